// The attention section over an encoder's states through the C++ host mirror: MXFP4 projections, rotary positions,
// cross-attention and the gated MXFP4 output projection of one item, each stage against double precision on the host from the
// previous stage's own output. Exit status 1 if a stage leaves its bound. The refusals (throwing wrappers) run first.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>
#include <vector>

#include "../../kiln_amd/host/kiln_gpu.hpp"

#define CK(x)                                                                              \
    do {                                                                                   \
        hipError_t e_ = (x);                                                               \
        if (e_ != hipSuccess) {                                                            \
            fprintf(stderr, "%s:%d %s: %s\n", __FILE__, __LINE__, #x, hipGetErrorString(e_)); \
            std::exit(2);                                                                  \
        }                                                                                  \
    } while (0)

typedef _Float16 f16;
template <class T>
struct Dev {
    T* p = nullptr;
    size_t n;
    explicit Dev(size_t n_) : n(n_) { CK(hipMalloc(&p, n * sizeof(T))); }
    explicit Dev(const std::vector<T>& v) : Dev(v.size()) { CK(hipMemcpy(p, v.data(), n * sizeof(T), hipMemcpyHostToDevice)); }
    ~Dev() { (void)hipFree(p); }
    Dev(const Dev&) = delete;
    std::vector<T> host() const {
        std::vector<T> v(n);
        CK(hipMemcpy(v.data(), p, n * sizeof(T), hipMemcpyDeviceToHost));
        return v;
    }
};

static const double GRID[8] = {0, 0.5, 1, 1.5, 2, 3, 4, 6};
// the values that codes and scales stand for
static std::vector<double> values(const std::vector<uint8_t>& c, const std::vector<uint8_t>& s, int rows, int cols) {
    std::vector<double> v((size_t)rows * cols);
    for (size_t i = 0; i < v.size(); i++) {
        const int code = c[i / 2] >> (4 * (i & 1)) & 15;
        v[i] = (code & 8 ? -1.0 : 1.0) * GRID[code & 7] * std::ldexp(1.0, (int)s[i / 32] - 127);
    }
    return v;
}
struct Layer {
    int rows, cols;
    std::vector<double> w;
    kiln::Mxfp4Weight* W;
};
static Layer layer(std::mt19937& rng, int rows, int cols) {
    std::normal_distribution<float> nd(0.f, 1.f / std::sqrt((float)cols));
    std::vector<float> w((size_t)rows * cols);
    for (auto& x : w) x = nd(rng);
    Dev<float> d(w);
    Dev<uint8_t> codes(w.size() / 2), scales(w.size() / 32);
    kiln::mxfp4_quantize(codes.p, scales.p, d.p, KILN_F32, cols, rows, cols);
    Layer l{rows, cols, {}, new kiln::Mxfp4Weight(codes.p, scales.p, rows, cols)};
    CK(hipDeviceSynchronize());
    l.w = values(codes.host(), scales.host(), rows, cols);
    return l;
}
static std::vector<double> quantised(const void* x, int dtype, int rows, int cols) {
    Dev<uint8_t> codes((size_t)rows * cols / 2), scales((size_t)rows * cols / 32);
    kiln::mxfp4_quantize(codes.p, scales.p, x, dtype, cols, rows, cols);
    CK(hipDeviceSynchronize());
    return values(codes.host(), scales.host(), rows, cols);
}
static int bad = 0;
static void stage(const char* name, double worst) {
    printf("%-28s worst error / bound %.3f\n", name, worst);
    if (!(worst <= 1.0)) bad = 1;
}
// y = x W^T in fp16 against double: K / 128 + 8 roundings of 2^-23 of the magnitudes, then fp16's
static double project(const std::vector<f16>& y, const std::vector<double>& x, const Layer& l, int T) {
    double worst = 0;
    for (int t = 0; t < T; t++)
        for (int n = 0; n < l.rows; n++) {
            double a = 0, m = 0;
            for (int k = 0; k < l.cols; k++) {
                const double p = x[(size_t)t * l.cols + k] * l.w[(size_t)n * l.cols + k];
                a += p;
                m += std::fabs(p);
            }
            const double tol = (l.cols / 128 + 8) * std::ldexp(m, -23);
            worst = std::max(worst, std::fabs((double)y[(size_t)t * l.rows + n] - a) / (tol + std::ldexp(std::fabs(a) + tol, -11) + 0x1p-25));
        }
    return worst;
}

int main() {
    int thrown = 0;
    try { kiln::RopeFreqs f(3); } catch (const std::runtime_error&) { thrown++; }
    try { kiln::Mxfp4Weight w(nullptr, nullptr, 8, 40); } catch (const std::runtime_error&) { thrown++; }
    try { kiln::cross_attn(nullptr, 96, nullptr, 96, nullptr, 96, nullptr, 96, KILN_F16, 1, 4, 4, 1, 1, 96, 0.1f); } catch (const std::runtime_error&) { thrown++; }
    if (thrown != 3) {
        printf("refusals: %d of 3 threw\n", thrown);
        return 1;
    }

    const int T = 70, S = 45, H = 4, Hkv = 2, Dh = 64, D = H * Dh, KV = Hkv * Dh, TEXT = 96, real = 41;
    std::mt19937 rng(11);
    std::normal_distribution<float> nd(0.f, 1.f);
    std::vector<f16> x((size_t)T * D), e((size_t)S * TEXT);
    for (auto& v : x) v = (f16)nd(rng);
    for (auto& v : e) v = (f16)nd(rng);
    Layer lq = layer(rng, D, D), lkv = layer(rng, 2 * KV, TEXT), lo = layer(rng, D, D);
    Dev<f16> dx(x), de(e), q((size_t)T * D), kv((size_t)S * 2 * KV), at((size_t)T * D);
    std::vector<float> gate(D), y0((size_t)T * D);
    for (auto& v : gate) v = nd(rng);
    for (auto& v : y0) v = nd(rng);
    Dev<float> dgate(gate), y(y0);
    Dev<int32_t> klen(std::vector<int32_t>{real});
    const size_t wsn = std::max({kiln_linear_mxfp4_workspace_bytes(T, D, D), kiln_linear_mxfp4_workspace_bytes(S, 2 * KV, TEXT),
                                 kiln_cross_attn_workspace_bytes(1, T, S, H, Hkv, Dh), (size_t)16});
    Dev<uint8_t> ws(wsn);

    kiln::linear_mxfp4(q.p, D, dx.p, KILN_F16, D, T, *lq.W, kiln::Epi16::F16, nullptr, 0.f, ws.p, wsn);
    kiln::linear_mxfp4(kv.p, 2 * KV, de.p, KILN_F16, TEXT, S, *lkv.W, kiln::Epi16::F16, nullptr, 0.f, ws.p, wsn);
    CK(hipDeviceSynchronize());
    const auto hq = q.host(), hkv = kv.host();
    stage("MXFP4 query projection", project(hq, quantised(dx.p, KILN_F16, T, D), lq, T));
    stage("MXFP4 key/value projection", project(hkv, quantised(de.p, KILN_F16, S, TEXT), lkv, S));

    kiln::RopeFreqs fr(Dh, 10000.0, KILN_ROPE_BANDS, 4.0, 32.0, 1.0, 4.0);
    kiln::rope(q.p, D, q.p, D, KILN_F16, T, H, Dh, fr, false, nullptr, 500);
    kiln::rope(kv.p, 2 * KV, kv.p, 2 * KV, KILN_F16, S, Hkv, Dh, fr, false, nullptr, 0);  // the keys; the values stay
    CK(hipDeviceSynchronize());
    const auto rq = q.host(), rkv = kv.host();
    double worst = 0;
    for (int t = 0; t < T; t++)
        for (int h = 0; h < H; h++)
            for (int i = 0; i < Dh / 2; i++) {
                const double a = (500.0 + t) * fr.host()[i], c = std::cos(a), s = std::sin(a);
                const size_t at0 = (size_t)t * D + h * Dh + i, at1 = at0 + Dh / 2;
                const double u = (double)hq[at0], v = (double)hq[at1], m = (std::fabs(u) + std::fabs(v)) * 9 * 0x1p-24;
                worst = std::max(worst, std::fabs((double)rq[at0] - (u * c - v * s)) / (m + std::ldexp(std::fabs(u * c - v * s) + m, -11) + 0x1p-25));
                worst = std::max(worst, std::fabs((double)rq[at1] - (v * c + u * s)) / (m + std::ldexp(std::fabs(v * c + u * s) + m, -11) + 0x1p-25));
            }
    for (int t = 0; t < S; t++)
        if (std::memcmp(&rkv[(size_t)t * 2 * KV + KV], &hkv[(size_t)t * 2 * KV + KV], KV * 2)) worst = 2;  // values untouched
    stage("rotary positions", worst);

    kiln::cross_attn(at.p, D, q.p, D, kv.p, 2 * KV, kv.p + KV, 2 * KV, KILN_F16, 1, T, S, H, Hkv, Dh, 0.125f, klen.p, nullptr, ws.p, wsn);
    CK(hipDeviceSynchronize());
    const auto ha = at.host();
    worst = 0;
    for (int t = 0; t < T; t++)
        for (int h = 0; h < H; h++) {
            double p[S], sc[S], smax = -INFINITY, smag = 0, l = 0;
            for (int j = 0; j < real; j++) {
                double a = 0, m = 0;
                for (int d = 0; d < Dh; d++) {
                    const double z = (double)rq[(size_t)t * D + h * Dh + d] * (double)rkv[(size_t)j * 2 * KV + h * Hkv / H * Dh + d];
                    a += z;
                    m += std::fabs(z);
                }
                sc[j] = 0.125 * a;
                smax = std::max(smax, sc[j]);
                smag = std::max(smag, 0.125 * m);
            }
            for (int j = 0; j < real; j++) l += p[j] = std::exp(sc[j] - smax);
            for (int d = 0; d < Dh; d++) {
                double o = 0, w = 0, vs = 0;
                for (int j = 0; j < real; j++) {
                    const double v = (double)rkv[(size_t)j * 2 * KV + KV + h * Hkv / H * Dh + d];
                    o += p[j] / l * v;
                    w += p[j] / l * std::fabs(v);
                    vs += std::fabs(v);
                }
                const double tol = (0x1p-11 + 4 * 0x1p-22 * 3 * smag + 80 * 0x1p-24 + 0x1p-21) * w + 0x1p-25 * vs;
                worst = std::max(worst, std::fabs((double)ha[(size_t)t * D + h * Dh + d] - o) / (tol + std::ldexp(std::fabs(o) + tol, -11) + 0x1p-25));
            }
        }
    stage("cross-attention", worst);

    kiln::linear_mxfp4(y.p, D, at.p, KILN_F16, D, T, *lo.W, kiln::Epi16::Resid, dgate.p, 0.f, ws.p, wsn);
    CK(hipDeviceSynchronize());
    const auto hy = y.host();
    const auto xa = quantised(at.p, KILN_F16, T, D);
    worst = 0;
    for (int t = 0; t < T; t++)
        for (int n = 0; n < D; n++) {
            double a = 0, m = 0;
            for (int k = 0; k < D; k++) {
                const double z = xa[(size_t)t * D + k] * lo.w[(size_t)n * D + k];
                a += z;
                m += std::fabs(z);
            }
            const double g = gate[n], want = (double)y0[(size_t)t * D + n] + g * a;
            const double tol = (D / 128 + 8) * std::ldexp(m, -23) * std::fabs(g) + std::ldexp(std::fabs(g * a), -23) + std::ldexp(std::fabs(want), -24);
            worst = std::max(worst, std::fabs((double)hy[(size_t)t * D + n] - want) / (tol + 1e-30));
        }
    stage("gated MXFP4 projection", worst);
    delete lq.W;
    delete lkv.W;
    delete lo.W;
    return bad;
}
