// A text encoder's layer through the C++ host mirror: residual + RMS norm to MXFP8, the stacked projection, causal attention over packed
// prompts behind a shared prefix, the output projection onto the residual stream, each stage against double precision on the host from the
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
// the values that MXFP4 codes and scales stand for
static std::vector<double> values(const std::vector<uint8_t>& c, const std::vector<uint8_t>& s, int rows, int cols) {
    std::vector<double> v((size_t)rows * cols);
    for (size_t i = 0; i < v.size(); i++) {
        const int code = c[i / 2] >> (4 * (i & 1)) & 15;
        v[i] = (code & 8 ? -1.0 : 1.0) * GRID[code & 7] * std::ldexp(1.0, (int)s[i / 32] - 127);
    }
    return v;
}
// .. and MXFP8's
static double e4m3(int c) {
    const int e = c >> 3 & 15, m = c & 7;
    const double v = e ? std::ldexp(8.0 + m, e - 10) : std::ldexp((double)m, -9);
    return c & 128 ? -v : v;
}
static std::vector<double> values8(const std::vector<uint8_t>& c, const std::vector<uint8_t>& s) {
    std::vector<double> v(c.size());
    for (size_t i = 0; i < v.size(); i++) v[i] = e4m3(c[i]) * std::ldexp(1.0, (int)s[i / 32] - 127);
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
static int bad = 0;
static void stage(const char* name, double worst) {
    printf("%-28s worst error / bound %.3f\n", name, worst);
    if (!(worst <= 1.0)) bad = 1;
}

int main() {
    int thrown = 0;
    kiln::PromptBatch none{1, 4, 5, nullptr};
    try { kiln::prompt_attn((void*)64, 96, (void*)6400, 96, (void*)12800, 96, (void*)25600, 96, KILN_F16, none, 1, 1, 96, 0.1f); } catch (const std::runtime_error&) { thrown++; }
    try { kiln::add_rmsnorm(nullptr, KILN_F16, nullptr, nullptr, KILN_F16, nullptr, KILN_F32, nullptr, 2, 40000, 1e-6f); } catch (const std::runtime_error&) { thrown++; }
    try { kiln::mxfp8_quantize(nullptr, nullptr, nullptr, KILN_F16, 40, 2, 40); } catch (const std::runtime_error&) { thrown++; }
    if (thrown != 3) {
        printf("refusals: %d of 3 threw\n", thrown);
        return 1;
    }

    const int H = 4, Hkv = 2, Dh = 64, D = H * Dh, KV = Hkv * Dh, W = D + 2 * KV, P = 37, B = 3;
    const std::vector<int32_t> starts{0, 40, 41, 70};
    const int T = starts[B];
    const float eps = 1e-6f, scale = 0.125f;
    std::mt19937 rng(12);
    std::normal_distribution<float> nd(0.f, 1.f);
    std::vector<f16> x((size_t)T * D), pk((size_t)P * KV), pv((size_t)P * KV);
    std::vector<float> res((size_t)T * D);
    std::vector<uint16_t> w(D);
    for (auto& v : x) v = (f16)nd(rng);
    for (auto& v : pk) v = (f16)nd(rng);
    for (auto& v : pv) v = (f16)nd(rng);
    for (auto& v : res) v = 2 * nd(rng);
    for (auto& v : w) {
        const float f = 1 + nd(rng) / 4;
        uint32_t b;
        std::memcpy(&b, &f, 4);
        v = (uint16_t)(b >> 16);
    }
    Layer lqkv = layer(rng, W, D), lo = layer(rng, D, D);
    Dev<f16> dx(x), qkv((size_t)T * W), at((size_t)T * D), dpk(pk), dpv(pv);
    Dev<float> dres(res);
    Dev<uint16_t> dw(w);
    Dev<uint8_t> codes((size_t)T * D), scales((size_t)T * D / 32);
    Dev<int32_t> ds(starts);
    Dev<uint8_t> ws(std::max<size_t>(kiln_prompt_attn_workspace_bytes(B, T, T, P, H, Hkv, Dh), 16));

    kiln::add_rmsnorm_mxfp8(codes.p, scales.p, dres.p, dx.p, KILN_F16, dres.p, KILN_F32, dw.p, T, D, eps);
    CK(hipDeviceSynchronize());
    const auto h = dres.host();
    const auto n8 = values8(codes.host(), scales.host());
    double worst = 0;
    for (int t = 0; t < T; t++) {
        double ss = 0;
        for (int i = 0; i < D; i++) ss += std::pow((double)x[t * D + i] + res[t * D + i], 2);
        const double r = 1 / std::sqrt(ss / D + eps);
        for (int b = 0; b < D / 32; b++) {
            double y[32], top = 0;
            for (int i = 0; i < 32; i++) {
                const size_t j = (size_t)t * D + b * 32 + i;
                const double s = (double)x[j] + res[j];
                uint32_t bits = (uint32_t)w[b * 32 + i] << 16;
                float f;
                std::memcpy(&f, &bits, 4);
                y[i] = s * r * f;
                top = std::max(top, std::fabs(y[i]));
                worst = std::max(worst, std::fabs((double)h[j] - s) / (std::ldexp(std::fabs(s), -24) + 1e-30));
            }
            // half a step of a code: 2^-4 of a value's power of two, at least 2^-10 of the scale's, which is at most top / 224
            for (int i = 0; i < 32; i++)
                worst = std::max(worst, std::fabs(n8[(size_t)t * D + b * 32 + i] - y[i]) / (std::fabs(y[i]) * (1 / 16. + 1e-5) + std::ldexp(top / 224, -10) * 1.001));
        }
    }
    stage("residual and norm to MXFP8", worst);

    kiln::linear_mxfp8(qkv.p, W, codes.p, scales.p, T, *lqkv.W, kiln::Epi16::F16);
    CK(hipDeviceSynchronize());
    const auto hq = qkv.host();
    worst = 0;
    for (int t = 0; t < T; t++)
        for (int n = 0; n < W; n++) {
            double a = 0, m = 0;
            for (int k = 0; k < D; k++) {
                const double p = n8[(size_t)t * D + k] * lqkv.w[(size_t)n * D + k];
                a += p;
                m += std::fabs(p);
            }
            const double tol = (D * 0x1p-24 + 7 * 0x1p-13) * m;  // of eight products seven are cut 13 bits below the largest
            worst = std::max(worst, std::fabs((double)hq[(size_t)t * W + n] - a) / (tol + std::ldexp(std::fabs(a) + tol, -11) + 0x1p-25));
        }
    stage("MXFP8 projection", worst);

    kiln::PromptBatch batch{B, T, T, ds.p};
    batch.pk = dpk.p;
    batch.pv = dpv.p;
    batch.ldpk = batch.ldpv = KV;
    batch.P = P;
    kiln::prompt_attn(at.p, D, qkv.p, W, qkv.p + D, W, qkv.p + D + KV, W, KILN_F16, batch, H, Hkv, Dh, scale, ws.p, ws.n);
    CK(hipDeviceSynchronize());
    const auto ha = at.host();
    worst = 0;
    for (int s = 0; s < B; s++)
        for (int t = starts[s]; t < starts[s + 1]; t++)
            for (int hd = 0; hd < H; hd++) {
                const int kv = hd * Hkv / H, n = P + t - starts[s] + 1;
                auto key = [&](int j, int d) { return j < P ? (double)pk[(size_t)j * KV + kv * Dh + d] : (double)hq[(size_t)(starts[s] + j - P) * W + D + kv * Dh + d]; };
                auto val = [&](int j, int d) { return j < P ? (double)pv[(size_t)j * KV + kv * Dh + d] : (double)hq[(size_t)(starts[s] + j - P) * W + D + KV + kv * Dh + d]; };
                std::vector<double> p(n);
                double smax = -INFINITY, smag = 0, l = 0;
                for (int j = 0; j < n; j++) {
                    double a = 0, m = 0;
                    for (int d = 0; d < Dh; d++) {
                        const double z = (double)hq[(size_t)t * W + hd * Dh + d] * key(j, d);
                        a += z;
                        m += std::fabs(z);
                    }
                    p[j] = scale * a;
                    smax = std::max(smax, p[j]);
                    smag = std::max(smag, scale * m);
                }
                for (auto& z : p) l += z = std::exp(z - smax);
                for (int d = 0; d < Dh; d++) {
                    double o = 0, wm = 0, vs = 0;
                    for (int j = 0; j < n; j++) {
                        o += p[j] / l * val(j, d);
                        wm += p[j] / l * std::fabs(val(j, d));
                        vs += std::fabs(val(j, d));
                    }
                    const double tol = (0x1p-11 + 4 * 0x1p-22 * 3 * smag + 80 * 0x1p-24 + 0x1p-21) * wm + 0x1p-32 * vs;
                    worst = std::max(worst, std::fabs((double)ha[(size_t)t * D + hd * Dh + d] - o) / (tol + std::ldexp(std::fabs(o) + tol, -11) + 0x1p-25));
                }
            }
    stage("causal attention", worst);

    kiln::mxfp8_quantize(codes.p, scales.p, at.p, KILN_F16, D, T, D);
    kiln::linear_mxfp8(dres.p, D, codes.p, scales.p, T, *lo.W, kiln::Epi16::Resid);
    CK(hipDeviceSynchronize());
    const auto hy = dres.host();
    const auto a8 = values8(codes.host(), scales.host());
    worst = 0;
    for (int t = 0; t < T; t++)
        for (int n = 0; n < D; n++) {
            double a = 0, m = 0;
            for (int k = 0; k < D; k++) {
                const double z = a8[(size_t)t * D + k] * lo.w[(size_t)n * D + k];
                a += z;
                m += std::fabs(z);
            }
            const double want = (double)h[(size_t)t * D + n] + a;
            worst = std::max(worst, std::fabs((double)hy[(size_t)t * D + n] - want) / (D * 0x1p-24 * m + 0x1p-17 * m + std::ldexp(std::fabs(want) + std::fabs(a), -23) + 1e-30));
        }
    stage("output onto the residual", worst);
    delete lqkv.W;
    delete lo.W;
    return bad;
}
