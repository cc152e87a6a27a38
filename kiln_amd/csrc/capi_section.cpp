// C ABI of the attention section over an encoder's states: rotary positions, cross-attention, MXFP4 quantisation and linear
// layers. Argument checks and dispatch; declarations and contracts: include/kiln_attn.h.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdlib.h>

#include <algorithm>

#include "../../include/kiln_attn.h"
#include "capi_util.hpp"
#include "internal.hpp"
#include "mxfp4.hpp"

using kiln::DT;
using namespace kiln::capi;

namespace {

bool dtype_ok(int d) { return d == KILN_F32 || d == KILN_F16 || d == KILN_BF16; }
size_t esize(int d) { return d == KILN_F32 ? 4 : 2; }
bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
// a row stride holds the row's columns (one row needs none)
bool ld_ok(int ld, long long cols, int T) { return T <= 1 || ld >= cols; }
constexpr int MAX_ROWS = 1 << 30;

// Windows of T rows of wx and wy bytes, lx and ly bytes apart, share none
bool apart(const void* x, long long lx, long long wx, const void* y, long long ly, long long wy, int T) {
    const long long bx = (long long)(intptr_t)x, by = (long long)(intptr_t)y;
    const long long ex = bx + (T - 1) * lx + wx, ey = by + (T - 1) * ly + wy;
    if (ex <= by || ey <= bx) return true;
    if (T == 1 || lx != ly) return false;
    // columns side by side in one row stride
    const long long d = ((by - bx) % lx + lx) % lx;
    return d >= wx && lx - d >= wy;
}

}  // namespace

extern "C" {

int kiln_rope_freqs(double* host_freqs, float* mscale, int rot, double theta, int scaling, double factor, double trained,
                    double slow, double fast) {
    if (!host_freqs || !mscale) return fail(KILN_EINVAL, "rope_freqs: null pointer");
    if (rot < 2 || rot % 2) return fail(KILN_EINVAL, "rope_freqs: rot %d must be even and positive", rot);
    if (scaling < KILN_ROPE_NONE || scaling > KILN_ROPE_BANDS) return fail(KILN_EINVAL, "rope_freqs: scaling %d", scaling);
    if (!(theta > 0) || !isfinite(theta) || !(factor >= 1) || !isfinite(factor))
        return fail(KILN_EINVAL, "rope_freqs: theta %g must be positive, factor %g at least 1", theta, factor);
    if (scaling == KILN_ROPE_NTK && rot == 2) return fail(KILN_EINVAL, "rope_freqs: NTK scaling needs rot > 2");
    const bool turns = scaling == KILN_ROPE_RAMP || scaling == KILN_ROPE_BANDS;
    if (turns && (!(trained > 0) || !isfinite(trained) || !(slow > 0) || !(fast > slow) || !isfinite(fast)))
        return fail(KILN_EINVAL, "rope_freqs: trained %g, slow %g, fast %g need trained > 0 and 0 < slow < fast", trained, slow, fast);
    if (scaling == KILN_ROPE_RAMP && !(theta > 1)) return fail(KILN_EINVAL, "rope_freqs: the ramp needs theta > 1");
    const double two_pi = 6.283185307179586477;
    const double base = scaling == KILN_ROPE_NTK ? theta * pow(factor, (double)rot / (rot - 2)) : theta;
    double lo = 0, hi = 0;
    if (scaling == KILN_ROPE_RAMP) {
        auto pair_of = [&](double n) { return rot * log(trained / (two_pi * n)) / (2 * log(theta)); };
        lo = std::max(floor(pair_of(fast)), 0.0);
        hi = std::min(ceil(pair_of(slow)), (double)(rot - 1));
    }
    for (int i = 0; i < rot / 2; i++) {
        double f = pow(base, -2.0 * i / rot);
        if (scaling == KILN_ROPE_LINEAR) f /= factor;
        if (turns) {
            const double stretched = scaling == KILN_ROPE_RAMP ? std::clamp((i - lo) / std::max(hi - lo, 0.001), 0.0, 1.0)
                                                               : 1 - std::clamp((trained * f / two_pi - slow) / (fast - slow), 0.0, 1.0);
            f = f / factor * stretched + f * (1 - stretched);
        }
        host_freqs[i] = f;
    }
    *mscale = scaling == KILN_ROPE_RAMP ? (float)(0.1 * log(factor) + 1) : 1.f;
    return KILN_OK;
}

int kiln_rope(void* y, int ldy, const void* x, int ldx, int dtype, int T, int H, int Dh, int rot, int interleaved, const int32_t* pos,
              int pos0, const double* freqs, float mscale, kiln_stream_t stream) {
    kiln::prof::Scope prof_("rope", (hipStream_t)stream);
    if (!dtype_ok(dtype)) return fail(KILN_EINVAL, "rope: dtype %d", dtype);
    if (T < 0 || H <= 0 || Dh <= 0 || rot < 2 || rot % 2 || rot > Dh)
        return fail(KILN_EINVAL, "rope: bad sizes T=%d H=%d Dh=%d rot=%d", T, H, Dh, rot);
    if (Dh > 1024 || H > 65535 || T > MAX_ROWS)
        return fail(KILN_EUNSUPPORTED, "rope: Dh=%d above 1024, H=%d above 65535 or T=%d above 2^30", Dh, H, T);
    if (!T) return KILN_OK;
    if (!x || !y || !freqs) return fail(KILN_EINVAL, "rope: null pointer");
    const long long W = (long long)H * Dh;
    if (!ld_ok(ldx, W, T) || !ld_ok(ldy, W, T)) return fail(KILN_EINVAL, "rope: row stride %d or %d below %lld", ldx, ldy, W);
    if (!aligned(x, esize(dtype)) || !aligned(y, esize(dtype)) || !aligned(freqs, 8) || !aligned(pos, 4))
        return fail(KILN_EUNSUPPORTED, "rope: a pointer is not aligned to its elements");
    const long long e = (long long)esize(dtype);
    if (!(x == y && (T == 1 || ldx == ldy)) && !apart(x, ldx * e, W * e, y, ldy * e, W * e, T)) return fail(KILN_EINVAL, "rope: x and y overlap");
    return hip_check(kiln::launch_rope(y, (size_t)(T == 1 ? W : ldy), x, (size_t)(T == 1 ? W : ldx), (DT)dtype, T, H, Dh, rot,
                                       interleaved != 0, pos, pos0, freqs, mscale, (hipStream_t)stream),
                     "rope launch");
}

size_t kiln_cross_attn_workspace_bytes(int B, int Tq, int Tk, int Hq, int Hkv, int Dh) {
    if (B <= 0 || Tq <= 0 || Tk <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || (Dh != 64 && Dh != 128)) return 0;
    if (Tk > MAX_ROWS || (long long)Tq * (Hq / Hkv) > MAX_ROWS) return 0;
    return kiln::cross_attn_workspace(B, Tq, Tk, Hq, Hkv, Dh);
}

int kiln_cross_attn_form(int B, int Tq, int Tk, int Hq, int Hkv, int Dh) {
    if (B <= 0 || Tq <= 0 || Tk < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || (Dh != 64 && Dh != 128)) return 0;
    if (Tk > MAX_ROWS || (long long)Tq * (Hq / Hkv) > MAX_ROWS) return 0;
    return kiln::cross_attn_form(B, Tq, Tk, Hq, Hkv, Dh);
}

int kiln_cross_attn(void* out, int ldo, long long bso, const void* q, int ldq, long long bsq, const void* k, int ldk, long long bsk,
                    const void* v, int ldv, long long bsv, int dtype, int B, int Tq, int Tk, int Hq, int Hkv, int Dh, float scale,
                    const int32_t* klen, const uint8_t* kmask, long long bsm, void* workspace, size_t ws_bytes, kiln_stream_t stream) {
    kiln::prof::Scope prof_("attention", (hipStream_t)stream);
    if (dtype != KILN_F16 && dtype != KILN_BF16) return fail(KILN_EINVAL, "cross_attn: dtype %d (fp16 or bf16)", dtype);
    if (B < 0 || Tq < 0 || Tk < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv)
        return fail(KILN_EINVAL, "cross_attn: bad sizes B=%d Tq=%d Tk=%d Hq=%d Hkv=%d", B, Tq, Tk, Hq, Hkv);
    if (Dh != 64 && Dh != 128) return fail(KILN_EUNSUPPORTED, "cross_attn: head size %d (64 or 128)", Dh);
    if (!(scale > 0.f) || !isfinite(scale * kiln::LOG2E))
        return fail(KILN_EINVAL, "cross_attn: scale %g must be positive, and finite times log2(e)", (double)scale);
    if (!B || !Tq) return KILN_OK;
    if (!out || !q || (Tk && (!k || !v))) return fail(KILN_EINVAL, "cross_attn: null pointer");
    const long long G = Hq / Hkv, rows = Tq * G;
    if (rows > MAX_ROWS || Tk > MAX_ROWS || (rows / 16 + 1) * B * Hkv > MAX_ROWS)
        return fail(KILN_EUNSUPPORTED, "cross_attn: too many rows or keys (B=%d Tq=%d Tk=%d)", B, Tq, Tk);
    const struct {
        const char* name;
        const void* p;
        int ld, T, H;
        long long bs;
    } ten[4] = {{"out", out, ldo, Tq, Hq, bso}, {"q", q, ldq, Tq, Hq, bsq}, {"k", k, ldk, Tk, Hkv, bsk}, {"v", v, ldv, Tk, Hkv, bsv}};
    for (const auto& t : ten) {
        if (!ld_ok(t.ld, (long long)t.H * Dh, t.T)) return fail(KILN_EINVAL, "cross_attn: %s row stride %d", t.name, t.ld);
        if (!aligned(t.p, 16) || (t.T > 1 && t.ld % 8) || (B > 1 && t.bs % 8) || (t.T > 1 && t.ld > (1 << 24)))
            return fail(KILN_EUNSUPPORTED, "cross_attn: %s rows not 16-byte aligned, or more than 2^24 elements apart", t.name);
    }
    if (!aligned(klen, 4)) return fail(KILN_EUNSUPPORTED, "cross_attn: klen not aligned");
    // items' outputs one behind the other, or side by side in rows that hold them all
    const long long W = (long long)Hq * Dh, abso = bso < 0 ? -bso : bso;
    if (B > 1 && abso < (Tq - 1) * (long long)ldo + W && (abso < W || ldo < (B - 1) * abso + W))
        return fail(KILN_EINVAL, "cross_attn: items' outputs overlap (bso %lld, ldo %d)", bso, ldo);
    if (workspace && !aligned(workspace, 16)) return fail(KILN_EUNSUPPORTED, "cross_attn: workspace not 16-byte aligned");
    kiln::CrossLaunch c{};
    c.out = out;
    c.q = q;
    c.k = k;
    c.v = v;
    c.ldo = (size_t)(Tq == 1 ? 0 : ldo);
    c.ldq = (size_t)(Tq == 1 ? 0 : ldq);
    c.ldk = (size_t)(Tk <= 1 ? Dh : ldk);
    c.ldv = (size_t)(Tk <= 1 ? Dh : ldv);
    c.bso = bso;
    c.bsq = bsq;
    c.bsk = bsk;
    c.bsv = bsv;
    c.dt = (DT)dtype;
    c.B = B;
    c.Tq = Tq;
    c.Tk = Tk;
    c.Hq = Hq;
    c.Hkv = Hkv;
    c.Dh = Dh;
    c.scale = scale;
    c.klen = klen;
    c.kmask = kmask;
    c.bsm = bsm;
    c.ws = workspace;
    c.ws_bytes = ws_bytes;
    return hip_check(kiln::launch_cross_attn(c, (hipStream_t)stream), "cross_attn launch");
}

// rows x cols of an MXFP4 matrix: KILN_OK, or the refusal
static int mx_sizes(const char* what, int rows, int cols) {
    if (rows < 0 || cols <= 0) return fail(KILN_EINVAL, "%s: bad sizes rows=%d cols=%d", what, rows, cols);
    if (cols % kiln::MXB) return fail(KILN_EUNSUPPORTED, "%s: cols %d must be a multiple of 32", what, cols);
    if (rows > MAX_ROWS || cols > MAX_ROWS) return fail(KILN_EUNSUPPORTED, "%s: more than 2^30 rows or columns", what);
    return KILN_OK;
}

int kiln_mxfp4_quantize(uint8_t* codes, uint8_t* scales, const void* x, int dtype, int ldx, int rows, int cols, kiln_stream_t stream) {
    kiln::prof::Scope prof_("mxfp4", (hipStream_t)stream);
    if (!dtype_ok(dtype)) return fail(KILN_EINVAL, "mxfp4_quantize: dtype %d", dtype);
    if (int r = mx_sizes("mxfp4_quantize", rows, cols)) return r;
    if (!rows) return KILN_OK;
    if (!codes || !scales || !x) return fail(KILN_EINVAL, "mxfp4_quantize: null pointer");
    if (!ld_ok(ldx, cols, rows)) return fail(KILN_EINVAL, "mxfp4_quantize: row stride %d below %d", ldx, cols);
    if (!aligned(codes, 16) || !aligned(x, esize(dtype))) return fail(KILN_EUNSUPPORTED, "mxfp4_quantize: alignment");
    return hip_check(kiln::launch_mx_quantize(codes, scales, x, (DT)dtype, (size_t)ldx, rows, cols, (hipStream_t)stream), "mxfp4_quantize launch");
}

int kiln_mxfp4_dequantize(void* y, int dtype, int ldy, const uint8_t* codes, const uint8_t* scales, int rows, int cols,
                          kiln_stream_t stream) {
    kiln::prof::Scope prof_("mxfp4", (hipStream_t)stream);
    if (!dtype_ok(dtype)) return fail(KILN_EINVAL, "mxfp4_dequantize: dtype %d", dtype);
    if (int r = mx_sizes("mxfp4_dequantize", rows, cols)) return r;
    if (!rows) return KILN_OK;
    if (!codes || !scales || !y) return fail(KILN_EINVAL, "mxfp4_dequantize: null pointer");
    if (!ld_ok(ldy, cols, rows)) return fail(KILN_EINVAL, "mxfp4_dequantize: row stride %d below %d", ldy, cols);
    if (!aligned(codes, 16) || !aligned(y, esize(dtype))) return fail(KILN_EUNSUPPORTED, "mxfp4_dequantize: alignment");
    return hip_check(kiln::launch_mx_dequantize(y, (DT)dtype, (size_t)ldy, codes, scales, rows, cols, (hipStream_t)stream),
                     "mxfp4_dequantize launch");
}

size_t kiln_linear_mxfp4_weight_bytes(int rows, int cols) {
    if (rows <= 0 || cols <= 0 || cols % kiln::MXB || rows > MAX_ROWS || cols > MAX_ROWS) return 0;
    return kiln::mx_code_bytes(rows, cols) + kiln::mx_scale_bytes(rows, cols);
}

int kiln_linear_mxfp4_prepare_weight(uint8_t* wp, const uint8_t* codes, const uint8_t* scales, int rows, int cols, kiln_stream_t stream) {
    kiln::prof::Scope prof_("mxfp4", (hipStream_t)stream);
    if (int r = mx_sizes("linear_mxfp4_prepare_weight", rows, cols)) return r;
    if (!rows) return fail(KILN_EINVAL, "linear_mxfp4_prepare_weight: no rows");
    if (!wp || !codes || !scales) return fail(KILN_EINVAL, "linear_mxfp4_prepare_weight: null pointer");
    if (!aligned(wp, 16) || !aligned(codes, 16)) return fail(KILN_EUNSUPPORTED, "linear_mxfp4_prepare_weight: not 16-byte aligned");
    return hip_check(kiln::launch_mx_pack(wp, codes, scales, rows, cols, (hipStream_t)stream), "linear_mxfp4_prepare_weight launch");
}

size_t kiln_linear_mxfp4_workspace_bytes(int T, int rows, int cols) {
    if (T <= 0 || !kiln_linear_mxfp4_weight_bytes(rows, cols) || T > MAX_ROWS) return 0;
    return kiln::linear_mx_workspace(T, rows, cols);
}

int kiln_linear_mxfp4_tile(int T, int rows, int cols) {
    if (T <= 0 || !kiln_linear_mxfp4_weight_bytes(rows, cols) || T > MAX_ROWS) return 0;
    return kiln::linear_mx_tile(T, rows, cols);
}

int kiln_linear_mxfp4(void* y, int ldy, const void* x, int dtype, int ldx, int T, const uint8_t* wp, int rows, int cols, int epi,
                      const float* gate, float beta, void* workspace, size_t ws_bytes, kiln_stream_t stream) {
    kiln::prof::Scope prof_("gemm_mxfp4", (hipStream_t)stream);
    if (!dtype_ok(dtype)) return fail(KILN_EINVAL, "linear_mxfp4: dtype %d", dtype);
    if (epi < KILN_EPI_F32 || epi > KILN_EPI_RESID) return fail(KILN_EINVAL, "linear_mxfp4: epilogue %d", epi);
    if (int r = mx_sizes("linear_mxfp4", rows, cols)) return r;
    if (T < 0 || !rows) return fail(KILN_EINVAL, "linear_mxfp4: bad sizes T=%d rows=%d", T, rows);
    if (!T) return KILN_OK;
    if ((long long)(T / 64 + 1) * (rows / 64 + 1) > MAX_ROWS)
        return fail(KILN_EUNSUPPORTED, "linear_mxfp4: T=%d x rows=%d above 2^42 outputs", T, rows);
    if (!y || !x || !wp) return fail(KILN_EINVAL, "linear_mxfp4: null pointer");
    if (!ld_ok(ldx, cols, T) || !ld_ok(ldy, rows, T)) return fail(KILN_EINVAL, "linear_mxfp4: row stride (ldx %d, ldy %d)", ldx, ldy);
    const size_t ye = epi == KILN_EPI_F32 || epi == KILN_EPI_RESID ? 4 : 2;
    if (!aligned(wp, 16) || !aligned(x, esize(dtype)) || !aligned(y, ye) || !aligned(gate, 4) || !aligned(workspace, 16))
        return fail(KILN_EUNSUPPORTED, "linear_mxfp4: alignment");
    // in place the few-row form would read what other workgroups have written
    const long long xe = (long long)esize(dtype);
    if (!apart(x, ldx * xe, cols * xe, y, ldy * (long long)ye, rows * (long long)ye, T))
        return fail(KILN_EINVAL, "linear_mxfp4: x and y overlap");
    const size_t need = kiln::linear_mx_workspace(T, rows, cols);
    if (need && (!workspace || ws_bytes < need))
        return fail(KILN_ENOMEM, "linear_mxfp4: workspace %zu bytes < %zu needed", workspace ? ws_bytes : (size_t)0, need);
    return hip_check(kiln::launch_linear_mx(y, (size_t)ldy, x, (DT)dtype, (size_t)ldx, T, wp, rows, cols, epi, gate, beta,
                                            static_cast<uint8_t*>(workspace), (hipStream_t)stream),
                     "linear_mxfp4 launch");
}

}  // extern "C"
