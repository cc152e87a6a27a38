// C ABI of a text encoder's layer: causal attention over packed sequences, the residual's addition with the RMS norm, MXFP8 rows and
// linear layers on them. Argument checks and dispatch; declarations and contracts: include/kiln_attn.h.
#include <hip/hip_runtime.h>
#include <math.h>

#include "../../include/kiln_attn.h"
#include "capi_util.hpp"
#include "internal.hpp"
#include "mxfp4.hpp"

using kiln::DT;
using namespace kiln::capi;

extern "C" {

constexpr int MAX_SEQS = 1 << 14;  // each workgroup goes over all of them for its place

// sizes that kiln_prompt_attn takes
static bool prompt_sizes(int B, int Tq, int Tk, int P, int Hq, int Hkv, int Dh) {
    if (B <= 0 || B > MAX_SEQS || Tq <= 0 || Tk < 0 || P < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || (Dh != 64 && Dh != 128)) return false;
    const long long rows = (long long)Tq * (Hq / Hkv);
    return rows <= MAX_ROWS && Tk <= MAX_ROWS && P <= MAX_ROWS && (rows / 16 + B) * Hkv < 1 << 24;
}

size_t kiln_prompt_attn_workspace_bytes(int B, int Tq, int Tk, int P, int Hq, int Hkv, int Dh) {
    return prompt_sizes(B, Tq, Tk, P, Hq, Hkv, Dh) ? kiln::prompt_attn_workspace(B, Tq, Tk, P, Hq, Hkv, Dh) : 0;
}

int kiln_prompt_attn_form(int B, int Tq, int Tk, int P, int Hq, int Hkv, int Dh) {
    return prompt_sizes(B, Tq, Tk, P, Hq, Hkv, Dh) ? kiln::prompt_attn_form(B, Tq, Tk, P, Hq, Hkv, Dh) : 0;
}

int kiln_prompt_attn(void* out, int ldo, const void* q, int ldq, const void* k, int ldk, const void* v, int ldv, int dtype, int Tq, int Tk,
                     int Hq, int Hkv, int Dh, float scale, int B, const int32_t* q_start, const int32_t* k_start, const int32_t* k_len,
                     const void* pk, int ldpk, const void* pv, int ldpv, int P, void* workspace, size_t ws_bytes, kiln_stream_t stream) {
    kiln::prof::Scope prof_("attention", (hipStream_t)stream);
    if (dtype != KILN_F16 && dtype != KILN_BF16) return fail(KILN_EINVAL, "prompt_attn: dtype %d (fp16 or bf16)", dtype);
    if (B < 0 || Tq < 0 || Tk < 0 || P < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv)
        return fail(KILN_EINVAL, "prompt_attn: bad sizes B=%d Tq=%d Tk=%d P=%d Hq=%d Hkv=%d", B, Tq, Tk, P, Hq, Hkv);
    if (Dh != 64 && Dh != 128) return fail(KILN_EUNSUPPORTED, "prompt_attn: head size %d (64 or 128)", Dh);
    if (!(scale > 0.f) || !isfinite(scale * kiln::LOG2E))
        return fail(KILN_EINVAL, "prompt_attn: scale %g must be positive, and finite times log2(e)", (double)scale);
    if (!k_start != !k_len) return fail(KILN_EINVAL, "prompt_attn: k_start and k_len go together");
    if (!B || !Tq) return KILN_OK;
    if (!q_start && B != 1) return fail(KILN_EINVAL, "prompt_attn: %d sequences without q_start", B);
    if (!k_start && Tk != Tq) return fail(KILN_EINVAL, "prompt_attn: keys of the queries' own rows, but Tq=%d, Tk=%d", Tq, Tk);
    if (!out || !q || (Tk && (!k || !v)) || (P && (!pk || !pv))) return fail(KILN_EINVAL, "prompt_attn: null pointer");
    if (!prompt_sizes(B, Tq, Tk, P, Hq, Hkv, Dh))
        return fail(KILN_EUNSUPPORTED, "prompt_attn: too many rows, keys or sequences (B=%d Tq=%d Tk=%d P=%d)", B, Tq, Tk, P);
    const struct {
        const char* name;
        const void* p;
        int ld, T, H;
    } ten[6] = {{"out", out, ldo, Tq, Hq}, {"q", q, ldq, Tq, Hq}, {"k", k, ldk, Tk, Hkv}, {"v", v, ldv, Tk, Hkv}, {"prefix k", pk, ldpk, P, Hkv}, {"prefix v", pv, ldpv, P, Hkv}};
    for (const auto& t : ten) {
        if (!t.T) continue;
        if (!ld_ok(t.ld, (long long)t.H * Dh, t.T)) return fail(KILN_EINVAL, "prompt_attn: %s row stride %d", t.name, t.ld);
        if (!aligned(t.p, 16) || (t.T > 1 && (t.ld % 8 || t.ld > (1 << 24))))
            return fail(KILN_EUNSUPPORTED, "prompt_attn: %s rows not 16-byte aligned, or more than 2^24 elements apart", t.name);
        if (t.p != out && !apart(out, ldo * 2LL, Hq * 2LL * Dh, Tq, t.p, t.ld * 2LL, t.H * 2LL * Dh, t.T))
            return fail(KILN_EINVAL, "prompt_attn: out and %s overlap", t.name);
        if (t.p == out && &t != ten) return fail(KILN_EINVAL, "prompt_attn: out and %s overlap", t.name);
    }
    if (!aligned(q_start, 4) || !aligned(k_start, 4) || !aligned(k_len, 4)) return fail(KILN_EUNSUPPORTED, "prompt_attn: starts or lengths not aligned");
    if (workspace && !aligned(workspace, 16)) return fail(KILN_EUNSUPPORTED, "prompt_attn: workspace not 16-byte aligned");
    kiln::PromptLaunch c{};
    c.out = out;
    c.q = q;
    c.k = k;
    c.v = v;
    c.pk = pk;
    c.pv = pv;
    c.ldo = (size_t)(Tq == 1 ? 0 : ldo);
    c.ldq = (size_t)(Tq == 1 ? 0 : ldq);
    c.ldk = (size_t)(Tk <= 1 ? Dh : ldk);
    c.ldv = (size_t)(Tk <= 1 ? Dh : ldv);
    c.ldpk = (size_t)(P <= 1 ? Dh : ldpk);
    c.ldpv = (size_t)(P <= 1 ? Dh : ldpv);
    c.dt = (DT)dtype;
    c.B = B;
    c.Tq = Tq;
    c.Tk = Tk;
    c.P = P;
    c.Hq = Hq;
    c.Hkv = Hkv;
    c.Dh = Dh;
    c.scale = scale;
    c.q_start = q_start;
    c.k_start = k_start;
    c.k_len = k_len;
    c.ws = workspace;
    c.ws_bytes = ws_bytes;
    return hip_check(kiln::launch_prompt_attn(c, (hipStream_t)stream), "prompt_attn launch");
}

// both norms: y in ydt (scales null), or MXFP8 codes
static int add_rmsnorm(const char* what, void* y, int ydt, int ldy, uint8_t* scales, void* h, int ldh, const void* x, int xdt, int ldx,
                       const void* res, int rdt, int ldr, const uint16_t* w, int rows, int dim, float eps, kiln_stream_t stream) {
    if (!dtype_ok(xdt) || (!scales && !dtype_ok(ydt)) || (res && !dtype_ok(rdt))) return fail(KILN_EINVAL, "%s: dtype", what);
    if (rows < 0 || dim <= 0) return fail(KILN_EINVAL, "%s: bad sizes rows=%d dim=%d", what, rows, dim);
    if (rows > MAX_ROWS || dim > 32768) return fail(KILN_EUNSUPPORTED, "%s: rows=%d above 2^30 or dim=%d above 32768", what, rows, dim);
    if (!(eps > 0.f) || !isfinite(eps)) return fail(KILN_EINVAL, "%s: eps %g must be positive and finite", what, (double)eps);
    if (!res != !h) return fail(KILN_EINVAL, "%s: the residual and the sum go together", what);
    if (!rows) return KILN_OK;
    if (!y || !x) return fail(KILN_EINVAL, "%s: null pointer", what);
    if (!ld_ok(ldx, dim, rows) || (!scales && !ld_ok(ldy, dim, rows)) || (res && (!ld_ok(ldr, dim, rows) || !ld_ok(ldh, dim, rows))))
        return fail(KILN_EINVAL, "%s: a row stride is below %d", what, dim);
    const long long xe = (long long)esize(xdt), re = (long long)esize(rdt), ye = scales ? 1 : (long long)esize(ydt), ly = scales ? dim : ldy;
    if (!aligned(x, xe) || !aligned(y, scales ? 16 : ye) || !aligned(w, 2) || (res && (!aligned(res, re) || !aligned(h, re))))
        return fail(KILN_EUNSUPPORTED, "%s: alignment", what);
    // a row's thread reads its columns of x and the residual before it writes them: y over x and the sum over the residual are in place
    // where they lie the same
    const bool y_in_x = y == x && !scales && ydt == xdt && (rows == 1 || ldy == ldx);
    if (!y_in_x && !apart(y, ly * ye, dim * ye, rows, x, ldx * xe, dim * xe, rows)) return fail(KILN_EINVAL, "%s: y and x overlap", what);
    if (res) {
        const bool h_in_res = h == res && (rows == 1 || ldh == ldr);
        if (!h_in_res && !apart(h, ldh * re, dim * re, rows, res, ldr * re, dim * re, rows)) return fail(KILN_EINVAL, "%s: the sum and the residual overlap", what);
        if (!apart(h, ldh * re, dim * re, rows, x, ldx * xe, dim * xe, rows)) return fail(KILN_EINVAL, "%s: the sum and x overlap", what);
        if (!apart(y, ly * ye, dim * ye, rows, res, ldr * re, dim * re, rows) || !apart(y, ly * ye, dim * ye, rows, h, ldh * re, dim * re, rows))
            return fail(KILN_EINVAL, "%s: y overlaps the residual or the sum", what);
    }
    const struct {
        const char* name;
        const void* p;
        long long ld, width;
        int T;
        bool written;
    } buf[] = {{"y", y, ly * ye, dim * ye, rows, true}, {"the sum", h, ldh * re, dim * re, rows, true}, {"x", x, ldx * xe, dim * xe, rows, false},
               {"the residual", res, ldr * re, dim * re, rows, false}, {"the weight", w, dim * 2LL, dim * 2LL, 1, false}};
    const long long sw = (long long)rows * (dim / 32);
    for (const auto& b : buf) {
        if (!b.p) continue;
        if (scales && !apart(scales, sw, sw, 1, b.p, b.ld, b.width, b.T)) return fail(KILN_EINVAL, "%s: the scales and %s overlap", what, b.name);
        if (w && b.written && !apart(w, dim * 2LL, dim * 2LL, 1, b.p, b.ld, b.width, b.T))
            return fail(KILN_EINVAL, "%s: the weight and %s overlap", what, b.name);
    }
    kiln::RmsLaunch c{};
    c.y = y;
    c.scales = scales;
    c.h = h;
    c.x = x;
    c.res = res;
    c.w = w;
    c.ydt = (DT)ydt;
    c.xdt = (DT)xdt;
    c.rdt = (DT)rdt;
    c.ldy = (size_t)(rows == 1 ? dim : ly);
    c.ldh = (size_t)(rows == 1 ? dim : ldh);
    c.ldx = (size_t)(rows == 1 ? dim : ldx);
    c.ldr = (size_t)(rows == 1 ? dim : ldr);
    c.rows = rows;
    c.dim = dim;
    c.eps = eps;
    return hip_check(kiln::launch_add_rmsnorm(c, (hipStream_t)stream), what);
}

int kiln_add_rmsnorm(void* y, int ydtype, int ldy, void* h, int ldh, const void* x, int xdtype, int ldx, const void* res, int rdtype, int ldr,
                     const uint16_t* w_bf16, int rows, int dim, float eps, kiln_stream_t stream) {
    kiln::prof::Scope prof_("norm", (hipStream_t)stream);
    return add_rmsnorm("add_rmsnorm", y, ydtype, ldy, nullptr, h, ldh, x, xdtype, ldx, res, rdtype, ldr, w_bf16, rows, dim, eps, stream);
}

int kiln_add_rmsnorm_mxfp8(uint8_t* codes, uint8_t* scales, void* h, int ldh, const void* x, int xdtype, int ldx, const void* res, int rdtype,
                           int ldr, const uint16_t* w_bf16, int rows, int dim, float eps, kiln_stream_t stream) {
    kiln::prof::Scope prof_("norm", (hipStream_t)stream);
    if (int r = mx_sizes("add_rmsnorm_mxfp8", rows, dim)) return r;
    if (rows && !scales) return fail(KILN_EINVAL, "add_rmsnorm_mxfp8: null pointer");
    static uint8_t none;  // no rows: the checks alone
    return add_rmsnorm("add_rmsnorm_mxfp8", codes, KILN_F32, dim, scales ? scales : &none, h, ldh, x, xdtype, ldx, res, rdtype, ldr, w_bf16, rows, dim, eps, stream);
}

int kiln_mxfp8_quantize(uint8_t* codes, uint8_t* scales, const void* x, int dtype, int ldx, int rows, int cols, kiln_stream_t stream) {
    kiln::prof::Scope prof_("mxfp8", (hipStream_t)stream);
    if (!dtype_ok(dtype)) return fail(KILN_EINVAL, "mxfp8_quantize: dtype %d", dtype);
    if (int r = mx_sizes("mxfp8_quantize", rows, cols)) return r;
    if (!rows) return KILN_OK;
    if (!codes || !scales || !x) return fail(KILN_EINVAL, "mxfp8_quantize: null pointer");
    if (!ld_ok(ldx, cols, rows)) return fail(KILN_EINVAL, "mxfp8_quantize: row stride %d below %d", ldx, cols);
    if (!aligned(codes, 16) || !aligned(x, esize(dtype))) return fail(KILN_EUNSUPPORTED, "mxfp8_quantize: alignment");
    return hip_check(kiln::launch_mx8_quantize(codes, scales, x, (DT)dtype, (size_t)ldx, rows, cols, (hipStream_t)stream), "mxfp8_quantize launch");
}

int kiln_mxfp8_dequantize(void* y, int dtype, int ldy, const uint8_t* codes, const uint8_t* scales, int rows, int cols, kiln_stream_t stream) {
    kiln::prof::Scope prof_("mxfp8", (hipStream_t)stream);
    if (!dtype_ok(dtype)) return fail(KILN_EINVAL, "mxfp8_dequantize: dtype %d", dtype);
    if (int r = mx_sizes("mxfp8_dequantize", rows, cols)) return r;
    if (!rows) return KILN_OK;
    if (!codes || !scales || !y) return fail(KILN_EINVAL, "mxfp8_dequantize: null pointer");
    if (!ld_ok(ldy, cols, rows)) return fail(KILN_EINVAL, "mxfp8_dequantize: row stride %d below %d", ldy, cols);
    if (!aligned(codes, 16) || !aligned(y, esize(dtype))) return fail(KILN_EUNSUPPORTED, "mxfp8_dequantize: alignment");
    return hip_check(kiln::launch_mx8_dequantize(y, (DT)dtype, (size_t)ldy, codes, scales, rows, cols, (hipStream_t)stream), "mxfp8_dequantize launch");
}

// rows x cols of a weight and T rows of linear_mxfp8: KILN_OK, or the refusal
static int mx8_linear_sizes(int T, int rows, int cols) {
    if (int r = mx_sizes("linear_mxfp8", rows, cols)) return r;
    if (T < 0 || !rows) return fail(KILN_EINVAL, "linear_mxfp8: bad sizes T=%d rows=%d", T, rows);
    if (cols > 1 << 22) return fail(KILN_EUNSUPPORTED, "linear_mxfp8: cols %d above 2^22", cols);
    if (T > MAX_ROWS || (long long)(T / 64 + 1) * (rows / 64 + 1) > MAX_ROWS)
        return fail(KILN_EUNSUPPORTED, "linear_mxfp8: T=%d above 2^30, or T x rows=%d above 2^42 outputs", T, rows);
    return KILN_OK;
}

int kiln_linear_mxfp8_tile(int T, int rows, int cols, int epi) {
    if (T <= 0 || epi < KILN_EPI_F32 || epi > KILN_EPI_RESID || mx8_linear_sizes(T, rows, cols)) return 0;
    return kiln::linear_mx8_tile(T, rows, cols, epi);
}

int kiln_linear_mxfp8(void* y, int ldy, const uint8_t* codes, const uint8_t* scales, int T, const uint8_t* wp, int rows, int cols, int epi,
                      const float* gate, float beta, kiln_stream_t stream) {
    kiln::prof::Scope prof_("gemm_mxfp8", (hipStream_t)stream);
    if (epi < KILN_EPI_F32 || epi > KILN_EPI_RESID) return fail(KILN_EINVAL, "linear_mxfp8: epilogue %d", epi);
    if (int r = mx8_linear_sizes(T, rows, cols)) return r;
    if (!T) return KILN_OK;
    if (!y || !codes || !scales || !wp) return fail(KILN_EINVAL, "linear_mxfp8: null pointer");
    if (!ld_ok(ldy, rows, T)) return fail(KILN_EINVAL, "linear_mxfp8: row stride %d below %d", ldy, rows);
    const long long ye = epi == KILN_EPI_F32 || epi == KILN_EPI_RESID ? 4 : 2;
    if (!aligned(wp, 16) || !aligned(codes, 16) || !aligned(y, ye) || !aligned(gate, 4)) return fail(KILN_EUNSUPPORTED, "linear_mxfp8: alignment");
    if (!apart(codes, cols, cols, T, y, ldy * ye, rows * ye, T) || !apart(scales, cols / 32, cols / 32, T, y, ldy * ye, rows * ye, T))
        return fail(KILN_EINVAL, "linear_mxfp8: y overlaps the codes or the scales");
    return hip_check(kiln::launch_linear_mx8(y, (size_t)ldy, codes, scales, T, wp, rows, cols, epi, gate, beta, (hipStream_t)stream),
                     "linear_mxfp8 launch");
}

}  // extern "C"
