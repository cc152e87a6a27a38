// The MXFP4 linear layer (kiln_linear_mxfp4): y = epilogue(Q(x) Wq^T) with v_mfma_scale_f32_16x16x128_f8f6f4, both operands
// 4-bit codes with a scale per 32 values (mxfp4.hpp). Products of codes and powers of two are exact; sums are fp32. The layer of MXFP8 rows
// (kiln_linear_mxfp8) is compiled with it: gemm_mxfp8.hpp, included at the end.
#include <hip/hip_runtime.h>

#include <math.h>

#include <algorithm>

#include "gemm16.hpp"
#include "mxfp4.hpp"

namespace kiln {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) uint32_t lds_u32;

struct MxGemmParams {
    const uint8_t* xc;  // x in the operand layout (the tiled form)
    const uint8_t* xs;
    const void* x;      // x as it is (the few-row form, which quantises it itself)
    size_t ldx;
    const uint8_t* wc;
    const uint8_t* ws;
    int T, N, K, kbs;
    void* y;
    size_t ldy;
    const float* gate;
    float beta;
    int vec;            // rows and base of y take stores of 4 elements (1), of 16 bytes (2)
    int tiles_m, tiles_n, total, per;
};

// A and B blocks' scale bytes are selected from a register of four: J, I are constants
template <int J, int I>
__device__ __forceinline__ floatx4 mx_mfma(u32x4 a, uint32_t sa, u32x4 b, uint32_t sb, floatx4 c) {
    const i32x8 A = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
    const i32x8 B = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, 4, 4, J, (int)sa, I, (int)sb);  // 4: E2M1
}
__device__ __forceinline__ floatx4 mx_mfma_at(int j, int i, u32x4 a, uint32_t sa, u32x4 b, uint32_t sb, floatx4 c) {
    switch (j * 4 + i) {  // j and i are constants once the loops around are unrolled
#define MX_CASE(J, I) case J * 4 + I: return mx_mfma<J, I>(a, sa, b, sb, c);
#define MX_ROW(J) MX_CASE(J, 0) MX_CASE(J, 1) MX_CASE(J, 2) MX_CASE(J, 3)
        MX_ROW(0) MX_ROW(1) MX_ROW(2) MX_ROW(3)
#undef MX_ROW
#undef MX_CASE
    }
    return c;
}

// GELU(v) = v Phi(v) = max(v, 0) - |v| Phi(-|v|), with Phi(-z) = 2^P(z): log2 Phi(-z) is smooth on all of z >= 0, and P is its
// polynomial of degree 7 with the least largest error on [0, 6] (2^-18.2 of Phi; below 2^-17 with fp32's roundings), decreasing
// beyond, where |v| Phi(-|v|) < 2^-27 is nothing to fp16. Relative to GELU itself the error is no larger (Phi(-z) <= 1/2), a
// hundredth of the fp16 rounding that follows. 10 operations and one exp against erfc's 17, a reciprocal and an exp: the GELU
// of 6912 x 8192 outputs takes some 24 us instead of 40. -inf gives 0, inf inf, NaN NaN.
__device__ __forceinline__ float mx_gelu(float v) {
    const float z = fabsf(v);
    float q = -1.83525563e-6f;
    q = fmaf(q, z, 6.16068428e-5f);
    q = fmaf(q, z, -9.30587179e-4f);
    q = fmaf(q, z, 8.50810017e-3f);
    q = fmaf(q, z, -5.39603643e-2f);
    q = fmaf(q, z, -0.458464354f);
    q = fmaf(q, z, -1.15125084f);
    q = fmaf(q, z, -0.999995291f);
    return fmaf(-fminf(z, 3.0e38f), __builtin_amdgcn_exp2f(q), fmaxf(v, 0.f));
}

// columns n .. n + 3 of row m
template <int EPI>
__device__ __forceinline__ void mx_store(const MxGemmParams& p, int m, int n, floatx4 v) {
    if (m >= p.T || n >= p.N) return;
    constexpr bool F32 = EPI == KILN_EPI_F32 || EPI == KILN_EPI_RESID;
    if constexpr (EPI == KILN_EPI_GELU16)
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = mx_gelu(v[e]);
    const size_t off = (size_t)m * p.ldy + n;
    if (p.vec && n + 4 <= p.N) {
        if constexpr (F32) {
            float* dst = static_cast<float*>(p.y) + off;
            if (EPI == KILN_EPI_RESID || p.beta != 0.f) {
                const floatx4 o = *reinterpret_cast<const floatx4*>(dst);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    v[e] = EPI == KILN_EPI_RESID ? o[e] + (p.gate ? p.gate[n + e] : 1.f) * v[e] : v[e] + p.beta * o[e];
            }
            *reinterpret_cast<floatx4*>(dst) = v;
        } else {
            *reinterpret_cast<half4*>(static_cast<_Float16*>(p.y) + off) =
                half4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (n + e >= p.N) break;
        if constexpr (F32) {
            float* dst = static_cast<float*>(p.y) + off + e;
            if constexpr (EPI == KILN_EPI_RESID) *dst += (p.gate ? p.gate[n + e] : 1.f) * v[e];
            else *dst = p.beta != 0.f ? v[e] + p.beta * *dst : v[e];
        } else {
            static_cast<_Float16*>(p.y)[off + e] = (_Float16)v[e];
        }
    }
}

// The tile of a wave: acc[nb][mb] holds columns n0 + 16 nb + 4 (lane / 16) .. + 3 of row m0 + 16 mb + lane % 16. WAVES waves share the LDS
// bytes of the ring that the products are done with (this function waits for the others').
template <int EPI, int NB, int MB, int WAVES, int LDS>
__device__ __forceinline__ void mx_store_tile(const MxGemmParams& p, const floatx4 (&acc)[NB][MB], uint8_t* lds8, int wv, int lane, int m0,
                                              int n0) {
    const int g = lane >> 4, rl = lane & 15;
    if (p.vec < 2) {
#pragma unroll
        for (int mb = 0; mb < MB; mb++)
#pragma unroll
            for (int nb = 0; nb < NB; nb++) mx_store<EPI>(p, m0 + mb * 16 + rl, n0 + nb * 16 + 4 * g, acc[nb][mb]);
        return;
    }
    // Aligned rows leave through LDS as whole rows of the wave's columns, 16 bytes a lane, instead of 8- or 16-byte pieces of
    // 16 rows per store. The wave's region holds RB row blocks; 16-byte chunks lie permuted by the row (both sides conflict-free).
    constexpr bool F32 = EPI == KILN_EPI_F32 || EPI == KILN_EPI_RESID;
    constexpr int RB = F32 ? MB / 2 : MB, CH = NB * 16 * (F32 ? 4 : 2) / 16, PER = F32 ? 4 : 8;  // chunks of a row, values of a chunk
    static_assert(RB * 16 * CH * 16 * WAVES <= LDS, "the waves' regions fit in the ring");
    uint8_t* stg = lds8 + wv * (RB * 16 * CH * 16);
    __builtin_amdgcn_s_waitcnt(0xC07F);
    __builtin_amdgcn_s_barrier();  // every wave is done with the ring
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int h = 0; h < MB / RB; h++) {
#pragma unroll
        for (int r = 0; r < RB; r++)
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
                floatx4 v = acc[nb][h * RB + r];
                if constexpr (EPI == KILN_EPI_GELU16)
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = mx_gelu(v[e]);
                const int row = r * 16 + rl;
                if constexpr (F32)
                    *reinterpret_cast<floatx4*>(stg + row * CH * 16 + ((nb * 4 + g) ^ (row & (CH - 1))) * 16) = v;
                else
                    *reinterpret_cast<half4*>(stg + row * CH * 16 + ((nb * 2 + (g >> 1)) ^ (row & (CH - 1))) * 16 + (g & 1) * 8) =
                        half4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
            }
        __builtin_amdgcn_wave_barrier();  // a wave's LDS operations keep their order
#pragma unroll 4
        for (int i = 0; i < RB * 16 * CH / 64; i++) {
            const int row = (i * 64 + lane) / CH, c = (i * 64 + lane) % CH;
            const u32x4 v = *reinterpret_cast<const u32x4*>(stg + row * CH * 16 + (c ^ (row & (CH - 1))) * 16);
            const int m = m0 + h * RB * 16 + row, n = n0 + c * PER;
            if (m >= p.T || n >= p.N) continue;
            const size_t off = (size_t)m * p.ldy + n;
            if constexpr (F32) {
                const floatx4 f = __builtin_bit_cast(floatx4, v);
                mx_store<EPI>(p, m, n, f);
            } else if (n + PER <= p.N) {
                *reinterpret_cast<u32x4*>(static_cast<_Float16*>(p.y) + off) = v;
            } else {
                const half8 hv = __builtin_bit_cast(half8, v);
#pragma unroll
                for (int e = 0; e < PER; e++)
                    if (n + e < p.N) static_cast<_Float16*>(p.y)[off + e] = hv[e];
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// ---- few rows: a workgroup takes 16 weight rows and every row of x ----
//
// Eight waves share out the k blocks; each quantises its part of x in registers (a lane of the operand layout holds exactly
// one block of 32) and reads its units of the weight, 1 KB each, straight from memory. The waves' sums meet in LDS.
// Bound by the latency of two dependent loads and the launch: one launch, no workspace. 1 row x 8192 x 2048 with GELU, 9 MB, in 5.4 us
// (an empty launch is 2.2, the bytes 1.7).
constexpr int FEW_WAVES = 8;
template <class E, int EPI, int MB, bool VEC>
__global__ __launch_bounds__(FEW_WAVES * 64) void k_mx_few(const MxGemmParams p) {
    __shared__ floatx4 red[FEW_WAVES][MB][64];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nb = blockIdx.x, r = lane & 15;
    floatx4 acc[MB];
#pragma unroll
    for (int mb = 0; mb < MB; mb++) acc[mb] = floatx4{0.f, 0.f, 0.f, 0.f};
    const uint8_t* wc = p.wc + (size_t)nb * MX_UNIT + lane * 16;
    const uint8_t* wsc = p.ws + (size_t)(nb >> 2) * MX_SUNIT + lane * 4 + (nb & 3);
    const size_t rgs = mx_rg(p.N);
    const E* x = static_cast<const E*>(p.x);
    struct Ops {
        u32x4 w;
        uint32_t sw;
        MxVals<E, MXB> v[MB];
    };
    auto inside = [&](int mb, int kb) { return mb * 16 + r < p.T && kb * 128 + 32 * (lane >> 4) < p.K; };
    auto load = [&](Ops& o, int kb) {
        kb = min(kb, p.kbs - 1);
        o.w = *reinterpret_cast<const u32x4*>(wc + kb * rgs * 4 * MX_UNIT);
        o.sw = wsc[kb * rgs * MX_SUNIT];
#pragma unroll
        for (int mb = 0; mb < MB; mb++) {
            const bool in = inside(mb, kb);
            const E* src = x + (in ? (mb * 16 + r) * p.ldx + kb * 128 + 32 * (lane >> 4) : 0);
            if constexpr (VEC) o.v[mb].load(src);
            else o.v[mb].load_any(src, in ? MXB : 0);
        }
    };
    auto mul = [&](const Ops& o, int kb) {
#pragma unroll
        for (int mb = 0; mb < MB; mb++) {
            uint32_t s;
            u32x4 c = mx_block<E>(o.v[mb], s);
            if (!inside(mb, kb)) c = u32x4{0, 0, 0, 0}, s = 0;
            acc[mb] = mx_mfma<0, 0>(o.w, o.sw, c, s, acc[mb]);
        }
    };
    if constexpr (MB * sizeof(E) <= 4) {  // two k blocks in flight, where the registers hold them
        Ops o[2];
        load(o[0], wv);
        load(o[1], wv + FEW_WAVES);
        for (int kb = wv; kb < p.kbs; kb += 2 * FEW_WAVES) {
            mul(o[0], kb);
            load(o[0], kb + 2 * FEW_WAVES);
            if (kb + FEW_WAVES < p.kbs) mul(o[1], kb + FEW_WAVES);
            load(o[1], kb + 3 * FEW_WAVES);
        }
    } else {
        for (int kb = wv; kb < p.kbs; kb += FEW_WAVES) {
            Ops o;
            load(o, kb);
            mul(o, kb);
        }
    }
#pragma unroll
    for (int mb = 0; mb < MB; mb++) red[wv][mb][lane] = acc[mb];
    __syncthreads();
    if (wv < MB) {
        floatx4 t = red[0][wv][lane];
#pragma unroll
        for (int w = 1; w < FEW_WAVES; w++) t += red[w][wv][lane];
        mx_store<EPI>(p, wv * 16 + r, nb * 16 + 4 * (lane >> 4), t);
    }
}

// ---- small products: operands from the quantised rows straight into registers ----
//
// A workgroup takes 16 NB weight rows x 16 MB rows of x; its eight waves share out the k blocks, each reading whole 1 KB units
// of both operands (from L2) two k blocks ahead of their products, and meet in LDS. No ring to fill: what bounds it at these sizes
// is the latency of a few loads, then L2's rate. 64 x 2048 x 8192 in 9.7 us with its quantise pass (128 x 128 tiles: 21.3).
constexpr int THIN_WAVES = 8;
template <int EPI, int NB, int MB>
__global__ __launch_bounds__(THIN_WAVES * 64, 2) void k_mx_thin(const MxGemmParams p) {
    extern __shared__ __attribute__((aligned(16))) floatx4 thin_red[];  // [wave][block][lane]
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ti = (int)(blockIdx.x & 7) * p.per + (int)(blockIdx.x >> 3);  // an XCD's range: the row tiles of a W tile together
    if (ti >= p.total) return;
    const int tm = ti % p.tiles_m, tn = ti / p.tiles_m, nb0 = tn * NB, mb0 = tm * MB;
    const uint8_t* wc = p.wc + (size_t)nb0 * MX_UNIT + lane * 16;
    const uint8_t* xc = p.xc + (size_t)mb0 * MX_UNIT + lane * 16;
    const uint8_t* wsc = p.ws + (size_t)(nb0 >> 2) * MX_SUNIT + lane * 4;
    const uint8_t* xsc = p.xs + (size_t)(mb0 >> 2) * MX_SUNIT + lane * 4;
    const size_t wrg = mx_rg(p.N), xrg = mx_rg(p.T);
    const int wsh = 8 * (nb0 & 3), xsh = 8 * (mb0 & 3);  // the tile's first block's byte of a scale unit
    struct Ops {
        u32x4 w[NB], x[MB];
        uint32_t sw, sx;
    } ops[2];
    auto load = [&](Ops& o, int kb) {
        kb = min(kb, p.kbs - 1);
#pragma unroll
        for (int i = 0; i < NB; i++) o.w[i] = *reinterpret_cast<const u32x4*>(wc + (kb * wrg * 4 + i) * MX_UNIT);
#pragma unroll
        for (int i = 0; i < MB; i++) o.x[i] = *reinterpret_cast<const u32x4*>(xc + (kb * xrg * 4 + i) * MX_UNIT);
        o.sw = *reinterpret_cast<const uint32_t*>(wsc + kb * wrg * MX_SUNIT);
        o.sx = *reinterpret_cast<const uint32_t*>(xsc + kb * xrg * MX_SUNIT);
    };
    floatx4 acc[NB][MB];
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
        for (int j = 0; j < MB; j++) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    auto mul = [&](const Ops& o) {
        const uint32_t sw = o.sw >> wsh, sx = o.sx >> xsh;
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int j = 0; j < MB; j++) acc[i][j] = mx_mfma_at(i, j, o.w[i], sw, o.x[j], sx, acc[i][j]);
    };
    load(ops[0], wv);
    load(ops[1], wv + THIN_WAVES);
    for (int kb = wv; kb < p.kbs; kb += 2 * THIN_WAVES) {
        mul(ops[0]);
        load(ops[0], kb + 2 * THIN_WAVES);
        if (kb + THIN_WAVES < p.kbs) mul(ops[1]);
        load(ops[1], kb + 3 * THIN_WAVES);
    }
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
        for (int j = 0; j < MB; j++) thin_red[(wv * NB * MB + i * MB + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    for (int b = wv; b < NB * MB; b += THIN_WAVES) {
        floatx4 t = thin_red[b * 64 + lane];
#pragma unroll
        for (int w = 1; w < THIN_WAVES; w++) t += thin_red[(w * NB * MB + b) * 64 + lane];
        mx_store<EPI>(p, (mb0 + b % MB) * 16 + (lane & 15), (nb0 + b / MB) * 16 + 4 * (lane >> 4), t);
    }
}
template <int EPI, int NB, int MB>
static hipError_t mx_thin(MxGemmParams p, hipStream_t s) {
    p.tiles_m = (p.T + 16 * MB - 1) / (16 * MB);
    p.tiles_n = (p.N + 16 * NB - 1) / (16 * NB);
    p.total = p.tiles_m * p.tiles_n;
    p.per = (p.total + 7) / 8;
    if (hipError_t e = grid_check((size_t)p.per * 8, THIN_WAVES * 64)) return e;
    hipLaunchKernelGGL((k_mx_thin<EPI, NB, MB>), dim3(p.per * 8), dim3(THIN_WAVES * 64), THIN_WAVES * NB * MB * 1024, s, p);
    return hipGetLastError();
}

// ---- tiles ----
//
// WN x WM waves of 16 NB x 16 MB blocks. A stage of the LDS ring holds one k block of 128: the tile's units of W and of x
// (1 KB each) and their scales, all by LDS DMA in the operand layout, so that every operand read is 1 KB without conflicts.
//
// 256 x 256 (8 waves of 64 x 128): 8192^3 in 271 us with its quantise pass (36), 4.1 PFLOP/s, the matrix cores busy 64% of the product's
// time at 1.74 GHz (alone, on random operands in registers, the matrix instructions reach 6.9 PFLOP/s on this chip at 1.7 GHz, on zeros
// 9.2). Three 1 KB operand reads per 8 products; four waves of 128 x 128 would need two, but their registers spill into moves:
// 40% slower. 6912 x 8192 x 2048 takes 75 us, with GELU 97, matrix cores busy 40% and 29%: 864 tiles in four rounds that would be
// 3.4, and each round's start and epilogue. Two workgroups of 128 x 256 per CU (one's epilogue beside the other's products, in
// step or staggered) measured the same.
// 128 x 128 (4 waves of 64 x 64): 1537 x 2048 x 2048 in 10.4 us, fp32 out 12.7, about 0.3 us a k block of 17 KB whatever the ring's depth
// (4 to 9 stages) or the number of waves. Two thirds of the requests hit the L2, next to nothing comes from HBM; what it waits
// for is not known.
template <int WN_, int WM_, int NB_, int MB_, int NST_, int WGS_>
struct MxCfg {
    static constexpr int WN = WN_, WM = WM_, NB = NB_, MB = MB_, NST = NST_, WGS = WGS_, WAVES = WN * WM, THREADS = WAVES * 64;
    static constexpr int BN = WN * NB * 16, BM = WM * MB * 16;
    static constexpr int UN = BN / 16, UM = BM / 16, SN = (BN + 63) / 64, SM = (BM + 63) / 64;
    static constexpr int CODE_DMA = (UN + UM) / WAVES, SCALE_DMA = (SN + SM + WAVES - 1) / WAVES, DPS = CODE_DMA + SCALE_DMA;
    static constexpr int SC_OFF = (UN + UM) * MX_UNIT, STAGE = SC_OFF + (SN + SM) * MX_SUNIT, LDS = NST * STAGE;
    static_assert((UN + UM) % WAVES == 0 && NB % 4 == 0 && MB % 4 == 0 && LDS * WGS <= 160 * 1024, "tile");
};

template <int EPI, class C>
__global__ __launch_bounds__(C::THREADS, C::WAVES * C::WGS / 4) void k_mx_gemm(const MxGemmParams p) {
#ifdef __HIP_DEVICE_COMPILE__  // the host pass only needs the kernel's handle
    extern __shared__ __attribute__((aligned(16))) uint8_t lds8[];
    constexpr int NB = C::NB, MB = C::MB;
    // blocks go round the 8 XCDs: each takes a contiguous range of tiles, in groups of row tiles that share W in its L2
    const int ti = (int)(blockIdx.x & 7) * p.per + (int)(blockIdx.x >> 3);
    if (ti >= p.total) return;
    int tm, tn;
    raster_tile(ti, 4, p.tiles_m, p.tiles_n, tm, tn);
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wn = wv % C::WN, wm = wv / C::WN;
    const int wrg = mx_rg(p.N), xrg = mx_rg(p.T);  // row groups that exist

    // DMA pieces of this wave: units wv, wv + WAVES, .. of the stage (W's first), then the scale units; row blocks past the
    // matrix re-read its last one (their results are not stored)
    typedef __attribute__((address_space(3))) void* lds_p;
    const uint8_t* src[C::CODE_DMA];
    size_t kstep[C::CODE_DMA];  // bytes from a k block to the next
#pragma unroll
    for (int i = 0; i < C::CODE_DMA; i++) {
        const int u = wv + i * C::WAVES;
        src[i] = (u < C::UN ? p.wc + (size_t)min(tn * C::UN + u, 4 * wrg - 1) * MX_UNIT
                            : p.xc + (size_t)min(tm * C::UM + u - C::UN, 4 * xrg - 1) * MX_UNIT) + lane * 16;
        kstep[i] = (size_t)4 * MX_UNIT * (u < C::UN ? wrg : xrg);
    }
    const uint8_t* ssrc[C::SCALE_DMA];
    size_t skstep[C::SCALE_DMA];
    int sdst[C::SCALE_DMA];
#pragma unroll
    for (int i = 0; i < C::SCALE_DMA; i++) {
        const int u = (wv + i * C::WAVES) % (C::SN + C::SM);  // a wave without one copies another's again
        sdst[i] = C::SC_OFF + u * MX_SUNIT;
        ssrc[i] = (u < C::SN ? p.ws + (size_t)min(tn * C::BN / 64 + u, wrg - 1) * MX_SUNIT
                             : p.xs + (size_t)min(tm * C::BM / 64 + u - C::SN, xrg - 1) * MX_SUNIT) + lane * 4;
        skstep[i] = (size_t)MX_SUNIT * (u < C::SN ? wrg : xrg);
    }
    typedef const __attribute__((address_space(1))) void* glb_p;
    // piece i of the next k block to copy (`more`: there is one after it; past the end the last one again)
    auto dma_piece = [&](int i, bool more, int stage) {
        uint8_t* base = lds8 + stage * C::STAGE;
        if (i < C::CODE_DMA) {
            __builtin_amdgcn_global_load_lds((glb_p)src[i], (lds_p)(base + (wv + i * C::WAVES) * MX_UNIT), 16, 0, 0);
            src[i] += more ? kstep[i] : 0;
        } else if (i < C::DPS) {
            __builtin_amdgcn_global_load_lds((glb_p)ssrc[i - C::CODE_DMA], (lds_p)(base + sdst[i - C::CODE_DMA]), 4, 0, 0);
            ssrc[i - C::CODE_DMA] += more ? skstep[i - C::CODE_DMA] : 0;
        }
    };
    auto dma = [&](int step, int stage) {
#pragma unroll
        for (int i = 0; i < C::DPS; i++) dma_piece(i, step + 1 < p.kbs, stage);
    };

    const uint32_t lds_base = (uint32_t)(size_t)(__attribute__((address_space(3))) uint8_t*)lds8;
    floatx4 acc[NB][MB];
#pragma unroll
    for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int mb = 0; mb < MB; mb++) acc[nb][mb] = floatx4{0.f, 0.f, 0.f, 0.f};

    constexpr int XB = MB <= 4 ? 2 : 1;  // x's operands double where the registers hold them, read ahead like W's
    u32x4 fw[2][NB], fx[XB][MB];
    uint32_t sw[2][NB / 4], sx[2][MB / 4];
    const uint32_t wa = lds_base + wn * NB * MX_UNIT + lane * 16, xa = lds_base + (C::UN + wm * MB) * MX_UNIT + lane * 16;
    const uint32_t swa = lds_base + C::SC_OFF + wn * NB / 4 * MX_SUNIT + lane * 4;
    const uint32_t sxa = lds_base + C::SC_OFF + (C::SN + wm * MB / 4) * MX_SUNIT + lane * 4;
    auto read_w = [&](int b, uint32_t st) {
#pragma unroll
        for (int nb = 0; nb < NB; nb++) fw[b][nb] = *reinterpret_cast<const lds_u32x4*>((size_t)(wa + st + nb * MX_UNIT));
#pragma unroll
        for (int i = 0; i < NB / 4; i++) sw[b][i] = *reinterpret_cast<const lds_u32*>((size_t)(swa + st + i * MX_SUNIT));
#pragma unroll
        for (int i = 0; i < MB / 4; i++) sx[b][i] = *reinterpret_cast<const lds_u32*>((size_t)(sxa + st + i * MX_SUNIT));
    };
    auto read_x = [&](int b, int mb, uint32_t st) { fx[b & (XB - 1)][mb] = *reinterpret_cast<const lds_u32x4*>((size_t)(xa + st + mb * MX_UNIT)); };

#pragma unroll
    for (int s = 0; s < C::NST - 1; s++) dma(s, s);
    wait_vmcnt<(C::NST - 2) * C::DPS>();
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    read_w(0, 0);
#pragma unroll
    for (int mb = 0; mb < MB; mb++) read_x(0, mb, 0);
    int next = 1;  // the stage of step i + 1
    // Step i: its operands are in registers. Those of step i + 1 landed in every wave; the stage of step i - 1, whose reads every
    // wave finished before its products of i - 1, is refilled (past the end with the last block again: the count of loads
    // in flight stays the same). The operands of i + 1 are read between the products of i.
    auto step = [&](int i, auto tag) {
        constexpr int cur = decltype(tag)::value;
        wait_vmcnt<(C::NST - 3) * C::DPS>();
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        const int ds = next >= 2 ? next - 2 : next - 2 + C::NST;
        const uint32_t st = next * C::STAGE;
#pragma unroll
        for (int mb = 0; mb < MB; mb++) {
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
                acc[nb][mb] = mx_mfma_at(nb & 3, mb & 3, fw[cur][nb], sw[cur][nb / 4], fx[cur & (XB - 1)][mb], sx[cur][mb / 4], acc[nb][mb]);
            __builtin_amdgcn_sched_barrier(0);
            if (XB == 1) read_x(0, mb, st);
            else if (mb < MB / 2) {
                read_x(cur ^ 1, 2 * mb, st);
                read_x(cur ^ 1, 2 * mb + 1, st);
            }
            if (mb == 0) {
#pragma unroll
                for (int u = 0; u < NB / 4; u++) sw[cur ^ 1][u] = *reinterpret_cast<const lds_u32*>((size_t)(swa + st + u * MX_SUNIT));
#pragma unroll
                for (int u = 0; u < MB / 4; u++) sx[cur ^ 1][u] = *reinterpret_cast<const lds_u32*>((size_t)(sxa + st + u * MX_SUNIT));
            }
            if (mb < MB / 2) {
#pragma unroll
                for (int n = 0; n < 2 * NB / MB; n++) {
                    const int nb = mb * (2 * NB / MB) + n;
                    fw[cur ^ 1][nb] = *reinterpret_cast<const lds_u32x4*>((size_t)(wa + st + nb * MX_UNIT));
                }
            }
#pragma unroll
            for (int n = 0; n < (C::DPS + MB - 1) / MB; n++) dma_piece(mb * ((C::DPS + MB - 1) / MB) + n, i + C::NST < p.kbs, ds);
            __builtin_amdgcn_sched_barrier(0);
        }
        next = next == C::NST - 1 ? 0 : next + 1;
    };
    int i = 0;
    for (; i + 2 <= p.kbs; i += 2) {
        step(i, std::integral_constant<int, 0>{});
        step(i + 1, std::integral_constant<int, 1>{});
    }
    if (i < p.kbs) step(i, std::integral_constant<int, 0>{});
    wait_vmcnt<0>();  // no copy into LDS outlives the ring
    const int m0 = tm * C::BM + wm * MB * 16, n0 = tn * C::BN + wn * NB * 16;
    mx_store_tile<EPI, NB, MB, C::WAVES, C::LDS>(p, acc, lds8, wv, lane, m0, n0);
#endif
}

using MxBig = MxCfg<4, 2, 4, 8, 4, 1>;  // 256 x 256 (n x m), 8 waves, 136 KB
using MxMid = MxCfg<2, 2, 4, 4, 4, 2>;  // 128 x 128, 4 waves, 68 KB

template <int EPI, class C>
static hipError_t mx_tiles(MxGemmParams p, hipStream_t s) {
    p.tiles_m = (p.T + C::BM - 1) / C::BM;
    p.tiles_n = (p.N + C::BN - 1) / C::BN;
    p.total = p.tiles_m * p.tiles_n;
    p.per = (p.total + 7) / 8;
    if (hipError_t e = grid_check((size_t)p.per * 8, C::THREADS)) return e;
    hipLaunchKernelGGL((k_mx_gemm<EPI, C>), dim3(p.per * 8), dim3(C::THREADS), C::LDS, s, p);
    return hipGetLastError();
}
template <class E, int EPI>
static hipError_t mx_few(const MxGemmParams& p, hipStream_t s) {
    const bool vec = ((uintptr_t)p.x & 15) == 0 && (p.T == 1 || p.ldx * sizeof(E) % 16 == 0);
    const int mb = p.T <= 16 ? 1 : p.T <= 32 ? 2 : 4;
    auto pick = [&]() {
        if (mb == 1) return vec ? k_mx_few<E, EPI, 1, true> : k_mx_few<E, EPI, 1, false>;
        if (mb == 2) return vec ? k_mx_few<E, EPI, 2, true> : k_mx_few<E, EPI, 2, false>;
        return vec ? k_mx_few<E, EPI, 4, true> : k_mx_few<E, EPI, 4, false>;
    };
    if (hipError_t e = grid_check((p.N + 15) / 16, FEW_WAVES * 64)) return e;
    hipLaunchKernelGGL(pick(), dim3((p.N + 15) / 16), dim3(FEW_WAVES * 64), 0, s, p);
    return hipGetLastError();
}

// The form of a product.
enum MxKind { MX_FEW, MX_THIN22, MX_THIN44, MX_MID, MX_BIG };
// Few rows quantise in the product, one launch: as long as 16 of them, or little of x, is quantised anew in each workgroup (fp16
// out, the whole call among others, against the next best form: 2048 x 2048, T = 32 7.6 / 8.5 us, T = 64 10.5 / 8.3;
// 2048 x 8192, T = 8 7.6 / 8.2, T = 17 12.5 / 8.6; 1024 x 1024, T = 64 6.8 / 8.4).
static bool mx_few_rows(int T, int N, int K) {
    const int mb = (T + 15) / 16, groups = std::max(1, (N + 15) / 16 / cu_count());
    return T <= 64 && (mb == 1 || (long)(mb > 2 ? 4 : mb) * mx_kb(K) * groups <= 32);
}
// Modelled time of the other forms' product kernel in us: workgroups that follow each other on a CU, each with a fixed cost and one
// per k block, and what the tiles in flight take from each other. Fitted to T = 17 .. 6912 x {1024 x 1024, 2048 x 2048,
// 8192 x 2048, 2048 x 8192}; where two forms meet they measured within 5% (8192 x 2048, T = 128 8.7 and T = 200 12.2 with 64 x 64,
// 10.6 and 10.5 with 128 x 128 tiles; T = 1537 28.5 with 128 x 128, 25.9 with 256 x 256).
static MxKind mx_choose(int T, int N, int K) {
    if (mx_few_rows(T, N, K)) return MX_FEW;
    const double cus = cu_count(), kb = mx_kb(K);
    auto tiles = [&](int bn, int bm) { return (double)((N + bn - 1) / bn) * ((T + bm - 1) / bm); };
    const double t22 = tiles(32, 32), t44 = tiles(64, 64), tm = tiles(128, 128), tb = tiles(256, 256);
    const double cost[4] = {0.8 + 0.01 * kb + (0.25 + 0.05 * kb) * t22 / cus,
                            ceil(t44 / cus) * (1.2 + 0.045 * kb) + 0.125 * kb * t44 / cus,
                            1.9 * std::max(1.0, tm / cus) + kb * (0.155 + 0.22 * tm / cus),
                            ceil(tb / cus) * (5.0 + 0.55 * kb) + 0.35 * kb * tb / cus};
    return (MxKind)(MX_THIN22 + (std::min_element(cost, cost + 4) - cost));
}
size_t linear_mx_workspace(int T, int rows, int cols) {
    return mx_few_rows(T, rows, cols) ? 0 : mx_code_bytes(T, cols) + mx_scale_bytes(T, cols);
}

int linear_mx_tile(int T, int rows, int cols) {
    switch (mx_choose(T, rows, cols)) {
        case MX_FEW: return 16 << 16 | (T <= 16 ? 16 : T <= 32 ? 32 : 64);
        case MX_THIN22: return 32 << 16 | 32;
        case MX_THIN44: return 64 << 16 | 64;
        case MX_MID: return MxMid::BN << 16 | MxMid::BM;
        default: return MxBig::BN << 16 | MxBig::BM;
    }
}

template <int EPI>
static hipError_t linear_mx_epi(MxGemmParams p, DT dt, uint8_t* ws, hipStream_t s) {
    const MxKind kind = mx_choose(p.T, p.N, p.K);
    if (kind == MX_FEW) {
        if (dt == DT::F32) return mx_few<float, EPI>(p, s);
        if (dt == DT::F16) return mx_few<_Float16, EPI>(p, s);
        return mx_few<__bf16, EPI>(p, s);
    }
    if (hipError_t e = launch_mx_quantize_pack(ws, p.x, dt, p.ldx, p.T, p.K, s)) return e;
    p.xc = ws;
    p.xs = ws + mx_code_bytes(p.T, p.K);
    switch (kind) {
        case MX_THIN22: return mx_thin<EPI, 2, 2>(p, s);
        case MX_THIN44: return mx_thin<EPI, 4, 4>(p, s);
        case MX_MID: return mx_tiles<EPI, MxMid>(p, s);
        default: return mx_tiles<EPI, MxBig>(p, s);
    }
}

hipError_t launch_linear_mx(void* y, size_t ldy, const void* x, DT dt, size_t ldx, int T, const uint8_t* wp, int rows, int cols, int epi,
                            const float* gate, float beta, uint8_t* ws, hipStream_t s) {
    MxGemmParams p{};
    p.x = x;
    p.ldx = ldx;
    p.wc = wp;
    p.ws = wp + mx_code_bytes(rows, cols);
    p.T = T;
    p.N = rows;
    p.K = cols;
    p.kbs = mx_kb(cols);
    p.y = y;
    p.ldy = ldy;
    p.gate = gate;
    p.beta = beta;
    const int e4 = epi == KILN_EPI_F32 || epi == KILN_EPI_RESID ? 16 : 8;
    p.vec = ((uintptr_t)y & (e4 - 1)) == 0 && (T == 1 || ldy % 4 == 0);
    if (p.vec && ((uintptr_t)y & 15) == 0 && (T == 1 || ldy * e4 / 4 % 16 == 0)) p.vec = 2;
    switch (epi) {
        case KILN_EPI_F32: return linear_mx_epi<KILN_EPI_F32>(p, dt, ws, s);
        case KILN_EPI_F16: return linear_mx_epi<KILN_EPI_F16>(p, dt, ws, s);
        case KILN_EPI_GELU16: return linear_mx_epi<KILN_EPI_GELU16>(p, dt, ws, s);
        default: return linear_mx_epi<KILN_EPI_RESID>(p, dt, ws, s);
    }
}

}  // namespace kiln

// the layer of MXFP8 rows shares the epilogues above
#include "gemm_mxfp8.hpp"
