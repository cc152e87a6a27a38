// Attention of B x Tq queries to Tk encoder states of another length (kiln_cross_attn): O = softmax(s Q K^T) V per head,
// Hkv key heads each shared by G = Hq / Hkv query heads, keys bounded by a length and a mask per item. fp16 or bf16 rows,
// read where they lie: no prepare pass (a context of a few hundred states is used once per layer).
//
// The G query heads of a key head and their Tq tokens are the rows of one problem, r = t G + g, so that a key is read once
// for all of them. Scores are computed transposed, S^T = K Q^T, and O^T = V^T P^T, with v_mfma_f32_16x16x32: a lane of the
// S^T accumulators holds eight of a 32-key tile's keys for one row, which is the B operand of the second product as it
// is, if V's keys come in the same order: two transposing LDS reads per 16 dimensions.
//
// Keys come in tiles of 32: K and V rows go to LDS by buffer DMA, 16 bytes a lane, and the 16-byte chunks of a row lie
// permuted (k_swz, v_swz) so that both kinds of read spread over the banks; the permutation is on the global side. Rows past
// the length or masked out lie outside the descriptor's range and arrive as zeros, whatever they hold: their scores are set
// to -inf by the tile's bit mask, and 0 times an infinity or a NaN never happens.
//
// Softmax in one pass: running maximum m and sum l per row in fp32, in units of log2. The maximum moves (and O and l are
// rescaled) only when a tile's exceeds it by more than 8, so P <= 2^8 and most tiles need no exchange between lanes. P is
// rounded to the inputs' type, half a step of it (2^-11 fp16, 2^-8 bf16) per weight, as far off as the output's own rounding.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "internal.hpp"

namespace kiln {

struct CrossParams {
    const void* q;
    const void* k;
    const void* v;
    void* o;
    long long bsq, bsk, bsv, bso;
    size_t ldq, ldk, ldv, ldo;
    int B, Tq, Tk, Hkv, G;
    const int* klen;
    const uint8_t* kmask;
    long long bsm;
    float sc;  // scale log2(e)
    int rows;                       // Tq G
    int rtiles, ksplit, total, per;  // row tiles, key ranges of one, work items, items per XCD
    float* part;                    // ksplit > 1: partial results [item][row of the tile][DH], then [item][row](m, l)
};

constexpr int XKT = 32;       // keys of a tile
constexpr float XRESCALE = 8.f;

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4v lds_s4v;
typedef __attribute__((address_space(3))) u32x4 lds_x4;
typedef __attribute__((address_space(3))) void* lds_ptr;

template <class E>
struct XMma;
template <>
struct XMma<_Float16> {
    static __device__ __forceinline__ floatx4 mul(u32x4 a, u32x4 b, floatx4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, half2v{(_Float16)a, (_Float16)b});
    }
};
template <>
struct XMma<__bf16> {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ floatx4 mul(u32x4 a, u32x4 b, floatx4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, b2{(__bf16)a, (__bf16)b});
    }
};

template <int N>
__device__ __forceinline__ void x_wait_vmcnt() {
    __builtin_amdgcn_s_waitcnt((N & 0xF) | (0x7 << 4) | (0xF << 8) | ((N >> 4) << 14));
}
// position of 16-byte chunk c of key row r: K is read 16 keys x one chunk at a time (eight neighbouring keys take eight
// positions), V four keys x a pair of chunks at a time (four neighbouring keys take four pairs)
__device__ __forceinline__ int k_swz(int c, int r) { return c ^ (r & 7); }
__device__ __forceinline__ int v_swz(int c, int r) { return c ^ (((r & 3) << 1) | ((r >> 2) & 1)); }

// QB 16-row blocks per wave; KW = 1: four waves with rows of their own share the tiles; KW = 4: four waves with the same
// rows, each with a quarter of the keys and tiles of its own, whose results meet in LDS
template <class E, int DH, int QB, int KW>
struct XCfg {
    static constexpr int RW = 16 * QB, RT = RW * 4 / KW;              // rows of a wave, of the workgroup
    static constexpr int PC = DH / 8;                                 // 16-byte chunks of a row
    static constexpr int TILE = XKT * DH * 2, STAGE = 2 * TILE;       // K tile, V tile
    static constexpr int NS = KW == 4 ? 2 : 4;                        // stages of a ring
    static constexpr int THREADS_PER_RING = 256 / KW;
    static constexpr int DMA = XKT * PC / THREADS_PER_RING;           // 16-byte pieces per thread, for K and for V each
    static constexpr int RING = NS * STAGE;
    static constexpr int BITS = 4 * 32 * 4;                           // each wave's mask windows: 2 x 16 words
    static constexpr int MERGE = KW == 4 ? 4 * RW * (DH + 2) * 4 : 0; // the waves' results
    static constexpr int LDS = (RING * KW > MERGE ? RING * KW : MERGE) + BITS;
};

template <class E, int DH, int QB, int KW>
__global__ __launch_bounds__(256) void k_cross_attn(const CrossParams p) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass drops a kernel template whose target builtins it cannot check
    using C = XCfg<E, DH, QB, KW>;
    using M = XMma<E>;
    extern __shared__ __attribute__((aligned(16))) uint8_t xlds[];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, c16 = lane & 15;
    // blocks go round the 8 XCDs: each takes a contiguous range of items, so that the row tiles of a key head share its L2
    const int item = (int)(blockIdx.x & 7) * p.per + (int)(blockIdx.x >> 3);
    if (item >= p.total) return;
    const int rt = item % p.rtiles, ks = item / p.rtiles % p.ksplit, bh = item / p.rtiles / p.ksplit;
    const int hk = bh % p.Hkv, b = bh / p.Hkv;
    const int L = p.klen ? max(0, min(p.klen[b], p.Tk)) : p.Tk;
    const int nt = (L + XKT - 1) / XKT;
    // this workgroup's tiles, this wave's tiles
    const int g0 = (int)((long long)nt * ks / p.ksplit), g1 = (int)((long long)nt * (ks + 1) / p.ksplit);
    const int t0 = KW == 1 ? g0 : g0 + (g1 - g0) * wv / 4, t1 = KW == 1 ? g1 : g0 + (g1 - g0) * (wv + 1) / 4;
    const uint8_t* mask = p.kmask ? p.kmask + (long long)b * p.bsm : nullptr;

    uint8_t* ring = xlds + (KW == 4 ? wv * C::RING : 0);
    const uint32_t lds_base = (uint32_t)(size_t)(__attribute__((address_space(3))) uint8_t*)ring;
    uint32_t* bits = reinterpret_cast<uint32_t*>(xlds + C::LDS - C::BITS) + wv * 32;

    // The keys of tile j as bits. With a mask: windows of 16 tiles (512 keys) in LDS, two of them, each wave its own.
    auto fill_window = [&](int w) {  // window w of this wave's tiles: tiles t0 + 16 w ..
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const long long key = (long long)(t0 + 16 * w) * XKT + 64 * i + lane;
            const unsigned long long m = __ballot(key < L && mask[key < L ? key : 0] != 0);
            if (lane == i) *reinterpret_cast<unsigned long long*>(bits + (w & 1) * 16 + 2 * i) = m;
        }
        __builtin_amdgcn_wave_barrier();
    };
    auto tile_bits = [&](int j) -> uint32_t {
        if (j >= t1) return 0u;
        if (mask) return __builtin_amdgcn_readfirstlane(bits[(j - t0) & 31]);
        const int left = L - j * XKT;
        return left >= XKT ? ~0u : (1u << left) - 1u;
    };

    // DMA of tile j: a thread's pieces are chunks of fixed rows; a masked row's offset is beyond every range
    const int tr = KW == 4 ? lane : (int)threadIdx.x;
    const uint8_t* kb = static_cast<const uint8_t*>(p.k) + ((long long)b * p.bsk + (long long)hk * DH) * 2;
    const uint8_t* vb = static_cast<const uint8_t*>(p.v) + ((long long)b * p.bsv + (long long)hk * DH) * 2;
    uint32_t ko[C::DMA], vo[C::DMA];
    int prow[C::DMA];
#pragma unroll
    for (int i = 0; i < C::DMA; i++) {
        const int pc = i * C::THREADS_PER_RING + tr, r = pc / C::PC, c = pc % C::PC;
        prow[i] = r;
        ko[i] = (uint32_t)(r * p.ldk * 2 + k_swz(c, r) * 16);
        vo[i] = (uint32_t)(r * p.ldv * 2 + v_swz(c, r) * 16);
    }
    auto dma = [&](int j, int stage) {
        if (mask && j < t1 && ((j - t0) & 15) == 0) fill_window((j - t0) >> 4);
        const int left = j < t1 ? min(XKT, L - j * XKT) : 0;
        const long long row0 = (long long)j * XKT;
        const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(kb + (j < t1 ? row0 * (long long)p.ldk * 2 : 0)), (short)0,
            left > 0 ? (int)((left - 1) * p.ldk * 2 + DH * 2) : 0, 0x00020000 /* raw */);
        const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(vb + (j < t1 ? row0 * (long long)p.ldv * 2 : 0)), (short)0,
            left > 0 ? (int)((left - 1) * p.ldv * 2 + DH * 2) : 0, 0x00020000);
        uint8_t* dst = ring + stage * C::STAGE + (KW == 4 ? 0 : wv * 1024);
        const uint32_t m = mask ? tile_bits(j) : ~0u;
#pragma unroll
        for (int i = 0; i < C::DMA; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_ptr)(dst + i * C::THREADS_PER_RING * 16), 16,
                                                     m >> prow[i] & 1 ? ko[i] : 0x7ffffff0u, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < C::DMA; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_ptr)(dst + C::TILE + i * C::THREADS_PER_RING * 16), 16,
                                                     m >> prow[i] & 1 ? vo[i] : 0x7ffffff0u, 0, 0, 0);
    };

    // Q: the B operands of S^T, lane (row c16, chunk 4 cc + g); rows past the last read row 0 and are not stored
    const int row0 = rt * C::RT + (KW == 4 ? 0 : wv * C::RW);
    u32x4 qf[QB][DH / 32];
#pragma unroll
    for (int qb = 0; qb < QB; qb++) {
        const int r = row0 + 16 * qb + c16, rr = r < p.rows ? r : 0, t = rr / p.G, h = hk * p.G + rr % p.G;
        const uint8_t* src = static_cast<const uint8_t*>(p.q) + ((long long)b * p.bsq + (long long)t * p.ldq + (long long)h * DH + 8 * g) * 2;
#pragma unroll
        for (int cc = 0; cc < DH / 32; cc++) qf[qb][cc] = *reinterpret_cast<const u32x4*>(src + 64 * cc);
    }

    floatx4 o[DH / 16][QB];
    float m[QB], mn[QB], l[QB];  // running maximum; its negative as subtracted (0 while the maximum is -inf); this lane's sum
#pragma unroll
    for (int qb = 0; qb < QB; qb++) {
        m[qb] = -INFINITY;
        mn[qb] = 0.f;
        l[qb] = 0.f;
#pragma unroll
        for (int db = 0; db < DH / 16; db++) o[db][qb] = floatx4{0.f, 0.f, 0.f, 0.f};
    }

#pragma unroll
    for (int s = 0; s < C::NS - 1; s++) dma(t0 + s, s);
    int stage = 0;
    for (int j = t0; j < t1; j++) {
        // tile j landed (past the last tile the copies go on with empty ranges, which keeps the count); every wave that
        // shares the ring is done with tile j - 1, whose stage is refilled
        x_wait_vmcnt<(C::NS - 2) * 2 * C::DMA>();
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
        if constexpr (KW == 1) __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (C::NS > 2) dma(j + C::NS - 1, stage == 0 ? C::NS - 1 : stage - 1);
        else dma(j + 1, stage ^ 1);
        const uint32_t bt = tile_bits(j);
        const uint32_t ka = lds_base + stage * C::STAGE, va = ka + C::TILE;
        floatx4 s[2][QB];
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
            const int r = 16 * kk + c16;
#pragma unroll
            for (int cc = 0; cc < DH / 32; cc++) {
                const u32x4 kf = *reinterpret_cast<const lds_x4*>((size_t)(ka + r * DH * 2 + k_swz(4 * cc + g, r) * 16));
#pragma unroll
                for (int qb = 0; qb < QB; qb++)
                    s[kk][qb] = M::mul(kf, qf[qb][cc], cc == 0 ? floatx4{0.f, 0.f, 0.f, 0.f} : s[kk][qb]);
            }
        }
        if (bt != ~0u) {
#pragma unroll
            for (int kk = 0; kk < 2; kk++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (!(bt >> (16 * kk + 4 * g + i) & 1))
#pragma unroll
                        for (int qb = 0; qb < QB; qb++) s[kk][qb][i] = -INFINITY;
        }
        float top[QB];
        bool moves = false;
#pragma unroll
        for (int qb = 0; qb < QB; qb++) {
            float t = fmaxf(s[0][qb][0], s[1][qb][0]);
#pragma unroll
            for (int i = 1; i < 4; i++) t = fmaxf(t, fmaxf(s[0][qb][i], s[1][qb][i]));
            top[qb] = t * p.sc;
            moves |= top[qb] > m[qb] + XRESCALE;  // from -inf: any score that is not
        }
        if (__any(moves)) {
#pragma unroll
            for (int qb = 0; qb < QB; qb++) {
                const float t = quad_max(top[qb]);
                if (t > m[qb]) {
                    const float f = __builtin_amdgcn_exp2f(m[qb] - t);
                    m[qb] = t;
                    mn[qb] = -t;
                    l[qb] *= f;
#pragma unroll
                    for (int db = 0; db < DH / 16; db++) o[db][qb] *= f;
                }
            }
        }
        u32x4 pf[QB];
#pragma unroll
        for (int qb = 0; qb < QB; qb++) {
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                e[i] = __builtin_amdgcn_exp2f(fmaf(s[i / 4][qb][i % 4], p.sc, mn[qb]));
                l[qb] += e[i];
            }
#pragma unroll
            for (int i = 0; i < 4; i++) pf[qb][i] = M::pack(e[2 * i], e[2 * i + 1]);
        }
#pragma unroll
        for (int db = 0; db < DH / 16; db++) {
            // lane: keys 16 jh + 4 g .. + 3 of dimension 16 db + c16, from the rows and 8-byte pieces the 16 lanes name
            const int r = 4 * g + (c16 >> 2), c = 2 * db + ((c16 & 3) >> 1), h8 = (c16 & 1) * 8;
            const s4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v*)(size_t)(va + r * DH * 2 + v_swz(c, r) * 16 + h8));
            const s4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v*)(size_t)(va + (r + 16) * DH * 2 + v_swz(c, r + 16) * 16 + h8));
            const u32x2 a = __builtin_bit_cast(u32x2, lo), d = __builtin_bit_cast(u32x2, hi);
            const u32x4 vf = {a[0], a[1], d[0], d[1]};
#pragma unroll
            for (int qb = 0; qb < QB; qb++) o[db][qb] = M::mul(vf, pf[qb], o[db][qb]);
        }
        stage = stage == C::NS - 1 ? 0 : stage + 1;
    }
    x_wait_vmcnt<0>();  // no copy into LDS outlives its ring

#pragma unroll
    for (int qb = 0; qb < QB; qb++) l[qb] = quad_sum(l[qb]);

    if constexpr (KW == 1) {
#pragma unroll
        for (int qb = 0; qb < QB; qb++) {
            const int r = row0 + 16 * qb + c16;
            if (r >= p.rows) continue;
            if (p.ksplit > 1) {
                const size_t at = (size_t)item * C::RT + (wv * C::RW + 16 * qb + c16);
#pragma unroll
                for (int db = 0; db < DH / 16; db++) *reinterpret_cast<floatx4*>(p.part + at * DH + 16 * db + 4 * g) = o[db][qb];
                if (g == 0) *reinterpret_cast<float2*>(p.part + (size_t)p.total * C::RT * DH + at * 2) = make_float2(m[qb], l[qb]);
                continue;
            }
            const float inv = l[qb] > 0.f || l[qb] != l[qb] ? 1.f / l[qb] : 0.f;  // no key: zeros
            const int t = r / p.G, h = hk * p.G + r % p.G;
            uint8_t* dst = static_cast<uint8_t*>(p.o) + ((long long)b * p.bso + (long long)t * p.ldo + (long long)h * DH + 4 * g) * 2;
#pragma unroll
            for (int db = 0; db < DH / 16; db++)
                *reinterpret_cast<u32x2*>(dst + 32 * db) =
                    u32x2{M::pack(o[db][qb][0] * inv, o[db][qb][1] * inv), M::pack(o[db][qb][2] * inv, o[db][qb][3] * inv)};
        }
    } else {
        // the four waves' results of the same 16 QB rows
        __syncthreads();
        float* ro = reinterpret_cast<float*>(xlds);
        float* rml = ro + 4 * C::RW * DH;
#pragma unroll
        for (int qb = 0; qb < QB; qb++) {
#pragma unroll
            for (int db = 0; db < DH / 16; db++)
                *reinterpret_cast<floatx4*>(ro + (wv * C::RW + 16 * qb + c16) * DH + 16 * db + 4 * g) = o[db][qb];
            if (g == 0) {
                rml[(wv * C::RW + 16 * qb + c16) * 2] = m[qb];
                rml[(wv * C::RW + 16 * qb + c16) * 2 + 1] = l[qb];
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < C::RW * DH / 4; i += 256) {
            const int rl = i / (DH / 4), d = (i % (DH / 4)) * 4, r = row0 + rl;
            if (r >= p.rows) break;  // rows ascend with i
            float mm = -INFINITY, ll = 0.f;
#pragma unroll
            for (int w = 0; w < 4; w++) mm = fmaxf(mm, rml[(w * C::RW + rl) * 2]);
            const float me = mm == -INFINITY ? 0.f : mm;
            floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float f = __builtin_amdgcn_exp2f(rml[(w * C::RW + rl) * 2] - me);
                ll += f * rml[(w * C::RW + rl) * 2 + 1];
                acc += f * *reinterpret_cast<const floatx4*>(ro + (w * C::RW + rl) * DH + d);
            }
            if (p.ksplit > 1) {
                const size_t at = (size_t)item * C::RT + rl;
                *reinterpret_cast<floatx4*>(p.part + at * DH + d) = acc;
                if (d == 0) *reinterpret_cast<float2*>(p.part + (size_t)p.total * C::RT * DH + at * 2) = make_float2(mm, ll);
                continue;
            }
            const float inv = ll > 0.f || ll != ll ? 1.f / ll : 0.f;
            const int t = r / p.G, h = hk * p.G + r % p.G;
            uint8_t* dst = static_cast<uint8_t*>(p.o) + ((long long)b * p.bso + (long long)t * p.ldo + (long long)h * DH + d) * 2;
            *reinterpret_cast<u32x2*>(dst) = u32x2{M::pack(acc[0] * inv, acc[1] * inv), M::pack(acc[2] * inv, acc[3] * inv)};
        }
    }
#endif
}

// the key ranges of each row joined, in the ranges' order: DH / 4 lanes to a row
template <class E, int DH>
__global__ __launch_bounds__(256) void k_cross_merge(const CrossParams p, int RT) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, n = (size_t)p.B * p.Hkv * p.rows * (DH / 4);
    if (i >= n) return;
    const int d = (int)(i % (DH / 4)) * 4;
    const size_t rr = i / (DH / 4), bh = rr / p.rows;
    const int r = (int)(rr - bh * p.rows), rt = r / RT, rl = r - rt * RT, hk = (int)(bh % p.Hkv), b = (int)(bh / p.Hkv);
    const float* ml = p.part + (size_t)p.total * RT * DH;
    const size_t at0 = ((bh * p.ksplit) * p.rtiles + rt) * RT + rl, step = (size_t)p.rtiles * RT;
    float mm = -INFINITY, ll = 0.f;
    for (int k = 0; k < p.ksplit; k++) mm = fmaxf(mm, ml[(at0 + k * step) * 2]);
    const float me = mm == -INFINITY ? 0.f : mm;
    floatx4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < p.ksplit; k++) {
        const float2 e = *reinterpret_cast<const float2*>(ml + (at0 + k * step) * 2);
        const float f = __builtin_amdgcn_exp2f(e.x - me);
        ll += f * e.y;
        acc += f * *reinterpret_cast<const floatx4*>(p.part + (at0 + k * step) * DH + d);
    }
    const float inv = ll > 0.f || ll != ll ? 1.f / ll : 0.f;
    const int t = r / p.G, h = hk * p.G + r % p.G;
    uint8_t* dst = static_cast<uint8_t*>(p.o) + ((long long)b * p.bso + (long long)t * p.ldo + (long long)h * DH + d) * 2;
    *reinterpret_cast<u32x2*>(dst) =
        u32x2{XMma<E>::pack(acc[0] * inv, acc[1] * inv), XMma<E>::pack(acc[2] * inv, acc[3] * inv)};
}

// The form of a call: rows and key ranges per workgroup.
struct XForm {
    int qb, kw, rt, ksplit;
};
static XForm cross_form(int B, int Tq, int Tk, int Hq, int Hkv, int Dh) {
    const long rows = (long)Tq * (Hq / Hkv), heads = (long)B * Hkv, cus = cu_count(), tiles = (Tk + XKT - 1) / XKT;
    if (rows <= 16) {
        // one row block: the waves split the keys, and ranges of at least 8 tiles (2 per wave) fill the chip
        const long ks = std::min<long>({(2 * cus + heads - 1) / heads, tiles / 8, 256});
        return {1, 4, 16, (int)std::max<long>(1, ks)};
    }
    const int qb = rows * heads >= 128 * cus ? 2 : 1, rt = 64 * qb;
    const long units = (rows + rt - 1) / rt * heads;
    const long ks = units >= cus ? 1 : std::min<long>({2 * cus / units, tiles / 8, 256});
    return {qb, 1, rt, (int)std::max<long>(1, ks)};
}
size_t cross_attn_workspace(int B, int Tq, int Tk, int Hq, int Hkv, int Dh) {
    const XForm f = cross_form(B, Tq, Tk, Hq, Hkv, Dh);
    if (f.ksplit == 1) return 0;
    const size_t rtiles = ((size_t)Tq * (Hq / Hkv) + f.rt - 1) / f.rt;
    return (size_t)B * Hkv * f.ksplit * rtiles * f.rt * (Dh + 2) * sizeof(float);
}

template <class E, int DH, int QB, int KW>
static hipError_t cross_launch(CrossParams p, hipStream_t s) {
    using C = XCfg<E, DH, QB, KW>;
    p.rtiles = (p.rows + C::RT - 1) / C::RT;
    p.total = p.B * p.Hkv * p.ksplit * p.rtiles;
    p.per = (p.total + 7) / 8;
    hipLaunchKernelGGL((k_cross_attn<E, DH, QB, KW>), dim3(p.per * 8), dim3(256), C::LDS, s, p);
    if (hipError_t e = hipGetLastError()) return e;
    if (p.ksplit == 1) return hipSuccess;
    const size_t n = (size_t)p.B * p.Hkv * p.rows * (DH / 4);
    hipLaunchKernelGGL((k_cross_merge<E, DH>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, p, C::RT);
    return hipGetLastError();
}
template <class E, int DH>
static hipError_t cross_of(const CrossParams& p, const XForm& f, hipStream_t s) {
    if (f.kw == 4) return cross_launch<E, DH, 1, 4>(p, s);
    if (f.qb == 1) return cross_launch<E, DH, 1, 1>(p, s);
    return cross_launch<E, DH, 2, 1>(p, s);
}

hipError_t launch_cross_attn(const CrossLaunch& c, hipStream_t s) {
    XForm f = cross_form(c.B, c.Tq, c.Tk, c.Hq, c.Hkv, c.Dh);
    if (c.ws_bytes < cross_attn_workspace(c.B, c.Tq, c.Tk, c.Hq, c.Hkv, c.Dh) || !c.ws) f.ksplit = 1;
    CrossParams p{};
    p.q = c.q;
    p.k = c.k;
    p.v = c.v;
    p.o = c.out;
    p.bsq = c.bsq;
    p.bsk = c.bsk;
    p.bsv = c.bsv;
    p.bso = c.bso;
    p.ldq = c.ldq;
    p.ldk = c.ldk;
    p.ldv = c.ldv;
    p.ldo = c.ldo;
    p.B = c.B;
    p.Tq = c.Tq;
    p.Tk = c.Tk;
    p.Hkv = c.Hkv;
    p.G = c.Hq / c.Hkv;
    p.klen = c.klen;
    p.kmask = c.kmask;
    p.bsm = c.bsm;
    p.sc = c.scale * LOG2E;
    p.rows = c.Tq * p.G;
    p.ksplit = f.ksplit;
    p.part = static_cast<float*>(c.ws);
    if (c.dt == DT::F16) return c.Dh == 64 ? cross_of<_Float16, 64>(p, f, s) : cross_of<_Float16, 128>(p, f, s);
    return c.Dh == 64 ? cross_of<__bf16, 64>(p, f, s) : cross_of<__bf16, 128>(p, f, s);
}

}  // namespace kiln
