// Attention of B x Tq queries to Tk encoder states of another length (kiln_cross_attn): O = softmax(s Q K^T) V per head,
// Hkv key heads each shared by G = Hq / Hkv query heads, keys bounded by a length and a mask per item. fp16 or bf16 rows,
// read where they lie: no prepare pass (a context of a few hundred states is used once per layer).
//
// The G query heads of a key head and their Tq tokens are the rows of one problem, r = t G + g, so that a key is read once
// for all of them. Scores are computed transposed, S^T = K Q^T, and O^T = V^T P^T, with v_mfma_f32_16x16x32: a lane of the
// S^T accumulators holds eight of a 32-key tile's keys for one row, which is the B operand of the second product as it
// is, if V's keys come in the same order: two transposing LDS reads per 16 dimensions.
//
// Keys come in tiles of 32: K and V rows go to LDS by buffer DMA, 16 bytes a lane, the chunks of a row permuted (k_swz, v_swz) so
// that both kinds of operand read lie in all banks. Rows past the length, and V's masked rows, lie outside the descriptor's range
// and arrive as zeros, whatever they hold: their scores are set to -inf by the tile's bit mask, and 0 times an infinity or a NaN
// never happens.
//
// Softmax in one pass: running maximum m and sum l per row in fp32, in units of log2. The maximum moves (and O and l are
// rescaled) only when a tile's exceeds it by more than 8, so most tiles need no exchange between lanes. P is taken as 2^lift times
// the weight and rounded to the inputs' type, half a step of it (2^-11 fp16, 2^-8 bf16) per weight, as far off as the output's own
// rounding. The factor is in O and l alike. In fp16 it is 2^7: P is 2^15 at most, and weights down to 2^-32 of the largest count
// (2^-25 without), of which a long context may have enough: 2^17 keys at 2^-25.5 are 2^-8.5 of the output. bf16 has fp32's
// exponents, for weights and for values: there P sums to less than 1 over all keys (lift = -9 - log2 Tk, to the integer below), so that no
// finite value overflows on its way; at the other end, products with values below 2^-117 Tk leave fp32's normal range.
// The exponent is one fma, s sc + (lift - m): exact products against a rounded m, off by half a unit of m's last place for all
// keys of a row alike. While |m| is at most 2^20 that is a factor of 2^(1/16), in O and l alike; beyond, where it would grow out of
// the weights' range, products are rounded as m was before it is taken off (`far`: a branch that a wave takes or not).
//
// Bound, with many rows, by matrix and vector work in turn (16 multiply-adds, 16 exponentials, 8 conversions and some 14 maxima after
// 16 and before 18 products per wave and tile of 32 rows, Dh 128): 2 x 4096 x 4096, 16 heads of 128, 277 us, 990 TFLOP/s, the matrix
// cores busy 47% of the time; 2 x 4096 x 512 51 us, of which Q in and O out are ~15. With few rows by the keys' bytes: 8 x 1 x 8192,
// 16 heads on 4 of 128, 134 MB in 25 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "attn16.hpp"
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
    float sc;                       // scale log2(e)
    float lift;                     // log2 of the weights' factor
    int rows;                       // Tq G
    int rtiles, ksplit, ct;         // row tiles, key ranges of one (ct tiles each), ..
    int total, per;                 // .. work items, items per XCD
    float* part;                    // ksplit > 1: partial results [item][row of the tile][DH], then [item][row](m, l)
};

// A workgroup's geometry: NW waves of 16 QB rows. SHARED: the waves have rows of their own and share a ring of NS tiles.
// Otherwise every wave has the same rows, a ring and a share of the keys of its own; the results of four meet in LDS.
template <int DH_, int QB_, int NW_, bool SHARED_, int NS_>
struct XCfg {
    static constexpr int DH = DH_, QB = QB_, NW = NW_, NS = NS_;
    static constexpr bool SHARED = SHARED_;
    static constexpr int THREADS = 64 * NW, RW = 16 * QB, RT = SHARED ? RW * NW : RW;  // rows of a wave, of the workgroup
    static constexpr int PC = DH / 8;                                  // 16-byte chunks of a row
    static constexpr int TILE = XKT * DH * 2, STAGE = 2 * TILE;        // K tile, V tile
    static constexpr int RTHREADS = SHARED ? THREADS : 64;             // threads that fill a ring
    static constexpr int DMA = XKT * PC / RTHREADS;                    // 16-byte pieces per thread, for K and for V each
    static constexpr int RING = NS * STAGE, RINGS = SHARED ? RING : RING * NW;
    static constexpr int BITS = NW * 32 * 4;                           // each wave's mask windows: 2 x 16 words
    static constexpr int MERGE = !SHARED && NW > 1 ? NW * RW * (DH + 2) * 4 : 0;
    static constexpr int LDS = (RINGS > MERGE ? RINGS : MERGE) + BITS;
    static constexpr int WAVES = QB == 1 && NW > 1 && LDS <= 40 * 1024 ? 4 : LDS <= 80 * 1024 || NW == 1 || NW == 8 ? 2 : 1;  // per SIMD that registers have to allow
};

template <class E, class C, bool MASK>
__global__ __launch_bounds__(C::THREADS, C::WAVES) void k_cross_attn(const CrossParams p) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass drops a kernel template whose target builtins it cannot check
    using M = XMma<E>;
    constexpr int DH = C::DH, QB = C::QB;
    extern __shared__ __attribute__((aligned(16))) uint8_t xlds[];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, c16 = lane & 15;
    // blocks go round the 8 XCDs: each takes a contiguous range of items, so that the row tiles of a key head share its L2
    // (the key heads of a row tile side by side instead: B = 2, 4096 x 4096, 16 heads of 128 295 -> 314 us)
    const int item = (int)(blockIdx.x & 7) * p.per + (int)(blockIdx.x >> 3);
    if (item >= p.total) return;
    const int rt = item % p.rtiles, ks = item / p.rtiles % p.ksplit, bh = item / p.rtiles / p.ksplit;
    const int hk = bh % p.Hkv, b = bh / p.Hkv;
    const int L = p.klen ? max(0, min(p.klen[b], p.Tk)) : p.Tk;
    const int nt = (L + XKT - 1) / XKT;
    // this workgroup's tiles, this wave's tiles
    const int g0 = ks * p.ct, g1 = min(nt, g0 + p.ct);
    if (p.ksplit > 1 && g0 >= g1) return;  // the merge leaves ranges past the item's keys out
    const int t0 = C::SHARED ? g0 : g0 + max(g1 - g0, 0) * wv / C::NW, t1 = C::SHARED ? g1 : g0 + max(g1 - g0, 0) * (wv + 1) / C::NW;

    uint8_t* ring = xlds + (C::SHARED ? 0 : wv * C::RING);
    const uint32_t lds_base = (uint32_t)(size_t)(__attribute__((address_space(3))) uint8_t*)ring;
    const uint8_t* mask = MASK ? p.kmask + (long long)b * p.bsm : nullptr;
    uint32_t* bits = reinterpret_cast<uint32_t*>(xlds + C::LDS - C::BITS) + wv * 32;

    // The keys of tile j < t1 as bits. With a mask: windows of 16 tiles (512 keys) in LDS, two of them, each wave its own.
    auto fill_window = [&](int w) {  // window w of this wave's tiles: tiles t0 + 16 w .., at least one key
        const long long key0 = (long long)(t0 + 16 * w) * XKT + lane;
        uint8_t byte[8];  // all loads before the first is looked at
#pragma unroll
        for (int i = 0; i < 8; i++) byte[i] = mask[min(key0 + 64 * i, (long long)L - 1)];
        uint32_t word = 0;  // lane j < 16: the window's word j, stored as what tile_bits reads
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const unsigned long long m = __ballot((byte[i] != 0) & (key0 + 64 * i < L));
            if (lane >> 1 == i) word = lane & 1 ? (uint32_t)(m >> 32) : (uint32_t)m;
        }
        if (lane < 16) bits[(w & 1) * 16 + lane] = word;
        __builtin_amdgcn_wave_barrier();
    };
    auto tile_bits = [&](int j) -> uint32_t {
        if constexpr (MASK) return __builtin_amdgcn_readfirstlane(bits[(j - t0) & 31]);
        const int left = L - j * XKT;
        return left >= XKT ? ~0u : (1u << left) - 1u;
    };

    // DMA of the tiles' K and V in turn: a thread's pieces are chunks of fixed rows of a tile; the descriptor's range ends with
    // the item's last row (empty past the last tile), and a masked V row's offset is beyond every range
    struct Stream {
        const uint8_t* src;     // the next tile to copy
        uint32_t ld2;           // bytes from row to row
        int j;                  // its index
        uint32_t off[C::DMA];
    } kst, vst;
    kst.ld2 = (uint32_t)p.ldk * 2;
    vst.ld2 = (uint32_t)p.ldv * 2;
    kst.src = static_cast<const uint8_t*>(p.k) + ((long long)b * p.bsk + (long long)hk * DH) * 2 + (long long)t0 * XKT * kst.ld2;
    vst.src = static_cast<const uint8_t*>(p.v) + ((long long)b * p.bsv + (long long)hk * DH) * 2 + (long long)t0 * XKT * vst.ld2;
    kst.j = vst.j = t0;
    int prow[C::DMA];
#pragma unroll
    for (int i = 0; i < C::DMA; i++) {
        const int pc = i * C::RTHREADS + (C::SHARED ? (int)threadIdx.x : lane), r = pc / C::PC, c = pc % C::PC;
        prow[i] = r;
        kst.off[i] = r * kst.ld2 + k_swz<DH>(c, r) * 16;
        vst.off[i] = r * vst.ld2 + v_swz<DH>(c, r) * 16;
    }
    // V's copies leave masked rows out; K's need not: a masked key's score is replaced, whatever it came to. So the first K tiles
    // are under way while the mask is read.
    auto copy = [&](Stream& t, uint32_t at, auto masked) {
        constexpr bool M_ = decltype(masked)::value;
        uint32_t m = ~0u;
        const int left = t.j < t1 ? min(XKT, L - t.j * XKT) : 0;
        if constexpr (M_) {
            if (left > 0) {
                if (((t.j - t0) & 15) == 0) fill_window((t.j - t0) >> 4);
                m = tile_bits(t.j);
            }
        }
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(t.src), (short)0, left > 0 ? (int)((left - 1) * t.ld2 + DH * 2) : 0, 0x00020000 /* raw */);
        uint8_t* dst = ring + at + (C::SHARED ? wv * 1024 : 0);
#pragma unroll
        for (int i = 0; i < C::DMA; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(dst + i * C::RTHREADS * 16), 16,
                                                     !M_ || (m >> prow[i] & 1) ? t.off[i] : 0x7ffffff0u, 0, 0, 0);
        if (t.j + 1 < t1) t.src += (size_t)XKT * t.ld2;
        t.j++;
    };
    auto copy_k = [&](int stage) { copy(kst, stage * C::STAGE, std::false_type{}); };
    auto copy_v = [&](int stage) { copy(vst, stage * C::STAGE + C::TILE, std::integral_constant<bool, MASK>{}); };

    // Q: the B operands of S^T, lane (row c16, chunk 4 cc + g); rows past the last read row 0 and are not stored
    const int row0 = rt * C::RT + (C::SHARED ? wv * C::RW : 0);
    u32x4 qf[QB][DH / 32];
#pragma unroll
    for (int qb = 0; qb < QB; qb++) {
        const int r = row0 + 16 * qb + c16, rr = r < p.rows ? r : 0, t = rr / p.G, h = hk * p.G + rr % p.G;
        const uint8_t* src = static_cast<const uint8_t*>(p.q) + ((long long)b * p.bsq + (long long)t * p.ldq + (long long)h * DH + 8 * g) * 2;
#pragma unroll
        for (int cc = 0; cc < DH / 32; cc++) qf[qb][cc] = *reinterpret_cast<const u32x4*>(src + 64 * cc);
    }

    floatx4 o[DH / 16][QB], l[QB];  // l: every register of a lane holds its row's sum (P^T times ones)
    const float lift = std::is_same<E, _Float16>::value ? XLIFT16 : p.lift;
    float m[QB], mn[QB];            // running maximum; lift minus it (lift while it is -inf)
    bool far = false;               // a row's maximum is far from zero: scores come to the weights less it, in log2
#pragma unroll
    for (int qb = 0; qb < QB; qb++) {
        m[qb] = -INFINITY;
        mn[qb] = lift;
        l[qb] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int db = 0; db < DH / 16; db++) o[db][qb] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    const uint32_t one2 = M::pack(1.f, 1.f);
    const u32x4 ones = {one2, one2, one2, one2};
    // operand addresses within a stage; the chunks' permutation is the same for rows 16 apart
    uint32_t kaddr[DH / 32], vaddr[DH / 16];
#pragma unroll
    for (int cc = 0; cc < DH / 32; cc++) kaddr[cc] = lds_base + c16 * DH * 2 + k_swz<DH>(4 * cc + g, c16) * 16;
    // V: keys 16 jh + 4 g .. + 3 of dimension 16 db + c16, from the rows and 8-byte pieces that the 16 lanes name
    const int vr = 4 * g + (c16 >> 2);
#pragma unroll
    for (int db = 0; db < DH / 16; db++)
        vaddr[db] = lds_base + C::TILE + vr * DH * 2 + v_swz<DH>(2 * db + ((c16 & 3) >> 1), vr) * 16 + (c16 & 1) * 8;

    // pieces of a tile's work
    auto read_k = [&](uint32_t st, u32x4 (&kf)[2][DH / 32]) {
#pragma unroll
        for (int kk = 0; kk < 2; kk++)
#pragma unroll
            for (int cc = 0; cc < DH / 32; cc++)
                kf[kk][cc] = *reinterpret_cast<const lds_x4*>((size_t)(kaddr[cc] + st + kk * 16 * DH * 2));
    };
    auto read_v = [&](uint32_t st, int db) {
        const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v*)(size_t)(vaddr[db] + st)));
        const u32x2 d = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v*)(size_t)(vaddr[db] + st + 16 * DH * 2)));
        return u32x4{a[0], a[1], d[0], d[1]};
    };
    auto scores = [&](const u32x4 (&kf)[2][DH / 32], floatx4 (&s)[2][QB]) {
#pragma unroll
        for (int cc = 0; cc < DH / 32; cc++)
#pragma unroll
            for (int kk = 0; kk < 2; kk++)
#pragma unroll
                for (int qb = 0; qb < QB; qb++)
                    s[kk][qb] = M::mul(kf[kk][cc], qf[qb][cc], cc == 0 ? floatx4{0.f, 0.f, 0.f, 0.f} : s[kk][qb]);
    };
    auto hide = [&](int j, floatx4 (&s)[2][QB]) {
        const uint32_t bt = tile_bits(j);
        if (bt == ~0u) return;
#pragma unroll
        for (int kk = 0; kk < 2; kk++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (!(bt >> (16 * kk + 4 * g + i) & 1))
#pragma unroll
                    for (int qb = 0; qb < QB; qb++) s[kk][qb][i] = -INFINITY;
    };
    auto largest = [&](const floatx4 (&s)[2][QB], float (&top)[QB]) {
#pragma unroll
        for (int qb = 0; qb < QB; qb++) {
            float t = fmaxf(s[0][qb][0], s[1][qb][0]);
#pragma unroll
            for (int i = 1; i < 4; i++) t = fmaxf(fmaxf(t, s[0][qb][i]), s[1][qb][i]);
            top[qb] = t * p.sc;
        }
    };
    auto rescale = [&](const float (&top)[QB], floatx4 (&s)[2][QB]) {
#pragma clang fp contract(off)  // tops are rounded products, and so are far scores, which are then at most 8 above m
        bool moves = false;
#pragma unroll
        for (int qb = 0; qb < QB; qb++) moves |= top[qb] - m[qb] > XRESCALE;  // from -inf: any score that is not
        if (__any(moves)) {
            bool big = false;
#pragma unroll
            for (int qb = 0; qb < QB; qb++) {
                const float t = fmaxf(m[qb], quad_max(top[qb]));
                const float f = t > m[qb] ? __builtin_amdgcn_exp2f(m[qb] - t) : 1.f;
                m[qb] = t;
                big |= fabsf(t) > XFAR && t != -INFINITY;
                l[qb] *= f;
#pragma unroll
                for (int db = 0; db < DH / 16; db++) o[db][qb] *= f;
            }
            far = __any(big);
#pragma unroll
            for (int qb = 0; qb < QB; qb++) mn[qb] = far || m[qb] == -INFINITY ? lift : lift - m[qb];
        }
        if (far) {
#pragma unroll
            for (int qb = 0; qb < QB; qb++)
#pragma unroll
                for (int i = 0; i < 8; i++)
                    s[i / 4][qb][i % 4] = s[i / 4][qb][i % 4] * p.sc - (m[qb] == -INFINITY ? 0.f : m[qb]);
        }
    };
    auto weights = [&](const floatx4 (&s)[2][QB], u32x4 (&pf)[QB]) {
        const float sc = far ? 1.f : p.sc;
#pragma unroll
        for (int qb = 0; qb < QB; qb++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                pf[qb][i] = M::pack(__builtin_amdgcn_exp2f(fmaf(s[i / 2][qb][2 * i % 4], sc, mn[qb])),
                                    __builtin_amdgcn_exp2f(fmaf(s[i / 2][qb][2 * i % 4 + 1], sc, mn[qb])));
    };

    if constexpr (C::SHARED) {
        // A step computes the scores of tile j + 1 ahead of the weights and products of tile j. It would let the scores' products run
        // beside the exponentials, but the branch around `hide` and the loop's break part them: as compiled, a wave's matrix and vector
        // work follow each other, and overlap only with another wave's. K of tile j + 1 and V of tile j landed (past the
        // last tile the copies go on with empty ranges, which keeps the count); every wave is done with K of tile j and V of tile
        // j - 1, whose places take K of tile j + NS and V of tile j + NS - 1. Stages are constants: the reads' offsets too.
        constexpr int NS = C::NS;
        static_assert(NS % 2 == 0, "the scores' two sets go with the stages");
        floatx4 s[2][2][QB];
        float top[QB];
        u32x4 kf[2][DH / 32], vf[DH / 16], pf[QB];
        copy_k(0);
#pragma unroll
        for (int i = 1; i < NS; i++) {
            copy_k(i);
            copy_v(i - 1);
        }
        x_wait_vmcnt<2 * (NS - 1) * C::DMA>();
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        if (t0 < t1) {
            read_k(0, kf);
            scores(kf, s[0]);
            hide(t0, s[0]);
            largest(s[0], top);
        }
        auto step = [&](int j, auto parity, auto st) {  // st: the stage of tile j, a constant or not
            constexpr int cur = decltype(parity)::value;
            x_wait_vmcnt<2 * (NS - 2) * C::DMA>();
            __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            copy_k(st);
            copy_v((st + NS - 1) % NS);
            read_k((st + 1) % NS * C::STAGE, kf);
#pragma unroll
            for (int db = 0; db < DH / 16; db++) vf[db] = read_v(st * C::STAGE, db);
            rescale(top, s[cur]);
            __builtin_amdgcn_sched_barrier(0);
            weights(s[cur], pf);
            scores(kf, s[cur ^ 1]);
            __builtin_amdgcn_sched_barrier(0);
            if (j + 1 < t1) hide(j + 1, s[cur ^ 1]);
#pragma unroll
            for (int qb = 0; qb < QB; qb++) l[qb] = M::mul(ones, pf[qb], l[qb]);
#pragma unroll
            for (int db = 0; db < DH / 16; db++)
#pragma unroll
                for (int qb = 0; qb < QB; qb++) o[db][qb] = M::mul(vf[db], pf[qb], o[db][qb]);
            largest(s[cur ^ 1], top);
        };
        using P0 = std::integral_constant<int, 0>;
        using P1 = std::integral_constant<int, 1>;
        if constexpr (QB == 1) {  // the compiler spills 16-row waves' registers in the loop of four
            for (int j = t0, st = 0; j < t1; j += 2, st = (st + 2) % NS) {
                step(j, P0{}, st);
                if (j + 1 >= t1) break;
                step(j + 1, P1{}, st + 1);
            }
        } else {
            static_assert(NS == 4, "the loop names its stages");
            for (int j = t0; j < t1; j += 4) {
                step(j, P0{}, P0{});
                if (j + 1 >= t1) break;
                step(j + 1, P1{}, P1{});
                if (j + 2 >= t1) break;
                step(j + 2, P0{}, std::integral_constant<int, 2>{});
                if (j + 3 >= t1) break;
                step(j + 3, P1{}, std::integral_constant<int, 3>{});
            }
        }
    } else {
        int stage = 0;
        auto next = [](int i) { return i == C::NS - 1 ? 0 : i + 1; };
#pragma unroll
        for (int i = 0; i < C::NS - 1; i++) {
            copy_k(i);
            copy_v(i);
        }
        for (int j = t0; j < t1; j++) {
            x_wait_vmcnt<(C::NS - 2) * 2 * C::DMA>();
            __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): this wave is done with tile j - 1, whose stage is refilled
            __builtin_amdgcn_sched_barrier(0);
            const int into = stage == 0 ? C::NS - 1 : stage - 1;
            copy_k(into);
            copy_v(into);
            const uint32_t st = stage * C::STAGE;
            floatx4 s[2][QB];
            float top[QB];
            u32x4 kf[2][DH / 32], pf[QB];
            read_k(st, kf);
            scores(kf, s);
            hide(j, s);
            largest(s, top);
            rescale(top, s);
            weights(s, pf);
#pragma unroll
            for (int qb = 0; qb < QB; qb++) l[qb] = M::mul(ones, pf[qb], l[qb]);
#pragma unroll
            for (int db = 0; db < DH / 16; db++) {
                const u32x4 vf = read_v(st, db);
#pragma unroll
                for (int qb = 0; qb < QB; qb++) o[db][qb] = M::mul(vf, pf[qb], o[db][qb]);
            }
            stage = next(stage);
        }
    }
    x_wait_vmcnt<0>();  // no copy into LDS outlives its ring

    auto store4 = [&](int r, int d, float a0, float a1, float a2, float a3) {
        const int t = r / p.G, h = hk * p.G + r % p.G;
        uint8_t* dst = static_cast<uint8_t*>(p.o) + ((long long)b * p.bso + (long long)t * p.ldo + (long long)h * DH + d) * 2;
        *reinterpret_cast<u32x2*>(dst) = u32x2{M::pack(a0, a1), M::pack(a2, a3)};
    };
    if constexpr (C::SHARED || C::NW == 1) {
        if (p.ksplit > 1) {
#pragma unroll
            for (int qb = 0; qb < QB; qb++) {
                const int r = row0 + 16 * qb + c16;
                if (r >= p.rows) continue;
                const size_t at = (size_t)item * C::RT + (r - rt * C::RT);
#pragma unroll
                for (int db = 0; db < DH / 16; db++) *reinterpret_cast<floatx4*>(p.part + at * DH + 16 * db + 4 * g) = o[db][qb];
                if (g == 0) *reinterpret_cast<float2*>(p.part + (size_t)p.total * C::RT * DH + at * 2) = make_float2(m[qb], l[qb][0]);
            }
            return;
        }
        // rows leave through LDS, whole and 16 bytes a lane (8-byte pieces of 16 rows per store: 10 of 57 us in the same case);
        // a row's chunks lie permuted by its number
        static_assert(C::RW * DH * 2 * C::NW <= C::RINGS, "the waves' rows fit in the rings");
        uint8_t* stg = xlds + wv * C::RW * DH * 2;
        if constexpr (C::SHARED) __builtin_amdgcn_s_barrier();  // every wave is done with the ring, and its copies landed
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int qb = 0; qb < QB; qb++) {
            const int r = 16 * qb + c16;
            const float inv = l[qb][0] > 0.f || l[qb][0] != l[qb][0] ? 1.f / l[qb][0] : 0.f;  // no key: zeros
#pragma unroll
            for (int db = 0; db < DH / 16; db++)
                *reinterpret_cast<u32x2*>(stg + r * DH * 2 + ((2 * db + (g >> 1)) ^ (r & (C::PC - 1))) * 16 + (g & 1) * 8) =
                    u32x2{M::pack(o[db][qb][0] * inv, o[db][qb][1] * inv), M::pack(o[db][qb][2] * inv, o[db][qb][3] * inv)};
        }
        __builtin_amdgcn_wave_barrier();  // a wave's LDS operations keep their order
#pragma unroll
        for (int i = 0; i < C::RW * C::PC / 64; i++) {
            const int rl = (i * 64 + lane) / C::PC, c = lane % C::PC, r = row0 + rl;
            const u32x4 v = *reinterpret_cast<const u32x4*>(stg + rl * DH * 2 + (c ^ (rl & (C::PC - 1))) * 16);
            if (r >= p.rows) continue;
            const int t = r / p.G, h = hk * p.G + r % p.G;
            *reinterpret_cast<u32x4*>(static_cast<uint8_t*>(p.o) + ((long long)b * p.bso + (long long)t * p.ldo + (long long)h * DH + c * 8) * 2) = v;
        }
    } else {
        // the waves' results of the same 16 QB rows
        __syncthreads();
        float* ro = reinterpret_cast<float*>(xlds);
        float* rml = ro + C::NW * C::RW * DH;
#pragma unroll
        for (int qb = 0; qb < QB; qb++) {
#pragma unroll
            for (int db = 0; db < DH / 16; db++)
                *reinterpret_cast<floatx4*>(ro + (wv * C::RW + 16 * qb + c16) * DH + 16 * db + 4 * g) = o[db][qb];
            if (g == 0) {
                rml[(wv * C::RW + 16 * qb + c16) * 2] = m[qb];
                rml[(wv * C::RW + 16 * qb + c16) * 2 + 1] = l[qb][0];
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < C::RW * DH / 4; i += C::THREADS) {
            const int rl = i / (DH / 4), d = (i % (DH / 4)) * 4, r = row0 + rl;
            if (r >= p.rows) break;  // rows ascend with i
            float mm = -INFINITY, ll = 0.f;
#pragma unroll
            for (int w = 0; w < C::NW; w++) mm = fmaxf(mm, rml[(w * C::RW + rl) * 2]);
            const float me = mm == -INFINITY ? 0.f : mm;
            floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < C::NW; w++) {
                const float f = __builtin_amdgcn_exp2f(rml[(w * C::RW + rl) * 2] - me);
                ll += f * rml[(w * C::RW + rl) * 2 + 1];
                acc += f * *reinterpret_cast<const floatx4*>(ro + (w * C::RW + rl) * DH + d);
            }
            const float inv = ll > 0.f || ll != ll ? 1.f / ll : 0.f;
            store4(r, d, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
        }
    }
#endif
}

// The key ranges of a row joined, in the ranges' order: a workgroup per row. Its first threads hold the ranges' maxima and sums
// (at most 256), then DH / 4 threads a group take every 4 GR / DH th range.
template <class E, int DH>
__global__ __launch_bounds__(256) void k_cross_merge(const CrossParams p, int RT) {
    constexpr int GR = 256 / (DH / 4);
    __shared__ float fac[256], red[8];
    __shared__ floatx4 acc_s[GR][DH / 4];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const size_t rr = blockIdx.x, bh = rr / p.rows;
    const int r = (int)(rr - bh * p.rows), rt = r / RT, rl = r - rt * RT, hk = (int)(bh % p.Hkv), b = (int)(bh / p.Hkv);
    const int L = p.klen ? max(0, min(p.klen[b], p.Tk)) : p.Tk;
    const int n = ((L + XKT - 1) / XKT + p.ct - 1) / p.ct;  // the item's ranges
    const float* ml = p.part + (size_t)p.total * RT * DH;
    const size_t at0 = ((bh * p.ksplit) * p.rtiles + rt) * RT + rl, step = (size_t)p.rtiles * RT;
    const int gr = tid / (DH / 4), d = tid % (DH / 4);
    const float* src = p.part + at0 * DH + 4 * d;
    floatx4 ahead[4];  // a group's first ranges, under way while the factors are found
#pragma unroll
    for (int i = 0; i < 4; i++)
        ahead[i] = gr + i * GR < n ? *reinterpret_cast<const floatx4*>(src + (gr + i * GR) * step * DH) : floatx4{0.f, 0.f, 0.f, 0.f};
    float2 e = make_float2(-INFINITY, 0.f);
    if (tid < n) e = *reinterpret_cast<const float2*>(ml + (at0 + tid * step) * 2);
    float mm = e.x;
#pragma unroll
    for (int i = 32; i; i >>= 1) mm = fmaxf(mm, __shfl_xor(mm, i, 64));
    if (lane == 0) red[wv] = mm;
    __syncthreads();
    mm = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float f = __builtin_amdgcn_exp2f(e.x - (mm == -INFINITY ? 0.f : mm));
    fac[tid] = f;
    float ll = f * e.y;
#pragma unroll
    for (int i = 32; i; i >>= 1) ll += __shfl_xor(ll, i, 64);
    if (lane == 0) red[4 + wv] = ll;
    __syncthreads();
    ll = (red[4] + red[5]) + (red[6] + red[7]);
    floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (gr + i * GR < n) acc += fac[gr + i * GR] * ahead[i];
#pragma unroll 4
    for (int k = gr + 4 * GR; k < n; k += GR) acc += fac[k] * *reinterpret_cast<const floatx4*>(src + k * step * DH);
    acc_s[gr][d] = acc;
    __syncthreads();
    if (tid >= DH / 4) return;
#pragma unroll
    for (int i = 1; i < GR; i++) acc += acc_s[i][d];
    const float inv = ll > 0.f || ll != ll ? 1.f / ll : 0.f;
    const int t = r / p.G, h = hk * p.G + r % p.G;
    uint8_t* dst = static_cast<uint8_t*>(p.o) + ((long long)b * p.bso + (long long)t * p.ldo + (long long)h * DH + 4 * d) * 2;
    *reinterpret_cast<u32x2*>(dst) =
        u32x2{XMma<E>::pack(acc[0] * inv, acc[1] * inv), XMma<E>::pack(acc[2] * inv, acc[3] * inv)};
}

// The form of a call. ONE: a wave alone has 16 rows and a range of the keys; FOUR: four waves with the same 16 rows split the
// keys; S16, S32, S64: four waves of 16, 32 or 64 rows share the keys.
enum XKind { X_ONE, X_FOUR, X_S16, X_S32, X_S64 };
struct XForm {
    XKind kind;
    int rt, ksplit, ct;  // rows of a workgroup, key ranges, tiles of a range
};
static XForm cross_form(int B, int Tq, int Tk, int Hq, int Hkv, int Dh, bool split) {
    const long rows = (long)Tq * (Hq / Hkv), heads = (long)B * Hkv, cus = cu_count(), tiles = std::max(1, (Tk + XKT - 1) / XKT);
    const auto ranges = [&](XKind k, int rt, long ct) {
        ct = std::max(ct, (tiles + 255) / 256);  // the merge takes 256 ranges
        const long n = split ? (tiles + ct - 1) / ct : 1;
        return XForm{k, rt, (int)n, (int)(n == 1 ? tiles : ct)};
    };
    if (rows <= 16) {
        // One row block, bound by the keys' bytes: single waves of 32 KB of LDS and a mask's windows, four a CU, with ranges that fill
        // the chip three times over (a shorter item's ranges past its length end at once), at least 4 tiles each. Few keys in
        // four waves of one workgroup need no merge. In us, four waves / ranges: 1 x 3000, 20 heads of 128 24.8 / 11.6; 1 x 2048, 16 of 64
        // 10.4 / 10.3; 4 x 512, 16 of 128 8.4 / 10.6; 64 x 100, 16 of 128 (1024 heads) 21.5 / 11.5 in one range.
        if (heads >= 2 * cus) return {X_ONE, 16, 1, (int)tiles};
        if (!split || (tiles <= 32 && heads <= cus)) return {X_FOUR, 16, 1, (int)tiles};
        return ranges(X_ONE, 16, std::max<long>(4, (tiles * heads + 3 * cus - 1) / (3 * cus)));
    }
    // More rows per wave read LDS less often per product, but two workgroups per CU have to come of them. In us, 16 / 32 / 64 rows:
    // 2 x 4096 x 512, 10 heads of 64 26.7 / 23.1 / 27.7, 16 heads - / 32.1 / 29.9; 2 x 4096 x 77, 16 of 128 28.7 / 23.9;
    // 1 x 2048 x 2048, 16 of 128 (256 workgroups of 128 rows) 54.1 / 58.2; 2 x 1024 x 77, 20 of 64 8.4 / 10.2.
    const long u64 = (rows + 255) / 256 * heads, u32 = (rows + 127) / 128 * heads, u16 = (rows + 63) / 64 * heads;
    if (Dh == 64 && tiles >= 8 && u64 >= 2 * cus) return {X_S64, 256, 1, (int)tiles};
    if (u32 >= 2 * cus) return {X_S32, 128, 1, (int)tiles};
    if (u16 >= cus || tiles < 16) return {X_S16, 64, 1, (int)tiles};
    return ranges(X_S16, 64, std::max<long>(8, tiles * u16 / (2 * cus)));
}
size_t cross_attn_workspace(int B, int Tq, int Tk, int Hq, int Hkv, int Dh) {
    const XForm f = cross_form(B, Tq, Tk, Hq, Hkv, Dh, true);
    if (f.ksplit == 1) return 0;
    const size_t rtiles = ((size_t)Tq * (Hq / Hkv) + f.rt - 1) / f.rt;
    return (size_t)B * Hkv * f.ksplit * rtiles * f.rt * (Dh + 2) * sizeof(float);
}

int cross_attn_form(int B, int Tq, int Tk, int Hq, int Hkv, int Dh) {
    const XForm f = cross_form(B, Tq, Tk, Hq, Hkv, Dh, true);
    return f.rt << 16 | (f.kind == X_FOUR ? 4 : 1) << 8 | (f.ksplit > 1);
}

template <class E, class C>
static hipError_t cross_launch(CrossParams p, hipStream_t s) {
    p.rtiles = (p.rows + C::RT - 1) / C::RT;
    p.total = p.B * p.Hkv * p.ksplit * p.rtiles;
    p.per = (p.total + 7) / 8;
    if (hipError_t e = grid_check((size_t)p.per * 8, C::THREADS)) return e;
    auto kern = p.kmask ? k_cross_attn<E, C, true> : k_cross_attn<E, C, false>;
    hipLaunchKernelGGL(kern, dim3(p.per * 8), dim3(C::THREADS), C::LDS, s, p);
    if (hipError_t e = hipGetLastError()) return e;
    if (p.ksplit == 1) return hipSuccess;
    hipLaunchKernelGGL((k_cross_merge<E, C::DH>), dim3((unsigned)((size_t)p.B * p.Hkv * p.rows)), dim3(256), 0, s, p, C::RT);
    return hipGetLastError();
}
template <class E, int DH>
static hipError_t cross_of(const CrossParams& p, XKind k, hipStream_t s) {
    switch (k) {
        case X_ONE: return cross_launch<E, XCfg<DH, 1, 1, false, 2>>(p, s);
        case X_FOUR: return cross_launch<E, XCfg<DH, 1, 4, false, 2>>(p, s);
        case X_S16: return cross_launch<E, XCfg<DH, 1, 4, true, 4>>(p, s);
        case X_S32: return cross_launch<E, XCfg<DH, 2, 4, true, 4>>(p, s);
        default: return cross_launch<E, XCfg<64, 4, 4, true, 4>>(p, s);
    }
}

hipError_t launch_cross_attn(const CrossLaunch& c, hipStream_t s) {
    // sizes that need no workspace run the same form with one and without
    const size_t need = cross_attn_workspace(c.B, c.Tq, c.Tk, c.Hq, c.Hkv, c.Dh);
    const bool split = need == 0 || (c.ws && c.ws_bytes >= need);
    const XForm f = cross_form(c.B, c.Tq, c.Tk, c.Hq, c.Hkv, c.Dh, split);
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
    p.lift = XLIFT16;
    if (c.dt == DT::BF16) {
        p.lift = -1.f - XRESCALE;
        for (long n = 1; n < c.Tk; n *= 2) p.lift -= 1.f;
    }
    p.rows = c.Tq * p.G;
    p.ksplit = f.ksplit;
    p.ct = f.ct;
    p.part = static_cast<float*>(c.ws);
    if (c.dt == DT::F16) return c.Dh == 64 ? cross_of<_Float16, 64>(p, f.kind, s) : cross_of<_Float16, 128>(p, f.kind, s);
    return c.Dh == 64 ? cross_of<__bf16, 64>(p, f.kind, s) : cross_of<__bf16, 128>(p, f.kind, s);
}

}  // namespace kiln
