// Causal attention over packed sequences (kiln_prompt_attn): for each of B sequences O = softmax(s Q K^T) V per head, its nq queries
// being the last of its nk keys, so that query i sees the keys up to i + nk - nq; P prefix keys in front are seen by all. Hkv key
// heads each shared by G = Hq / Hkv query heads. fp16 or bf16 rows, read where they lie; lengths on the device.
//
// The G query heads of a key head and a sequence's tokens are the rows of one problem, r = t G + g. Products, the layout of tiles in
// LDS, the softmax in one pass with a maximum that moves in steps of 2^8, the weights' factor and scores far from zero: as in
// cross_attn.hip. A row tile's keys end with its last row's; tiles that not every row of a wave sees whole are masked by row.
//
// A hidden key's score is replaced, whatever it came to. Its weight 0 times an infinity or a NaN of V would still be a NaN in rows that
// must not see it: in tiles where that can be, a product of V with zeros finds them (8 matrix instructions), and they go to the rows
// that see them one by one (`keep_apart`), the others' operand holding zeros in their place.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "attn16.hpp"
#include "common.hpp"
#include "internal.hpp"

namespace kiln {

struct PromptParams {
    const void* q;
    const void* k;
    const void* v;
    const void* pk;
    const void* pv;
    void* o;
    size_t ldq, ldk, ldv, ldo, ldpk, ldpv;
    int B, Tq, Tk, P, Hkv, G;
    const int* q_start;  // [B + 1], or null: one sequence of all rows
    const int* k_start;  // [B], k_len [B], or null: the queries' own rows
    const int* k_len;
    float sc;            // scale log2(e)
    float lift;          // log2 of the weights' factor
    int nw;              // keys shared out: workgroups per key head
    size_t rows_part;    // .. partial results by row in front of those by workgroup
    float* part;         // .. partial results [.][DH], then [.](m, l)
    float* part_ml;
    uint32_t* cuts;      // .. of each row: its first workgroup, and << 16 their number; then the tiles of a workgroup's part
};

// How the keys go over the workgroups. WHOLE: a workgroup per key head and row tile. SPLIT: every key head's tiles of keys, row tile by row tile,
// are one line that its nw workgroups share out in equal parts; a row tile that is cut leaves partial results, joined by k_prompt_merge.
// PACK: as SPLIT, but the prefix's keys come first and once for all sequences' rows, whose own keys follow without it.
enum PromptMode { PM_WHOLE, PM_SPLIT, PM_PACK };
constexpr int PROMPT_LEAST = 4;  // tiles of a workgroup's part

// A sequence's rows: queries q0 .. q0 + nq - 1, keys k0 .. k0 + nk - 1, inside the tensors whatever the lengths on the device say
struct PromptSeq {
    int q0, nq, k0, nk;
};
__device__ __forceinline__ PromptSeq prompt_seq(const PromptParams& p, int s) {
    PromptSeq r{0, p.Tq, 0, p.Tq};
    if (p.q_start) {
        r.q0 = max(0, min(p.q_start[s], p.Tq));
        r.nq = max(0, min(p.q_start[s + 1], p.Tq) - r.q0);
    }
    r.k0 = r.q0;
    r.nk = r.nq;
    if (p.k_start) {
        r.k0 = max(0, min(p.k_start[s], p.Tk));
        r.nk = max(0, min(p.k_len[s], p.Tk - r.k0));
    }
    return r;
}

// Keys that the last row of a sequence's row tile `place` sees, and its tiles (one at least: a row without keys is zeros) behind np of the prefix
template <int RT>
__device__ __forceinline__ int prompt_keys(const PromptParams& p, const PromptSeq& q, int place) {
    const int rows = q.nq * p.G;
    return max(0, min(q.nk, (min(rows, (place + 1) * RT) - 1) / p.G + q.nk - q.nq + 1));
}
template <int RT>
__device__ __forceinline__ int prompt_tiles(const PromptParams& p, const PromptSeq& q, int place, int np) {
    return max(1, np + (prompt_keys<RT>(p, q, place) + XKT - 1) / XKT);
}
// the sum over a wave's lanes, in all of them
__device__ __forceinline__ int wave_sum(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x121, 0xF, 0xF, false);  // row_ror 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x122, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x124, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x128, 0xF, 0xF, false);
    auto r = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
    v = (int)(r[0] + r[1]);
    r = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
    return __builtin_amdgcn_readfirstlane((int)(r[0] + r[1]));
}

// the sum over the lanes up to a lane's own
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast 15 to rows 1 and 3, 31 to rows 2 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}

// A key head's line of tiles: `ahead` of the prefix over all rows (PACK), then each sequence's; `each` tiles to a workgroup
template <int RT, PromptMode MODE>
struct PromptLine {
    int lane, np, ahead, total, each, first;  // first: the tiles of sequence `lane`
    __device__ __forceinline__ int of(const PromptParams& p, int s) const {
        if (s >= p.B) return 0;
        const PromptSeq q = prompt_seq(p, s);
        int n = 0;
        for (int i = 0; i * RT < q.nq * p.G; i++) n += prompt_tiles<RT>(p, q, i, MODE == PM_PACK ? 0 : np);
        return n;
    }
    __device__ __forceinline__ explicit PromptLine(const PromptParams& p) {
        lane = threadIdx.x & 63;
        np = (p.P + XKT - 1) / XKT;
        ahead = MODE == PM_PACK ? (p.Tq * p.G + RT - 1) / RT * np : 0;
        first = of(p, lane);
        int n = first;
        for (int s = 64; s < p.B; s += 64) n += of(p, s + lane);
        total = ahead + wave_sum(n);
        each = max(PROMPT_LEAST, (total + p.nw - 1) / p.nw);
    }
    // the sequence that holds place `at` of the line (>= ahead), or -1; at: counted from the sequence's first tile
    __device__ __forceinline__ int find(const PromptParams& p, int& at) const {
        at -= ahead;
        for (int s0 = 0; s0 < p.B; s0 += 64) {
            const int n = s0 ? of(p, s0 + lane) : first, up = wave_scan(n);
            const unsigned long long past = __ballot(up > at);
            if (past) {
                const int i = __ffsll(past) - 1;
                at -= __builtin_amdgcn_readlane(up - n, i);
                return s0 + i;
            }
            at -= __builtin_amdgcn_readlane(up, 63);
        }
        return -1;
    }
};

// Row tile number `rank` of all sequences' tiles of RT rows, in the order of falling place in their sequence (the longest ranges of keys
// first): its sequence and place, or -1 past the last. With F(n) the number of tiles at place n or later, F(n + 1) <= rank < F(n).
template <int RT>
__device__ __forceinline__ int prompt_find(const PromptParams& p, int rank, int& place) {
    const int lane = threadIdx.x & 63;
    auto tiles = [&](int s) {
        if (s >= p.B) return 0;
        const PromptSeq q = prompt_seq(p, s);
        return (q.nq * p.G + RT - 1) / RT;
    };
    if (p.B == 1) {
        place = __builtin_amdgcn_readfirstlane(tiles(0)) - 1 - rank;
        return place >= 0 ? 0 : -1;
    }
    int own[4], most = 0;  // of the first 256 sequences; more are read again
#pragma unroll
    for (int c = 0; c < 4; c++) {
        own[c] = c * 64 < p.B ? tiles(c * 64 + lane) : 0;
        most = max(most, own[c]);
    }
    for (int s = 256; s < p.B; s += 64) most = max(most, tiles(s + lane));
    auto from = [&](int n) {  // F(n)
        int sum = 0;
#pragma unroll
        for (int c = 0; c < 4; c++) sum += max(0, own[c] - n);
        for (int s = 256; s < p.B; s += 64) sum += max(0, tiles(s + lane) - n);
        return wave_sum(sum);
    };
    if (rank >= from(0)) return -1;
#pragma unroll
    for (int i = 32; i; i >>= 1) most = max(most, __shfl_xor(most, i, 64));
    int lo = 0, hi = __builtin_amdgcn_readfirstlane(most), fhi = 0;  // F(lo) > rank >= F(hi) = fhi
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2, f = from(mid);
        if (f > rank) lo = mid;
        else hi = mid, fhi = f;
    }
    place = lo;
    // the sequences with a tile at this place, in their order
    int want = rank - fhi;
    for (int s0 = 0; s0 < p.B; s0 += 64) {
        const unsigned long long has = __ballot(tiles(s0 + lane) > lo);
        const int n = __popcll(has);
        if (want < n) {
            // lane i counts the set bits below it
            const int below = __popcll(has & ((1ull << lane) - 1));
            return s0 + __ffsll((unsigned long long)__ballot((has >> lane & 1) && below == want)) - 1;
        }
        want -= n;
    }
    return -1;
}

template <class E, class C, PromptMode MODE>
__global__ __launch_bounds__(C::THREADS, C::WAVES) void k_prompt_attn(const PromptParams p) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass drops a kernel template whose target builtins it cannot check
    using M = XMma<E>;
    constexpr int DH = C::DH, QB = C::QB;
    static_assert(C::SHARED || C::NW == 1, "waves share the keys, or one has them to itself");
    extern __shared__ __attribute__((aligned(16))) uint8_t xlds[];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, c16 = lane & 15;
    // key heads side by side: blocks go round the 8 XCDs, so that a head's row tiles share the L2s of few, and every XCD has long and
    // short ones
    const int hk = (int)(blockIdx.x % p.Hkv), bx = (int)(blockIdx.x / p.Hkv);
    // a row tile: sequence (-1: the prefix's pass over all rows), place in it, its tiles t0 .. t1 - 1 of kt
    int s = 0, jt = 0, t0 = 0, t1, kt, left_u = 0, each = 0;
    PromptSeq sq;
    if constexpr (MODE == PM_WHOLE) {
        s = prompt_find<C::RT>(p, bx, jt);
        if (s < 0) return;
        sq = prompt_seq(p, s);
    } else {
        const PromptLine<C::RT, MODE> line(p);
        each = line.each;
        if (bx == 0 && hk == 0 && threadIdx.x == 0) p.cuts[(size_t)p.Tq * p.G] = each;
        int u = bx * each;
        left_u = min(line.total - u, each);
        if (left_u <= 0) return;
        if (u < line.ahead) {
            s = -1;
            jt = u / line.np;
            t0 = u % line.np;
        } else {
            s = line.find(p, u);
            sq = prompt_seq(p, s);
            for (int n; u >= (n = prompt_tiles<C::RT>(p, sq, jt, MODE == PM_PACK ? 0 : line.np)); jt++) u -= n;
            t0 = u;
        }
    }
    for (;;) {
    const bool ahead = MODE == PM_PACK && s < 0;
    if (ahead) sq = PromptSeq{0, p.Tq, 0, 0};
    const int rows = sq.nq * p.G, diff = sq.nk - sq.nq;
    const int np = MODE == PM_PACK && !ahead ? 0 : (p.P + XKT - 1) / XKT;
    const int row0 = jt * C::RT + (C::SHARED ? wv * C::RW : 0);
    // the row tile's own keys
    const int L = ahead ? 0 : prompt_keys<C::RT>(p, sq, jt);
    kt = max(1, np + (L + XKT - 1) / XKT);
    t1 = MODE == PM_WHOLE ? kt : min(kt, t0 + left_u);

    uint8_t* ring = xlds;
    const uint32_t lds_base = (uint32_t)(size_t)(__attribute__((address_space(3))) uint8_t*)ring;

    // DMA of the tiles' K and V in turn: a thread's pieces are chunks of fixed rows of a tile; the descriptor's range ends with
    // the last row (empty past the last tile)
    struct Stream {
        const uint8_t* src;     // the next tile to copy
        uint32_t ld2;           // bytes from row to row
        int j;                  // its index
        uint32_t off[C::DMA];
    } kst, vst;
    const uint8_t* own_k = static_cast<const uint8_t*>(p.k) + ((long long)sq.k0 * p.ldk + (long long)hk * DH) * 2;
    const uint8_t* own_v = static_cast<const uint8_t*>(p.v) + ((long long)sq.k0 * p.ldv + (long long)hk * DH) * 2;
    auto place_k = [&](uint32_t ld2) {
        kst.ld2 = ld2;
#pragma unroll
        for (int i = 0; i < C::DMA; i++) {
            const int pc = i * C::RTHREADS + (C::SHARED ? (int)threadIdx.x : lane), r = pc / C::PC, c = pc % C::PC;
            kst.off[i] = r * ld2 + k_swz<DH>(c, r) * 16;
        }
    };
    auto place_v = [&](uint32_t ld2) {
        vst.ld2 = ld2;
#pragma unroll
        for (int i = 0; i < C::DMA; i++) {
            const int pc = i * C::RTHREADS + (C::SHARED ? (int)threadIdx.x : lane), r = pc / C::PC, c = pc % C::PC;
            vst.off[i] = r * ld2 + v_swz<DH>(c, r) * 16;
        }
    };
    kst.j = vst.j = t0;
    if (t0 < np) {
        place_k((uint32_t)p.ldpk * 2);
        place_v((uint32_t)p.ldpv * 2);
        kst.src = static_cast<const uint8_t*>(p.pk) + (long long)hk * DH * 2 + (long long)t0 * XKT * kst.ld2;
        vst.src = static_cast<const uint8_t*>(p.pv) + (long long)hk * DH * 2 + (long long)t0 * XKT * vst.ld2;
    } else {
        place_k((uint32_t)p.ldk * 2);
        place_v((uint32_t)p.ldv * 2);
        kst.src = own_k + (long long)(t0 - np) * XKT * kst.ld2;
        vst.src = own_v + (long long)(t0 - np) * XKT * vst.ld2;
    }
    auto left_of = [&](int j) { return j < np ? p.P - j * XKT : L - (j - np) * XKT; };  // keys from tile j's first on
    auto copy = [&](Stream& t, uint32_t at) {
        const int left = t.j < t1 ? min(XKT, left_of(t.j)) : 0;
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(t.src), (short)0, left > 0 ? (int)((left - 1) * t.ld2 + DH * 2) : 0, 0x00020000 /* raw */);
        uint8_t* dst = ring + at + (C::SHARED ? wv * 1024 : 0);
#pragma unroll
        for (int i = 0; i < C::DMA; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(dst + i * C::RTHREADS * 16), 16, t.off[i], 0, 0, 0);
        if (t.j + 1 < t1) t.src += (size_t)XKT * t.ld2;
        t.j++;
    };
    auto copy_k = [&](int stage) {
        copy(kst, stage * C::STAGE);
        if (kst.j == np && np < t1) {  // from the prefix to the sequence's own keys
            place_k((uint32_t)p.ldk * 2);
            kst.src = own_k;
        }
    };
    auto copy_v = [&](int stage) {
        copy(vst, stage * C::STAGE + C::TILE);
        if (vst.j == np && np < t1) {
            place_v((uint32_t)p.ldv * 2);
            vst.src = own_v;
        }
    };

    // Q: the B operands of S^T, lane (row c16, chunk 4 cc + g); rows past the last read the last and are not stored. lim: the own keys
    // that a row sees
    u32x4 qf[QB][DH / 32];
    int lim[QB];
#pragma unroll
    for (int qb = 0; qb < QB; qb++) {
        const int r = min(row0 + 16 * qb + c16, rows - 1), t = r / p.G, h = hk * p.G + r % p.G;
        const uint8_t* src = static_cast<const uint8_t*>(p.q) + ((long long)(sq.q0 + t) * p.ldq + (long long)h * DH + 8 * g) * 2;
#pragma unroll
        for (int cc = 0; cc < DH / 32; cc++) qf[qb][cc] = *reinterpret_cast<const u32x4*>(src + 64 * cc);
        lim[qb] = t + diff + 1;
    }
    // of the wave's first and last row
    const int lim0 = min(row0, rows - 1) / p.G + diff + 1, lim1 = min(row0 + C::RW - 1, rows - 1) / p.G + diff + 1;

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
    // tile j's keys that a row sees: the first lim - (its first own key), or all up to the prefix's end
    auto hide = [&](int j, floatx4 (&s)[2][QB]) {
        const bool pre = j < np;
        const int key0 = (j - np) * XKT;
        if ((pre ? p.P - j * XKT : lim0 - key0) >= XKT) return;
#pragma unroll
        for (int qb = 0; qb < QB; qb++) {
            const int seen = (pre ? p.P - j * XKT : lim[qb] - key0) - 4 * g;
#pragma unroll
            for (int kk = 0; kk < 2; kk++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (16 * kk + i >= seen) s[kk][qb][i] = -INFINITY;
        }
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
    // Tile j, that rows of this wave see different parts of: infinities and NaNs of V leave the operands; the rows that see them take
    // their products here. V's rows are read from the stage itself, four dimensions of a key a lane, as the accumulators lie.
    auto keep_apart = [&](int j, uint32_t st, u32x4 (&vf)[DH / 16], const u32x4 (&pf)[QB]) __attribute__((always_inline)) {
        floatx4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int db = 0; db < DH / 16; db++) z = M::mul(vf[db], u32x4{0, 0, 0, 0}, z);
        const float zs = (z[0] + z[1]) + (z[2] + z[3]);
        if (!__any(zs != 0.f)) return;  // 0, or NaN
        constexpr uint32_t EXP = std::is_same<E, _Float16>::value ? 0x7c00u : 0x7f80u;
#pragma unroll
        for (int db = 0; db < DH / 16; db++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint32_t w = vf[db][i];
                if ((w & EXP) == EXP) w &= 0xffff0000u;
                if ((w >> 16 & EXP) == EXP) w &= 0xffffu;
                vf[db][i] = w;
            }
#pragma clang loop unroll(disable)
        for (int at = 0; at < XKT * DH / 16; at++) {
            const int key = at / (DH / 16), db = at % (DH / 16);
            const u32x2 v4 = *reinterpret_cast<const __attribute__((address_space(3))) u32x2*>(
                (size_t)(lds_base + st + C::TILE + key * DH * 2 + v_swz<DH>(2 * db + (g >> 1), key) * 16 + (g & 1) * 8));
            bool odd[4];
#pragma unroll
            for (int i = 0; i < 4; i++) odd[i] = (v4[i / 2] >> (16 * (i & 1)) & EXP) == EXP;
            if (!__any(odd[0] | odd[1] | odd[2] | odd[3])) continue;
            // the weights of this key: element 4 (key / 16) + key % 4 of the lanes of group key / 4 % 4
            const int w = 2 * (key >> 4) + (key >> 1 & 1);
#pragma unroll
            for (int qb = 0; qb < QB; qb++) {
                const uint32_t word = w == 0 ? pf[qb][0] : w == 1 ? pf[qb][1] : w == 2 ? pf[qb][2] : pf[qb][3];
                const uint16_t pb = (uint16_t)(__shfl(word, 16 * (key >> 2 & 3) + c16, 64) >> (16 * (key & 1)));
                const float pw = (float)__builtin_bit_cast(E, pb);
                const bool sees = (j - np) * XKT + key < lim[qb];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint16_t vb = (uint16_t)(v4[i / 2] >> (16 * (i & 1)));
                    const float x = odd[i] && sees ? pw * (float)__builtin_bit_cast(E, vb) : 0.f;
#pragma unroll
                    for (int d = 0; d < DH / 16; d++)
                        if (d == db) o[d][qb][i] += x;
                }
            }
        }
    };

    auto apart = [&](int j) { return j >= np && lim0 < lim1 && lim0 - (j - np) * XKT < XKT; };
    if constexpr (C::SHARED) {
        // A step computes the scores of tile j + 1 ahead of the weights and products of tile j. K of tile j + 1 and V of tile j landed (past
        // the last tile the copies go on with empty ranges, which keeps the count); every wave is done with K of tile j and V of tile
        // j - 1, whose places take K of tile j + NS and V of tile j + NS - 1.
        constexpr int NS = C::NS;
        static_assert(NS % 2 == 0, "the scores' two sets go with the stages");
        floatx4 sc[2][2][QB];
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
        read_k(0, kf);
        scores(kf, sc[0]);
        hide(t0, sc[0]);
        largest(sc[0], top);
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
            rescale(top, sc[cur]);
            __builtin_amdgcn_sched_barrier(0);
            weights(sc[cur], pf);
            scores(kf, sc[cur ^ 1]);
            __builtin_amdgcn_sched_barrier(0);
            if (apart(j)) keep_apart(j, st * C::STAGE, vf, pf);
            if (j + 1 < t1) hide(j + 1, sc[cur ^ 1]);
#pragma unroll
            for (int qb = 0; qb < QB; qb++) l[qb] = M::mul(ones, pf[qb], l[qb]);
#pragma unroll
            for (int db = 0; db < DH / 16; db++)
#pragma unroll
                for (int qb = 0; qb < QB; qb++) o[db][qb] = M::mul(vf[db], pf[qb], o[db][qb]);
            largest(sc[cur ^ 1], top);
        };
        using P0 = std::integral_constant<int, 0>;
        using P1 = std::integral_constant<int, 1>;
        if constexpr (QB == 1) {
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
            floatx4 sc[2][QB];
            float top[QB];
            u32x4 kf[2][DH / 32], vf[DH / 16], pf[QB];
            read_k(st, kf);
            scores(kf, sc);
            hide(j, sc);
            largest(sc, top);
            rescale(top, sc);
            weights(sc, pf);
#pragma unroll
            for (int db = 0; db < DH / 16; db++) vf[db] = read_v(st, db);
            if (apart(j)) keep_apart(j, st, vf, pf);
#pragma unroll
            for (int qb = 0; qb < QB; qb++) l[qb] = M::mul(ones, pf[qb], l[qb]);
#pragma unroll
            for (int db = 0; db < DH / 16; db++)
#pragma unroll
                for (int qb = 0; qb < QB; qb++) o[db][qb] = M::mul(vf[db], pf[qb], o[db][qb]);
            stage = stage == C::NS - 1 ? 0 : stage + 1;
        }
    }
    x_wait_vmcnt<0>();  // no copy into LDS outlives its ring

    const bool whole = MODE == PM_WHOLE || (t0 == 0 && t1 == kt);
    if (MODE != PM_WHOLE && hk == 0 && !ahead && t0 == 0) {  // where the merge finds these rows' parts (the same for every key head)
        const uint32_t n = kt <= left_u ? 1 : 1 + (kt - left_u + each - 1) / each;
        for (int i = threadIdx.x; i < C::RT && jt * C::RT + i < rows; i += C::THREADS) p.cuts[(size_t)sq.q0 * p.G + jt * C::RT + i] = (uint32_t)bx | n << 16;
    }
    if (MODE != PM_WHOLE && (MODE == PM_PACK || !whole)) {
        // partial results: of a whole row tile by row (PACK), else by workgroup: one that begins before it, one that ends behind it
        size_t base = p.rows_part + (((size_t)hk * p.nw + bx) * 2 + (t0 > 0 ? 0 : 1)) * C::RT + (C::SHARED ? wv * C::RW : 0);
        if (MODE == PM_PACK && whole) base = ((size_t)(ahead ? p.Hkv : 0) + hk) * p.Tq * p.G + (size_t)sq.q0 * p.G + row0;
#pragma unroll
        for (int qb = 0; qb < QB; qb++) {
            if (row0 + 16 * qb + c16 >= rows) continue;
            const size_t at = base + 16 * qb + c16;
#pragma unroll
            for (int db = 0; db < DH / 16; db++) *reinterpret_cast<floatx4*>(p.part + at * DH + 16 * db + 4 * g) = o[db][qb];
            if (g == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m[qb], l[qb][0]);
        }
        if constexpr (C::SHARED) __builtin_amdgcn_s_barrier();  // every wave is done with the ring
    } else {
    // rows leave through LDS, whole and 16 bytes a lane; a row's chunks lie permuted by its number
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
        if (r >= rows) continue;
        const int t = r / p.G, h = hk * p.G + r % p.G;
        *reinterpret_cast<u32x4*>(static_cast<uint8_t*>(p.o) + ((long long)(sq.q0 + t) * p.ldo + (long long)h * DH + c * 8) * 2) = v;
    }
    if (MODE != PM_WHOLE && C::SHARED) {
        __builtin_amdgcn_s_waitcnt(0xC07F);
        __builtin_amdgcn_s_barrier();  // every wave's rows are out of LDS
    }
    }
    if constexpr (MODE == PM_WHOLE) return;
    // the next row tile of the line
    left_u -= t1 - t0;
    if (left_u <= 0) return;
    __builtin_amdgcn_s_waitcnt(0xC07F);
    __builtin_amdgcn_sched_barrier(0);
    t0 = 0;
    if (++jt * C::RT >= rows) {
        jt = 0;
        do {
            if (++s >= p.B) return;
            sq = prompt_seq(p, s);
        } while (sq.nq == 0);
    }
    }
#endif
}

// The partial results of a row joined, in the line's order: a wave per row
template <class E, int DH, int RT, PromptMode MODE>
__global__ __launch_bounds__(256) void k_prompt_merge(const PromptParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int lane = threadIdx.x & 63, hk = (int)(blockIdx.x % p.Hkv);
    const long long R = (long long)(blockIdx.x / p.Hkv) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (R >= (long long)p.Tq * p.G) return;
    const int t = (int)(R / p.G);
    // the row's sequence: the last that claims it
    int s = -1;
    for (int s0 = 0; s0 < p.B; s0 += 64) {
        bool in = false;
        if (s0 + lane < p.B) {
            const PromptSeq q = prompt_seq(p, s0 + lane);
            in = t >= q.q0 && t - q.q0 < q.nq;
        }
        const unsigned long long has = __ballot(in);
        if (has) s = s0 + 63 - __clzll(has);
    }
    if (s < 0) return;
    const uint32_t cut = p.cuts[R];
    const int r = (int)(R - (long long)prompt_seq(p, s).q0 * p.G), w = cut & 0xffff, n = cut >> 16;
    if (MODE == PM_SPLIT && n == 1) return;  // written by its workgroup
    int w2 = 0, n2 = 0;
    if (MODE == PM_PACK) {
        const int np = (p.P + XKT - 1) / XKT, each = (int)p.cuts[(size_t)p.Tq * p.G], at = (int)(R / RT) * np;
        w2 = at / each;
        n2 = (at + np - 1) / each - w2 + 1;
    }
    const size_t all = (size_t)p.Tq * p.G;
    auto index = [&](int i) -> size_t {  // of the row's partial result i
        const bool own = MODE == PM_SPLIT || i < n;
        const int k = own ? i : i - n;
        if ((own ? n : n2) == 1) return ((size_t)(own ? 0 : p.Hkv) + hk) * all + R;
        return p.rows_part + (((size_t)hk * p.nw + (own ? w : w2) + k) * 2 + (k == 0 ? 1 : 0)) * RT + (own ? r % RT : (int)(R % RT));
    };
    const int parts = n + n2;
    float mm = -INFINITY;
    for (int i = lane; i < parts; i += 64) mm = fmaxf(mm, p.part_ml[index(i) * 2]);
#pragma unroll
    for (int i = 32; i; i >>= 1) mm = fmaxf(mm, __shfl_xor(mm, i, 64));
    const float me = mm == -INFINITY ? 0.f : mm;
    constexpr int PER = DH / 64;
    typedef float vec __attribute__((ext_vector_type(PER)));
    vec acc = 0.f;
    float ll = 0.f;
    for (int i0 = 0; i0 < parts; i0 += 64) {
        float f = 0.f;
        if (i0 + lane < parts) {
            const float2 e = *reinterpret_cast<const float2*>(p.part_ml + index(i0 + lane) * 2);
            f = __builtin_amdgcn_exp2f(e.x - me);
            ll += f * e.y;
        }
        const int end = min(64, parts - i0);
        for (int i = 0; i < end; i += 4) {  // four in flight; past the last the factor is 0
            vec v[4];
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = *reinterpret_cast<const vec*>(p.part + index(i0 + min(i + k, end - 1)) * DH + PER * lane);
#pragma unroll
            for (int k = 0; k < 4; k++) acc += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), i + k)) * v[k];
        }
    }
#pragma unroll
    for (int i = 32; i; i >>= 1) ll += __shfl_xor(ll, i, 64);
    const float inv = ll > 0.f || ll != ll ? 1.f / ll : 0.f;
    uint8_t* dst = static_cast<uint8_t*>(p.o) + ((long long)t * p.ldo + (long long)(hk * p.G + (int)(R % p.G)) * DH + PER * lane) * 2;
    if constexpr (PER == 2) *reinterpret_cast<uint32_t*>(dst) = XMma<E>::pack(acc[0] * inv, acc[1] * inv);
    else *reinterpret_cast<uint16_t*>(dst) = __builtin_bit_cast(uint16_t, (E)(acc[0] * inv));
#endif
}

// The form of a call. Rows, keys and work are guesses from the tensors' sizes: lengths are on the device.
struct PromptForm {
    PromptMode mode;
    bool one;   // single waves of 16 rows (else four that share the keys)
    int rt;     // rows of a workgroup
    int nw;     // keys shared out: workgroups per key head
};
static PromptForm prompt_form(int B, int Tq, int Tk, int P, int Hq, int Hkv, int Dh, bool split) {
    const long G = Hq / Hkv, cus = cu_count(), rows = std::max<long>(1, (long)Tq * G / B), keys = Tk / B + P;
    const long tiles = std::max<long>(B, (long)Tq * G / 64) * Hkv;
    // the line's places are counted in 32 bits, whatever the lengths
    const bool fits = ((long)Tq * G / 16 + B) * ((Tk + (long)P) / XKT + 2) < 1 << 29;
    if (!split || !fits || keys <= 16 * XKT || (rows > 16 && tiles >= 2 * cus)) {
        const long tiles128 = std::max<long>(B, (long)Tq * G / 128) * Hkv;
        return {PM_WHOLE, false, tiles128 >= 2 * cus ? 128 : 64, 0};
    }
    const bool pack = P >= 2 * XKT && B > 1 && rows <= 32;
    const long slots = rows <= 16 ? 4 * cus : 2 * cus;
    const int rt = rows <= 16 ? 16 : pack || rows < 128 ? 64 : 128;
    return {pack ? PM_PACK : PM_SPLIT, rows <= 16, rt, (int)std::min<long>(0xffff, std::max<long>(1, slots / Hkv))};
}
static size_t prompt_rows_part(const PromptForm& f, int Tq, int Hq) { return f.mode == PM_PACK ? (size_t)2 * Tq * Hq : 0; }
static size_t prompt_parts(const PromptForm& f, int Tq, int Hq, int Hkv) {
    return f.mode == PM_WHOLE ? 0 : prompt_rows_part(f, Tq, Hq) + (size_t)Hkv * f.nw * 2 * f.rt;
}
size_t prompt_attn_workspace(int B, int Tq, int Tk, int P, int Hq, int Hkv, int Dh) {
    const size_t parts = prompt_parts(prompt_form(B, Tq, Tk, P, Hq, Hkv, Dh, true), Tq, Hq, Hkv);
    return parts ? parts * (Dh + 2) * sizeof(float) + ((size_t)Tq * (Hq / Hkv) + 1) * sizeof(uint32_t) : 0;
}

template <class E, class C>
static hipError_t prompt_whole(const PromptParams& p, hipStream_t s) {
    // every sequence rounds its rows up to whole tiles
    const size_t tiles = ((size_t)p.Tq * p.G) / C::RT + p.B;
    if (hipError_t e = grid_check(tiles * p.Hkv, C::THREADS)) return e;
    hipLaunchKernelGGL((k_prompt_attn<E, C, PM_WHOLE>), dim3((unsigned)(tiles * p.Hkv)), dim3(C::THREADS), C::LDS, s, p);
    return hipGetLastError();
}
template <class E, class C, PromptMode MODE>
static hipError_t prompt_split(const PromptParams& p, hipStream_t s) {
    const size_t merges = ((size_t)p.Tq * p.G + 3) / 4 * p.Hkv;
    if (hipError_t e = grid_check(merges, 256)) return e;
    hipLaunchKernelGGL((k_prompt_attn<E, C, MODE>), dim3(p.nw * p.Hkv), dim3(C::THREADS), C::LDS, s, p);
    if (hipError_t e = hipGetLastError()) return e;
    hipLaunchKernelGGL((k_prompt_merge<E, C::DH, C::RT, MODE>), dim3((unsigned)merges), dim3(256), 0, s, p);
    return hipGetLastError();
}
template <class E, int DH>
static hipError_t prompt_of(const PromptParams& p, const PromptForm& f, hipStream_t s) {
    if (f.mode == PM_WHOLE) return f.rt == 128 ? prompt_whole<E, XCfg<DH, 2, 4, true, 4>>(p, s) : prompt_whole<E, XCfg<DH, 1, 4, true, 4>>(p, s);
    if (f.mode == PM_SPLIT)
        return f.one         ? prompt_split<E, XCfg<DH, 1, 1, false, 2>, PM_SPLIT>(p, s)
               : f.rt == 128 ? prompt_split<E, XCfg<DH, 2, 4, true, 4>, PM_SPLIT>(p, s)
                             : prompt_split<E, XCfg<DH, 1, 4, true, 4>, PM_SPLIT>(p, s);
    return f.one ? prompt_split<E, XCfg<DH, 1, 1, false, 2>, PM_PACK>(p, s) : prompt_split<E, XCfg<DH, 1, 4, true, 4>, PM_PACK>(p, s);
}

hipError_t launch_prompt_attn(const PromptLaunch& c, hipStream_t s) {
    PromptParams p{};
    p.q = c.q;
    p.k = c.k;
    p.v = c.v;
    p.pk = c.pk;
    p.pv = c.pv;
    p.o = c.out;
    p.ldq = c.ldq;
    p.ldk = c.ldk;
    p.ldv = c.ldv;
    p.ldo = c.ldo;
    p.ldpk = c.ldpk;
    p.ldpv = c.ldpv;
    p.B = c.B;
    p.Tq = c.Tq;
    p.Tk = c.Tk;
    p.P = c.P;
    p.Hkv = c.Hkv;
    p.G = c.Hq / c.Hkv;
    p.q_start = c.q_start;
    p.k_start = c.k_start;
    p.k_len = c.k_len;
    p.sc = c.scale * LOG2E;
    p.lift = -1.f - XRESCALE;  // bf16: the weights of all keys sum to less than 1
    for (long n = 1; n < (long)c.Tk + c.P; n *= 2) p.lift -= 1.f;
    // sizes that need no workspace run the same form with one and without
    const size_t need = prompt_attn_workspace(c.B, c.Tq, c.Tk, c.P, c.Hq, c.Hkv, c.Dh);
    const PromptForm f = prompt_form(c.B, c.Tq, c.Tk, c.P, c.Hq, c.Hkv, c.Dh, need == 0 || (c.ws && c.ws_bytes >= need));
    p.nw = f.nw;
    p.rows_part = prompt_rows_part(f, c.Tq, c.Hq);
    p.part = static_cast<float*>(c.ws);
    const size_t parts = prompt_parts(f, c.Tq, c.Hq, c.Hkv);
    p.part_ml = p.part + parts * c.Dh;
    p.cuts = reinterpret_cast<uint32_t*>(p.part_ml + parts * 2);
    if (c.dt == DT::F16) return c.Dh == 64 ? prompt_of<_Float16, 64>(p, f, s) : prompt_of<_Float16, 128>(p, f, s);
    return c.Dh == 64 ? prompt_of<__bf16, 64>(p, f, s) : prompt_of<__bf16, 128>(p, f, s);
}

}  // namespace kiln
