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
//
// What bounds it (16 heads on 8 of 128 where nothing else is said, two workgroups or four single waves a CU; a single wave's
// ring is 32 KB of LDS, of which five would fit, and half of that for heads of 64). Whole prompts: the matrix cores and
// the vector work of the softmax, which in one wave follow each other and beside another wave's overlap: 8192 tokens 241 to 260 us, 1.06 to 1.14
// PFLOP/s. 24 prompts of 2048 446, 0.92 PFLOP/s: of a workgroup's 37 us some 8 are its start and end, of which another workgroup of the CU
// hides a part: finding its tile 1.0, the first keys' and Q's way 2.4, the first scores 0.7, the tiles one by one (12% slower than two or four in
// a row), the rows' way out 1.2. 4 x 120 tokens 8.3, one such chain. Single tokens after 16 x 8191 keys: memory, 408 MB in 76 us, 5.4 TB/s, then the merge
// (4.6). 3 x 100 rows after 4000 keys (32 heads on 4 of 64): 20.6, of it one round of 256 workgroups with 16 tiles at least (16.8 in a trace) and the
// merge (5.0). A prefix of 4096 keys before 32 single tokens with 300 of their own: 17.1 (12.0 and 4.4); without sharing 570 MB would be read, with it
// 41. Every workgroup looks through all sequences for its place: 512 single tokens after 50 keys 80 us, 1024 208, 4096 2137.
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
    uint32_t g_mul;      // r / G = r g_mul >> g_shift, exactly for r < 2^31
    int g_shift;
    const int* q_start;  // [B + 1], or null: one sequence of all rows
    const int* k_start;  // [B], k_len [B], or null: the queries' own rows
    const int* k_len;
    float sc;            // scale log2(e)
    float lift;          // log2 of the weights' factor
    int nw;              // keys shared out: parts per key head that are aimed at
    int items;           // .. the most that can come of it
    float* part;         // .. partial results [key head][item][row of the tile][DH], then [.](m, l)
    float* part_ml;
    uint32_t* cuts;      // .. of each row: its first item, their number; then the tiles of an item
};

// How the keys go over the workgroups. WHOLE: a workgroup per key head and row tile. SPLIT: row tiles are cut into items of about equal numbers
// of key tiles, as many over all sequences as fill the chip, a workgroup each; the partial results of a row are joined by
// k_prompt_merge. PACK: as SPLIT, but the prefix's keys are taken once for all sequences' rows, whose own keys follow without it.
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

__device__ __forceinline__ int prompt_token(const PromptParams& p, int r) { return (int)((uint64_t)(uint32_t)r * p.g_mul >> p.g_shift); }  // r / G
// the sequences, the first 64 of them a lane each
struct PromptSeqs {
    PromptSeq mine;  // of sequence `lane` (none: no rows)
    __device__ __forceinline__ explicit PromptSeqs(const PromptParams& p) : mine{0, 0, 0, 0} {
        const int lane = threadIdx.x & 63;
        if (lane < p.B) mine = prompt_seq(p, lane);
    }
    __device__ __forceinline__ PromptSeq lane_of(const PromptParams& p, int s0) const {  // sequence s0 + lane
        if (s0 == 0) return mine;
        const int s = s0 + (int)(threadIdx.x & 63);
        return s < p.B ? prompt_seq(p, s) : PromptSeq{0, 0, 0, 0};
    }
    __device__ __forceinline__ PromptSeq get(const PromptParams& p, int s) const {  // s the same in all lanes
        if (s >= 64) return prompt_seq(p, s);
        return {__builtin_amdgcn_readlane(mine.q0, s), __builtin_amdgcn_readlane(mine.nq, s), __builtin_amdgcn_readlane(mine.k0, s),
                __builtin_amdgcn_readlane(mine.nk, s)};
    }
};

// Keys that the last row of a sequence's row tile `place` sees
template <int RT>
__device__ __forceinline__ int prompt_keys(const PromptParams& p, const PromptSeq& q, int place) {
    return max(0, min(q.nk, min(q.nq - 1, prompt_token(p, (place + 1) * RT - 1)) + q.nk - q.nq + 1));
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

// A key head's items: `ahead` of the prefix over all rows (PACK; each row tile `per` of them), then each sequence's. A sequence's row tiles are all
// cut into as many as its longest needs to have at most `each` key tiles in one (early ones of a causal prompt have fewer, or none).
template <int RT, PromptMode MODE>
struct PromptItems {
    int np, each, per, ahead;
    __device__ __forceinline__ static int row_tiles(const PromptParams& p, const PromptSeq& q) { return (q.nq * p.G + RT - 1) / RT; }
    __device__ __forceinline__ int key_tiles(const PromptSeq& q) const { return max(1, (MODE == PM_PACK ? 0 : np) + (q.nk + XKT - 1) / XKT); }
    __device__ __forceinline__ int cuts(const PromptSeq& q) const { return (key_tiles(q) + each - 1) / each; }
    __device__ __forceinline__ PromptItems(const PromptParams& p, const PromptSeqs& seqs) {
        np = (p.P + XKT - 1) / XKT;
        const int all = (p.Tq * p.G + RT - 1) / RT;  // row tiles of all rows
        uint32_t n = 0;
        for (int s0 = 0; s0 < p.B; s0 += 64) {
            const PromptSeq q = seqs.lane_of(p, s0);
            n += (uint32_t)(row_tiles(p, q) * key_tiles(q));
        }
        // below 2^29 where the starts ascend; where they do not, n may be anything, and the prefix's items still stay below their number
        const int pre = MODE == PM_PACK ? all * np : 0, total = (int)((uint32_t)wave_sum((int)n) + (uint32_t)(pre + p.nw - 1));
        each = max(PROMPT_LEAST, max(total / p.nw, (pre + p.nw - 1) / p.nw));
        per = (np + each - 1) / each;
        ahead = MODE == PM_PACK ? all * per : 0;
    }
    // the sequence that holds item `at` >= ahead, or -1; at: counted from the sequence's first
    __device__ __forceinline__ int find(const PromptParams& p, const PromptSeqs& seqs, int& at) const {
        at -= ahead;
        for (int s0 = 0; s0 < p.B; s0 += 64) {
            const PromptSeq q = seqs.lane_of(p, s0);
            const int n = row_tiles(p, q) * cuts(q), up = wave_scan(n);
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

// Row tile number `rank` of all sequences' tiles of RT rows: its sequence and place there, or -1 past the last. The order goes by bands of places,
// 2^n to 2^(n+1) - 1, the highest first, so that the longest ranges of keys do not begin last; in a band sequence by sequence, so that the tiles
// that run at one time share their keys in the L2s. F(n): the number of tiles at place n or later.
template <int RT>
__device__ __forceinline__ int prompt_find(const PromptParams& p, const PromptSeqs& seqs, int rank, int& place) {
    auto tiles = [&](int s0) { return (seqs.lane_of(p, s0).nq * p.G + RT - 1) / RT; };
    const int own = tiles(0);
    if (p.B == 1) {
        place = __builtin_amdgcn_readfirstlane(own) - 1 - rank;
        return place >= 0 ? 0 : -1;
    }
    // F(n); less than 2^24 where the starts ascend, and no overflow where they do not
    auto from = [&](int n) {
        int sum = max(0, own - n);
        for (int s0 = 64; s0 < p.B; s0 += 64) sum = min(sum + max(0, tiles(s0) - n), 1 << 24);
        return wave_sum(sum);
    };
    if (rank >= from(0)) return -1;
    int lo = 0, hi = 1, fhi;  // F(lo) > rank >= F(hi) = fhi
    while ((fhi = from(hi)) > rank) lo = hi, hi *= 2;
    rank -= fhi;
    for (int s0 = 0; s0 < p.B; s0 += 64) {
        const int n = max(0, min(s0 ? tiles(s0) : own, hi) - lo), up = wave_scan(n);  // tiles in the band
        const unsigned long long past = __ballot(up > rank);
        if (past) {
            const int i = __ffsll(past) - 1;
            place = lo + __builtin_amdgcn_readlane(up, i) - 1 - rank;
            return s0 + i;
        }
        rank -= __builtin_amdgcn_readlane(up, 63);
    }
    return -1;
}

// A workgroup's geometry: RV waves of 16 QB rows, KG times: key groups that take every KG-th tile, each with a ring of NS tiles that its
// waves share, and join their results in LDS. One wave alone: a ring of its own.
template <int DH_, int QB_, int RV_, int KG_, int NS_>
struct PCfg {
    static constexpr int DH = DH_, QB = QB_, RV = RV_, KG = KG_, NS = NS_, NW = RV * KG;
    static constexpr bool SHARED = NW > 1;
    static constexpr int THREADS = 64 * NW, GTHREADS = 64 * RV, RW = 16 * QB, RT = RW * RV;  // threads of a key group, rows of a wave, of the workgroup
    static constexpr int PC = DH / 8;                                  // 16-byte chunks of a row
    static constexpr int TILE = XKT * DH * 2, STAGE = 2 * TILE;        // K tile, V tile
    static constexpr int DMA = XKT * PC / GTHREADS;                    // 16-byte pieces per thread, for K and for V each
    static constexpr int RING = NS * STAGE;
    static constexpr int JOIN = (KG - 1) * RT * (DH + 8) * 4;          // a lane's accumulators, and m and l of its rows
    static constexpr int LDS = RING * KG > JOIN ? RING * KG : JOIN;
    static constexpr int WAVES = 2;                                    // per SIMD that registers have to allow
};

template <class E, class C, PromptMode MODE>
__global__ __launch_bounds__(C::THREADS, C::WAVES) void k_prompt_attn(const PromptParams p) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass drops a kernel template whose target builtins it cannot check
    using M = XMma<E>;
    constexpr int DH = C::DH, QB = C::QB;
    extern __shared__ __attribute__((aligned(16))) uint8_t xlds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kg = wave / C::RV, wv = wave % C::RV;  // key group, rows' wave
    const int g = lane >> 4, c16 = lane & 15;
    // key heads side by side: blocks go round the 8 XCDs, so that a head's row tiles share the L2s of few, and every XCD has long and
    // short ones
    const int hk = (int)(blockIdx.x % p.Hkv), bx = (int)(blockIdx.x / p.Hkv);
    // a row tile: its sequence and place there; all its tiles, or (part) item `cut` of `cuts`
    int s = 0, jt = 0, cut = 0, cuts = 1;
    bool ahead = false;  // the prefix's pass over all rows
    const PromptSeqs seqs(p);
    if constexpr (MODE == PM_WHOLE) {
        s = prompt_find<C::RT>(p, seqs, bx, jt);
        if (s < 0) return;
    } else {
        const PromptItems<C::RT, MODE> items(p, seqs);
        if (bx == 0 && hk == 0 && threadIdx.x == 0) p.cuts[(size_t)p.Tq * p.G * 2] = items.each;
        ahead = bx < items.ahead;
        int at = bx;
        if (ahead) {
            cuts = items.per;
        } else {
            s = items.find(p, seqs, at);
            if (s < 0) return;
            cuts = items.cuts(seqs.get(p, s));
        }
        jt = at / cuts;
        cut = at % cuts;
    }
    const PromptSeq sq = ahead ? PromptSeq{0, p.Tq, 0, 0} : seqs.get(p, s);
    const int rows = sq.nq * p.G, diff = sq.nk - sq.nq;
    const int P = MODE == PM_PACK && !ahead ? 0 : p.P;
    const int row0 = jt * C::RT + wv * C::RW;
    // the row tile's own keys; its tiles: the prefix's whole ones, the own keys', the prefix's end (order is nothing to a softmax, and so those
    // with keys to hide come last)
    const int L = ahead ? 0 : prompt_keys<C::RT>(p, sq, jt);
    const int fp = P / XKT, own_end = fp + (L + XKT - 1) / XKT, kt = max(1, own_end + (P % XKT ? 1 : 0));
    const int t0 = MODE == PM_WHOLE ? 0 : (int)((long long)kt * cut / cuts), t1 = MODE == PM_WHOLE ? kt : (int)((long long)kt * (cut + 1) / cuts);
    if (MODE != PM_WHOLE && hk == 0 && !ahead && cut == 0)  // where the merge finds these rows' parts (the same for every key head)
        for (int i = threadIdx.x; i < C::RT && jt * C::RT + i < rows; i += C::THREADS)
            *reinterpret_cast<uint2*>(p.cuts + ((size_t)sq.q0 * p.G + jt * C::RT + i) * 2) = make_uint2(bx, cuts);

    uint8_t* ring = xlds + kg * C::RING;
    const uint32_t lds_base = (uint32_t)(size_t)(__attribute__((address_space(3))) uint8_t*)ring;

    // DMA of this key group's tiles t0 + kg, t0 + kg + KG, .., K and V in turn: a thread's pieces are chunks of fixed rows of a tile; the
    // descriptor's range ends with the last row of the prefix or of the own keys, and is empty from tile t1 on
    struct Stream {
        const uint8_t* src;  // the next tile to copy
        uint32_t ld2;        // bytes from row to row
        int left;            // rows from its first on
        int j, end;          // its number, and where the rows' stretch ends
        uint32_t off[C::DMA];
    } kst, vst;
    auto place = [&](Stream& t, const void* pre, size_t ld_pre, const void* own, size_t ld_own, auto is_k) {  // the stretch of tile t.j
        const bool mine = t.j >= fp && t.j < own_end;
        const size_t ld = mine ? ld_own : ld_pre;
        const uint32_t ld2 = t.ld2 = (uint32_t)ld * 2;
        const int tile = t.j < fp ? t.j : mine ? t.j - fp : fp;  // its place in the stretch's rows
        const int rows = t.j >= t1 ? 0 : mine ? min(L, (t1 - fp) * XKT) : min(P, t1 * XKT);
        t.end = t.j < fp ? fp : mine ? own_end : 0x7fffffff;
        t.src = static_cast<const uint8_t*>(mine ? own : pre) + ((mine ? (long long)sq.k0 * ld : 0) + (long long)hk * DH) * 2 + (long long)tile * XKT * ld2;
        t.left = rows - tile * XKT;
#pragma unroll
        for (int i = 0; i < C::DMA; i++) {
            const int pc = i * C::GTHREADS + wv * 64 + lane, r = pc / C::PC, c = pc % C::PC;
            t.off[i] = r * ld2 + (decltype(is_k)::value ? k_swz<DH>(c, r) : v_swz<DH>(c, r)) * 16;
        }
    };
    auto copy = [&](Stream& t, uint32_t at, const void* pre, size_t ld_pre, const void* own, size_t ld_own, auto is_k) {
        if (t.j >= t.end) place(t, pre, ld_pre, own, ld_own, is_k);
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(t.src), (short)0, t.left > 0 ? (int)((min(t.left, XKT) - 1) * t.ld2 + DH * 2) : 0, 0x00020000 /* raw */);
        uint8_t* dst = ring + at + wv * 1024;
#pragma unroll
        for (int i = 0; i < C::DMA; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(dst + i * C::GTHREADS * 16), 16, t.off[i], 0, 0, 0);
        t.src += (size_t)C::KG * XKT * t.ld2;
        t.left -= C::KG * XKT;
        t.j += C::KG;
    };
    kst.j = vst.j = t0 + kg;
    place(kst, p.pk, p.ldpk, p.k, p.ldk, std::true_type{});
    place(vst, p.pv, p.ldpv, p.v, p.ldv, std::false_type{});
    auto copy_k = [&](int stage) { copy(kst, stage * C::STAGE, p.pk, p.ldpk, p.k, p.ldk, std::true_type{}); };
    auto copy_v = [&](int stage) { copy(vst, stage * C::STAGE + C::TILE, p.pv, p.ldpv, p.v, p.ldv, std::false_type{}); };

    // Q: the B operands of S^T, lane (row c16, chunk 4 cc + g); rows past the last read the last and are not stored. lim: the own keys
    // that a row sees
    u32x4 qf[QB][DH / 32];
    int lim[QB];
#pragma unroll
    for (int qb = 0; qb < QB; qb++) {
        const int r = min(row0 + 16 * qb + c16, rows - 1), t = prompt_token(p, r), h = hk * p.G + r - t * p.G;
        const uint8_t* src = static_cast<const uint8_t*>(p.q) + ((long long)(sq.q0 + t) * p.ldq + (long long)h * DH + 8 * g) * 2;
#pragma unroll
        for (int cc = 0; cc < DH / 32; cc++) qf[qb][cc] = *reinterpret_cast<const u32x4*>(src + 64 * cc);
        lim[qb] = t + diff + 1;
    }
    const int lim0 = prompt_token(p, min(row0, rows - 1)) + diff + 1;  // of the wave's first row

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
    // The first tile with keys that some row of the wave does not see (the prefix's end, at last); own ones from `from_apart` on hold keys that
    // some row of the workgroup sees, up to L, but the wave's first does not (with 32 or more query heads on a key head none of the wave's may).
    const int from_hide = min(C::KG > 1 ? min(t1, own_end) : own_end, fp + max(lim0, 0) / XKT);
    const int from_apart = lim0 < L ? fp + max(lim0, 0) / XKT : 0x7fffffff;
    // a row sees the first lim - (its first own key) of tile j's keys, or all up to the prefix's end; none of a tile past the last
    auto hide = [&](int j, floatx4 (&s)[2][QB]) {
        if (j < from_hide) return;
#pragma unroll
        for (int qb = 0; qb < QB; qb++) {
            const int seen = (C::KG > 1 && j >= t1 ? 0 : j < own_end ? lim[qb] - (j - fp) * XKT : P % XKT) - 4 * g;
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
    // Tile j, with keys that not all rows of this wave see: infinities and NaNs of V leave the operands; the rows that see them take
    // their products here. V's rows are read from the stage itself, four dimensions of a key a lane, as the accumulators lie.
    auto keep_apart = [&](int j, uint32_t st, u32x4 (&vf)[DH / 16], const u32x4 (&pf)[QB]) __attribute__((always_inline)) {
        floatx4 z[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int db = 0; db < DH / 16; db++) z[db & 1] = M::mul(vf[db], u32x4{0, 0, 0, 0}, z[db & 1]);
        z[0] += z[1];
        const float zs = (z[0][0] + z[0][1]) + (z[0][2] + z[0][3]);
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
                const bool sees = (j - fp) * XKT + key < lim[qb];
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

    if constexpr (C::SHARED) {
        // A step computes the scores of tile j + 1 ahead of the weights and products of tile j. K of tile j + 1 and V of tile j landed (past
        // the last tile the copies go on with empty ranges, which keeps the count); every wave is done with K of tile j and V of tile
        // j - 1, whose places take K of tile j + NS and V of tile j + NS - 1.
        constexpr int NS = C::NS, KG = C::KG;
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
        hide(t0 + kg, sc[0]);
        largest(sc[0], top);
        auto begin = [&](auto st) {
            x_wait_vmcnt<2 * (NS - 2) * C::DMA>();
            __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
        };
        // (behind the reads of V: the compiler has each wait for all copies that are under way)
        auto copies = [&](auto st) {
            __builtin_amdgcn_sched_barrier(0);
            copy_k(st);
            copy_v((st + NS - 1) % NS);
            __builtin_amdgcn_sched_barrier(0);
        };
        auto products = [&]() {
#pragma unroll
            for (int qb = 0; qb < QB; qb++) l[qb] = M::mul(ones, pf[qb], l[qb]);
#pragma unroll
            for (int db = 0; db < DH / 16; db++)
#pragma unroll
                for (int qb = 0; qb < QB; qb++) o[db][qb] = M::mul(vf[db], pf[qb], o[db][qb]);
        };
        auto step = [&](auto parity, auto st) {  // a tile with nothing to hide, nor the next, at a stage that is a constant
            constexpr int cur = decltype(parity)::value;
            begin(st);
            read_k((st + 1) % NS * C::STAGE, kf);
#pragma unroll
            for (int db = 0; db < DH / 16; db++) vf[db] = read_v(st * C::STAGE, db);
            copies(st);
            rescale(top, sc[cur]);
            __builtin_amdgcn_sched_barrier(0);
            weights(sc[cur], pf);
            scores(kf, sc[cur ^ 1]);
            __builtin_amdgcn_sched_barrier(0);
            products();
            largest(sc[cur ^ 1], top);
        };
        auto step_any = [&](int j, int st) {  // any tile, any stage
            begin(st);
            read_k((st + 1) % NS * C::STAGE, kf);
#pragma unroll
            for (int db = 0; db < DH / 16; db++) vf[db] = read_v(st * C::STAGE, db);
            copies(st);
            rescale(top, sc[0]);
            __builtin_amdgcn_sched_barrier(0);
            weights(sc[0], pf);
            scores(kf, sc[0]);
            __builtin_amdgcn_sched_barrier(0);
            if (j >= from_apart && j < own_end) keep_apart(j, st * C::STAGE, vf, pf);
            products();
            hide(j + KG, sc[0]);
            largest(sc[0], top);
        };
        using P0 = std::integral_constant<int, 0>;
        using P1 = std::integral_constant<int, 1>;
        // First the tiles with nothing to hide in any wave, two steps at a time, their stages constants; then the others one by one. (The
        // groups take the same number of steps: the second's last tile may lie past the end.)
        const int special = min(t1, min(own_end, fp + max(prompt_token(p, min(jt * C::RT, rows - 1)) + diff + 1, 0) / XKT));
        int j = t0 + kg, st = 0;
        for (; j - kg + NS * KG + KG - 1 < special; j += NS * KG) {
            step(P0{}, P0{});
            step(P1{}, P1{});
            if constexpr (NS == 4) {
                step(P0{}, std::integral_constant<int, 2>{});
                step(P1{}, std::integral_constant<int, 3>{});
            }
        }
        for (; j - kg < t1; j += KG, st = (st + 1) % NS) step_any(j, st);
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
            if (j >= from_apart && j < own_end) keep_apart(j, st, vf, pf);
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
    if constexpr (C::KG > 1) {
        // the second group's results go to the first's lanes, which hold the same rows and dimensions
        static_assert(C::KG == 2, "two groups");
        floatx4* jo = reinterpret_cast<floatx4*>(xlds) + wv * (DH / 16 * QB + QB) * 64 + lane;
        __builtin_amdgcn_s_waitcnt(0xC07F);
        __builtin_amdgcn_s_barrier();  // every wave is done with the rings, and its copies landed
        __builtin_amdgcn_sched_barrier(0);
        if (kg == 1) {
#pragma unroll
            for (int qb = 0; qb < QB; qb++) {
#pragma unroll
                for (int db = 0; db < DH / 16; db++) jo[(qb * (DH / 16) + db) * 64] = o[db][qb];
                jo[(QB * (DH / 16) + qb) * 64] = floatx4{m[qb], l[qb][0], 0.f, 0.f};
            }
        }
        __syncthreads();
        if (kg == 0) {
#pragma unroll
            for (int qb = 0; qb < QB; qb++) {
                const floatx4 e = jo[(QB * (DH / 16) + qb) * 64];
                const float t = fmaxf(m[qb], e[0]), te = t == -INFINITY ? 0.f : t;
                const float f0 = __builtin_amdgcn_exp2f(m[qb] - te), f1 = __builtin_amdgcn_exp2f(e[0] - te);
                m[qb] = t;
                l[qb][0] = f0 * l[qb][0] + f1 * e[1];
#pragma unroll
                for (int db = 0; db < DH / 16; db++) o[db][qb] = f0 * o[db][qb] + f1 * jo[(qb * (DH / 16) + db) * 64];
            }
        }
        __syncthreads();
    }

    if (kg != 0) return;
    if (MODE == PM_PACK || (MODE == PM_SPLIT && cuts > 1)) {
        const size_t base = ((size_t)hk * p.items + bx) * C::RT + wv * C::RW;
#pragma unroll
        for (int qb = 0; qb < QB; qb++) {
            if (row0 + 16 * qb + c16 >= rows) continue;
            const size_t at = base + 16 * qb + c16;
#pragma unroll
            for (int db = 0; db < DH / 16; db++) *reinterpret_cast<floatx4*>(p.part + at * DH + 16 * db + 4 * g) = o[db][qb];
            if (g == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m[qb], l[qb][0]);
        }
        return;
    }
    // rows leave through LDS, whole and 16 bytes a lane; a row's chunks lie permuted by its number
    static_assert(C::RT * DH * 2 <= C::LDS, "the waves' rows fit in the rings");
    uint8_t* stg = xlds + wv * C::RW * DH * 2;
    if constexpr (C::SHARED && C::KG == 1) __builtin_amdgcn_s_barrier();  // every wave is done with the ring, and its copies landed
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
        const int t = prompt_token(p, r), h = hk * p.G + r - t * p.G;
        *reinterpret_cast<u32x4*>(static_cast<uint8_t*>(p.o) + ((long long)(sq.q0 + t) * p.ldo + (long long)h * DH + c * 8) * 2) = v;
    }
#endif
}

// The partial results of a row joined, in the line's order: a wave per row. Loads in flight are what it waits for: 16 where there are many (a token
// after 8191 keys 17.8 -> 14.8 us, of 64 parts; 32 tokens behind a prefix of 4096 17.9 -> 17.1, of 21), 4 where a few are left.
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
    const uint2 cut = *reinterpret_cast<const uint2*>(p.cuts + R * 2);
    const int r = (int)(R - (long long)prompt_seq(p, s).q0 * p.G), w = (int)cut.x, n = (int)cut.y;
    if (cut.x >= (uint32_t)p.items || cut.y > (uint32_t)p.items - cut.x) return;  // (starts that do not ascend: a tile too many, never begun)
    if (MODE == PM_SPLIT && n == 1) return;  // written by its workgroup
    int n2 = 0;
    if (MODE == PM_PACK) {
        const int np = (p.P + XKT - 1) / XKT, each = (int)p.cuts[(size_t)p.Tq * p.G * 2];
        n2 = (np + each - 1) / each;
    }
    auto index = [&](int i) -> size_t {  // of the row's partial result i
        const bool own = MODE == PM_SPLIT || i < n;
        return ((size_t)hk * p.items + (own ? w + i : (int)(R / RT) * n2 + i - n)) * RT + (own ? r % RT : (int)(R % RT));
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
        auto take = [&](int i, auto n) {  // n at once
            constexpr int N = decltype(n)::value;
            vec v[N];
#pragma unroll
            for (int k = 0; k < N; k++) v[k] = *reinterpret_cast<const vec*>(p.part + index(i0 + min(i + k, end - 1)) * DH + PER * lane);
#pragma unroll
            for (int k = 0; k < N; k++) acc += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), i + k)) * (i + k < end ? v[k] : vec(0.f));
        };
        int i = 0;
        for (; i + 8 < end; i += 16) take(i, std::integral_constant<int, 16>{});
        for (; i < end; i += 4) take(i, std::integral_constant<int, 4>{});
    }
#pragma unroll
    for (int i = 32; i; i >>= 1) ll += __shfl_xor(ll, i, 64);
    const float inv = ll > 0.f || ll != ll ? 1.f / ll : 0.f;
    uint8_t* dst = static_cast<uint8_t*>(p.o) + ((long long)t * p.ldo + (long long)(hk * p.G + (int)(R % p.G)) * DH + PER * lane) * 2;
    if constexpr (PER == 2) *reinterpret_cast<uint32_t*>(dst) = XMma<E>::pack(acc[0] * inv, acc[1] * inv);
    else *reinterpret_cast<uint16_t*>(dst) = __builtin_bit_cast(uint16_t, (E)(acc[0] * inv));
#endif
}

// The form of a call. Rows, keys and work are guesses from the tensors' sizes, the same for every sequence: lengths are on the device. Where one has
// most of the keys, or many read the same ones, WHOLE may be taken for long ranges: a token after 8191 keys among 63 after 50 112 us (alone, shared
// out, 14.8), 32 tokens that all read one place of 8192 keys 110.
struct PromptForm {
    PromptMode mode;
    int rt;     // rows of a workgroup: 16 (a wave alone), 64 (two row waves by two key groups), 128 (four row waves)
    int nw;     // keys shared out: workgroups per key head
};
//
// The times of both ways are modelled in us. WHOLE: a workgroup's start and its longest range of keys, once per round of workgroups. Shared
// out: the merge and two starts, then all tiles over the whole chip. Per 32 keys of a 64-row tile 0.4 us (heads of 64: 0.22). Fitted to, WHOLE / shared
// out, 16 heads on 8 of 128: 3 x 100 rows after 4000 keys (32 on 4 of 64) 37.3 / 20.7; 300 after 8000 106 / 40; 8 x 100 after 1000 20.5 / 23.1; 40 after
// 1000 18.9 / 12.5; single tokens, 16 after 8191 175 / 81; 2 after 600 12.5 / 9.7; 64 after 600 22.3 / 23.8; 32 after 200 8.7 / 9.9. A prefix once for
// all: 64 tokens behind 8192 140 / 30, 8 x 8 behind 4000 51 / 15.
// Up to 16 rows a sequence take 16-row tiles, but 64-row ones where a prefix before many sequences passes through LDS too often. Fitted to, 16 / 64
// rows, tokens with 200 keys of their own behind a prefix: 32 behind 1000 13.6 / 17.0, behind 4096 18.0 / 20.5; 64 behind 1000 20.4 / 24.9, behind 8192 37.9 /
// 29.2, behind 4096 (32 heads on 4 of 64) 21.4 / 17.3; 128 with 100 behind 4096 35.1 / 33.7; 8 x 8 behind 4000 17.2 / 19.1.
// 128 rows share a tile's way from LDS among more, but have to fill the chip some rounds over, or have few keys each: 64 / 128 rows, 24 prompts
// of up to 2000 400 / 290, one of 8192 287 / 254, of 4096 80 / 95, of 3000 49 / 68; 8 of up to 500 22.4 / 19.2.
static PromptForm prompt_form(int B, int Tq, int Tk, int P, int Hq, int Hkv, int Dh, bool split) {
    const long G = Hq / Hkv, cus = cu_count(), rows = std::max<long>(1, (long)Tq * G / B);
    const double tile = Dh == 64 ? 0.22 : 0.4, own = tile * Tk / B / XKT, pre = tile * P / XKT;
    auto tiles = [&](long rt) { return std::max<long>(B, (long)Tq * G / rt) * Hkv; };
    const double fill = tiles(64) / (2.0 * cus), least = 0.05;  // of a round
    const bool pack = P >= 2 * XKT && B > 1 && rows <= 32;
    const double whole = 5 + (own + pre) * std::max(1.0, fill);
    const double pre_fill = pack ? ((double)Tq * G / 64 + 1) * Hkv / (2.0 * cus) : fill;
    const double shared = (rows <= 16 ? 9 : 15) + 1.5 * (own * std::max(fill, least) + pre * std::max(pre_fill, least));
    // items are counted in 32 bits, whatever the lengths
    const bool fits = ((long)Tq * G / 16 + B) * ((Tk + (long)P) / XKT + 2) < 1 << 29;
    if (!split || !fits || whole <= shared) return {PM_WHOLE, tiles(128) >= 4 * cus || (own + pre <= 16 * tile && fill > 1) ? 128 : 64, 0};
    const double unit = (Dh == 64 ? 0.55 : 1) * Hkv * 32 / cus, own_tiles = (double)Tk / XKT + B;  // of a 16-row tile by 32 keys of 8 heads of 128
    auto units = [&](long rt) { return unit * (((double)Tq * G / rt + 1) * P / XKT + own_tiles); };
    const int rt = rows > 16 || (pack && 15 + 0.0165 * units(64) < 8 + 0.0115 * units(16)) ? 64 : 16;
    // one round of workgroups: four single waves a CU, or two of 64 rows, less what the row tiles' rounding adds
    const long slots = (rt == 16 ? 4 : 2) * cus / Hkv, over = (long)Tq * G / rt + B;
    return {pack ? PM_PACK : PM_SPLIT, rt, (int)std::max<long>(std::max<long>(1, slots / 2), slots - over)};
}
// items per key head at most: every row tile rounds its parts up
static size_t prompt_items(const PromptForm& f, int B, int Tq, int G) {
    return f.mode == PM_WHOLE ? 0 : f.nw + (size_t)Tq * G / f.rt + B + (f.mode == PM_PACK ? (size_t)Tq * G / f.rt + 1 : 0);
}
size_t prompt_attn_workspace(int B, int Tq, int Tk, int P, int Hq, int Hkv, int Dh) {
    const PromptForm f = prompt_form(B, Tq, Tk, P, Hq, Hkv, Dh, true);
    const size_t rows = prompt_items(f, B, Tq, Hq / Hkv) * Hkv * f.rt;
    return rows ? rows * (Dh + 2) * sizeof(float) + ((size_t)Tq * (Hq / Hkv) * 2 + 2) * sizeof(uint32_t) : 0;
}

int prompt_attn_form(int B, int Tq, int Tk, int P, int Hq, int Hkv, int Dh) {
    const PromptForm f = prompt_form(B, Tq, Tk, P, Hq, Hkv, Dh, true);
    return f.rt << 16 | (int)f.mode;
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
    if (hipError_t e = grid_check((size_t)p.items * p.Hkv, C::THREADS)) return e;
    hipLaunchKernelGGL((k_prompt_attn<E, C, MODE>), dim3((unsigned)((size_t)p.items * p.Hkv)), dim3(C::THREADS), C::LDS, s, p);
    if (hipError_t e = hipGetLastError()) return e;
    hipLaunchKernelGGL((k_prompt_merge<E, C::DH, C::RT, MODE>), dim3((unsigned)merges), dim3(256), 0, s, p);
    return hipGetLastError();
}
template <class E, int DH>
static hipError_t prompt_of(const PromptParams& p, const PromptForm& f, hipStream_t s) {
    using One = PCfg<DH, 1, 1, 1, 2>;
    using R64 = PCfg<DH, 2, 2, 2, 2>;
    using R128 = PCfg<DH, 2, 4, 1, 4>;
    if (f.mode == PM_WHOLE) return f.rt == 128 ? prompt_whole<E, R128>(p, s) : prompt_whole<E, R64>(p, s);
    if (f.mode == PM_PACK) return f.rt == 16 ? prompt_split<E, One, PM_PACK>(p, s) : prompt_split<E, R64, PM_PACK>(p, s);
    return f.rt == 16 ? prompt_split<E, One, PM_SPLIT>(p, s) : prompt_split<E, R64, PM_SPLIT>(p, s);
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
    p.g_shift = 31;
    while ((1 << (p.g_shift - 31)) < p.G) p.g_shift++;
    p.g_mul = (uint32_t)(((1ull << p.g_shift) + p.G - 1) / p.G);
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
    p.items = (int)prompt_items(f, c.B, c.Tq, p.G);
    const size_t rows = (size_t)p.items * c.Hkv * f.rt;
    p.part = static_cast<float*>(c.ws);
    p.part_ml = p.part + rows * c.Dh;
    p.cuts = reinterpret_cast<uint32_t*>(p.part_ml + rows * 2);
    if (c.dt == DT::F16) return c.Dh == 64 ? prompt_of<_Float16, 64>(p, f, s) : prompt_of<_Float16, 128>(p, f, s);
    return c.Dh == 64 ? prompt_of<__bf16, 64>(p, f, s) : prompt_of<__bf16, 128>(p, f, s);
}

}  // namespace kiln
