// Rotary positions of a projection's heads: kiln_rope.
//
// For token t at position p and pair i of a head, with a = p f_i:  (u, v) -> m (u cos a - v sin a, v cos a + u sin a).
// Pairs are (i, i + rot/2) or (2i, 2i + 1) of the head's first rot dimensions; the others pass unchanged.
//
// Bound by memory: every element is read and written once. The angle is the one part that is not: p f_i is taken in 64
// bits (at position 10^6 a 32-bit product is off by 0.06 rad) and reduced to a fraction of a turn before its sine and
// cosine, which are full-precision 32-bit ones. A workgroup takes tb tokens, computes their rot/2 pairs of (cos, sin) once
// into LDS, and turns all of their heads with them, so the angles cost 1/H of an evaluation per pair. 16-byte loads and
// stores where the rows and the pair halves allow them; any alignment and any even rot otherwise. 32768 tokens x 20 heads of 128
// in fp16: 69 us, 4.8 TB/s (a large copy 5.2).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.hpp"
#include "internal.hpp"

namespace kiln {

struct RopeParams {
    const void* x;
    void* y;
    size_t ldx, ldy;
    int T, H, Dh, rot;
    const int* pos;
    int pos0;
    const double* freqs;
    float mscale;
    int tb, hb;               // tokens and heads of a workgroup
    int np, nu;               // units of a head: np pair units, then copies of the dimensions that do not turn
    uint64_t inv_hu, inv_u;   // ceil(2^32 / (hb nu)), ceil(2^32 / nu): exact quotients below 2^16
};

constexpr int ROPE_THREADS = 256, ROPE_MAX_UNITS = 1 << 16;

template <class E, int N>
struct RopeVec {
    typedef E T __attribute__((ext_vector_type(N)));
};
template <class E>
struct RopeVec<E, 1> {
    typedef E T;
};
template <class E>
__device__ __forceinline__ float rope_get(const E& v, int) { return (float)v; }
template <class E>
__device__ __forceinline__ void rope_set(E& v, int, float f) { v = (E)f; }
#define ROPE_VEC_OPS(E, N)                                                                              \
    __device__ __forceinline__ float rope_get(const typename RopeVec<E, N>::T& v, int e) { return (float)v[e]; } \
    __device__ __forceinline__ void rope_set(typename RopeVec<E, N>::T& v, int e, float f) { v[e] = (E)f; }
ROPE_VEC_OPS(float, 4)
ROPE_VEC_OPS(_Float16, 8)
ROPE_VEC_OPS(__bf16, 8)

// N elements a unit's half (half pairs) or a whole unit (interleaved pairs); 1 for the general form
template <class E, int N, bool INTER>
__global__ __launch_bounds__(ROPE_THREADS) void k_rope(const RopeParams p) {
    extern __shared__ float2 cs[];  // [tb][rot / 2]: m cos, m sin
    using V = typename RopeVec<E, N>::T;
    const int t0 = blockIdx.x * p.tb, h0 = blockIdx.y * p.hb;
    const int nt = min(p.tb, p.T - t0), nh = min(p.hb, p.H - h0), half = p.rot >> 1;
    for (int j = threadIdx.x; j < nt * half; j += ROPE_THREADS) {
        const int t = j / half, i = j - t * half;
        const double at = p.pos ? (double)p.pos[t0 + t] : (double)p.pos0 + (double)(t0 + t);
        const double turns = at * p.freqs[i] * 0.15915494309189533577;
        float s, c;
        sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
        cs[j] = make_float2(p.mscale * c, p.mscale * s);
    }
    __syncthreads();
    const E* x = static_cast<const E*>(p.x);
    E* y = static_cast<E*>(p.y);
    const int units = nt * p.hb * p.nu;
    for (int j = threadIdx.x; j < units; j += ROPE_THREADS) {
        const int t = (int)(((uint64_t)(uint32_t)j * p.inv_hu) >> 32), r = j - t * (p.hb * p.nu);
        const int h = (int)(((uint64_t)(uint32_t)r * p.inv_u) >> 32), u = r - h * p.nu;
        if (h >= nh) continue;
        const E* xr = x + (size_t)(t0 + t) * p.ldx + (size_t)(h0 + h) * p.Dh;
        E* yr = y + (size_t)(t0 + t) * p.ldy + (size_t)(h0 + h) * p.Dh;
        const float2* ct = cs + t * half;
        if (u >= p.np) {
            const int d = p.rot + (u - p.np) * N;
            *reinterpret_cast<V*>(yr + d) = *reinterpret_cast<const V*>(xr + d);
        } else if constexpr (INTER && N > 1) {
            V v = *reinterpret_cast<const V*>(xr + u * N), o;
#pragma unroll
            for (int e = 0; e < N; e += 2) {
                const float2 k = ct[(u * N + e) >> 1];
                const float a = rope_get(v, e), b = rope_get(v, e + 1);
                rope_set(o, e, a * k.x - b * k.y);
                rope_set(o, e + 1, b * k.x + a * k.y);
            }
            *reinterpret_cast<V*>(yr + u * N) = o;
        } else {
            const int d0 = INTER ? 2 * u : u * N, d1 = INTER ? 2 * u + 1 : half + u * N;
            V a = *reinterpret_cast<const V*>(xr + d0), b = *reinterpret_cast<const V*>(xr + d1), oa, ob;
#pragma unroll
            for (int e = 0; e < N; e++) {
                const float2 k = ct[u * N + e];
                const float fa = rope_get(a, e), fb = rope_get(b, e);
                rope_set(oa, e, fa * k.x - fb * k.y);
                rope_set(ob, e, fb * k.x + fa * k.y);
            }
            *reinterpret_cast<V*>(yr + d0) = oa;
            *reinterpret_cast<V*>(yr + d1) = ob;
        }
    }
}

template <class E>
static hipError_t rope_of(RopeParams p, bool inter, bool aligned, hipStream_t s) {
    constexpr int N = 16 / (int)sizeof(E);
    const bool vec = aligned && p.Dh % N == 0 && p.rot % (inter ? N : 2 * N) == 0;
    const int n = vec ? N : 1;
    p.np = vec && inter ? p.rot / n : p.rot / 2 / n;
    p.nu = p.np + (p.x == p.y ? 0 : (p.Dh - p.rot) / n);  // in place the rest stays where it is
    // a workgroup takes about 1024 units of whole tokens; a few tokens are spread over workgroups by heads
    p.hb = std::min(p.H, std::max(1, ROPE_MAX_UNITS / 2 / p.nu));
    p.tb = std::max(1, std::min({1024 / (p.hb * p.nu), 32, 8192 / p.rot}));
    while (p.tb > 1 && (p.T + p.tb - 1) / p.tb < 2 * cu_count()) p.tb /= 2;
    if (p.tb == 1 && p.T < cu_count()) p.hb = std::min(p.hb, std::max(1, ROPE_THREADS / p.nu));
    p.inv_hu = ((1ull << 32) + p.hb * p.nu - 1) / (p.hb * p.nu);
    p.inv_u = ((1ull << 32) + p.nu - 1) / p.nu;
    const dim3 grid((p.T + p.tb - 1) / p.tb, (p.H + p.hb - 1) / p.hb);
    if (hipError_t e = grid_check(grid.x, ROPE_THREADS)) return e;
    const size_t lds = (size_t)p.tb * (p.rot / 2) * sizeof(float2);
    auto kern = vec ? (inter ? k_rope<E, N, true> : k_rope<E, N, false>) : (inter ? k_rope<E, 1, true> : k_rope<E, 1, false>);
    hipLaunchKernelGGL(kern, grid, dim3(ROPE_THREADS), lds, s, p);
    return hipGetLastError();
}

hipError_t launch_rope(void* y, size_t ldy, const void* x, size_t ldx, DT dt, int T, int H, int Dh, int rot, bool inter,
                       const int* pos, int pos0, const double* freqs, float mscale, hipStream_t s) {
    RopeParams p{};
    p.x = x;
    p.y = y;
    p.ldx = ldx;
    p.ldy = ldy;
    p.T = T;
    p.H = H;
    p.Dh = Dh;
    p.rot = rot;
    p.pos = pos;
    p.pos0 = pos0;
    p.freqs = freqs;
    p.mscale = mscale;
    const size_t e = dt == DT::F32 ? 4 : 2;
    const bool aligned = (((uintptr_t)x | (uintptr_t)y) & 15) == 0 && (T == 1 || ((ldx | ldy) * e) % 16 == 0);
    switch (dt) {
        case DT::F32: return rope_of<float>(p, inter, aligned, s);
        case DT::F16: return rope_of<_Float16>(p, inter, aligned, s);
        default: return rope_of<__bf16>(p, inter, aligned, s);
    }
}

}  // namespace kiln
