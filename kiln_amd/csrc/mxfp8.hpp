// Microscaled 8-bit floating point (MXFP8): 32 neighbours of a row share the scale 2^(s - 127) of one byte s, and each is an e4m3 code
// (sign, exponents 2^-6 .. 2^8, three bits of mantissa; steps of 2^-9 below 2^-6; largest 448, no infinities, 0x7f NaN).
#pragma once
#include "mxfp4.hpp"

namespace kiln {

typedef short s16x2 __attribute__((ext_vector_type(2)));

// The scale byte of a block whose largest magnitude has the fp32 bits `top`: the smallest power of two 2^e with top <= 448 2^e, so that no
// value saturates and every one is rounded by half a step of its own (with 2^(floor(log2 top) - 8), MXFP4's rule, magnitudes in
// 448 .. 512 times the scale would lose up to an eighth). 448 is 1.75 2^8: a larger mantissa takes the next exponent. Exponents below
// 2^-127 stop there; a block with an infinity or a NaN takes the NaN byte.
__device__ __forceinline__ uint32_t mx8_scale(uint32_t top) {
    if (top >= 0x7f800000u) return 255u;
    const uint32_t e = (top + 0x1fffffu) >> 23;
    return e > 8 ? e - 8 : 0u;
}
// the codes of four values over a scale (round to nearest even)
__device__ __forceinline__ uint32_t mx8_codes4(float a, float b, float c, float d, float scale) {
    s16x2 r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, a, b, scale, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, scale, true);
    return __builtin_bit_cast(uint32_t, r);
}
// Eight neighbours of a lane, four lanes to a block: their codes and the block's scale byte
__device__ __forceinline__ u32x2 mx8_quad(const float (&v)[8], uint32_t& s) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);  // NaNs order above infinity
    s = mx8_scale(quad_umax(top));
    const float sc = mx_scale_f32(s);
    u32x2 c = {mx8_codes4(v[0], v[1], v[2], v[3], sc), mx8_codes4(v[4], v[5], v[6], v[7], sc)};
    if (s == 255) c = u32x2{0, 0};
    return c;
}


// Eight elements as fp32, from rows in fp32, fp16 or bf16; VEC: 16-byte aligned, all eight there (otherwise the first `have`, zeros after)
template <bool VEC, class E>
__device__ __forceinline__ void load8f(const E* p, int have, float (&v)[8]) {
    if constexpr (!VEC) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < have ? (float)p[i] : 0.f;
    } else {
        typedef E V __attribute__((ext_vector_type(16 / sizeof(E))));
#pragma unroll
        for (int j = 0; j < 8; j += 16 / (int)sizeof(E)) {
            const V x = *reinterpret_cast<const V*>(p + j);
#pragma unroll
            for (int e = 0; e < 16 / (int)sizeof(E); e++) v[j + e] = (float)x[e];
        }
    }
}
template <bool VEC, class E>
__device__ __forceinline__ void store8f(E* p, int have, const float (&v)[8]) {  // rounded to nearest even
    if constexpr (!VEC) {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < have) p[i] = (E)v[i];
    } else {
        typedef E V __attribute__((ext_vector_type(16 / sizeof(E))));
#pragma unroll
        for (int j = 0; j < 8; j += 16 / (int)sizeof(E)) {
            V x;
#pragma unroll
            for (int e = 0; e < 16 / (int)sizeof(E); e++) x[e] = (E)v[j + e];
            *reinterpret_cast<V*>(p + j) = x;
        }
    }
}

}  // namespace kiln
