// Microscaled 4-bit floating point (MXFP4): 32 neighbours of a row share the scale 2^(s - 127) of one byte s, and each is
// a code of sign and magnitude 0, 0.5, 1, 1.5, 2, 3, 4, 6 (the OCP microscaling formats' E2M1 with E8M0 scales).
//
// Operand layout of a [rows, cols] matrix, as the scaled matrix instruction of 16 x 16 x 128 reads it (lane l: row l % 16,
// k block of 32 l / 16):
//   codes   [KB][rows / 16][lane 64][16 bytes]   unit (k block of 128, row block): 1 KB, in the instruction's lane order
//   scales  [KB][rows / 64][lane 64][4 bytes]    byte j: row block 4 (row / 64) + j
// with rows padded to 64 and KB = ceil(cols / 128). Codes and scales of the padding are 0, so it adds nothing. The k block comes
// first: workgroups of a product are at about the same k block, and its row blocks side by side lie in all of an L2's channels
// (with the row block first they were KB kilobytes apart, often in the same few).
#pragma once
#include <algorithm>

#include "common.hpp"
#include "internal.hpp"

namespace kiln {

constexpr int MXB = 32;           // values that share a scale
constexpr int MX_UNIT = 1024;     // bytes of a unit of codes
constexpr int MX_SUNIT = 256;     // bytes of a unit of scales (64 rows)
__host__ __device__ inline int mx_kb(int cols) { return (cols + 127) / 128; }
__host__ __device__ inline int mx_rg(int rows) { return (rows + 63) / 64; }  // groups of 64 rows
__host__ __device__ inline size_t mx_code_bytes(int rows, int cols) { return (size_t)((rows + 63) / 64) * 4 * mx_kb(cols) * MX_UNIT; }
__host__ __device__ inline size_t mx_scale_bytes(int rows, int cols) { return (size_t)((rows + 63) / 64) * mx_kb(cols) * MX_SUNIT; }

typedef __bf16 bf2v __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// The scale byte of a block whose largest magnitude has the fp32 bits `top`: 2^(floor(log2 top) - 2), 2 being the largest
// exponent of a code, so that the largest value lands on 4 .. 8 and rounds to 4 or 6 (above 6: saturates). Exponents
// below 2^-127 stop there; a block with an infinity or a NaN has no scale and takes the NaN byte.
__device__ __forceinline__ uint32_t mx_scale(uint32_t top) {
    const uint32_t e = top >> 23;
    return e == 255 ? 255u : e >= 2 ? e - 2 : 0u;
}
// 2^(s - 127) as fp32; the byte 0 is the subnormal 2^-127
__device__ __forceinline__ float mx_scale_f32(uint32_t s) { return __uint_as_float(s ? s << 23 : 0x00400000u); }

// n neighbours of one lane as loaded: the largest magnitude's bits, and their codes for a scale (round to nearest even
// and saturate, the conversion instruction's own rule)
template <class E, int N>
struct MxVals;
template <int N>
struct MxVals<float, N> {
    floatx4 v[N / 4];
    __device__ __forceinline__ void load(const float* p) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) v[i] = reinterpret_cast<const floatx4*>(p)[i];
    }
    __device__ __forceinline__ void load_any(const float* p, int have) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i / 4][i % 4] = i < have ? p[i] : 0.f;
    }
    __device__ __forceinline__ uint32_t top() const {  // magnitudes order as their bits do, NaNs above infinity
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < N; i++) m = max(m, __float_as_uint(v[i / 4][i % 4]) & 0x7fffffffu);
        return m;
    }
    __device__ __forceinline__ uint32_t codes8(int i, float s) const {
        uint32_t c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2 * i][0], v[2 * i][1], s, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2 * i][2], v[2 * i][3], s, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2 * i + 1][0], v[2 * i + 1][1], s, 2);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2 * i + 1][2], v[2 * i + 1][3], s, 3);
    }
};
// the two 16-bit types: v holds bit patterns
template <class E, int N>
struct MxVals16 {
    u32x4 v[N / 8];
    __device__ __forceinline__ void load(const E* p) {
#pragma unroll
        for (int i = 0; i < N / 8; i++) v[i] = reinterpret_cast<const u32x4*>(p)[i];
    }
    __device__ __forceinline__ void load_any(const E* p, int have) {
        const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
        for (int i = 0; i < N / 2; i++)
            v[i / 4][i % 4] = (2 * i < have ? q[2 * i] : 0u) | (2 * i + 1 < have ? (uint32_t)q[2 * i + 1] << 16 : 0u);
    }
    template <class P>  // (bit_cast of a vector element's own expression reads element 0: through a value)
    __device__ __forceinline__ P pair(int i, int j) const {
        const uint32_t w = v[i][j];
        return __builtin_bit_cast(P, w);
    }
    __device__ __forceinline__ uint32_t top16() const {
        u16x2 m = {0, 0};
#pragma unroll
        for (int i = 0; i < N / 2; i++)
            m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, v[i / 4][i % 4] & 0x7fff7fffu));
        return m[0] > m[1] ? m[0] : m[1];
    }
};
template <int N>
struct MxVals<_Float16, N> : MxVals16<_Float16, N> {
    __device__ __forceinline__ uint32_t top() const {
        return __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)this->top16()));
    }
    __device__ __forceinline__ uint32_t codes8(int i, float s) const {
        uint32_t c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, this->template pair<half2v>(i, 0), s, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, this->template pair<half2v>(i, 1), s, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, this->template pair<half2v>(i, 2), s, 2);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, this->template pair<half2v>(i, 3), s, 3);
    }
};
template <int N>
struct MxVals<__bf16, N> : MxVals16<__bf16, N> {
    __device__ __forceinline__ uint32_t top() const { return this->top16() << 16; }
    __device__ __forceinline__ uint32_t codes8(int i, float s) const {
        uint32_t c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, this->template pair<bf2v>(i, 0), s, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, this->template pair<bf2v>(i, 1), s, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, this->template pair<bf2v>(i, 2), s, 2);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, this->template pair<bf2v>(i, 3), s, 3);
    }
};

__device__ __forceinline__ uint32_t quad_umax(uint32_t v) {  // over the four lanes of a quad
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
}

// Eight neighbours are a unit: n = rows * cols / 8 of them, row by row. The place of unit i in rows of stride ld: dense rows need no
// row number, others a 32-bit division (64-bit ones took a third of the kernels' time)
template <bool DENSE>
__device__ __forceinline__ size_t mx_place(size_t i, size_t n, uint32_t per_row, size_t ld) {
    if constexpr (DENSE) return i * 8;
    const size_t r = n >> 32 ? i / per_row : (uint32_t)i / per_row;
    return r * ld + (i - r * per_row) * 8;
}
// workgroups of 256 for n units, one each
inline unsigned mx_grid(size_t n) { return (unsigned)std::min<size_t>((n + 255) / 256, (size_t)cu_count() * 32); }
// 16-byte loads of the rows
inline bool rows16(const void* p, size_t ld, DT dt, int rows) {
    return ((uintptr_t)p & 15) == 0 && (rows == 1 || ld * (dt == DT::F32 ? 4 : 2) % 16 == 0);
}

// the 32 codes of a whole block in one lane, and its scale byte
template <class E>
__device__ __forceinline__ u32x4 mx_block(const MxVals<E, MXB>& x, uint32_t& scale) {
    scale = mx_scale(x.top());
    const float s = mx_scale_f32(scale);
    u32x4 c;
#pragma unroll
    for (int i = 0; i < 4; i++) c[i] = scale == 255 ? 0u : x.codes8(i, s);
    return c;
}

}  // namespace kiln
