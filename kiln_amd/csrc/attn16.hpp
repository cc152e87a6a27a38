// Pieces shared by the attention kernels that read K and V where they lie (cross_attn.hip, prompt_attn.hip): the matrix products of both
// 16-bit types, the permutation of a key tile's rows in LDS, the softmax's constants.
#pragma once
#include <hip/hip_runtime.h>

#include "common.hpp"

namespace kiln {

constexpr int XKT = 32;       // keys of a tile
constexpr float XRESCALE = 8.f, XLIFT16 = 7.f;  // log2: the maximum's slack, the factor of fp16 weights
constexpr float XFAR = 1 << 20;                 // log2: a maximum from which scores are rounded on their own

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
// Position of 16-byte chunk c of key row r in its LDS row. K is read 16 keys x one chunk at a time, V eight keys x a pair of
// chunks: either way 256 bytes that lie in all 64 banks, for rows of 256 bytes (Dh 128) and of 128. The permutation is on the
// side of the copies' sources, where it costs nothing (rows in order and padded blocks instead: the same time, more conflicts).
template <int DH>
__device__ __forceinline__ int k_swz(int c, int r) {
    return DH == 128 ? c ^ (r & 15) : c ^ ((r >> 1) & 7);
}
template <int DH>
__device__ __forceinline__ int v_swz(int c, int r) {
    return DH == 128 ? c ^ ((r & 7) << 1) : c ^ (((r >> 1) & 3) << 1);
}

}  // namespace kiln
