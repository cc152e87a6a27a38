// MXFP4 quantisation, its inverse, and the operand layout of the MXFP4 product (mxfp4.hpp). All bound by memory:
// 8192 x 2048 bf16 to codes 8.4 us, back 8.3 (5.0 and 5.1 TB/s); 6912 x 2048 fp16 to the operand layout 6.9 (5.2).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "mxfp4.hpp"

namespace kiln {

// x [rows, cols] to codes [rows, cols / 2] (even column in the low half) and scales [rows, cols / 32]. Four lanes take a
// block of 32, eight values each: loads of 16 or 32 contiguous bytes per lane, 4-byte stores of codes.
template <class E, bool VEC, bool DENSE>
__global__ __launch_bounds__(256) void k_mx_quantize(uint8_t* codes, uint8_t* scales, const E* x, size_t ldx, size_t n, uint32_t per_row) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const E* src = x + mx_place<DENSE>(i, n, per_row, ldx);
        MxVals<E, 8> v;
        if constexpr (VEC) v.load(src);
        else v.load_any(src, 8);
        const uint32_t s = mx_scale(quad_umax(v.top()));
        *reinterpret_cast<uint32_t*>(codes + i * 4) = s == 255 ? 0u : v.codes8(0, mx_scale_f32(s));
        if ((threadIdx.x & 3) == 0) scales[i >> 2] = (uint8_t)s;
    }
}

// The eight values of a code word times the scale, by the conversion instructions: exact in fp32 and bf16 (fp16 rounds outside
// its range). The scale NaN is put in by hand.
template <class E>
__device__ __forceinline__ void mx_values8(uint32_t c, uint32_t s, E (&o)[8]) {
    const float sc = mx_scale_f32(s);
    auto two = [&](auto pair, int i) {
        const bool nan = s == 255;
        o[2 * i] = nan ? (E)__uint_as_float(0x7fc00000u) : (E)pair[0];
        o[2 * i + 1] = nan ? (E)__uint_as_float(0x7fc00000u) : (E)pair[1];
    };
    if constexpr (sizeof(E) == 4) {
        two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, sc, 0), 0);
        two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, sc, 1), 1);
        two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, sc, 2), 2);
        two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, sc, 3), 3);
    } else if constexpr (std::is_same<E, _Float16>::value) {
        two(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, sc, 0), 0);
        two(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, sc, 1), 1);
        two(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, sc, 2), 2);
        two(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, sc, 3), 3);
    } else {
        two(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 0), 0);
        two(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 1), 1);
        two(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 2), 2);
        two(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 3), 3);
    }
}
template <class E, bool VEC, bool DENSE>
__global__ __launch_bounds__(256) void k_mx_dequantize(E* y, size_t ldy, const uint8_t* codes, const uint8_t* scales, size_t n,
                                                       uint32_t per_row) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        E o[8];
        mx_values8(*reinterpret_cast<const uint32_t*>(codes + i * 4), scales[i >> 2], o);
        E* dst = y + mx_place<DENSE>(i, n, per_row, ldy);
        if constexpr (VEC) {
            typedef E V __attribute__((ext_vector_type(16 / sizeof(E))));
#pragma unroll
            for (int j = 0; j < 8; j += 16 / (int)sizeof(E)) {
                V v;
#pragma unroll
                for (int e = 0; e < 16 / (int)sizeof(E); e++) v[e] = o[j + e];
                *reinterpret_cast<V*>(dst + j) = v;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) dst[j] = o[j];
        }
    }
}

// codes and scales (row-major) to the operand layout, one wave per (64 rows, k block of 128); the padding is written too
__global__ __launch_bounds__(256) void k_mx_pack(uint8_t* oc, uint8_t* os, const uint8_t* codes, const uint8_t* scales, int rows,
                                                 int cols, size_t units) {
    const size_t u = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (u >= units) return;
    const size_t rgs = mx_rg(rows), rg = u % rgs, kb = u / rgs;
    const int lane = threadIdx.x & 63, k = (int)kb * 128 + 32 * (lane >> 4);
    uint32_t sc = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const size_t r = rg * 64 + 16 * j + (lane & 15);
        u32x4 c = {0, 0, 0, 0};
        if (r < (size_t)rows && k < cols) {
            c = *reinterpret_cast<const u32x4*>(codes + r * (cols / 2) + k / 2);
            sc |= (uint32_t)scales[r * (cols / 32) + k / 32] << (8 * j);
        }
        *reinterpret_cast<u32x4*>(oc + ((kb * rgs + rg) * 4 + j) * MX_UNIT + lane * 16) = c;
    }
    *reinterpret_cast<uint32_t*>(os + (kb * rgs + rg) * MX_SUNIT + lane * 4) = sc;
}

// The rows of an activation straight to the operand layout: a workgroup takes 64 rows x 128 columns (four units of codes, one
// of scales). Four lanes share a block, so a load covers 256-byte pieces (fp16) of four rows, four loads in flight; the codes
// meet in LDS and leave as whole units. (A lane per block reads the same lines four times over: 6912 x 2048 fp16 10.7 us.)
template <class E, bool VEC>
__global__ __launch_bounds__(256) void k_mx_quantize_pack(uint8_t* oc, uint8_t* os, const E* x, size_t ldx, int rows, int cols, int kbs) {
    __shared__ __attribute__((aligned(16))) uint32_t lc[4][64][4];  // [row block][operand lane][8 codes]
    __shared__ __attribute__((aligned(16))) uint8_t ls[64][4];                                   // [operand lane][row block]
    const size_t rgs = mx_rg(rows), rg = blockIdx.x / kbs, kb = blockIdx.x % kbs;
    const int q = threadIdx.x & 15, k = (int)kb * 128 + 8 * q;
    MxVals<E, 8> v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const size_t r = rg * 64 + 16 * j + (threadIdx.x >> 4);
        const bool in = r < (size_t)rows && k < cols;
        const E* src = x + (in ? r * ldx + k : 0);
        if constexpr (VEC) v[j].load(src);
        else v[j].load_any(src, in ? 8 : 0);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int rl = threadIdx.x >> 4, lane = rl + 16 * (q >> 2);
        const bool in = rg * 64 + 16 * j + rl < (size_t)rows && k < cols;
        const uint32_t s = mx_scale(quad_umax(v[j].top()));
        lc[j][lane][q & 3] = in && s != 255 ? v[j].codes8(0, mx_scale_f32(s)) : 0u;
        if ((q & 3) == 0) ls[lane][j] = in ? (uint8_t)s : 0;
    }
    __syncthreads();
    const int j = threadIdx.x >> 6, lane = threadIdx.x & 63;
    *reinterpret_cast<u32x4*>(oc + ((kb * rgs + rg) * 4 + j) * MX_UNIT + lane * 16) = *reinterpret_cast<const u32x4*>(lc[j][lane]);
    if (j == 0) *reinterpret_cast<uint32_t*>(os + (kb * rgs + rg) * MX_SUNIT + lane * 4) = *reinterpret_cast<const uint32_t*>(ls[lane]);
}

template <class E>
static hipError_t quantize_of(uint8_t* codes, uint8_t* scales, const void* x, size_t ldx, int rows, int cols, bool vec, hipStream_t s) {
    const size_t n = (size_t)rows * (cols / 8);
    const bool dense = rows == 1 || ldx == (size_t)cols;
    auto kern = vec ? (dense ? k_mx_quantize<E, true, true> : k_mx_quantize<E, true, false>)
                    : (dense ? k_mx_quantize<E, false, true> : k_mx_quantize<E, false, false>);
    hipLaunchKernelGGL(kern, dim3(mx_grid(n)), dim3(256), 0, s, codes, scales, static_cast<const E*>(x), ldx, n, (uint32_t)(cols / 8));
    return hipGetLastError();
}
template <class E>
static hipError_t dequantize_of(void* y, size_t ldy, const uint8_t* codes, const uint8_t* scales, int rows, int cols, bool vec,
                                hipStream_t s) {
    const size_t n = (size_t)rows * (cols / 8);
    const bool dense = rows == 1 || ldy == (size_t)cols;
    auto kern = vec ? (dense ? k_mx_dequantize<E, true, true> : k_mx_dequantize<E, true, false>)
                    : (dense ? k_mx_dequantize<E, false, true> : k_mx_dequantize<E, false, false>);
    hipLaunchKernelGGL(kern, dim3(mx_grid(n)), dim3(256), 0, s, static_cast<E*>(y), ldy, codes, scales, n, (uint32_t)(cols / 8));
    return hipGetLastError();
}
template <class E>
static hipError_t quantize_pack_of(uint8_t* op, const void* x, size_t ldx, int rows, int cols, bool vec, hipStream_t s) {
    const int kbs = mx_kb(cols);
    const size_t wgs = ((size_t)rows + 63) / 64 * kbs;
    if (hipError_t e = grid_check(wgs, 256)) return e;
    auto kern = vec ? k_mx_quantize_pack<E, true> : k_mx_quantize_pack<E, false>;
    hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(256), 0, s, op, op + mx_code_bytes(rows, cols),
                       static_cast<const E*>(x), ldx, rows, cols, kbs);
    return hipGetLastError();
}
hipError_t launch_mx_quantize(uint8_t* codes, uint8_t* scales, const void* x, DT dt, size_t ldx, int rows, int cols, hipStream_t s) {
    const bool vec = rows16(x, ldx, dt, rows);
    if (dt == DT::F32) return quantize_of<float>(codes, scales, x, ldx, rows, cols, vec, s);
    if (dt == DT::F16) return quantize_of<_Float16>(codes, scales, x, ldx, rows, cols, vec, s);
    return quantize_of<__bf16>(codes, scales, x, ldx, rows, cols, vec, s);
}
hipError_t launch_mx_dequantize(void* y, DT dt, size_t ldy, const uint8_t* codes, const uint8_t* scales, int rows, int cols,
                                hipStream_t s) {
    const bool vec = rows16(y, ldy, dt, rows);
    if (dt == DT::F32) return dequantize_of<float>(y, ldy, codes, scales, rows, cols, vec, s);
    if (dt == DT::F16) return dequantize_of<_Float16>(y, ldy, codes, scales, rows, cols, vec, s);
    return dequantize_of<__bf16>(y, ldy, codes, scales, rows, cols, vec, s);
}
hipError_t launch_mx_pack(uint8_t* op, const uint8_t* codes, const uint8_t* scales, int rows, int cols, hipStream_t s) {
    const size_t units = (size_t)mx_rg(rows) * mx_kb(cols);
    if (hipError_t e = grid_check((units + 3) / 4, 256)) return e;
    hipLaunchKernelGGL(k_mx_pack, dim3((unsigned)((units + 3) / 4)), dim3(256), 0, s, op, op + mx_code_bytes(rows, cols), codes, scales,
                       rows, cols, units);
    return hipGetLastError();
}
hipError_t launch_mx_quantize_pack(uint8_t* op, const void* x, DT dt, size_t ldx, int rows, int cols, hipStream_t s) {
    const bool vec = rows16(x, ldx, dt, rows);
    if (dt == DT::F32) return quantize_pack_of<float>(op, x, ldx, rows, cols, vec, s);
    if (dt == DT::F16) return quantize_pack_of<_Float16>(op, x, ldx, rows, cols, vec, s);
    return quantize_pack_of<__bf16>(op, x, ldx, rows, cols, vec, s);
}

}  // namespace kiln
