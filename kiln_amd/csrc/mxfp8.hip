// MXFP8 quantisation and its inverse (mxfp8.hpp). Eight neighbours are a lane's unit, four lanes a block. Bound by memory: 6912 x 2048 fp16 either
// way 8.0 us (5.4 TB/s), x 8192 25.3 and 25.9 (6.7); 77 x 1024 2.3, a launch.
#include <hip/hip_runtime.h>

#include "mxfp8.hpp"

namespace kiln {

// x [rows, cols] to codes [rows, cols] and scales [rows, cols / 32]
template <class E, bool VEC, bool DENSE>
__global__ __launch_bounds__(256) void k_mx8_quantize(uint8_t* codes, uint8_t* scales, const E* x, size_t ldx, size_t n, uint32_t per_row) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        float v[8];
        load8f<VEC>(x + mx_place<DENSE>(i, n, per_row, ldx), 8, v);
        uint32_t s;
        *reinterpret_cast<u32x2*>(codes + i * 8) = mx8_quad(v, s);
        if ((threadIdx.x & 3) == 0) scales[i >> 2] = (uint8_t)s;
    }
}

// Codes times their scale, exact in fp32 (an e4m3 value has four bits, 2^-136 is the smallest product); other types round once.
template <class E, bool VEC, bool DENSE>
__global__ __launch_bounds__(256) void k_mx8_dequantize(E* y, size_t ldy, const uint8_t* codes, const uint8_t* scales, size_t n,
                                                        uint32_t per_row) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const u32x2 c = *reinterpret_cast<const u32x2*>(codes + i * 8);
        const uint32_t s = scales[i >> 2];
        const float sc = mx_scale_f32(s);
        float v[8];
#pragma unroll
        for (int w = 0; w < 2; w++) {
            const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[w], sc, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[w], sc, true);
            v[4 * w] = a[0];
            v[4 * w + 1] = a[1];
            v[4 * w + 2] = b[0];
            v[4 * w + 3] = b[1];
        }
        if (s == 255)
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = __uint_as_float(0x7fc00000u);
        store8f<VEC>(y + mx_place<DENSE>(i, n, per_row, ldy), 8, v);
    }
}

template <class E>
static hipError_t quantize8_of(uint8_t* codes, uint8_t* scales, const void* x, size_t ldx, int rows, int cols, bool vec, hipStream_t s) {
    const size_t n = (size_t)rows * (cols / 8);
    const bool dense = rows == 1 || ldx == (size_t)cols;
    auto kern = vec ? (dense ? k_mx8_quantize<E, true, true> : k_mx8_quantize<E, true, false>)
                    : (dense ? k_mx8_quantize<E, false, true> : k_mx8_quantize<E, false, false>);
    hipLaunchKernelGGL(kern, dim3(mx_grid(n)), dim3(256), 0, s, codes, scales, static_cast<const E*>(x), ldx, n, (uint32_t)(cols / 8));
    return hipGetLastError();
}
template <class E>
static hipError_t dequantize8_of(void* y, size_t ldy, const uint8_t* codes, const uint8_t* scales, int rows, int cols, bool vec, hipStream_t s) {
    const size_t n = (size_t)rows * (cols / 8);
    const bool dense = rows == 1 || ldy == (size_t)cols;
    auto kern = vec ? (dense ? k_mx8_dequantize<E, true, true> : k_mx8_dequantize<E, true, false>)
                    : (dense ? k_mx8_dequantize<E, false, true> : k_mx8_dequantize<E, false, false>);
    hipLaunchKernelGGL(kern, dim3(mx_grid(n)), dim3(256), 0, s, static_cast<E*>(y), ldy, codes, scales, n, (uint32_t)(cols / 8));
    return hipGetLastError();
}

hipError_t launch_mx8_quantize(uint8_t* codes, uint8_t* scales, const void* x, DT dt, size_t ldx, int rows, int cols, hipStream_t s) {
    const bool vec = rows16(x, ldx, dt, rows);
    if (dt == DT::F32) return quantize8_of<float>(codes, scales, x, ldx, rows, cols, vec, s);
    if (dt == DT::F16) return quantize8_of<_Float16>(codes, scales, x, ldx, rows, cols, vec, s);
    return quantize8_of<__bf16>(codes, scales, x, ldx, rows, cols, vec, s);
}
hipError_t launch_mx8_dequantize(void* y, DT dt, size_t ldy, const uint8_t* codes, const uint8_t* scales, int rows, int cols, hipStream_t s) {
    const bool vec = rows16(y, ldy, dt, rows);
    if (dt == DT::F32) return dequantize8_of<float>(y, ldy, codes, scales, rows, cols, vec, s);
    if (dt == DT::F16) return dequantize8_of<_Float16>(y, ldy, codes, scales, rows, cols, vec, s);
    return dequantize8_of<__bf16>(y, ldy, codes, scales, rows, cols, vec, s);
}

}  // namespace kiln
