// The residual's addition and the RMS norm of the sum in one pass (kiln_add_rmsnorm): h = x + res, y = h / sqrt(mean(h^2) + eps) w, y in
// fp32, 16 bits or as MXFP8 codes and scales (mxfp8.hpp). Every value is read once and kept in registers, as fp32, between the sum of
// squares and its use; the norm takes the sum before it is rounded to the residual's type.
//
// A row to a wave up to 2048 columns, to 4, 8 or 16 waves beyond: eight neighbours a lane and chunk, at most four chunks a lane, all loads
// under way before the first is used. Bound by memory: 6912 x 2048, bf16 x on a fp32 residual to MXFP8, 25.1 us (6.2 TB/s of what is read and
// written); 4096 columns, all bf16, 33.4 (6.8); 2000 x 32768, sixteen waves a row that meet at two barriers, 101 (5.2). One row of 2048: 3.3, a
// launch and one round trip.
#include <hip/hip_runtime.h>

#include "mxfp8.hpp"

namespace kiln {

struct RmsParams {
    void* y;
    uint8_t* scales;  // not null: y holds MXFP8 codes
    void* h;
    const void* x;
    const void* res;
    const uint16_t* w;
    size_t ldy, ldh, ldx, ldr;
    int rows, dim;
    float eps;
    DT ydt, xdt, rdt;
};

// Eight elements of 2 or 4 bytes as they lie, and as fp32
template <int BYTES, bool VEC>
struct Raw8 {
    u32x4 w[BYTES / 2];
    __device__ __forceinline__ void load(const void* base, size_t at, int have) {
        const uint8_t* p = static_cast<const uint8_t*>(base) + at * BYTES;
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < BYTES / 2; i++) w[i] = have > 0 ? reinterpret_cast<const u32x4*>(p)[i] : u32x4{0, 0, 0, 0};
        } else if constexpr (BYTES == 4) {
#pragma unroll
            for (int i = 0; i < 8; i++) w[i / 4][i % 4] = i < have ? reinterpret_cast<const uint32_t*>(p)[i] : 0u;
        } else {
            const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
            for (int i = 0; i < 4; i++) w[0][i] = (2 * i < have ? q[2 * i] : 0u) | (2 * i + 1 < have ? (uint32_t)q[2 * i + 1] << 16 : 0u);
        }
    }
    __device__ __forceinline__ void get(DT dt, float (&v)[8]) const {
        if constexpr (BYTES == 4) {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = __uint_as_float(w[i / 4][i % 4]);
        } else if (dt == DT::F16) {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[0][i / 2] >> (16 * (i & 1))));
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = __uint_as_float(i & 1 ? w[0][i / 2] & 0xffff0000u : w[0][i / 2] << 16);
        }
    }
};
template <bool VEC>
__device__ __forceinline__ void rms_store(void* base, DT dt, size_t at, int have, const float (&v)[8]) {
    if (dt == DT::F32) store8f<VEC>(static_cast<float*>(base) + at, have, v);
    else if (dt == DT::F16) store8f<VEC>(static_cast<_Float16*>(base) + at, have, v);
    else store8f<VEC>(static_cast<__bf16*>(base) + at, have, v);
}

// WAVES waves to a row, CH chunks of eight a lane; XB and RB: bytes of x's and the residual's elements (RB 0: none)
template <int XB, int RB, int WAVES, int CH, bool VEC>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void k_add_rmsnorm(const RmsParams p) {
    __shared__ float red[2][WAVES];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const size_t row = WAVES == 1 ? (size_t)blockIdx.x * 4 + wv : blockIdx.x;
    if (row >= (size_t)p.rows) return;  // (a wave of its own, or the whole workgroup)
    const int col0 = (WAVES == 1 ? lane : (int)threadIdx.x) * 8;
    auto have = [&](int c) { return p.dim - (col0 + c * WAVES * 512); };
    Raw8<XB, VEC> x[CH];
    Raw8<RB ? RB : 2, VEC> r[CH];
    Raw8<2, VEC> w[CH];
#pragma unroll
    for (int c = 0; c < CH; c++) x[c].load(p.x, row * p.ldx + col0 + c * WAVES * 512, have(c));
    if constexpr (RB != 0)
#pragma unroll
        for (int c = 0; c < CH; c++) r[c].load(p.res, row * p.ldr + col0 + c * WAVES * 512, have(c));
    if (p.w)
#pragma unroll
        for (int c = 0; c < CH; c++) w[c].load(p.w, col0 + c * WAVES * 512, have(c));
    float f[CH][8], ss = 0.f;
#pragma unroll
    for (int c = 0; c < CH; c++) {
        x[c].get(p.xdt, f[c]);
        if constexpr (RB != 0) {
            float t[8];
            r[c].get(p.rdt, t);
#pragma unroll
            for (int i = 0; i < 8; i++) f[c][i] += t[i];
            if (have(c) > 0) rms_store<VEC>(p.h, p.rdt, row * p.ldh + col0 + c * WAVES * 512, have(c), f[c]);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) ss = fmaf(f[c][i], f[c][i], ss);
    }
    auto all = [&](float v, int at) {  // over the row's lanes
        v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x121, 0xF, 0xF, false));
        v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x122, 0xF, 0xF, false));
        v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x124, 0xF, 0xF, false));
        v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x128, 0xF, 0xF, false));
        v = quad_sum(v);
        if constexpr (WAVES > 1) {
            if (lane == 0) red[at][wv] = v;
            __syncthreads();
            v = red[at][0];
#pragma unroll
            for (int i = 1; i < WAVES; i++) v += red[at][i];
        } else {  // the lanes add in different orders: one's sum for all, which then take the same branches
            v = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v)));
        }
        return v;
    };
    ss = all(ss, 0);
    float rs = 1.f / sqrtf(ss / (float)p.dim + p.eps);
    // Squares beyond fp32, or below its normal range where eps does not exceed them: of the row times a power of two (rows with infinities and
    // NaNs come here too, and keep them)
    constexpr float LITTLE = 0x1p-100f;
    if (!(ss < INFINITY) || (p.eps < LITTLE && ss < LITTLE)) {
        const bool big = !(ss < LITTLE);
        const float k = big ? 0x1p-80f : 0x1p80f;
        float s2 = 0.f;
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float v = f[c][i] * k;
                s2 = fmaf(v, v, s2);
            }
        s2 = all(s2, 1);
        rs = 1.f / sqrtf(s2 / (float)p.dim + p.eps * k * k);
        // in this order small values do not pass through subnormal ones
        const float a = big ? rs : k, b = big ? k : rs;
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) f[c][i] = f[c][i] * a * b;
        rs = 1.f;
    }
#pragma unroll
    for (int c = 0; c < CH; c++) {
        float t[8];
        if (p.w) w[c].get(DT::BF16, t);
        else
#pragma unroll
            for (int i = 0; i < 8; i++) t[i] = 1.f;
#pragma unroll
        for (int i = 0; i < 8; i++) t[i] *= f[c][i] * rs;
        if (p.scales) {  // dim % 32 == 0: a quad's lanes are all inside or all outside
            uint32_t s;
            const u32x2 codes = mx8_quad(t, s);
            if (have(c) <= 0) continue;
            const size_t at = row * p.dim + col0 + c * WAVES * 512;
            *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(p.y) + at) = codes;
            if ((lane & 3) == 0) p.scales[at >> 5] = (uint8_t)s;
        } else if (have(c) > 0) {
            rms_store<VEC>(p.y, p.ydt, row * p.ldy + col0 + c * WAVES * 512, have(c), t);
        }
    }
}

template <int XB, int RB, int WAVES, int CH>
static hipError_t rms_launch(const RmsParams& p, bool vec, hipStream_t s) {
    const size_t wgs = WAVES == 1 ? ((size_t)p.rows + 3) / 4 : (size_t)p.rows;
    if (hipError_t e = grid_check(wgs, WAVES == 1 ? 256 : 64 * WAVES)) return e;
    auto kern = vec ? k_add_rmsnorm<XB, RB, WAVES, CH, true> : k_add_rmsnorm<XB, RB, WAVES, CH, false>;
    hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(WAVES == 1 ? 256 : 64 * WAVES), 0, s, p);
    return hipGetLastError();
}
template <int XB, int RB>
static hipError_t rms_of(const RmsParams& p, bool vec, hipStream_t s) {
    if (p.dim <= 512) return rms_launch<XB, RB, 1, 1>(p, vec, s);
    if (p.dim <= 1024) return rms_launch<XB, RB, 1, 2>(p, vec, s);
    if (p.dim <= 2048) return rms_launch<XB, RB, 1, 4>(p, vec, s);
    if (p.dim <= 4096) return rms_launch<XB, RB, 4, 2>(p, vec, s);
    if (p.dim <= 8192) return rms_launch<XB, RB, 4, 4>(p, vec, s);
    if (p.dim <= 16384) return rms_launch<XB, RB, 8, 4>(p, vec, s);
    return rms_launch<XB, RB, 16, 4>(p, vec, s);
}

hipError_t launch_add_rmsnorm(const RmsLaunch& c, hipStream_t s) {
    RmsParams p{c.y, c.scales, c.h, c.x, c.res, c.w, c.ldy, c.ldh, c.ldx, c.ldr, c.rows, c.dim, c.eps, c.ydt, c.xdt, c.rdt};
    // 16-byte pieces of eight elements
    const bool vec = c.dim % 8 == 0 && rows16(c.x, c.ldx, c.xdt, c.rows) && (!c.w || ((uintptr_t)c.w & 15) == 0) &&
                     (c.scales || rows16(c.y, c.ldy, c.ydt, c.rows)) &&
                     (!c.res || (rows16(c.res, c.ldr, c.rdt, c.rows) && rows16(c.h, c.ldh, c.rdt, c.rows)));
    const int rb = !c.res ? 0 : c.rdt == DT::F32 ? 4 : 2;
    if (c.xdt == DT::F32) return rb == 0 ? rms_of<4, 0>(p, vec, s) : rb == 2 ? rms_of<4, 2>(p, vec, s) : rms_of<4, 4>(p, vec, s);
    return rb == 0 ? rms_of<2, 0>(p, vec, s) : rb == 2 ? rms_of<2, 2>(p, vec, s) : rms_of<2, 4>(p, vec, s);
}

}  // namespace kiln
