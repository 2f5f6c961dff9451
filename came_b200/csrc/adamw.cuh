// Device helpers of the AdamW step and of the gradient norm.
#pragma once

#include "common.cuh"

namespace came {

// ------------------------------------------------------------------------------------------
// 8 consecutive elements <-> fp32 registers.  fp32: one 32-byte access; 16-bit types: one of 16 bytes.
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ void load8(const float* p, float* v) {
    asm volatile("ld.global.L1::no_allocate.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "l"(p) : "memory");
}
__device__ __forceinline__ uint4 load16(const void* p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p) : "memory");
    return r;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float* v) { unpack_bf16x8(load16(p), v); }
__device__ __forceinline__ void load8(const __half* p, float* v) { unpack_f16x8(load16(p), v); }
__device__ __forceinline__ void store8(float* p, const float* v) {
    asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]),
                 "f"(v[5]), "f"(v[6]), "f"(v[7])
                 : "memory");
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float* v) { store_run<8>(p, v); }
__device__ __forceinline__ void store8(__half* p, const float* v) { store_run<8>(p, v); }

__device__ __forceinline__ float approx_sqrt(float x) {
    float y;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ------------------------------------------------------------------------------------------
// random bits: C. Wellons' 32-bit mixer "lowbias32" (two multiplications, three xor-shifts)
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t mix32(uint32_t x) {
    x ^= x >> 16;
    x *= 0x7feb352du;
    x ^= x >> 15;
    x *= 0x846ca68bu;
    return x ^ (x >> 16);
}

// ------------------------------------------------------------------------------------------
// float8 codes
// ------------------------------------------------------------------------------------------
// e8m0 byte of the scale for a block whose largest magnitude has these fp32 bits: 2^(exponent - TOP), at least 2^-126
template <int TOP>
__device__ __forceinline__ uint32_t e8m0_scale(uint32_t top_bits) { return (uint32_t)max((int)(top_bits >> 23) - TOP, 1); }
__device__ __forceinline__ float e8m0_value(uint32_t byte) { return __uint_as_float(byte ? byte << 23 : 0x00400000u); }      // (byte 0 is 2^-127)
__device__ __forceinline__ float e8m0_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }      // (byte in [1, 248])

// stochastic rounding: r < 2^BITS is added to the mantissa below the bits that stay, the rest is cut off
template <int BITS>
__device__ __forceinline__ float dither(float y, uint32_t r) { return __uint_as_float((__float_as_uint(y) + r) & ~((1u << BITS) - 1u)); }

__device__ __forceinline__ void half2_floats(uint32_t w, float* v) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    v[0] = f.x;
    v[1] = f.y;
}
__device__ __forceinline__ void e4m3_decode8(const uint2& c, float* v) {
    const uint32_t w[2] = {c.x, c.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t h;
        const uint16_t two = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(two));
        half2_floats(h, v + 2 * i);
    }
}
// e5m2 is the upper byte of fp16
__device__ __forceinline__ void e5m2_decode8(const uint2& c, float* v) {
    half2_floats(__byte_perm(c.x, 0u, 0x1404u), v);
    half2_floats(__byte_perm(c.x, 0u, 0x3424u), v + 2);
    half2_floats(__byte_perm(c.y, 0u, 0x1404u), v + 4);
    half2_floats(__byte_perm(c.y, 0u, 0x3424u), v + 6);
}
__device__ __forceinline__ uint32_t e4m3_encode4(const float* v) {
    uint16_t a, b;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(a) : "f"(v[1]), "f"(v[0]));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(b) : "f"(v[3]), "f"(v[2]));
    return (uint32_t)a | ((uint32_t)b << 16);
}
__device__ __forceinline__ uint32_t e5m2_encode4(const float* v) {
    uint16_t a, b;
    asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(a) : "f"(v[1]), "f"(v[0]));
    asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(b) : "f"(v[3]), "f"(v[2]));
    return (uint32_t)a | ((uint32_t)b << 16);
}
__device__ __forceinline__ uint2 e4m3_encode8(const float* v) { return make_uint2(e4m3_encode4(v), e4m3_encode4(v + 4)); }
__device__ __forceinline__ uint2 e5m2_encode8(const float* v) { return make_uint2(e5m2_encode4(v), e5m2_encode4(v + 4)); }

// ------------------------------------------------------------------------------------------
// gradient norm: sums of squares per CTA in 64 bits, added in a fixed order by every CTA that needs the total
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// all threads call; the same value in every thread.  red: one double per warp
__device__ __forceinline__ double block_sum64(double v, double* red) {
    v = warp_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = 0.0;
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) t += red[w];
    return t;
}
__device__ __forceinline__ double norm_of_partials(const double* parts, int n, double* red) {
    double t = 0.0;
    for (int i = threadIdx.x; i < n; i += blockDim.x) t += __ldcg(parts + i);
    return sqrt(block_sum64(t, red));
}
__device__ __forceinline__ double clip_coefficient(double norm, float max_norm) {
    const double c = (double)max_norm / (norm + 1e-6);
    return c > 1.0 ? 1.0 : c;      // (NaN stays)
}

}  // namespace came
