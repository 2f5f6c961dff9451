// Device helpers of the AdamW step and of the gradient norm.
#pragma once

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "launch.h"

namespace came {

constexpr int ADAMW_THREADS = 256, ADAMW_WARPS = ADAMW_THREADS / 32;

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
// the same for arguments and results that are normal numbers (others become zero)
__device__ __forceinline__ float fast_sqrt(float x) {
    float y;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float fast_rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {      // (a NaN does not count)
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
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

// two codes of a word of four (the lower or the upper two) to fp32
__device__ __forceinline__ float2 e4m3_pair(uint32_t w, int upper) {
    uint32_t h;
    const uint16_t two = (uint16_t)(upper ? w >> 16 : w);
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(two));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ float2 e5m2_pair(uint32_t w, int upper) {      // (e5m2 is the upper byte of fp16)
    const uint32_t h = __byte_perm(w, 0u, upper ? 0x3424u : 0x1404u);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

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

// ------------------------------------------------------------------------------------------
// what a warp needs of a tensor's step count and hyper-parameters
// ------------------------------------------------------------------------------------------
// What a tensor's step count and hyper-parameters make of the formulas
struct AdamwCoef {
    float c, b1, om1, b2, om2, size, root, eps, wd_lr;
    uint32_t key;
};

// The same for a warp's tensors as long as count and group stay the same
struct AdamwCache {
    float step;
    int group;
    AdamwCoef k;
};

// 1 - beta^t, from ln beta as a sum of two fp32 numbers  (out of line: rare, and long)
static __device__ __noinline__ double one_minus_power(float ln_hi, float ln_lo, double t) { return -expm1(t * ((double)ln_hi + (double)ln_lo)); }

// (all lanes of a warp)
__device__ __forceinline__ void adamw_coef(AdamwCache& cache, const CameTensorDesc& d, const CameHyper* hyp, bool clipped, double norm) {
    const float step = *static_cast<const float*>(d.res_row);
    if (step == cache.step && d.group == cache.group) return;      // (the same in every lane)
    const CameHyper& h = hyp[d.group];
    const double t = (double)step + 1.0;
    // even lanes: lr / (1 - b1^t); odd lanes: 1 / sqrt(1 - b2^t)
    const bool odd = threadIdx.x & 1;
    const double rest = one_minus_power(odd ? h.om_beta3 : h.beta3, odd ? h.reserved[1] : h.reserved[0], t);
    const float f = (float)(odd ? 1.0 / sqrt(rest) : (double)h.lr / rest);
    cache.step = step;
    cache.group = d.group;
    AdamwCoef& k = cache.k;
    k.size = __shfl_sync(0xffffffffu, f, 0);
    k.root = __shfl_sync(0xffffffffu, f, 1);
    k.c = clipped ? (float)((double)h.grad_scale * clip_coefficient(norm, h.clip_threshold)) : h.grad_scale;
    k.b1 = h.beta1; k.om1 = h.om_beta1;
    k.b2 = h.beta2; k.om2 = h.om_beta2;
    k.eps = h.eps0; k.wd_lr = h.wd_lr;
    k.key = mix32((uint32_t)t);
}

// The end of a CTA: the last one raises the step counts of the launch's tensors.  Every warp of every CTA has read the counts it
// needs by then.
__device__ __forceinline__ void adamw_count_step(const AdamwArgs& w) {
    __shared__ bool last;
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(w.ticket, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    for (int i = threadIdx.x; i < w.n_tensors; i += ADAMW_THREADS) atomicAdd(w.steps[i], 1.0f);      // (one address each: nothing to wait for)
    if (threadIdx.x == 0) *w.ticket = 0u;
}
// Launches that may begin while the one before them on the stream ends: after griddep_launch() of all its CTAs, which comes when a
// CTA has no more runs (earlier, the waiting CTAs would spread unevenly over the SMs: 1 % of a large step).  It is the end of
// that launch that griddep_wait() waits for; nothing in memory is touched before.
__device__ __forceinline__ void griddep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void griddep_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <typename... P, typename... A>
static cudaError_t launch_behind(void (*kernel)(P...), int grid, int threads, int smem, cudaStream_t st, const A&... args) {
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3((unsigned)grid);
    c.blockDim = dim3((unsigned)threads);
    c.dynamicSmemBytes = (size_t)smem;
    c.stream = st;
    c.attrs = &early;
    c.numAttrs = 1;
    static_assert((std::is_same_v<P, A> && ...), "the arguments are passed by their addresses");
    void* at[] = {const_cast<void*>(static_cast<const void*>(&args))...};      // (no copy of tables of 20 KB on the way)
    return cudaLaunchKernelExC(&c, reinterpret_cast<const void*>(kernel), at);
}
// The beginning: the norm of all gradients.  False: it is not finite, and the step does not take place.
__device__ __forceinline__ bool adamw_norm(const AdamwArgs& w, double* norm) {
    __shared__ double red[ADAMW_THREADS / 32];
    *norm = 0.0;
    if (!w.norm_parts) return true;
    *norm = norm_of_partials(w.norm_parts, w.n_parts, red);
    if (blockIdx.x == 0 && threadIdx.x == 0) *w.norm_out = (float)*norm;
    return isfinite(*norm);
}

// A CTA takes spans of w.span consecutive items, one of every gridDim.x; items of a span that lie in one tensor are one run of
// elements [lo, hi) of its n.
template <typename F>
__device__ __forceinline__ void for_runs(const StepArgs& a, const AdamwArgs& w, F f) {
    for (int64_t from = (int64_t)blockIdx.x * w.span; from < w.n; from += (int64_t)gridDim.x * w.span) {
        const int end = (int)min((int64_t)w.n, from + w.span);
        for (int item = (int)from; item < end;) {
            const Work wk = w.work[item];
            const CameTensorDesc& d = a.descs[wk.tensor];
            const int64_t n = d.rows * (d.cols ? d.cols : 1) * (d.batch > 1 ? (int64_t)d.batch : 1);
            const int64_t lo = (int64_t)wk.tile * ADAMW_ITEM, hi = min(lo + (int64_t)(end - item) * ADAMW_ITEM, n);
            item += (int)((hi - lo + ADAMW_ITEM - 1) / ADAMW_ITEM);
            f(d, wk.tensor, lo, hi, n);
        }
    }
}
// Host side: the span and the grid.  Every CTA (per_sm on each SM) has the same number of spans, of `most` items at most: a span
// in one piece spares the next run's set-up, but the shorter they are, the closer together lie the addresses that the GPU
// works on at a time.
static inline int adamw_spans(AdamwArgs& w, int per_sm, int most) {
    const int64_t ctas = (int64_t)persistent_grid_limit() * per_sm, rounds = (w.n + ctas * most - 1) / (ctas * most);
    w.span = (int)((w.n + ctas * rounds - 1) / (ctas * rounds));
    return (int)std::min(ctas, ((int64_t)w.n + w.span - 1) / w.span);
}

// host side: pick the instance for a launch's types
template <template <typename, typename> class Launch, typename P, typename... A>
static cudaError_t adamw_for_g(int g_dtype, const A&... args) {
    if (g_dtype == CAME_DT_F32) return Launch<P, float>::run(args...);
    if (g_dtype == CAME_DT_F16) return Launch<P, __half>::run(args...);
    return Launch<P, __nv_bfloat16>::run(args...);
}
template <template <typename, typename> class Launch, typename... A>
static cudaError_t adamw_for(const KernelKey& key, const A&... args) {
    if (key.p_dtype == CAME_DT_F32) return adamw_for_g<Launch, float>(key.g_dtype, args...);
    if (key.p_dtype == CAME_DT_F16) return adamw_for_g<Launch, __half>(key.g_dtype, args...);
    return adamw_for_g<Launch, __nv_bfloat16>(key.g_dtype, args...);
}
static AdamwHyp adamw_hyp(const CameHyper* host_hyp, int n_hyp) {
    AdamwHyp h{};
    if (host_hyp)
        for (int i = 0; i < n_hyp && i < ADAMW_MAX_HYP; ++i) h.h[i] = host_hyp[i];
    return h;
}

}  // namespace came
