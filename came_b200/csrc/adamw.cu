// AdamW over many tensors in one launch: states in fp32, or in float8 with a power-of-two scale per 256 elements.
//
//   m' = b1 m + (1 - b1) c g      v' = b2 v + (1 - b2) (c g)^2      c = grad_scale x clip coefficient
//   p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// t is counted on the device: every CTA reads it, the last one to finish adds 1, so that a captured step counts its own
// replays.  1 - b^t is formed as -expm1(t ln b) in 64 bits (at t = 1, b2 = 0.999 a difference in 32 bits keeps three
// digits), once per CTA and tensor set with the same count.
//
// Float8 states.  m is held as e4m3, v as e5m2 (its root then has the range and the relative step of m), both times a scale
// 2^k (one e8m0 byte) that puts the exponent of the block's largest magnitude at 2^7 resp. 2^14.  A scale that is a power of
// two leaves the grid where it is from step to step, so that only what a state gained is rounded, and it is rounded
// stochastically: a uniform number is added below the last mantissa bit that is kept, the rest is cut off.  Rounded to
// nearest, v would never fall at b2 = 0.999 (a step moves it by 0.1 %, half a spacing is 7 to 12 %).
// The random bits are a hash of the element's index and t: no state, the same in every run.
#include "adamw.cuh"
#include "launch.h"

namespace came {

constexpr int ADAMW_THREADS = 256;

struct AdamwHyp {
    CameHyper h[ADAMW_MAX_HYP];
};

// What a tensor's step count and hyper-parameters make of the formulas
struct AdamwCoef {
    float c, b1, om1, b2, om2, size, root, eps, wd_lr;
    uint32_t key;
};

// The same for a CTA's tensors as long as count and group stay the same
struct AdamwCache {
    float step;
    int group;
    AdamwCoef k;
};
struct AdamwShared {
    float size, root;
};

// 1 - beta^t, from ln beta as a sum of two fp32 numbers  (out of line: rare, and long)
static __device__ __noinline__ double one_minus_power(float ln_hi, float ln_lo, double t) { return -expm1(t * ((double)ln_hi + (double)ln_lo)); }

__device__ __forceinline__ void adamw_coef(AdamwCache& cache, const CameTensorDesc& d, const CameHyper* hyp, bool clipped, double norm,
                                           AdamwShared* sh) {
    const float step = *static_cast<const float*>(d.res_row);
    if (step == cache.step && d.group == cache.group) return;      // (the same in every thread)
    const CameHyper& h = hyp[d.group];
    const double t = (double)step + 1.0;
    __syncthreads();      // (the previous values have been read)
    if (threadIdx.x == 0) sh->size = (float)((double)h.lr / one_minus_power(h.beta3, h.reserved[0], t));
    if (threadIdx.x == 32) sh->root = (float)(1.0 / sqrt(one_minus_power(h.om_beta3, h.reserved[1], t)));
    __syncthreads();
    cache.step = step;
    cache.group = d.group;
    AdamwCoef& k = cache.k;
    k.c = clipped ? (float)((double)h.grad_scale * clip_coefficient(norm, h.clip_threshold)) : h.grad_scale;
    k.b1 = h.beta1; k.om1 = h.om_beta1;
    k.b2 = h.beta2; k.om2 = h.om_beta2;
    k.eps = h.eps0; k.wd_lr = h.wd_lr;
    k.size = sh->size; k.root = sh->root;
    k.key = mix32((uint32_t)t);
}

__device__ __forceinline__ float adamw_moment(float m, float g, const AdamwCoef& k) { return fmaf(k.b1, m, k.om1 * g); }
__device__ __forceinline__ float adamw_second(float v, float g, const AdamwCoef& k) { return fmaf(k.b2, v, k.om2 * (g * g)); }
// (root and quotient to 2 units in the last place: they scale an update of lr, itself added to p with its own rounding)
__device__ __forceinline__ float adamw_param(float p, float m, float v, const AdamwCoef& k) {
    const float den = fmaf(approx_sqrt(v), k.root, k.eps);
    return fmaf(-k.size, __fdividef(m, den), fmaf(-k.wd_lr, p, p));
}

// states in fp32
template <typename P, typename G>
__device__ __forceinline__ void adamw_elems(P* p, const G* g, float* m, float* v, int64_t at, int64_t end, bool vec, const AdamwCoef& k) {
    if (vec && at + 8 <= end) {
        float pv[8], gv[8], mv[8], vv[8];
        load8(g + at, gv);
        load8(m + at, mv);
        load8(v + at, vv);
        load8(p + at, pv);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = gv[i] * k.c;
            mv[i] = adamw_moment(mv[i], x, k);
            vv[i] = adamw_second(vv[i], x, k);
            pv[i] = adamw_param(pv[i], mv[i], vv[i], k);
        }
        store8(m + at, mv);
        store8(v + at, vv);
        store8(p + at, pv);
        return;
    }
    for (int64_t i = at; i < at + 8 && i < end; ++i) {
        const float x = to_f32(g[i]) * k.c, mn = adamw_moment(m[i], x, k), vn = adamw_second(v[i], x, k);
        m[i] = mn;
        v[i] = vn;
        p[i] = from_f32<P>(adamw_param(to_f32(p[i]), mn, vn, k));
    }
}

// states in float8: a warp owns a block, a lane 8 consecutive elements of it
template <typename P, typename G>
__device__ __forceinline__ void adamw_block8(P* p, const G* g, uint8_t* m, uint8_t* v, uint8_t* ms, uint8_t* vs, int64_t blk, int64_t n,
                                             bool vec, const AdamwCoef& k) {
    const int lane = threadIdx.x & 31;
    const int64_t at = blk * QBLOCK + 8 * lane;
    const bool full = vec && at + 8 <= n;
    float pv[8], gv[8], mv[8], vv[8];
    uint2 mc = make_uint2(0u, 0u), vc = make_uint2(0u, 0u);
    const float m_scale = e8m0_value(ms[blk]), v_scale = e8m0_value(vs[blk]);
    if (full) {
        load8(g + at, gv);
        mc = *reinterpret_cast<const uint2*>(m + at);
        vc = *reinterpret_cast<const uint2*>(v + at);
        load8(p + at, pv);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool in = at + i < n;
            gv[i] = in ? to_f32(g[at + i]) : 0.0f;
            pv[i] = in ? to_f32(p[at + i]) : 0.0f;
            const uint32_t a = in ? m[at + i] : 0u, b = in ? v[at + i] : 0u;
            (i < 4 ? mc.x : mc.y) |= a << (8 * (i & 3));
            (i < 4 ? vc.x : vc.y) |= b << (8 * (i & 3));
        }
    }
    e4m3_decode8(mc, mv);
    e5m2_decode8(vc, vv);
    float m_big = 0.0f, v_big = 0.0f;      // (a NaN does not count: it must not flush the rest of the block)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = gv[i] * k.c;
        mv[i] = adamw_moment(mv[i] * m_scale, x, k);
        vv[i] = adamw_second(vv[i] * v_scale, x, k);
        pv[i] = adamw_param(pv[i], mv[i], vv[i], k);
        m_big = fmaxf(m_big, fabsf(mv[i]));
        v_big = fmaxf(v_big, vv[i]);
    }
    const uint32_t m_top = __reduce_max_sync(0xffffffffu, __float_as_uint(m_big));
    const uint32_t v_top = __reduce_max_sync(0xffffffffu, __float_as_uint(v_big));
    const uint32_t m_byte = e8m0_scale<7>(m_top), v_byte = e8m0_scale<14>(v_top);
    const float m_inv = e8m0_inverse(m_byte), v_inv = e8m0_inverse(v_byte);
    // v > 0 stays above zero (its root divides); a block of zeros stays zero
    const float least = v_top ? 0x1p-16f : 0.0f;
    const uint32_t h = mix32((uint32_t)(at >> 3) + k.key);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t r = h * (0x9E3779B1u * (2u * i + 1u));
        mv[i] = dither<20>(mv[i] * m_inv, r & 0xfffffu);
        vv[i] = dither<21>(fmaxf(vv[i] * v_inv, least), r >> 11);
    }
    mc = e4m3_encode8(mv);
    vc = e5m2_encode8(vv);
    if (full) {
        *reinterpret_cast<uint2*>(m + at) = mc;
        *reinterpret_cast<uint2*>(v + at) = vc;
        store8(p + at, pv);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (at + i < n) {
                m[at + i] = (uint8_t)((i < 4 ? mc.x : mc.y) >> (8 * (i & 3)));
                v[at + i] = (uint8_t)((i < 4 ? vc.x : vc.y) >> (8 * (i & 3)));
                p[at + i] = from_f32<P>(pv[i]);
            }
    }
    if (lane == 0) { ms[blk] = (uint8_t)m_byte; vs[blk] = (uint8_t)v_byte; }
}

template <typename P, typename G, bool F8>
__global__ void __launch_bounds__(ADAMW_THREADS) k_adamw(const StepArgs a, const AdamwArgs w, const __grid_constant__ AdamwHyp by_value) {
    __shared__ AdamwShared sh;
    __shared__ double red[ADAMW_THREADS / 32];
    __shared__ bool last;
    const CameHyper* hyp = w.by_value ? by_value.h : a.hyp;
    double norm = 0.0;
    if (w.norm_parts) {
        norm = norm_of_partials(w.norm_parts, w.n_parts, red);
        if (blockIdx.x == 0 && threadIdx.x == 0) *w.norm_out = (float)norm;
        if (!isfinite(norm)) return;      // (in every CTA, and before anything is written: the step does not take place)
    }
    AdamwCache cache;
    cache.step = -1.0f;
    cache.group = -1;
    for (int item = blockIdx.x; item < w.n; item += gridDim.x) {
        const Work wk = w.work[item];
        const CameTensorDesc& d = a.descs[wk.tensor];
        adamw_coef(cache, d, hyp, w.norm_parts != nullptr, norm, &sh);
        const int64_t n = d.rows * (d.cols ? d.cols : 1) * (d.batch > 1 ? (int64_t)d.batch : 1);
        const int64_t lo = (int64_t)wk.tile * w.chunk, hi = min(lo + w.chunk, n);
        const bool vec = a.scr[wk.tensor].g_v == 8;
        P* p = static_cast<P*>(d.p);
        const G* g = static_cast<const G*>(d.g);
        if (F8) {
            for (int64_t b = lo / QBLOCK + (threadIdx.x >> 5); b * QBLOCK < hi; b += ADAMW_THREADS / 32)
                adamw_block8(p, g, static_cast<uint8_t*>(d.m), static_cast<uint8_t*>(d.sq_row), reinterpret_cast<uint8_t*>(d.m_absmax),
                             reinterpret_cast<uint8_t*>(d.sq_row_absmax), b, n, vec, cache.k);
        } else {
            for (int64_t at = lo + 8 * threadIdx.x; at < hi; at += 8 * ADAMW_THREADS)
                adamw_elems(p, g, static_cast<float*>(d.m), static_cast<float*>(d.sq_row), at, hi, vec, cache.k);
        }
    }
    // the last CTA counts the step: every other one has read the counts it needs
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(w.ticket, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (last) {
        for (int i = threadIdx.x; i < w.n_tensors; i += ADAMW_THREADS) *static_cast<float*>(a.descs[w.tensors[i].tensor].res_row) += 1.0f;
        if (threadIdx.x == 0) *w.ticket = 0u;
    }
}

template <typename P, typename G, bool F8>
static cudaError_t launch_one(const StepArgs& a, const AdamwArgs& w, const AdamwHyp& h, cudaStream_t st) {
    const int grid = min(w.n, persistent_grid_limit() * 8);
    k_adamw<P, G, F8><<<grid, ADAMW_THREADS, 0, st>>>(a, w, h);
    return cudaGetLastError();
}
template <typename P, bool F8>
static cudaError_t launch_g(int g_dtype, const StepArgs& a, const AdamwArgs& w, const AdamwHyp& h, cudaStream_t st) {
    if (g_dtype == CAME_DT_F32) return launch_one<P, float, F8>(a, w, h, st);
    if (g_dtype == CAME_DT_F16) return launch_one<P, __half, F8>(a, w, h, st);
    return launch_one<P, __nv_bfloat16, F8>(a, w, h, st);
}
template <bool F8>
static cudaError_t launch_p(const KernelKey& key, const StepArgs& a, const AdamwArgs& w, const AdamwHyp& h, cudaStream_t st) {
    if (key.p_dtype == CAME_DT_F32) return launch_g<float, F8>(key.g_dtype, a, w, h, st);
    if (key.p_dtype == CAME_DT_F16) return launch_g<__half, F8>(key.g_dtype, a, w, h, st);
    return launch_g<__nv_bfloat16, F8>(key.g_dtype, a, w, h, st);
}

cudaError_t launch_adamw(const KernelKey& key, const StepArgs& a, const AdamwArgs& args, const CameHyper* host_hyp, int n_hyp, cudaStream_t st) {
    AdamwArgs w = args;
    AdamwHyp h{};
    w.by_value = host_hyp != nullptr;
    if (host_hyp)
        for (int i = 0; i < n_hyp && i < ADAMW_MAX_HYP; ++i) h.h[i] = host_hyp[i];
    return key.mode == CAME_MODE_ADAMW8 ? launch_p<true>(key, a, w, h, st) : launch_p<false>(key, a, w, h, st);
}

}  // namespace came
