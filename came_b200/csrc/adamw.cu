// AdamW over many tensors in one launch, states in fp32.
//
//   m' = b1 m + (1 - b1) c g      v' = b2 v + (1 - b2) (c g)^2      c = grad_scale x clip coefficient
//   p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// t is counted on the device: every CTA reads it, the last one to finish adds 1, so that a captured step counts its own
// replays.  1 - b^t is formed as -expm1(t ln b) in 64 bits (at t = 1, b2 = 0.999 a difference in 32 bits keeps three
// digits), once per warp and set of tensors with the same count.
#include "adamw.cuh"
#include "launch.h"

namespace came {

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

template <typename P, typename G>
__global__ void __launch_bounds__(ADAMW_THREADS, 4) k_adamw(const StepArgs a, const AdamwArgs w, const __grid_constant__ AdamwHyp by_value) {
    const CameHyper* hyp = w.by_value ? by_value.h : a.hyp;
    double norm;
    if (!adamw_norm(w, &norm)) return;      // (in every CTA, and before anything is written)
    AdamwCache cache;
    cache.step = -1.0f;
    cache.group = -1;
    const int lane = threadIdx.x & 31;
    // an item is a warp's
    for (int item = blockIdx.x + gridDim.x * (threadIdx.x >> 5); item < w.n; item += gridDim.x * (ADAMW_THREADS / 32)) {
        const Work wk = w.work[item];
        const CameTensorDesc& d = a.descs[wk.tensor];
        const int64_t n = d.rows * (d.cols ? d.cols : 1) * (d.batch > 1 ? (int64_t)d.batch : 1);
        const int64_t lo = (int64_t)wk.tile * w.chunk, hi = min(lo + w.chunk, n);
        const bool vec = a.scr[wk.tensor].g_v == 8;
        adamw_coef(cache, d, hyp, w.norm_parts != nullptr, norm);
        for (int64_t at = lo + 8 * lane; at < hi; at += 8 * 32)
            adamw_elems(static_cast<P*>(d.p), static_cast<const G*>(d.g), static_cast<float*>(d.m), static_cast<float*>(d.sq_row), at, hi, vec,
                        cache.k);
    }
    adamw_count_step(a, w);
}

template <typename P, typename G> struct LaunchAdamw {
    static cudaError_t run(const StepArgs& a, const AdamwArgs& w, const AdamwHyp& h, cudaStream_t st) {
        k_adamw<P, G><<<min(w.n, persistent_grid_limit() * 4), ADAMW_THREADS, 0, st>>>(a, w, h);
        return cudaGetLastError();
    }
};

cudaError_t launch_adamw(const KernelKey& key, const StepArgs& a, const AdamwArgs& args, const CameHyper* host_hyp, int n_hyp, cudaStream_t st) {
    AdamwArgs w = args;
    w.by_value = host_hyp != nullptr;
    const AdamwHyp h = adamw_hyp(host_hyp, n_hyp);
    return key.mode == CAME_MODE_ADAMW8 ? launch_adamw8(key, a, w, h, st) : adamw_for<LaunchAdamw>(key, a, w, h, st);
}

}  // namespace came
