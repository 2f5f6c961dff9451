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

// Bound by DRAM: 22 (16-bit types) or 28 bytes an element.  The fewer the streams and the closer together their addresses, the
// better the rate: bf16, 1024 M elements, 3.44 ms with two CTAs per SM and spans of 4096 elements (the copy rate), 3.53 with
// spans of 16384, 3.65 with three CTAs, 3.75 with four, 3.56 with two CTAs whose warps take 4096 elements each.
constexpr int ADAMW_CTAS = 2;

__device__ __forceinline__ float adamw_moment(float m, float g, const AdamwCoef& k) { return fmaf(k.b1, m, k.om1 * g); }
__device__ __forceinline__ float adamw_second(float v, float g, const AdamwCoef& k) { return fmaf(k.b2, v, k.om2 * (g * g)); }
// (root and quotient to 2 units in the last place: they scale an update of lr, itself added to p with its own rounding)
__device__ __forceinline__ float adamw_param(float p, float m, float v, const AdamwCoef& k) {
    const float den = fmaf(approx_sqrt(v), k.root, k.eps);
    return fmaf(-k.size, __fdividef(m, den), fmaf(-k.wd_lr, p, p));
}

template <typename P, typename G>
__device__ __forceinline__ void adamw_one(P* p, const G* g, float* m, float* v, int64_t i, const AdamwCoef& k) {
    const float x = to_f32(g[i]) * k.c, mn = adamw_moment(m[i], x, k), vn = adamw_second(v[i], x, k);
    m[i] = mn;
    v[i] = vn;
    p[i] = from_f32<P>(adamw_param(to_f32(p[i]), mn, vn, k));
}
// 256 elements by a warp, a lane 8 consecutive ones; all loads before the first store
template <typename P, typename G>
__device__ __forceinline__ void adamw_run8(P* p, const G* g, float* m, float* v, int64_t at, const AdamwCoef& k) {
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
}
// 256 elements of tensors that do not all allow that: lane l takes l, l + 32, ..., so that a warp's accesses lie next to each
// other, all loads before the first store (fp16 off the boundaries, 256 M elements: 3100 us with 8 consecutive elements a lane,
// 1130 so)
template <typename P, typename G>
__device__ __forceinline__ void adamw_run1(P* p, const G* g, float* m, float* v, int64_t at, const AdamwCoef& k) {
    P pv[8];
    G gv[8];
    float mv[8], vv[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        gv[i] = g[at + 32 * i];
        mv[i] = m[at + 32 * i];
        vv[i] = v[at + 32 * i];
        pv[i] = p[at + 32 * i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = to_f32(gv[i]) * k.c, mn = adamw_moment(mv[i], x, k), vn = adamw_second(vv[i], x, k);
        m[at + 32 * i] = mn;
        v[at + 32 * i] = vn;
        p[at + 32 * i] = from_f32<P>(adamw_param(to_f32(pv[i]), mn, vn, k));
    }
}

template <typename P, typename G>
__global__ void __launch_bounds__(ADAMW_THREADS, ADAMW_CTAS) k_adamw(const StepArgs a, const AdamwArgs w, const __grid_constant__ AdamwHyp by_value) {
    const CameHyper* hyp = w.by_value ? by_value.h : a.hyp;
    double norm;
    if (!adamw_norm(w, &norm)) return;      // (in every CTA, and before anything is written)
    AdamwCache cache;
    cache.step = -1.0f;
    cache.group = -1;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for_runs(a, w, [&](const CameTensorDesc& d, int tensor, int64_t lo, int64_t hi, int64_t n) {
        const bool vec = a.scr[tensor].g_v == 8;
        adamw_coef(cache, d, hyp, w.norm_parts != nullptr, norm);
        P* p = static_cast<P*>(d.p);
        const G* g = static_cast<const G*>(d.g);
        float *m = static_cast<float*>(d.m), *v = static_cast<float*>(d.sq_row);
        const int64_t whole = lo + (hi - lo) / 256 * 256;
        int64_t at = lo + 256 * warp;
        if (vec)
            for (; at < whole; at += 256 * ADAMW_WARPS) adamw_run8(p, g, m, v, at + 8 * lane, cache.k);
        else
            for (; at < whole; at += 256 * ADAMW_WARPS) adamw_run1(p, g, m, v, at + lane, cache.k);
        if (at == whole)      // the warp whose turn it is
            for (at += lane; at < hi; at += 32) adamw_one(p, g, m, v, at, cache.k);
    });
    adamw_count_step(a, w);
}

template <typename P, typename G> struct LaunchAdamw {
    static cudaError_t run(const StepArgs& a, const AdamwArgs& w, const AdamwHyp& h, cudaStream_t st) {
        AdamwArgs x = w;
        const int grid = adamw_spans(x, ADAMW_CTAS, 2);
        k_adamw<P, G><<<grid, ADAMW_THREADS, 0, st>>>(a, x, h);
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
