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
// better the rate: bf16, 1024 M elements, 3.44 ms with two CTAs per SM whose warps take runs of 256 elements in turn and spans of
// 4096 elements (the copy rate), 3.53 with spans of 16384, 3.65 with three CTAs, 3.75 with four, 3.56 where a warp takes 4096
// elements for itself.
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
// 256 elements by a warp, all loads before the first store
template <typename P, typename G> struct Run8 {
    float p[8], g[8], m[8], v[8];
    __device__ __forceinline__ void step(const AdamwCoef& k) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = g[i] * k.c;
            m[i] = adamw_moment(m[i], x, k);
            v[i] = adamw_second(v[i], x, k);
            p[i] = adamw_param(p[i], m[i], v[i], k);
        }
    }
    // a lane 8 consecutive ones
    __device__ __forceinline__ void load(const P* ps, const G* gs, const float* ms, const float* vs, int64_t at) {
        load8(gs + at, g);
        load8(ms + at, m);
        load8(vs + at, v);
        load8(ps + at, p);
    }
    __device__ __forceinline__ void store(P* ps, float* ms, float* vs, int64_t at) const {
        store8(ms + at, m);
        store8(vs + at, v);
        store8(ps + at, p);
    }
    // tensors that do not all allow that: lane l takes l, l + 32, ..., so that a warp's accesses lie next to each other
    // (fp16 off the boundaries, 256 M elements: 3100 us with 8 consecutive elements a lane, 1090 so)
    __device__ __forceinline__ void load_across(const P* ps, const G* gs, const float* ms, const float* vs, int64_t at) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            g[i] = to_f32(gs[at + 32 * i]);
            m[i] = ms[at + 32 * i];
            v[i] = vs[at + 32 * i];
            p[i] = to_f32(ps[at + 32 * i]);
        }
    }
    __device__ __forceinline__ void store_across(P* ps, float* ms, float* vs, int64_t at) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            ms[at + 32 * i] = m[i];
            vs[at + 32 * i] = v[i];
            ps[at + 32 * i] = from_f32<P>(p[i]);
        }
    }
};

template <typename P, typename G>
__global__ void __launch_bounds__(ADAMW_THREADS, ADAMW_CTAS) k_adamw(const StepArgs a, const AdamwArgs w, const __grid_constant__ AdamwHyp by_value) {
    const CameHyper* hyp = w.by_value ? by_value.h : a.hyp;
    griddep_wait();
    double norm;
    if (!adamw_norm(w, &norm)) return;      // (in every CTA, and before anything is written)
    AdamwCache cache;
    cache.step = -1.0f;
    cache.group = -1;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for_runs(a, w, [&](const CameTensorDesc& d, int tensor, int64_t lo, int64_t hi, int64_t n) {
        const bool vec = a.scr[tensor].g_v == 8;
        P* p = static_cast<P*>(d.p);
        const G* g = static_cast<const G*>(d.g);
        float *m = static_cast<float*>(d.m), *v = static_cast<float*>(d.sq_row);
        const int64_t whole = lo + (hi - lo) / 256 * 256;
        int64_t at = lo + 256 * warp;
        adamw_coef(cache, d, hyp, w.norm_parts != nullptr, norm);
        const AdamwCoef& k = cache.k;
        if (vec)
            for (; at < whole; at += 256 * ADAMW_WARPS) {
                Run8<P, G> r;
                r.load(p, g, m, v, at + 8 * lane);
                r.step(k);
                r.store(p, m, v, at + 8 * lane);
            }
        else
            for (; at < whole; at += 256 * ADAMW_WARPS) {
                Run8<P, G> r;
                r.load_across(p, g, m, v, at + lane);
                r.step(k);
                r.store_across(p, m, v, at + lane);
            }
        if (at == whole)      // the warp whose turn it is
            for (at += lane; at < hi; at += 32) adamw_one(p, g, m, v, at, k);
    });
    griddep_launch();
    adamw_count_step(w);
}

template <typename P, typename G> struct LaunchAdamw {
    static cudaError_t run(const StepArgs& a, const AdamwArgs& w, const AdamwHyp& h, cudaStream_t st) {
        // (256 M elements, one tensor, spans of 2048 / 4096: fp32 1040 / 1113 us, bf16 890 / 857; fp32 decoders of width 768 to 4096:
        // 3 % slower to 6 % faster with the short ones)
        AdamwArgs x = w;
        const int grid = adamw_spans(x, ADAMW_CTAS, sizeof(P) + sizeof(G) <= 4 ? 2 : 1);
        return launch_behind(k_adamw<P, G>, grid, ADAMW_THREADS, 0, st, a, x, h);
    }
};

cudaError_t launch_adamw(const KernelKey& key, const StepArgs& a, const AdamwArgs& args, const CameHyper* host_hyp, int n_hyp, cudaStream_t st) {
    AdamwArgs w = args;
    w.by_value = host_hyp != nullptr;
    const AdamwHyp h = adamw_hyp(host_hyp, n_hyp);
    return key.mode == CAME_MODE_ADAMW8 ? launch_adamw8(key, a, w, h, st) : adamw_for<LaunchAdamw>(key, a, w, h, st);
}

}  // namespace came
