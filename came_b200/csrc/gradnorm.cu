// Norm of all gradients, and the clip that follows from it.
//
//   N = sqrt(sum_i (s_i g_i)^2)      c = min(1, max_norm / (N + 1e-6))      g_i' = c g_i
//
// One pass over the gradients leaves a sum per CTA; whoever needs N (every CTA of the scaling pass, every CTA of the AdamW
// step) adds those few hundred sums itself, always in the same order: no atomics, no launch in between.  Eight squares are
// added in fp32, those sums in 64 bits; where eight squares leave the safe range of fp32 they are formed in 64 bits, so that
// neither a huge nor a tiny gradient costs the norm its value.
#include "adamw.cuh"
#include "launch.h"

namespace came {

constexpr int NORM_THREADS = 256;
constexpr int NORM_CTAS = 4;      // per SM: 1.26 G bf16 elements in 368 us, 6 860 GB/s (the copy rate is 6 562; nothing is written)

__device__ __forceinline__ double squares8(const float* x) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(x[i], x[i], s);
    if (s > 1e-30f && s < 1e30f) return (double)s;
    double t = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) t = fma((double)x[i], (double)x[i], t);
    return t;
}
__device__ __forceinline__ void load_g8(const float* p, float* v) {
    const uint4 a = load16(p), b = load16(p + 4);
    v[0] = __uint_as_float(a.x); v[1] = __uint_as_float(a.y); v[2] = __uint_as_float(a.z); v[3] = __uint_as_float(a.w);
    v[4] = __uint_as_float(b.x); v[5] = __uint_as_float(b.y); v[6] = __uint_as_float(b.z); v[7] = __uint_as_float(b.w);
}
__device__ __forceinline__ void load_g8(const __nv_bfloat16* p, float* v) { load8(p, v); }
__device__ __forceinline__ void load_g8(const __half* p, float* v) { load8(p, v); }
__device__ __forceinline__ void store_g8(float* p, const float* v) { store_run<8>(p, v); }
__device__ __forceinline__ void store_g8(__nv_bfloat16* p, const float* v) { store_run<8>(p, v); }
__device__ __forceinline__ void store_g8(__half* p, const float* v) { store_run<8>(p, v); }

// elements in front of the first 16-byte boundary, at most n
template <typename T>
__device__ __forceinline__ int64_t head_of(const T* g, int64_t n) {
    const int64_t k = (int64_t)((16u - (uint32_t)(reinterpret_cast<uintptr_t>(g) & 15u)) & 15u) / (int64_t)sizeof(T);
    return k < n ? k : n;
}

// this thread's share of the squares of g[0 .. n)
template <typename T>
__device__ __forceinline__ double chunk_squares(const T* g, int64_t n) {
    const int64_t head = head_of(g, n), body = (n - head) / 8;
    double t = 0.0;
    int64_t i = threadIdx.x;
    for (; i + 3 * NORM_THREADS < body; i += 4 * NORM_THREADS) {
        float x[4][8];
#pragma unroll
        for (int u = 0; u < 4; ++u) load_g8(g + head + 8 * (i + u * NORM_THREADS), x[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u) t += squares8(x[u]);
    }
    for (; i < body; i += NORM_THREADS) {
        float x[8];
        load_g8(g + head + 8 * i, x);
        t += squares8(x);
    }
    for (int64_t k = threadIdx.x; k < head; k += NORM_THREADS) t += (double)to_f32(g[k]) * (double)to_f32(g[k]);
    for (int64_t k = head + 8 * body + threadIdx.x; k < n; k += NORM_THREADS) t += (double)to_f32(g[k]) * (double)to_f32(g[k]);
    return t;
}
__device__ __forceinline__ double chunk_squares_any(const void* g, int dtype, int64_t lo, int64_t n) {
    if (dtype == CAME_DT_F32) return chunk_squares(static_cast<const float*>(g) + lo, n);
    if (dtype == CAME_DT_F16) return chunk_squares(static_cast<const __half*>(g) + lo, n);
    return chunk_squares(static_cast<const __nv_bfloat16*>(g) + lo, n);
}

__global__ void __launch_bounds__(NORM_THREADS) k_grad_norm(const StepArgs a, const AdamwArgs w, const __grid_constant__ AdamwHyp by_value,
                                                           double* parts) {
    __shared__ double red[NORM_THREADS / 32];
    const CameHyper* hyp = w.by_value ? by_value.h : a.hyp;
    griddep_wait();
    double t = 0.0;
    for_runs(a, w, [&](const CameTensorDesc& d, int, int64_t lo, int64_t hi, int64_t) {
        const double s = (double)hyp[d.group].grad_scale;
        t += s * s * chunk_squares_any(d.g, d.g_dtype, lo, hi - lo);
    });
    griddep_launch();
    t = block_sum64(t, red);
    if (threadIdx.x == 0) parts[blockIdx.x] = t;
}

static int norm_spans(AdamwArgs& w) { return adamw_spans(w, NORM_CTAS, 16); }
int grad_norm_parts(int n) {
    AdamwArgs w{};
    w.n = n;
    return norm_spans(w);
}

cudaError_t launch_grad_norm(const StepArgs& a, const Work* work, int n, const CameHyper* host_hyp, int n_hyp, double* parts, cudaStream_t st) {
    AdamwArgs w{};
    w.work = work;
    w.n = n;
    w.by_value = host_hyp != nullptr;
    const int grid = norm_spans(w);
    return launch_behind(k_grad_norm, grid, NORM_THREADS, 0, st, a, w, adamw_hyp(host_hyp, n_hyp), parts);
}

// ---- tensors given by value: the table is a kernel argument (the limit is 32 764 bytes), nothing is uploaded -------------
template <int N> struct GradTable {
    void* g[N];
    int64_t n[N];
    int first[N + 1];      // chunk at which a tensor begins
    uint8_t dtype[N];
    int count, chunk;
};
// Tensors of a launch: the small table is passed faster (host time of a call: 64 gradients 9.4 us, 65 in the large one 11.3).
constexpr int CLIP_FEW = 64, CLIP_MOST = 1024;

// tensor that chunk c belongs to
template <int N>
__device__ __forceinline__ int tensor_of(const GradTable<N>& t, int c) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
template <int N>
__global__ void __launch_bounds__(NORM_THREADS) k_clip_norm(const __grid_constant__ GradTable<N> t, double* parts) {
    __shared__ double red[NORM_THREADS / 32];
    griddep_wait();
    double s = 0.0;
    for (int c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
        const int i = tensor_of(t, c);
        const int64_t lo = (int64_t)(c - t.first[i]) * t.chunk;
        s += chunk_squares_any(t.g[i], t.dtype[i], lo, min((int64_t)t.chunk, t.n[i] - lo));
    }
    griddep_launch();
    s = block_sum64(s, red);
    if (threadIdx.x == 0) parts[blockIdx.x] = s;
}

template <typename T>
__device__ __forceinline__ void chunk_scale(T* g, int64_t n, float c) {
    const int64_t head = head_of(g, n), body = (n - head) / 8;
    for (int64_t i = threadIdx.x; i < body; i += NORM_THREADS) {
        float x[8];
        load_g8(g + head + 8 * i, x);
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] *= c;
        store_g8(g + head + 8 * i, x);
    }
    for (int64_t k = threadIdx.x; k < head; k += NORM_THREADS) g[k] = from_f32<T>(to_f32(g[k]) * c);
    for (int64_t k = head + 8 * body + threadIdx.x; k < n; k += NORM_THREADS) g[k] = from_f32<T>(to_f32(g[k]) * c);
}
template <int N>
__global__ void __launch_bounds__(NORM_THREADS) k_clip_scale(const __grid_constant__ GradTable<N> t, const double* parts, int n_parts,
                                                            float max_norm, float* norm_out) {
    __shared__ double red[NORM_THREADS / 32];
    griddep_wait();
    const double norm = norm_of_partials(parts, n_parts, red);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const float c = (float)clip_coefficient(norm, max_norm);
    if (c == 1.0f) return;
    for (int k = blockIdx.x; k < t.first[t.count]; k += gridDim.x) {
        const int i = tensor_of(t, k);
        const int64_t lo = (int64_t)(k - t.first[i]) * t.chunk, n = min((int64_t)t.chunk, t.n[i] - lo);
        if (t.dtype[i] == CAME_DT_F32) chunk_scale(static_cast<float*>(t.g[i]) + lo, n, c);
        else if (t.dtype[i] == CAME_DT_F16) chunk_scale(static_cast<__half*>(t.g[i]) + lo, n, c);
        else chunk_scale(static_cast<__nv_bfloat16*>(t.g[i]) + lo, n, c);
    }
}

static inline int clip_grid(int chunks) { return max(1, min(chunks, persistent_grid_limit() * NORM_CTAS)); }
size_t clip_parts(int n_tensors) {
    return (size_t)(n_tensors / CLIP_MOST + 1) * (size_t)(persistent_grid_limit() * NORM_CTAS);
}

template <int N>
static void clip_table(GradTable<N>& t, const CameGradRef* grads, int n, int chunk) {
    t.count = n;
    t.chunk = chunk;
    int at = 0;
    for (int i = 0; i < n; ++i) {
        t.g[i] = grads[i].g;
        t.n[i] = grads[i].n;
        t.dtype[i] = (uint8_t)grads[i].dtype;
        t.first[i] = at;
        at += (int)((grads[i].n + chunk - 1) / chunk);
    }
    t.first[n] = at;
}
template <int N>
static cudaError_t clip_pass(const GradTable<N>& t, bool scale, double* parts, int* n_parts, float max_norm, float* norm, cudaStream_t st) {
    const int grid = clip_grid(t.first[t.count]);
    if (scale) return launch_behind(k_clip_scale<N>, grid, NORM_THREADS, 0, st, t, static_cast<const double*>(parts), *n_parts, max_norm, norm);
    double* const to = parts + *n_parts;
    *n_parts += grid;
    return launch_behind(k_clip_norm<N>, grid, NORM_THREADS, 0, st, t, to);
}

cudaError_t launch_clip(const CameGradRef* grads, int n, float max_norm, float* norm, double* parts, cudaStream_t st) {
    // Chunks of a tensor: as long as leaves two for every SM, since each is looked up and begun anew (chunks of 4096 / 16384 / 65536
    // elements: 528 bf16 gradients of 10 to 20 thousand 10.3 / 8.4 / 7.7 us, 1.26 G elements in 201 gradients 867 / 392 / 368);
    // at most 2^30 of them.
    double total = 0.0;
    for (int i = 0; i < n; ++i) total += (double)grads[i].n;
    int64_t chunk = 4096;
    while (chunk < 65536 && total / (double)chunk > 2.0 * persistent_grid_limit()) chunk *= 2;
    while (total / (double)chunk > (double)(1 << 30)) chunk *= 2;
    int n_parts = 0;
    cudaError_t e = cudaSuccess;
    const bool norm_only = isinf(max_norm);
    GradTable<CLIP_FEW> few;      // (filled once where one table holds all: 528 gradients 2 us less on the host)
    GradTable<CLIP_MOST> most;
    int filled = -1;
    for (int pass = 0; pass < (norm_only ? 1 : 2) && e == cudaSuccess; ++pass)
        for (int at = 0; at < n && e == cudaSuccess; at += CLIP_MOST) {
            const int k = min(n - at, CLIP_MOST);
            float* out = at == 0 ? norm : nullptr;
            if (at != filled) {
                if (k <= CLIP_FEW) clip_table(few, grads + at, k, (int)chunk);
                else clip_table(most, grads + at, k, (int)chunk);
                filled = at;
            }
            e = k <= CLIP_FEW ? clip_pass(few, pass == 1, parts, &n_parts, max_norm, out, st)
                              : clip_pass(most, pass == 1, parts, &n_parts, max_norm, out, st);
        }
    if (e == cudaSuccess && (norm_only || n == 0)) {      // the total alone: an empty table
        const GradTable<CLIP_FEW> none{};
        e = launch_behind(k_clip_scale<CLIP_FEW>, 1, NORM_THREADS, 0, st, none, static_cast<const double*>(parts), n_parts, max_norm, norm);
    }
    return e;
}

}  // namespace came
