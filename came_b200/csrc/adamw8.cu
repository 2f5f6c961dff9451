// AdamW over many tensors in one launch, moments in float8 (formulas and step count: adamw.cu).
//
// m is held as e4m3, v as e5m2 (its root then has the range and the relative step of m), both times a scale 2^k (one e8m0
// byte per 256 elements) that puts the exponent of the block's largest magnitude at 2^7 resp. 2^14.  A scale that is a power
// of two leaves the grid where it is from step to step, so that only what a moment gained is rounded, and it is rounded
// stochastically on the format's whole grid, subnormals included.  Rounded to nearest, v would never fall at b2 = 0.999 (a step
// moves it by 0.1 %, half a spacing is 7 to 12 %), and an m of few subnormal units would never die out at b1 = 0.9.
// The random bits are a hash of the element's index and t: no state, the same in every run.
//
// A warp owns blocks of 256 elements, a lane 8 consecutive elements of each; the block's largest magnitudes are one warp
// reduction.  Parameters, gradients and codes of the next STAGES - 1 blocks are on their way into a ring in shared memory
// by asynchronous copies of 16 (codes: 8) bytes.  Parameters and gradients that do not start on such a boundary are copied
// from the boundaries around them and shifted as they are read.
//
// Bound by instructions first, by DRAM close behind (10.03 bytes an element in 16-bit types): one element per lane and step takes
// 54 instructions; packed arithmetic, whole blocks without questions per block (span8_fast) and codes that are cut out of the
// rounded bits instead of converted leave 34.  256 M bf16 elements: 404 us (97 % of the copy rate); under the power cap, back to
// back, the clock falls to 1.6-1.8 GHz and 1.26 G elements take 2.14-2.19 ms (88-90 %).
#include <cfloat>

#include "adamw.cuh"
#include "launch.h"
#include "pipeline.cuh"

namespace came {

// Two CTAs of 8 warps per SM and a ring of four slots: more warps mean fewer registers (80 at three CTAs: spills, 461 us where two
// take 404 for 256 M bf16 elements), deeper rings bring nothing (five slots: 416 us).
constexpr int ADAMW8_CTAS = 2, ADAMW8_STAGES = 4;
// The fast root takes what is below 1.2e-38 for zero, the true one 1.1e-19 at most: with eps 2^24 times that (times the factor of
// the root) or more, no digit of their sum is lost.
constexpr float ADAMW8_LOST_ROOT = 2e-12f;

// A slot: 256 parameters and 256 gradients from the 32-byte boundary in front of them, then 16 bytes of codes (m, v) per lane.
// A sector (32 bytes) of memory has to lie in one sector of the slot: split over two it is fetched twice (fp32: 36 instead of
// 20 million sectors for 64 million elements, 940 instead of 690 us for 256 million).
template <typename P, typename G> struct Ring8 {
    static constexpr int G_OFF = QBLOCK * sizeof(P) + 32, MV_OFF = G_OFF + QBLOCK * sizeof(G) + 32;
    static constexpr int BYTES = MV_OFF + 32 * 16;
    static constexpr int STAGES = ADAMW8_STAGES;
    static constexpr int CTA_BYTES = BYTES * STAGES * (ADAMW_THREADS / 32);
};

constexpr int BSTEP = QBLOCK * ADAMW_WARPS;      // elements from a warp's block to its next one: the warps of a CTA take blocks in turn
// The blocks a warp is at: addresses of this lane's 8 elements of the first one
template <typename P, typename G> struct Span8 {
    P* p;
    const G* g;
    uint8_t *m, *v;
    int64_t left;               // elements of the tensor from the first block on
    uint32_t p_off, g_off;      // bytes that the tensors start behind a 32-byte boundary
    int async_lo, async_hi;     // blocks that are copied asynchronously: all of them, and the boundaries around them, lie inside the tensor
};

// 256 elements from `from`, a 32-byte boundary `off` bytes in front of them
template <typename T>
__device__ __forceinline__ void ring_copy(uint8_t* slot, const uint8_t* from, uint32_t off, int lane) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) cp16(slot + 512 * i + 16 * lane, from + 512 * i + 16 * lane, 16);
    if (16 * lane < off) cp16(slot + QBLOCK * sizeof(T) + 16 * lane, from + QBLOCK * sizeof(T) + 16 * lane, 16);
}
// this lane's 8 elements, as they lie in memory
template <typename T>
__device__ __forceinline__ void ring_read(const uint8_t* slot, uint32_t off, int lane, uint32_t* w) {
    constexpr int WORDS = 2 * sizeof(T);
    const uint8_t* at = slot + (off & 16) + lane * (4 * WORDS);
    uint32_t x[WORDS + 4];
#pragma unroll
    for (int i = 0; i < WORDS; i += 4) *reinterpret_cast<uint4*>(x + i) = *reinterpret_cast<const uint4*>(at + 4 * i);
    if ((off & 15) == 0) {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = x[i];
        return;
    }
    *reinterpret_cast<uint4*>(x + WORDS) = *reinterpret_cast<const uint4*>(at + 4 * WORDS);
    if (off & 4)
#pragma unroll
        for (int i = 0; i < WORDS + 3; ++i) x[i] = x[i + 1];
    if (off & 8)
#pragma unroll
        for (int i = 0; i < WORDS + 2; ++i) x[i] = x[i + 2];
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = __funnelshift_r(x[i], x[i + 1], 8 * (off & 3));
}
// some elements, one by one, to where ring_read with offset 0 looks for them; the others are zero
template <typename T>
__device__ __forceinline__ void ring_gather(uint8_t* slot, const T* src, int n, int lane) {
#pragma unroll
    for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(slot)[8 * lane + i] = i < n ? src[i] : from_f32<T>(0.0f);
}

template <typename P, typename G>
__device__ __forceinline__ void block8_fetch(uint8_t* slot, const Span8<P, G>& t, int b, int lane) {
    using R = Ring8<P, G>;
    if (b >= t.async_lo && b < t.async_hi) {
        ring_copy<P>(slot, reinterpret_cast<const uint8_t*>(t.p + b * BSTEP - 8 * lane) - t.p_off, t.p_off, lane);
        ring_copy<G>(slot + R::G_OFF, reinterpret_cast<const uint8_t*>(t.g + b * BSTEP - 8 * lane) - t.g_off, t.g_off, lane);
        cp8(slot + R::MV_OFF + lane * 16, t.m + b * BSTEP);
        cp8(slot + R::MV_OFF + lane * 16 + 8, t.v + b * BSTEP);
        return;
    }
    const int at = b * BSTEP, k = (int)max((int64_t)0, min((int64_t)8, t.left - at - 8 * lane));
    ring_gather(slot, t.p + at, k, lane);
    ring_gather(slot + R::G_OFF, t.g + at, k, lane);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        slot[R::MV_OFF + lane * 16 + i] = i < k ? t.m[at + i] : (uint8_t)0;
        slot[R::MV_OFF + lane * 16 + 8 + i] = i < k ? t.v[at + i] : (uint8_t)0;
    }
}

template <typename T> __device__ __forceinline__ u64 word_pair(const uint32_t* w, int j);
template <> __device__ __forceinline__ u64 word_pair<float>(const uint32_t* w, int j) { return pk_u32(w[2 * j], w[2 * j + 1]); }
template <> __device__ __forceinline__ u64 word_pair<__nv_bfloat16>(const uint32_t* w, int j) { return pk_u32(w[j] << 16, w[j] & 0xffff0000u); }
template <> __device__ __forceinline__ u64 word_pair<__half>(const uint32_t* w, int j) {
    return __half22float2(*reinterpret_cast<const __half2*>(w + j));
}

// A packed product with a rounding of its own: a product followed by a sum would be contracted into one rounding
__device__ __forceinline__ u64 mul2_rounded(u64 a, u64 b) { return fma2(a, b, splat(0.0f)); }

// What a lane makes of its 8 elements of a block
struct Result8 {
    float p[8];
    uint2 m, v;
    uint32_t m_top, v_top;      // bits of the block's largest magnitudes
};

// Stochastic rounding on the grid of an 8-bit format with SHIFT = 23 - (its mantissa bits): floor(|y| / u + r / 2^SHIFT) u, u the
// spacing at y.  y = x / 2^k is brought down by as much as lies between the least normal numbers of fp32 and of the format, 2^-120
// for e4m3 and 2^-112 for e5m2.  The spacing then is bit SHIFT of the fp32 number whatever its size, subnormals included:
// r < 2^SHIFT is added to the bits, and the code stands above bit SHIFT.  The product is truncated, which loses nothing
// of the floor.  Two neighbours become the upper and the lower half of a word, and from there bytes.
__device__ __forceinline__ uint32_t e4m3_halves(u64 x, uint32_t r0, uint32_t r1) {      // codes in the upper bytes
    const uint32_t w = __byte_perm(__float_as_uint(x.x) + (r0 & 0xfffffu), __float_as_uint(x.y) + (r1 & 0xfffffu), 0x7632u);
    return ((w << 4) & 0x7fff7fffu) | (w & 0x80008000u);
}
__device__ __forceinline__ uint32_t e5m2_halves(u64 x, uint32_t r0, uint32_t r1, int least) {      // (no sign)
    const int w0 = max((int)(__float_as_uint(x.x) + (r0 >> 11)), least), w1 = max((int)(__float_as_uint(x.y) + (r1 >> 11)), least);
    return __byte_perm((uint32_t)w0, (uint32_t)w1, 0x7632u) << 3;
}
// 2^-k 2^-120 resp. 2^-k 2^-112 for a scale byte k + 127; above these bytes the factor would leave fp32: part of it is taken
// off before
constexpr uint32_t M_BYTE_HIGH = 134, V_BYTE_HIGH = 142, M_PART = 115, V_PART = 100;
__device__ __forceinline__ float m_factor(uint32_t byte) { return __uint_as_float((M_BYTE_HIGH - byte) << 23); }
__device__ __forceinline__ float v_factor(uint32_t byte) { return __uint_as_float((V_BYTE_HIGH - byte) << 23); }

// Elements go in pairs through the packed fp32 instructions.  Moments: every product and sum is rounded by itself, as separate
// tensor operations round them, so that codes can be compared bit for bit (the scale is a power of two: scale * beta * code is
// beta * value).  m_keep, v_keep: beta * scale; group: index of the 8 elements in their tensor.
template <typename P, typename G, bool TINY_EPS>
__device__ __forceinline__ void block8_math(Result8& out, const uint32_t* pw, const uint32_t* gw, const uint4& codes, float m_beta, float v_beta,
                                            uint32_t group, const AdamwCoef& k) {
    const u64 m_keep = splat(m_beta), v_keep = splat(v_beta);
    const u64 c = splat(k.c), om1 = splat(k.om1), om2 = splat(k.om2);
    u64 m[4], v[4];
    float m_big = 0.0f, v_big = 0.0f;      // (a NaN does not count: it must not flush the rest of the block)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const u64 g = mul2(word_pair<G>(gw, j), c);
        m[j] = add2(mul2_rounded(e4m3_pair(j < 2 ? codes.x : codes.y, j & 1), m_keep), mul2_rounded(g, om1));
        v[j] = add2(mul2_rounded(e5m2_pair(j < 2 ? codes.z : codes.w, j & 1), v_keep), mul2_rounded(mul2(g, g), om2));
        m_big = max3(m_big, fabsf(m[j].x), fabsf(m[j].y));
        v_big = max3(v_big, v[j].x, v[j].y);
        const u64 root = TINY_EPS ? pk(approx_sqrt(v[j].x), approx_sqrt(v[j].y)) : pk(fast_sqrt(v[j].x), fast_sqrt(v[j].y));
        const u64 den = fma2(root, splat(k.root), splat(k.eps));
        const u64 q = TINY_EPS ? pk(__fdividef(m[j].x, den.x), __fdividef(m[j].y, den.y)) : mul2(m[j], pk(fast_rcp(den.x), fast_rcp(den.y)));
        const u64 old = word_pair<P>(pw, j), now = fma2(splat(-k.size), q, fma2(splat(-k.wd_lr), old, old));
        out.p[2 * j] = now.x;
        out.p[2 * j + 1] = now.y;
    }
    out.m_top = __reduce_max_sync(0xffffffffu, __float_as_uint(m_big));
    out.v_top = __reduce_max_sync(0xffffffffu, __float_as_uint(v_big));
    uint32_t m_byte = e8m0_scale<7>(out.m_top), v_byte = e8m0_scale<14>(out.v_top);
    if (m_byte >= M_BYTE_HIGH || v_byte >= V_BYTE_HIGH) {      // |m| from 2^14, v from 2^29 on
        const float m_part = m_byte >= M_BYTE_HIGH ? 0x1p-115f : 1.0f, v_part = v_byte >= V_BYTE_HIGH ? 0x1p-100f : 1.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            m[j] = __fmul2_rz(m[j], splat(m_part));      // (truncated twice is truncated once)
            v[j] = __fmul2_rz(pk(fminf(v[j].x, FLT_MAX), fminf(v[j].y, FLT_MAX)), splat(v_part));
        }
        if (m_byte >= M_BYTE_HIGH) m_byte -= M_PART;
        if (v_byte >= V_BYTE_HIGH) v_byte -= V_PART;
    }
    const u64 m_down = splat(m_factor(m_byte)), v_down = splat(v_factor(v_byte));
    const int least = out.v_top ? 1 << 21 : 0;      // v stays above zero (its root divides): at least 2^-16 after scaling; a block of zeros stays zero
    const uint32_t h = mix32(group + k.key);
    uint32_t r[8], mh[4], vh[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = h * (0x9E3779B1u * (2u * i + 1u));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        mh[j] = e4m3_halves(__fmul2_rz(m[j], m_down), r[2 * j], r[2 * j + 1]);
        vh[j] = e5m2_halves(__fmul2_rz(v[j], v_down), r[2 * j], r[2 * j + 1], least);
    }
    out.m = make_uint2(__byte_perm(mh[0], mh[1], 0x7531u), __byte_perm(mh[2], mh[3], 0x7531u));
    out.v = make_uint2(__byte_perm(vh[0], vh[1], 0x7531u), __byte_perm(vh[2], vh[3], 0x7531u));
}

// Scales of a warp's blocks: lane l holds those of block l
struct Scales8 {
    float m_beta, v_beta;       // old: beta * scale
    uint32_t m_top, v_top;      // new: bits of the largest magnitudes
};

// A block of any kind
template <typename P, typename G>
__device__ __forceinline__ void block8_step(uint8_t* slot, const Span8<P, G>& t, int b, int lane, uint32_t group, Scales8& sc,
                                            const AdamwCoef& k) {
    using R = Ring8<P, G>;
    const int at = b * BSTEP;
    const bool async = b >= t.async_lo && b < t.async_hi;
    uint32_t pw[2 * sizeof(P)], gw[2 * sizeof(G)];
    ring_read<G>(slot + R::G_OFF, async ? t.g_off : 0u, lane, gw);
    ring_read<P>(slot, async ? t.p_off : 0u, lane, pw);
    const uint4 codes = *reinterpret_cast<const uint4*>(slot + R::MV_OFF + lane * 16);
    Result8 r;
    const float m_beta = __shfl_sync(0xffffffffu, sc.m_beta, b), v_beta = __shfl_sync(0xffffffffu, sc.v_beta, b);
    if (k.eps < ADAMW8_LOST_ROOT * k.root) block8_math<P, G, true>(r, pw, gw, codes, m_beta, v_beta, group + BSTEP / 8 * b, k);
    else block8_math<P, G, false>(r, pw, gw, codes, m_beta, v_beta, group + BSTEP / 8 * b, k);
    if (lane == b) {
        sc.m_top = r.m_top;
        sc.v_top = r.v_top;
    }
    if (async) {
        *reinterpret_cast<uint2*>(t.m + at) = r.m;
        *reinterpret_cast<uint2*>(t.v + at) = r.v;
        if (t.p_off == 0 || (sizeof(P) == 2 && t.p_off == 16)) store8(t.p + at, r.p);
        else {      // through the slot: lanes next to each other write elements next to each other
            __syncwarp();      // (its parameters and gradients have been read)
            P* out = reinterpret_cast<P*>(slot);
            store_run<8>(out + 8 * lane, r.p);
            __syncwarp();
            P* to = t.p + at - 8 * lane;
#pragma unroll
            for (int i = 0; i < 8; ++i) to[32 * i + lane] = out[32 * i + lane];
            __syncwarp();
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (at + 8 * lane + i < t.left) {
            t.m[at + i] = (uint8_t)((i < 4 ? r.m.x : r.m.y) >> (8 * (i & 3)));
            t.v[at + i] = (uint8_t)((i < 4 ? r.v.x : r.v.y) >> (8 * (i & 3)));
            t.p[at + i] = from_f32<P>(r.p[i]);
        }
}

// Whole blocks of tensors on 32-byte boundaries, STAGES of them at a time (n a multiple of that): every place in the ring is
// known when this is compiled, and nothing is asked per block.  Returns with the ring empty.
template <typename P, typename G>
__device__ __forceinline__ void span8_fast(uint8_t* ring, Span8<P, G> t, int n, int lane, uint32_t group, Scales8& sc,
                                           const AdamwCoef& k) {
    using R = Ring8<P, G>;
    constexpr int S = R::STAGES;
    const uint8_t *p_from = reinterpret_cast<const uint8_t*>(t.p - 8 * lane) + 16 * lane, *g_from = reinterpret_cast<const uint8_t*>(t.g - 8 * lane) + 16 * lane;
    const uint8_t *m_from = t.m, *v_from = t.v;
    auto fetch = [&](int slot, int ahead) {      // the block `ahead` of the pointers
        uint8_t* to = ring + slot * R::BYTES;
#pragma unroll
        for (int i = 0; i < (int)sizeof(P) / 2; ++i) cp16(to + 512 * i + 16 * lane, p_from + ahead * BSTEP * (int)sizeof(P) + 512 * i, 16);
#pragma unroll
        for (int i = 0; i < (int)sizeof(G) / 2; ++i)
            cp16(to + R::G_OFF + 512 * i + 16 * lane, g_from + ahead * BSTEP * (int)sizeof(G) + 512 * i, 16);
        cp8(to + R::MV_OFF + lane * 16, m_from + ahead * BSTEP);
        cp8(to + R::MV_OFF + lane * 16 + 8, v_from + ahead * BSTEP);
    };
#pragma unroll
    for (int s = 0; s < S - 1; ++s) {
        fetch(s, s);
        cp_commit();
    }
    for (int b = 0; b < n; b += S) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
            __syncwarp();      // (the slot is filled again only after every lane has read what it held)
            if (s == 0 || b + S < n) fetch((s + S - 1) % S, s + S - 1);
            cp_commit();
            cp_wait<S - 1>();
            __syncwarp();
            const uint8_t* slot = ring + s * R::BYTES;
            uint32_t pw[2 * sizeof(P)], gw[2 * sizeof(G)];
            ring_read<G>(slot + R::G_OFF, 0u, lane, gw);
            ring_read<P>(slot, 0u, lane, pw);
            const uint4 codes = *reinterpret_cast<const uint4*>(slot + R::MV_OFF + lane * 16);
            Result8 r;
            block8_math<P, G, false>(r, pw, gw, codes, __shfl_sync(0xffffffffu, sc.m_beta, b + s), __shfl_sync(0xffffffffu, sc.v_beta, b + s),
                                     group + BSTEP / 8 * s, k);
            *reinterpret_cast<uint2*>(t.m + s * BSTEP) = r.m;
            *reinterpret_cast<uint2*>(t.v + s * BSTEP) = r.v;
            store8(t.p + s * BSTEP, r.p);
            if (lane == b + s) {
                sc.m_top = r.m_top;
                sc.v_top = r.v_top;
            }
        }
        p_from += S * BSTEP * (int)sizeof(P);
        g_from += S * BSTEP * (int)sizeof(G);
        m_from += S * BSTEP;
        v_from += S * BSTEP;
        t.p += S * BSTEP;
        t.m += S * BSTEP;
        t.v += S * BSTEP;
        group += BSTEP / 8 * S;
    }
    __syncwarp();
}

template <typename P, typename G>
__global__ void __launch_bounds__(ADAMW_THREADS, ADAMW8_CTAS) k_adamw8(const StepArgs a, const AdamwArgs w, const __grid_constant__ AdamwHyp by_value) {
    using R = Ring8<P, G>;
    extern __shared__ __align__(128) uint8_t ring_all[];
    const int lane = threadIdx.x & 31;
    uint8_t* ring = ring_all + (threadIdx.x >> 5) * (R::BYTES * R::STAGES);
    const CameHyper* hyp = w.by_value ? by_value.h : a.hyp;
    griddep_wait();
    double norm;
    if (!adamw_norm(w, &norm)) return;      // (in every CTA, and before anything is written)
    AdamwCache cache;
    cache.step = -1.0f;
    cache.group = -1;
    const int warp = threadIdx.x >> 5;
    for_runs(a, w, [&](const CameTensorDesc& d, int tensor, int64_t lo, int64_t hi, int64_t n) {
        const int64_t first = lo / QBLOCK + warp, at = first * QBLOCK + 8 * lane;
        const int blocks = (int)((hi + QBLOCK - 1) / QBLOCK - first + ADAMW_WARPS - 1) / ADAMW_WARPS;      // this warp's
        uint8_t *m_scale = reinterpret_cast<uint8_t*>(d.m_absmax) + first, *v_scale = reinterpret_cast<uint8_t*>(d.sq_row_absmax) + first;
        Span8<P, G> t{static_cast<P*>(d.p) + at, static_cast<const G*>(d.g) + at, static_cast<uint8_t*>(d.m) + at, static_cast<uint8_t*>(d.sq_row) + at,
                      n - first * QBLOCK, (uint32_t)(reinterpret_cast<uintptr_t>(d.p) & 31u), (uint32_t)(reinterpret_cast<uintptr_t>(d.g) & 31u), 0, 0};
        const bool shifted = (t.p_off | t.g_off) != 0;
        t.async_lo = shifted && first == 0 ? 1 : 0;
        const int64_t sure = t.left - (shifted ? 8 : 0) - QBLOCK;      // the last place where a block can start
        if (a.scr[tensor].g_v == 8 && sure >= 0) t.async_hi = (int)min((int64_t)blocks, sure / BSTEP + 1);
        uint32_t ms = 0u, vs = 0u;
        if (lane < blocks) {
            ms = m_scale[lane * ADAMW_WARPS];
            vs = v_scale[lane * ADAMW_WARPS];
        }
        adamw_coef(cache, d, hyp, w.norm_parts != nullptr, norm);
        Scales8 sc{cache.k.b1 * e8m0_value(ms), cache.k.b2 * e8m0_value(vs), 0u, 0u};
        const uint32_t group = (uint32_t)(at >> 3);
        int b = 0;
        if (!shifted && cache.k.eps >= ADAMW8_LOST_ROOT * cache.k.root && t.async_hi >= R::STAGES) {
            b = t.async_hi / R::STAGES * R::STAGES;
            span8_fast(ring, t, b, lane, group, sc, cache.k);
        }
#pragma unroll
        for (int s = 0; s < R::STAGES - 1; ++s) {
            if (b + s < blocks) block8_fetch(ring + s * R::BYTES, t, b + s, lane);
            cp_commit();
        }
        uint8_t *slot = ring, *ahead = ring + (R::STAGES - 1) * R::BYTES;
        for (; b < blocks; ++b) {
            // (a slot is filled again only after every lane has read what it held)
            __syncwarp();
            if (b + R::STAGES - 1 < blocks) block8_fetch(ahead, t, b + R::STAGES - 1, lane);
            cp_commit();
            cp_wait<R::STAGES - 1>();
            __syncwarp();
            block8_step(slot, t, b, lane, group, sc, cache.k);
            ahead = slot;
            slot = slot == ring + (R::STAGES - 1) * R::BYTES ? ring : slot + R::BYTES;
        }
        __syncwarp();
        if (lane < blocks) {
            m_scale[lane * ADAMW_WARPS] = (uint8_t)e8m0_scale<7>(sc.m_top);
            v_scale[lane * ADAMW_WARPS] = (uint8_t)e8m0_scale<14>(sc.v_top);
        }
    });
    griddep_launch();
    adamw_count_step(w);
}

template <typename P, typename G> struct LaunchAdamw8 {
    static cudaError_t run(const StepArgs& a, const AdamwArgs& w, const AdamwHyp& h, cudaStream_t st) {
        constexpr int smem = Ring8<P, G>::CTA_BYTES;
        const cudaError_t e = cudaFuncSetAttribute(k_adamw8<P, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        // Spans (256 M elements): 16-bit types are bound by instructions, a long span fills its ring less often (404 us with 16
        // items, 426 with 8, 509 with 4); fp32 is bound by DRAM, which likes addresses close together (683, 661, 642).
        AdamwArgs x = w;
        const int grid = adamw_spans(x, ADAMW8_CTAS, sizeof(P) + sizeof(G) <= 4 ? 16 : 4);
        return launch_behind(k_adamw8<P, G>, grid, ADAMW_THREADS, smem, st, a, x, h);
    }
};

cudaError_t launch_adamw8(const KernelKey& key, const StepArgs& a, const AdamwArgs& w, const AdamwHyp& h, cudaStream_t st) {
    return adamw_for<LaunchAdamw8>(key, a, w, h, st);
}

}  // namespace came
