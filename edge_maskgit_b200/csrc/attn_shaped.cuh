// attn_shaped.cuh -- what the two kernels of mgc_attention share: their arguments, the shaping of
// a score, which keys a query sees, and the exact row that repairs a NaN.
#pragma once
#include <cstdint>

#include "../../include/mgc.h"
#include "kernels.h"
#include "tma.cuh"

namespace mgc {

constexpr float ATTN_LOG2E = 1.4426950408889634f;

// The call, as the kernels get it.  Partial results (nsplit > 1), per split and row
// (b * Sq + i) * Hq + h: the unnormalised output f32 [D], then (row max in base 2, sum).
struct AttnCall {
    mgc_attention_args a;
    int g;                 // query heads per key head
    int nsplit, chunk;     // splits of the key range; keys per split (a multiple of the key tile)
    int cluster;           // few queries: the splits are one cluster, joined in distributed shared memory
    int wide;              // few queries: eight warps a block instead of four
    float* opart;
    float2* mlpart;
};

// Per-head constants of a score in the base-2 domain: t = s * log2 e.
struct ScoreShape {
    float c1;      // no cap: scale * log2 e; cap: scale / cap * 2 log2 e (the exponent of tanh)
    float cap2;    // cap * log2 e, 0 = none
    float slope2;  // slope * log2 e
    const float* table;   // + distance -dist_range..dist_range, or null
    int range;
};
__device__ __forceinline__ ScoreShape score_shape(const mgc_attention_args& a, int h) {
    ScoreShape s;
    s.cap2 = a.cap * ATTN_LOG2E;
    s.c1 = a.cap > 0.0f ? a.scale / a.cap * (2.0f * ATTN_LOG2E) : a.scale * ATTN_LOG2E;
    s.slope2 = a.slopes ? __ldg(a.slopes + h) * ATTN_LOG2E : 0.0f;
    s.range = a.dist_range;
    s.table = a.dist_bias ? a.dist_bias + (long long)h * (2LL * a.dist_range + 1) + a.dist_range : nullptr;
    return s;
}
// A bias in the base-2 domain.  The product with log2 e must not turn the lowest finite value into
// -inf: a -inf score hides its key, a finite one does not.
__device__ __forceinline__ float bias2(float b) {
    const float t = b * ATTN_LOG2E;
    return t == -INFINITY && b != -INFINITY ? -3.402823466e38f : t;
}
// cap * tanh(x / cap) in base 2, tanh(u) = 1 - 2 / (1 + e^2u): its absolute error (a few 2^-24
// times cap2) is an error of that size in the exponent of p.  The approximate tanh instruction
// (2^-11) would put percents on p at a cap of 50.
__device__ __forceinline__ float capped(float s, float c1, float cap2) {
    const float e = ex2_approx(s * c1);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return fmaf(-2.0f * cap2, r, cap2);
}
__device__ __forceinline__ float shaped(float s, const ScoreShape& f, int dist, int slope_dist) {
    float t = f.cap2 > 0.0f ? capped(s, f.c1, f.cap2) : s * f.c1;
    t = fmaf(-f.slope2, fabsf((float)slope_dist), t);
    if (f.table) t += bias2(__ldg(f.table + max(-f.range, min(f.range, dist))));
    return t;
}

// Positions and bounds of batch row b.
struct RowBounds { int len, pos0, prefix; };
__device__ __forceinline__ RowBounds row_bounds(const mgc_attention_args& a, int b) {
    RowBounds r;
    r.len = a.k_len ? max(0, min(a.Sk, __ldg(a.k_len + b))) : a.Sk;
    r.pos0 = a.q_pos ? max(-(1 << 29), min(1 << 29, __ldg(a.q_pos + b))) : a.Sk - a.Sq;
    r.prefix = a.causal ? (a.prefix ? max(0, __ldg(a.prefix + b)) : 0) : a.Sk;
    return r;
}
// Key j is seen by a query at position p (documents apart) iff j < key_end(p): below the row's
// length, and causally at most p or inside the prefix (not causal: prefix = Sk).
__device__ __forceinline__ int key_end(const RowBounds& r, int p) { return min(r.len, max(p + 1, r.prefix)); }

// The position that slopes count distances from.  A query before the first or behind the last key has the same
// -slope |p - nearest key| in all its scores, which the softmax does not see: counted from the nearest key,
// the distances that differ keep their bits, however far the query is.
__device__ __forceinline__ int slope_pos(const RowBounds& r, int p) { return max(0, min(p, r.len - 1)); }

// A result that the row may not have: NaN, or in bf16 an infinity (values up to 2^127 can pass the
// largest float in a sum of unnormalised products; f16's cannot).
template <bool BF16>
__device__ __forceinline__ bool suspect(float x) { return BF16 ? !isfinite(x) : isnan(x); }
// One row, exactly as the formulas have it, touching seen keys only, by one warp; o = this lane's
// dims d = lane + 32 u.  The kernels multiply a whole tile of v by probabilities that are 0 at
// unseen keys; a NaN or infinity that v holds there turns the row into NaN.  A row with a suspect
// result is therefore recomputed here: it stays NaN or infinite if a seen key made it so.  o is the
// average so far, not a sum, so it never exceeds the largest value.
template <bool BF16>
__device__ __noinline__ void exact_row(const mgc_attention_args& a, int g, int b, int h, int i, float (&o)[4]) {
    const int lane = threadIdx.x & 31;
    const RowBounds rb = row_bounds(a, b);
    const ScoreShape sh = score_shape(a, h);
    const int p = rb.pos0 + i, ps = slope_pos(rb, p), end = key_end(rb, p);
    const long long hk = h / g;
    const long long qo = b * a.q_stride[0] + i * a.q_stride[1] + h * a.q_stride[2];
    const long long ko = b * a.k_stride[0] + hk * a.k_stride[2], vo = b * a.v_stride[0] + hk * a.v_stride[2];
    const int doc = a.doc_q ? __ldg(a.doc_q + (long long)b * a.Sq + i) : 0;
    float m = -INFINITY, l = 0.0f;
    for (int u = 0; u < 4; u++) o[u] = 0.0f;
    for (int j0 = 0; j0 < end; j0 += 32) {
        const int j = j0 + lane;
        float t = -INFINITY;
        if (j < end && (!a.doc_q || (doc >= 0 && __ldg(a.doc_k + (long long)b * a.Sk + j) == doc))) {
            float s = 0.0f;
            for (int d = 0; d < a.D; d++) s = fmaf(load16<BF16>(a.q, qo + d), load16<BF16>(a.k, ko + j * a.k_stride[1] + d), s);
            t = shaped(s, sh, j - p, j - ps);
        }
        float mx = t;   // NaN scores reach l through ex2
        for (int k = 16; k; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
        const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.0f : mn;
        const float alpha = ex2_approx(m - base), pj = ex2_approx(t - base);
        const unsigned seen = __ballot_sync(0xffffffffu, !(t == -INFINITY));
        float ls = pj;
        for (int k = 16; k; k >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, k);
        const float before = l * alpha;
        l = before + ls;
        m = mn;
        if (l == 0.0f) continue;   // nothing seen yet
        const float inv = 1.0f / l;
        for (int u = 0; u < 4; u++) o[u] *= before * inv;
        for (int k = 0; k < 32; k++) {
            if (!(seen >> k & 1)) continue;
            const float pk = __shfl_sync(0xffffffffu, pj, k) * inv;
            for (int u = 0; u < 4; u++) {
                const int d = lane + 32 * u;
                if (d < a.D) o[u] = fmaf(pk, load16<BF16>(a.v, vo + (j0 + k) * a.v_stride[1] + d), o[u]);
            }
        }
    }
}

// Launches of the two kernels; the caller has checked the arguments.
void launch_attn_step(const AttnCall& c, cudaStream_t st);
void launch_attn_combine(const AttnCall& c, cudaStream_t st);

}  // namespace mgc
