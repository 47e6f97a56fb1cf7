// attn_shaped.cuh -- what the two kernels of mgc_attention share: their arguments, the shaping of
// a score, which keys a query sees, and the repair of a row whose result is NaN.
#pragma once
#include <cstdint>

#include "../../include/mgc.h"
#include "kernels.h"
#include "tma.cuh"

namespace mgc {

constexpr float ATTN_LOG2E = 1.4426950408889634f;

// The call, as the kernels get it.  Partial results (nsplit > 1), per split and row
// (b * Sq + i) * Hq + h: the unnormalised output f32 [D], then (base, sum): probabilities are 2^(t - base).
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
// Is key j, at a position below the row's end, of the query's document?
__device__ __forceinline__ bool same_doc(const mgc_attention_args& a, int b, int j, int doc) {
    return !a.doc_q || (doc >= 0 && __ldg(a.doc_k + (long long)b * a.Sk + j) == doc);
}
template <bool BF16>
__device__ __forceinline__ float4 load4(const void* p, long long at) {   // 8-byte aligned
    const uint2 x = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + at);
    const float2 lo = unpack16<BF16>(x.x), hi = unpack16<BF16>(x.y);
    return make_float4(lo.x, lo.y, hi.x, hi.y);
}

// Puts right the suspect results of one row that is in `out` already, by one warp; lane = dims 4 lane ..
// 4 lane + 3.  The kernels multiply a whole tile of v by probabilities that are 0 at unseen keys, so a NaN
// or infinity that v holds there makes a result NaN; each dim on its own, so the others are right.  (A row
// whose sum of probabilities is NaN has a NaN or infinite score at a key that it sees: all of it is NaN, and
// the caller leaves it.)
// First, what a suspect dim sees: a NaN, or infinities of both signs, and it is NaN; of one sign, and it is that
// infinity.  That takes a look at v, up to the first NaN, and is the usual case (one bad token makes every row behind it
// NaN: 1 x 4096, 32 heads of 128 over 8, computing those again took 350 ms).  What sees finite values only is computed
// again from the formulas, over seen keys, as an average so far and not a sum, so that it never exceeds the
// largest value.
template <bool BF16>
__device__ __noinline__ void repair_row(const mgc_attention_args& a, int g, int b, int h, int i) {
    constexpr unsigned ALL = 0xffffffffu;
    const int lane = threadIdx.x & 31, d0 = lane * 4;
    const bool dims = d0 < a.D;
    const RowBounds rb = row_bounds(a, b);
    const ScoreShape sh = score_shape(a, h);
    const int p = rb.pos0 + i, ps = slope_pos(rb, p), end = key_end(rb, p);
    const long long hk = h / g;
    const long long qo = b * a.q_stride[0] + i * a.q_stride[1] + h * a.q_stride[2];
    const long long ko = b * a.k_stride[0] + hk * a.k_stride[2], vo = b * a.v_stride[0] + hk * a.v_stride[2];
    const long long oo = b * a.out_stride[0] + i * a.out_stride[1] + h * a.out_stride[2];
    const int doc = a.doc_q ? __ldg(a.doc_q + (long long)b * a.Sq + i) : 0;
    float4 r = dims ? load4<BF16>(a.out, oo + d0) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float* rv = &r.x;
    unsigned bad = 0, nan = 0, pos = 0, neg = 0;   // bits: this lane's four dims
#pragma unroll
    for (int e = 0; e < 4; e++) bad |= suspect<BF16>(rv[e]) ? 1u << e : 0u;

    constexpr int AHEAD = 16;   // keys whose v is in flight
    for (int j0 = 0; j0 < end && __any_sync(ALL, bad & ~nan); j0 += AHEAD) {
        uint2 x[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            x[u] = make_uint2(0, 0);
            if (dims && j0 + u < end)
                x[u] = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(a.v) + vo + (j0 + u) * a.v_stride[1] + d0);
        }
        unsigned odd = 0;   // bits: keys with a value that is not finite in a suspect dim
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            const float2 lo = unpack16<BF16>(x[u].x), hi = unpack16<BF16>(x[u].y);
            const float f[4] = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
            for (int e = 0; e < 4; e++) odd |= (bad >> e & 1) && !isfinite(f[e]) ? 1u << u : 0u;
        }
        odd = __reduce_or_sync(ALL, odd);
        while (odd) {
            const int j = j0 + __ffs(odd) - 1;
            odd &= odd - 1;
            if (!same_doc(a, b, j, doc)) continue;
            float s = 0.0f;   // a key whose score is -inf is not seen
            if (dims) {
                const float4 x4 = load4<BF16>(a.q, qo + d0), y4 = load4<BF16>(a.k, ko + j * a.k_stride[1] + d0);
                s = fmaf(x4.w, y4.w, fmaf(x4.z, y4.z, fmaf(x4.y, y4.y, x4.x * y4.x)));
            }
            for (int k = 16; k; k >>= 1) s += __shfl_xor_sync(ALL, s, k);
            if (shaped(s, sh, j - p, j - ps) == -INFINITY) continue;
            if (dims) {
                const float4 f4 = load4<BF16>(a.v, vo + j * a.v_stride[1] + d0);
                const float f[4] = {f4.x, f4.y, f4.z, f4.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    nan |= isnan(f[e]) ? 1u << e : 0u;
                    pos |= f[e] == INFINITY ? 1u << e : 0u;
                    neg |= f[e] == -INFINITY ? 1u << e : 0u;
                }
            }
        }
    }
    nan |= pos & neg;
    const unsigned again = bad & ~(nan | pos | neg);
    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (__any_sync(ALL, again)) {
        float m = -INFINITY, l = 0.0f;
        for (int j0 = 0; j0 < end; j0 += 32) {
            const int j = j0 + lane;
            float t = -INFINITY;
            if (j < end && same_doc(a, b, j, doc)) {
                float s = 0.0f;
                for (int d = 0; d < a.D; d += 4) {
                    const float4 x4 = load4<BF16>(a.q, qo + d), y4 = load4<BF16>(a.k, ko + j * a.k_stride[1] + d);
                    s = fmaf(x4.w, y4.w, fmaf(x4.z, y4.z, fmaf(x4.y, y4.y, fmaf(x4.x, y4.x, s))));
                }
                t = shaped(s, sh, j - p, j - ps);
            }
            float mx = t;
            for (int k = 16; k; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(ALL, mx, k));
            const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.0f : mn;
            const float alpha = ex2_approx(m - base), pj = ex2_approx(t - base);
            const unsigned seen = __ballot_sync(ALL, !(t == -INFINITY));
            float ls = pj;
            for (int k = 16; k; k >>= 1) ls += __shfl_xor_sync(ALL, ls, k);
            const float before = l * alpha;
            l = before + ls;
            m = mn;
            if (l == 0.0f) continue;   // nothing seen yet
            const float inv = 1.0f / l;
            for (int e = 0; e < 4; e++) o[e] *= before * inv;
            for (int k = 0; k < 32; k++) {
                if (!(seen >> k & 1)) continue;
                const float pk = __shfl_sync(ALL, pj, k) * inv;
                if (dims) {
                    const float4 f = load4<BF16>(a.v, vo + (j0 + k) * a.v_stride[1] + d0);
                    o[0] = fmaf(pk, f.x, o[0]); o[1] = fmaf(pk, f.y, o[1]);
                    o[2] = fmaf(pk, f.z, o[2]); o[3] = fmaf(pk, f.w, o[3]);
                }
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (bad >> e & 1)
            store16<BF16>(a.out, oo + d0 + e, nan >> e & 1 ? NAN : pos >> e & 1 ? INFINITY : neg >> e & 1 ? -INFINITY : o[e]);
}

// Launches of the two kernels; the caller has checked the arguments.
void launch_attn_step(const AttnCall& c, cudaStream_t st);
void launch_attn_combine(const AttnCall& c, cudaStream_t st);

}  // namespace mgc
