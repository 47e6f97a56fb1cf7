// attn_step.cu -- mgc_attention for few queries against long keys (a decode step), and the join of
// split key ranges.
//
// Bound by the bytes of k and v, which are read once: the Sq * (Hq / Hkv) query rows that share a
// key head sit in one 16-row tensor-core tile (mma.sync m16n8k16; with 16 rows or fewer per key the
// tile is memory-bound by an order of magnitude, so the tcgen05 path with its 128-row tile would
// add nothing).  The key range is split over CTAs, and inside a CTA over four or eight warps.  Each warp has
// its own ring of 16-key stages filled by cp.async, so the main loop has no CTA-wide barrier; the
// online softmax keeps (max, sum, output) in registers, and warps and CTAs are joined at the end: up to
// 8 CTAs are one cluster and join in distributed shared memory, more leave partial results in the
// workspace for a second kernel.
#include <stdexcept>

#include "attn_shaped.cuh"

namespace mgc {
namespace {

constexpr int KT = 16, STAGES = 3;
template <int DP> constexpr int row_bytes() { return DP * 2 + 16; }   // odd in 16-byte units: ldmatrix without conflicts
template <int DP> constexpr int stage_bytes() { return 2 * KT * row_bytes<DP>(); }
template <int DP, int WARPS> constexpr int ring_bytes() { return WARPS * STAGES * stage_bytes<DP>(); }
template <int DP> constexpr int join_row() { return DP + 8; }   // floats: eight rows' writes meet no bank twice
template <int DP, int WARPS> constexpr int join_bytes() { return WARPS * 16 * (join_row<DP>() * 4 + 8); }
template <int DP> constexpr int part_bytes() { return 16 * (DP * 4 + 8); }   // a CTA's own result, for its cluster
template <int DP, int WARPS> constexpr int smem_bytes() {
    constexpr int ring = ring_bytes<DP, WARPS>(), join = join_bytes<DP, WARPS>() + part_bytes<DP>();
    return ring > join ? ring : join;
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// 16 bytes global -> shared, or zeros
__device__ __forceinline__ void cp16_or_zero(uint32_t dst, const void* src, bool copy) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(copy ? 16 : 0) : "memory");
}

// Writes one finished row (o = dims lane + 32 u, l their sum of probabilities), and puts suspect results right.
template <bool BF16>
__device__ __forceinline__ void write_row(const AttnCall& c, int b, int h, int i, const float (&o)[4], float l) {
    const int lane = threadIdx.x & 31;
    const long long at = b * c.a.out_stride[0] + i * c.a.out_stride[1] + h * c.a.out_stride[2];
    bool bad = false;
#pragma unroll
    for (int u = 0; u < 4; u++) {
        if (lane + 32 * u >= c.a.D) continue;
        bad |= suspect<BF16>(o[u]);
        store16<BF16>(c.a.out, at + lane + 32 * u, o[u]);
    }
    if (__any_sync(0xffffffffu, bad) && !isnan(l)) {
        __syncwarp();
        repair_row<BF16>(c.a, c.g, b, h, i);
    }
}

// The same from sums of unnormalised values: o = dims 4 lane .. 4 lane + 3.
template <bool BF16>
__device__ __forceinline__ void write_row4(const AttnCall& c, int b, int h, int i, float4 o, float l) {
    const int lane = threadIdx.x & 31;
    const bool dims = lane * 4 < c.a.D;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t* dst = reinterpret_cast<uint16_t*>(c.a.out) + b * c.a.out_stride[0] + i * c.a.out_stride[1] + h * c.a.out_stride[2];
    if (dims) reinterpret_cast<uint2*>(dst)[lane] = make_uint2(pack16<BF16>(o.x * inv, o.y * inv), pack16<BF16>(o.z * inv, o.w * inv));
    const bool bad = dims && (suspect<BF16>(o.x) || suspect<BF16>(o.y) || suspect<BF16>(o.z) || suspect<BF16>(o.w));
    if (__any_sync(0xffffffffu, bad) && !isnan(l)) {
        __syncwarp();
        repair_row<BF16>(c.a, c.g, b, h, i);
    }
}

// grid: splits x (batch row, key head, 16-row block), splits fastest
template <bool BF16, int DP, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) attn_step_kernel(const __grid_constant__ AttnCall c) {
    constexpr int RB = row_bytes<DP>(), SB = stage_bytes<DP>(), NK = DP / 16, CH = DP / 8;
    // Probabilities are 2^(t - base), with the base LIFT below the row's maximum.  In f16 they then go up to
    // 2^15, and those that are 2^-29 of the largest still have all their bits (a sum of many small ones behind
    // one large is right); bf16 needs no lift.  m below is this base.
    constexpr int LIFT = BF16 ? 0 : 15;
    extern __shared__ __align__(16) uint8_t smem[];
    griddep_wait();
    griddep_launch();
    const mgc_attention_args& a = c.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, qr = lane >> 2, qc = (lane & 3) * 2;
    const unsigned blocks = (unsigned)(a.Sq * c.g + 15) / 16;
    unsigned rest = blockIdx.x / (unsigned)c.nsplit;
    const int rows = a.Sq * c.g, split = (int)(blockIdx.x - rest * c.nsplit);
    const int blk = (int)(rest % blocks); rest /= blocks;
    const int hk = (int)(rest % (unsigned)a.Hkv), b = (int)(rest / (unsigned)a.Hkv);
    const RowBounds rb = row_bounds(a, b);

    // rows of this lane's fragments: blk * 16 + qr and + 8; row = query i * g + (h - hk * g)
    int row[2], qi[2], head[2], doc[2], end[2], pos[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
        row[u] = blk * 16 + qr + 8 * u;
        const int rr = min(row[u], rows - 1);
        qi[u] = rr / c.g;
        head[u] = hk * c.g + (rr - qi[u] * c.g);
        pos[u] = rb.pos0 + qi[u];
        doc[u] = a.doc_q ? __ldg(a.doc_q + (long long)b * a.Sq + qi[u]) : 0;
        end[u] = row[u] < rows && doc[u] >= 0 ? key_end(rb, pos[u]) : 0;
    }
    uint32_t qf[NK][4];
#pragma unroll
    for (int k = 0; k < NK; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int u = e & 1, d = k * 16 + qc + (e >> 1) * 8;
            const long long at = b * a.q_stride[0] + qi[u] * a.q_stride[1] + head[u] * a.q_stride[2] + d;
            qf[k][e] = d < a.D ? __ldg(reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint16_t*>(a.q) + at)) : 0u;
        }

    // this CTA's keys: the split's chunk, cut to what the block's last query sees
    const int last_q = min(blk * 16 + 15, rows - 1) / c.g;
    const int k_lo = split * c.chunk, k_hi = min(k_lo + c.chunk, key_end(rb, rb.pos0 + last_q));
    const int tiles = k_hi > k_lo ? (k_hi - k_lo + KT - 1) / KT : 0;
    const uint16_t* kp = reinterpret_cast<const uint16_t*>(a.k) + b * a.k_stride[0] + hk * a.k_stride[2];
    const uint16_t* vp = reinterpret_cast<const uint16_t*>(a.v) + b * a.v_stride[0] + hk * a.v_stride[2];
    const uint32_t ring = smem_u32(smem) + warp * STAGES * SB;
    const int mine = tiles > warp ? (tiles - warp + WARPS - 1) / WARPS : 0;   // tiles warp, warp + 4, ...

    const int ks = (int)a.k_stride[1], vs = (int)a.v_stride[1];   // (below 2^31: checked)
    auto load = [&](int n) {   // stage n % STAGES <- the warp's n-th tile; keys past the end read as zeros
        if (n < mine) {
            const int j0 = k_lo + (warp + n * WARPS) * KT;
            const uint32_t s = ring + (n % STAGES) * SB;
            const uint16_t* kt = kp + (long long)j0 * ks;
            const uint16_t* vt = vp + (long long)j0 * vs;
            if (a.D == DP && j0 + KT <= k_hi) {
#pragma unroll
                for (int i = 0; i < KT * CH / 32; i++) {
                    const int x = lane + 32 * i, r = x / CH, ch = x % CH;
                    cp16(s + r * RB + ch * 16, kt + (long long)r * ks + ch * 8);
                    cp16(s + KT * RB + r * RB + ch * 16, vt + (long long)r * vs + ch * 8);
                }
            } else {
#pragma unroll 1
                for (int x = lane; x < KT * CH; x += 32) {
                    const int r = x / CH, ch = x % CH;
                    const bool in = j0 + r < k_hi && ch * 8 < a.D;
                    cp16_or_zero(s + r * RB + ch * 16, in ? kt + (long long)r * ks + ch * 8 : kp, in);
                    cp16_or_zero(s + KT * RB + r * RB + ch * 16, in ? vt + (long long)r * vs + ch * 8 : vp, in);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // score constants of the two rows (ScoreShape, branches on the call's own values only)
    const ScoreShape s0 = score_shape(a, head[0]), s1 = score_shape(a, head[1]);
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[DP / 8][4];
#pragma unroll
    for (int d = 0; d < DP / 8; d++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[d][e] = 0.0f;
    for (int n = 0; n < STAGES - 1; n++) load(n);
    for (int n = 0; n < mine; n++) {
        load(n + STAGES - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        __syncwarp();
        const uint32_t s = ring + (n % STAGES) * SB;
        const int j0 = k_lo + (warp + n * WARPS) * KT;
        float sc[2][4] = {};
#pragma unroll
        for (int k = 0; k < NK; k++) {
            uint32_t kf[4];   // keys 0-7 and 8-15, d halves
            ldsm4(kf, s + (lane & 15) * RB + k * 32 + (lane >> 4) * 16);
            mma16816<BF16>(sc[0], qf[k], kf[0], kf[2]);
            mma16816<BF16>(sc[1], qf[k], kf[1], kf[3]);
        }
        // ---- shape; one branch for all eight scores at a time
        auto each = [&](auto f) {   // f(score, row 0 / 1, key)
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) f(sc[t][e], e >> 1, j0 + t * 8 + qc + (e & 1));
        };
        if (a.cap > 0.0f) each([&](float& x, int, int) { x = capped(x, s0.c1, s0.cap2); });
        else each([&](float& x, int, int) { x *= s0.c1; });
        if (a.slopes)
            each([&](float& x, int u, int j) {
                x = fmaf(u ? -s1.slope2 : -s0.slope2, fabsf((float)(j - slope_pos(rb, pos[u]))), x);
            });
        if (a.dist_bias)
            each([&](float& x, int u, int j) {
                x += bias2(__ldg((u ? s1.table : s0.table) + max(-s0.range, min(s0.range, j - pos[u]))));
            });
        if (a.doc_k)
            each([&](float& x, int u, int j) {
                if (__ldg(a.doc_k + (long long)b * a.Sk + min(j, a.Sk - 1)) != doc[u]) x = -INFINITY;
            });
        float mx[2] = {-INFINITY, -INFINITY};
        each([&](float& x, int u, int j) {
            x = j < end[u] ? x : -INFINITY;
            mx[u] = fmaxf(mx[u], x);
        });
        float alpha[2], base[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 1));
            mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 2));
            // (rounded up: p never passes 2^LIFT)
            const float mn = fmaxf(m[u], LIFT ? __fadd_ru(mx[u], -(float)LIFT) : mx[u]);
            base[u] = mn == -INFINITY ? 0.0f : mn;   // nothing seen yet: p = 2^-inf = 0
            alpha[u] = ex2_approx(m[u] - base[u]);
            m[u] = mn;
        }
        uint32_t pf[4];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            float p[4];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int e = 0; e < 2; e++) p[t * 2 + e] = ex2_approx(sc[t][u * 2 + e] - base[u]);
            l[u] = l[u] * alpha[u] + ((p[0] + p[1]) + (p[2] + p[3]));
            pf[u] = pack16<BF16>(p[0], p[1]);       // rounded to the type of v: what tensor cores multiply
            pf[u + 2] = pack16<BF16>(p[2], p[3]);
        }
        if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
            for (int d = 0; d < DP / 8; d++) {
                o[d][0] *= alpha[0]; o[d][1] *= alpha[0];
                o[d][2] *= alpha[1]; o[d][3] *= alpha[1];
            }
        }
        const uint32_t sv = s + KT * RB;
#pragma unroll
        for (int k = 0; k < NK; k++) {
            uint32_t vf[4];   // keys 0-7 / 8-15 of dims 16 k .. 16 k + 7, then of the next 8 dims
            ldsm4t(vf, sv + (lane & 15) * RB + k * 32 + (lane >> 4) * 16);
            mma16816<BF16>(o[2 * k], pf, vf[0], vf[1]);
            mma16816<BF16>(o[2 * k + 1], pf, vf[2], vf[3]);
        }
        __syncwarp();   // the stage is read before the next round refills it
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();   // the ring is free: join the warps through it
    constexpr int JR = join_row<DP>();
    float* so = reinterpret_cast<float*>(smem);                    // [WARPS][16][JR]
    float2* sml = reinterpret_cast<float2*>(so + WARPS * 16 * JR);  // [WARPS][16]
#pragma unroll
    for (int u = 0; u < 2; u++) {
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
        if ((lane & 3) == 0) sml[warp * 16 + qr + 8 * u] = make_float2(m[u], l[u]);
        if (row[u] >= rows) continue;
#pragma unroll
        for (int d = 0; d < DP / 8; d++)
            *reinterpret_cast<float2*>(so + (warp * 16 + qr + 8 * u) * JR + d * 8 + qc) = make_float2(o[d][2 * u], o[d][2 * u + 1]);
    }
    float* po = reinterpret_cast<float*>(smem + join_bytes<DP, WARPS>());   // [16][DP]
    float2* pml = reinterpret_cast<float2*>(po + 16 * DP);            // [16]
    __syncthreads();
    for (int r = warp; r < 16 && blk * 16 + r < rows; r += WARPS) {
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; w++) mm = fmaxf(mm, sml[w * 16 + r].x);
        const float base = mm == -INFINITY ? 0.0f : mm;
        float ll = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            const float2 ml = sml[w * 16 + r];
            const float f = ex2_approx(ml.x - base);
            ll += ml.y * f;
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (lane + 32 * u < DP) acc[u] += so[(w * 16 + r) * JR + lane + 32 * u] * f;
        }
        const int gr = blk * 16 + r, i = gr / c.g, h = hk * c.g + gr % c.g;
        if (c.cluster) {
            if (lane == 0) pml[r] = make_float2(mm, ll);
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (lane + 32 * u < DP) po[r * DP + lane + 32 * u] = acc[u];
        } else if (c.nsplit == 1) {
            const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
#pragma unroll
            for (int u = 0; u < 4; u++) acc[u] = ll == 0.0f ? 0.0f : acc[u] * inv;
            write_row<BF16>(c, b, h, i, acc, ll);
        } else {
            const long long all = (long long)a.B * a.Sq * a.Hq;
            const long long id = split * all + ((long long)b * a.Sq + i) * a.Hq + h;
            if (lane == 0) c.mlpart[id] = make_float2(mm, ll);
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (lane + 32 * u < a.D) c.opart[id * a.D + lane + 32 * u] = acc[u];
        }
    }
    if (!c.cluster) return;
    __syncwarp();
    cluster_sync_all();
    for (int r = warp * c.nsplit + split; r < 16 && blk * 16 + r < rows; r += WARPS * c.nsplit) {   // this CTA's rows
        float2 ml = make_float2(-INFINITY, 0.0f);   // lane = split
        if (lane < c.nsplit) {
            const uint32_t at = mapa_u32(pml + r, lane);
            asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(ml.x), "=f"(ml.y) : "r"(at) : "memory");
        }
        float mm = ml.x;
        for (int k = 16; k; k >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, k));
        const float f = ex2_approx(ml.x - (mm == -INFINITY ? 0.0f : mm));
        float ll = ml.y * f;
        for (int k = 16; k; k >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, k);
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);   // dims 4 lane ..
        const bool dims = lane * 4 < DP;
#pragma unroll
        for (int p = 0; p < 8; p++) {   // all remote reads in flight
            if (p >= c.nsplit) break;
            const float w = __shfl_sync(0xffffffffu, f, p);
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (dims)
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                             : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(mapa_u32(po + r * DP + lane * 4, p)) : "memory");
            acc.x = fmaf(x.x, w, acc.x); acc.y = fmaf(x.y, w, acc.y);
            acc.z = fmaf(x.z, w, acc.z); acc.w = fmaf(x.w, w, acc.w);
        }
        const int gr = blk * 16 + r;
        write_row4<BF16>(c, b, hk * c.g + gr % c.g, gr / c.g, acc, ll);
    }
    __syncwarp();
    cluster_sync_all();   // partial results live until every CTA has read them
}

// Joins the splits of one row per warp, in split order; lane = four dims.
template <bool BF16>
__global__ void __launch_bounds__(128) attn_combine_kernel(const __grid_constant__ AttnCall c) {
    griddep_wait();
    griddep_launch();
    const mgc_attention_args& a = c.a;
    const int lane = threadIdx.x & 31;
    const long long all = (long long)a.B * a.Sq * a.Hq, id = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (id >= all) return;
    float mm = -INFINITY;
    for (int s = lane; s < c.nsplit; s += 32) mm = fmaxf(mm, c.mlpart[s * all + id].x);
    for (int k = 16; k; k >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, k));
    const float base = mm == -INFINITY ? 0.0f : mm;
    const bool dims = lane * 4 < a.D;
    const float4* op = reinterpret_cast<const float4*>(c.opart + id * a.D) + lane;
    const long long step = all * a.D / 4;
    float ll = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = 0; s0 < c.nsplit; s0 += 32) {
        const int n = min(32, c.nsplit - s0);
        float f = 0.0f, lf = 0.0f;   // lane = split: its weight, its sum
        if (lane < n) {
            const float2 ml = c.mlpart[(s0 + lane) * all + id];
            f = ex2_approx(ml.x - base);   // 0 where the split saw nothing (its partial is 0)
            lf = ml.y * f;
        }
        for (int k = 16; k; k >>= 1) lf += __shfl_xor_sync(0xffffffffu, lf, k);
        ll += lf;
#pragma unroll 8
        for (int s = 0; s < n; s++) {   // independent loads: eight splits in flight
            const float w = __shfl_sync(0xffffffffu, f, s);
            if (dims) {
                const float4 o = __ldcs(op + (s0 + s) * step);
                acc.x = fmaf(o.x, w, acc.x); acc.y = fmaf(o.y, w, acc.y);
                acc.z = fmaf(o.z, w, acc.z); acc.w = fmaf(o.w, w, acc.w);
            }
        }
    }
    const long long bi = id / a.Hq;
    write_row4<BF16>(c, (int)(bi / a.Sq), (int)(id % a.Hq), (int)(bi % a.Sq), acc, ll);
}

template <bool BF16, int DP, int WARPS>
void launch_warps(const AttnCall& c, cudaStream_t st) {
    static std::atomic<uint64_t> done{0};
    auto kernel = attn_step_kernel<BF16, DP, WARPS>;
    constexpr int smem = smem_bytes<DP, WARPS>();
    allow_smem(kernel, smem, done);
    const long long blocks = (long long)c.a.B * c.a.Hkv * ((c.a.Sq * c.g + 15) / 16) * c.nsplit;
    if (blocks > 0x7fffffffLL) throw std::runtime_error("too many rows for one launch");
    if (c.cluster) {
        launch_clusters(kernel, (unsigned)blocks, WARPS * 32, smem, c.nsplit, st, c);
        return;
    }
    ++g_launch_count;
    const cudaError_t e = launch_k(kernel, dim3((unsigned)blocks), dim3(WARPS * 32), smem, st, c);
    if (e != cudaSuccess) throw std::runtime_error(std::string("launch failed: ") + cudaGetErrorString(e));
}
template <bool BF16, int DP>
void launch_step(const AttnCall& c, cudaStream_t st) {
    if (c.wide) launch_warps<BF16, DP, 8>(c, st);
    else launch_warps<BF16, DP, 4>(c, st);
}

template <bool BF16>
void dispatch_step(const AttnCall& c, cudaStream_t st) {
    switch ((c.a.D + 15) / 16) {
        case 1: launch_step<BF16, 16>(c, st); break;
        case 2: launch_step<BF16, 32>(c, st); break;
        case 3: launch_step<BF16, 48>(c, st); break;
        case 4: launch_step<BF16, 64>(c, st); break;
        case 5: launch_step<BF16, 80>(c, st); break;
        case 6: launch_step<BF16, 96>(c, st); break;
        case 7: launch_step<BF16, 112>(c, st); break;
        default: launch_step<BF16, 128>(c, st); break;
    }
}

}  // namespace

void launch_attn_step(const AttnCall& c, cudaStream_t st) {
    if (c.a.dtype == MGC_BF16) dispatch_step<true>(c, st);
    else dispatch_step<false>(c, st);
}

void launch_attn_combine(const AttnCall& c, cudaStream_t st) {
    const long long all = (long long)c.a.B * c.a.Sq * c.a.Hq, blocks = (all + 3) / 4;
    if (blocks > 0x7fffffffLL) throw std::runtime_error("too many rows for one launch");
    // (launched while the partial results are still being made: the kernel waits for them itself)
    launch_after(c.a.dtype == MGC_BF16 ? attn_combine_kernel<true> : attn_combine_kernel<false>, (unsigned)blocks, 128, st, c);
}

}  // namespace mgc
