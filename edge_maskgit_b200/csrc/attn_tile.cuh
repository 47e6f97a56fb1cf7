// attn_tile.cuh -- mgc_attention for many queries, on tcgen05 tensor cores.
//
// One CTA owns up to two 128-query tiles of one head and walks the key tiles (128 keys) that any of
// its rows sees.  Copies, products and softmax run in separate warps:
//   warp 8   loads Q once, then K and V tiles through two rings (tensor maps, 128-byte swizzle)
//   warp 9   issues S = Q K^T into TMEM and, once P is there, O += P V with P read from TMEM
//   warps 0-3, 4-7   the softmax of query tile 0 and 1: one thread owns one row, so the running
//            maximum and sum need no exchange between threads (warps 10, 11 only complete a
//            warpgroup, whose registers move together)
// P (16 bits) overwrites the first half of its S.  While one tile's softmax runs, the tensor cores
// work on the other's products.  Probabilities are relative to a base that follows the row's maximum
// in large steps only, so the output in TMEM is hardly ever rescaled and no pass over a tile has to
// find its maximum first; in floating point this costs no precision.
#pragma once
#include <climits>

#include "attn_shaped.cuh"

namespace mgc {
namespace at {

constexpr int QT = 128, KT = 128, THREADS = 384;
constexpr uint32_t SLAB = 128 * 128;   // 128 rows of 64 16-bit values
template <int DP> constexpr uint32_t tile_bytes() { return SLAB * (DP / 64); }
template <int DP> constexpr int kv_stages() { return DP == 64 ? 3 : 2; }
constexpr int WIN = 264;   // entries of one copy of a tile's bias window (256 used)
constexpr uint32_t OFF_TABLE = 0;                        // [2 tiles][2 buffers][4 copies][WIN] f32 bias by distance
constexpr uint32_t OFF_DOC = OFF_TABLE + 16 * WIN * 4;    // [2][2][128] int32 document numbers
constexpr uint32_t OFF_BAR = OFF_DOC + 4 * 128 * 4, OFF_TILES = OFF_BAR + 512;   // (from a 1024-byte boundary)
constexpr uint32_t HEAD = (OFF_TILES + 1023) / 1024 * 1024;
template <int DP> constexpr uint32_t smem() { return 1024 + HEAD + (2 + 2 * kv_stages<DP>()) * tile_bytes<DP>(); }
// TMEM columns: S0 | S1 | O0 | O1, and with heads of up to 64 there is room for P0 | P1: then S is
// free as soon as it is read, and the next one is ready before P is done.
constexpr uint32_t TM_O = 256, TM_P = 384;

enum Mode { CAP = 1, SLOPE = 2, TABLE = 4 };

struct TileCall {
    AttnCall c;
    int tiles_per_cta;      // 1 or 2 query tiles
    int qblocks;            // CTAs along the queries
    int q_outer;            // 1: the last queries of every head first (causal: the long rows first)
    // [B][key tiles] or null: x = lowest number >= 0 of the tile (INT_MAX: none), with the sign bit
    // set if some are negative; y = the highest
    const int2* doc_range;
    int* dev_error;         // the library's device error word
    int kmul[3], vmul[3], qmul[3];   // 0 where a stride is 0 (batch, -, head): the map has one entry there
};

// A tile whose bias is linear in the key (or that has none) forms its exponents in one step, s c1 + (bias - base),
// with one rounding at the end, while base and bias were rounded on their own.  Up to this size of the bias
// and of the row's maximum (in base 2) those roundings are below 2^-3.  Beyond it a lowest bias would
// lose the scores, and a maximum of 2^27 could lie 16 above its own base, past f16's largest value: such a
// tile forms t = s c1 + bias of each key first, and t minus the base is exact where it matters.
constexpr float LINEAR_MAX = 1048576.0f;

// What the softmax of one row needs of one key tile.
struct RowTile {
    float c1;              // no cap: scale in base 2 (sign in `flip`); cap: scale / cap
    uint32_t flip;
    float cap2, slope2;
    float d0;              // distance of the tile's key 0, as slopes count it
    float lin_a, lin_b;    // the bias of key j where it is linear: lin_a + lin_b * j
    const float* win;      // bias of key j at win[j], 16-byte aligned
    int lim;               // keys below the row's end
    const int4* docs;      // documents of the tile's keys, or null
    int doc;
    float k0, k1, k2;      // cap: t = s (k0 + k1 s^2 + k2 s^4) while |s c1| <= CAP_RAW
};
// cap tanh(u) in base 2 for |u| <= 1/3, u (c0 + c1 u^2 + c2 u^4), fitted here to a relative error of
// 2.2e-6: scores well below their cap, the usual case, take four FP32 operations a pair.
constexpr float CAP_RAW = 1.0f / 3.0f;

// cap tanh(u) in base 2 for |u| <= 1: u (c0 + c1 u^2 + ...), fitted here; as stored, relative error 6.9e-7
// (times the cap: an error of that size in the exponent).  A score within the cap, the usual case,
// then takes no MUFU operation; tanh from its definition would take two beside the one of 2^x.
__device__ __forceinline__ uint64_t capped_poly(uint64_t u, uint64_t cap2) {
    const uint64_t w = mul2(u, u);
    uint64_t p = fma2(w, pack2(-0.00310273808f, -0.00310273808f), pack2(0.0168325986f, 0.0168325986f));
    p = fma2(p, w, pack2(-0.0516843035f, -0.0516843035f));
    p = fma2(p, w, pack2(0.132842583f, 0.132842583f));
    p = fma2(p, w, pack2(-0.333293984f, -0.333293984f));
    p = fma2(p, w, pack2(0.999999486f, 0.999999486f));
    return mul2(mul2(u, cap2), p);
}

__device__ __forceinline__ void flip32(uint32_t* s, const RowTile& x) {   // a negative scale
    if (x.flip) {
#pragma unroll
        for (int j = 0; j < 32; j++) s[j] ^= x.flip;
    }
}
// Scores of 32 keys, from key `first` of the tile, become t, shaped scores in base 2 (MODE 0: they
// stay raw, to be scaled in one fma with the base).
template <int MODE>
__device__ __forceinline__ void shape32(uint32_t* s, const RowTile& x, int first) {
    const uint64_t c2 = pack2(x.c1, x.c1);
    auto S = [&](int j) -> float { return __uint_as_float(s[j]); };
    if (!(MODE & CAP)) flip32(s, x);
    if (MODE & CAP) {
        float hi[2] = {-INFINITY, -INFINITY}, lo[2] = {INFINITY, INFINITY};
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
            hi[(j >> 1) & 1] = max3(hi[(j >> 1) & 1], S(j), S(j + 1));
            lo[(j >> 1) & 1] = min3(lo[(j >> 1) & 1], S(j), S(j + 1));
        }
        const float top = fmaxf(fmaxf(hi[0], hi[1]), -fminf(lo[0], lo[1])) * fabsf(x.c1);
        if (__all_sync(0xffffffffu, top <= 1.0f)) {   // (a NaN score escapes the comparison and stays NaN)
            const uint64_t cp2 = pack2(x.cap2, x.cap2);
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
                float a, b;
                unpack2(capped_poly(mul2(pack2(S(j), S(j + 1)), c2), cp2), a, b);
                s[j] = __float_as_uint(a);
                s[j + 1] = __float_as_uint(b);
            }
        } else {
            const float k = x.c1 * (2.0f * ATTN_LOG2E);
#pragma unroll
            for (int j = 0; j < 32; j++) s[j] = __float_as_uint(capped(S(j), k, x.cap2));
        }
    }
    if (MODE & (SLOPE | TABLE)) {
        const float d0 = x.d0 + (float)first;
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
            float b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (MODE & TABLE) {
                const float4 f = *reinterpret_cast<const float4*>(x.win + first + j);
                b[0] = f.x; b[1] = f.y; b[2] = f.z; b[3] = f.w;
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (MODE & SLOPE) b[e] = fmaf(-x.slope2, fabsf(d0 + (float)(j + e)), b[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const uint64_t t2 = pack2(S(j + e), S(j + e + 1)), b2 = pack2(b[e], b[e + 1]);
                float u, v;
                unpack2((MODE & CAP) ? add2(t2, b2) : fma2(t2, c2, b2), u, v);
                s[j + e] = __float_as_uint(u);
                s[j + e + 1] = __float_as_uint(v);
            }
        }
    }
}
// Unseen keys' scores become -inf.
__device__ __forceinline__ void mask32(uint32_t* s, const RowTile& x, int first) {
    const int lim = x.lim - first;
    if (x.lim < KT) {
#pragma unroll
        for (int j = 0; j < 32; j++) s[j] = j < lim ? s[j] : 0xFF800000u;
    }
    if (x.docs) {
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
            const int4 d = x.docs[(first + j) / 4];
            s[j] = d.x == x.doc ? s[j] : 0xFF800000u;
            s[j + 1] = d.y == x.doc ? s[j + 1] : 0xFF800000u;
            s[j + 2] = d.z == x.doc ? s[j + 2] : 0xFF800000u;
            s[j + 3] = d.w == x.doc ? s[j + 3] : 0xFF800000u;
        }
    }
}
// hi[] = max(hi[], s[]), NaN where a score is
__device__ __forceinline__ void max32(float (&hi)[4], const uint32_t* s) {
#pragma unroll
    for (int j = 0; j < 32; j += 2)
        hi[(j >> 1) & 3] = max3_nan(hi[(j >> 1) & 3], __uint_as_float(s[j]), __uint_as_float(s[j + 1]));
}

// 32 columns of a row's output in TMEM, times f.
__device__ __forceinline__ void scale_o(uint32_t taddr, float f) {
    uint32_t v[32];
    tmem_ld32(taddr, v);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 32; e++) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
    tmem_st32(taddr, v);
}

// GIVE_UP: a self-test, in which one warp of each block acts as if its wait for a tile's second scores had run out.
template <bool BF16, int DP, int MODE, bool GIVE_UP = false>
__global__ void __launch_bounds__(THREADS, 1) attn_tile_kernel(const __grid_constant__ CUtensorMap mq,
                                                               const __grid_constant__ CUtensorMap mk,
                                                               const __grid_constant__ CUtensorMap mv,
                                                               const __grid_constant__ TileCall tc) {
    constexpr int NST = kv_stages<DP>(), NSLAB = DP / 64;
    constexpr bool SEP = DP == 64;
    constexpr uint32_t TB = tile_bytes<DP>();
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = align1024_smem(smem_raw);
    uint8_t* sQ = sm + HEAD;
    uint8_t* sK = sQ + 2 * TB;
    uint8_t* sV = sK + NST * TB;
    uint64_t* bars = (uint64_t*)(sm + OFF_BAR);
    uint64_t* q_full = bars;               // [2] a query tile landed
    uint64_t* k_full = bars + 2;           // [NST]
    uint64_t* k_empty = k_full + NST;
    uint64_t* v_full = k_empty + NST;
    uint64_t* v_empty = v_full + NST;
    uint64_t* s_full = v_empty + NST;      // [2] S is in TMEM, and the product before it is done
    uint64_t* p_full = s_full + 2;         // [2] P is in TMEM (4 warps)
    uint64_t* o_full = p_full + 2;         // [2] a product with P is done
    uint64_t* s_free = o_full + 2;         // [2] S was read (4 warps; SEP)
    uint64_t* p_half = s_free + 2;         // [2] the first half of P is in TMEM (4 warps)
    uint64_t* drained = p_half + 2;        // every product is done
    uint32_t* tmem_slot = (uint32_t*)(drained + 1);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    int* range = (int*)(tmem_slot + 2);    // lo0, lo1, hi0, hi1, then a tile's lowest / highest document

    const AttnCall& c = tc.c;
    const mgc_attention_args& a = c.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    unsigned rest = blockIdx.x / (unsigned)c.nsplit;
    const int split = (int)(blockIdx.x - rest * c.nsplit);
    int qb, h, b;
    if (tc.q_outer) {
        h = (int)(rest % (unsigned)a.Hq); rest /= (unsigned)a.Hq;
        b = (int)(rest % (unsigned)a.B);
        qb = tc.qblocks - 1 - (int)(rest / (unsigned)a.B);
    } else {
        qb = (int)(rest % (unsigned)tc.qblocks); rest /= (unsigned)tc.qblocks;
        h = (int)(rest % (unsigned)a.Hq);
        b = (int)(rest / (unsigned)a.Hq);
    }
    const int hk = h / c.g, q0 = qb * tc.tiles_per_cta * QT;
    griddep_wait();
    griddep_launch();
    const RowBounds rb = row_bounds(a, b);
    const int nkt = (a.Sk + KT - 1) / KT;

    // ---- the key tiles [lo, hi) of each query tile
    const int kt_first = split * (c.chunk / KT), kt_last = min(nkt, kt_first + c.chunk / KT);
    int lo[2], hi[2];
#pragma unroll
    for (int w = 0; w < 2; w++) {
        const int first = q0 + w * QT, last = min(first + QT, a.Sq) - 1;
        lo[w] = kt_first;
        hi[w] = w < tc.tiles_per_cta && last >= first
                    ? max(lo[w], min(kt_last, (key_end(rb, rb.pos0 + last) + KT - 1) / KT)) : lo[w];
    }
    // Step i works on key tile order(i): from the diagonal (the last query's position) down to the first,
    // then up from there.  A bias that falls with the distance has its largest values first, so bases
    // are not moved from tile to tile, and causally the tile with the mask comes first.
    bool on[2];
    int lo_all, n, centre;
    auto steps = [&] {
        on[0] = hi[0] > lo[0];
        on[1] = hi[1] > lo[1];
        lo_all = min(on[0] ? lo[0] : INT_MAX, on[1] ? lo[1] : INT_MAX);
        const int hi_all = max(on[0] ? hi[0] : 0, on[1] ? hi[1] : 0);
        n = hi_all > lo_all ? hi_all - lo_all : 0;
        centre = max(lo_all, min(hi_all - 1, (rb.pos0 + min(q0 + tc.tiles_per_cta * QT, a.Sq) - 1) >> 7));
    };
    auto order = [&](int i) { return i <= centre - lo_all ? centre - i : lo_all + i; };
    auto active = [&](int w, int i) {
        const int kt = order(i);
        return on[w] && i >= 0 && i < n && kt >= lo[w] && kt < hi[w];
    };
    // ---- copies (by one thread)
    auto copy = [&](uint8_t* dst, const CUtensorMap* map, int pos, int head, int batch, uint64_t* bar) {
        mbar_arrive_expect_tx(bar, TB);
#pragma unroll
        for (int s = 0; s < NSLAB; s++) tma_load_4d(dst + s * SLAB, map, s * 64, pos, head, batch, bar);
    };
    auto copy_k = [&](int i) { copy(sK + i % NST * TB, &mk, order(i) * KT, hk * tc.kmul[2], b * tc.kmul[0], k_full + i % NST); };
    auto copy_v = [&](int i) { copy(sV + i % NST * TB, &mv, order(i) * KT, hk * tc.vmul[2], b * tc.vmul[0], v_full + i % NST); };
    auto first_copies = [&] {   // both query tiles and a ring of key tiles
        for (int i = 0; i < min(n, NST); i++) {
            if (i == 0 && on[0]) copy(sQ, &mq, q0, h * tc.qmul[2], b * tc.qmul[0], q_full);
            copy_k(i);
            if (i == 0 && on[1]) copy(sQ + TB, &mq, q0 + QT, h * tc.qmul[2], b * tc.qmul[0], q_full + 1);
            copy_v(i);
        }
    };
    steps();

    if (tid == 256) {   // (warp 8, which issues the copies)
        for (int i = 0; i < 2; i++) {
            mbar_init(q_full + i, 1); mbar_init(s_full + i, 1); mbar_init(p_full + i, 4); mbar_init(o_full + i, 1);
            mbar_init(s_free + i, 4); mbar_init(p_half + i, 4);
        }
        for (int i = 0; i < NST; i++) {
            mbar_init(k_full + i, 1); mbar_init(k_empty + i, 1); mbar_init(v_full + i, 1); mbar_init(v_empty + i, 1);
        }
        mbar_init(drained, 1);
        *abort_flag = 0;
        mbar_fence_init();
        if (!a.doc_q) first_copies();   // under the rest of the set-up
    }
    if (tid < 2) {
        range[tid] = INT_MAX; range[2 + tid] = 0; range[4 + tid] = INT_MAX; range[6 + tid] = -1;
    }
    if (warp == 9) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (a.doc_q) {   // only tiles that share a document number with the queries (sorted or not)
        if (warp < 8) {
            const int w = warp >> 2, i = q0 + w * QT + (tid & 127);
            const int d = w < tc.tiles_per_cta && i < a.Sq ? __ldg(a.doc_q + (long long)b * a.Sq + i) : -1;
            int mn = d >= 0 ? d : INT_MAX, mx = d;
            for (int k = 16; k; k >>= 1) {
                mn = min(mn, __shfl_xor_sync(0xffffffffu, mn, k));
                mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, k));
            }
            if (lane == 0) { atomicMin(range + 4 + w, mn); atomicMax(range + 6 + w, mx); }
        }
        __syncthreads();
        for (int kt = kt_first + tid; kt < kt_last; kt += THREADS) {
            const int2 r = __ldg(tc.doc_range + (long long)b * nkt + kt);
#pragma unroll
            for (int w = 0; w < 2; w++)
                if (r.y >= range[4 + w] && (r.x & INT_MAX) <= range[6 + w]) { atomicMin(range + w, kt); atomicMax(range + 2 + w, kt + 1); }
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 2; w++) {
            lo[w] = max(lo[w], range[w]);
            hi[w] = min(hi[w], range[2 + w]);
        }
        steps();
        if (tid == 256) first_copies();
    }

    // Registers: 384 threads start with 168 each (64512); the 256 softmax threads take 216, the
    // other warpgroup keeps 72: 256 * 216 + 128 * 72 = 64512, all of the launch's own.
    // (Inside the branches: where they meet again the compiler has to assume the smaller number.)
    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 8) {
        // ---------------------------------------------------------------- copies
        if (lane == 0 && n > 0) {
            int i = min(n, NST), ks = i, vs = i;   // (the first ring is under way); copies of K and V requested
            for (; i < n; i++) {
                const int par = (i / NST - 1) & 1;
                if (!mbar_wait(k_empty + i % NST, par, abort_flag, 51, tc.dev_error)) break;
                copy_k(i);
                ks++;
                if (!mbar_wait(v_empty + i % NST, par, abort_flag, 52, tc.dev_error)) break;
                copy_v(i);
                vs++;
            }
            // The block must not end with copies under way.  They have landed where all of them were used; after
            // a wait that gave up, here or in another warp, some may not have been.
            volatile int never = 0;
            for (int w = 0; w < 2; w++) if (on[w]) mbar_wait(q_full + w, 0, &never, 53, tc.dev_error);
            for (int t = max(0, ks - NST); t < ks; t++) mbar_wait(k_full + t % NST, (t / NST) & 1, &never, 53, tc.dev_error);
            for (int t = max(0, vs - NST); t < vs; t++) mbar_wait(v_full + t % NST, (t / NST) & 1, &never, 53, tc.dev_error);
        }
    } else if (warp == 9) {
        // ---------------------------------------------------------------- products
        // The whole warp walks the loop, so that descriptors stay in uniform registers; one elected
        // lane issues.
        if (n > 0) {
            const int dsteps = (a.D + 15) / 16;
            constexpr uint32_t idesc_s = idesc_make(1, BF16, BF16, QT, KT);
            const uint32_t idesc_o = idesc_make(1, BF16, BF16, QT, (uint32_t)dsteps * 16) | IDESC_B_MN;
            const uint64_t dq0 = sdesc_sw128(smem_u32(sQ)), dk0 = sdesc_sw128(smem_u32(sK));
            const uint64_t dv0 = sdesc_mn_sw128(smem_u32(sV), SLAB);
            const bool lead = elect_one();
            auto qk = [&](int w, int st) {
                const uint64_t dq = dq0 + w * (TB >> 4), dk = dk0 + (uint32_t)st * (TB >> 4);
                if (lead) {
#pragma unroll
                    for (int k = 0; k < DP / 16; k++) {
                        if (k < dsteps) {
                            const uint32_t off = (k >> 2) * (SLAB >> 4) + 2 * (k & 3);
                            mma_f16(tmem + w * KT, dq + off, dk + off, idesc_s, k > 0);
                        }
                    }
                    mma_commit(s_full + w);
                }
            };
            auto pv = [&](int w, int st, bool first, int k0, int k1) {
                const uint64_t dv = dv0 + (uint32_t)st * (TB >> 4);
                if (lead) {
#pragma unroll
                    for (int k = k0; k < k1; k++)
                        mma_f16_ts(tmem + TM_O + w * DP, tmem + (SEP ? TM_P + w * (KT / 2) : w * KT) + k * 8,
                                   dv + k * (2048 >> 4), idesc_o, k > 0 || !first);
                    if (k1 == KT / 16) mma_commit(o_full + w);
                }
            };
            bool ok = true;
            int ns[2] = {0, 0}, np[2] = {0, 0};   // scores and products issued
            int st = 0, par = 0;                  // ring stage and parity of step i
            for (int i = -1; ok && i < n; i++) {
                const int st1 = i < 0 ? 0 : st + 1 == NST ? 0 : st + 1, par1 = i < 0 ? 0 : st1 == 0 ? par ^ 1 : par;
                if (i + 1 < n && !(ok = mbar_wait(k_full + st1, par1, abort_flag, 54, tc.dev_error))) break;
                // (the copy of a tile between the two ranges is used by neither, but has to land)
                if (i >= 0 && !(ok = mbar_wait(v_full + st, par, abort_flag, 56, tc.dev_error))) break;
                auto score = [&](int w) {   // S of step i + 1
                    if (!active(w, i + 1)) return;
                    if (ns[w] == 0) ok = ok && mbar_wait(q_full + w, 0, abort_flag, 57, tc.dev_error);
                    else if (SEP) ok = ok && mbar_wait(s_free + w, (ns[w] - 1) & 1, abort_flag, 62, tc.dev_error);
                    if (!ok) return;
                    tc_fence_after();
                    qk(w, st1);
                    ns[w]++;
                };
                auto product = [&](int w) {   // O += P V of step i
                    if (!active(w, i)) return;
                    if (!SEP) {
                        ok = ok && mbar_wait(p_half + w, np[w] & 1, abort_flag, 64, tc.dev_error);
                        if (!ok) return;
                        tc_fence_after();
                        pv(w, st, np[w] == 0, 0, KT / 32);
                    }
                    ok = ok && mbar_wait(p_full + w, np[w] & 1, abort_flag, 55, tc.dev_error);
                    if (!ok) return;
                    tc_fence_after();
                    pv(w, st, np[w] == 0, SEP ? 0 : KT / 32, KT / 16);
                    np[w]++;
                };
                if (SEP) {
                    score(0); product(0);
                    score(1); product(1);
                } else {   // S(i + 1) takes the place of P(i)
                    product(0); score(0);
                    product(1); score(1);
                }
                if (!ok) break;
                if (lead) {
                    if (i >= 0) mma_commit(v_empty + st);
                    if (i + 1 < n) mma_commit(k_empty + st1);
                }
                st = st1;
                par = par1;
            }
            if (lead) {   // the TMEM is freed behind the last product, also after a wait that gave up
                volatile int never = 0;
                mma_commit(drained);
                mbar_wait(drained, 0, &never, 65, tc.dev_error);
            }
            __syncwarp();
        }
    }
    } else {
        // ---------------------------------------------------------------- softmax: thread = row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int w = warp >> 2, r = tid & 127;
        const int row_i = q0 + w * QT + r, qi = min(row_i, a.Sq - 1);
        const int p = rb.pos0 + qi;
        const ScoreShape sh = score_shape(a, h);
        const bool live = w < tc.tiles_per_cta && row_i < a.Sq;
        // (rows past the last query compute on as copies of it, so that they force no masking)
        const int doc = a.doc_q ? __ldg(a.doc_q + (long long)b * a.Sq + qi) : 0;
        const int end = doc >= 0 ? key_end(rb, p) : 0;
        const bool idle = q0 + w * QT + (warp & 3) * 32 >= a.Sq;   // a warp of such rows only
        const uint32_t t_row = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t tS = t_row + w * KT, tO = t_row + TM_O + w * DP, tP = SEP ? t_row + TM_P + w * (KT / 2) : tS;
        float* win = reinterpret_cast<float*>(sm + OFF_TABLE) + w * 8 * WIN;
        int* sdoc = reinterpret_cast<int*>(sm + OFF_DOC) + w * 256;
        const int bar_id = 1 + w;
        RowTile x;
        // (a scale of 0 must not meet the -inf of a masked score)
        x.c1 = (MODE & CAP) ? a.scale / a.cap : fmaxf(fabsf(sh.c1), 1.17549435e-38f);
        x.flip = sh.c1 < 0.0f ? 0x80000000u : 0u;   // a negative scale
        x.cap2 = sh.cap2;
        x.slope2 = sh.slope2;
        x.doc = doc < 0 ? -2 : doc;   // (a padding query matches no key, not a padding key either)
        x.k0 = 0.999997882f * x.cap2 * x.c1;
        x.k1 = -0.332985124f * x.cap2 * x.c1 * x.c1 * x.c1;
        x.k2 = 0.124804431f * x.cap2 * x.c1 * x.c1 * x.c1 * x.c1 * x.c1;
        // Probabilities are 2^(t - base).  base is set at the first scores to SHIFT below their maximum,
        // whose probability is then a power of two and rounds to itself, and again only when a score
        // passes it by SLACK: the sum and the output so far are then scaled, in f32.  So no pass over the
        // tile has to find its maximum first.  In f16 probabilities go up to 2^15, which it holds, and its
        // smallest normal number is 2^-25 of the row's maximum or less (a sum of many small ones behind one
        // large is right); bf16 has room for more.  (base is rounded up: no score lies more than SHIFT above it.)
        constexpr float SHIFT = BF16 ? 3.0f : 11.0f, SLACK = BF16 ? 40.0f : 15.0f;

        // bias window and documents of key tile kt: fetched a tile ahead
        float pre_b[2] = {0.0f, 0.0f};
        int pre_d = 0;
        int2 pre_r = make_int2(0, 0);
        auto fetch = [&](int kt) {
            if (MODE & TABLE) {
                const int d0 = kt * KT - (rb.pos0 + q0 + w * QT) - 127;   // distance of window entry 0
#pragma unroll
                for (int u = 0; u < 2; u++) pre_b[u] = __ldg(sh.table + max(-sh.range, min(sh.range, d0 + r + 128 * u)));
            }
            if (a.doc_k) {   // (padding, and keys past the length, get one number, and a padding query another)
                pre_d = kt * KT + r < rb.len ? max(-1, __ldg(a.doc_k + (long long)b * a.Sk + kt * KT + r)) : -1;
                pre_r = __ldg(tc.doc_range + (long long)b * nkt + kt);
            }
        };
        // All of the tile's distances beyond the table's range on one side: one bias for all, and the window is
        // neither filled nor looked at, so the tile has to be linear for each of its rows: no caps, slopes that
        // count from one side, and a bias that does not absorb the scores (the type's lowest value, say).
        auto is_flat = [&](int kt) {
            const int dist_lo = kt * KT - (rb.pos0 + q0 + w * QT) - 127, dist_hi = dist_lo + 254;
            bool flat = (MODE & TABLE) && !(MODE & CAP) && (dist_lo >= sh.range || dist_hi <= -sh.range) &&
                        (fabsf(pre_b[0]) <= LINEAR_MAX || pre_b[0] == -INFINITY);
            if ((MODE & SLOPE) && (MODE & TABLE) && flat) {
                const int first = slope_pos(rb, rb.pos0 + q0 + w * QT), last = slope_pos(rb, rb.pos0 + min(q0 + w * QT + QT, a.Sq) - 1);
                const int k0 = kt * KT, far = max(abs(k0 - first), abs(k0 - last)) + 127;
                flat = (k0 >= last || k0 + 127 <= first) && fabsf(x.slope2) * (float)far <= LINEAR_MAX;
            }
            return flat;
        };
        float base = 0.0f, l = 0.0f;
        bool fresh = true, ok = true;   // fresh: the row has seen nothing yet, base is not set
        // (selected, not indexed by w: arrays would go to local memory)
        const int lo_w = w ? lo[1] : lo[0], hi_w = w ? hi[1] : hi[0], n_w = max(0, hi_w - lo_w);
        const int lo_o = w ? lo[0] : lo[1], hi_o = w ? hi[0] : hi[1];
        auto mine = [&](int i) { const int kt = order(i); return kt >= lo_w && kt < hi_w; };
        auto others = [&](int i) { const int kt = order(i); return i >= 0 && i < n && kt >= lo_o && kt < hi_o; };
        int i = 0, it = 0;   // step, this tile's steps so far
        while (i < n && !mine(i)) i++;
        if (n_w > 0) fetch(order(i));
        for (int next; it < n_w; i = next, it++) {
            const int kt = order(i), buf = it & 1;
            for (next = i + 1; next < n && !mine(next);) next++;
            const bool flat = is_flat(kt);
            if (((MODE & TABLE) && !flat) || a.doc_k) {
                if ((MODE & TABLE) && !flat) {   // four copies, each shifted by one entry: every row reads aligned vectors
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const float v = bias2(pre_b[u]);
                        const int e = r + 128 * u;
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            if (e >= k) win[(buf * 4 + k) * WIN + e - k] = v;
                    }
                }
                if (a.doc_k) sdoc[buf * 128 + r] = pre_d;
                named_bar_sync(bar_id, 128);
            }
            x.d0 = (float)(kt * KT - slope_pos(rb, p));
            x.lin_a = x.lin_b = 0.0f;
            bool linear = false;
            if (MODE & (SLOPE | TABLE)) {
                linear = flat;
                if (!(MODE & TABLE))
                    linear = __all_sync(0xffffffffu, (x.d0 >= 0.0f || x.d0 <= -127.0f) &&
                                                         fabsf(x.slope2) * (fabsf(x.d0) + 127.0f) <= LINEAR_MAX);
                x.lin_b = x.d0 >= 0.0f ? -x.slope2 : x.slope2;
                x.lin_a = ((MODE & SLOPE) ? x.lin_b * x.d0 : 0.0f) + (flat ? bias2(pre_b[0]) : 0.0f);
            }
            x.win = win + (buf * 4 + ((127 - r) & 3)) * WIN + ((127 - r) & ~3);
            x.lim = end - kt * KT;
            x.docs = nullptr;
            bool none = x.lim <= 0;   // this row sees nothing of the tile
            if (a.doc_k) {
                if (!__all_sync(0xffffffffu, pre_r.x == pre_r.y && doc == pre_r.x)) x.docs = reinterpret_cast<const int4*>(sdoc + buf * 128);
                none = none || doc > pre_r.y || doc < (pre_r.x & INT_MAX);
                // (the document numbers hide the keys past the length too)
                if (x.docs && !a.causal) x.lim = KT;
            }
            const bool masked = x.docs || !__all_sync(0xffffffffu, x.lim >= KT);
            const bool skip = idle || __all_sync(0xffffffffu, none);
            if (((MODE & TABLE) || a.doc_k) && next < n) fetch(order(next));

            ok = __all_sync(0xffffffffu, mbar_wait(s_full + w, it & 1, abort_flag, 58, tc.dev_error));
            if (GIVE_UP && it == 1 && warp == 1) {
                if (lane == 0) {
                    *abort_flag = 58;
                    atomicExch(tc.dev_error, 58);
                }
                ok = false;
            }
            if (!ok) break;
            tc_fence_after();
            // keys behind the row's length are not in the tensor maps' bounds: v may hold NaN there
            if (rb.len < a.Sk && rb.len - kt * KT < KT && rb.len > kt * KT && !(w == 1 && others(i))) {
                const int st = i % NST;
                ok = __all_sync(0xffffffffu, mbar_wait(v_full + st, (i / NST) & 1, abort_flag, 59, tc.dev_error));
                if (!ok) break;
                if (r >= rb.len - kt * KT) {
#pragma unroll
                    for (int sl = 0; sl < NSLAB; sl++)
#pragma unroll
                        for (int ch = 0; ch < 8; ch++)
                            *reinterpret_cast<uint4*>(sV + st * TB + sl * SLAB + r * 128 + ch * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_async_smem();
            }
            // (SEP) the next S may come; P and O are free once the product before is done
            auto s_is_read = [&] {
                if (!SEP) return;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(s_free + w);
            };
            auto wait_product = [&] {
                if (!SEP || it == 0) return;
                ok = __all_sync(0xffffffffu, mbar_wait(o_full + w, (it - 1) & 1, abort_flag, 61, tc.dev_error));
                tc_fence_after();
            };
            auto half_done = [&] {   // P of the first 64 keys is in TMEM
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_half + w);
            };
            if (skip) {   // no scores to look at: probabilities of 0
                s_is_read();
                wait_product();
                uint32_t zero[16];
#pragma unroll
                for (int e = 0; e < 16; e++) zero[e] = 0;
#pragma unroll
                for (int q = 0; q < 4; q++) tmem_st16(tP + q * 16, zero);
                if (!SEP) half_done();
            } else {
                uint32_t s[128];
                bool raw = MODE == 0;   // s holds scores to be shaped with the exponentials, not t
                float hi[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, lo_s[4] = {INFINITY, INFINITY, INFINITY, INFINITY};
#pragma unroll
                for (int q = 0; q < 4; q++) tmem_ld32(tS + q * 32, reinterpret_cast<uint32_t(&)[32]>(s[q * 32]));
#pragma unroll
                for (int q = 0; q < 4; q++) tmem_ld_done(reinterpret_cast<uint32_t(&)[32]>(s[q * 32]));
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    if (MODE == CAP) {
                        max32(hi, s + q * 32);
#pragma unroll
                        for (int j = 0; j < 32; j += 2)
                            lo_s[(j >> 1) & 3] = min3(lo_s[(j >> 1) & 3], __uint_as_float(s[q * 32 + j]), __uint_as_float(s[q * 32 + j + 1]));
                    }
                }
                if (MODE != CAP) {
                    // (a tile whose bias is linear in the key keeps its raw scores: t is cheap to form twice)
                    raw = MODE == 0 || ((MODE & CAP) == 0 && linear);
                    if (!raw || x.flip) {
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            if (raw) flip32(s + q * 32, x);
                            else shape32<MODE>(s + q * 32, x, q * 32);
                        }
                    }
                    if (masked) {
#pragma unroll
                        for (int q = 0; q < 4; q++) mask32(s + q * 32, x, q * 32);
                    }
                    if ((MODE & SLOPE) && raw) {
#pragma unroll
                        for (int j = 0; j < 128; j += 2)
                            hi[(j >> 1) & 3] = max3_nan(hi[(j >> 1) & 3], fmaf(__uint_as_float(s[j]), x.c1, fmaf((float)j, x.lin_b, x.lin_a)),
                                                        fmaf(__uint_as_float(s[j + 1]), x.c1, fmaf((float)(j + 1), x.lin_b, x.lin_a)));
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; q++) max32(hi, s + q * 32);
                    }
                }
                float mx = max3_nan(max3_nan(hi[0], hi[1], hi[2]), hi[3], hi[3]);
                if (raw && !(MODE & SLOPE) && mx != -INFINITY) mx = fmaf(mx, x.c1, x.lin_a);
                if (MODE == CAP) {
                    const float low = fminf(fminf(lo_s[0], lo_s[1]), fminf(lo_s[2], lo_s[3]));
                    raw = !masked && __all_sync(0xffffffffu, fmaxf(mx, -low) * fabsf(x.c1) <= CAP_RAW && mx == mx);
                    if (raw) {   // capped scores keep their order
                        mx = x.c1 < 0.0f ? low : mx;
                        const float w2 = mx * mx;
                        mx *= fmaf(fmaf(w2, x.k2, x.k1), w2, x.k0);
                    } else {
                        hi[0] = hi[1] = hi[2] = hi[3] = -INFINITY;
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            shape32<MODE>(s + q * 32, x, q * 32);
                            if (masked) mask32(s + q * 32, x, q * 32);
                            max32(hi, s + q * 32);
                        }
                        mx = max3_nan(max3_nan(hi[0], hi[1], hi[2]), hi[3], hi[3]);
                    }
                }
                s_is_read();
                const bool set = fresh ? mx != -INFINITY : mx - base > SLACK;   // (base + SLACK could round up)
                const bool large = !(MODE & CAP) && raw && fabsf(mx) > LINEAR_MAX && mx != -INFINITY;
                const bool move = __any_sync(0xffffffffu, set || large);
                wait_product();
                if (move) {
                    if (!(MODE & CAP) && __any_sync(0xffffffffu, large)) {
                        raw = false;   // scores of that size round like their maximum
#pragma unroll
                        for (int j = 0; j < 128; j++)
                            s[j] = __float_as_uint(fmaf(__uint_as_float(s[j]), x.c1, fmaf((float)j, x.lin_b, x.lin_a)));
                    }
                    float alpha = 1.0f;
                    if (set) {
                        const float nb = __fadd_ru(mx, -SHIFT);
                        if (!fresh) alpha = ex2_approx(base - nb);
                        l *= alpha;
                        base = nb;
                        fresh = false;
                    }
                    if (it > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll 1
                        for (int d = 0; d < DP; d += 32) scale_o(tO + d, alpha);
                    }
                }
                const uint64_t nb2 = pack2(-base, -base);
                uint64_t sum2[4] = {0, 0, 0, 0};
                auto probs = [&](auto arg) {   // arg: two entries of s -> two exponents
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        uint32_t pk[16];
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const int j = q * 32 + 2 * e;
                            float u, v;
                            unpack2(arg(pack2(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), j), u, v);
                            u = ex2_approx(u);
                            v = ex2_approx(v);
                            sum2[e & 3] = add2(sum2[e & 3], pack2(u, v));
                            pk[e] = pack16<BF16>(u, v);   // rounded to the type of v: what tensor cores multiply
                        }
                        tmem_st16(tP + q * 16, pk);
                        if (!SEP && q == 1) half_done();
                    }
                };
                const uint64_t c2 = pack2(x.c1, x.c1);
                if (MODE == CAP && raw) {
                    const uint64_t k0 = pack2(x.k0, x.k0), k1 = pack2(x.k1, x.k1), k2 = pack2(x.k2, x.k2);
                    probs([&](uint64_t t, int) {
                        const uint64_t w2 = mul2(t, t);
                        return fma2(t, fma2(fma2(w2, k2, k1), w2, k0), nb2);
                    });
                } else if ((MODE & SLOPE) && raw) {
                    const float la = x.lin_a - base;
                    probs([&](uint64_t t, int j) {
                        return fma2(t, c2, pack2(fmaf((float)j, x.lin_b, la), fmaf((float)(j + 1), x.lin_b, la)));
                    });
                } else {   // raw scores, or t already: one form
                    const float k = raw ? x.c1 : 1.0f, off = (raw ? x.lin_a : 0.0f) - base;
                    const uint64_t k2 = pack2(k, k), off2 = pack2(off, off);
                    probs([&](uint64_t t, int) { return fma2(t, k2, off2); });
                }
                float e0, e1, e2, e3;
                unpack2(add2(sum2[0], sum2[1]), e0, e1);
                unpack2(add2(sum2[2], sum2[3]), e2, e3);
                l += (e0 + e1) + (e2 + e3);
                if (mx != mx) l = mx;   // a NaN score: the row is NaN
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + w);
        }
        // A warp whose wait gave up still meets the tile's other warps at its remaining steps: one of them may
        // see the scores that it waits for before it sees the flag, and nothing bounds the wait at a meeting.
        if (!ok && ((MODE & TABLE) || a.doc_k)) {
#pragma unroll 1
            while (++it < n_w) {
                bool meet = true;   // (with documents, at each step)
                if ((MODE & TABLE) && !a.doc_k) {
                    for (i++; !mine(i);) i++;
                    fetch(order(i));
                    meet = !is_flat(order(i));
                }
                if (meet) named_bar_sync(bar_id, 128);
            }
        }
        // ---------------------------------------------------------------- output
        if (ok && n_w > 0) ok = __all_sync(0xffffffffu, mbar_wait(o_full + w, (n_w - 1) & 1, abort_flag, 60, tc.dev_error));
        tc_fence_after();
        if (ok && w < tc.tiles_per_cta && q0 + w * QT + (warp & 3) * 32 < a.Sq) {
            const bool any = n_w > 0 && !fresh;
            const float inv = any ? 1.0f / l : 0.0f;
            const long long row = ((long long)b * a.Sq + row_i) * a.Hq + h, id = (long long)split * a.B * a.Sq * a.Hq + row;
            if (c.nsplit > 1 && live) c.mlpart[id] = make_float2(any ? base : -INFINITY, l);
            uint16_t* dst = reinterpret_cast<uint16_t*>(a.out) + b * a.out_stride[0] + qi * a.out_stride[1] + h * a.out_stride[2];
            bool bad = false;
#pragma unroll
            for (int d = 0; d < DP; d += 32) {
                if (d >= a.D) break;
                uint32_t o[32];
                if (n_w > 0) {
                    tmem_ld32(tO + d, o);
                    tmem_ld_wait();
                }
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    const float v = any ? __uint_as_float(o[e]) : 0.0f;
                    bad |= d + e < a.D && suspect<BF16>(v);
                    o[e] = __float_as_uint(c.nsplit > 1 ? v : v * inv);
                }
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    if (d + e >= a.D || !live) break;
                    if (c.nsplit > 1) {
                        float4* op = reinterpret_cast<float4*>(c.opart + id * a.D + d + e);
                        op[0] = make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]), __uint_as_float(o[e + 3]));
                        op[1] = make_float4(__uint_as_float(o[e + 4]), __uint_as_float(o[e + 5]), __uint_as_float(o[e + 6]), __uint_as_float(o[e + 7]));
                    } else {
                        uint4 v;
                        v.x = pack16<BF16>(__uint_as_float(o[e]), __uint_as_float(o[e + 1]));
                        v.y = pack16<BF16>(__uint_as_float(o[e + 2]), __uint_as_float(o[e + 3]));
                        v.z = pack16<BF16>(__uint_as_float(o[e + 4]), __uint_as_float(o[e + 5]));
                        v.w = pack16<BF16>(__uint_as_float(o[e + 6]), __uint_as_float(o[e + 7]));
                        *reinterpret_cast<uint4*>(dst + d + e) = v;
                    }
                }
                __syncwarp();
            }
            bad = bad && !isnan(l) && live && c.nsplit == 1;   // (split: the join looks for it)
            for (unsigned todo = __ballot_sync(0xffffffffu, bad); todo; todo &= todo - 1)
                repair_row<BF16>(a, c.g, b, h, q0 + w * QT + (warp & 3) * 32 + __ffs(todo) - 1);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <bool BF16, int DP, int MODE, bool GIVE_UP = false>
void launch_tile(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const TileCall& t, cudaStream_t st) {
    static std::atomic<uint64_t> done{0};
    auto kernel = attn_tile_kernel<BF16, DP, MODE, GIVE_UP>;
    allow_smem(kernel, smem<DP>(), done);
    const long long grid = (long long)t.qblocks * t.c.a.B * t.c.a.Hq * t.c.nsplit;
    if (grid > 0x7fffffffLL) throw std::runtime_error("too many rows for one launch");
    ++g_launch_count;
    const cudaError_t e = launch_k(kernel, dim3((unsigned)grid), dim3(THREADS), smem<DP>(), st, mq, mk, mv, t);
    if (e != cudaSuccess) throw std::runtime_error(std::string("launch failed: ") + cudaGetErrorString(e));
}

template <bool BF16, int DP>
void dispatch_mode(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const TileCall& t, cudaStream_t st) {
    const mgc_attention_args& a = t.c.a;
    switch ((a.cap > 0.0f ? CAP : 0) | (a.slopes ? SLOPE : 0) | (a.dist_bias ? TABLE : 0)) {
        case 0: launch_tile<BF16, DP, 0>(mq, mk, mv, t, st); break;
        case 1: launch_tile<BF16, DP, 1>(mq, mk, mv, t, st); break;
        case 2: launch_tile<BF16, DP, 2>(mq, mk, mv, t, st); break;
        case 3: launch_tile<BF16, DP, 3>(mq, mk, mv, t, st); break;
        case 4: launch_tile<BF16, DP, 4>(mq, mk, mv, t, st); break;
        case 5: launch_tile<BF16, DP, 5>(mq, mk, mv, t, st); break;
        case 6: launch_tile<BF16, DP, 6>(mq, mk, mv, t, st); break;
        default: launch_tile<BF16, DP, 7>(mq, mk, mv, t, st); break;
    }
}

// One translation unit per type (and head size): they compile side by side.
void launch_tile_f16_64(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const TileCall&, cudaStream_t);
void launch_tile_f16_128(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const TileCall&, cudaStream_t);
void launch_tile_bf16_64(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const TileCall&, cudaStream_t);
void launch_tile_bf16_128(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const TileCall&, cudaStream_t);
void launch_tile_gives_up(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const TileCall&, cudaStream_t);   // f16, up to 64, a table

}  // namespace at
}  // namespace mgc
