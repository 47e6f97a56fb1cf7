// linear16.cu -- mgc_linear: y = act(x W^T + bias) + resid in f16 / bf16 on tcgen05 tensor cores.
//
// Both kernels compute the transposed product: W's rows are the MMA's M axis (TMEM lanes) and x's
// rows its N axis (TMEM columns).  A warp then holds 32 consecutive outputs n of one row m in its
// lanes, so results, residual and bias move between registers and memory in consecutive addresses
// without a staging tile, whatever the alignment of y's rows, and a call with few rows (one token)
// wastes columns of a narrow tile instead of 127 lanes of a wide one.
//
// Operands come by tensor maps with the 128-byte swizzle, 64 k at a time; what lies outside the
// tensors reads as zero, so K, N and M need no padding.
#include <algorithm>
#include <atomic>

#include "../../include/mgc.h"
#include "kernels.h"
#include "tma.cuh"

namespace mgc {
namespace {

constexpr int BK = 64;         // k per stage: one 128-byte swizzle row
constexpr int TILE_N = 128;    // outputs n per CTA (TMEM lanes)
constexpr uint32_t A_BYTES = TILE_N * BK * 2;

struct LinArgs {
    int M, N, K;
    const float* bias;
    const void* resid; long long ldr;
    void* y; long long ldy;
    int act;
};

// x Phi(x) = max(x, 0) - |x| h(|x|), h(a) = 0.5 erfc(a / sqrt 2) = e^(-a^2 / 2) t P(t), t = 1 / (1 + 0.26 a):
// the form of Abramowitz and Stegun 7.1.26, with seven coefficients fitted here to a relative error
// of 8.4e-7 on 0 <= a <= 13 (beyond, h is below 2^-120), so small results keep their precision.
// 11 FP32 operations and two MUFU against erff's ~25 and a branch: the epilogue of a 256 x 256 tile
// has to fit under its MMAs.
__device__ __forceinline__ float gelu16(float x) {
    const float a = fminf(fabsf(x), 30.0f);
    float t;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.26f, a, 1.0f)));
    float p = fmaf(-0.0729497778f, t, 0.229241262f);
    p = fmaf(p, t, -0.107327773f);
    p = fmaf(p, t, 0.167471854f);
    p = fmaf(p, t, 0.0727312424f);
    p = fmaf(p, t, 0.107331982f);
    p = fmaf(p, t, 0.103501627f);
    const float h = ex2_approx(a * a * -0.7213475204f) * (p * t);
    const float half = 0.5f * x;
    return fmaf(-a, h, half + fabsf(half));   // (max(x, 0) with a NaN that stays one; x + |x| would overflow)
}
// x / (1 + e^-x), from e^-|x| so that nothing overflows: small results keep their precision too.
__device__ __forceinline__ float silu16(float x) {
    float e, r;   // (e may be subnormal: no flush)
    asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(fabsf(x) * -1.4426950409f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return x * (x < 0.0f ? e : 1.0f) * r;
}
__device__ __forceinline__ float act16(float v, int a) { return a == 1 ? gelu16(v) : a == 2 ? silu16(v) : v; }
template <int N>
__device__ __forceinline__ void act16_all(float (&v)[N], int a) {
    if (a == 1) {
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = gelu16(v[j]);
    } else if (a == 2) {
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = silu16(v[j]);
    }
}

// 32 accumulators of one output n, for x rows m .. m + 31: a warp moves 32 consecutive n of a row
// at a time, 2 bytes a lane.
template <bool BF16>
__device__ __forceinline__ void finish_cols(const uint32_t (&acc)[32], const LinArgs& a, int m, int n, float bias,
                                            int cols = 32) {
    const int rows = min(cols, a.M - m);   // (a 16-column tile has 16)
    uint16_t* y = reinterpret_cast<uint16_t*>(a.y) + m * a.ldy + n;
    const uint16_t* r = a.resid ? reinterpret_cast<const uint16_t*>(a.resid) + m * a.ldr + n : nullptr;
    float v[32], res[32];
    if (r) {
#pragma unroll
        for (int j = 0; j < 32; j++) {
            res[j] = j < rows ? load16<BF16>(r, 0) : 0.0f;
            r += a.ldr;
        }
    }
#pragma unroll
    for (int j = 0; j < 32; j++) v[j] = __uint_as_float(acc[j]) + bias;
    act16_all(v, a.act);
    if (r) {
#pragma unroll
        for (int j = 0; j < 32; j++) v[j] += res[j];
    }
#pragma unroll
    for (int j = 0; j < 32; j++) {
        if (j < rows) store16<BF16>(y, 0, v[j]);
        y += a.ldy;
    }
}

// 32 accumulators of one x row m, for outputs n .. n + 31 (N a multiple of 8; bias, and the rows of y
// and resid, 16-byte aligned): 16 bytes a move.
template <bool BF16>
__device__ __forceinline__ void finish_row(const uint32_t (&acc)[32], const LinArgs& a, int m, int n) {
    const int groups = min(4, (a.N - n) / 8);
    uint4 res[4];
    if (a.resid) {
        const uint4* r = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.resid) + m * a.ldr + n);
#pragma unroll
        for (int g = 0; g < 4; g++) res[g] = g < groups ? __ldcs(r + g) : make_uint4(0, 0, 0, 0);
    }
    float v[32];
    if (a.bias) {
#pragma unroll
        for (int g = 0; g < 4; g++) {
            float4 b0 = make_float4(0, 0, 0, 0), b1 = b0;
            if (g < groups) {
                const float4* b = reinterpret_cast<const float4*>(a.bias + n + 8 * g);
                b0 = __ldg(b);
                b1 = __ldg(b + 1);
            }
            const float b[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
#pragma unroll
            for (int j = 0; j < 8; j++) v[8 * g + j] = __uint_as_float(acc[8 * g + j]) + b[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 32; j++) v[j] = __uint_as_float(acc[j]);
    }
    act16_all(v, a.act);
    uint4* y = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.y) + m * a.ldy + n);
#pragma unroll
    for (int g = 0; g < 4; g++) {
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float2 f = make_float2(v[8 * g + 2 * j], v[8 * g + 2 * j + 1]);
            if (a.resid) {
                const float2 x = unpack16<BF16>((&res[g].x)[j]);
                f.x += x.x;
                f.y += x.y;
            }
            o[j] = pack16<BF16>(f.x, f.y);
        }
        if (g < groups) y[g] = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

// ------------------------------------------------------------------ few rows or few tiles
// One 128 n x BN m tile, its k range split over the CTAs of a cluster so that a small product
// still reads its weight with every SM.  The partial sums meet in distributed shared memory and
// are added in rank order: no workspace, no atomics, one launch.
namespace ls {
constexpr int THREADS = 192;   // warp 0 copies, warp 1 issues MMAs, warps 2-5 read the result
template <int BN> constexpr int stages() { return BN <= 32 ? 5 : BN <= 64 ? 8 : 6; }
template <int BN> constexpr uint32_t stage_bytes() { return A_BYTES + BN * BK * 2; }
template <int BN> constexpr uint32_t ring() { return stages<BN>() * stage_bytes<BN>(); }
template <int BN> constexpr uint32_t smem() { return 1024 + ring<BN>() + 256; }
}  // namespace ls

template <bool BF16, int BN>
__global__ void __launch_bounds__(ls::THREADS) linear_split_kernel(const __grid_constant__ CUtensorMap mw,
                                                                   const __grid_constant__ CUtensorMap mx,
                                                                   const LinArgs a, int split) {
    constexpr int ST = ls::stages<BN>();
    constexpr uint32_t SB = ls::stage_bytes<BN>(), COLS = BN < 32 ? 32 : BN;
    static_assert((uint32_t)(BN + 8) * TILE_N * 4 <= ls::ring<BN>(), "the partial tile reuses the ring");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = align1024_smem(smem_raw);
    uint64_t* full = (uint64_t*)(sm + ls::ring<BN>());
    uint64_t* empty = full + ST;
    uint64_t* done = empty + ST;
    uint32_t* tmem_slot = (uint32_t*)(done + 1);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = blockIdx.x % split, tile = blockIdx.x / split;
    const int ntn = (a.N + TILE_N - 1) / TILE_N;
    const int n0 = tile % ntn * TILE_N, m0 = tile / ntn * BN;
    const int ks = (a.K + BK - 1) / BK;
    const int k0 = (int)((long long)ks * rank / split), nk = (int)((long long)ks * (rank + 1) / split) - k0;

    auto load = [&](int i) {
        const int s = i % ST;
        mbar_arrive_expect_tx(full + s, SB);
        tma_load_2d(sm + s * SB, &mw, (k0 + i) * BK, n0, full + s);
        tma_load_2d(sm + s * SB + A_BYTES, &mx, (k0 + i) * BK, m0, full + s);
    };
    if (tid == 0) {
        for (int i = 0; i < ST; i++) { mbar_init(full + i, 1); mbar_init(empty + i, 1); }
        mbar_init(done, 1);
        *abort_flag = 0;
        mbar_fence_init();
        griddep_wait();
        for (int i = 0; i < min(ST, nk); i++) load(i);   // under the rest of the set-up
    }
    if (warp == 1) tmem_alloc(tmem_slot, COLS);
    griddep_wait();
    griddep_launch();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0 && lane == 0) {
        int i = min(ST, nk);
        for (; i < nk; i++) {
            if (!mbar_wait(empty + i % ST, (i / ST - 1) & 1, abort_flag, 41)) break;
            load(i);
        }
        if (i < nk) {   // gave up: let the copies in flight land
            volatile int never = 0;
            for (int t = std::max(0, i - ST); t < i; t++) mbar_wait(full + t % ST, (t / ST) & 1, &never, 42);
        }
    } else if (warp == 1 && lane == 0) {
        constexpr uint32_t idesc = idesc_make(1, BF16, BF16, TILE_N, BN);
        bool ok = true;
        for (int i = 0; i < nk; i++) {
            const int s = i % ST;
            if (!(ok = mbar_wait(full + s, (i / ST) & 1, abort_flag, 43))) break;
            tc_fence_after();
            const uint64_t da = sdesc_sw128(smem_u32(sm + s * SB)), db = sdesc_sw128(smem_u32(sm + s * SB + A_BYTES));
#pragma unroll
            for (int k = 0; k < BK / 16; k++) mma_f16(tmem, da + 2 * k, db + 2 * k, idesc, (i | k) != 0);
            mma_commit(empty + s);
        }
        if (ok) mma_commit(done);
    }
    // every warp waits for the accumulator: past it nothing reads or writes the ring any more
    __syncwarp();
    const bool ok = __all_sync(0xffffffffu, mbar_wait(done, 0, abort_flag, 44));
    tc_fence_after();
    const int quad = warp & 3, n = n0 + quad * 32 + lane;   // warps 2-5: TMEM lanes 32 (warp % 4) ..
    const uint32_t t_row = tmem + ((uint32_t)(quad * 32) << 16);
    const float bias = warp >= 2 && a.bias && n < a.N ? __ldg(a.bias + n) : 0.0f;
    if (split == 1) {
        if (warp >= 2 && ok) {
#pragma unroll 1
            for (int c = 0; c < BN; c += 32) {
                if (m0 + c >= a.M) break;
                uint32_t acc[32];
                if (BN >= 32) tmem_ld32(t_row + c, acc);
                else tmem_ld16(t_row + c, acc);
                tmem_ld_wait();
                if (BN < 32) for (int j = 16; j < 32; j++) acc[j] = 0;
                if (n < a.N) finish_cols<BF16>(acc, a, m0 + c, n, bias, min(32, BN));
            }
        }
    } else {
        float* part = reinterpret_cast<float*>(sm);   // [BN][128 n]
        const int cols = min(BN, a.M - m0);
        if (warp >= 2 && ok) {
#pragma unroll 1
            for (int c = 0; c < cols; c += 16) {
                uint32_t acc[16];
                tmem_ld16(t_row + c, acc);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; j++) part[(c + j) * TILE_N + quad * 32 + lane] = __uint_as_float(acc[j]);
            }
        }
        __syncwarp();
        cluster_sync_all();
        if (warp >= 2 && ok && n < a.N) {
            constexpr int G = BN == 16 ? 2 : 8;   // columns in flight: remote reads take a microsecond
            const int c0 = cols * rank / split, c1 = cols * (rank + 1) / split;   // this CTA's columns
#pragma unroll 1
            for (int c = c0; c < c1; c += G) {
                float v[G], res[G];
#pragma unroll
                for (int j = 0; j < G; j++) {
                    v[j] = 0.0f;
                    res[j] = a.resid && c + j < c1 ? load16<BF16>(a.resid, (m0 + c + j) * a.ldr + n) : 0.0f;
                }
#pragma unroll 4
                for (int p = 0; p < split; p++) {
                    const uint32_t at = mapa_u32(part + c * TILE_N + quad * 32 + lane, p);
#pragma unroll
                    for (int j = 0; j < G; j++) {   // (columns past c1 lie inside the ring: read, not used)
                        float x;
                        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(at + j * TILE_N * 4) : "memory");
                        v[j] += x;
                    }
                }
#pragma unroll
                for (int j = 0; j < G; j++) {
                    if (c + j >= c1) break;
                    v[j] = act16(v[j] + bias, a.act);
                    if (a.resid) v[j] += res[j];
                    store16<BF16>(a.y, (m0 + c + j) * a.ldy + n, v[j]);
                }
            }
        }
        __syncwarp();
        cluster_sync_all();   // the partial tiles live until every CTA has read them
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, COLS);
    }
}

// ------------------------------------------------------------------ many tiles
// A pair of CTAs owns 256 n x 256 m: each loads its half of both operands (64 KB of a stage's
// 64 KB arrive once per pair), the even CTA issues M256 x N256 MMAs that read both halves, and each
// CTA keeps its 128 n x 256 m accumulator in its own TMEM, twice, so that the epilogue of one tile
// runs under the MMAs of the next.  Persistent over tiles.
namespace lp {
constexpr int ST = 6, THREADS = 384;   // warp 0 copies, warp 1 issues MMAs, warps 4-11 read results
constexpr int TN = 256, TM = 256;
constexpr uint32_t SB = 2 * A_BYTES, RING = ST * SB, SMEM = 1024 + RING + 256;
// tiles walk 16 m-tiles before the next n-tile, so that both operands come from L2 (8192 x 4096 x 14336:
// 727 us; 8 m-tiles 738, 4 769, 32 776)
constexpr int GROUP = 16;
}  // namespace lp

// ROWS: x's rows are the lanes (a thread holds consecutive n of one row and moves 16 bytes at a
// time, 1/8 of the instructions), where y's and resid's rows allow it; else W's rows are, as above.
template <bool BF16, bool ROWS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(lp::THREADS, 1)
    linear_pair_kernel(const __grid_constant__ CUtensorMap mw, const __grid_constant__ CUtensorMap mx, const LinArgs a) {
    using namespace lp;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = align1024_smem(smem_raw);
    uint64_t* full = (uint64_t*)(sm + RING);   // [ST] even CTA: both CTAs' copies of the stage landed
    uint64_t* empty = full + ST;               // [ST] the MMAs that read the stage are done
    uint64_t* acc_full = empty + ST;           // [2]
    uint64_t* acc_empty = acc_full + 2;        // [2] even CTA: 16 epilogue warps have read it
    uint32_t* tmem_slot = (uint32_t*)(acc_empty + 2);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_ctarank();
    const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
    const int ks = (a.K + BK - 1) / BK;
    const int ntn = (a.N + TN - 1) / TN, ntm = (a.M + TM - 1) / TM;
    const int tiles = ntn * ntm;
    auto tile_at = [&](int t, int& n0, int& m0) {
        const int per = GROUP * ntn, g = t / per, first = g * GROUP, size = min(GROUP, ntm - first), r = t - g * per;
        m0 = (first + r % size) * TM;
        n0 = r / size * TN;
    };

    if (tid == 0) {
        for (int i = 0; i < ST; i++) { mbar_init(full + i, 1); mbar_init(empty + i, 1); }
        for (int i = 0; i < 2; i++) { mbar_init(acc_full + i, 1); mbar_init(acc_empty + i, 16); }
        *abort_flag = 0;
        mbar_fence_init();
        tma_prefetch_map(&mw);
        tma_prefetch_map(&mx);
    }
    if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
    griddep_wait();
    griddep_launch();
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();   // both CTAs' barriers are initialised
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0 && lane == 0) {
        int it = 0;
        bool ok = true;
        for (int t = pair; ok && t < tiles; t += npairs) {
            int n0, m0;
            tile_at(t, n0, m0);
            for (int k = 0; k < ks; k++, it++) {
                const int s = it % ST;
                if (it >= ST && !(ok = mbar_wait(empty + s, (it / ST - 1) & 1, abort_flag, 45))) break;
                if (rank == 0) mbar_arrive_expect_tx(full + s, 2 * SB);
                const uint32_t bar = mapa_u32(full + s, 0);
                tma_load_2d_pair(sm + s * SB + (ROWS ? A_BYTES : 0), &mw, k * BK, n0 + (int)rank * 128, bar);
                tma_load_2d_pair(sm + s * SB + (ROWS ? 0 : A_BYTES), &mx, k * BK, m0 + (int)rank * 128, bar);
            }
        }
        if (!ok && rank == 0) {
            volatile int never = 0;
            for (int t = max(0, it - ST); t < it; t++) mbar_wait(full + t % ST, (t / ST) & 1, &never, 42);
        }
    } else if (warp == 1 && lane == 0 && rank == 0) {
        constexpr uint32_t idesc = idesc_make(1, BF16, BF16, TN, TM);
        int it = 0, n = 0;
        bool ok = true;
        for (int t = pair; ok && t < tiles; t += npairs, n++) {
            const int b = n & 1;
            if (n >= 2 && !(ok = mbar_wait(acc_empty + b, (n / 2 - 1) & 1, abort_flag, 46))) break;
            tc_fence_after();
            for (int k = 0; k < ks; k++, it++) {
                const int s = it % ST;
                if (!(ok = mbar_wait(full + s, (it / ST) & 1, abort_flag, 47))) break;
                tc_fence_after();
                const uint64_t da = sdesc_sw128(smem_u32(sm + s * SB)), db = sdesc_sw128(smem_u32(sm + s * SB + A_BYTES));
#pragma unroll
                for (int kk = 0; kk < BK / 16; kk++)
                    mma_f16_pair(tmem + b * TM, da + 2 * kk, db + 2 * kk, idesc, (k | kk) != 0);
                mma_commit_pair(empty + s);
            }
            if (ok) mma_commit_pair(acc_full + b);
        }
    } else if (warp >= 4) {
        const int quad = warp & 3, half = (warp - 4) >> 2;
        int n = 0;
        for (int t = pair; t < tiles; t += npairs, n++) {
            const int b = n & 1;
            int n0, m0;
            tile_at(t, n0, m0);
            const int own = (ROWS ? m0 : n0) + (int)rank * 128 + quad * 32 + lane;   // this lane's row or output
            const float bias = !ROWS && a.bias && own < a.N ? __ldg(a.bias + own) : 0.0f;
            if (!__all_sync(0xffffffffu, mbar_wait(acc_full + b, (n / 2) & 1, abort_flag, 48))) break;
            tc_fence_after();
            const uint32_t t_row = tmem + ((uint32_t)(quad * 32) << 16) + b * TM + half * 128;
#pragma unroll 1
            for (int c = 0; c < 128; c += 32) {
                const int other = (ROWS ? n0 : m0) + half * 128 + c;
                if (other >= (ROWS ? a.N : a.M)) break;
                uint32_t acc[32];
                tmem_ld32(t_row + c, acc);
                tmem_ld_wait();
                if (own < (ROWS ? a.M : a.N)) {
                    if (ROWS) finish_row<BF16>(acc, a, own, other);
                    else finish_cols<BF16>(acc, a, other, own, bias);
                }
                __syncwarp();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(mapa_u32(acc_empty + b, 0));
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();   // no CTA leaves while its pair may still signal or read it
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, 512);
    }
}

// ------------------------------------------------------------------ host
CUtensorMap operand_map(const void* p, bool bf16, int rows, int K, long long ld, int box_rows) {
    const uint64_t dims[2] = {(uint64_t)K, (uint64_t)rows}, strides[1] = {(uint64_t)ld};
    const uint32_t box[2] = {BK, (uint32_t)box_rows};
    return make_map16(p, bf16, 2, dims, strides, box);
}

template <bool BF16, int BN>
void run_split(const void* w, long long ldw, const void* x, long long ldx, const LinArgs& a, int split, cudaStream_t st) {
    static std::atomic<uint64_t> done{0};
    auto kernel = linear_split_kernel<BF16, BN>;
    allow_smem(kernel, ls::smem<BN>(), done);
    const CUtensorMap mw = operand_map(w, BF16, a.N, a.K, ldw, TILE_N), mx = operand_map(x, BF16, a.M, a.K, ldx, BN);
    const long long tiles = (long long)((a.N + TILE_N - 1) / TILE_N) * ((a.M + BN - 1) / BN);
    if (tiles * split > 0x7fffffffLL) throw std::runtime_error("M * N is too large for one launch");
    launch_clusters(kernel, (unsigned)(tiles * split), ls::THREADS, ls::smem<BN>(), split, st, mw, mx, a, split);
}

template <bool BF16>
void run_linear(const void* w, long long ldw, const void* x, long long ldx, const LinArgs& a, cudaStream_t st) {
    const int sms = current_sms();
    const long long big = (long long)((a.N + lp::TN - 1) / lp::TN) * ((a.M + lp::TM - 1) / lp::TM);
    const int ks = (a.K + BK - 1) / BK;
    // The kernel, tile and split of the least estimated time, in us, from measurements on a B200: a tile
    // of bn columns takes 16 KB + 128 bn bytes a k step, which an SM gets from L2 at about 55 bytes a
    // clock; set-up and launch 3.5 us; a split adds its join.  Measured against the estimate: 257 x
    // 768 x 2304 in 64 columns 7.3 (7.1), in 128 8.0 (8.3), in 128 split in two 12.5 (10.6), in
    // pairs 13.4 (12.5); 100 x 2048 x 2048 in 64 split in four 9.8 (9.5); 4097 x 768 x 768 in 128 16.0
    // (13.2), in pairs 14.1 (12.5); 1 x 4096 x 4096 in 16 split in four 10.9 (8.5), in two 14.2 (9.7).
    const long long pair_waves = (big + sms / 2 - 1) / (sms / 2);
    double best = 9.0 + ks * 0.29 + (double)(pair_waves - 1) * std::max(ks * 0.29, 5.0);
    int bn = 256, split = 1;
    for (int n = 16; n <= 128; n *= 2) {
        if (n > 16 && n / 2 >= a.M) break;   // no wider than the rows need
        const long long tiles = (long long)((a.N + TILE_N - 1) / TILE_N) * ((a.M + n - 1) / n);
        const int per_sm = n <= 32 ? 2 : 1;   // blocks whose shared memory fits an SM
        for (int sp = 1; sp <= 8 && ks / sp >= 2; sp *= 2) {
            const long long ctas = tiles * sp;
            if (sp > 1 && (ctas > sms * per_sm || sp > 4 * per_sm)) break;   // (8 CTAs with an SM each rarely fit a GPC)
            const long long side = std::min<long long>(per_sm, (ctas + sms - 1) / sms);   // that share an SM
            const long long waves = (ctas + sms * per_sm - 1) / (sms * per_sm);
            const double step = (16384 + 128 * n) / 55.0 / 1850.0 * side;
            const double us = 3.5 + waves * ((double)((ks + sp - 1) / sp) * step + 0.2 + 0.006 * n) + (sp > 1 ? 0.8 + 0.03 * n : 0.0);
            if (us < best) { best = us; bn = n; split = sp; }
        }
    }
    if (bn == 256) {
        const bool rows = a.N % 8 == 0 && a.ldy % 8 == 0 && ((uintptr_t)a.y | (uintptr_t)a.bias) % 16 == 0 &&
                          (!a.resid || (a.ldr % 8 == 0 && (uintptr_t)a.resid % 16 == 0));
        if (big > 0x7fffffffLL) throw std::runtime_error("M * N is too large for one launch");
        const CUtensorMap mw = operand_map(w, BF16, a.N, a.K, ldw, 128), mx = operand_map(x, BF16, a.M, a.K, ldx, 128);
        const unsigned pairs = (unsigned)std::min<long long>(big, sms / 2);
        static std::atomic<uint64_t> done[2];
        auto kernel = rows ? linear_pair_kernel<BF16, true> : linear_pair_kernel<BF16, false>;
        allow_smem(kernel, lp::SMEM, done[rows]);
        launch_clusters(kernel, 2 * pairs, lp::THREADS, lp::SMEM, 0, st, mw, mx, a);
        return;
    }
    if (bn == 16) run_split<BF16, 16>(w, ldw, x, ldx, a, split, st);
    else if (bn == 32) run_split<BF16, 32>(w, ldw, x, ldx, a, split, st);
    else if (bn == 64) run_split<BF16, 64>(w, ldw, x, ldx, a, split, st);
    else run_split<BF16, 128>(w, ldw, x, ldx, a, split, st);
}

}  // namespace
}  // namespace mgc

using namespace mgc;

extern "C" int mgc_linear(int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, int M, int N, int K,
                          const float* bias, int act, const void* resid, int64_t ldr, void* y, int64_t ldy, void* stream) {
    return guarded("mgc_linear", [&] {
        auto need = [](bool ok, const char* m) { if (!ok) throw std::invalid_argument(m); };
        need(dtype == MGC_F16 || dtype == MGC_BF16, "dtype must be F16 or BF16");
        need(M >= 0 && N >= 0, "negative size");
        // (tiles and k steps are counted up to the next multiple of 256 and one more, in 32 bits)
        need(M <= 0x7ffffc00 && N <= 0x7ffffc00 && K <= 0x7ffffc00, "M, N and K must be at most 2^31 - 1024");
        need(K > 0 && K % 8 == 0, "K must be a positive multiple of 8");
        need(act >= 0 && act <= 2, "act must be 0 (none), 1 (GELU) or 2 (SiLU)");
        if (M == 0 || N == 0) return;
        need(x && w && y, "x, w and y must not be NULL");
        need(((uintptr_t)x | (uintptr_t)w) % 16 == 0, "x and w must be 16-byte aligned");
        need(((uintptr_t)y | (uintptr_t)resid) % 2 == 0 && (uintptr_t)bias % 4 == 0, "y, resid and bias must be aligned to their type");
        need((M == 1 || (ldx >= K && ldx % 8 == 0)) && (N == 1 || (ldw >= K && ldw % 8 == 0)),
             "ldx and ldw must be multiples of 8 and at least K");
        need(M == 1 || (ldy >= N && (!resid || ldr >= N)), "ldy and ldr must be at least N");
        need(y != resid || ldy == ldr || M == 1, "in place, ldy must be ldr");
        LinArgs a{M, N, K, bias, resid, ldr, y, ldy, act};
        if (dtype == MGC_BF16) run_linear<true>(w, ldw, x, ldx, a, (cudaStream_t)stream);
        else run_linear<false>(w, ldw, x, ldx, a, (cudaStream_t)stream);
    });
}
