// logits.cu -- mgc_logits_adjust: penalties for repeated tokens, a bias and a bit mask on logits.
//
//   z = z > 0 ? z / rep : z * rep,  z -= freq * c + pres     for tokens seen c > 0 times
//   z += bias[v];   z = -inf where the token's bit is 0
//
// Bound by memory: each logit is read and written once, everything else (a row's history, a shared
// bias or mask) comes from L2.  One CTA owns a chunk of consecutive tokens of one row.  It counts the
// row's history into shared memory for those tokens only, so counting needs neither a second kernel
// nor a [R][V] table in global memory: the price is that each of a row's chunks reads the history
// again, from L2.  Chunks are up to 8192 tokens, which keeps that small; with few rows they are
// shorter, so that all SMs have work.  After the count each warp works on its own segments, with no barrier
// between warps.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/mgc.h"
#include "kernels.h"
#include "tma.cuh"

namespace mgc {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;

struct LogitArgs {
    const void* z; long long ld;
    int R, V, chunks;
    const int32_t* hist; long long ld_hist; int L;
    const int32_t* hist_len;
    const float* pen; long long ld_pen;
    const float* bias; long long ld_bias;
    const uint32_t* allowed; long long ld_allowed;
    void* out; long long ld_out;
};

template <int N, int SHIFT>
__device__ __forceinline__ void add_at(float (&z)[N], const float (&x)[N + 4]) {
#pragma unroll
    for (int j = 0; j < N; j++) z[j] += x[j + SHIFT];
}
// A token that the history holds `count` times.
__device__ __forceinline__ float penalise(float z, uint32_t count, float rep, float freq, float pres) {
    return count ? (z > 0.0f ? z / rep : z * rep) - (freq * (float)count + pres) : z;
}

template <int DT> struct Elem;   // DT: 0 f32, 1 f16, 2 bf16; a 16-byte vector holds N values
template <> struct Elem<0> {
    static constexpr int N = 4, SIZE = 4;
    __device__ static float get(const uint4& v, int i) { return __uint_as_float((&v.x)[i]); }
    __device__ static void set2(uint4& v, int i, float a, float b) {
        (&v.x)[i] = __float_as_uint(a);
        (&v.x)[i + 1] = __float_as_uint(b);
    }
    __device__ static float load(const void* p, long long i) { return reinterpret_cast<const float*>(p)[i]; }
    __device__ static void store(void* p, long long i, float v) { reinterpret_cast<float*>(p)[i] = v; }
};
template <bool BF16> struct Elem16 {
    static constexpr int N = 8, SIZE = 2;
    __device__ static float get(const uint4& v, int i) {
        const float2 f = unpack16<BF16>((&v.x)[i >> 1]);
        return i & 1 ? f.y : f.x;
    }
    __device__ static void set2(uint4& v, int i, float a, float b) { (&v.x)[i >> 1] = pack16<BF16>(a, b); }
    __device__ static float load(const void* p, long long i) { return load16<BF16>(p, i); }
    __device__ static void store(void* p, long long i, float v) { store16<BF16>(p, i, v); }
};
template <> struct Elem<1> : Elem16<false> {};
template <> struct Elem<2> : Elem16<true> {};

// A chunk starts at a 16-byte boundary of the logits' memory, so rows that begin in the middle of one
// (odd V) still move whole vectors: chunk c of a row holds tokens [c * chunk - lead, ...), lead = the
// values between the boundary below the row's first logit and that logit.
// SEGS: segments of 32 vectors per warp and chunk; their logits are all requested at the start (a
// warp that fetched one segment ahead kept 16 KB per SM in flight: 2 TB/s).
template <int DT, int SEGS, bool HIST, bool BIAS, bool MASK>
__global__ void __launch_bounds__(kThreads, 3) logits_adjust_kernel(const LogitArgs a) {
    using E = Elem<DT>;
    constexpr int N = E::N, SEG = 32 * N;
    extern __shared__ __align__(16) uint32_t s_count[];   // [chunk]
    griddep_wait();
    griddep_launch();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int chunk = SEGS * kWarps * SEG;
    const long long r = blockIdx.x / a.chunks;
    const int c = (int)(blockIdx.x % a.chunks);
    const char* zrow = reinterpret_cast<const char*>(a.z) + r * a.ld * E::SIZE;
    char* orow = reinterpret_cast<char*>(a.out) + r * a.ld_out * E::SIZE;
    const int lead = (int)((reinterpret_cast<uintptr_t>(zrow) & 15) / E::SIZE);
    const bool out_vec = ((reinterpret_cast<uintptr_t>(zrow) ^ reinterpret_cast<uintptr_t>(orow)) & 15) == 0;
    const int t0 = c * chunk - lead;   // token of the chunk's first value (may be < 0); V + chunk < 2^31
    if (t0 >= a.V) return;   // (chunks are counted for the longest lead: a row with less may not fill the last)
    const float* brow = BIAS ? a.bias + r * a.ld_bias : nullptr;

    auto seg_at = [&](int k) { return (k * kWarps + warp) * SEG; };   // segment k's place in the chunk
    // a segment without a row's end (nor, where bias is read in aligned pieces, its neighbourhood)
    auto inside = [&](int t) { return t >= (BIAS ? 4 : 0) && t + SEG + (BIAS ? 4 : 0) <= a.V; };
    uint4 v[SEGS];
#pragma unroll
    for (int k = 0; k < SEGS; k++) {
        const int t = t0 + seg_at(k);
        if (inside(t)) v[k] = *reinterpret_cast<const uint4*>(zrow + (long long)(t + lane * N) * E::SIZE);
    }
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    bool any = false;
    if (HIST) {
        int n = a.L;
        if (a.hist_len) n = max(0, min(a.L, __ldg(a.hist_len + r)));
        const float* pen = a.pen + r * a.ld_pen;
        rep = __ldg(pen); freq = __ldg(pen + 1); pres = __ldg(pen + 2);
        for (int i = tid; i < chunk / 4; i += kThreads) reinterpret_cast<uint4*>(s_count)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        const int32_t* h = a.hist + r * a.ld_hist;
        const int first = max(t0, 0);
        const unsigned span = (unsigned)(min(t0 + chunk, a.V) - first);   // > 0: t0 < V
        auto count = [&](int tok) {
            if ((unsigned)tok - (unsigned)first < span) {   // (a negative number is a large one)
                atomicAdd(s_count + (tok - t0), 1u);   // integers: the order does not matter
                any = true;
            }
        };
        // four at a time from the first 16-byte boundary on
        const int head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(h) & 15)) & 15) / 4), quads = (n - head) / 4;
        if (tid < head) count(__ldg(h + tid));
#pragma unroll 4
        for (int i = tid; i < quads; i += kThreads) {
            const int4 q = __ldg(reinterpret_cast<const int4*>(h + head) + i);
            count(q.x); count(q.y); count(q.z); count(q.w);
        }
        const int done = head + quads * 4;
        if (tid < n - done) count(__ldg(h + done + tid));
        any = __syncthreads_or(any);
    }

    const uint32_t* mask = MASK ? a.allowed + r * a.ld_allowed : nullptr;
#pragma unroll
    for (int k = 0; k < SEGS; k++) {
        const int at = seg_at(k) + lane * N, t = t0 + at;
        if (inside(t0 + seg_at(k))) {
            float z[N];
#pragma unroll
            for (int j = 0; j < N; j++) z[j] = E::get(v[k], j);
            if (HIST && any) {
#pragma unroll
                for (int j = 0; j < N; j += 4) {
                    const uint4 u = *reinterpret_cast<const uint4*>(s_count + at + j);
                    if (u.x | u.y | u.z | u.w) {
                        z[j] = penalise(z[j], u.x, rep, freq, pres);
                        z[j + 1] = penalise(z[j + 1], u.y, rep, freq, pres);
                        z[j + 2] = penalise(z[j + 2], u.z, rep, freq, pres);
                        z[j + 3] = penalise(z[j + 3], u.w, rep, freq, pres);
                    }
                }
            }
            if (BIAS) {
                // aligned loads around the N values, which start at one of four places (the same for the warp)
                const int shift = (int)(reinterpret_cast<uintptr_t>(brow + t) >> 2 & 3);
                const float4* q = reinterpret_cast<const float4*>(brow + t - shift);
                float x[N + 4];
#pragma unroll
                for (int j = 0; j < N / 4; j++) {
                    const float4 f = __ldg(q + j);
                    x[4 * j] = f.x; x[4 * j + 1] = f.y; x[4 * j + 2] = f.z; x[4 * j + 3] = f.w;
                }
                if (shift == 0) add_at<N, 0>(z, x);
                else {
                    const float4 f = __ldg(q + N / 4);
                    x[N] = f.x; x[N + 1] = f.y; x[N + 2] = f.z; x[N + 3] = f.w;
                    if (shift == 1) add_at<N, 1>(z, x);
                    else if (shift == 2) add_at<N, 2>(z, x);
                    else add_at<N, 3>(z, x);
                }
            }
            if (MASK) {   // N bits from token t on: at most two words
                const uint32_t lo = __ldg(mask + (t >> 5)), hi = __ldg(mask + ((t + N - 1) >> 5));
                const uint32_t bits = __funnelshift_r(lo, hi, (uint32_t)(t & 31));
#pragma unroll
                for (int j = 0; j < N; j++) z[j] = bits >> j & 1 ? z[j] : -INFINITY;
            }
            uint4 o;
#pragma unroll
            for (int j = 0; j < N; j += 2) E::set2(o, j, z[j], z[j + 1]);
            if (out_vec) *reinterpret_cast<uint4*>(orow + (long long)t * E::SIZE) = o;
            else {
#pragma unroll
                for (int j = 0; j < N; j++) E::store(orow, t + j, E::get(o, j));
            }
        } else {   // the segment of a row's first or last logits
#pragma unroll 1
            for (int j = 0; j < N; j++) {
                const int i = seg_at(k) + j * 32 + lane, x = t0 + i;
                if (x < 0 || x >= a.V) continue;
                float z = E::load(zrow, x);
                if (HIST) z = penalise(z, s_count[i], rep, freq, pres);
                if (BIAS) z += __ldg(brow + x);
                if (MASK && !(__ldg(mask + (x >> 5)) >> (x & 31) & 1)) z = -INFINITY;
                E::store(orow, x, z);
            }
        }
    }
}

template <int DT, int SEGS, bool HIST, bool BIAS, bool MASK>
void launch_one(const LogitArgs& a, cudaStream_t st) {
    static std::atomic<uint64_t> done{0};
    auto kernel = logits_adjust_kernel<DT, SEGS, HIST, BIAS, MASK>;
    const uint32_t smem = HIST ? SEGS * kWarps * 32 * Elem<DT>::N * 4 : 0;   // at most 32 KB
    if (smem) allow_smem(kernel, smem, done);
    ++g_launch_count;
    const cudaError_t e = launch_k(kernel, dim3((unsigned)((long long)a.chunks * a.R)), dim3(kThreads), smem, st, a);
    if (e != cudaSuccess) throw std::runtime_error(std::string("launch failed: ") + cudaGetErrorString(e));
}
template <int DT, int SEGS>
void launch_segs(LogitArgs& a, long long chunks, cudaStream_t st) {
    a.chunks = (int)chunks;
    if (chunks * a.R > 0x7fffffffLL) throw std::runtime_error("R * V is too large for one launch");
    const bool h = a.hist, b = a.bias, m = a.allowed;
    if (h && b && m) launch_one<DT, SEGS, true, true, true>(a, st);
    else if (h && b) launch_one<DT, SEGS, true, true, false>(a, st);
    else if (h && m) launch_one<DT, SEGS, true, false, true>(a, st);
    else if (h) launch_one<DT, SEGS, true, false, false>(a, st);
    else if (b && m) launch_one<DT, SEGS, false, true, true>(a, st);
    else if (b) launch_one<DT, SEGS, false, true, false>(a, st);
    else if (m) launch_one<DT, SEGS, false, false, true>(a, st);
    else launch_one<DT, SEGS, false, false, false>(a, st);
}

// Long chunks read the history less often (256 x 128257 bf16 with all parts: 57 us; twice as long,
// fewer blocks fit an SM: 62; half as long: 80); short ones give every SM work when there are few rows.
template <int DT>
void launch_logits(LogitArgs& a, cudaStream_t st) {
    constexpr int N = Elem<DT>::N;
    const long long enough = 4LL * current_sms();
    // a row may start up to N - 1 values past a boundary
    auto chunks = [&](int segs) { return ((long long)a.V + N - 1 + kWarps * 32 * N * segs - 1) / (kWarps * 32 * N * segs); };
    if (chunks(2) * a.R >= enough) launch_segs<DT, 2>(a, chunks(2), st);
    else launch_segs<DT, 1>(a, chunks(1), st);
}

}  // namespace
}  // namespace mgc

using namespace mgc;

extern "C" int mgc_logits_adjust(int dtype, const void* z, int64_t ld, int R, int V, const int32_t* hist,
                                 int64_t ld_hist, int L, const int32_t* hist_len, const float* pen, int64_t ld_pen,
                                 const float* bias, int64_t ld_bias, const uint32_t* allowed, int64_t ld_allowed,
                                 void* out, int64_t ld_out, void* stream) {
    return guarded("mgc_logits_adjust", [&] {
        auto need = [](bool ok, const char* m) { if (!ok) throw std::invalid_argument(m); };
        need(dtype == MGC_F32 || dtype == MGC_F16 || dtype == MGC_BF16, "dtype must be F32, F16 or BF16");
        need(R >= 0 && V >= 0 && L >= 0, "negative size");
        need(V <= 1 << 30, "V must be at most 2^30");
        if (R == 0 || V == 0) return;
        need(z && out, "logits and out must not be NULL");
        need((hist != nullptr) == (pen != nullptr), "history and penalties are given together");
        const int size = dtype == MGC_F32 ? 4 : 2;
        need(((uintptr_t)z | (uintptr_t)out) % size == 0, "logits and out must be aligned to their type");
        need(((uintptr_t)hist | (uintptr_t)hist_len | (uintptr_t)pen | (uintptr_t)bias | (uintptr_t)allowed) % 4 == 0,
             "history, penalties, bias and allowed must be 4-byte aligned");
        need(ld >= V || R == 1, "ld must be at least V");
        need(ld_out >= V || R == 1, "ld_out must be at least V");
        need(z != out || ld == ld_out || R == 1, "in place, ld_out must be ld");
        need(!hist || ld_hist == 0 || ld_hist >= L, "ld_history must be 0 or at least L");
        need(!pen || ld_pen == 0 || ld_pen >= 3, "ld_penalties must be 0 or at least 3");
        need(!bias || ld_bias == 0 || ld_bias >= V, "ld_bias must be 0 or at least V");
        need(!allowed || ld_allowed == 0 || ld_allowed >= ((int64_t)V + 31) / 32,
             "ld_allowed must be 0 or at least (V + 31) / 32");
        LogitArgs a{z, ld, R, V, 0, hist, ld_hist, L, hist_len, pen, ld_pen, bias, ld_bias, allowed, ld_allowed, out, ld_out};
        if (L == 0) a.hist = nullptr;   // an empty history
        const cudaStream_t st = (cudaStream_t)stream;
        if (dtype == MGC_F32) launch_logits<0>(a, st);
        else if (dtype == MGC_F16) launch_logits<1>(a, st);
        else launch_logits<2>(a, st);
    });
}
