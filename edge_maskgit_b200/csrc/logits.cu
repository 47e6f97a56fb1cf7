// logits.cu -- mgc_logits_adjust: penalties for repeated tokens, a bias and a bit mask on logits.
//
//   z = z > 0 ? z / rep : z * rep,  z -= freq * c + pres     for tokens seen c > 0 times
//   z += bias[v];   z = -inf where the token's bit is 0
//
// Bound by memory: each logit is read and written once, everything else (a row's history, a shared
// bias or mask) comes from L2.  One CTA owns kChunk consecutive tokens of one row.  It counts the
// row's history into shared memory for those tokens only, so counting needs neither a second
// kernel nor a [R][V] table in global memory: the price is that each of a row's chunks reads the
// history again, which stays in L2.  The logits' own loads are issued before the count.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/mgc.h"
#include "kernels.h"
#include "tma.cuh"

namespace mgc {
namespace {

constexpr int kThreads = 256;

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

// One logit: the formulas above, in f32.
__device__ __forceinline__ float adjust(float z, uint32_t count, float rep, float freq, float pres, float bias,
                                        bool allowed) {
    if (count) z = (z > 0.0f ? z / rep : z * rep) - (freq * (float)count + pres);
    z += bias;
    return allowed ? z : -INFINITY;
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

// VPT 16-byte vectors per thread.  A chunk starts at a 16-byte boundary of the logits' memory, so
// rows that begin in the middle of one (odd V) still load whole vectors: chunk c of a row holds
// tokens [c * CHUNK - lead, (c + 1) * CHUNK - lead), lead = the values between the boundary below
// the row's first logit and that logit.
template <int DT, int VPT, bool HIST, bool BIAS, bool MASK>
__global__ void __launch_bounds__(kThreads) logits_adjust_kernel(const LogitArgs a) {
    using E = Elem<DT>;
    constexpr int N = E::N, CHUNK = kThreads * VPT * N;
    __shared__ __align__(16) uint32_t s_count[HIST ? CHUNK : 4];
    __shared__ __align__(16) float s_bias[BIAS ? CHUNK : 4];
    griddep_wait();
    griddep_launch();
    const int tid = threadIdx.x;
    const long long r = blockIdx.x / a.chunks;
    const int c = (int)(blockIdx.x % a.chunks);
    const char* zrow = reinterpret_cast<const char*>(a.z) + r * a.ld * E::SIZE;
    char* orow = reinterpret_cast<char*>(a.out) + r * a.ld_out * E::SIZE;
    const int lead = (int)((reinterpret_cast<uintptr_t>(zrow) & 15) / E::SIZE);
    const bool out_vec = ((reinterpret_cast<uintptr_t>(zrow) ^ reinterpret_cast<uintptr_t>(orow)) & 15) == 0;
    const long long t0 = (long long)c * CHUNK - lead;   // token of the chunk's first value (may be < 0)

    uint4 v[VPT];
    auto first = [&](int i) { return t0 + (long long)(i * kThreads + tid) * N; };
    auto whole = [&](long long t) { return t >= 0 && t + N <= a.V; };
#pragma unroll
    for (int i = 0; i < VPT; i++) {
        const long long t = first(i);
        if (whole(t)) v[i] = *reinterpret_cast<const uint4*>(zrow + t * E::SIZE);
    }
    if (BIAS) {   // 4-byte copies: a row of an odd-sized table starts anywhere
        const float* b = a.bias + r * a.ld_bias;
#pragma unroll 4
        for (int i = tid; i < CHUNK; i += kThreads) {
            const long long t = t0 + i;
            if (t >= 0 && t < a.V)
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(s_bias + i)), "l"(b + t) : "memory");
        }
    }
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    bool any = false;
    if (HIST) {
        for (int i = tid; i < CHUNK / 4; i += kThreads) reinterpret_cast<uint4*>(s_count)[i] = make_uint4(0, 0, 0, 0);
        int n = a.L;
        if (a.hist_len) n = max(0, min(a.L, __ldg(a.hist_len + r)));
        const float* pen = a.pen + r * a.ld_pen;
        rep = __ldg(pen); freq = __ldg(pen + 1); pres = __ldg(pen + 2);
        __syncthreads();
        const int32_t* h = a.hist + r * a.ld_hist;
#pragma unroll 4
        for (int i = tid; i < n; i += kThreads) {
            const int tok = __ldg(h + i);
            const long long at = tok - t0;
            if (tok >= 0 && tok < a.V && at >= 0 && at < CHUNK) {
                atomicAdd(s_count + at, 1u);   // integers: the order does not matter
                any = true;
            }
        }
    }
    if (BIAS) cp_async_wait_all();
    if (HIST) any = __syncthreads_or(any);
    else if (BIAS) __syncthreads();

    const uint32_t* mask = MASK ? a.allowed + r * a.ld_allowed : nullptr;
#pragma unroll
    for (int i = 0; i < VPT; i++) {
        const long long t = first(i);
        const int at = (i * kThreads + tid) * N;
        if (whole(t)) {
            float b[N];
            uint32_t n[N], bits = ~0u;
            if (BIAS) {
#pragma unroll
                for (int j = 0; j < N; j += 4) {
                    const float4 f = *reinterpret_cast<const float4*>(s_bias + at + j);
                    b[j] = f.x; b[j + 1] = f.y; b[j + 2] = f.z; b[j + 3] = f.w;
                }
            }
            if (HIST && any) {
#pragma unroll
                for (int j = 0; j < N; j += 4) {
                    const uint4 u = *reinterpret_cast<const uint4*>(s_count + at + j);
                    n[j] = u.x; n[j + 1] = u.y; n[j + 2] = u.z; n[j + 3] = u.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < N; j++) n[j] = 0;
            }
            if (MASK) {   // N bits from token t on: at most two words
                const uint32_t lo = __ldg(mask + (t >> 5));
                const uint32_t hi = __ldg(mask + ((t + N - 1) >> 5));
                bits = __funnelshift_r(lo, hi, (uint32_t)(t & 31));
            }
            uint4 o;
#pragma unroll
            for (int j = 0; j < N; j += 2)
                E::set2(o, j,
                        adjust(E::get(v[i], j), n[j], rep, freq, pres, BIAS ? b[j] : 0.0f, bits >> j & 1),
                        adjust(E::get(v[i], j + 1), n[j + 1], rep, freq, pres, BIAS ? b[j + 1] : 0.0f, bits >> (j + 1) & 1));
            if (out_vec) *reinterpret_cast<uint4*>(orow + t * E::SIZE) = o;
            else {
#pragma unroll
                for (int j = 0; j < N; j++) E::store(orow, t + j, E::get(o, j));
            }
        } else {   // a row's first or last few logits
#pragma unroll 1
            for (int j = 0; j < N; j++) {
                const long long x = t + j;
                if (x < 0 || x >= a.V) continue;
                const bool ok = !MASK || (__ldg(mask + (x >> 5)) >> (x & 31) & 1);
                E::store(orow, x, adjust(E::load(zrow, x), HIST ? s_count[at + j] : 0, rep, freq, pres,
                                         BIAS ? s_bias[at + j] : 0.0f, ok));
            }
        }
    }
}

template <int DT, int VPT>
void launch_logits(LogitArgs& a, cudaStream_t st) {
    constexpr int CHUNK = kThreads * VPT * Elem<DT>::N;
    // a row may start up to N - 1 values past a boundary
    a.chunks = (int)(((long long)a.V + Elem<DT>::N - 1 + CHUNK - 1) / CHUNK);
    const long long grid = (long long)a.chunks * a.R;
    if (grid > 0x7fffffffLL) throw std::runtime_error("R * V is too large for one launch");
    const bool h = a.hist, b = a.bias, m = a.allowed;
    auto go = [&](auto kernel) {
        ++g_launch_count;
        const cudaError_t e = launch_k(kernel, dim3((unsigned)grid), dim3(kThreads), 0, st, a);
        if (e != cudaSuccess) throw std::runtime_error(std::string("launch failed: ") + cudaGetErrorString(e));
    };
    if (h && b && m) go(logits_adjust_kernel<DT, VPT, true, true, true>);
    else if (h && b) go(logits_adjust_kernel<DT, VPT, true, true, false>);
    else if (h && m) go(logits_adjust_kernel<DT, VPT, true, false, true>);
    else if (h) go(logits_adjust_kernel<DT, VPT, true, false, false>);
    else if (b && m) go(logits_adjust_kernel<DT, VPT, false, true, true>);
    else if (b) go(logits_adjust_kernel<DT, VPT, false, true, false>);
    else if (m) go(logits_adjust_kernel<DT, VPT, false, false, true>);
    else go(logits_adjust_kernel<DT, VPT, false, false, false>);
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
        if (dtype == MGC_F32) launch_logits<0, 4>(a, st);
        else if (dtype == MGC_F16) launch_logits<1, 2>(a, st);
        else launch_logits<2, 2>(a, st);
    });
}
