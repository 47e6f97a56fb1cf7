// attn_shaped.cu -- mgc_attention: argument checks, the choice of kernel and split, workspace.
#include <algorithm>
#include <cmath>

#include "attn_tile.cuh"

namespace mgc {
namespace {

struct Plan {
    AttnCall c{};
    bool tile = false;          // the 128-row tcgen05 kernel
    at::TileCall t{};
    uint64_t doc_bytes = 0, opart_bytes = 0, bytes = 0;   // workspace: document ranges, partials, (max, sum)
};

// Lowest and highest document number of every 128-key tile (TileCall::doc_range).
__global__ void __launch_bounds__(128) doc_range_kernel(const int32_t* __restrict__ doc, int Sk, int nkt, int2* out) {
    griddep_wait();
    griddep_launch();
    __shared__ int2 part[4];
    const int kt = blockIdx.x % nkt, b = blockIdx.x / nkt, j = kt * 128 + threadIdx.x;
    const int d = j < Sk ? __ldg(doc + (long long)b * Sk + j) : INT_MAX;
    int mn = d < 0 ? INT_MAX : d, mx = j < Sk ? d : -1;
    for (int k = 16; k; k >>= 1) {
        mn = min(mn, __shfl_xor_sync(0xffffffffu, mn, k));
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, k));
    }
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = make_int2(mn, mx);
    const bool padding = __syncthreads_or(d < 0);
    if (threadIdx.x == 0) {
        for (int w = 1; w < 4; w++) { mn = min(mn, part[w].x); mx = max(mx, part[w].y); }
        out[blockIdx.x] = make_int2(padding ? mn | INT_MIN : mn, mx);
    }
}

void check(const mgc_attention_args& a) {
    auto need = [](bool ok, const char* m) { if (!ok) throw std::invalid_argument(m); };
    need(a.dtype == MGC_F16 || a.dtype == MGC_BF16, "dtype must be F16 or BF16");
    need(a.B >= 0 && a.Sq >= 0 && a.Sk >= 0, "negative size");
    need(a.Hkv > 0 && a.Hq > 0 && a.Hq % a.Hkv == 0, "Hq must be a positive multiple of Hkv");
    need(a.D >= 8 && a.D <= 128 && a.D % 8 == 0, "D must be a multiple of 8 from 8 to 128");
    need(a.causal == 0 || a.causal == 1, "causal must be 0 or 1");
    // Capped scores carry an absolute error of up to 2^-20 cap, at 1024 what one rounding step of an f16
    // result is; and the constants of the cap, (scale / cap)^5 cap at most, have to be finite.
    need(std::fabs(a.scale) <= 0x1p100f, "scale must be at most 2^100");
    need(a.cap == 0.0f || (a.cap >= 0x1p-10f && a.cap <= 0x1p10f), "cap must be 0 or from 2^-10 to 2^10");
    need(a.cap == 0.0f || std::fabs(a.scale) <= 0x1p20f * a.cap, "scale must be at most 2^20 cap");
    need(a.dist_range >= 0 && a.dist_range <= (1 << 30), "dist_range must be from 0 to 2^30");
    need((a.doc_q != nullptr) == (a.doc_k != nullptr), "doc_q and doc_k are given together");
    need(a.reserved == 0, "reserved must be 0");
    need((long long)a.Sq * (a.Hq / a.Hkv) < (1LL << 28) && a.Sk < (1 << 28), "Sq or Sk is too large");
}

void check_pointers(const mgc_attention_args& a) {
    auto need = [](bool ok, const char* m) { if (!ok) throw std::invalid_argument(m); };
    need(a.q && a.out && (a.Sk == 0 || (a.k && a.v)), "q, k, v and out must not be NULL");
    need((((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.out) & 15) == 0, "q, k, v and out must be 16-byte aligned");
    need((((uintptr_t)a.slopes | (uintptr_t)a.dist_bias | (uintptr_t)a.prefix | (uintptr_t)a.k_len | (uintptr_t)a.q_pos |
           (uintptr_t)a.doc_q | (uintptr_t)a.doc_k) & 3) == 0, "tables must be 4-byte aligned");
    const int sizes_q[3] = {a.B, a.Sq, a.Hq}, sizes_k[3] = {a.B, a.Sk, a.Hkv};
    for (int i = 0; i < 3; i++) {
        auto ok = [&](int64_t s, int n) { return n <= 1 || (s >= 0 && s % 8 == 0 && s < (1LL << 38)); };
        need(ok(a.q_stride[i], sizes_q[i]) && ok(a.k_stride[i], sizes_k[i]) && ok(a.v_stride[i], sizes_k[i]) &&
                 ok(a.out_stride[i], sizes_q[i]),
             "strides must be multiples of 8, not negative");
        need(sizes_q[i] <= 1 || a.out_stride[i] >= a.D, "out's strides must be at least D");
        need(i != 1 || a.Sk <= 1 || (a.k_stride[1] < (1LL << 31) && a.v_stride[1] < (1LL << 31)),
             "k's and v's position strides must be below 2^31");
    }
}

Plan plan(const mgc_attention_args& args) {
    check(args);
    Plan p;
    p.c.a = args;
    mgc_attention_args& a = p.c.a;
    // the stride of a dimension of size 1 is never used: make it a harmless one
    const int sizes_q[3] = {a.B, a.Sq, a.Hq}, sizes_k[3] = {a.B, a.Sk, a.Hkv};
    for (int i = 0; i < 3; i++) {
        if (sizes_q[i] <= 1) a.q_stride[i] = a.out_stride[i] = 0;
        if (sizes_k[i] <= 1) a.k_stride[i] = a.v_stride[i] = 0;
    }
    p.c.g = a.Hq / a.Hkv;
    p.c.nsplit = 1;
    p.c.chunk = std::max(16, (a.Sk + 15) / 16 * 16);
    if (a.B == 0 || a.Sq == 0) return p;
    const int rows = a.Sq * p.c.g, sms = current_sms();
    // A position stride of 0 (one key repeated) has no tensor map; the other kernel takes any.
    const bool maps = a.Sk > 0 && (a.Sq == 1 || a.q_stride[1] > 0) && (a.Sk == 1 || (a.k_stride[1] > 0 && a.v_stride[1] > 0));
    // The other kernel also serves small problems (its set-up is a third of the tiles'): blocks of 16 rows times
    // keys, about where the two take equal time in a graph.  Over 334 shapes (32 to 1000 queries, 40 to 4000
    // keys, 1 to 16 rows, 4 to 32 heads of 48 to 128) the chosen ones take 2 % more in all than the better
    // of the two each time: 1 x 257 x 16 heads of 48 (70 thousand) 8.0 against 10.3 us, 4 x 257 (280 thousand) 19.0 / 19.6, 1 x
    // 513 x 16 of 64 (271 thousand) 20.0 / 13.7; 1 x 128 x 32 heads of 128 over 8 (33 thousand) 7.7 / 7.9, 1 x 300 (180
    // thousand) 28.2 / 12.2.  It is furthest off for many short rows (16 x 128 x 8 of 64, 131 thousand: 14.6 / 7.4, the
    // first is taken) and for 32 queries of many rows (16 x 32 x 2000 keys x 16 of 48: 40.6 / 60.2, the second is).
    const long long block_keys = (long long)a.B * a.Hkv * ((rows + 15) / 16) * a.Sk;
    p.tile = maps && a.Sq >= 32 && block_keys > (a.D <= 64 ? 160000 : 32000);
    if (p.tile) {
        const long long heads = (long long)a.B * a.Hq;
        const int nkt = (a.Sk + at::KT - 1) / at::KT, nqt = (a.Sq + at::QT - 1) / at::QT;
        at::TileCall& t = p.t;
        t.tiles_per_cta = heads * ((nqt + 1) / 2) >= sms ? 2 : 1;
        t.qblocks = (nqt + t.tiles_per_cta - 1) / t.tiles_per_cta;
        t.q_outer = a.causal;
        const long long ctas = heads * t.qblocks;
        const int split = (int)std::max<long long>(1, std::min<long long>(sms / ctas, nkt / 4));
        const int per = (nkt + split - 1) / split;
        p.c.chunk = per * at::KT;
        p.c.nsplit = (nkt + per - 1) / per;
        for (int i = 0; i < 3; i += 2) {
            t.qmul[i] = a.q_stride[i] != 0;
            t.kmul[i] = a.k_stride[i] != 0;
            t.vmul[i] = a.v_stride[i] != 0;
        }
        if (a.doc_k) p.doc_bytes = ((uint64_t)a.B * nkt * sizeof(int2) + 15) / 16 * 16;
    } else {
        const long long heads = (long long)a.B * a.Hkv * ((rows + 15) / 16);
        // As many ranges of keys as run at once (two blocks an SM with large heads, three with small ones),
        // of 128 keys at least.  Long ones of several rows are cut to 1024 keys, or to 32 ranges where those
        // are longer, so that rows of unequal length balance, unless there are several rounds of blocks anyway.  Up to
        // 8 ranges are one cluster and join in one launch (4 rows x 4096 keys x 8 heads of 128: 17.5 us,
        // by a second kernel 20; clusters of 16 took 35).
        const long long slots = (long long)sms * (a.D > 64 ? 2 : 3);
        const long long n = std::max<long long>(1, slots / heads);
        auto up64 = [](long long x) { return (x + 63) / 64 * 64; };
        long long chunk = std::max<long long>(128, up64((a.Sk + n - 1) / n));
        if (chunk > 2048 && a.B > 1 && heads < 4 * slots)
            chunk = std::min(chunk, std::max<long long>(1024, up64((a.Sk + 31) / 32)));
        if (a.Sk > chunk) {
            p.c.chunk = (int)chunk;
            p.c.nsplit = (int)((a.Sk + chunk - 1) / chunk);
            p.c.cluster = p.c.nsplit <= 8;
            // Few heads and not too many keys: a cluster of 8 blocks of eight warps, one launch and no workspace,
            // which saves the host 3 to 5 us a call and costs the GPU up to 3 us.  Its GPU time is about
            // 6.2 us + 7.3 ps * keys * (D + 32); it is taken where calls gain at least what graph replays lose.
            // One row, 1 to 8 heads, call (GPU) in us, against two launches:
            //   heads of 128: 1100 keys 9.9 (7.7) / 14.8 (6.9), 2000 10.3 (8.4) / 14.8 (7.0), 4096 12.6 (11.1) /
            //   14.9 (8.3), 6000 16.4 (13.7) / 14.8 (11.2), 8192 18.6 (16.3) / 15.2 (11.6)
            //   heads of 64: 2000 9.9 (6.8) / 14.8 (6.3), 4096 10.3 (8.4) / 14.8 (7.3), 6000 12.8 (10.0) / 14.9 (10.5),
            //   8192 13.5 (11.5) / 14.9 (10.0)
            // (16 heads, two rounds of such clusters: 2000 keys 14.5 (12.4) / 14.8 (7.2))
            if (p.c.nsplit > 8 && (long long)a.Sk * (a.D + 32) <= 655360 && heads * 16 <= sms) {
                p.c.chunk = (int)up64((a.Sk + 7) / 8);
                p.c.nsplit = (a.Sk + p.c.chunk - 1) / p.c.chunk;
                p.c.cluster = p.c.wide = 1;
            }
        }
    }
    p.bytes = p.doc_bytes;
    if (p.c.nsplit > 1 && !p.c.cluster) {
        const uint64_t all = (uint64_t)a.B * a.Sq * a.Hq * p.c.nsplit;
        p.opart_bytes = (all * a.D * 4 + 15) / 16 * 16;
        p.bytes += p.opart_bytes + all * 8;
    }
    return p;
}

CUtensorMap operand_map(const void* p, bool bf16, int D, int S, int H, int B, const int64_t* stride) {
    const uint64_t dims[4] = {(uint64_t)D, (uint64_t)S, (uint64_t)H, (uint64_t)B};
    const uint64_t strides[3] = {(uint64_t)stride[1], (uint64_t)stride[2], (uint64_t)stride[0]};
    const uint32_t box[4] = {64, 128, 1, 1};
    return make_map16(p, bf16, 4, dims, strides, box);
}

void run_tile(Plan& p, cudaStream_t st, bool gives_up = false) {
    const mgc_attention_args& a = p.c.a;
    const bool bf16 = a.dtype == MGC_BF16;
    if (a.doc_k) {
        const int nkt = (a.Sk + at::KT - 1) / at::KT;
        int2* range = reinterpret_cast<int2*>(a.workspace);
        if ((long long)a.B * nkt > 0x7fffffffLL) throw std::runtime_error("too many rows for one launch");
        ++g_launch_count;
        const cudaError_t e = launch_k(doc_range_kernel, dim3((unsigned)(a.B * nkt)), dim3(128), 0, st, a.doc_k, a.Sk, nkt, range);
        if (e != cudaSuccess) throw std::runtime_error(std::string("launch failed: ") + cudaGetErrorString(e));
        p.t.doc_range = range;
    }
    p.t.c = p.c;
    p.t.dev_error = dev_error_address();
    const CUtensorMap mq = operand_map(a.q, bf16, a.D, a.Sq, a.Hq, a.B, a.q_stride);
    const CUtensorMap mk = operand_map(a.k, bf16, a.D, a.Sk, a.Hkv, a.B, a.k_stride);
    const CUtensorMap mv = operand_map(a.v, bf16, a.D, a.Sk, a.Hkv, a.B, a.v_stride);
    if (gives_up) return at::launch_tile_gives_up(mq, mk, mv, p.t, st);
    (bf16 ? (a.D <= 64 ? at::launch_tile_bf16_64 : at::launch_tile_bf16_128)
          : (a.D <= 64 ? at::launch_tile_f16_64 : at::launch_tile_f16_128))(mq, mk, mv, p.t, st);
}

void place_workspace(Plan& p) {
    if (!p.bytes) return;
    const mgc_attention_args& a = p.c.a;
    if (!a.workspace || ((uintptr_t)a.workspace & 15) || a.workspace_bytes < p.bytes)
        throw std::invalid_argument("workspace must be 16-byte aligned and hold mgc_attention_workspace() bytes");
    uint8_t* ws = reinterpret_cast<uint8_t*>(a.workspace);
    p.c.opart = reinterpret_cast<float*>(ws + p.doc_bytes);
    p.c.mlpart = reinterpret_cast<float2*>(ws + p.doc_bytes + p.opart_bytes);
}

}  // namespace
}  // namespace mgc

using namespace mgc;

extern "C" {

int mgc_attention_workspace(const mgc_attention_args* args, uint64_t* bytes) {
    return guarded("mgc_attention_workspace", [&] {
        if (!args || !bytes) throw std::invalid_argument("args and bytes must not be NULL");
        *bytes = plan(*args).bytes;
    });
}

int mgc_attention(const mgc_attention_args* args, void* stream) {
    return guarded("mgc_attention", [&] {
        if (!args) throw std::invalid_argument("args must not be NULL");
        Plan p = plan(*args);
        if (args->B == 0 || args->Sq == 0) return;
        check_pointers(*args);
        place_workspace(p);
        const cudaStream_t st = (cudaStream_t)stream;
        if (p.tile) run_tile(p, st);
        else launch_attn_step(p.c, st);
        if (p.c.nsplit > 1 && !p.c.cluster) launch_attn_combine(p.c, st);
    });
}

int mgc_selftest_attention_gives_up(const mgc_attention_args* args, void* stream) {
    return guarded("mgc_selftest_attention_gives_up", [&] {
        if (!args) throw std::invalid_argument("args must not be NULL");
        Plan p = plan(*args);
        if (!p.tile || args->dtype != MGC_F16 || args->D > 64 || !args->dist_bias || args->cap != 0.0f || args->slopes)
            throw std::invalid_argument("takes calls of the tile kernel in f16, heads of up to 64, a distance table only");
        check_pointers(*args);
        place_workspace(p);
        run_tile(p, (cudaStream_t)stream, true);
        const cudaError_t e = cudaStreamSynchronize((cudaStream_t)stream);
        if (e != cudaSuccess) throw std::runtime_error(cudaGetErrorString(e));
    });
}

}  // extern "C"
