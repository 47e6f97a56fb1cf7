// attn_shaped.cu -- mgc_attention: argument checks, the choice of kernel and split, workspace.
#include <algorithm>
#include <cmath>

#include "attn_shaped.cuh"

namespace mgc {
namespace {

struct Plan {
    AttnCall c{};
    bool tile = false;          // the 128-row tcgen05 kernel
    uint64_t opart_bytes = 0, bytes = 0;
};

void check(const mgc_attention_args& a) {
    auto need = [](bool ok, const char* m) { if (!ok) throw std::invalid_argument(m); };
    need(a.dtype == MGC_F16 || a.dtype == MGC_BF16, "dtype must be F16 or BF16");
    need(a.B >= 0 && a.Sq >= 0 && a.Sk >= 0, "negative size");
    need(a.Hkv > 0 && a.Hq > 0 && a.Hq % a.Hkv == 0, "Hq must be a positive multiple of Hkv");
    need(a.D >= 8 && a.D <= 128 && a.D % 8 == 0, "D must be a multiple of 8 from 8 to 128");
    need(a.causal == 0 || a.causal == 1, "causal must be 0 or 1");
    need(std::isfinite(a.scale), "scale must be finite");
    need(a.cap >= 0.0f && std::isfinite(a.cap), "cap must be finite and not negative");
    need(a.dist_range >= 0 && a.dist_range <= (1 << 30), "dist_range must be from 0 to 2^30");
    need((a.doc_q != nullptr) == (a.doc_k != nullptr), "doc_q and doc_k are given together");
    need(a.reserved == 0, "reserved must be 0");
    need((long long)a.Sq * (a.Hq / a.Hkv) < (1LL << 30) && a.Sk < (1 << 30), "Sq or Sk is too large");
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
    const long long heads = (long long)a.B * a.Hkv * ((rows + 15) / 16);
    const long long want = std::max<long long>(1, (4LL * sms + heads - 1) / heads);
    long long chunk = ((a.Sk + want - 1) / want + 63) / 64 * 64;
    chunk = std::max<long long>(128, std::min<long long>(1024, chunk));
    if (heads >= 4LL * sms && a.Sk <= 4096) chunk = (a.Sk + 63) / 64 * 64;
    if (a.Sk > chunk) {
        p.c.chunk = (int)chunk;
        p.c.nsplit = (int)((a.Sk + chunk - 1) / chunk);
    }
    if (p.c.nsplit > 1) {
        const uint64_t all = (uint64_t)a.B * a.Sq * a.Hq * p.c.nsplit;
        p.opart_bytes = (all * a.D * 4 + 15) / 16 * 16;
        p.bytes = p.opart_bytes + all * 8;
    }
    return p;
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
        if (p.bytes) {
            if (!args->workspace || ((uintptr_t)args->workspace & 15) || args->workspace_bytes < p.bytes)
                throw std::invalid_argument("workspace must be 16-byte aligned and hold mgc_attention_workspace() bytes");
            p.c.opart = reinterpret_cast<float*>(args->workspace);
            p.c.mlpart = reinterpret_cast<float2*>(reinterpret_cast<uint8_t*>(args->workspace) + p.opart_bytes);
        }
        const cudaStream_t st = (cudaStream_t)stream;
        launch_attn_step(p.c, st);
        if (p.c.nsplit > 1) launch_attn_combine(p.c, st);
    });
}

}  // extern "C"
