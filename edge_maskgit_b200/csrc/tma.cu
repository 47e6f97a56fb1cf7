// tma.cu -- host-side helpers of the 16-bit operators: tensor maps, device properties, errors.
#include <cudaTypedefs.h>

#include <atomic>
#include <mutex>

#include "kernels.h"
#include "tma.cuh"

namespace mgc {

static PFN_cuTensorMapEncodeTiled_v12000 encode_tiled() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = (PFN_cuTensorMapEncodeTiled_v12000)p;
    });
    if (!fn) throw std::runtime_error("cuTensorMapEncodeTiled is not available");
    return fn;
}

CUtensorMap make_map16(const void* base, bool bf16, int rank, const uint64_t* dims, const uint64_t* strides,
                       const uint32_t* box) {
    CUtensorMap m;
    cuuint64_t d[5], st[4];
    cuuint32_t bx[5], es[5];
    for (int i = 0; i < rank; i++) {
        d[i] = dims[i];
        bx[i] = box[i];
        es[i] = 1;
        if (i > 0) {
            st[i - 1] = strides[i - 1] * 2;
            if (strides[i - 1] == 0) d[i] = 1;
            if (d[i] == 1) st[i - 1] = (dims[0] * 2 + 15) / 16 * 16;   // never stepped over: any valid stride
        }
    }
    const CUresult r = encode_tiled()(&m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                                      (cuuint32_t)rank, const_cast<void*>(base), d, st, bx, es,
                                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw std::runtime_error("cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
    return m;
}

int current_sms() {
    constexpr int kMax = 64;
    static std::atomic<int> known[kMax];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMax) throw std::runtime_error("no usable current device");
    int n = known[dev].load();
    if (n == 0) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
            throw std::runtime_error("cannot read the device's SM count");
        known[dev].store(n);
    }
    return n;
}

int* dev_error_address() {
    constexpr int kMax = 64;
    static std::atomic<int*> known[kMax];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMax) throw std::runtime_error("no usable current device");
    int* p = known[dev].load();
    if (!p) {
        void* v = nullptr;
        const cudaError_t e = cudaGetSymbolAddress(&v, g_dev_error);
        if (e != cudaSuccess) throw std::runtime_error(std::string("cudaGetSymbolAddress: ") + cudaGetErrorString(e));
        known[dev].store(p = (int*)v);
    }
    return p;
}

void set_error_for(const char* what, const char* msg) { set_last_error((std::string(what) + ": " + msg).c_str()); }

}  // namespace mgc
