// ops_common.cu -- host helpers of the operator files and the stall counter.
#include <mutex>

#include "ops_common.h"

namespace nesle {
namespace ops {

__device__ unsigned int g_stalls;

static std::mutex g_mu;
constexpr int kMaxDevices = 64;

// The device address of the stall counter (looked up once a device).
int stall_counter(int device, unsigned int** out) {
    static unsigned int* addr[kMaxDevices] = {};
    if (device < 0 || device >= kMaxDevices) return invalid("device ordinal out of range");
    std::lock_guard<std::mutex> lock(g_mu);
    if (!addr[device]) {
        void* p = nullptr;
        if (int rc = cuda_status(cudaGetSymbolAddress(&p, g_stalls), "stall counter")) return rc;
        addr[device] = static_cast<unsigned int*>(p);
    }
    *out = addr[device];
    return NESLE_OK;
}

int sm_count(int device) {
    static int count[kMaxDevices] = {};
    if (device < 0 || device >= kMaxDevices) return 1;
    if (!count[device]) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n < 1) return 1;
        count[device] = n;
    }
    return count[device];
}

int encode_map(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const uint64_t* dims,
               const uint64_t* strides, const uint32_t* box, CUtensorMapSwizzle swizzle) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static Encode encode = nullptr;
    if (!encode) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult found{};
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found);
        if (e != cudaSuccess || found != cudaDriverEntryPointSuccess || !fn)
            return set_error(NESLE_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
        encode = reinterpret_cast<Encode>(fn);
    }
    cuuint64_t d[5], s[4];
    cuuint32_t b[5], e[5];
    for (int i = 0; i < rank; ++i) {
        d[i] = dims[i];
        b[i] = box[i];
        e[i] = 1;
        if (i) s[i - 1] = strides[i - 1];
    }
    const CUresult r = encode(map, type, static_cast<cuuint32_t>(rank), const_cast<void*>(base), d, s, b, e,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(NESLE_ERR_CUDA, ("cuTensorMapEncodeTiled: error " + std::to_string((int)r)).c_str());
    return NESLE_OK;
}

}  // namespace ops
}  // namespace nesle

using namespace nesle;

extern "C" int nesle_ops_stalls(int device, uint32_t* count) {
    return ops::guarded([&]() -> int {
        if (!count) return ops::invalid("ops_stalls: null argument");
        ops::OnDevice on(device);
        if (!on.ok) return ops::invalid("ops_stalls: device ordinal out of range");
        unsigned int* p = nullptr;
        if (int rc = ops::stall_counter(device, &p)) return rc;
        return ops::cuda_status(cudaMemcpy(count, p, sizeof(uint32_t), cudaMemcpyDeviceToHost), "ops_stalls");
    });
}
