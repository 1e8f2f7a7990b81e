// ops_common.h -- what the operator files (ops_*.cu) share: error reporting,
// the device guard, element types and tensor-map encoding.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <exception>
#include <string>

#include "../../include/nesle_b200.h"
#include "../../include/nesle_ops.h"

namespace nesle {

// Sets the thread's last error (nesle_last_error) and returns `code`; in capi.cu.
int set_error(int code, const char* message) noexcept;

namespace ops {

inline int invalid(const char* m) { return set_error(NESLE_ERR_INVALID, m); }

inline int cuda_status(cudaError_t e, const char* where) {
    if (e == cudaSuccess) return NESLE_OK;
    return set_error(NESLE_ERR_CUDA, (std::string(where) + ": " + cudaGetErrorString(e)).c_str());
}

// Whether every pointer lies on `bytes`, as loads of elements of that size want it.
template <class... P>
bool all_on(uintptr_t bytes, P... pointers) {
    return (... && (reinterpret_cast<uintptr_t>(pointers) % bytes == 0));
}
// Memory of `rows` rows of `bytes`, `pitch` apart.
struct Memory {
    uintptr_t at;
    uint64_t rows;
    int64_t pitch;
    uint64_t bytes;
    Memory(const void* p, uint64_t rows_, int64_t pitch_, uint64_t bytes_) : at(reinterpret_cast<uintptr_t>(p)), rows(rows_), pitch(pitch_), bytes(bytes_) {}
    uintptr_t end() const { return at && rows && bytes ? at + (rows - 1) * pitch + bytes : at; }
};
// Whether two may share a byte.
inline bool may_overlap(const Memory& a, const Memory& b) {
    if (a.at >= b.end() || b.at >= a.end()) return false;
    if (a.pitch != b.pitch || a.pitch <= 0) return true;
    const uint64_t pitch = a.pitch, d = b.at >= a.at ? (b.at - a.at) % pitch : (pitch - (a.at - b.at) % pitch) % pitch;
    return d < a.bytes || d + b.bytes > pitch;  // b's rows begin d after a's, modulo the pitch
}
inline uintptr_t element_size(int dtype) { return dtype == NESLE_F32 ? 4 : 2; }

// Runs a C entry's body: no C++ exception leaves the library.
template <class F>
int guarded(F&& body) noexcept {
    try {
        return body();
    } catch (const std::exception& e) {
        return set_error(NESLE_ERR_RUNTIME, e.what());
    } catch (...) {
        return set_error(NESLE_ERR_RUNTIME, "unknown C++ exception");
    }
}

// Makes `device` current for the scope.  cudaSetDevice is called even where it already is: a thread that has made no CUDA
// call yet (the autograd engine's, for one) has no context bound, and encoding a tensor map needs one.
struct OnDevice {
    int prev = -1;
    bool ok = true;
    explicit OnDevice(int device) { ok = cudaGetDevice(&prev) == cudaSuccess && cudaSetDevice(device) == cudaSuccess; }
    ~OnDevice() {
        int cur = -1;
        if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
    }
};

int sm_count(int device);

// The device address of the stall counter, which kernels add to when a wait gives up.
int stall_counter(int device, unsigned int** out);

// A tiled tensor map over `rank` dimensions, innermost first; `strides` are the
// byte strides of dimensions 1..rank-1.  Zero fill.
int encode_map(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const uint64_t* dims,
               const uint64_t* strides, const uint32_t* box, CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B);

// Allows a kernel its dynamic shared memory on the current device, `device`: once for each.
template <auto* kKernel>
int allow_smem(int bytes, int device, const char* where) {
    static std::atomic<uint64_t> done{0};
    const uint64_t bit = device >= 0 && device < 64 ? uint64_t(1) << device : 0;
    if (done.load(std::memory_order_relaxed) & bit) return NESLE_OK;
    const int rc = cuda_status(
        cudaFuncSetAttribute(reinterpret_cast<const void*>(kKernel), cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), where);
    if (!rc) done.fetch_or(bit, std::memory_order_relaxed);
    return rc;
}

template <class T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }

}  // namespace ops
}  // namespace nesle
