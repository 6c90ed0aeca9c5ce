// Host-side checks shared by the entry points of include/tmt_mx.h and of the LayerNorm checkpoints.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>
#include <stdexcept>
#include <string>

namespace tmt {
void set_error(const char* fmt, ...);

inline void cuda_ok(cudaError_t e, const char* what) {
    if (e != cudaSuccess) throw std::runtime_error(std::string(what) + " failed: " + cudaGetErrorString(e));
}

// Every tensor is 16-byte aligned and lies in the current device's memory or in managed memory. A pointer of another device or
// of the host would fault there, so it is refused here.
inline void check_tensors(std::initializer_list<const void*> ptrs, uintptr_t align = 16) {
    int dev = 0;
    cuda_ok(cudaGetDevice(&dev), "cudaGetDevice");
    for (const void* p : ptrs) {
        if (!p) throw std::runtime_error("null argument");
        if (reinterpret_cast<uintptr_t>(p) & (align - 1)) throw std::runtime_error("a tensor must start on a " + std::to_string(align) + "-byte boundary");
        cudaPointerAttributes a{};
        cuda_ok(cudaPointerGetAttributes(&a, p), "cudaPointerGetAttributes");
        if (a.type == cudaMemoryTypeUnregistered || a.type == cudaMemoryTypeHost) throw std::runtime_error("a tensor lies in host memory");
        if (a.type == cudaMemoryTypeDevice && a.device != dev)
            throw std::runtime_error("a tensor lies on device " + std::to_string(a.device) + ", the current device is " + std::to_string(dev));
    }
}

inline int sm_count() {
    int dev = 0, sms = 0;
    cuda_ok(cudaGetDevice(&dev), "cudaGetDevice");
    cuda_ok(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev), "cudaDeviceGetAttribute");
    return sms;
}

}  // namespace tmt

#define MX_GUARD(...)                                                    \
    try { __VA_ARGS__; return 0; }                                       \
    catch (const std::exception& e) { tmt::set_error("%s", e.what()); return -1; } \
    catch (...) { tmt::set_error("unknown error"); return -1; }
