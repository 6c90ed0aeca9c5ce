// Host-side checks shared by the entry points of include/tmt_mx.h and of the LayerNorm checkpoints.
#pragma once
#include <cuda_runtime.h>

#include <atomic>
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

// What the calls ask of the current device again and again, asked for once per device: `ask` fills in a value, which is not 0.
template <class T, class Ask>
T per_device(std::atomic<T> (&known)[64], Ask ask) {
    int dev = 0;
    cuda_ok(cudaGetDevice(&dev), "cudaGetDevice");
    if (dev < 64) {
        const T v = known[dev].load(std::memory_order_acquire);
        if (v) return v;
    }
    const T v = ask(dev);
    if (dev < 64) known[dev].store(v, std::memory_order_release);
    return v;
}

inline int sm_count() {
    static std::atomic<int> known[64];
    return per_device(known, [](int dev) {
        int sms = 0;
        cuda_ok(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev), "cudaDeviceGetAttribute");
        return sms;
    });
}

}  // namespace tmt

#define MX_GUARD(...)                                                    \
    try { __VA_ARGS__; return 0; }                                       \
    catch (const std::exception& e) { tmt::set_error("%s", e.what()); return -1; } \
    catch (...) { tmt::set_error("unknown error"); return -1; }
