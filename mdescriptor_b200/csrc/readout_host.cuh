// Host-side pieces shared by the readout operators' C entry points.
#pragma once

#include "host_errors.cuh"
#include "readout.cuh"

#include <atomic>

namespace mdsoap {
namespace readout {

inline void need(bool ok, const char* message) {
    if (!ok) raise(MDSOAP_INVALID_ARGUMENT, message);
}

// Makes a device current for the length of a call; the caller's stays what it
// was (a framework's next allocation goes by it).
struct OnDevice {
    int before = 0, now;
    explicit OnDevice(int device) : now(device) {
        check(cudaGetDevice(&before), "cudaGetDevice");
        if (before != now) check(cudaSetDevice(now), "cudaSetDevice");
    }
    ~OnDevice() {
        if (before != now) cudaSetDevice(before);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
};

// Streaming multiprocessors of a device, asked for once.
inline int sm_count(int device) {
    static std::atomic<int> known[64];
    const bool slot = device >= 0 && device < 64;
    if (slot)
        if (const int sms = known[device].load(std::memory_order_relaxed)) return sms;
    int sms = 0;
    check(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device), "device attribute");
    if (slot) known[device].store(sms, std::memory_order_relaxed);
    return sms;
}

// Raises a kernel's limit of dynamic shared memory, once on each device.
template <class K>
void allow_shared(K kernel, int bytes, std::atomic<uint64_t>& done, int device, const char* what) {
    const uint64_t bit = uint64_t(1) << (device & 63);
    if (device < 64 && (done.load(std::memory_order_acquire) & bit)) return;
    check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), what);
    done.fetch_or(bit, std::memory_order_release);
}

template <class F>
void by_type(int32_t dtype, F&& body) {
    switch (dtype) {
        case MDSOAP_FLOAT32: body(float{}); break;
        case MDSOAP_BFLOAT16: body(__nv_bfloat16{}); break;
        case MDSOAP_FLOAT16: body(__half{}); break;
        default: raise(MDSOAP_INVALID_ARGUMENT, "readout: element type must be float32, bfloat16 or float16");
    }
}

}  // namespace readout
}  // namespace mdsoap
