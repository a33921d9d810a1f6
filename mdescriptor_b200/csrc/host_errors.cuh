// Host-side errors shared by the translation units that hold C entry points:
// the thread's last message, CUDA status mapping and the engine's allocator.
#pragma once

#include "../../include/mdsoap.h"

#include <cuda_runtime.h>

#include <cstdlib>
#include <exception>
#include <string>

namespace mdsoap {

inline thread_local std::string g_error;

inline int fail(int status, const std::string& message) {
    g_error = message;
    return status;
}

struct Failure {
    int status;
    std::string message;
};

[[noreturn]] inline void raise(int status, const std::string& message) { throw Failure{status, message}; }

inline void check(cudaError_t err, const char* what) {
    if (err == cudaSuccess) return;
    const std::string text = std::string(what) + ": " + cudaGetErrorString(err);
    if (err == cudaErrorMemoryAllocation) raise(MDSOAP_OUT_OF_MEMORY, text);
    if (err == cudaErrorNoDevice || err == cudaErrorInsufficientDriver || err == cudaErrorInvalidDevice ||
        err == cudaErrorDevicesUnavailable || err == cudaErrorInitializationError)
        raise(MDSOAP_DEVICE_UNAVAILABLE, text);
    raise(MDSOAP_INTERNAL, text);
}

// Injected allocation failure, for the out-of-memory tests: with
// MDSOAP_TEST_FAIL_ALLOC=<bytes> set, every engine device allocation of at
// least that many bytes returns cudaErrorMemoryAllocation without calling
// cudaMalloc, so the OUT_OF_MEMORY path (status, plugin exception, adapter
// error code) is exercised on the host, with no real exhaustion of a GPU.
inline cudaError_t engine_malloc(void** ptr, size_t bytes) {
    if (const char* env = std::getenv("MDSOAP_TEST_FAIL_ALLOC")) {
        const long long limit = std::atoll(env);
        if (limit > 0 && bytes >= (size_t)limit) {
            *ptr = nullptr;
            return cudaErrorMemoryAllocation;
        }
    }
    return cudaMalloc(ptr, bytes);
}

// The body of a C entry point: no exception leaves it.
template <class F>
int entry(F&& body) {
    try {
        body();
        return MDSOAP_OK;
    } catch (const Failure& f) {
        return fail(f.status, f.message);
    } catch (const std::exception& e) {
        return fail(MDSOAP_INTERNAL, e.what());
    } catch (...) {
        return fail(MDSOAP_INTERNAL, "unknown error");
    }
}

}  // namespace mdsoap
