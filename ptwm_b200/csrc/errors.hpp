// Error string, CUDA error macro and device guard of every translation unit of
// libptwm_b200.so.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>
#include <string>

#include "../../include/ptwm_b200.h"

namespace ptwm {

// Last error of the calling thread (returned by ptwm_b200_last_error).
std::string& last_error_ref();
inline int64_t fail(int64_t rc, const std::string& m) { last_error_ref() = m; return rc; }

#define CUDA_TRY(expr)                                                                                        \
    do {                                                                                                      \
        cudaError_t e_ = (expr);                                                                              \
        if (e_ != cudaSuccess) {                                                                              \
            cudaGetLastError(); /* reported here: the thread's next call does not find it again */            \
            return ::ptwm::fail(PTWM_RC_CUDA, std::string(#expr) + ": " + cudaGetErrorString(e_));            \
        }                                                                                                     \
    } while (0)

// Makes `dev` current for the scope and restores the previous device.
struct DeviceGuard {
    int prev = -1;
    cudaError_t err;
    explicit DeviceGuard(int dev) {
        err = cudaGetDevice(&prev);
        if (err == cudaSuccess && prev != dev) err = cudaSetDevice(dev);
        if (err != cudaSuccess) cudaGetLastError();  // `err` has it: the thread's next call does not find it again
    }
    ~DeviceGuard() { if (prev >= 0) cudaSetDevice(prev); }
};

}  // namespace ptwm
