// The context of the C ABI and how its entry points report errors, for the translation units that implement them.
#ifndef ASP_CTX_H
#define ASP_CTX_H

#include <cuda_runtime.h>
#include <stdint.h>

#include <string>
#include <vector>

#include "../../include/asp_b200.h"
#include "memory.h"

namespace asp
{
std::string &last_error(); // of this thread: asp_last_error

inline asp_status cuda_fail(cudaError_t e, const char *what)
{
    last_error() = std::string(what) + ": " + cudaGetErrorString(e);
    return ASP_ERR_CUDA;
}
inline asp_status fail(asp_status s, const std::string &msg)
{
    last_error() = msg;
    return s;
}
#define ASP_CUDA(call)                                             \
    do                                                             \
    {                                                              \
        cudaError_t e__ = (call);                                  \
        if (e__ != cudaSuccess) return asp::cuda_fail(e__, #call); \
    } while (0)

// Makes `device` current for the lifetime of the object and restores the caller's device afterwards:
// every entry point that launches or allocates runs under one, so a process that holds contexts on
// several GPUs never launches into a stream of a device that is not current.
struct DeviceGuard
{
    int prev = -1;
    cudaError_t err = cudaSuccess;
    explicit DeviceGuard(int device)
    {
        err = cudaGetDevice(&prev);
        if (err == cudaSuccess && prev != device) err = cudaSetDevice(device);
        else if (err == cudaSuccess) prev = -1; // nothing to restore
    }
    ~DeviceGuard()
    {
        if (prev >= 0) cudaSetDevice(prev);
    }
};
#define ASP_ON_DEVICE(ctx)                   \
    asp::DeviceGuard guard__((ctx)->device); \
    if (guard__.err != cudaSuccess) return asp::cuda_fail(guard__.err, "cudaSetDevice")
} // namespace asp

struct asp_ctx
{
    int device = 0;
    uint64_t serial = 0; // of this context, never given to another one
    cudaStream_t stream = nullptr;
    cudaEvent_t ev0 = nullptr, ev1 = nullptr;
    // side streams: the sub-matrix kernels of one SpMV run concurrently (the reference gives every
    // sub-matrix kernel its own stream, code_builder.cc:1515-1518)
    static const int kAux = 3;
    cudaStream_t aux[kAux] = {nullptr, nullptr, nullptr};
    cudaEvent_t ev_fork = nullptr, ev_join[kAux] = {nullptr, nullptr, nullptr};
    int sm_count = 0;
    int max_smem_optin = 0;
    // scratch x / y used by asp_time and asp_spmv_host; grown on demand
    void *x = nullptr, *y = nullptr;
    size_t x_bytes = 0, y_bytes = 0;
    // copy streams and events of the pipelined host SpMV, created on first use
    cudaStream_t h2d = nullptr, d2h = nullptr;
    std::vector<cudaEvent_t> pipe_events;
    asp::Stager stager;
    unsigned *fault = nullptr; // page-locked: set by a kernel that gives up a bounded wait, read by asp_synchronize
};

#endif
