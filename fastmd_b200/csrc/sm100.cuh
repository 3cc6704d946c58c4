// What the tensor-core kernels share: bounded mbarrier waits, tcgen05 fences and commits, and the driver entry
// points behind the tensor maps.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "common.cuh"

namespace fmd {

// Every mbarrier wait gives up after this long (about a second).
constexpr unsigned long long kWaitNs = 1000000000ull;

__device__ __forceinline__ uint32_t su32(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(bar)), "r"(count) : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.shared::cta.b64 st, [%0];\n\t}" ::"r"(su32(bar))
                 : "memory");
}

__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(
                     su32(bar)),
                 "r"(bytes)
                 : "memory");
}

__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}

__device__ __forceinline__ unsigned long long global_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

// Waits for the phase of `parity` to complete. Gives up after kWaitNs, or
// as soon as another role of the CTA has given up (abort != 0, unless
// `ignore_abort`); returns false then and sets the CTA's abort word.
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, volatile int32_t* abort,
                                          bool ignore_abort = false) {
    const uint32_t a = su32(bar);
    if (mbar_try_wait(a, parity)) return true;
    const unsigned long long t0 = global_ns();
    while (true) {
        if (mbar_try_wait(a, parity)) return true;
        if (!ignore_abort && *abort) return false;
        if (global_ns() - t0 > kWaitNs) {
            *abort = 1;
            return false;
        }
    }
}

__device__ __forceinline__ void tc_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}

__device__ __forceinline__ void tc_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(su32(bar))
                 : "memory");
}

// ------------------------------------------------------------------- host

using EncodeTiled = PFN_cuTensorMapEncodeTiled_v12000;
using CtxGetCurrent = PFN_cuCtxGetCurrent_v4000;

struct DriverCalls {
    EncodeTiled encode = nullptr;
    CtxGetCurrent ctx_get_current = nullptr;
};

// Driver entry points through the runtime (no link against libcuda).
inline const DriverCalls& driver_calls() {
    static DriverCalls calls;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            calls.encode = reinterpret_cast<EncodeTiled>(p);
        if (cudaGetDriverEntryPoint("cuCtxGetCurrent", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            calls.ctx_get_current = reinterpret_cast<CtxGetCurrent>(p);
    });
    return calls;
}

// The tensor-map encoder is a driver call: a host thread on which the runtime has not yet made the
// primary context current (a fresh autograd worker, say) gets it bound first.
inline fmd_status bind_context(const DriverCalls& drv) {
    CUcontext current = nullptr;
    if (drv.ctx_get_current(&current) != CUDA_SUCCESS || current == nullptr) {
        int dev_index = 0;
        cudaError_t err = cudaGetDevice(&dev_index);
        if (err == cudaSuccess) err = cudaSetDevice(dev_index);
        if (err != cudaSuccess) return record_cuda_error(err);
    }
    return FMD_OK;
}

}  // namespace fmd
