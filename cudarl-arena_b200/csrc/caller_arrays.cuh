// caller_arrays.cuh -- what the entry points on the caller's own device arrays share: where an array is, its types, and the arithmetic on two floats at once.
#pragma once
#include "internal.h"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>
#include <cstdio>

namespace cudarl {

// A call of the runtime that fails is remembered by it until somebody asks.  What has been reported here is forgotten there, so that no later call takes it for its own.
inline int fail_cuda(const char* what, cudaError_t e) noexcept {
    cudaGetLastError();
    char text[256];
    std::snprintf(text, sizeof text, "%s: %s", what, cudaGetErrorString(e));
    return fail_global(1000 + (int)e, text);
}

// A launch that answers for itself (cudaGetLastError after a launch would also give what an earlier call has left).
template <class... Params, class... Args>
inline cudaError_t launch(void (*kernel)(Params...), unsigned grid, unsigned block, cudaStream_t st, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid); cfg.blockDim = dim3(block); cfg.stream = st;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

inline size_t type_bytes(int type) { return type == CUDARL_F32 ? 4u : 2u; }

// The one device that all arrays of a call are on.  An address of the host, or of another device than the first array's, would be a fault in the
// kernel and is refused here.
class CallerArrays {
    int device_ = -1;
public:
    int device() const { return device_; }
    void expect(int device) { device_ = device; }
    int check(const char* name, const void* p, size_t align) noexcept {
        char text[160];
        if (reinterpret_cast<uintptr_t>(p) % align) {
            std::snprintf(text, sizeof text, "%s is not aligned to %zu bytes", name, align);
            return fail_global(-1, text);
        }
        cudaPointerAttributes a;
        const cudaError_t e = cudaPointerGetAttributes(&a, p);
        if (e != cudaSuccess) return fail_cuda("cudaPointerGetAttributes", e);
        if (a.type == cudaMemoryTypeManaged) return 0;
        if (a.type != cudaMemoryTypeDevice) {
            std::snprintf(text, sizeof text, "%s is not device memory", name);
            return fail_global(-1, text);
        }
        if (device_ < 0) device_ = a.device;
        if (a.device != device_) {
            std::snprintf(text, sizeof text, "%s is on device %d, other arrays are on device %d", name, a.device, device_);
            return fail_global(-1, text);
        }
        return 0;
    }
    int check_if(const char* name, const void* p, size_t align) noexcept { return p ? check(name, p, align) : 0; }
};

// Makes a device current for the length of a call (a negative one leaves what is).
class CurrentDevice {
    int before_ = -1;
public:
    cudaError_t set(int device) noexcept {
        if (device < 0) return cudaSuccess;
        int now = 0;
        cudaError_t e = cudaGetDevice(&now);
        if (e != cudaSuccess || now == device) return e;
        e = cudaSetDevice(device);
        if (e == cudaSuccess) before_ = now;
        return e;
    }
    ~CurrentDevice() { if (before_ >= 0) cudaSetDevice(before_); }
};

// Of the current device.
inline cudaError_t multiprocessors(int* out) noexcept {
    int device = 0;
    const cudaError_t e = cudaGetDevice(&device);
    return e != cudaSuccess ? e : cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, device);
}

// One value as a float, and a float rounded to nearest into one.
template <int TYPE> struct Of;
template <> struct Of<CUDARL_F32> {
    using T = float;
    static __device__ __forceinline__ float get(T v) { return v; }
    static __device__ __forceinline__ T put(float v) { return v; }
};
template <> struct Of<CUDARL_BF16> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ float get(T v) { return __bfloat162float(v); }
    static __device__ __forceinline__ T put(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Of<CUDARL_F16> {
    using T = __half;
    static __device__ __forceinline__ float get(T v) { return __half2float(v); }
    static __device__ __forceinline__ T put(float v) { return __float2half_rn(v); }
};

// Two floats for the instructions that take two: half as many to issue, each of the two rounded as by itself.  (mul2 into add2 may become one fma2.)
typedef unsigned long long Two;
__device__ __forceinline__ Two two(float a, float b) { Two r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void apart(Two v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) { Two r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ Two add2(Two a, Two b) { Two r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ Two mul2(Two a, Two b) { Two r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }

}  // namespace cudarl
