// Shared pieces of the memory-over-ticks kernels (fg_rotate.cu, fg_decay.cu): values of the three types as fp32, and the
// entry points' error handling. No counterpart in the reference, whose fly actor has no memory (flyguy/fly.py:76).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <string>

#include "fg_once.h"
#include "flyguy_b200.h"

namespace fgm {

constexpr int kSms = 148;                                    // of a B200, the only device these are built for

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <class T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

__device__ __forceinline__ float warp_sum(float s) {
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

// pairs of fp32 in one instruction
__device__ __forceinline__ uint64_t two(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}
__device__ __forceinline__ void halves(uint64_t x, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x));
}
// the two halves' sum
__device__ __forceinline__ float sum2(uint64_t x) {
    float a, b;
    halves(x, a, b);
    return a + b;
}

struct MemErr {
    std::string msg;
};
std::string& last_error();

#define MCK(call)                                                                                         \
    do {                                                                                                  \
        cudaError_t e_ = (call);                                                                          \
        if (e_ != cudaSuccess) throw ::fgm::MemErr{std::string(#call) + ": " + cudaGetErrorString(e_)};  \
    } while (0)

// runs f; whatever it throws becomes -1 and the calling thread's message
template <class F>
long long mem_guard(F&& f) {
    try {
        const long long r = f();
        last_error().clear();
        return r;
    } catch (const MemErr& e) {
        last_error() = e.msg;
    } catch (const std::exception& e) {
        last_error() = e.what();
    }
    return -1;
}

inline void need(bool ok, const char* what) {
    if (!ok) throw MemErr{what};
}

// f with a value of the type that FG_F32 / FG_BF16 / FG_F16 names
template <class F>
void by_type(long long type, F&& f) {
    if (type == FG_F32) f(float());
    else if (type == FG_BF16) f(__nv_bfloat16());
    else if (type == FG_F16) f(__half());
    else throw MemErr{"unknown type"};
}

// kernel may be launched with so many bytes of shared memory on the current device
template <class K>
void allow_shared(K* kernel, int bytes) {
    MCK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
}
inline int current_device() {
    int d = 0;
    MCK(cudaGetDevice(&d));
    return d;
}

}  // namespace fgm
