// Device-scope loads and stores for data exchanged between workgroups of one
// launch (the split-K partials of the short-prompt prefill GEMM).  MI355X
// has one L2 per XCD and they are not coherent with each other, so such data
// is accessed with device-scope (sc1) operations -- the code the compiler
// emits for agent-scope relaxed atomics -- instead of cached ones.  Data
// produced by an earlier launch needs none of this: the kernel boundary
// writes back and invalidates the caches.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace tmg {

__device__ __forceinline__ float ld_dev(const float *p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ void st_dev(float *p, float v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The same for two neighbouring floats, 8-byte aligned.
__device__ __forceinline__ float2 ld_dev2(const float *p) {
    const unsigned long long v = __hip_atomic_load(reinterpret_cast<const unsigned long long *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

__device__ __forceinline__ void st_dev2(float *p, float x, float y) {
    const unsigned long long v = (unsigned long long)__float_as_uint(y) << 32 | __float_as_uint(x);
    __hip_atomic_store(reinterpret_cast<unsigned long long *>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

}  // namespace tmg
