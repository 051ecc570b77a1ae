// What the sequence operators (linear attention, norms) share: element types, vector access, reductions.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pathsig_hip.h"

namespace psig {

void set_error(const char *fmt, ...);

namespace seq {

using bf16 = __bf16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(bf16 x) { return (float)x; }
// (round to nearest, ties to even)
template <typename T>
__device__ __forceinline__ T from_float(float x) {
    return (T)x;
}

// N consecutive elements as one access of up to 16 bytes (N = 1: of one element)
template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
    T v[N];
};

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

inline int launch_status(const char *what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return PATHSIG_OK;
    set_error("%s: %s", what, hipGetErrorString(e));
    return PATHSIG_ERR_LAUNCH;
}

}  // namespace seq
}  // namespace psig
