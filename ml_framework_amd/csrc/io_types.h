// io_types.h -- the three activation types of the sequence operators (fp32,
// fp16, bf16): storage, conversion and 4- / 16-byte loads. Arithmetic is fp32;
// a value is rounded (to nearest even) once, on its way to memory.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/seera_hip.h"

namespace seera {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(f16_t v) { return (float)v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return (float)v; }

template <class T>
__device__ __forceinline__ T from_f32(float v) {
    return (T)v;
}

// N consecutive values, loaded and stored as one access (the address must be
// aligned to all of them).
template <class T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

// Bytes of one value of a SEERA_DTYPE_*, 0 for an unknown one.
inline int dtype_bytes(int dtype) {
    return dtype == SEERA_DTYPE_F32 ? 4 : dtype == SEERA_DTYPE_F16 || dtype == SEERA_DTYPE_BF16 ? 2 : 0;
}

inline bool aligned_to(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace seera
