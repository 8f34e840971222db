// Device helpers shared by the kernels around sampled codes (kernels_sample.hip) and codebook lookup (kernels_lookup.hip):
// the three element types of their matrices and loads / stores of 2, 4, 8 or 16 bytes of them.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "vq_common.h"

namespace vq {

// Elements are held in their own type and computed with in f32.  The one rounding to 16 bits is the conversion back, to
// nearest even (a cast of __bf16 / _Float16 is).
template <class T> __device__ __forceinline__ float widen(T v) { return (float)v; }
template <class T> __device__ __forceinline__ T narrow(float v) { return (T)v; }

// BYTES of consecutive elements, moved by one load or store; the address is a multiple of BYTES
template <class T, int BYTES>
struct alignas(BYTES) Pack {
    static constexpr int E = BYTES / (int)sizeof(T);
    T v[E];
};

}  // namespace vq
