// Element types and row access of the token-model operators: rows of adjacent elements at any alignment, arithmetic in
// 32 bits, one rounding (to nearest even) on the way out.
#pragma once
#include <hip/hip_runtime.h>

#include "subblock.h"

namespace hfuse {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <class T>
__device__ __forceinline__ float to_f32(T v) {
  return (float)v;
}
template <class T>
__device__ __forceinline__ T from_f32(float v) {
  return (T)v;   // round to nearest even (v_cvt_pk_bf16_f32 / v_cvt_f16_f32)
}

// Sum over the 64 lanes, in every lane: a butterfly, so the order of the additions is fixed.
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

// Calls f with a value of the type that `type` (HF_F32 / HF_BF16 / HF_F16) names.
template <class F>
hipError_t with_type(int type, F f) {
  switch (type) {
    case 0: return f(float{});
    case 1: return f(bf16_t{});
    default: return f(f16_t{});
  }
}

}  // namespace hfuse
