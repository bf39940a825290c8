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

// N adjacent elements.  Rows may start at any element, so the types used for memory are aligned to one element only
// (gfx950 loads 16 bytes from any address; a wave's 1 KiB then touches nine 128-byte lines instead of eight).
template <class T, int N>
struct VecOf {
  typedef T type __attribute__((ext_vector_type(N)));
  typedef type mem __attribute__((aligned(sizeof(T))));
};
template <class T>
struct VecOf<T, 1> {
  typedef T type;
  typedef T mem;
};
template <class T, int N>
using vec_t = typename VecOf<T, N>::type;

// Elements of a 16-byte access, the width of every row access where a row is that long.
template <class T>
constexpr int kVec = 16 / (int)sizeof(T);

template <class T, int N>
__device__ __forceinline__ vec_t<T, N> load_vec(const T *p) {
  return *reinterpret_cast<const typename VecOf<T, N>::mem *>(p);
}
template <class T, int N>
__device__ __forceinline__ vec_t<T, N> load_vec_stream(const T *p) {
  return __builtin_nontemporal_load(reinterpret_cast<const typename VecOf<T, N>::mem *>(p));
}
template <class T, int N>
__device__ __forceinline__ void store_vec(T *p, vec_t<T, N> v) {
  *reinterpret_cast<typename VecOf<T, N>::mem *>(p) = v;
}
template <class T, int N>
__device__ __forceinline__ void store_vec_stream(T *p, vec_t<T, N> v) {
  __builtin_nontemporal_store(v, reinterpret_cast<typename VecOf<T, N>::mem *>(p));
}
template <class T, int N>
__device__ __forceinline__ float elem(const vec_t<T, N> &v, int i) {
  if constexpr (N == 1) return to_f32(v);
  else return to_f32(v[i]);
}
template <class T, int N>
__device__ __forceinline__ vec_t<T, N> round_vec(const float *f) {
  vec_t<T, N> v;
  if constexpr (N == 1) v = from_f32<T>(f[0]);
  else {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = from_f32<T>(f[i]);
  }
  return v;
}

// A row of `cols` elements (cols >= N) is covered by ceil(cols / N) accesses of N elements.  Where N does not divide cols
// the last one is moved back to end with the row: it repeats elements of the one before, and stores to them repeat the
// same values.  Slot j starts at column slot_column(j); its first slot_repeats(j) elements are repeats.
template <int N>
__device__ __forceinline__ int row_slots(int cols) {
  return (int)(((unsigned)cols + (N - 1)) / N);
}
template <int N>
__device__ __forceinline__ int slot_column(int j, int cols) {
  return min(j * N, cols - N);
}
template <int N>
__device__ __forceinline__ int slot_repeats(int j, int cols) {
  return max(0, j * N - (cols - N));
}

// Sum over aligned groups of LANES lanes (a power of two up to 64; FROM: already summed over groups of so many), in every
// lane, of a float, of two side by side (their steps fill each other's waits) or, up to 16 lanes, of a double.  The steps inside 16 lanes are DPP moves (quad permutes, mirrors
// of 8 and of 16: each pairs lanes whose partial sums cover disjoint halves, as an xor would).
template <int CTRL>
__device__ __forceinline__ int dpp_move(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, false);
}
template <int CTRL>
__device__ __forceinline__ float dpp_move(float v) {
  return __builtin_bit_cast(float, dpp_move<CTRL>(__builtin_bit_cast(int, v)));
}
template <int CTRL>
__device__ __forceinline__ float2 dpp_move(float2 v) {
  return make_float2(dpp_move<CTRL>(v.x), dpp_move<CTRL>(v.y));
}
template <int CTRL>
__device__ __forceinline__ double dpp_move(double v) {
  const int2 w = __builtin_bit_cast(int2, v);
  return __builtin_bit_cast(double, make_int2(dpp_move<CTRL>(w.x), dpp_move<CTRL>(w.y)));
}
__device__ __forceinline__ float lane_xor(float v, int m) { return __shfl_xor(v, m); }
__device__ __forceinline__ float2 lane_xor(float2 v, int m) { return make_float2(__shfl_xor(v.x, m), __shfl_xor(v.y, m)); }
template <int LANES, int FROM = 1, class V>
__device__ __forceinline__ V lanes_sum(V v) {
  if constexpr (LANES >= 2 && FROM < 2) v += dpp_move<0xB1>(v);    // quad_perm [1,0,3,2]
  if constexpr (LANES >= 4 && FROM < 4) v += dpp_move<0x4E>(v);    // quad_perm [2,3,0,1]
  if constexpr (LANES >= 8) v += dpp_move<0x141>(v);               // row_half_mirror
  if constexpr (LANES >= 16) v += dpp_move<0x140>(v);              // row_mirror
  if constexpr (LANES >= 32) v += lane_xor(v, 16);
  if constexpr (LANES >= 64) v += lane_xor(v, 32);
  return v;
}

// s / n, rounded once, with inv = 1 / n rounded: the remainder of the first quotient is exact.  (s * inv alone misses whole
// quotients: 1000.0f * 1000 * (1.0f / 1000) is 1000.00006, which makes -0.02 of a constant row where the variance is 0.)
__device__ __forceinline__ float quotient(float s, float n, float inv) {
  const float q = s * inv, better = fmaf(fmaf(-q, n, s), inv, q);
  return fabsf(q) <= 3.402823466e38f ? better : q;   // infinities stay
}

// Column slots of a row shared by `lanes` threads, VPT slots each: thread t has slots t, t + lanes, ...
template <int VEC, int VPT>
struct RowSlots {
  int col[VPT];       // first column (threads behind the row repeat its last slot)
  int skip[VPT];      // elements of the slot that are not this thread's to count: repeats, or all VEC behind the row
  bool whole[VPT];    // wave-uniform: no lane of the wave skips anything
  __device__ __forceinline__ RowSlots(int t, int lanes, int cols) {
    const int slots = row_slots<VEC>(cols);
#pragma unroll
    for (int k = 0; k < VPT; k++) {
      const int j = t + k * lanes;
      col[k] = slot_column<VEC>(min(j, slots - 1), cols);
      skip[k] = j < slots ? slot_repeats<VEC>(j, cols) : VEC;
      whole[k] = __ballot(skip[k] != 0) == 0;
    }
  }
};

// Inputs too large to be in the 256 MB memory-side cache from whatever wrote them are read past the caches.
inline bool past_caches(size_t bytes) { return bytes > ((size_t)256 << 20); }

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
