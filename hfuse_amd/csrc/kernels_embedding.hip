// Token embedding: rows of a table by token id, scaled, and the gradient of the table.
#include <algorithm>

#include "device/rows.h"
#include "launch.h"

namespace hfuse {
namespace {

constexpr int kThreads = 256;

// One workgroup a token.
template <class T, class I>
__global__ __launch_bounds__(kThreads) void embedding_kernel(hf_embedding_args a) {
  for (int64_t i = blockIdx.x; i < a.ntokens; i += gridDim.x) {
    const int64_t t = (int64_t) static_cast<const I *>(a.tokens)[i];
    T *out = static_cast<T *>(a.out) + i * a.out_stride;
    const bool used = t >= 0 && t < a.vocab;
    const T *w = static_cast<const T *>(a.weight) + (used ? t : 0) * a.weight_stride;
    for (int64_t c = threadIdx.x; c < a.cols; c += kThreads)
      out[c] = used ? (a.scale == 1.0f ? w[c] : from_f32<T>(to_f32(w[c]) * a.scale)) : from_f32<T>(0.0f);
  }
}

// One workgroup a row of the table and kThreads columns: it looks through all tokens for its own.
template <class T, class O, class I>
__global__ __launch_bounds__(kThreads) void embedding_backward_kernel(hf_embedding_backward_args a) {
  const I *tokens = static_cast<const I *>(a.tokens);
  const int lane = (int)threadIdx.x & 63;
  const int64_t c = (int64_t)blockIdx.y * kThreads + threadIdx.x;
  for (int64_t v = blockIdx.x; v < a.vocab; v += gridDim.x) {
    float acc = 0.0f;
    if (v != a.padding_idx) {
      for (int64_t base = 0; base < a.ntokens; base += 64) {
        const int64_t i = base + lane;
        unsigned long long mine = __ballot(i < a.ntokens && (int64_t)tokens[i] == v);
        while (mine) {
          const int64_t row = base + __builtin_ctzll(mine);
          mine &= mine - 1;
          if (c < a.cols) acc += to_f32(static_cast<const T *>(a.dy)[row * a.dy_stride + c]);
        }
      }
    }
    if (c < a.cols) static_cast<O *>(a.dweight)[v * a.dweight_stride + c] = from_f32<O>(acc * a.scale);
  }
}

template <class T, class O, class I>
hipError_t embed_backward(const hf_embedding_backward_args &a, hipStream_t s) {
  const unsigned tiles = (unsigned)((a.cols + kThreads - 1) / kThreads);
  if (tiles > 65535u) return hipErrorInvalidValue;
  const unsigned grid = (unsigned)std::min<int64_t>(a.vocab, 1 << 20);
  hipLaunchKernelGGL((embedding_backward_kernel<T, O, I>), dim3(grid, tiles), dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace

size_t embedding_backward_workspace(const hf_embedding_backward_args &, int) { return 0; }

hipError_t launch_embedding(const hf_embedding_args &a, int cus, hipStream_t s) {
  if (a.ntokens == 0) return hipSuccess;
  const unsigned grid = (unsigned)std::min<int64_t>(a.ntokens, (int64_t)cus * 64);
  return with_type(a.type, [&](auto t) {
    using T = decltype(t);
    if (a.index_type == HF_I64) hipLaunchKernelGGL((embedding_kernel<T, int64_t>), dim3(grid), dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL((embedding_kernel<T, int32_t>), dim3(grid), dim3(kThreads), 0, s, a);
    return hipGetLastError();
  });
}

hipError_t launch_embedding_backward(const hf_embedding_backward_args &a, int cus, hipStream_t s) {
  (void)cus;
  return with_type(a.type, [&](auto t) {
    using T = decltype(t);
    if (a.index_type == HF_I64)
      return a.out_type == HF_F32 ? embed_backward<T, float, int64_t>(a, s) : embed_backward<T, T, int64_t>(a, s);
    return a.out_type == HF_F32 ? embed_backward<T, float, int32_t>(a, s) : embed_backward<T, T, int32_t>(a, s);
  });
}

}  // namespace hfuse
