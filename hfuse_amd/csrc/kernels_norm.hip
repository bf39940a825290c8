// Layer norm over the last dimension and its gradient.
#include <algorithm>

#include "device/rows.h"
#include "launch.h"

namespace hfuse {
namespace {

constexpr int kThreads = 256;

// Sum over the workgroup, in every thread.
__device__ __forceinline__ float block_sum(float v, float *part) {
  v = wave_sum(v);
  __syncthreads();   // the slots may still be read for the sum before
  if ((threadIdx.x & 63u) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0f;
#pragma unroll
  for (int w = 0; w < kThreads / 64; w++) v += part[w];
  return v;
}

// One workgroup a row: mean, mean square of the differences, output; the row is read three times (cache hits).
template <class T, class P>
__global__ __launch_bounds__(kThreads) void layer_norm_kernel(hf_layer_norm_args a) {
  __shared__ float part[kThreads / 64];
  const int cols = (int)a.cols, tid = (int)threadIdx.x;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    T *y = static_cast<T *>(a.y) + row * a.y_stride;
    float s = 0.0f;
    for (int c = tid; c < cols; c += kThreads) s += to_f32(x[c]);
    const float mean = block_sum(s, part) / (float)cols;
    s = 0.0f;
    for (int c = tid; c < cols; c += kThreads) {
      const float d = to_f32(x[c]) - mean;
      s += d * d;
    }
    const float rstd = 1.0f / sqrtf(block_sum(s, part) / (float)cols + a.eps);
    for (int c = tid; c < cols; c += kThreads) {
      const float w = a.weight ? to_f32(static_cast<const P *>(a.weight)[c]) : 1.0f;
      const float b = a.bias ? to_f32(static_cast<const P *>(a.bias)[c]) : 0.0f;
      y[c] = from_f32<T>((to_f32(x[c]) - mean) * rstd * w + b);
    }
    if (tid == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
  }
}

template <class T, class P>
__global__ __launch_bounds__(kThreads) void layer_norm_dx_kernel(hf_layer_norm_backward_args a) {
  __shared__ float part[kThreads / 64];
  const int cols = (int)a.cols, tid = (int)threadIdx.x;
  const P *weight = static_cast<const P *>(a.weight);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    const T *dy = static_cast<const T *>(a.dy) + row * a.dy_stride;
    T *dx = static_cast<T *>(a.dx) + row * a.dx_stride;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float sg = 0.0f, sgh = 0.0f;
    for (int c = tid; c < cols; c += kThreads) {
      const float g = to_f32(dy[c]) * (weight ? to_f32(weight[c]) : 1.0f);
      sg += g;
      sgh += g * ((to_f32(x[c]) - mean) * rstd);
    }
    sg = block_sum(sg, part) / (float)cols;
    sgh = block_sum(sgh, part) / (float)cols;
    for (int c = tid; c < cols; c += kThreads) {
      const float g = to_f32(dy[c]) * (weight ? to_f32(weight[c]) : 1.0f);
      const float h = (to_f32(x[c]) - mean) * rstd;
      dx[c] = from_f32<T>(rstd * (g - sg - h * sgh));
    }
  }
}

// One thread a column, down all rows.
template <class T, class P>
__global__ __launch_bounds__(kThreads) void layer_norm_dparams_kernel(hf_layer_norm_backward_args a) {
  const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= a.cols) return;
  const T *x = static_cast<const T *>(a.x) + c, *dy = static_cast<const T *>(a.dy) + c;
  float dw = 0.0f, db = 0.0f;
  for (int64_t row = 0; row < a.rows; row++) {
    const float g = to_f32(dy[row * a.dy_stride]);
    db += g;
    if (a.dweight) dw += g * ((to_f32(x[row * a.x_stride]) - a.mean[row]) * a.rstd[row]);
  }
  if (a.dweight) static_cast<P *>(a.dweight)[c] = from_f32<P>(dw);
  if (a.dbias) static_cast<P *>(a.dbias)[c] = from_f32<P>(db);
}

template <class T, class P>
hipError_t norm_forward(const hf_layer_norm_args &a, int cus, hipStream_t s) {
  const int64_t grid = std::min<int64_t>(a.rows, (int64_t)cus * 64);
  hipLaunchKernelGGL((layer_norm_kernel<T, P>), dim3((unsigned)grid), dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

template <class T, class P>
hipError_t norm_backward(const hf_layer_norm_backward_args &a, int cus, hipStream_t s) {
  if (a.dx && a.rows > 0) {
    const int64_t grid = std::min<int64_t>(a.rows, (int64_t)cus * 64);
    hipLaunchKernelGGL((layer_norm_dx_kernel<T, P>), dim3((unsigned)grid), dim3(kThreads), 0, s, a);
  }
  if (a.dweight || a.dbias) {
    const int64_t grid = (a.cols + kThreads - 1) / kThreads;
    hipLaunchKernelGGL((layer_norm_dparams_kernel<T, P>), dim3((unsigned)grid), dim3(kThreads), 0, s, a);
  }
  return hipGetLastError();
}

}  // namespace

size_t layer_norm_backward_workspace(const hf_layer_norm_backward_args &, int) { return 0; }

hipError_t launch_layer_norm(const hf_layer_norm_args &a, int cus, hipStream_t s) {
  if (a.rows == 0) return hipSuccess;
  return with_type(a.type, [&](auto t) {
    using T = decltype(t);
    return a.param_type == HF_F32 ? norm_forward<T, float>(a, cus, s) : norm_forward<T, T>(a, cus, s);
  });
}

hipError_t launch_layer_norm_backward(const hf_layer_norm_backward_args &a, int cus, hipStream_t s) {
  return with_type(a.type, [&](auto t) {
    using T = decltype(t);
    return a.param_type == HF_F32 ? norm_backward<T, float>(a, cus, s) : norm_backward<T, T>(a, cus, s);
  });
}

}  // namespace hfuse
