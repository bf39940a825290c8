// The gradient of layer norm: with h = (x - mean) rstd and g = dy w,
//   dx = rstd (g - mean(g) - h mean(g h)),  dweight = sum over rows of dy h,  dbias = sum over rows of dy.
//
// Bound by HBM: x and dy are read once and dx is written once, about 14 operations an element.  Measured on an MI355X:
// 32768 x 8192 bf16 274 us + 5 us for the sums of the parts = 5.8 TB/s, 5003 x 1155 f16 12.7 + 4.2 us, 64 x 1024 5.9 + 2.5;
// 16384 x 8192 f32, whose rows take workgroups of 1024 that form h and g twice, 305 + 5 us = 5.2 TB/s.  The part draws so much
// power there that arithmetic costs time although it hides behind the memory: h and g formed twice instead of kept in
// registers 289 -> 395 us (32768 x 8192 bf16, many in turn).
#include <algorithm>

#include "device/rows.h"
#include "launch.h"

// Every product and sum as it is written: elements that two slots hold come out alike whichever stores last.
#pragma clang fp contract(off)

namespace hfuse {
namespace {

// One pass over the rows: a group of lanes holds a row of x and of dy in registers, VPT slots of 16 bytes each, forms the
// two sums over the row that dx needs, writes dx, and adds dy * h and dy to the 32-bit sums of its columns, which stay in
// registers for all rows of the group.  The next row is on its way meanwhile.  A workgroup leaves one row of sums for
// dweight and one for dbias in `parts`; sum_parts_kernel adds them up in an order of its own.  One workgroup a CU
// (100 to 160 registers a thread, three or four waves a SIMD): two write twice the parts, 15.1 + 5.1 against 12.7 + 4.2 us at
// 5003 x 1155 f16, 276 + 7.3 against 274 + 5.1 at 32768 x 8192 bf16, and win 0.6 of 19 us at 131072 x 128.  LANES: lanes to a
// row, 0 for whole waves whose number the launch says.
template <class T, class P, int VEC, int VPT, int LANES, int BLOCK, bool PARAMS>
__global__ __launch_bounds__(BLOCK) void layer_norm_grad_kernel(hf_layer_norm_backward_args a, float *parts, int wide_lanes, bool stream) {
  constexpr bool kKeep = BLOCK < 1024 || VPT == 1;   // a workgroup of 1024 has 128 registers a thread: weights from the caches, h and g computed twice
  constexpr bool kAhead = BLOCK < 1024 || VPT * VEC < 16;   // ... and a second row of the longest does not fit
  constexpr bool kWide = LANES == 0 || LANES > 64;   // a row is whole waves
  __shared__ float2 part[2][16];
  const int lanes = LANES ? LANES : wide_lanes, groups = (int)blockDim.x / lanes;
  const int cols = (int)a.cols, t = (int)threadIdx.x % lanes, group = (int)threadIdx.x / lanes;
  const RowSlots<VEC, VPT> map(t, lanes, cols);
  const P *weight = static_cast<const P *>(a.weight);
  const bool want_dx = a.dx != nullptr, want_h = want_dx || a.dweight;   // dbias alone reads dy only
  auto load_weight = [&](int k) { return weight && want_dx ? load_vec<P, VEC>(weight + map.col[k]) : (vec_t<P, VEC>)(P)1.0f; };
  vec_t<P, VEC> kept[kKeep ? VPT : 1];
  if constexpr (kKeep) {
#pragma unroll
    for (int k = 0; k < VPT; k++) kept[k] = load_weight(k);
  }
  float dw[PARAMS ? VPT : 1][VEC], db[PARAMS ? VPT : 1][VEC];
#pragma unroll
  for (int k = 0; k < (PARAMS ? VPT : 1); k++)
#pragma unroll
    for (int e = 0; e < VEC; e++) dw[k][e] = db[k][e] = 0.0f;

  const float n = (float)cols, inv = 1.0f / n;
  const int64_t step = (int64_t)gridDim.x * groups;
  vec_t<T, VEC> next_x[VPT], next_dy[VPT];
  float next_mean = 0.0f, next_rstd = 0.0f;
  auto fetch = [&](int64_t row) {
    row = min(row, a.rows - 1);
    const T *dy = static_cast<const T *>(a.dy) + row * a.dy_stride;
#pragma unroll
    for (int k = 0; k < VPT; k++) next_dy[k] = stream ? load_vec_stream<T, VEC>(dy + map.col[k]) : load_vec<T, VEC>(dy + map.col[k]);
    if (want_h) {
      const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
#pragma unroll
      for (int k = 0; k < VPT; k++) next_x[k] = stream ? load_vec_stream<T, VEC>(x + map.col[k]) : load_vec<T, VEC>(x + map.col[k]);
      next_mean = a.mean[row];
      next_rstd = a.rstd[row];
    }
  };
#pragma unroll
  for (int k = 0; k < VPT; k++) next_x[k] = (vec_t<T, VEC>)(T)0.0f;
  if (kAhead) fetch((int64_t)blockIdx.x * groups + group);
  int turn = 0;
  for (int64_t base = (int64_t)blockIdx.x * groups; base < a.rows; base += step) {   // all groups of a workgroup make the same trips
    const int64_t row = base + group;
    const bool mine = row < a.rows;
    if (!kAhead) fetch(row);
    const float mean = next_mean, rstd = next_rstd;
    vec_t<T, VEC> x[VPT], dy[VPT];
#pragma unroll
    for (int k = 0; k < VPT; k++) {
      x[k] = next_x[k];
      dy[k] = next_dy[k];
    }
    if (kAhead && base + step < a.rows) fetch(row + step);
    float sg = 0.0f, sgh = 0.0f, hs[kKeep ? VPT : 1][VEC], gs[kKeep ? VPT : 1][VEC];
    auto h_of = [&](int k, int e) { return (elem<T, VEC>(x[k], e) - mean) * rstd; };
#pragma unroll
    for (int k = 0; k < VPT; k++) {
      const vec_t<P, VEC> w = kKeep ? kept[kKeep ? k : 0] : load_weight(k);
      auto slot = [&](auto whole) {
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          const float d = elem<T, VEC>(dy[k], e), h = h_of(k, e), g = d * elem<P, VEC>(w, e);
          if constexpr (kKeep) {
            hs[k][e] = h;
            gs[k][e] = g;
          }
          if (whole() || e >= map.skip[k]) {
            sg += g;
            sgh = fmaf(g, h, sgh);
          }
          if (PARAMS && mine) {   // (repeated columns are summed twice, alike)
            dw[k][e] = fmaf(d, h, dw[k][e]);
            db[k][e] += d;
          }
        }
      };
      if (map.whole[k]) slot([] { return true; });
      else slot([] { return false; });
    }
    if (!want_dx) continue;
    sg = lanes_sum<(kWide ? 64 : LANES)>(sg);
    sgh = lanes_sum<(kWide ? 64 : LANES)>(sgh);
    if constexpr (kWide) {   // the waves of the row, 16 at most
      if ((threadIdx.x & 63u) == 0) part[turn][threadIdx.x >> 6] = make_float2(sg, sgh);
      __syncthreads();   // two slots in turn: a slot is written again only behind the other one's barrier
      const int i = (int)threadIdx.x & 15, waves = lanes >> 6;
      const float2 v = i < waves ? part[turn][group * waves + i] : make_float2(0.0f, 0.0f);
      sg = lanes_sum<16>(v.x);
      sgh = lanes_sum<16>(v.y);
      turn ^= 1;
    }
    sg = quotient(sg, n, inv) * rstd;   // (of a constant g, such as the gradient of a sum, nothing is left)
    sgh *= inv * rstd;
    if (mine) {
      T *dx = static_cast<T *>(a.dx) + row * a.dx_stride;
#pragma unroll
      for (int k = 0; k < VPT; k++) {
        if (map.skip[k] == VEC) continue;
        float out[VEC];
        if constexpr (kKeep) {
#pragma unroll
          for (int e = 0; e < VEC; e++) out[e] = fmaf(gs[k][e], rstd, -fmaf(hs[k][e], sgh, sg));
        } else {
          const vec_t<P, VEC> w = load_weight(k);
#pragma unroll
          for (int e = 0; e < VEC; e++) out[e] = fmaf(elem<T, VEC>(dy[k], e) * elem<P, VEC>(w, e), rstd, -fmaf(h_of(k, e), sgh, sg));
        }
        store_vec_stream<T, VEC>(dx + map.col[k], round_vec<T, VEC>(out));
      }
    }
  }

  if constexpr (PARAMS) {
    const size_t width = (size_t)row_slots<VEC>(cols) * VEC;
    float *dw_part = parts + (size_t)blockIdx.x * 2 * width, *db_part = dw_part + width;
    // sets of threads with sums of their own: the groups, or the waves where a wave holds several
    const int span = kWide ? lanes : 64, sets = (int)blockDim.x / span;
    __shared__ float sums[(BLOCK - 64) * VEC];
    const int set = (int)threadIdx.x / span, in_set = (int)threadIdx.x % span;
#pragma unroll
    for (int k = 0; k < VPT; k++) {
#pragma unroll
      for (int which = 0; which < 2; which++) {
        float v[VEC];
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          v[e] = which ? db[k][e] : dw[k][e];
          if constexpr (!kWide)
#pragma unroll
            for (int m = LANES; m < 64; m <<= 1) v[e] += __shfl_xor(v[e], m);   // the groups inside a wave
        }
        if (sets > 1) {
          if (set > 0)
#pragma unroll
            for (int e = 0; e < VEC; e++) sums[((set - 1) * VEC + e) * span + in_set] = v[e];
          __syncthreads();
          if (set == 0)
            for (int i = 0; i < sets - 1; i++)
#pragma unroll
              for (int e = 0; e < VEC; e++) v[e] += sums[(i * VEC + e) * span + in_set];
          __syncthreads();
        }
        if (set == 0 && in_set < lanes && map.skip[k] != VEC)
          store_vec<float, VEC>((which ? db_part : dw_part) + (size_t)(t + k * lanes) * VEC, round_vec<float, VEC>(v));
      }
    }
  }
}

// Rows too long for the registers of a workgroup: dx by itself, the rows read twice (the second time from the caches) ...
template <class T, class P>
__global__ __launch_bounds__(1024) void layer_norm_long_dx_kernel(hf_layer_norm_backward_args a) {
  constexpr int VEC = kVec<T>;
  __shared__ float2 part[2][16];
  const int cols = (int)a.cols, tid = (int)threadIdx.x, slots = row_slots<VEC>(cols);
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride, *dy = static_cast<const T *>(a.dy) + row * a.dy_stride;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float sg = 0.0f, sgh = 0.0f;
    auto weights = [&](int c) { return a.weight ? load_vec<P, VEC>(static_cast<const P *>(a.weight) + c) : (vec_t<P, VEC>)(P)1.0f; };
    for (int j = tid; j < slots; j += 1024) {
      const int c = slot_column<VEC>(j, cols), skip = slot_repeats<VEC>(j, cols);
      const vec_t<T, VEC> xv = load_vec<T, VEC>(x + c), dv = load_vec<T, VEC>(dy + c);
      const vec_t<P, VEC> wv = weights(c);
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        const float g = elem<T, VEC>(dv, e) * elem<P, VEC>(wv, e);
        if (e >= skip) {
          sg += g;
          sgh = fmaf(g, (elem<T, VEC>(xv, e) - mean) * rstd, sgh);
        }
      }
    }
    sg = lanes_sum<64>(sg);
    sgh = lanes_sum<64>(sgh);
    if ((tid & 63) == 0) part[turn][tid >> 6] = make_float2(sg, sgh);
    __syncthreads();
    sg = sgh = 0.0f;
    for (int i = 0; i < 16; i++) {
      sg += part[turn][i].x;
      sgh += part[turn][i].y;
    }
    sg /= (float)cols;
    sgh /= (float)cols;
    T *dx = static_cast<T *>(a.dx) + row * a.dx_stride;
    for (int j = tid; j < slots; j += 1024) {
      const int c = slot_column<VEC>(j, cols);
      const vec_t<T, VEC> xv = load_vec<T, VEC>(x + c), dv = load_vec<T, VEC>(dy + c);
      const vec_t<P, VEC> wv = weights(c);
      float out[VEC];
#pragma unroll
      for (int e = 0; e < VEC; e++)
        out[e] = rstd * (elem<T, VEC>(dv, e) * elem<P, VEC>(wv, e) - fmaf((elem<T, VEC>(xv, e) - mean) * rstd, sgh, sg));
      store_vec<T, VEC>(dx + c, round_vec<T, VEC>(out));
    }
  }
}

// ... and the sums down the columns, a thread a slot over every gridDim.y-th row.
template <class T>
__global__ __launch_bounds__(256) void layer_norm_long_params_kernel(hf_layer_norm_backward_args a, float *parts) {
  constexpr int VEC = kVec<T>;
  const int cols = (int)a.cols, slots = row_slots<VEC>(cols), j = (int)(blockIdx.x * 256 + threadIdx.x);
  if (j >= slots) return;
  const int c = slot_column<VEC>(j, cols);
  const T *x = static_cast<const T *>(a.x) + c, *dy = static_cast<const T *>(a.dy) + c;
  float dw[VEC], db[VEC];
#pragma unroll
  for (int e = 0; e < VEC; e++) dw[e] = db[e] = 0.0f;
#pragma unroll 4
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const vec_t<T, VEC> dv = load_vec<T, VEC>(dy + row * a.dy_stride);
    if (a.dweight) {
      const vec_t<T, VEC> xv = load_vec<T, VEC>(x + row * a.x_stride);
      const float mean = a.mean[row], rstd = a.rstd[row];
#pragma unroll
      for (int e = 0; e < VEC; e++) dw[e] = fmaf(elem<T, VEC>(dv, e), (elem<T, VEC>(xv, e) - mean) * rstd, dw[e]);
    }
#pragma unroll
    for (int e = 0; e < VEC; e++) db[e] += elem<T, VEC>(dv, e);
  }
  const size_t width = (size_t)slots * VEC;
  float *part = parts + (size_t)blockIdx.y * 2 * width + (size_t)j * VEC;
  store_vec<float, VEC>(part, round_vec<float, VEC>(dw));
  store_vec<float, VEC>(part + width, round_vec<float, VEC>(db));
}

// dweight and dbias from `nparts` rows of sums each: 64 columns a workgroup, whose sixteen waves take the rows in turn;
// their sums are added in the order of the waves.  Column c of the parts is slot c / vec, element c % vec.
template <class P>
__global__ __launch_bounds__(1024) void sum_parts_kernel(const float *parts, int nparts, int vec, int cols, P *dweight, P *dbias) {
  __shared__ float sums[16][64];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int width = (int)(((unsigned)cols + (unsigned)vec - 1) / (unsigned)vec) * vec;
  const int at = (int)blockIdx.x * 64 + lane;
  P *out = blockIdx.y ? dbias : dweight;
  if (!out) return;
  const float *p = parts + (size_t)blockIdx.y * width + min(at, width - 1);
  float s = 0.0f;
#pragma unroll 8
  for (int i = wave; i < nparts; i += 16) s += p[(size_t)i * 2 * (size_t)width];
  sums[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && at < width) {
    s = 0.0f;
    for (int i = 0; i < 16; i++) s += sums[i][lane];
    out[min(at / vec * vec, cols - vec) + at % vec] = from_f32<P>(s);
  }
}

// How the gradient is cut: lanes to a row, slots to a lane, threads of a workgroup, workgroups.
struct GradPlan {
  int vec, vpt, lanes, block, bound;   // bound: the launch bound of the kernel that runs
  bool in_registers;
  unsigned grid;   // workgroups with a part of the columns' sums each
  size_t bytes;
};

GradPlan plan_grad(const hf_layer_norm_backward_args &a, int cus) {
  GradPlan p;
  const int full = a.type == HF_F32 ? kVec<float> : kVec<bf16_t>;
  p.vec = a.cols < full ? 1 : full;
  const int64_t slots = (a.cols + p.vec - 1) / p.vec;
  const int waves = (int)std::min<int64_t>((slots + 63) / 64, 65);   // wavefronts with one slot a lane
  p.in_registers = waves <= (p.vec == 4 ? 64 : 32);
  // Two slots a lane, one where that leaves fewer lanes without a slot (their arithmetic costs the same), more where a
  // workgroup would not hold the row.
  p.vpt = waves == 1 || (waves < 8 && waves % 2) ? 1 : waves <= 32 ? 2 : 4;
  p.lanes = p.vpt == 4 ? 1024 : (waves + p.vpt - 1) / p.vpt * 64;
  if (waves == 1)
    for (p.lanes = 8; p.lanes < slots;) p.lanes *= 2;
  // As many groups as 512 threads hold; up to 1024 threads with one slot a lane, and two groups of five or six waves.
  p.bound = p.lanes <= 64 ? 512 : p.vpt == 1 || p.lanes > 768 ? 1024 : 768;
  p.block = std::max(1, (p.vpt == 1 && p.lanes > 64 ? 1024 : p.lanes > 256 && p.lanes <= 384 ? 768 : 512) / p.lanes) * p.lanes;
  if (p.in_registers) {
    const int64_t groups = p.block / p.lanes, sets = (a.rows + groups - 1) / groups;
    const int64_t trips = std::max<int64_t>(1, (sets + cus - 1) / cus);
    p.grid = (unsigned)((sets + trips - 1) / trips);   // every workgroup makes `trips` trips, or one less
  } else {
    p.grid = (unsigned)std::min<int64_t>(a.rows, 128);
  }
  const size_t width = (size_t)((a.cols + p.vec - 1) / p.vec) * p.vec;
  p.bytes = a.dweight || a.dbias ? (size_t)p.grid * 2 * width * sizeof(float) : 0;
  return p;
}

template <class T, class P, int VEC, int VPT, int LANES, int BLOCK>
hipError_t grad_rows(const hf_layer_norm_backward_args &a, const GradPlan &p, hipStream_t s) {
  const bool stream = past_caches((size_t)a.rows * (size_t)a.cols * sizeof(T) * 2);
  if (a.dweight || a.dbias)
    hipLaunchKernelGGL((layer_norm_grad_kernel<T, P, VEC, VPT, LANES, BLOCK, true>), dim3(p.grid), dim3(p.block), 0, s, a,
                       static_cast<float *>(a.workspace), p.lanes, stream);
  else
    hipLaunchKernelGGL((layer_norm_grad_kernel<T, P, VEC, VPT, LANES, BLOCK, false>), dim3(p.grid), dim3(p.block), 0, s, a, nullptr, p.lanes, stream);
  return hipGetLastError();
}

template <class T, class P>
hipError_t grad_in_registers(const hf_layer_norm_backward_args &a, const GradPlan &p, hipStream_t s) {
  constexpr int VEC = kVec<T>;
  if (p.vec == 1) return grad_rows<T, P, 1, 1, 8, 512>(a, p, s);
  switch (p.lanes) {
    case 8: return grad_rows<T, P, VEC, 1, 8, 512>(a, p, s);
    case 16: return grad_rows<T, P, VEC, 1, 16, 512>(a, p, s);
    case 32: return grad_rows<T, P, VEC, 1, 32, 512>(a, p, s);
    case 64: return p.vpt == 1 ? grad_rows<T, P, VEC, 1, 64, 512>(a, p, s) : grad_rows<T, P, VEC, 2, 64, 512>(a, p, s);
  }
  if (p.vpt == 1) return grad_rows<T, P, VEC, 1, 0, 1024>(a, p, s);
  if (p.bound == 768) return grad_rows<T, P, VEC, 2, 0, 768>(a, p, s);
  if (p.vpt == 2) return grad_rows<T, P, VEC, 2, 0, 1024>(a, p, s);
  if constexpr (VEC == 4)
    if (p.vpt == 4) return grad_rows<T, P, VEC, 4, 1024, 1024>(a, p, s);
  return hipErrorInvalidValue;
}

template <class T, class P>
hipError_t norm_backward(const hf_layer_norm_backward_args &a, int cus, hipStream_t s) {
  const GradPlan p = plan_grad(a, cus);
  const bool params = a.dweight || a.dbias;
  float *parts = static_cast<float *>(a.workspace);
  if (a.rows > 0 && p.in_registers) {
    const hipError_t e = grad_in_registers<T, P>(a, p, s);
    if (e != hipSuccess) return e;
  } else if (a.rows > 0) {
    if (a.dx) hipLaunchKernelGGL((layer_norm_long_dx_kernel<T, P>), dim3((unsigned)std::min<int64_t>(a.rows, (int64_t)cus * 2)), dim3(1024), 0, s, a);
    if (params) hipLaunchKernelGGL((layer_norm_long_params_kernel<T>), dim3((unsigned)((a.cols + kVec<T> * 256 - 1) / (kVec<T> * 256)), p.grid), dim3(256), 0, s, a, parts);
  }
  if (params) {
    const int64_t width = (a.cols + p.vec - 1) / p.vec * p.vec;
    hipLaunchKernelGGL((sum_parts_kernel<P>), dim3((unsigned)((width + 63) / 64), 2), dim3(1024), 0, s, parts, (int)(a.rows > 0 ? p.grid : 0), p.vec,
                       (int)a.cols, static_cast<P *>(a.dweight), static_cast<P *>(a.dbias));
  }
  return hipGetLastError();
}

}  // namespace

size_t layer_norm_backward_workspace(const hf_layer_norm_backward_args &a, int cus) { return plan_grad(a, cus).bytes; }

hipError_t launch_layer_norm_backward(const hf_layer_norm_backward_args &a, int cus, hipStream_t s) {
  return with_type(a.type, [&](auto t) {
    using T = decltype(t);
    return a.param_type == HF_F32 ? norm_backward<T, float>(a, cus, s) : norm_backward<T, T>(a, cus, s);
  });
}

}  // namespace hfuse
