// Layer norm over the last dimension: mean = sum(x) / n, var = sum((x - mean)^2) / n, y = (x - mean) / sqrt(var + eps) w + b.
//
// Bound by HBM: a row is read once and written once, about 8 operations an element (2 a byte in 16 bits).  Measured on an
// MI355X: 32768 x 8192 bf16 with float32 parameters 184 us = 5.8 TB/s (196 a launch under the profiler; a copy of 2 GiB
// reaches 4.9 TB/s there), 3001 x 1155 float32 8.2 us, one row of 4096 bf16 2.5 us (an empty kernel takes 1.3).  The variance
// is the mean of squared differences from the mean, not of squares, and where a row's sum is not exact the mean of the
// differences corrects both (centred): rows with a large mean lose nothing.  Outputs are stored past the caches, and
// inputs read past them where they cannot be there (past_caches): 193 -> 185 us.
#include <algorithm>
#include <type_traits>

#include "device/rows.h"
#include "launch.h"

// Every product and sum as it is written: elements that two slots hold come out alike whichever stores last.
#pragma clang fp contract(off)

namespace hfuse {
namespace {

// The sum of a row of 32-bit elements is rounded, so their differences d are taken from a number near the mean.  By how
// much it is off is the mean of d, whose terms are as small as the row's spread: mean(x) = near + mean(d), and
// var = mean(d^2) - mean(d)^2.  Of a constant row, d is a few units of x's last place, and their sum is exact.  A row whose
// mean is smaller than its spread needs none of it: the differences are rounded themselves, by as much as the sum was.
// 16-bit rows with a large mean have exact sums of up to 2^16 (bf16) or 2^13 elements (f16): 8 or 11 bits an element and one
// for every doubling make 24, and of f16 rows of more than 2^13 columns the sums of the waves are added in 64 bits.  Their
// mean is rounded once, 2^-16 or 2^-13 of the elements' own step, and nothing is corrected: the two operations an element would
// cost 184 -> 197 us at 32768 x 8192 bf16, and 360 -> 392 at 32768 x 16384 f16, where adding in 64 bits costs 360 -> 374.
struct Centre {
  float shift, rstd;   // d - shift: the difference from the mean
};
__device__ __forceinline__ Centre centred(float near, float sum_d, float sum_d2, float n, float inv, float eps) {
  Centre c;
  const float square = sum_d2 * inv;
  c.shift = near * near > square ? quotient(sum_d, n, inv) : 0.0f;   // (nor do rows out of range, of infinities or of NaN)
  const float var = fmaf(-c.shift, c.shift, square);
  c.rstd = rsqrtf((var < 0.0f ? 0.0f : var) + eps);                  // (a NaN stays)
  return c;
}

// A group of lanes holds a row in registers, VPT slots of 16 bytes each: the row is read once, the mean and then the mean
// square of the differences come from the registers, and the next row is on its way meanwhile.  A workgroup keeps its
// weights in registers for its rows.  LANES: lanes to a row, 0 for whole waves whose number the launch says.
template <class T, class P, int VEC, int VPT, int LANES, int BLOCK>
__global__ __launch_bounds__(BLOCK) void layer_norm_rows_kernel(hf_layer_norm_args a, int wide_lanes, bool stream) {
  constexpr bool kKeep = VPT <= 2 || BLOCK < 1024;   // weights and biases fit the registers next to two rows
  constexpr bool kCentre = sizeof(T) == 4;
  constexpr bool kWideJoin = std::is_same<T, f16_t>::value && VPT > 1 && BLOCK == 1024;   // f16 rows of more than 2^13 columns
  __shared__ float part[16];
  __shared__ float2 part2[16];
  const int lanes = LANES ? LANES : wide_lanes, groups = (int)blockDim.x / lanes;
  const int cols = (int)a.cols, t = (int)threadIdx.x % lanes, group = (int)threadIdx.x / lanes;
  const RowSlots<VEC, VPT> map(t, lanes, cols);
  const P *weight = static_cast<const P *>(a.weight), *bias = static_cast<const P *>(a.bias);
  auto load_params = [&](int k, vec_t<P, VEC> &w, vec_t<P, VEC> &b) {
    w = weight ? load_vec<P, VEC>(weight + map.col[k]) : (vec_t<P, VEC>)(P)1.0f;
    b = bias ? load_vec<P, VEC>(bias + map.col[k]) : (vec_t<P, VEC>)(P)0.0f;
  };
  vec_t<P, VEC> w[kKeep ? VPT : 1], b[kKeep ? VPT : 1];
  if constexpr (kKeep) {
#pragma unroll
    for (int k = 0; k < VPT; k++) load_params(k, w[k], b[k]);
  }
  const float n = (float)cols, inv = 1.0f / n;
  const double inv64 = kWideJoin ? 1.0 / (double)cols : 0.0;
  const int64_t step = (int64_t)gridDim.x * groups;
  // Sums over a row, of one value or two.  The waves of a wide one, 16 at most, leave theirs in LDS, and every lane has one of
  // them behind the barrier.  A row has two sums in arrays of their own: each is written again only behind the other's barrier.
  auto of_waves = [&](auto v, auto *part) {
    if ((threadIdx.x & 63u) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    const int i = (int)threadIdx.x & 15, waves = lanes >> 6;
    return i < waves ? part[group * waves + i] : decltype(v){};
  };
  auto sum_row = [&](auto v, auto *part) {
    v = lanes_sum<(LANES ? LANES : 64)>(v);
    if constexpr (LANES == 0) v = lanes_sum<16>(of_waves(v, part));
    return v;
  };
  vec_t<T, VEC> next[VPT];
  auto fetch = [&](int64_t row) {
    const T *x = static_cast<const T *>(a.x) + min(row, a.rows - 1) * a.x_stride;
#pragma unroll
    for (int k = 0; k < VPT; k++) next[k] = stream ? load_vec_stream<T, VEC>(x + map.col[k]) : load_vec<T, VEC>(x + map.col[k]);
  };
  fetch((int64_t)blockIdx.x * groups + group);
  for (int64_t base = (int64_t)blockIdx.x * groups; base < a.rows; base += step) {   // all groups of a workgroup make the same trips
    const int64_t row = base + group;
    vec_t<T, VEC> x[VPT];
#pragma unroll
    for (int k = 0; k < VPT; k++) x[k] = next[k];
    if (base + step < a.rows) fetch(row + step);
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < VPT; k++) {
      if (map.whole[k]) {
#pragma unroll
        for (int e = 0; e < VEC; e++) s += elem<T, VEC>(x[k], e);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; e++) s += e >= map.skip[k] ? elem<T, VEC>(x[k], e) : 0.0f;
      }
    }
    float near;
    if constexpr (kWideJoin) {   // (a wave has 2^11 elements at most: four waves' sums are exact)
      const float four = lanes_sum<4>(of_waves(lanes_sum<64>(s), part));
      near = (float)(lanes_sum<16, 4>((double)four) * inv64);
    } else {
      near = quotient(sum_row(s, part), n, inv);
    }
    s = 0.0f;
    float s2 = 0.0f, d[VPT][VEC];
#pragma unroll
    for (int k = 0; k < VPT; k++) {
#pragma unroll
      for (int e = 0; e < VEC; e++) d[k][e] = elem<T, VEC>(x[k], e) - near;
      if (map.whole[k]) {
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          if constexpr (kCentre) s += d[k][e];
          s2 = fmaf(d[k][e], d[k][e], s2);
        }
      } else {
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          const float counted = e >= map.skip[k] ? d[k][e] : 0.0f;
          if constexpr (kCentre) s += counted;
          s2 = fmaf(counted, counted, s2);
        }
      }
    }
    Centre c = {0.0f, 0.0f};
    if constexpr (kCentre) {
      const float2 sums = sum_row(make_float2(s, s2), part2);
      c = centred(near, sums.x, sums.y, n, inv, a.eps);
    } else {
      c.rstd = rsqrtf(sum_row(s2, &part2[0].x) * inv + a.eps);
    }
    if (row < a.rows) {
      T *y = static_cast<T *>(a.y) + row * a.y_stride;
#pragma unroll
      for (int k = 0; k < VPT; k++) {
        if (map.skip[k] == VEC) continue;
        vec_t<P, VEC> wk, bk;
        if constexpr (kKeep) {
          wk = w[k];
          bk = b[k];
        } else {
          load_params(k, wk, bk);
        }
        float out[VEC];
#pragma unroll
        for (int e = 0; e < VEC; e++) out[e] = fmaf((kCentre ? d[k][e] - c.shift : d[k][e]) * c.rstd, elem<P, VEC>(wk, e), elem<P, VEC>(bk, e));
        store_vec_stream<T, VEC>(y + map.col[k], round_vec<T, VEC>(out));
      }
      if (t == 0) {
        if (a.mean) a.mean[row] = kCentre ? near + c.shift : near;
        if (a.rstd) a.rstd[row] = c.rstd;
      }
    }
  }
}

// Rows too long for the registers of a workgroup: the same sums, the row read three times (twice from the caches).
template <class T, class P>
__global__ __launch_bounds__(1024) void layer_norm_long_kernel(hf_layer_norm_args a) {
  constexpr int VEC = kVec<T>;
  __shared__ float part[3][16];
  const int cols = (int)a.cols, tid = (int)threadIdx.x, slots = row_slots<VEC>(cols);
  const float n = (float)cols, inv = 1.0f / n;
  auto leave = [&](float v, int which) {
    v = lanes_sum<64>(v);
    if ((tid & 63) == 0) part[which][tid >> 6] = v;
  };
  auto sum_of = [&](int which) {   // behind a barrier; written again only behind another sum's
    float v = 0.0f;
    for (int i = 0; i < 16; i++) v += part[which][i];
    return v;
  };
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    float s = 0.0f;
    for (int j = tid; j < slots; j += 1024) {
      const vec_t<T, VEC> v = load_vec<T, VEC>(x + slot_column<VEC>(j, cols));
      const int skip = slot_repeats<VEC>(j, cols);
#pragma unroll
      for (int e = 0; e < VEC; e++) s += e >= skip ? elem<T, VEC>(v, e) : 0.0f;
    }
    leave(s, 0);
    __syncthreads();
    const float near = quotient(sum_of(0), n, inv);
    s = 0.0f;
    float s2 = 0.0f;
    for (int j = tid; j < slots; j += 1024) {
      const vec_t<T, VEC> v = load_vec<T, VEC>(x + slot_column<VEC>(j, cols));
      const int skip = slot_repeats<VEC>(j, cols);
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        const float d = e >= skip ? elem<T, VEC>(v, e) - near : 0.0f;
        s += d;
        s2 = fmaf(d, d, s2);
      }
    }
    leave(s, 1);
    leave(s2, 2);
    __syncthreads();
    const Centre centre = centred(near, sum_of(1), sum_of(2), n, inv, a.eps);
    T *y = static_cast<T *>(a.y) + row * a.y_stride;
    for (int j = tid; j < slots; j += 1024) {
      const int c = slot_column<VEC>(j, cols);
      const vec_t<T, VEC> v = load_vec<T, VEC>(x + c);
      const vec_t<P, VEC> w = a.weight ? load_vec<P, VEC>(static_cast<const P *>(a.weight) + c) : (vec_t<P, VEC>)(P)1.0f;
      const vec_t<P, VEC> b = a.bias ? load_vec<P, VEC>(static_cast<const P *>(a.bias) + c) : (vec_t<P, VEC>)(P)0.0f;
      float out[VEC];
#pragma unroll
      for (int e = 0; e < VEC; e++) out[e] = fmaf((elem<T, VEC>(v, e) - near - centre.shift) * centre.rstd, elem<P, VEC>(w, e), elem<P, VEC>(b, e));
      store_vec<T, VEC>(y + c, round_vec<T, VEC>(out));
    }
    if (tid == 0) {
      if (a.mean) a.mean[row] = near + centre.shift;
      if (a.rstd) a.rstd[row] = centre.rstd;
    }
  }
}

// Two rows a group of lanes in turn, if every CU has eight workgroups then: the second row is on its way while the first
// is finished, and a workgroup is gone before its reads and writes fall into step with everyone's.  (65536 x 4096 bf16, trips
// 1 / 2 / 3 / 4: 207 / 183 / 183 / 188 us.)  Float32 parameters next to 16-bit rows are as many bytes as two rows, and a
// workgroup of 1024 is alone on half a CU: four (194 -> 187 us at 65536 x 4096, 209 -> 190 us at 16384 x 16384).
template <class T, class P, int VEC, int VPT, int LANES, int BLOCK>
hipError_t norm_rows(const hf_layer_norm_args &a, int lanes, int cus, hipStream_t s) {
  const int groups = std::max(1, 256 / lanes);
  const int64_t sets = (a.rows + groups - 1) / groups;
  const int64_t kTrips = sizeof(P) > sizeof(T) || lanes > 512 ? 4 : 2;
  int64_t trips = std::max<int64_t>(1, std::min(kTrips, sets / (cus * 8)));
  while ((sets + trips - 1) / trips * (groups * lanes) >= (int64_t)1 << 32) trips *= 2;   // a grid has less than 2^32 threads
  const unsigned grid = (unsigned)((sets + trips - 1) / trips);   // every workgroup makes `trips` trips, or one less
  hipLaunchKernelGGL((layer_norm_rows_kernel<T, P, VEC, VPT, LANES, BLOCK>), dim3(grid), dim3((unsigned)(groups * lanes)), 0, s, a, lanes,
                     past_caches((size_t)a.rows * (size_t)a.cols * sizeof(T)));
  return hipGetLastError();
}

template <class T, class P>
hipError_t norm_forward(const hf_layer_norm_args &a, int cus, hipStream_t s) {
  constexpr int VEC = kVec<T>;
  if (a.cols < VEC) return norm_rows<T, P, 1, 1, 8, 256>(a, 8, cus, s);
  const int64_t slots = (a.cols + VEC - 1) / VEC;
  if (slots <= 8) return norm_rows<T, P, VEC, 1, 8, 256>(a, 8, cus, s);
  if (slots <= 16) return norm_rows<T, P, VEC, 1, 16, 256>(a, 16, cus, s);
  if (slots <= 32) return norm_rows<T, P, VEC, 1, 32, 256>(a, 32, cus, s);
  if (slots <= 64) return norm_rows<T, P, VEC, 1, 64, 256>(a, 64, cus, s);
  const int waves = (int)std::min<int64_t>((slots + 63) / 64, 65);   // wavefronts with one slot a lane
  // Fewer rows than CUs: a row's latency is all there is, and one slot a thread is the shortest (one row of 2048 / 4096 bf16
  // 2.3 / 2.5 us, with two slots 2.8 / 2.8); with more rows it is slower (4096 x 1024: 5.0 us against 4.5).
  if (a.rows <= cus && waves <= 16) return norm_rows<T, P, VEC, 1, 0, 1024>(a, waves * 64, cus, s);
  // Two slots a lane (with four 8192 x 4096 bf16 takes 24.0 instead of 22.8 us, 65536 x 4096 180 instead of 184; with one
  // 22.6 and 192), one or three where that leaves fewer lanes without a slot: their arithmetic costs the same.
  if (waves == 2) return norm_rows<T, P, VEC, 2, 64, 256>(a, 64, cus, s);
  if (waves == 3) return norm_rows<T, P, VEC, 3, 64, 256>(a, 64, cus, s);
  if (waves <= 16 && waves % 2 && waves % 3 == 0) return norm_rows<T, P, VEC, 3, 0, 512>(a, waves / 3 * 64, cus, s);
  if (waves < 8 && waves % 2) return norm_rows<T, P, VEC, 1, 0, 1024>(a, waves * 64, cus, s);
  if (waves <= 16) return norm_rows<T, P, VEC, 2, 0, 512>(a, (waves + 1) / 2 * 64, cus, s);
  if (waves <= 32) return norm_rows<T, P, VEC, 2, 0, 1024>(a, (waves + 1) / 2 * 64, cus, s);
  if (waves <= 48) return norm_rows<T, P, VEC, 3, 0, 1024>(a, (waves + 2) / 3 * 64, cus, s);
  if (waves <= 64) return norm_rows<T, P, VEC, 4, 0, 1024>(a, (waves + 3) / 4 * 64, cus, s);
  const unsigned grid = (unsigned)std::min<int64_t>(a.rows, (int64_t)cus * 2);
  hipLaunchKernelGGL((layer_norm_long_kernel<T, P>), dim3(grid), dim3(1024), 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_layer_norm(const hf_layer_norm_args &a, int cus, hipStream_t s) {
  if (a.rows == 0) return hipSuccess;
  return with_type(a.type, [&](auto t) {
    using T = decltype(t);
    return a.param_type == HF_F32 ? norm_forward<T, float>(a, cus, s) : norm_forward<T, T>(a, cus, s);
  });
}

}  // namespace hfuse
