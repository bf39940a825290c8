// Token embedding, out[i] = scale W[t_i], and the gradient of the table, dW[v] = scale sum of dy[i] over i with t_i = v.
//
// Both are bound by HBM.  Measured on an MI355X with 131072 tokens and a table of 128000 x 4096 bf16, ids of a learnt
// vocabulary (the k-th with a probability of about 1 / k): lookup 264 us (1.07 GB written, 0.67 GB fetched for 0.27 GB of
// distinct rows: 6.6 TB/s; 279 us a launch under the profiler); gradient, with the first id as padding, 370 us on the GPU and
// 406 a call in a row of them for 2.06 GB = 5.1-5.6 TB/s: the sort and the rows of zeros beside it 134, the sums 225, the
// shared tokens 11.
#include <algorithm>

#include "device/rows.h"
#include "launch.h"

namespace hfuse {
namespace {

// A group of `lanes` lanes copies U of its slots of a row at once: all its reads are on their way before the first store.
// (U 1 / 2 / 4 / 8: 337 / 276 / 270 / 301 us for the batch above, 4.6 / 4.8 / 5.4 / 7.4 us for 4999 rows of 1001 f16.)
// Stores go past the caches, which keep the table's frequent rows (rows of 128 bf16: 87 -> 51 us for a million tokens).
template <class T, class I, int VEC, int U>
__global__ __launch_bounds__(256) void embedding_kernel(hf_embedding_args a, int lanes_log2, unsigned tiles) {
  const unsigned lanes = 1u << lanes_log2, lane = threadIdx.x & (lanes - 1);
  const int cols = (int)a.cols, slots = row_slots<VEC>(cols);
  const unsigned long long groups = (unsigned long long)a.ntokens * tiles, step = ((unsigned long long)gridDim.x * 256u) >> lanes_log2;
  for (unsigned long long group = ((unsigned long long)blockIdx.x * 256u + threadIdx.x) >> lanes_log2; group < groups; group += step) {
    const int64_t i = (int64_t)(group / tiles);
    const int first = (int)(group % tiles) * U * (int)lanes + (int)lane;
    const int64_t t = (int64_t) static_cast<const I *>(a.tokens)[i];
    const bool used = t >= 0 && t < a.vocab;
    const T *w = static_cast<const T *>(a.weight) + (used ? t : 0) * a.weight_stride;
    T *out = static_cast<T *>(a.out) + i * a.out_stride;
    int col[U];
    vec_t<T, VEC> v[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      col[u] = slot_column<VEC>(min(first + u * (int)lanes, slots - 1), cols);   // (lanes behind the row repeat its last slot)
      v[u] = used ? load_vec<T, VEC>(w + col[u]) : (vec_t<T, VEC>)(T)0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (a.scale != 1.0f) {   // (1: the table's bits)
        float f[VEC];
#pragma unroll
        for (int e = 0; e < VEC; e++) f[e] = elem<T, VEC>(v[u], e) * a.scale;
        v[u] = round_vec<T, VEC>(f);
      }
      if (first + u * (int)lanes < slots) store_vec_stream<T, VEC>(out + col[u], v[u]);
    }
  }
}

// ------------------------------------------------------------------ the gradient of the table
// Few tokens take few_tokens_kernel, below.  Else the usable tokens are sorted with their positions by a stable radix sort (count_digits_kernel and place_digits_kernel
// for each digit), the dy rows of each token are summed from the sorted list (sum_rows_kernel), and tokens whose rows were
// shared out are joined (join_rows_kernel).  The rows of zeros -- most of the table in a small batch -- are written by
// further workgroups of the sort's launches: a sort of some thousand tokens waits for memory most of the time on a few
// CUs and leaves the rest of the part and its write bandwidth to them.  dy is read and the zeros are written past the
// caches: otherwise the reads push the dirty zeros out of the memory-side cache and wait for them (sums 301 -> 224 us).
// No floating-point atomics: every sum has one order, whatever the order in which workgroups run.

constexpr int kSortWaves = 4;
constexpr int kSortThreads = 64 * kSortWaves;
constexpr int kSortKeys = 4;                              // tokens a thread has in one step
constexpr int kSortStep = kSortThreads * kSortKeys;
constexpr int kMaxDigitBits = 9;
constexpr int kMaxBuckets = 1 << kMaxDigitBits;
constexpr int kSortTiles = 128;                           // workgroups of a sort launch at most

// What the launches hand on, in the caller's workspace.
struct TableScratch {
  uint2 *order, *other;     // {position, token} sorted by token, positions ascending; the list before the last digit
  unsigned *counts;         // [tile][bucket] of the digit in hand
  unsigned *owner;          // owner[v] = a position that names token v, if any does; anything otherwise
  unsigned *last;           // per shared token: the last chunk with a row of it
  unsigned *state;          // [0] usable tokens, [1] shared tokens
  unsigned *shared;         // the shared tokens, each by the chunk it starts in
  float *partial;           // two rows of sums a chunk: of the token it begins inside of, and of the token it ends inside of
  unsigned tile, tiles;     // positions of a sort workgroup (a multiple of kSortStep), sort workgroups
  unsigned chunk, nchunks;  // entries summed by one group of lanes
};

// Rows [row, row + rows) of the gradient, 2^lanes_log2 lanes each: those that no token names become zeros.
struct ZeroRows {
  unsigned row, rows;
  int lanes_log2;
  unsigned element;   // bytes of an element
};

__device__ __forceinline__ void zero_row(const hf_embedding_backward_args &a, const ZeroRows &z, size_t v, unsigned lane) {
  const unsigned lanes = 1u << z.lanes_log2, bytes = (unsigned)a.cols * z.element;
  unsigned char *row = static_cast<unsigned char *>(a.dweight) + v * (size_t)a.dweight_stride * z.element;
  typedef unsigned short word_t;   // rows are aligned to an element, of two bytes or more
  if (bytes >= 16) {
    for (unsigned j = lane * 16u; j < bytes; j += lanes * 16u)
      store_vec_stream<word_t, 8>(reinterpret_cast<word_t *>(row + min(j, bytes - 16u)), (vec_t<word_t, 8>)(word_t)0);
  } else {
    for (unsigned j = lane * 2u; j < bytes; j += lanes * 2u) *reinterpret_cast<word_t *>(row + j) = 0;
  }
}

template <class I>
__device__ __forceinline__ void write_zero_rows(const hf_embedding_backward_args &a, const unsigned *owner, const ZeroRows &z, unsigned block) {
  const size_t at = (size_t)block * 256u + threadIdx.x;
  const size_t r = at >> z.lanes_log2;
  if (r >= z.rows) return;
  const size_t v = z.row + r;
  // `owner` was never cleared: what it says is a claim, true if the position it gives names this token
  const unsigned i = owner[v];
  if (i < (unsigned)a.ntokens && (int64_t) static_cast<const I *>(a.tokens)[i] == (int64_t)v && (int64_t)v != a.padding_idx) return;
  zero_row(a, z, v, (unsigned)at & ((1u << z.lanes_log2) - 1u));
}

// Entry i of the list in hand: of the tokens themselves for the first digit ({i, ~0} for one outside the table or equal to
// padding_idx), of the list that the digit before left for the others.
template <class I, bool FIRST>
__device__ __forceinline__ uint2 list_entry(const hf_embedding_backward_args &a, const uint2 *in, unsigned i, unsigned n) {
  if (i >= n) return make_uint2(0, ~0u);
  if constexpr (!FIRST) {
    return in[i];
  } else {
    unsigned lo, hi = 0;
    if constexpr (sizeof(I) == 8) {
      const uint2 t = static_cast<const uint2 *>(a.tokens)[i];
      lo = t.x;
      hi = t.y;
    } else {
      lo = static_cast<const unsigned *>(a.tokens)[i];
    }
    const bool used = hi == 0 && lo < (unsigned)a.vocab && (a.padding_idx < 0 || lo != (unsigned)a.padding_idx);
    return make_uint2(i, used ? lo : ~0u);
  }
}

// Numbers the equal digits of a wave's 64 entries in the order of the lanes, behind the ones the wave has counted before.
// The lanes with the same digit are found with one ballot a bit.
__device__ __forceinline__ unsigned rank_equal(unsigned digit, bool used, int bits, unsigned lane, unsigned *count) {
  unsigned long long same = __ballot(used);
  for (int b = 0; b < bits; b++) {
    const bool one = (digit >> b) & 1u;
    const unsigned long long ones = __ballot(one);
    same &= one ? ones : ~ones;
  }
  unsigned rank = 0;
  if (used) {
    const int leader = __builtin_ctzll(same);
    if ((int)lane == leader) rank = atomicAdd(&count[digit], (unsigned)__builtin_popcountll(same));
    rank = (unsigned)__shfl((int)rank, leader) + (unsigned)__builtin_popcountll(same & ((1ull << lane) - 1ull));
  }
  return rank;
}

// Inclusive sum over the threads of a workgroup in their order, and the sum of all; one barrier.
template <int WAVES>
__device__ __forceinline__ unsigned scan_block(unsigned v, unsigned *part, unsigned &all) {
  const unsigned lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const unsigned u = __shfl_up(v, m);
    if (lane >= (unsigned)m) v += u;
  }
  if (lane == 63) part[wave] = v;
  __syncthreads();
  all = 0;
#pragma unroll
  for (unsigned w = 0; w < WAVES; w++) {
    if (w < wave) v += part[w];
    all += part[w];
  }
  return v;
}

// Workgroups [0, tiles): how often each value of the digit occurs in a tile; the first digit's launch notes an owner of
// every token on the way.  Behind them: rows of zeros (of the other digits' launches).
template <class I, bool FIRST>
__global__ __launch_bounds__(kSortThreads) void count_digits_kernel(hf_embedding_backward_args a, TableScratch sc, const uint2 *in, int shift,
                                                                    int bits, ZeroRows z) {
  __shared__ unsigned count[kMaxBuckets];
  const unsigned tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  if (FIRST && blockIdx.x == 0 && tid == 0) sc.state[1] = 0;
  if (blockIdx.x >= sc.tiles) {
    if constexpr (!FIRST) write_zero_rows<I>(a, sc.owner, z, blockIdx.x - sc.tiles);
    return;
  }
  const unsigned buckets = 1u << bits, n = FIRST ? (unsigned)a.ntokens : sc.state[0];
  for (unsigned b = tid; b < buckets; b += kSortThreads) count[b] = 0;
  __syncthreads();
  const unsigned from = blockIdx.x * sc.tile, to = min(from + sc.tile, n);
  for (unsigned step = from; step < to; step += kSortStep) {
    unsigned key[kSortKeys];
#pragma unroll
    for (int u = 0; u < kSortKeys; u++) key[u] = list_entry<I, FIRST>(a, in, step + (wave * kSortKeys + u) * 64u + lane, to).y;
#pragma unroll
    for (int u = 0; u < kSortKeys; u++) {
      if (FIRST && key[u] != ~0u) sc.owner[key[u]] = step + (wave * kSortKeys + u) * 64u + lane;   // any of them will do
      const unsigned d = (key[u] >> shift) & (buckets - 1);
      const unsigned long long used = __ballot(key[u] != ~0u);
      if (!used) continue;
      const unsigned d0 = (unsigned)__builtin_amdgcn_readlane((int)d, __builtin_ctzll(used));
      if ((__ballot(d == d0) & used) == used) {   // a run of one token: one addition, not 64 to one address
        if (lane == 0) atomicAdd(&count[d0], (unsigned)__builtin_popcountll(used));
      } else if (key[u] != ~0u) {
        atomicAdd(&count[d], 1u);
      }
    }
  }
  __syncthreads();
  for (unsigned b = tid; b < buckets; b += kSortThreads) sc.counts[blockIdx.x * buckets + b] = count[b];
}

// Workgroups [0, tiles): every entry of a tile to its place, behind all entries of smaller digits and all equal ones before
// it.  Where the equal ones of other tiles end is summed from their counts; inside the tile a wave numbers its equal
// entries with ballots, bit by bit of the digit, and the waves follow each other.  Behind them: rows of zeros.
template <class I, bool FIRST>
__global__ __launch_bounds__(kSortThreads) void place_digits_kernel(hf_embedding_backward_args a, TableScratch sc, const uint2 *in, uint2 *out,
                                                                    int shift, int bits, ZeroRows z) {
  __shared__ unsigned count[kSortWaves][kMaxBuckets], base[kMaxBuckets], scan[kSortWaves];
  const unsigned tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  if (blockIdx.x >= sc.tiles) {
    write_zero_rows<I>(a, sc.owner, z, blockIdx.x - sc.tiles);
    return;
  }
  const unsigned buckets = 1u << bits;
  constexpr int kOwn = kMaxBuckets / kSortThreads;   // buckets 2 tid and 2 tid + 1 are this thread's
  unsigned before[kOwn] = {0, 0}, total[kOwn] = {0, 0};
  if (tid * kOwn < buckets) {   // (one bit: two buckets)
    constexpr unsigned kAhead = 8;   // counts on their way at once (the registers of 16 cost the rows of zeros a tenth of their rate)
    for (unsigned t = 0; t < sc.tiles; t += kAhead) {
      uint2 c[kAhead];
#pragma unroll
      for (unsigned i = 0; i < kAhead; i++)
        c[i] = *reinterpret_cast<const uint2 *>(sc.counts + min(t + i, sc.tiles - 1) * buckets + tid * kOwn);
#pragma unroll
      for (unsigned i = 0; i < kAhead; i++) {
        if (t + i < blockIdx.x) {
          before[0] += c[i].x;
          before[1] += c[i].y;
        }
        if (t + i < sc.tiles) {
          total[0] += c[i].x;
          total[1] += c[i].y;
        }
      }
    }
  }
  unsigned all;
  const unsigned upto = scan_block<kSortWaves>(total[0] + total[1], scan, all);
  if (tid * kOwn < buckets) {
    base[tid * kOwn] = upto - total[0] - total[1] + before[0];
    base[tid * kOwn + 1] = upto - total[1] + before[1];
  }
  if (FIRST && blockIdx.x == 0 && tid == 0) sc.state[0] = all;

  const unsigned n = FIRST ? (unsigned)a.ntokens : all;
  const unsigned from = blockIdx.x * sc.tile, to = min(from + sc.tile, n);
  for (unsigned step = from; step < to; step += kSortStep) {
    uint2 entry[kSortKeys];
#pragma unroll
    for (int u = 0; u < kSortKeys; u++) entry[u] = list_entry<I, FIRST>(a, in, step + (wave * kSortKeys + u) * 64u + lane, to);
    for (unsigned b = lane; b < buckets; b += 64) count[wave][b] = 0;   // a wave's counters are its own
    unsigned rank[kSortKeys];
#pragma unroll
    for (int u = 0; u < kSortKeys; u++)
      rank[u] = rank_equal((entry[u].y >> shift) & (buckets - 1), entry[u].y != ~0u, bits, lane, count[wave]);
    __syncthreads();
    for (unsigned b = tid; b < buckets; b += kSortThreads) {   // counts -> first places; the tile's next step follows
      unsigned at = base[b];
#pragma unroll
      for (int w = 0; w < kSortWaves; w++) {
        const unsigned c = count[w][b];
        count[w][b] = at;
        at += c;
      }
      base[b] = at;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kSortKeys; u++)
      if (entry[u].y != ~0u) out[count[wave][(entry[u].y >> shift) & (buckets - 1)] + rank[u]] = entry[u];
    __syncthreads();   // (a faster wave clears its own counters only, but `base` and the places above are everyone's)
  }
}

// As many tokens as a thread each holds kSortKeys of need no list in memory: one launch, and no workspace.  A workgroup has
// `rows` rows of the table over one tile of columns (`lanes` slots), looks through all tokens for them, and finds none most
// of the time: then it writes zeros.  Else it sorts the positions of its own tokens in LDS, and each group of lanes sums a
// row of the table at a time; a token with more than kFewOwn positions is summed by all groups, joined in their order.
// Bound by the stores of the zeros, and by the latency of launch and fetch in small tables.  Against a list sorted by one
// workgroup, three launches in turn: 256 tokens of 32000 x 768 f32 24.9 -> 20.1 us (4.9 TB/s), 1000 of 50000 x 2048 bf16
// 43 -> 34, of 128000 x 8192 383 -> 300 (7.0 TB/s), 1000 x 768 19 -> 12.6.  The worst case, 1024 times one token of 512
// columns, is one CU's to read and takes 18 -> 32.
constexpr unsigned kFewTokens = kSortStep;
constexpr unsigned kFewRows = 256;   // one thread each
constexpr unsigned kFewOwn = 64;
template <class T, class O, class I, int VEC>
__global__ __launch_bounds__(kSortThreads) void few_tokens_kernel(hf_embedding_backward_args a, unsigned rows, int row_bits, int lanes_log2,
                                                                  unsigned tiles) {
  __shared__ unsigned count[kSortWaves][kFewRows], start[kFewRows + 1], scan[kSortWaves];
  __shared__ unsigned short list[kFewTokens];
  __shared__ float sums[kSortWaves][64 * VEC];
  const unsigned tid = threadIdx.x, wave = tid >> 6;
  const unsigned tile = blockIdx.x % tiles, first = blockIdx.x / tiles * rows, mine = min(rows, (unsigned)a.vocab - first);
  unsigned r[kSortKeys];
  bool any = false;
#pragma unroll
  for (int u = 0; u < kSortKeys; u++) {
    const unsigned key = list_entry<I, true>(a, nullptr, (wave * kSortKeys + u) * 64u + (tid & 63u), (unsigned)a.ntokens).y;
    r[u] = key - first;   // (an unusable key is at least 2^31 off)
    any |= r[u] < mine;
  }
  const bool present = __syncthreads_or(any);
  if (present) {
    for (unsigned b = tid & 63u; b < rows; b += 64) count[wave][b] = 0;   // a wave's counters are its own
    unsigned rank[kSortKeys];
#pragma unroll
    for (int u = 0; u < kSortKeys; u++) rank[u] = rank_equal(r[u] & (kFewRows - 1), r[u] < mine, row_bits, tid & 63u, count[wave]);
    __syncthreads();
    unsigned total = 0, all;
    if (tid < rows)
      for (int w = 0; w < kSortWaves; w++) total += count[w][tid];
    unsigned at = scan_block<kSortWaves>(total, scan, all) - total;
    if (tid < rows) {
      start[tid] = at;
      if (tid == rows - 1) start[rows] = all;
      for (int w = 0; w < kSortWaves; w++) {
        const unsigned c = count[w][tid];
        count[w][tid] = at;
        at += c;
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kSortKeys; u++)
      if (r[u] < mine) list[count[wave][r[u]] + rank[u]] = (unsigned short)((wave * kSortKeys + u) * 64u + (tid & 63u));
    __syncthreads();
  }

  const int lanes = 1 << lanes_log2, lane = (int)tid & (lanes - 1), cols = (int)a.cols, slots = row_slots<VEC>(cols);
  const unsigned group = tid >> lanes_log2, groups = kSortThreads >> lanes_log2;
  const int slot = (int)tile * lanes + lane, col = slot_column<VEC>(min(slot, slots - 1), cols);
  const T *dy = static_cast<const T *>(a.dy) + col;
  O *out = static_cast<O *>(a.dweight) + (size_t)first * (size_t)a.dweight_stride + col;
  float acc[VEC];
  auto sum = [&](unsigned from, unsigned to, unsigned step) {   // of every step-th position of the list
    constexpr int U = 8;
#pragma unroll
    for (int e = 0; e < VEC; e++) acc[e] = 0.0f;
    for (unsigned k = from; k < to; k += U * step) {
      vec_t<T, VEC> row[U];
#pragma unroll
      for (int u = 0; u < U; u++) row[u] = load_vec<T, VEC>(dy + (size_t)list[min(k + u * step, to - 1)] * (size_t)a.dy_stride);
#pragma unroll
      for (int u = 0; u < U; u++)
        if (k + u * step < to)
#pragma unroll
          for (int e = 0; e < VEC; e++) acc[e] += elem<T, VEC>(row[u], e);
    }
  };
  auto put = [&](unsigned b) {
    float v[VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) v[e] = acc[e] * a.scale;
    store_vec_stream<O, VEC>(out + (size_t)b * (size_t)a.dweight_stride, round_vec<O, VEC>(v));
  };
  if (!present) {
    if (slot < slots)
      for (unsigned b = group; b < mine; b += groups) store_vec_stream<O, VEC>(out + (size_t)b * (size_t)a.dweight_stride, (vec_t<O, VEC>)(O)0.0f);
    return;
  }
  for (unsigned b = group; b < mine; b += groups) {
    if (start[b + 1] - start[b] > kFewOwn) continue;
    sum(start[b], start[b + 1], 1);
    if (slot < slots) put(b);
  }
  for (unsigned b = 0; b < mine; b++) {
    if (start[b + 1] - start[b] <= kFewOwn) continue;
    sum(start[b] + group, start[b + 1], groups);
    for (int m = lanes; m < 64; m <<= 1)   // the groups of a wave
#pragma unroll
      for (int e = 0; e < VEC; e++) acc[e] += __shfl_xor(acc[e], m);
#pragma unroll
    for (int e = 0; e < VEC; e++) sums[wave][e * 64 + (int)(tid & 63u)] = acc[e];
    __syncthreads();
    if (group == 0 && slot < slots) {
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        acc[e] = sums[0][e * 64 + lane];
        for (int w = 1; w < kSortWaves; w++) acc[e] += sums[w][e * 64 + lane];
      }
      put(b);
    }
    __syncthreads();   // the sums are reused by the next row
  }
}

// Some more tokens (kSortFewTokens at most) next to a small table, one launch: workgroup 0 sorts them in its LDS, digit by
// digit; the others have `rows` rows of the table each, look through the tokens themselves and write the rows of zeros.
constexpr int kSortFewWaves = 8, kSortFewKeys = 8;   // keys: of a thread
constexpr int64_t kSortFewTokens = 64 * kSortFewWaves * kSortFewKeys, kSortFewBytes = 65536;   // bytes: of the table to a workgroup
template <class I>
__global__ __launch_bounds__(64 * kSortFewWaves) void sort_few_kernel(hf_embedding_backward_args a, TableScratch sc, int passes, int bits,
                                                                      unsigned rows, ZeroRows z) {
  constexpr int WAVES = kSortFewWaves, KEYS = kSortFewKeys;
  constexpr unsigned kThreads = 64 * WAVES;
  constexpr int kOwn = (kMaxBuckets + kThreads - 1) / kThreads;   // buckets of a thread
  __shared__ uint2 list[kThreads * KEYS];
  __shared__ unsigned count[WAVES][kMaxBuckets], scan[WAVES];
  const unsigned tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  uint2 entry[KEYS];
#pragma unroll
  for (int u = 0; u < KEYS; u++) entry[u] = list_entry<I, true>(a, nullptr, (wave * KEYS + u) * 64u + lane, (unsigned)a.ntokens);
  if (blockIdx.x > 0) {
    unsigned *present = count[0];   // a flag a row, kThreads of them at most
    const size_t first = (size_t)(blockIdx.x - 1) * rows;
    const unsigned mine = (unsigned)min((size_t)rows, (size_t)a.vocab - first);
    present[tid] = 0;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < KEYS; u++) {
      const size_t r = (size_t)entry[u].y - first;
      if (entry[u].y != ~0u && r < mine) present[r] = 1;
    }
    __syncthreads();
    for (unsigned r = tid >> z.lanes_log2; r < mine; r += kThreads >> z.lanes_log2)
      if (!present[r]) zero_row(a, z, first + r, tid & ((1u << z.lanes_log2) - 1u));
    return;
  }
  const unsigned buckets = 1u << bits;
  unsigned used = 0;
  for (int pass = 0; pass < passes; pass++) {
    const int shift = pass * bits;
    for (unsigned b = lane; b < buckets; b += 64) count[wave][b] = 0;   // a wave's counters are its own
    unsigned rank[KEYS];
#pragma unroll
    for (int u = 0; u < KEYS; u++)
      rank[u] = rank_equal((entry[u].y >> shift) & (buckets - 1), entry[u].y != ~0u, bits, lane, count[wave]);
    __syncthreads();
    unsigned total = 0;
    for (unsigned b = tid * kOwn; b < min((tid + 1) * kOwn, buckets); b++)
      for (int w = 0; w < WAVES; w++) total += count[w][b];
    unsigned at = scan_block<WAVES>(total, scan, used) - total;
    for (unsigned b = tid * kOwn; b < min((tid + 1) * kOwn, buckets); b++)
      for (int w = 0; w < WAVES; w++) {
        const unsigned c = count[w][b];
        count[w][b] = at;
        at += c;
      }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < KEYS; u++)
      if (entry[u].y != ~0u) list[count[wave][(entry[u].y >> shift) & (buckets - 1)] + rank[u]] = entry[u];
    __syncthreads();
#pragma unroll
    for (int u = 0; u < KEYS; u++) {
      const unsigned i = (wave * KEYS + u) * 64u + lane;
      entry[u] = i < used ? list[i] : make_uint2(0, ~0u);
    }
    __syncthreads();   // the list and the counters are written again
  }
#pragma unroll
  for (int u = 0; u < KEYS; u++)
    if (entry[u].y != ~0u) sc.order[(wave * KEYS + u) * 64u + lane] = entry[u];
  if (tid == 0) {
    sc.state[0] = used;
    sc.state[1] = 0;
  }
}

// First entry of [lo, hi) whose token is larger than `id` (hi if there is none); the list is sorted.  The ones up to `id`
// are counted, 64 at a time by a whole wave and 8 by a thread: a chunk's worth takes one wait for memory or a few.
template <bool WIDE>
__device__ __forceinline__ unsigned first_above(const uint2 *order, unsigned lo, unsigned hi, unsigned id) {
  while (lo < hi) {
    unsigned n = 0;
    if constexpr (WIDE) {
      const unsigned at = lo + (threadIdx.x & 63u);
      n = (unsigned)__builtin_popcountll(__ballot(at < hi && order[min(at, hi - 1)].y <= id));
    } else {
#pragma unroll
      for (unsigned i = 0; i < 8; i++) n += lo + i < hi && order[min(lo + i, hi - 1)].y <= id;
    }
    lo += n;
    if (n < (WIDE ? 64 : 8)) break;
  }
  return lo;
}

// A group of `lanes` lanes sums the rows of one chunk of `order` over one tile of columns (`lanes` slots).  A token whose rows
// cross one chunk boundary at most belongs to the chunk it starts in, which follows it to its end; a token that crosses
// more is shared: every chunk sums its own part of it.
template <class T, class O, int VEC, bool WIDE>
__global__ __launch_bounds__(256) void sum_rows_kernel(hf_embedding_backward_args a, TableScratch sc, int lanes_log2, unsigned tiles) {
  const int lanes = WIDE ? 64 : 1 << lanes_log2;
  const unsigned global = blockIdx.x * 256u + threadIdx.x;
  const unsigned group = WIDE ? (unsigned)__builtin_amdgcn_readfirstlane((int)(global >> 6)) : global >> lanes_log2;
  const int lane = (int)(threadIdx.x & (unsigned)(lanes - 1));
  const unsigned c = group / tiles;
  const int tile = (int)(group % tiles);
  const unsigned used = sc.state[0], k0 = c * sc.chunk;
  if (c >= sc.nchunks || k0 >= used) return;
  const uint2 *order = sc.order;
  const unsigned k1 = min(k0 + sc.chunk, used);
  const unsigned id0 = order[k0].y, idl = order[k1 - 1].y;
  const bool cont0 = k0 > 0 && order[k0 - 1].y == id0;                       // started in a chunk before
  const bool crosses = k1 < used && order[k1].y == idl;                      // goes on in the chunk behind
  const bool starts = !(cont0 && idl == id0);
  const bool shared0 = cont0 && ((crosses && idl == id0) || (k0 > sc.chunk && order[k0 - sc.chunk - 1].y == id0));
  const bool sharedl = starts && crosses && k1 + sc.chunk < used && order[k1 + sc.chunk].y == idl;
  const unsigned begin = cont0 && !shared0 ? first_above<WIDE>(order, k0, k1, id0) : k0;   // the rest of that token is the other chunk's
  const unsigned end = starts && crosses && !sharedl ? first_above<WIDE>(order, k1, min(k1 + sc.chunk, used), idl) : k1;
  if (tile == 0 && lane == 0) {
    if (sharedl) sc.shared[atomicAdd(&sc.state[1], 1u)] = c;   // in any order: each is joined by itself
    if (shared0 && !(crosses && idl == id0)) sc.last[id0] = c;
  }

  const int cols = (int)a.cols, slots = row_slots<VEC>(cols);
  const int slot = tile * lanes + lane, col = slot_column<VEC>(min(slot, slots - 1), cols);   // (lanes behind the row store nothing)
  const T *dy = static_cast<const T *>(a.dy) + col;
  float acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; e++) acc[e] = 0.0f;

  // the sum of a token's rows of this chunk: to its row of the gradient, or to the parts of a shared token
  auto put = [&](unsigned id) {
    const bool part0 = shared0 && id == id0, partl = sharedl && id == idl;
    if (slot < slots) {
      if (part0 || partl) {
        store_vec<float, VEC>(sc.partial + (((size_t)c * 2 + (part0 ? 0 : 1)) * (size_t)slots + (size_t)slot) * VEC, round_vec<float, VEC>(acc));
      } else {
        float s[VEC];
#pragma unroll
        for (int e = 0; e < VEC; e++) s[e] = acc[e] * a.scale;
        store_vec<O, VEC>(static_cast<O *>(a.dweight) + (size_t)id * (size_t)a.dweight_stride + col, round_vec<O, VEC>(s));
      }
    }
#pragma unroll
    for (int e = 0; e < VEC; e++) acc[e] = 0.0f;
  };
  auto add = [&](const vec_t<T, VEC> &row) {
#pragma unroll
    for (int e = 0; e < VEC; e++) acc[e] += elem<T, VEC>(row, e);
  };
  // As many entries as the group has lanes at a time, one in each: a row's address is one v_readlane (a whole wave) or one
  // shuffle away, and the tokens' last rows are the bits of one ballot.  The next U rows are on their way while U are added
  // (narrow rows, 4 / 8: 131072 tokens of 128 bf16 columns 75 / 71 us; wide ones: the same).
  constexpr int U = WIDE ? 4 : 8;
  const int group_base = WIDE ? 0 : (int)(threadIdx.x & 63u) & ~(lanes - 1);
  for (unsigned base = begin; base < end; base += (unsigned)lanes) {
    const int m = (int)min((unsigned)lanes, end - base);
    const uint2 mine = order[min(base + (unsigned)lane, end - 1)];
    const unsigned behind = order[min(base + (unsigned)lane + 1, end - 1)].y;
    const unsigned long long lasts = __ballot(behind != mine.y || base + (unsigned)lane + 1 >= end) >> group_base;
    auto of_lane = [&](unsigned v, int i) {
      return WIDE ? (unsigned)__builtin_amdgcn_readlane((int)v, i) : (unsigned)__shfl((int)v, group_base + i);
    };
    auto fetch = [&](vec_t<T, VEC> (&row)[U], int at) {
#pragma unroll
      for (int u = 0; u < U; u++) row[u] = load_vec_stream<T, VEC>(dy + (size_t)of_lane(mine.x, min(at + u, m - 1)) * (size_t)a.dy_stride);
    };
    auto take = [&](const vec_t<T, VEC> (&row)[U], int at) {
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (at + u < m) {
          add(row[u]);
          if ((lasts >> (at + u)) & 1ull) put(of_lane(mine.y, at + u));
        }
      }
    };
    vec_t<T, VEC> one[U], two[U];
    fetch(one, 0);
    for (int at = 0; at < m; at += 2 * U) {
      fetch(two, at + U);
      take(one, at);
      if (at + 2 * U < m) fetch(one, at + 2 * U);
      take(two, at + U);
    }
  }
}

// The shared tokens: a workgroup adds up the parts of one token over one tile of slots.  Its groups of lanes (one a wave
// where rows are wide) take the parts in turn and their sums are added in the order of the groups.
template <class O, int VEC, int WAVES, bool WIDE>
__global__ __launch_bounds__(64 * WAVES) void join_rows_kernel(hf_embedding_backward_args a, TableScratch sc, int lanes_log2, unsigned tiles) {
  __shared__ float sums[WAVES][64 * VEC];
  const int lanes = WIDE ? 64 : 1 << lanes_log2, lane = (int)threadIdx.x & (lanes - 1);
  const unsigned group = WIDE ? threadIdx.x >> 6 : threadIdx.x >> lanes_log2, groups = WIDE ? WAVES : (64u * WAVES) >> lanes_log2;
  const int cols = (int)a.cols, slots = row_slots<VEC>(cols);
  const unsigned long long items = (unsigned long long)sc.state[1] * tiles;
  for (unsigned long long item = blockIdx.x; item < items; item += gridDim.x) {
    const unsigned c = sc.shared[item / tiles];
    const int slot = (int)(item % tiles) * lanes + lane;
    const unsigned id = sc.order[(c + 1) * sc.chunk - 1].y;   // (a shared token fills the chunk behind: this one is full)
    const unsigned last = sc.last[id];
    const size_t width = (size_t)slots * VEC;
    const float *p = sc.partial + (size_t)min(slot, slots - 1) * VEC;
    float acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) acc[e] = 0.0f;
#pragma unroll 8
    for (unsigned q = c + group; q <= last; q += groups) {
      const vec_t<float, VEC> v = load_vec<float, VEC>(p + ((size_t)q * 2 + (q == c ? 1 : 0)) * width);
#pragma unroll
      for (int e = 0; e < VEC; e++) acc[e] += elem<float, VEC>(v, e);
    }
    if constexpr (!WIDE)   // the groups of a wave
      for (int m = lanes; m < 64; m <<= 1)
#pragma unroll
        for (int e = 0; e < VEC; e++) acc[e] += __shfl_xor(acc[e], m);
#pragma unroll
    for (int e = 0; e < VEC; e++) sums[threadIdx.x >> 6][e * 64 + ((int)threadIdx.x & 63)] = acc[e];
    __syncthreads();
    if (group == 0 && slot < slots) {
      float s[VEC];
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        s[e] = 0.0f;
        for (int w = 0; w < WAVES; w++) s[e] += sums[w][e * 64 + lane];
        s[e] *= a.scale;
      }
      store_vec<O, VEC>(static_cast<O *>(a.dweight) + (size_t)id * (size_t)a.dweight_stride + slot_column<VEC>(slot, cols), round_vec<O, VEC>(s));
    }
    __syncthreads();   // the sums are reused by the next item
  }
}

// Entries of a chunk at most, and the waves a CU should have at least before chunks are made smaller for more of them: a
// small chunk shares more tokens out, which costs narrow rows more than the waves bring.
constexpr int kMaxChunk = 64, kWideWaves = 16, kNarrowWaves = 4;

// How the launches are cut: columns into slots and tiles, sorted entries into chunks, the token's bits into digits.
struct TablePlan {
  int vec, lanes_log2, slots, passes, digit_bits, zero_log2;
  unsigned col_tiles, chunk, nchunks, tile, tiles;
  size_t owner_at, last_at, shared_at, counts_at, order_at, other_at, partial_at, bytes;   // the state is at the front
};

TablePlan plan_table(const hf_embedding_backward_args &a, int cus) {
  TablePlan p = {};
  const int vec = a.type == HF_F32 ? kVec<float> : kVec<bf16_t>;
  p.vec = a.cols >= vec ? vec : 1;
  p.slots = (int)((a.cols + p.vec - 1) / p.vec);
  p.lanes_log2 = 6;
  while (p.lanes_log2 > 3 && (1 << (p.lanes_log2 - 1)) >= p.slots) p.lanes_log2--;   // (eight lanes at least: they hold the entries)
  const int lanes = 1 << p.lanes_log2;
  p.col_tiles = (unsigned)((p.slots + lanes - 1) / lanes);
  if (a.ntokens <= kFewTokens) return p;   // few_tokens_kernel: no list, no workspace
  p.chunk = kMaxChunk;
  while (p.chunk > 8 && a.ntokens / p.chunk * p.col_tiles * lanes < (int64_t)cus * (lanes == 64 ? kWideWaves : kNarrowWaves) * 64) p.chunk /= 2;
  while (a.ntokens / p.chunk * p.col_tiles * lanes >= (int64_t)1 << 31) p.chunk *= 2;   // lanes are numbered in 32 bits
  p.nchunks = (unsigned)((a.ntokens + p.chunk - 1) / p.chunk);
  int bits = 1;
  while (((int64_t)1 << bits) < a.vocab) bits++;
  p.passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
  p.digit_bits = (bits + p.passes - 1) / p.passes;
  const int64_t steps = (a.ntokens + kSortStep - 1) / kSortStep;
  p.tile = (unsigned)((steps + kSortTiles - 1) / kSortTiles * kSortStep);
  p.tiles = (unsigned)((a.ntokens + p.tile - 1) / p.tile);
  const int64_t row_bytes = a.cols * (a.out_type == HF_F32 ? 4 : 2);
  p.zero_log2 = 0;   // lanes to a row of zeros: as many as it has 16-byte stores
  while (((int64_t)16 << p.zero_log2) < row_bytes) p.zero_log2++;
  while (p.zero_log2 > 0 && (a.vocab << p.zero_log2) >= (int64_t)1 << 31) p.zero_log2--;   // lanes are numbered in 32 bits
  size_t at = 16;
  auto take = [&at](size_t bytes) {
    const size_t here = at;
    at = (at + bytes + 15) & ~(size_t)15;
    return here;
  };
  p.owner_at = take((size_t)a.vocab * sizeof(unsigned));
  p.last_at = take((size_t)a.vocab * sizeof(unsigned));
  p.shared_at = take((size_t)p.nchunks * sizeof(unsigned));
  p.counts_at = take(((size_t)p.tiles << p.digit_bits) * sizeof(unsigned));
  p.order_at = take((size_t)a.ntokens * sizeof(uint2));
  p.other_at = take(p.passes > 1 ? (size_t)a.ntokens * sizeof(uint2) : 0);
  p.partial_at = take((size_t)p.nchunks * 2 * (size_t)p.slots * (size_t)p.vec * sizeof(float));
  p.bytes = at;
  return p;
}

template <class T, class O, int VEC>
hipError_t sum_tokens(const hf_embedding_backward_args &a, const TablePlan &p, const TableScratch &sc, int cus, hipStream_t s) {
  const unsigned long long sums = ((((unsigned long long)p.nchunks * p.col_tiles) << p.lanes_log2) + 255) / 256;
  const dim3 grid((unsigned)sums);
  const unsigned long long items = (unsigned long long)p.nchunks * p.col_tiles;   // of the join, at most
  if constexpr (VEC > 1) {   // (rows of less than a slot are 8 lanes wide)
    if (p.lanes_log2 == 6) {
      hipLaunchKernelGGL((sum_rows_kernel<T, O, VEC, true>), grid, dim3(256), 0, s, a, sc, 6, p.col_tiles);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
      hipLaunchKernelGGL((join_rows_kernel<O, VEC, 16, true>), dim3((unsigned)std::min<unsigned long long>(items, (unsigned long long)cus * 4)), dim3(1024),
                         0, s, a, sc, 6, p.col_tiles);
      return hipGetLastError();
    }
  }
  hipLaunchKernelGGL((sum_rows_kernel<T, O, VEC, false>), grid, dim3(256), 0, s, a, sc, p.lanes_log2, p.col_tiles);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((join_rows_kernel<O, VEC, 4, false>), dim3((unsigned)std::min<unsigned long long>(items, (unsigned long long)cus * 16)), dim3(256),
                     0, s, a, sc, p.lanes_log2, p.col_tiles);
  return hipGetLastError();
}

template <class I>
hipError_t sort_few(const hf_embedding_backward_args &a, const TablePlan &p, const TableScratch &sc, const ZeroRows &all, hipStream_t s) {
  constexpr int64_t kThreads = 64 * kSortFewWaves;
  int64_t rows = std::max<int64_t>(1, std::min<int64_t>(kThreads, kSortFewBytes / (a.cols * (int64_t)all.element)));
  while (rows < kThreads && a.vocab / rows * kThreads >= (int64_t)1 << 31) rows = std::min(rows * 2, kThreads);   // a grid has less than 2^32 threads
  ZeroRows z = all;
  while (((int64_t)1 << z.lanes_log2) > kThreads) z.lanes_log2--;   // a workgroup's rows are its own
  const unsigned blocks = (unsigned)((a.vocab + rows - 1) / rows);
  hipLaunchKernelGGL((sort_few_kernel<I>), dim3(1 + blocks), dim3(kThreads), 0, s, a, sc, p.passes, p.digit_bits, (unsigned)rows, z);
  return hipGetLastError();
}

template <class I>
hipError_t sort_tokens(const hf_embedding_backward_args &a, const TablePlan &p, const TableScratch &sc, const ZeroRows &all, hipStream_t s) {
  // One launch instead of two a digit: 24 against 30 us for 4096 tokens of a 2000 x 768 float32 table.  One workgroup's sort
  // of 4096 tokens (11 us) is only worth it next to a small table (50000 x 2048 bf16: 54 against 52 us).
  if (a.ntokens <= kSortFewTokens && a.vocab * a.cols * (int64_t)all.element <= (int64_t)64 << 20) return sort_few<I>(a, p, sc, all, s);
  // the rows of zeros are shared evenly among the launches behind the first, which finds out what they are
  const unsigned parts = 2u * (unsigned)p.passes - 1u;
  ZeroRows z = {0, 0, all.lanes_log2, all.element};
  unsigned part = 0;
  auto zero_blocks = [&] {
    z.row = (unsigned)((unsigned long long)all.rows * part / parts);
    z.rows = (unsigned)((unsigned long long)all.rows * (part + 1) / parts) - z.row;
    part++;
    return (unsigned)((((unsigned long long)z.rows << z.lanes_log2) + 255) / 256);
  };
  // the lists change places with every digit, so that the last one fills sc.order
  uint2 *in = nullptr, *out = p.passes % 2 ? sc.order : sc.other;
  for (int pass = 0; pass < p.passes; pass++) {
    const int shift = pass * p.digit_bits;
    unsigned blocks = p.tiles;
    if (pass == 0) {
      hipLaunchKernelGGL((count_digits_kernel<I, true>), dim3(blocks), dim3(kSortThreads), 0, s, a, sc, in, shift, p.digit_bits, z);
    } else {
      blocks += zero_blocks();   // (sets z)
      hipLaunchKernelGGL((count_digits_kernel<I, false>), dim3(blocks), dim3(kSortThreads), 0, s, a, sc, in, shift, p.digit_bits, z);
    }
    blocks = p.tiles + zero_blocks();
    if (pass == 0)
      hipLaunchKernelGGL((place_digits_kernel<I, true>), dim3(blocks), dim3(kSortThreads), 0, s, a, sc, in, out, shift, p.digit_bits, z);
    else
      hipLaunchKernelGGL((place_digits_kernel<I, false>), dim3(blocks), dim3(kSortThreads), 0, s, a, sc, in, out, shift, p.digit_bits, z);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    in = out;
    out = out == sc.order ? sc.other : sc.order;
  }
  return hipSuccess;
}

template <class T, class O, int VEC>
hipError_t few_tokens(const hf_embedding_backward_args &a, const TablePlan &p, int cus, hipStream_t s) {
  const int64_t row_bytes = ((int64_t)VEC * sizeof(O)) << p.lanes_log2;   // of a tile
  // 8 KiB of the table to a workgroup (4 / 16 / 32: 52 / 38 / 45 against 34 us for 1000 tokens of 50000 x 2048 bf16); less
  // in a small table, which would leave CUs idle (1000 x 768: 18 -> 12.6 us)
  int64_t rows = std::max<int64_t>(1, std::min<int64_t>(kFewRows, 8192 / row_bytes));
  while (rows > 1 && a.vocab / rows * p.col_tiles < 2 * cus) rows /= 2;
  while (rows < kFewRows && a.vocab / rows * p.col_tiles >= 1 << 23) rows = std::min<int64_t>(rows * 2, kFewRows);   // a grid has less than 2^32 threads
  int bits = 0;
  while ((1 << bits) < rows) bits++;
  const unsigned blocks = (unsigned)((a.vocab + rows - 1) / rows * p.col_tiles);
  if (a.index_type == HF_I64)
    hipLaunchKernelGGL((few_tokens_kernel<T, O, int64_t, VEC>), dim3(blocks), dim3(kSortThreads), 0, s, a, (unsigned)rows, bits, p.lanes_log2, p.col_tiles);
  else
    hipLaunchKernelGGL((few_tokens_kernel<T, O, int32_t, VEC>), dim3(blocks), dim3(kSortThreads), 0, s, a, (unsigned)rows, bits, p.lanes_log2, p.col_tiles);
  return hipGetLastError();
}

template <class T>
hipError_t embed_backward(const hf_embedding_backward_args &a, int cus, hipStream_t s) {
  const TablePlan p = plan_table(a, cus);
  if (a.ntokens <= kFewTokens) {
    if (a.out_type == HF_F32) return p.vec == 1 ? few_tokens<T, float, 1>(a, p, cus, s) : few_tokens<T, float, kVec<T>>(a, p, cus, s);
    return p.vec == 1 ? few_tokens<T, T, 1>(a, p, cus, s) : few_tokens<T, T, kVec<T>>(a, p, cus, s);
  }
  unsigned char *ws = static_cast<unsigned char *>(a.workspace);
  TableScratch sc;
  sc.state = reinterpret_cast<unsigned *>(ws);
  sc.owner = reinterpret_cast<unsigned *>(ws + p.owner_at);
  sc.last = reinterpret_cast<unsigned *>(ws + p.last_at);
  sc.shared = reinterpret_cast<unsigned *>(ws + p.shared_at);
  sc.counts = reinterpret_cast<unsigned *>(ws + p.counts_at);
  sc.order = reinterpret_cast<uint2 *>(ws + p.order_at);
  sc.other = reinterpret_cast<uint2 *>(ws + p.other_at);
  sc.partial = reinterpret_cast<float *>(ws + p.partial_at);
  sc.tile = p.tile;
  sc.tiles = p.tiles;
  sc.chunk = p.chunk;
  sc.nchunks = p.nchunks;
  const ZeroRows all = {0, (unsigned)a.vocab, p.zero_log2, a.out_type == HF_F32 ? 4u : 2u};
  const hipError_t e = a.index_type == HF_I64 ? sort_tokens<int64_t>(a, p, sc, all, s) : sort_tokens<int32_t>(a, p, sc, all, s);
  if (e != hipSuccess) return e;
  if (a.out_type == HF_F32)
    return p.vec == 1 ? sum_tokens<T, float, 1>(a, p, sc, cus, s) : sum_tokens<T, float, kVec<T>>(a, p, sc, cus, s);
  return p.vec == 1 ? sum_tokens<T, T, 1>(a, p, sc, cus, s) : sum_tokens<T, T, kVec<T>>(a, p, sc, cus, s);
}

}  // namespace

size_t embedding_backward_workspace(const hf_embedding_backward_args &a, int cus) { return plan_table(a, cus).bytes; }

namespace {
template <class T, class I, int VEC, int U>
hipError_t look_up(const hf_embedding_args &a, int lanes_log2, hipStream_t s) {
  const int64_t slots = (a.cols + VEC - 1) / VEC, per_tile = (int64_t)U << lanes_log2, tiles = (slots + per_tile - 1) / per_tile;
  const int64_t blocks = std::min<int64_t>((((a.ntokens * tiles) << lanes_log2) + 255) / 256, 1 << 23);   // a grid has less than 2^32 threads
  hipLaunchKernelGGL((embedding_kernel<T, I, VEC, U>), dim3((unsigned)blocks), dim3(256), 0, s, a, lanes_log2, (unsigned)tiles);
  return hipGetLastError();
}

template <class T, class I>
hipError_t embed_forward(const hf_embedding_args &a, int cus, hipStream_t s) {
  constexpr int VEC = kVec<T>;
  const bool narrow = a.cols < VEC;
  const int64_t slots = narrow ? a.cols : (a.cols + VEC - 1) / VEC;
  int lanes_log2 = 6;
  while (lanes_log2 > 0 && (1 << (lanes_log2 - 1)) >= slots) lanes_log2--;
  if (narrow) return look_up<T, I, 1, 1>(a, lanes_log2, s);
  const int64_t waves = (a.ntokens * slots) >> 6;   // with one slot a lane
  if (slots > 64 && waves > (int64_t)cus * 32) return look_up<T, I, VEC, 2>(a, lanes_log2, s);
  return look_up<T, I, VEC, 1>(a, lanes_log2, s);
}
}  // namespace

hipError_t launch_embedding(const hf_embedding_args &a, int cus, hipStream_t s) {
  if (a.ntokens == 0) return hipSuccess;
  return with_type(a.type, [&](auto t) {
    using T = decltype(t);
    return a.index_type == HF_I64 ? embed_forward<T, int64_t>(a, cus, s) : embed_forward<T, int32_t>(a, cus, s);
  });
}

hipError_t launch_embedding_backward(const hf_embedding_backward_args &a, int cus, hipStream_t s) {
  return with_type(a.type, [&](auto t) { return embed_backward<decltype(t)>(a, cus, s); });
}

}  // namespace hfuse
