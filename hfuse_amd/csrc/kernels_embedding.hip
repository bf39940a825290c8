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

// ------------------------------------------------------------------ the gradient of the table
// Three launches.  (1) group_tokens_kernel sorts the positions by token, stably, and writes the rows of zeros.
// (2) sum_rows_kernel sums the dy rows of each token.  (3) join_rows_kernel adds up the tokens whose rows were shared out.
// No floating-point atomics: every sum has one order, whatever the order in which workgroups run.

// What the launches hand on, in the caller's workspace.
struct TableScratch {
  uint2 *order;        // {position, token} sorted by token, positions ascending
  unsigned *starts;    // starts[v]: first entry of token v in `order`; starts[vocab] = number of usable tokens
  unsigned *nlong;     // tokens whose rows more than one chunk sums ...
  unsigned *longs;     // ... each by the chunk it starts in
  float *partial;      // two rows of sums a chunk: of the token it starts inside of, and of the token it ends inside of
  int chunk;           // entries a chunk has
  int nchunks;
};

constexpr int kGroupThreads = 1024;
constexpr int kGroupWaves = kGroupThreads / 64;
constexpr int kMaxRange = 768;             // tokens of a workgroup's range: a thread each, and 48 KiB of counters
constexpr int kHitWords = 64;              // 64-bit words a wave has to remember which of its loads held a token of the range

// A usable token, or ~0 for one outside the table or equal to padding_idx.
template <class I>
__device__ __forceinline__ unsigned token_key(const I *tokens, unsigned i, unsigned n, unsigned vocab, unsigned pad) {
  if (i >= n) return ~0u;
  unsigned lo, hi = 0;
  if constexpr (sizeof(I) == 8) {
    const uint2 t = reinterpret_cast<const uint2 *>(tokens)[i];
    lo = t.x;
    hi = t.y;
  } else {
    lo = (unsigned)tokens[i];
  }
  return (hi == 0 && lo < vocab && lo != pad) ? lo : ~0u;
}

// Each workgroup owns the tokens [first, first + range) and looks through all positions twice: it counts, lays its tokens
// out behind those of the ranges below (which it counted as well), and places their positions.  A wave takes one
// contiguous part of the positions and has counters of its own, so that positions come out in order.  Between the two
// looks it writes zeros to the rows of its tokens that no position names, whose stores drain under the second look.
template <class I>
__global__ __launch_bounds__(kGroupThreads) void group_tokens_kernel(hf_embedding_backward_args a, TableScratch sc, int range,
                                                                     unsigned row_bytes, unsigned out_bytes) {
  extern __shared__ __align__(16) unsigned smem[];   // counters [wave][range], then the hit words
  __shared__ unsigned wave_part[kGroupWaves], below_part[kGroupWaves];
  __shared__ unsigned long long zero_rows[kGroupWaves];
  const I *tokens = static_cast<const I *>(a.tokens);
  const unsigned n = (unsigned)a.ntokens, vocab = (unsigned)a.vocab;
  const unsigned pad = a.padding_idx < 0 ? ~0u : (unsigned)a.padding_idx;
  const unsigned first = blockIdx.x * (unsigned)range, owned = min((unsigned)range, vocab - first);
  const unsigned tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  unsigned *count = smem + wave * (unsigned)range;
  unsigned long long *hits = reinterpret_cast<unsigned long long *>(smem + ((kGroupWaves * (unsigned)range + 1u) & ~1u)) + wave * kHitWords;

  for (unsigned i = lane; i < (unsigned)range; i += 64) count[i] = 0;   // a wave's counters are its own: no barrier

  const unsigned loads = (n + 63u) / 64u, per = (loads + kGroupWaves - 1) / kGroupWaves;
  const unsigned from = min(wave * per, loads), to = min(from + per, loads);
  unsigned below = 0;
  constexpr int U = 8;   // loads in flight
  for (unsigned l = from; l < to; l += U) {
    unsigned key[U];
#pragma unroll
    for (int u = 0; u < U; u++) key[u] = l + u < to ? token_key(tokens, (l + u) * 64u + lane, n, vocab, pad) : ~0u;
    unsigned found = 0;
#pragma unroll
    for (int u = 0; u < U; u++) {
      below += key[u] < first;
      const unsigned t = key[u] - first;
      const unsigned long long mine = __ballot(t < owned);   // (an unusable key is at least 2^31 off)
      if (mine) {
        found |= 1u << u;
        const unsigned t0 = __builtin_amdgcn_readlane(t, __builtin_ctzll(mine));
        const unsigned long long same = __ballot(t == t0) & mine;
        if (same == mine) {                      // one token (a run of padding): one addition, not 64 to one address
          if (lane == 0) atomicAdd(&count[t0], (unsigned)__builtin_popcountll(mine));
        } else if ((mine >> lane) & 1u) {
          atomicAdd(&count[t], 1u);
        }
      }
    }
    const unsigned at = l - from;                // U divides 64: the flags of one trip fall into one word
    if (lane == 0 && at < 64u * kHitWords) {
      const unsigned long long bits = (unsigned long long)found << (at & 63u);
      hits[at >> 6] = (at & 63u) ? hits[at >> 6] | bits : bits;
    }
  }
  below = (unsigned)__builtin_amdgcn_readfirstlane((int)wave_sum_u32(below));
  if (lane == 0) below_part[wave] = below;
  __syncthreads();

  // counts -> first entries: over the waves of one token, then over the tokens
  unsigned total = 0;
  if (tid < owned)
    for (int w = 0; w < kGroupWaves; w++) {
      const unsigned c = smem[w * range + tid];
      smem[w * range + tid] = total;
      total += c;
    }
  const unsigned long long zeros = __ballot(tid < owned && total == 0);
  unsigned upto = total;                         // inclusive sum over the lanes
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const unsigned v = __shfl_up(upto, m);
    if (lane >= (unsigned)m) upto += v;
  }
  if (lane == 63) wave_part[wave] = upto;
  if (lane == 0) zero_rows[wave] = zeros;
  __syncthreads();
  unsigned start = upto - total;
  for (unsigned w = 0; w < kGroupWaves; w++) {
    start += below_part[w];
    if (w < wave) start += wave_part[w];
  }
  if (tid < owned) {
    sc.starts[first + tid] = start;
    if (first + tid == vocab - 1) sc.starts[vocab] = start + total;
    for (int w = 0; w < kGroupWaves; w++) smem[w * range + tid] += start;
  }
  if (blockIdx.x == 0 && tid == 0) *sc.nlong = 0;

  __syncthreads();   // the first entries of all waves' counters

  // rows of zeros, a wave a row
  auto write_zeros = [&] {
    unsigned char *out = static_cast<unsigned char *>(a.dweight);
    for (unsigned r = wave; r < owned; r += kGroupWaves) {
      if (!((zero_rows[r >> 6] >> (r & 63u)) & 1ull)) continue;
      unsigned char *row = out + (size_t)(first + r) * (size_t)a.dweight_stride * out_bytes;
      if (row_bytes >= 16) {
        const unsigned slots = (row_bytes + 15u) / 16u;
        for (unsigned j = lane; j < slots; j += 64) store_vec<unsigned short, 8>(reinterpret_cast<unsigned short *>(row + min(j * 16u, row_bytes - 16u)), (vec_t<unsigned short, 8>)(0));
      } else if (lane * 2u < row_bytes) {
        reinterpret_cast<unsigned short *>(row)[lane] = 0;
      }
    }
  };
  // second look, at the loads that held a token of the range
  auto place = [&] {
    const unsigned bits = 32u - (unsigned)__builtin_clz(max(owned, 2u) - 1u);
    const bool remembered = per <= 64u * kHitWords;
    for (unsigned g = 0; g * 64u < to - from; g++) {
      unsigned long long todo = ~0ull;
      if (remembered) {
        const unsigned long long h = hits[g];
        todo = ((unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(h >> 32)) << 32) | (unsigned)__builtin_amdgcn_readfirstlane((int)h);
      } else if (to - from - g * 64u < 64u) {
        todo = (1ull << (to - from - g * 64u)) - 1ull;
      }
      while (todo) {
        constexpr int B = 4;
        unsigned key[B], pos[B];
  #pragma unroll
        for (int b = 0; b < B; b++) {
          pos[b] = ~0u;
          if (todo) {
            pos[b] = (from + g * 64u + (unsigned)__builtin_ctzll(todo)) * 64u + lane;
            todo &= todo - 1;
          }
          key[b] = pos[b] == ~0u ? ~0u : token_key(tokens, pos[b], n, vocab, pad);
        }
  #pragma unroll
        for (int b = 0; b < B; b++) {
          const unsigned t = key[b] - first;
          const bool in = t < owned;
          unsigned long long same = __ballot(in);
          if (!same) continue;
          for (unsigned bit = 0; bit < bits; bit++) {   // the lanes with my token
            const bool one = (t >> bit) & 1u;
            const unsigned long long ones = __ballot(in && one);
            same &= one ? ones : ~ones;
          }
          if (in) {
            const int leader = __builtin_ctzll(same);
            unsigned at = 0;
            if ((int)lane == leader) at = atomicAdd(&count[t], (unsigned)__builtin_popcountll(same));
            at = (unsigned)__shfl((int)at, leader);
            at += (unsigned)__builtin_popcountll(same & ((1ull << lane) - 1ull));
            sc.order[at] = make_uint2(pos[b], key[b]);
          }
        }
      }
    }
  };
  if (wave & 1u) {   // half the waves store while the others look
    write_zeros();
    place();
  } else {
    place();
    write_zeros();
  }
}

// A group of `lanes` lanes sums the rows of one chunk of `order` over one tile of columns (lanes * VPT slots).  A token
// with at most `chunk` rows belongs to the chunk it starts in, which follows it to its end; a token with more is shared:
// every chunk sums its own part of it.
template <class T, class O, int VEC, int VPT, bool WIDE>
__global__ __launch_bounds__(256) void sum_rows_kernel(hf_embedding_backward_args a, TableScratch sc, int lanes_log2, int tiles) {
  const int lanes = WIDE ? 64 : 1 << lanes_log2;
  const unsigned global = blockIdx.x * 256u + threadIdx.x;
  unsigned group = WIDE ? (unsigned)__builtin_amdgcn_readfirstlane((int)(global >> 6)) : global >> lanes_log2;
  const int lane = (int)(threadIdx.x & (unsigned)(lanes - 1));
  const int c = (int)(group / (unsigned)tiles), tile = (int)(group % (unsigned)tiles);
  const unsigned used = sc.starts[a.vocab];
  const unsigned k0 = (unsigned)c * (unsigned)sc.chunk;
  if (c >= sc.nchunks || k0 >= used) return;
  const unsigned k1 = min(k0 + (unsigned)sc.chunk, used);
  const unsigned id0 = sc.order[k0].y, idl = sc.order[k1 - 1].y;
  const unsigned s0 = sc.starts[id0], e0 = sc.starts[id0 + 1], sl = sc.starts[idl], el = sc.starts[idl + 1];
  const bool long0 = e0 - s0 > (unsigned)sc.chunk && s0 < k0;    // continues a shared token
  const bool longl = el - sl > (unsigned)sc.chunk && sl >= k0;   // a shared token starts here
  const unsigned begin = (s0 < k0 && !long0) ? e0 : k0;          // the end of an earlier chunk's token is that chunk's
  const unsigned end = (el - sl > (unsigned)sc.chunk) ? k1 : (sl >= k0 ? el : min(el, k1));
  if (longl && tile == 0 && lane == 0) sc.longs[atomicAdd(sc.nlong, 1u)] = (unsigned)c;   // in any order: each is joined by itself

  const int cols = (int)a.cols, slots = row_slots<VEC>(cols);
  int col[VPT], slot[VPT];
#pragma unroll
  for (int v = 0; v < VPT; v++) {
    slot[v] = (tile * VPT + v) * lanes + lane;
    col[v] = slot_column<VEC>(min(slot[v], slots - 1), cols);   // lanes behind the row repeat its last slot and store nothing
  }
  const T *dy = static_cast<const T *>(a.dy);
  float acc[VPT][VEC];
#pragma unroll
  for (int v = 0; v < VPT; v++)
#pragma unroll
    for (int e = 0; e < VEC; e++) acc[v][e] = 0.0f;

  constexpr int U = 4;
  for (unsigned k = begin; k < end; k += U) {
    uint2 entry[U];
    unsigned next;
#pragma unroll
    for (int u = 0; u < U; u++) entry[u] = sc.order[min(k + u, end - 1)];
    next = sc.order[min(k + U, end - 1)].y;
    vec_t<T, VEC> row[U][VPT];
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int v = 0; v < VPT; v++) row[u][v] = load_vec<T, VEC>(dy + (size_t)entry[u].x * (size_t)a.dy_stride + col[v]);
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (k + u < end) {
#pragma unroll
        for (int v = 0; v < VPT; v++)
#pragma unroll
          for (int e = 0; e < VEC; e++) acc[v][e] += elem<T, VEC>(row[u][v], e);
        const unsigned id = entry[u].y;
        if (k + u + 1 == end || id != (u + 1 < U ? entry[u + 1 < U ? u + 1 : u].y : next)) {   // the token's last row here
          const bool part0 = long0 && id == id0, partl = longl && id == idl;
#pragma unroll
          for (int v = 0; v < VPT; v++) {
            if (slot[v] < slots) {
              if (part0 || partl) {
                float *p = sc.partial + ((size_t)c * 2 + (part0 ? 0 : 1)) * ((size_t)slots * VEC) + (size_t)slot[v] * VEC;
                store_vec<float, VEC>(p, round_vec<float, VEC>(acc[v]));
              } else {
                float s[VEC];
#pragma unroll
                for (int e = 0; e < VEC; e++) s[e] = acc[v][e] * a.scale;
                store_vec<O, VEC>(static_cast<O *>(a.dweight) + (size_t)id * (size_t)a.dweight_stride + col[v], round_vec<O, VEC>(s));
              }
            }
#pragma unroll
            for (int e = 0; e < VEC; e++) acc[v][e] = 0.0f;
          }
        }
      }
    }
  }
}

// The shared tokens: a workgroup adds up the parts of one token over 64 slots; its sixteen waves take the parts in turn
// and their sums are added in the order of the waves.
constexpr int kJoinWaves = 16;
template <class O, int VEC>
__global__ __launch_bounds__(64 * kJoinWaves) void join_rows_kernel(hf_embedding_backward_args a, TableScratch sc, int tiles) {
  __shared__ float sums[kJoinWaves][64 * VEC];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int cols = (int)a.cols, slots = row_slots<VEC>(cols);
  const unsigned items = *sc.nlong * (unsigned)tiles;
  for (unsigned item = blockIdx.x; item < items; item += gridDim.x) {
    const unsigned c = sc.longs[item / (unsigned)tiles];
    const int slot = (int)(item % (unsigned)tiles) * 64 + lane;
    const unsigned id = sc.order[min((c + 1) * (unsigned)sc.chunk, sc.starts[a.vocab]) - 1].y;
    const unsigned last = (sc.starts[id + 1] - 1) / (unsigned)sc.chunk;   // the chunk its last row is in
    const size_t width = (size_t)slots * VEC;
    const float *p = sc.partial + (size_t)min(slot, slots - 1) * VEC;
    float acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) acc[e] = 0.0f;
#pragma unroll 4
    for (unsigned q = c + (unsigned)wave; q <= last; q += kJoinWaves) {
      const vec_t<float, VEC> v = load_vec<float, VEC>(p + ((size_t)q * 2 + (q == c ? 1 : 0)) * width);
#pragma unroll
      for (int e = 0; e < VEC; e++) acc[e] += elem<float, VEC>(v, e);
    }
#pragma unroll
    for (int e = 0; e < VEC; e++) sums[wave][e * 64 + lane] = acc[e];
    __syncthreads();
    if (wave == 0 && slot < slots) {
      float s[VEC];
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        s[e] = 0.0f;
        for (int w = 0; w < kJoinWaves; w++) s[e] += sums[w][e * 64 + lane];
        s[e] *= a.scale;
      }
      store_vec<O, VEC>(static_cast<O *>(a.dweight) + (size_t)id * (size_t)a.dweight_stride + slot_column<VEC>(slot, cols), round_vec<O, VEC>(s));
    }
    __syncthreads();   // the sums are reused by the next item
  }
}

// How the launches are cut: columns into slots and tiles, sorted entries into chunks.
struct TablePlan {
  int vec, vpt, lanes_log2, tiles, chunk, nchunks, range, slots;
  unsigned ranges;
  size_t order_at, longs_at, partial_at, bytes;   // starts and nlong are at the front
};

size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }

TablePlan plan_table(const hf_embedding_backward_args &a, int cus) {
  TablePlan p;
  const int vec = a.type == HF_F32 ? kVec<float> : kVec<bf16_t>;
  p.vec = a.cols >= vec ? vec : 1;
  p.slots = (int)((a.cols + p.vec - 1) / p.vec);
  p.lanes_log2 = 6;
  while (p.lanes_log2 > 0 && (1 << (p.lanes_log2 - 1)) >= p.slots) p.lanes_log2--;
  const int lanes = 1 << p.lanes_log2;
  p.vpt = p.slots > 64 ? 2 : 1;
  p.tiles = (p.slots + lanes * p.vpt - 1) / (lanes * p.vpt);
  p.chunk = 64;
  while (p.chunk > 8 && a.ntokens / p.chunk * p.tiles * lanes < (int64_t)cus * 16 * 64) p.chunk /= 2;
  while (a.ntokens / p.chunk * p.tiles * lanes >= (int64_t)1 << 31) p.chunk *= 2;   // lanes are numbered in 32 bits
  p.nchunks = (int)((a.ntokens + p.chunk - 1) / p.chunk);
  p.range = (int)std::min<int64_t>(kMaxRange, (a.vocab + cus - 1) / cus);
  p.ranges = (unsigned)((a.vocab + p.range - 1) / p.range);
  size_t at = round16(((size_t)a.vocab + 2) * sizeof(unsigned));
  p.order_at = at;
  at = round16(at + (size_t)a.ntokens * sizeof(uint2));
  p.longs_at = at;
  at = round16(at + (size_t)p.nchunks * sizeof(unsigned));
  p.partial_at = at;
  p.bytes = round16(at + (size_t)p.nchunks * 2 * (size_t)p.slots * (size_t)p.vec * sizeof(float));
  return p;
}

template <class T, class O, int VEC>
hipError_t sum_tokens(const hf_embedding_backward_args &a, const TablePlan &p, const TableScratch &sc, int cus, hipStream_t s) {
  const unsigned long long blocks = ((((unsigned long long)p.nchunks * (unsigned)p.tiles) << p.lanes_log2) + 255) / 256;
  if (p.vpt == 2)
    hipLaunchKernelGGL((sum_rows_kernel<T, O, VEC, 2, true>), dim3((unsigned)blocks), dim3(256), 0, s, a, sc, 6, p.tiles);
  else if (p.lanes_log2 == 6)
    hipLaunchKernelGGL((sum_rows_kernel<T, O, VEC, 1, true>), dim3((unsigned)blocks), dim3(256), 0, s, a, sc, 6, p.tiles);
  else
    hipLaunchKernelGGL((sum_rows_kernel<T, O, VEC, 1, false>), dim3((unsigned)blocks), dim3(256), 0, s, a, sc, p.lanes_log2, p.tiles);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int join_tiles = (p.slots + 63) / 64;
  const unsigned grid = (unsigned)std::min<unsigned long long>((unsigned long long)p.nchunks * (unsigned)join_tiles, (unsigned long long)cus * 4);
  hipLaunchKernelGGL((join_rows_kernel<O, VEC>), dim3(grid), dim3(64 * kJoinWaves), 0, s, a, sc, join_tiles);
  return hipGetLastError();
}

template <class T>
hipError_t embed_backward(const hf_embedding_backward_args &a, int cus, hipStream_t s) {
  const TablePlan p = plan_table(a, cus);
  unsigned char *ws = static_cast<unsigned char *>(a.workspace);
  TableScratch sc;
  sc.starts = reinterpret_cast<unsigned *>(ws);
  sc.nlong = sc.starts + a.vocab + 1;
  sc.order = reinterpret_cast<uint2 *>(ws + p.order_at);
  sc.longs = reinterpret_cast<unsigned *>(ws + p.longs_at);
  sc.partial = reinterpret_cast<float *>(ws + p.partial_at);
  sc.chunk = p.chunk;
  sc.nchunks = p.nchunks;
  const unsigned out_bytes = a.out_type == HF_F32 ? 4 : 2;
  const size_t lds = (((size_t)kGroupWaves * p.range + 1) & ~(size_t)1) * 4 + (size_t)kGroupWaves * kHitWords * 8;
  if (a.index_type == HF_I64)
    hipLaunchKernelGGL(group_tokens_kernel<int64_t>, dim3(p.ranges), dim3(kGroupThreads), lds, s, a, sc, p.range, (unsigned)a.cols * out_bytes, out_bytes);
  else
    hipLaunchKernelGGL(group_tokens_kernel<int32_t>, dim3(p.ranges), dim3(kGroupThreads), lds, s, a, sc, p.range, (unsigned)a.cols * out_bytes, out_bytes);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.ntokens == 0) return e;
  if (a.out_type == HF_F32)
    return p.vec == 1 ? sum_tokens<T, float, 1>(a, p, sc, cus, s) : sum_tokens<T, float, kVec<T>>(a, p, sc, cus, s);
  return p.vec == 1 ? sum_tokens<T, T, 1>(a, p, sc, cus, s) : sum_tokens<T, T, kVec<T>>(a, p, sc, cus, s);
}

}  // namespace

size_t embedding_backward_workspace(const hf_embedding_backward_args &a, int cus) { return plan_table(a, cus).bytes; }

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
  return with_type(a.type, [&](auto t) { return embed_backward<decltype(t)>(a, cus, s); });
}

}  // namespace hfuse
