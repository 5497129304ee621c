// Scaled embedding lookup and its weight gradient.
//
//   out[i] = s W[t_i],      dW[v] = s sum over i with t_i = v of dy[i]
//
// in fp32 with one rounding; an id outside [0, V) gives a row of NaN and no
// gradient, and the padding row's gradient is zero.
//
// The gradient is a sum by token: the positions are grouped by token id and
// the rows of dy read once in that order.  HBM bound: dy is read once and the
// V rows of dW are written once, most of them zeros.
//
//   1. Group r of G has the ids with id mod G = r (G a power of two, so
//      neighbouring ids, whose frequencies are alike, spread over the groups).
//      embed_split_kernel sorts blocks of 2048 positions by group, in LDS;
//      embed_group_kernel, a work-group a group, sorts the group's parts of all
//      blocks by id: each wave counts its share of them, and places them in order
//      behind those of the waves before it.  (Without the split, every
//      work-group reading all ids, in step and from the same L2 channels, 131072
//      ids took 70 us, 20 this way.)  Further work-groups of both launches
//      fill dW with zeros meanwhile (a wave's loads wait for its own
//      earlier stores, so not the same ones).
//   2. embed_sum_kernel: the list in pieces of S positions; each is summed by
//      token, and a token's row is stored where all its positions lie within the
//      piece, a partial sum where they do not.
//   3. embed_join_kernel: tokens that cross pieces, from their partial sums.
//
// 16384 positions of 768 columns in bf16 into 50257 rows: 38 us, where reading dy
// and writing dW at the rate of a large copy take 20; 131072: 103 us and 54.  The
// rows of dy, 1.5 KB each in no order of addresses, arrive at 3.4 TB/s, with 8 or
// 16 of them in flight a thread.
//
// Up to 2048 positions, whose four launches would be latency, embed_small_kernel
// does all but the zeros: a work-group reads all ids, sorts its group's positions
// in LDS and sums them.  (Writing the rows of its absent ids too, 77 MB of rows
// 256 ids apart, took 35 us; the fill ahead of it takes 13.)
//
// Every order is that of the positions: results do not change from run to run.
#include <algorithm>

#include "attn_kernels.h"

namespace t2t {

namespace {

constexpr int kEmbThreads = 256;
constexpr int kEmbItems = 4;
constexpr int kEmbedSmall = 2048;      // positions that embed_small_kernel sums
constexpr int kLongRow = 64;           // positions: from here a row is all waves' there
constexpr int kGroupThreads = 512;
constexpr int kGroupWaves = kGroupThreads / 64;
constexpr int kGroupSteps = 4;         // of 64 positions, loaded at once
constexpr int kSplitItems = 4;         // positions a thread
constexpr int kSplitBlock = kGroupThreads * kSplitItems;
constexpr int kSumThreads = 256;
constexpr int kJoinWaves = 16;
constexpr int kLongRun = 32;           // pieces: from here the work-group joins a token

// VEC values of T in one access of up to 16 bytes.
template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Pack {
  T v[VEC];
};

// A thread moves kEmbItems pieces, the loads of all in flight at once.
template <typename T, int VEC>
__global__ __launch_bounds__(kEmbThreads) void embed_kernel(EmbedArgs a) {
  const uint32_t nv = a.C / VEC;
  const int64_t first = (int64_t)blockIdx.x * (kEmbThreads * kEmbItems);
  const int64_t n0 = first / nv;
  const uint32_t r0 = (uint32_t)(first - n0 * nv) + threadIdx.x;
  Pack<T, VEC> w[kEmbItems];
  int64_t t[kEmbItems];
#pragma unroll
  for (int k = 0; k < kEmbItems; ++k) {
    const int64_t n = n0 + (r0 + k * kEmbThreads) / nv;
    t[k] = a.tokens[n < a.N ? n : a.N - 1];
  }
#pragma unroll
  for (int k = 0; k < kEmbItems; ++k) {
    const int64_t row = (uint64_t)t[k] < (uint64_t)a.V ? t[k] : 0;  // (a row to read, unused)
    w[k] = reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(a.weight) +
                                                 row * a.w_stride)[(r0 + k * kEmbThreads) % nv];
  }
#pragma unroll
  for (int k = 0; k < kEmbItems; ++k) {
    const uint32_t r = r0 + k * kEmbThreads;
    const int64_t n = n0 + r / nv;
    if (n >= a.N) return;
    const float scale = (uint64_t)t[k] < (uint64_t)a.V ? a.scale : __builtin_nanf("");
    Pack<T, VEC> o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o.v[e] = (T)((float)w[k].v[e] * scale);
    reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(a.out) + n * (int64_t)a.C)[r % nv] = o;
  }
}

// An id as 32 bits; one outside 32 bits as the largest number, which is no row.
__device__ __forceinline__ uint32_t id_of(int64_t t) {
  return (uint64_t)t >> 32 ? 0xffffffffu : (uint32_t)t;
}

// Bytes [from, to) of dW, multiples of 16 but for the end of dW.
__device__ __forceinline__ void fill_zeros(void* dw, int64_t from, int64_t to, int block,
                                           int blocks) {
  const int64_t n = to / 16, step = (int64_t)blocks * kGroupThreads;
  const int64_t first = (int64_t)block * kGroupThreads + threadIdx.x;
  uint4* dst = static_cast<uint4*>(dw);
  for (int64_t i = from / 16 + first; i < n; i += step) dst[i] = make_uint4(0, 0, 0, 0);
  const int rest = (int)(to % 16) / 2;  // the 16-bit words behind the whole pieces
  if (first < rest) reinterpret_cast<uint16_t*>(dst + n)[first] = 0;
}

// The lanes of `active` whose v, of `bits` bits, is this lane's.
__device__ __forceinline__ uint64_t same_lanes(uint32_t v, int bits, uint64_t active) {
  uint64_t same = active;
  for (int b = 0; b < bits; ++b) {
    const bool one = v >> b & 1;
    const uint64_t ones = __ballot(one);
    same &= one ? ones : ~ones;
  }
  return same;
}

// Where the active lanes' values go: behind the earlier ones of the same v,
// counted in cursor[v], in the order of the lanes.
__device__ __forceinline__ int place(int* cursor, uint32_t v, int bits, bool active) {
  const int lane = threadIdx.x & 63;
  const uint64_t same = same_lanes(v, bits, __ballot(active));
  const int leader = __ffsll((unsigned long long)same) - 1;
  int at = 0;
  if (active && lane == leader) at = atomicAdd(&cursor[v], __popcll(same));
  at = __shfl(at, active ? leader : lane, 64);
  return at + __popcll(same & ((1ull << lane) - 1));
}

// counts[wave][n] to where the first value of each kind goes: behind those of
// smaller kinds and of earlier waves, from `base` on.  Returns the end.
__device__ __forceinline__ int starts_of(int* counts, int n, int base, int* red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int k0 = 0; k0 < n; k0 += kGroupThreads) {
    const int k = k0 + threadIdx.x;
    int count = 0;
    if (k < n)
#pragma unroll
      for (int w = 0; w < kGroupWaves; ++w) count += counts[w * n + k];
    int x = count;  // inclusive over the wave
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int y = __shfl_up(x, off, 64);
      if (lane >= off) x += y;
    }
    if (lane == 63) red[wave] = x;
    __syncthreads();
    int at = base + x - count;
#pragma unroll
    for (int w = 0; w < kGroupWaves; ++w) {
      if (w < wave) at += red[w];
      base += red[w];
    }
    if (k < n)
#pragma unroll
      for (int w = 0; w < kGroupWaves; ++w) {
        const int c = counts[w * n + k];
        counts[w * n + k] = at;
        at += c;
      }
    __syncthreads();
  }
  return base;
}

// A block of 2048 positions sorted by group: (position, id) to split[block],
// where each group's part starts to bounds[block][G + 1].
__global__ __launch_bounds__(kGroupThreads) void embed_split_kernel(EmbedGradArgs a) {
  extern __shared__ int lds[];
  if ((int)blockIdx.x >= a.blocks) {
    fill_zeros(a.dweight, 0, a.zero_split, blockIdx.x - a.blocks, gridDim.x - a.blocks);
    return;
  }
  const int G = 1 << a.group_log2, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int* cursor = lds;                  // [kGroupWaves][G]
  int* red = lds + kGroupWaves * G;   // [kGroupWaves]
  const int64_t b0 = (int64_t)blockIdx.x * kSplitBlock;
  const int i0 = wave * 64 * kSplitItems + lane;
  uint32_t id[kSplitItems];
#pragma unroll
  for (int k = 0; k < kSplitItems; ++k) {
    const int64_t i = b0 + i0 + 64 * k;
    id[k] = i < a.N ? id_of(a.tokens[i]) : 0;
  }
  for (int i = threadIdx.x; i < kGroupWaves * G; i += kGroupThreads) cursor[i] = 0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSplitItems; ++k)
    if (b0 + i0 + 64 * k < a.N) atomicAdd(&cursor[wave * G + (id[k] & (G - 1))], 1);
  __syncthreads();
  const int all = starts_of(cursor, G, 0, red);
  int* bounds = a.bounds + (int64_t)blockIdx.x * (G + 1);
  for (int g = threadIdx.x; g < G; g += kGroupThreads) bounds[g] = cursor[g];  // wave 0's start
  if (threadIdx.x == 0) bounds[G] = all;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSplitItems; ++k) {
    const bool in = b0 + i0 + 64 * k < a.N;
    const int at = place(cursor + wave * G, id[k] & (G - 1), a.group_log2, in);
    if (in) a.split[b0 + at] = make_int2((int)(b0 + i0 + 64 * k), (int)id[k]);
  }
}

// Calls f(position, id, active) for the wave's share of the group's positions
// in the sorted blocks, in order, all lanes at once.
template <typename F>
__device__ __forceinline__ void group_share(const EmbedGradArgs& a, uint32_t r, const F& f) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t G = 1u << a.group_log2;
  const int part = (a.blocks + kGroupWaves - 1) / kGroupWaves;
  const int b0 = wave * part, b1 = min(a.blocks, b0 + part);
  for (int b = b0; b < b1; b += kGroupSteps) {
    int at[kGroupSteps], end[kGroupSteps];
    int2 e[kGroupSteps];
#pragma unroll
    for (int k = 0; k < kGroupSteps; ++k) {
      const int* bounds = a.bounds + (int64_t)min(b + k, b1 - 1) * (G + 1) + r;
      at[k] = bounds[0];
      end[k] = b + k < b1 ? bounds[1] : at[k];
    }
#pragma unroll
    for (int k = 0; k < kGroupSteps; ++k) {
      e[k] = make_int2(0, 0);
      if (at[k] + lane < end[k]) e[k] = a.split[(int64_t)(b + k) * kSplitBlock + at[k] + lane];
    }
#pragma unroll
    for (int k = 0; k < kGroupSteps; ++k) {
      if (at[k] < end[k]) f(e[k].x, (uint32_t)e[k].y, at[k] + lane < end[k]);
      for (int i = at[k] + 64; i < end[k]; i += 64) {
        int2 more = make_int2(0, 0);
        if (i + lane < end[k]) more = a.split[(int64_t)(b + k) * kSplitBlock + i + lane];
        f(more.x, (uint32_t)more.y, i + lane < end[k]);
      }
    }
  }
}

// The row of an id in its group; `none` for one without a gradient.
__device__ __forceinline__ int row_in_group(const EmbedGradArgs& a, uint32_t id, int none) {
  return id < (uint32_t)a.V && id != (uint32_t)a.padding ? (int)(id >> a.group_log2) : none;
}

// The list of a group's positions by id.  Row R, behind the others, takes ids
// without a gradient; they are in the list as token -1, so that it has every
// position and needs no count.
__global__ __launch_bounds__(kGroupThreads) void embed_group_kernel(EmbedGradArgs a) {
  extern __shared__ int lds[];
  const uint32_t G = 1u << a.group_log2;
  if (blockIdx.x >= G) {
    fill_zeros(a.dweight, a.zero_split, a.zero_bytes, blockIdx.x - G, gridDim.x - G);
    return;
  }
  const uint32_t r = blockIdx.x;
  const int R = a.rows_per_group + 1, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int* cursor = lds;                  // [kGroupWaves][R]
  int* red = lds + kGroupWaves * R;   // [kGroupWaves]
  for (int i = threadIdx.x; i < kGroupWaves * R; i += kGroupThreads) cursor[i] = 0;
  // Positions of smaller groups.
  int before = 0;
  for (int b = threadIdx.x; b < a.blocks; b += kGroupThreads)
    before += a.bounds[(int64_t)b * (G + 1) + r];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) before += __shfl_xor(before, off, 64);
  if (lane == 0) red[wave] = before;
  __syncthreads();
  int base = 0;
#pragma unroll
  for (int w = 0; w < kGroupWaves; ++w) base += red[w];

  group_share(a, r, [&](int, uint32_t id, bool own) {
    if (own) atomicAdd(&cursor[wave * R + row_in_group(a, id, R - 1)], 1);
  });
  __syncthreads();
  starts_of(cursor, R, base, red);
  group_share(a, r, [&](int i, uint32_t id, bool own) {
    const int row = own ? row_in_group(a, id, R - 1) : 0;
    const int at = place(cursor + wave * R, row, a.row_bits, own);
    if (own) a.list[at] = row == R - 1 ? make_int2(0, -1) : make_int2(i, (int)id);
  });
}

__global__ __launch_bounds__(kGroupThreads) void embed_zero_kernel(EmbedGradArgs a) {
  fill_zeros(a.dweight, 0, a.zero_bytes, blockIdx.x, gridDim.x);
}

// The rows of a short list (at most kEmbedSmall positions) in one launch, a
// work-group a group of ids.  A row of up to kLongRow positions is summed by a
// wave, a longer one by all of them: each a contiguous share, then the shares.
template <typename T, int VEC>
__global__ __launch_bounds__(kGroupThreads) void embed_small_kernel(EmbedGradArgs a) {
  extern __shared__ int lds[];
  const uint32_t G = 1u << a.group_log2, r = blockIdx.x;
  const int R = a.rows_per_group + 1, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // The counters, and when they are done with, the shares [kGroupWaves][64 VEC].
  int* cursor = lds;
  float* shares = reinterpret_cast<float*>(lds);
  int* start = lds + kGroupWaves * max(R, 64 * VEC);  // [R + 1]: a row's first in the list
  int* list = start + R + 1;                          // [N]: positions
  int* red = list + a.N;                              // [kGroupWaves]
  for (int i = threadIdx.x; i < kGroupWaves * R; i += kGroupThreads) cursor[i] = 0;
  // A wave has kEmbedSmall / 8 positions at most, in order.
  constexpr int kSteps = kEmbedSmall / kGroupThreads;
  const int part = ((a.N + kGroupWaves - 1) / kGroupWaves + 63) & ~63;
  const int i0 = wave * part + lane, i1 = min(a.N, (wave + 1) * part);
  int row[kSteps];  // -1: another group's
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int i = i0 + 64 * k;
    const uint32_t id = i < i1 ? id_of(a.tokens[i]) : r ^ 1;
    row[k] = (id & (G - 1)) == r ? row_in_group(a, id, R - 1) : -1;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSteps; ++k)
    if (row[k] >= 0) atomicAdd(&cursor[wave * R + row[k]], 1);
  __syncthreads();
  const int all = starts_of(cursor, R, 0, red);
  for (int i = threadIdx.x; i < R; i += kGroupThreads) start[i] = cursor[i];  // wave 0's
  if (threadIdx.x == 0) start[R] = all;
  __syncthreads();
  for (int k = 0; k < kSteps; ++k) {
    int mine = -1;
#pragma unroll
    for (int j = 0; j < kSteps; ++j) mine = j == k ? row[j] : mine;
    if (!__ballot(mine >= 0)) continue;
    const int at = place(cursor + wave * R, mine < 0 ? 0 : mine, a.row_bits, mine >= 0);
    if (mine >= 0) list[at] = i0 + 64 * k;
  }
  __syncthreads();

  // The sum of positions [s, e) of the list in the lane's columns, in order.
  const auto sum = [&](int s, int e, int c, float (&acc)[VEC]) {
    const T* dy = static_cast<const T*>(a.dy) + c;
    for (; s < e; s += 8) {
      Pack<T, VEC> d[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)  // (behind the end: the last one again, unused)
        d[k] = *reinterpret_cast<const Pack<T, VEC>*>(
            dy + (int64_t)list[min(s + k, e - 1)] * a.dy_stride);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (s + k < e)
#pragma unroll
          for (int v = 0; v < VEC; ++v) acc[v] += (float)d[k].v[v];
    }
  };
  const auto store = [&](int row, int c, const float (&acc)[VEC]) {
    Pack<T, VEC> o;
#pragma unroll
    for (int v = 0; v < VEC; ++v) o.v[v] = (T)(acc[v] * a.scale);
    *reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(a.dweight) +
                                     (((int64_t)row << a.group_log2) + r) * a.C + c) = o;
  };
  // Rows by their number of positions: f(row) for each, in turn by wave where
  // the waves share them out.
  const auto rows = [&](int least, int most, bool shared, const auto& f) {
    int turn = 0;
    for (int r0 = 0; r0 < R - 1; r0 += 64) {
      const int mine = r0 + lane;
      const bool there = mine < R - 1 && ((int64_t)mine << a.group_log2) + r < a.V;
      const int count = there ? start[mine + 1] - start[mine] : -1;
      for (uint64_t left = __ballot(count >= least && count <= most); left; left &= left - 1) {
        if (!shared || turn++ % kGroupWaves == wave) f(r0 + __ffsll((unsigned long long)left) - 1);
      }
    }
  };
  rows(1, kLongRow, true, [&](int row) {
    for (int c = lane * VEC; c < a.C; c += 64 * VEC) {
      float acc[VEC] = {};
      sum(start[row], start[row + 1], c, acc);
      store(row, c, acc);
    }
  });
  rows(kLongRow + 1, kEmbedSmall, false, [&](int row) {
    const int s = start[row], e = start[row + 1], share = (e - s + kGroupWaves - 1) / kGroupWaves;
    for (int c0 = 0; c0 < a.C; c0 += 64 * VEC) {
      const int c = c0 + lane * VEC;
      float acc[VEC] = {};
      if (c < a.C) sum(min(e, s + wave * share), min(e, s + (wave + 1) * share), c, acc);
#pragma unroll
      for (int v = 0; v < VEC; ++v) shares[(wave * 64 + lane) * VEC + v] = acc[v];
      __syncthreads();
      if (wave == 0 && c < a.C) {
        for (int w = 1; w < kGroupWaves; ++w)
#pragma unroll
          for (int v = 0; v < VEC; ++v) acc[v] += shares[(w * 64 + lane) * VEC + v];
        store(row, c, acc);
      }
      __syncthreads();
    }
  });
}

// A thread sums VEC columns of a piece of S positions, the loads of kSumBatch
// of them in flight at once.  Lanes go on into the next piece where a row is no
// multiple of a wave's columns (the whole gradient of 65536 rows of 512 columns
// 51.9 us, of 131072 rows of 768 103.3 us; with waves of their own for each piece,
// a quarter of whose lanes 768 columns leave idle, 54.8 and 105.5 us).
template <typename T, int VEC, int S>
__global__ __launch_bounds__(kSumThreads) void embed_sum_kernel(EmbedGradArgs a) {
  constexpr int kSumBatch = 8;  // (16 of pieces of 32: as fast)
  const int M = a.N;
  const uint32_t per = a.C / VEC;
  const int64_t first = (int64_t)blockIdx.x * kSumThreads, piece0 = first / per;
  const uint32_t column = (uint32_t)(first - piece0 * per) + threadIdx.x;
  const int64_t piece = piece0 + column / per;
  const int c = (int)(column % per) * VEC;
  const int64_t e0 = piece * S;
  if (e0 >= M) return;
  const int n = (int)min((int64_t)S, M - e0);
  const int2* __restrict__ list = a.list + e0;
  const T* __restrict__ dy = static_cast<const T*>(a.dy) + c;
  const int before = e0 ? list[-1].y : -2, after = e0 + n < M ? list[n].y : -2;
  float acc[VEC] = {};
  bool from_before = list[0].y == before;
#pragma unroll 1  // (unrolled, most of a short list's time went into fetching code)
  for (int b = 0; b < n; b += kSumBatch) {
    // (positions behind the end: the first one, unused; what lies behind the list
    // in the workspace may be read)
    int token[kSumBatch], pos[kSumBatch];
    Pack<T, VEC> d[kSumBatch];
#pragma unroll
    for (int e = 0; e < kSumBatch; e += 2) {
      const int4 at = *reinterpret_cast<const int4*>(list + b + e);
      pos[e] = b + e < n ? at.x : 0;
      token[e] = at.y;
      pos[e + 1] = b + e + 1 < n ? at.z : 0;
      token[e + 1] = at.w;
    }
#pragma unroll
    for (int e = 0; e < kSumBatch; ++e) {
      d[e] = *reinterpret_cast<const Pack<T, VEC>*>(dy + (int64_t)pos[e] * a.dy_stride);
    }
    __builtin_amdgcn_sched_barrier(0);  // none of the loads moves to its use
    const int next = b + kSumBatch < n ? list[b + kSumBatch].y : after;
#pragma unroll
    for (int e = 0; e < kSumBatch; ++e) {
      if (b + e >= n) break;
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] += (float)d[e].v[k];
      const bool ends = b + e + 1 == n;
      const int follows = ends ? after : e + 1 < kSumBatch ? token[(e + 1) % kSumBatch] : next;
      if (!ends && follows == token[e]) continue;
      const bool to_after = ends && follows == token[e];
      if (token[e] >= 0) {
        if (from_before || to_after) {
          float* p = a.part + (2 * piece + !from_before) * a.C + c;
#pragma unroll
          for (int k = 0; k < VEC; ++k) p[k] = acc[k];
        } else {
          Pack<T, VEC> o;
#pragma unroll
          for (int k = 0; k < VEC; ++k) o.v[k] = (T)(acc[k] * a.scale);
          *reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(a.dweight) + (int64_t)token[e] * a.C +
                                           c) = o;
        }
      }
      from_before = false;
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
    }
  }
}

// Tokens that start in a piece and go on behind it: the sum of their partial
// sums, in order.  A work-group has 16 pieces and 64 VEC columns; a wave joins the
// token of its piece, and the one of kLongRun pieces or more that may start in
// one of the 16 (no second one can) is shared: each wave a contiguous part, then
// the waves.
template <int VEC>
__device__ __forceinline__ void add_part(const EmbedGradArgs& a, int64_t slot, int c,
                                         float (&sum)[VEC]) {
  const Pack<float, VEC> p = *reinterpret_cast<const Pack<float, VEC>*>(a.part + slot * a.C + c);
#pragma unroll
  for (int k = 0; k < VEC; ++k) sum[k] += p.v[k];
}

template <typename T, int VEC>
__device__ __forceinline__ void store_row(const EmbedGradArgs& a, int token, int c,
                                          const float (&sum)[VEC]) {
  Pack<T, VEC> o;
#pragma unroll
  for (int k = 0; k < VEC; ++k) o.v[k] = (T)(sum[k] * a.scale);
  *reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(a.dweight) + (int64_t)token * a.C + c) = o;
}

template <typename T, int VEC>
__global__ __launch_bounds__(64 * kJoinWaves) void embed_join_kernel(EmbedGradArgs a) {
  __shared__ float red[kJoinWaves][64 * VEC];
  __shared__ int long_piece, ends;
  const int M = a.N, S = a.piece;
  const int pieces = (int)(((int64_t)M + S - 1) / S);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int piece = blockIdx.x * kJoinWaves + wave;
  const int64_t e0 = (int64_t)piece * S, e1 = e0 + S;
  const int c = (blockIdx.y * 64 + lane) * VEC;
  if (threadIdx.x == 0) {
    long_piece = -1;
    ends = 0x7fffffff;
  }
  __syncthreads();
  if (e1 < M) {
    const int token = a.list[e1].y;
    const bool starts = token >= 0 && a.list[e1 - 1].y == token &&
                        !(a.list[e0].y == token && e0 && a.list[e0 - 1].y == token);
    if (starts) {
      // Lane l: does piece + 1 + l start with the token?
      const int q = piece + 1 + lane;
      const int64_t at = q < pieces ? (int64_t)q * S : e1;
      const uint64_t more = __ballot(q < pieces && a.list[at].y == token);
      const int run = __ffsll((unsigned long long)~more) - 1;  // pieces behind; -1: 64 or more
      if (run < 0 || run >= kLongRun) {
        if (lane == 0) long_piece = piece;
      } else if (c < a.C) {
        float sum[VEC] = {};
        add_part<VEC>(a, 2 * (int64_t)piece + 1, c, sum);
#pragma unroll 8
        for (int s = 1; s <= run; ++s) add_part<VEC>(a, 2 * (int64_t)(piece + s), c, sum);
        store_row<T, VEC>(a, token, c, sum);
      }
    }
  }
  __syncthreads();
  const int first = long_piece;
  if (first < 0) return;
  const int token = a.list[(int64_t)(first + 1) * S].y;
  int last = 0;  // the last piece that the token reaches
  for (int p = first + 1;; p += 64 * kJoinWaves) {
    const int q = p + threadIdx.x + 1;  // does piece q start with the token?
    if (q >= pieces || a.list[(int64_t)q * S].y != token) atomicMin(&ends, q - 1);
    __syncthreads();
    last = ends;
    __syncthreads();
    if (last != 0x7fffffff) break;
  }
  const int count = last - first + 1;
  const int share = (count + kJoinWaves - 1) / kJoinWaves;
  const int s0 = wave * share, s1 = min(count, s0 + share);
  float sum[VEC] = {};
  if (c < a.C) {
#pragma unroll 8
    for (int s = s0; s < s1; ++s) add_part<VEC>(a, 2 * (int64_t)(first + s) + (s == 0), c, sum);
  }
#pragma unroll
  for (int k = 0; k < VEC; ++k) red[wave][lane * VEC + k] = sum[k];
  __syncthreads();
  if (wave || c >= a.C) return;
#pragma unroll
  for (int w = 1; w < kJoinWaves; ++w)
#pragma unroll
    for (int k = 0; k < VEC; ++k) sum[k] += red[w][lane * VEC + k];
  store_row<T, VEC>(a, token, c, sum);
}

template <typename T, int VEC>
hipError_t launch_embed_t(const EmbedArgs& a, hipStream_t stream) {
  // (a launch has fewer than 2^32 threads: of more pieces there are several)
  const int64_t nv = a.C / VEC, most = (1ll << 31) / nv;
  constexpr int per = kEmbThreads * kEmbItems;
  for (int64_t n0 = 0; n0 < a.N; n0 += most) {
    EmbedArgs part = a;
    part.tokens += n0;
    part.out = static_cast<T*>(a.out) + n0 * a.C;
    part.N = std::min(a.N - n0, most);
    hipLaunchKernelGGL((embed_kernel<T, VEC>), dim3((unsigned)((part.N * nv + per - 1) / per)),
                       dim3(kEmbThreads), 0, stream, part);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T, int VEC, int S>
hipError_t launch_sum(const EmbedGradArgs& a, int64_t pieces, hipStream_t stream) {
  const int64_t threads = pieces * (a.C / VEC);
  const dim3 grid((unsigned)((threads + kSumThreads - 1) / kSumThreads));
  hipLaunchKernelGGL((embed_sum_kernel<T, VEC, S>), grid, dim3(kSumThreads), 0, stream, a);
  return hipGetLastError();
}

template <typename T, int VEC>
hipError_t launch_sum_piece(const EmbedGradArgs& a, int64_t pieces, hipStream_t stream) {
  return a.piece == 16 ? launch_sum<T, VEC, 16>(a, pieces, stream)
                       : launch_sum<T, VEC, 32>(a, pieces, stream);
}

template <typename T, int VEC>
hipError_t launch_join(const EmbedGradArgs& a, int64_t pieces, hipStream_t stream) {
  hipLaunchKernelGGL((embed_join_kernel<T, VEC>),
                     dim3((unsigned)((pieces + kJoinWaves - 1) / kJoinWaves),
                          (unsigned)((a.C + 64 * VEC - 1) / (64 * VEC))),
                     dim3(64 * kJoinWaves), 0, stream, a);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_grad_t(const EmbedGradArgs& a, bool vector, hipStream_t stream) {
  constexpr int kVec = 16 / (int)sizeof(T);
  const int G = 1 << a.group_log2, R = a.rows_per_group + 1;
  const auto fills = [](int64_t bytes) {  // work-groups; four 16-byte pieces a thread at least
    const int64_t n = (bytes / 16 + 4 * kGroupThreads - 1) / (4 * kGroupThreads);
    return (int)(n < 1 ? 1 : n < 768 ? n : 768);
  };
  if (a.N <= kEmbedSmall) {
    hipLaunchKernelGGL(embed_zero_kernel, dim3(fills(a.zero_bytes)), dim3(kGroupThreads), 0,
                       stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.N == 0) return e;
    const int vec = vector ? kVec : 1;
    const int lds = (kGroupWaves * std::max(R, 64 * vec) + R + 1 + a.N + kGroupWaves) * 4;
    if (vector)
      hipLaunchKernelGGL((embed_small_kernel<T, kVec>), dim3(G), dim3(kGroupThreads), lds, stream,
                         a);
    else
      hipLaunchKernelGGL((embed_small_kernel<T, 1>), dim3(G), dim3(kGroupThreads), lds, stream, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(embed_split_kernel, dim3(a.blocks + fills(a.zero_split)),
                     dim3(kGroupThreads), (kGroupWaves * G + kGroupWaves) * 4, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(embed_group_kernel, dim3(G + fills(a.zero_bytes - a.zero_split)),
                     dim3(kGroupThreads), (kGroupWaves * R + kGroupWaves) * 4, stream, a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t pieces = ((int64_t)a.N + a.piece - 1) / a.piece;
  e = vector ? launch_sum_piece<T, kVec>(a, pieces, stream)
             : launch_sum_piece<T, 1>(a, pieces, stream);
  if (e != hipSuccess) return e;
  return vector ? launch_join<T, 4>(a, pieces, stream) : launch_join<T, 1>(a, pieces, stream);
}

}  // namespace

// Groups: 256, more where a group's rows would not fit the LDS counters (8 ints
// a row: 32 KiB).  Positions a piece: few for short lists, whose waves would not
// fill the card.
EmbedPlan embed_plan(int64_t N, int64_t V, int C) {
  EmbedPlan p{};
  p.group_log2 = 8;
  while ((V >> p.group_log2) > 1024) ++p.group_log2;
  const int64_t G = 1ll << p.group_log2;
  p.rows_per_group = (int)((V + G - 1) >> p.group_log2);
  p.piece = N <= 32768 ? 16 : 32;
  p.bytes = 256;  // (never none)
  if (N <= kEmbedSmall) return p;
  p.blocks = (int)((N + kSplitBlock - 1) / kSplitBlock);
  const auto whole = [](int64_t n) { return (n + 255) / 256 * 256; };
  const int64_t pieces = (N + p.piece - 1) / p.piece;
  p.split_at = whole(N * (int64_t)sizeof(int2));
  p.bounds_at = p.split_at + whole(N * (int64_t)sizeof(int2));
  p.part_at = p.bounds_at + whole(p.blocks * (G + 1) * 4);
  p.bytes = p.part_at + 2 * pieces * C * 4;
  return p;
}

// The sum is one launch, which has fewer than 2^32 threads along an axis of its grid.
bool embed_grad_fits(int64_t N, int64_t V, int C, bool f32, bool vector) {
  if (N <= kEmbedSmall) return true;
  const int64_t piece = embed_plan(N, V, C).piece, pieces = (N + piece - 1) / piece;
  const int64_t threads = pieces * (C / (vector ? (f32 ? 4 : 8) : 1));
  return threads <= (1ll << 32) - kSumThreads;
}

hipError_t launch_embed(const EmbedArgs& a, bool f32, bool vector, hipStream_t stream) {
  if (a.N == 0) return hipSuccess;
  if (f32)
    return vector ? launch_embed_t<float, 4>(a, stream) : launch_embed_t<float, 1>(a, stream);
  return vector ? launch_embed_t<__bf16, 8>(a, stream) : launch_embed_t<__bf16, 1>(a, stream);
}

hipError_t launch_embed_grad(EmbedGradArgs a, void* workspace, bool f32, bool vector,
                             hipStream_t stream) {
  const EmbedPlan p = embed_plan(a.N, a.V, a.C);
  char* ws = static_cast<char*>(workspace);
  a.list = reinterpret_cast<int2*>(ws);
  a.split = reinterpret_cast<int2*>(ws + p.split_at);
  a.bounds = reinterpret_cast<int*>(ws + p.bounds_at);
  a.part = reinterpret_cast<float*>(ws + p.part_at);
  a.group_log2 = p.group_log2;
  a.rows_per_group = p.rows_per_group;
  a.row_bits = 0;
  while (p.rows_per_group >> a.row_bits) ++a.row_bits;  // the row behind the last too
  a.piece = p.piece;
  a.blocks = p.blocks;
  a.zero_bytes = a.V * a.C * (f32 ? 4 : 2);
  a.zero_split = a.zero_bytes / 32 * 16;  // about half in each launch
  return f32 ? launch_grad_t<float>(a, vector, stream) : launch_grad_t<__bf16>(a, vector, stream);
}

}  // namespace t2t
