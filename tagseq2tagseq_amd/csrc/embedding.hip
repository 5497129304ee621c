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
//   1. embed_group_kernel: work-group r of G takes the tokens with
//      id mod G = r (G a power of two, so neighbouring ids, whose frequencies
//      are alike, spread over the work-groups).  Every work-group reads all ids
//      (from L2): it counts those with a smaller remainder, which is where its
//      list starts, and the occurrences of its own ids; on a second reading
//      each wave places its positions, in order, behind those of the waves
//      before it.  No work-group waits for another.  Further work-groups of the
//      same launch fill dW with zeros meanwhile (a wave's loads wait for its
//      own earlier stores, so not the same ones).
//   2. embed_sum_kernel: the list in pieces of S positions; a wave sums 64 VEC
//      columns over a piece, all its loads in flight at once, and stores a
//      token's row where all its positions lie within the piece, and a partial
//      sum where they do not.
//   3. embed_join_kernel: tokens that cross pieces, from their partial sums.
//
// Every order is that of the positions: results do not change from run to run.
#include "attn_kernels.h"

namespace t2t {

namespace {

constexpr int kEmbThreads = 256;
constexpr int kEmbItems = 4;
constexpr int kSumBatch = 16;
constexpr int kGroupThreads = 1024;
constexpr int kGroupWaves = kGroupThreads / 64;
constexpr int kGroupSteps = 8;         // of 64 positions, loaded at once
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

// cursor[wave][row]: first the occurrences of the group's row in the wave's
// part of the tokens, then where the wave's next one goes.
__global__ __launch_bounds__(kGroupThreads) void embed_group_kernel(EmbedGradArgs a) {
  extern __shared__ int lds[];
  if (blockIdx.x >= 1u << a.group_log2) {  // the zeros of dW, bytes of whole 16-byte pieces
    const int64_t n = a.zero_bytes / 16, step = (int64_t)a.fill_groups * kGroupThreads;
    const int64_t i0 = (int64_t)(blockIdx.x - (1u << a.group_log2)) * kGroupThreads + threadIdx.x;
    uint4* dst = static_cast<uint4*>(a.dweight);
    for (int64_t i = i0; i < n; i += step) dst[i] = make_uint4(0, 0, 0, 0);
    const int rest = (int)(a.zero_bytes % 16) / 2;  // and the 16-bit words behind them
    if (i0 < rest) reinterpret_cast<uint16_t*>(dst + n)[i0] = 0;
    return;
  }
  const int R = a.rows_per_group;
  int* cursor = lds;                  // [kGroupWaves][R]
  int* red = lds + kGroupWaves * R;   // [kGroupWaves]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t G = 1u << a.group_log2, r = blockIdx.x;
  for (int i = threadIdx.x; i < kGroupWaves * R; i += kGroupThreads) cursor[i] = 0;
  __syncthreads();

  const int N = a.N;
  const int part = ((N + kGroupWaves - 1) / kGroupWaves + 63) & ~63;
  const int i0 = wave * part, i1 = min(N, i0 + part);
  int before = 0;
#pragma unroll 8
  for (int i = i0 + lane; i < i1; i += 64) {
    const int64_t t = a.tokens[i];
    const bool valid = (uint64_t)t < (uint64_t)a.V && t != a.padding;
    const uint32_t rest = (uint32_t)t & (G - 1);
    before += valid && rest < r;
    if (valid && rest == r) atomicAdd(&cursor[wave * R + (int)(t >> a.group_log2)], 1);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) before += __shfl_xor(before, off, 64);
  if (lane == 0) red[wave] = before;
  __syncthreads();  // the counts too
  int base = 0;
#pragma unroll
  for (int w = 0; w < kGroupWaves; ++w) base += red[w];
  __syncthreads();

  // Exclusive sums over rows, then over the waves within a row.
  for (int r0 = 0; r0 < R; r0 += kGroupThreads) {
    const int row = r0 + threadIdx.x;
    int count = 0;
    if (row < R)
#pragma unroll
      for (int w = 0; w < kGroupWaves; ++w) count += cursor[w * R + row];
    int x = count;  // inclusive over the wave
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int y = __shfl_up(x, off, 64);
      if (lane >= off) x += y;
    }
    if (lane == 63) red[wave] = x;
    __syncthreads();
    int at = base + x - count, all = 0;
#pragma unroll
    for (int w = 0; w < kGroupWaves; ++w) {
      if (w < wave) at += red[w];
      all += red[w];
    }
    if (row < R)
#pragma unroll
      for (int w = 0; w < kGroupWaves; ++w) {
        const int c = cursor[w * R + row];
        cursor[w * R + row] = at;
        at += c;
      }
    base += all;
    __syncthreads();
  }
  if (r == G - 1 && threadIdx.x == 0) *a.count = base;

  // Second reading: 64 positions at a time, one token id after the other.
  for (int s0 = i0; s0 < i1; s0 += 64 * kGroupSteps) {
    int64_t ts[kGroupSteps];
#pragma unroll
    for (int k = 0; k < kGroupSteps; ++k) {
      const int i = s0 + 64 * k + lane;
      ts[k] = i < i1 ? a.tokens[i] : -1;
    }
#pragma unroll
    for (int k = 0; k < kGroupSteps; ++k) {
      const int64_t t = ts[k];
      const bool own =
          (uint64_t)t < (uint64_t)a.V && t != a.padding && ((uint32_t)t & (G - 1)) == r;
      const int row = own ? (int)(t >> a.group_log2) : -1;
      uint64_t left = __ballot(own);
      while (left) {
        const int leader = __ffsll((unsigned long long)left) - 1;
        const int lrow = __builtin_amdgcn_readlane(row, leader);
        const uint64_t same = __ballot(row == lrow);
        int at = 0;
        if (lane == leader) at = atomicAdd(&cursor[wave * R + lrow], __popcll(same));
        at = __builtin_amdgcn_readlane(at, leader);
        if (row == lrow) {
          at += __popcll(same & ((1ull << lane) - 1));
          a.list[at] = make_int2(s0 + 64 * k + lane, (int)t);
        }
        left &= ~same;
      }
    }
  }
}

// A wave sums 64 VEC columns of a piece of S positions, lane l the columns
// VEC l .. of the wave's block, kSumBatch positions' loads in flight at once.
// The positions are the same for all lanes.
template <typename T, int VEC, int S>
__global__ __launch_bounds__(kSumThreads) void embed_sum_kernel(EmbedGradArgs a) {
  const int M = *a.count, lane = threadIdx.x & 63;
  const int blocks = (a.C + 64 * VEC - 1) / (64 * VEC);
  const int item = __builtin_amdgcn_readfirstlane(
      (int)(blockIdx.x * (kSumThreads / 64) + (threadIdx.x >> 6)));
  const int piece = item / blocks;
  const int c = (item % blocks) * 64 * VEC + lane * VEC;
  const int64_t e0 = (int64_t)piece * S;
  if (e0 >= M) return;
  const int n = (int)min((int64_t)S, M - e0);
  const int2* __restrict__ list = a.list + e0;
  const bool in = c < a.C;
  const T* __restrict__ dy = static_cast<const T*>(a.dy) + (in ? c : 0);
  const int before = e0 ? list[-1].y : -1, after = e0 + n < M ? list[n].y : -1;
  float acc[VEC] = {};
  bool from_before = list[0].y == before;
#pragma unroll
  for (int b = 0; b < S; b += kSumBatch) {
    if (b >= n) break;
    // (positions behind the piece's end: its last one again, unused)
    int token[kSumBatch];
    Pack<T, VEC> d[kSumBatch];
#pragma unroll
    for (int e = 0; e < kSumBatch; ++e) {
      const int2 at = list[min(b + e, n - 1)];
      token[e] = at.y;
      d[e] = *reinterpret_cast<const Pack<T, VEC>*>(dy + (int64_t)at.x * a.dy_stride);
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
      if (in) {
        if (from_before || to_after) {
          float* p = a.part + (2 * (int64_t)piece + !from_before) * a.C + c;
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
  const int M = *a.count, S = a.piece;
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
    const bool starts = a.list[e1 - 1].y == token &&
                        !(a.list[e0].y == token && e0 && a.list[e0 - 1].y == token);
    if (starts) {
      // Lane l: does piece + 1 + l start with the token?
      const int q = piece + 1 + lane;
      const uint64_t more = __ballot(q < pieces && a.list[q < pieces ? (int64_t)q * S : e1].y == token);
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
  const int64_t items = a.N * (a.C / VEC);
  constexpr int per = kEmbThreads * kEmbItems;
  const dim3 grid((unsigned)((items + per - 1) / per));
  hipLaunchKernelGGL((embed_kernel<T, VEC>), grid, dim3(kEmbThreads), 0, stream, a);
  return hipGetLastError();
}

template <typename T, int VEC, int S>
hipError_t launch_sum(const EmbedGradArgs& a, int64_t pieces, hipStream_t stream) {
  const int64_t waves = pieces * ((a.C + 64 * VEC - 1) / (64 * VEC));
  constexpr int per = kSumThreads / 64;
  hipLaunchKernelGGL((embed_sum_kernel<T, VEC, S>), dim3((unsigned)((waves + per - 1) / per)),
                     dim3(kSumThreads), 0, stream, a);
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
  const int lds = (kGroupWaves * a.rows_per_group + kGroupWaves) * 4;
  hipLaunchKernelGGL(embed_group_kernel, dim3((1u << a.group_log2) + a.fill_groups),
                     dim3(kGroupThreads), lds, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.N == 0) return e;
  const int64_t pieces = ((int64_t)a.N + a.piece - 1) / a.piece;
  // Columns a lane: 16 bytes, or half where that leaves fewer lanes idle (768
  // columns of bf16: three waves of 256 instead of one and a half of 512).
  constexpr int kWide = 16 / sizeof(T), kHalf = kWide / 2;
  const auto covered = [&](int vec) { return (a.C + 64 * vec - 1) / (64 * vec) * vec; };
  if (!vector)
    e = launch_sum_piece<T, 1>(a, pieces, stream);
  else if (covered(kHalf) < covered(kWide))
    e = launch_sum_piece<T, kHalf>(a, pieces, stream);
  else
    e = launch_sum_piece<T, kWide>(a, pieces, stream);
  if (e != hipSuccess || pieces < 2) return e;
  return vector ? launch_join<T, 4>(a, pieces, stream) : launch_join<T, 1>(a, pieces, stream);
}

}  // namespace

// Grouping work-groups: 256 (each reads every id), more where a group's rows
// would not fit the LDS counters (16 ints a row: 40 KiB).  Positions a piece: few
// for short lists, whose waves would not fill the card.
EmbedPlan embed_plan(int64_t N, int64_t V, int C) {
  EmbedPlan p{};
  p.group_log2 = 8;
  while ((V >> p.group_log2) >= 640) ++p.group_log2;
  p.rows_per_group = (int)((V + (1ll << p.group_log2) - 1) >> p.group_log2);
  p.piece = N <= 32768 ? 16 : 32;
  const int64_t pieces = (N + p.piece - 1) / p.piece;
  p.list_at = 256;  // behind the count
  p.part_at = (p.list_at + N * (int64_t)sizeof(int2) + 255) / 256 * 256;
  p.bytes = p.part_at + 2 * pieces * C * 4;
  return p;
}

hipError_t launch_embed(const EmbedArgs& a, bool f32, bool vector, hipStream_t stream) {
  if (a.N == 0) return hipSuccess;
  if (f32) return vector ? launch_embed_t<float, 4>(a, stream) : launch_embed_t<float, 1>(a, stream);
  return vector ? launch_embed_t<__bf16, 8>(a, stream) : launch_embed_t<__bf16, 1>(a, stream);
}

hipError_t launch_embed_grad(EmbedGradArgs a, void* workspace, bool f32, bool vector,
                             hipStream_t stream) {
  const EmbedPlan p = embed_plan(a.N, a.V, a.C);
  char* ws = static_cast<char*>(workspace);
  a.count = reinterpret_cast<int*>(ws);
  a.list = reinterpret_cast<int2*>(ws + p.list_at);
  a.part = reinterpret_cast<float*>(ws + p.part_at);
  a.group_log2 = p.group_log2;
  a.rows_per_group = p.rows_per_group;
  a.piece = p.piece;
  a.zero_bytes = a.V * a.C * (f32 ? 4 : 2);
  const int64_t fills = (a.zero_bytes / 16 + 4 * kGroupThreads - 1) / (4 * kGroupThreads);
  a.fill_groups = (int)(fills < 1 ? 1 : fills < 512 ? fills : 512);
  return f32 ? launch_grad_t<float>(a, vector, stream) : launch_grad_t<__bf16>(a, vector, stream);
}

}  // namespace t2t
