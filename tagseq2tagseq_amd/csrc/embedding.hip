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
//      list starts, and the occurrences of its own ids, and writes the zero
//      rows of its absent ids; on a second reading each wave places its
//      positions, in order, behind those of the waves before it.  No work-group
//      waits for another.
//   2. embed_sum_kernel: the list in pieces of S positions; a lane sums its
//      columns over a piece and stores a token's row where all its positions
//      lie within the piece, and a partial sum where they do not.
//   3. embed_join_kernel: tokens that cross pieces, from their partial sums.
//
// Every order is that of the positions: results do not change from run to run.
#include "attn_kernels.h"

namespace t2t {

namespace {

constexpr int kEmbThreads = 256;
constexpr int kGroupThreads = 1024;
constexpr int kGroupWaves = kGroupThreads / 64;
constexpr int kSumThreads = 256;
constexpr int kJoinWaves = 4;

// VEC values of T in one access of up to 16 bytes.
template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Pack {
  T v[VEC];
};

template <typename T, int VEC>
__global__ __launch_bounds__(kEmbThreads) void embed_kernel(EmbedArgs a) {
  const int nv = a.C / VEC;
  const int64_t first = (int64_t)blockIdx.x * kEmbThreads;
  const int64_t n0 = first / nv;
  const uint32_t r = (uint32_t)(first - n0 * nv) + threadIdx.x;
  const int64_t n = n0 + r / (uint32_t)nv;
  const int c = r % (uint32_t)nv;
  if (n >= a.N) return;
  const int64_t t = a.tokens[n];
  Pack<T, VEC> o;
  if (t >= 0 && t < a.V) {
    const Pack<T, VEC> w =
        reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(a.weight) + t * a.w_stride)[c];
#pragma unroll
    for (int e = 0; e < VEC; ++e) o.v[e] = (T)((float)w.v[e] * a.scale);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) o.v[e] = (T)__builtin_nanf("");
  }
  reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(a.out) + n * (int64_t)a.C)[c] = o;
}

__device__ __forceinline__ int wg_sum(int x, int* red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  int s = 0;
#pragma unroll
  for (int w = 0; w < kGroupWaves; ++w) s += red[w];
  __syncthreads();
  return s;
}

// cursor[wave][row]: first the occurrences of the group's row in the wave's
// part of the tokens, then where the wave's next one goes.
template <typename T, int VEC>
__global__ __launch_bounds__(kGroupThreads) void embed_group_kernel(EmbedGradArgs a) {
  extern __shared__ int lds[];
  const int R = a.rows_per_group;
  int* cursor = lds;                     // [kGroupWaves][R]
  int* total = lds + kGroupWaves * R;    // [R]
  int* red = total + R;                  // [kGroupWaves]
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
    const bool valid = t >= 0 && t < a.V && t != a.padding;
    const uint32_t rest = (uint32_t)t & (G - 1);
    before += valid && rest < r;
    if (valid && rest == r) atomicAdd(&cursor[wave * R + (int)(t >> a.group_log2)], 1);
  }
  const int base = wg_sum(before, red);  // its barriers also end the counting

  // Exclusive sums over rows, then over the waves within a row.
  int done = 0;
  for (int r0 = 0; r0 < R; r0 += kGroupThreads) {
    const int row = r0 + threadIdx.x;
    int count = 0;
    if (row < R)
      for (int w = 0; w < kGroupWaves; ++w) count += cursor[w * R + row];
    int x = count;  // inclusive over the wave
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int y = __shfl_up(x, off, 64);
      if (lane >= off) x += y;
    }
    if (lane == 63) red[wave] = x;
    __syncthreads();
    int at = base + done + x - count;
    for (int w = 0; w < wave; ++w) at += red[w];
    int all = 0;
    for (int w = 0; w < kGroupWaves; ++w) all += red[w];
    if (row < R) {
      total[row] = count;
      for (int w = 0; w < kGroupWaves; ++w) {
        const int c = cursor[w * R + row];
        cursor[w * R + row] = at;
        at += c;
      }
    }
    done += all;
    __syncthreads();
  }
  if (r == G - 1 && threadIdx.x == 0) *a.count = base + done;

  // Rows of ids that do not occur (and the padding row): zeros.
  const int nv = a.C / VEC;
  Pack<T, VEC> zero;
#pragma unroll
  for (int e = 0; e < VEC; ++e) zero.v[e] = (T)0.f;
  for (int row = wave; row < R; row += kGroupWaves) {
    const int64_t v = ((int64_t)row << a.group_log2) + r;
    if (v >= a.V || total[row]) continue;
    Pack<T, VEC>* dst = reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(a.dweight) + v * a.C);
    for (int c = lane; c < nv; c += 64) dst[c] = zero;
  }

  // Second reading: 64 positions at a time, one token id after the other.
  for (int s = i0; s < i1; s += 64) {
    const int i = s + lane;
    const int64_t t = i < i1 ? a.tokens[i] : -1;
    const bool own = t >= 0 && t < a.V && t != a.padding && ((uint32_t)t & (G - 1)) == r;
    const int row = own ? (int)(t >> a.group_log2) : -1;
    uint64_t left = __ballot(own);
    while (left) {
      const int leader = __ffsll((unsigned long long)left) - 1;
      const int lrow = __shfl(row, leader, 64);
      const uint64_t same = __ballot(row == lrow);
      int at = 0;
      if (lane == leader) at = atomicAdd(&cursor[wave * R + lrow], __popcll(same));
      at = __shfl(at, leader, 64);
      if (row == lrow) {
        at += __popcll(same & ((1ull << lane) - 1));
        a.list[at] = make_int2(i, (int)t);
      }
      left &= ~same;
    }
  }
}

// A thread sums VEC columns of one piece.
template <typename T, int VEC>
__global__ __launch_bounds__(kSumThreads) void embed_sum_kernel(EmbedGradArgs a) {
  const int nv = a.C / VEC, M = *a.count;
  const int64_t first = (int64_t)blockIdx.x * kSumThreads;
  const int64_t k0 = first / nv;
  const uint32_t r = (uint32_t)(first - k0 * nv) + threadIdx.x;
  const int64_t piece = k0 + r / (uint32_t)nv;
  const int c = r % (uint32_t)nv;
  const int64_t e0 = piece * a.piece;
  if (e0 >= M) return;
  const int64_t e1 = min((int64_t)M, e0 + a.piece);
  const int before = e0 ? a.list[e0 - 1].y : -1;
  const int after = e1 < M ? a.list[e1].y : -1;
  float acc[VEC] = {};
  int64_t e = e0;
  while (e < e1) {
    const int token = a.list[e].y;
    const bool from_before = e == e0 && token == before;
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
    for (; e < e1; ++e) {
      const int2 at = a.list[e];
      if (at.y != token) break;
      const Pack<T, VEC> d = reinterpret_cast<const Pack<T, VEC>*>(
          static_cast<const T*>(a.dy) + (int64_t)at.x * a.dy_stride)[c];
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] += (float)d.v[k];
    }
    const bool to_after = e == e1 && token == after;
    if (from_before || to_after) {
      float* p = a.part + (2 * piece + !from_before) * a.C + c * VEC;
#pragma unroll
      for (int k = 0; k < VEC; ++k) p[k] = acc[k];
    } else {
      Pack<T, VEC> o;
#pragma unroll
      for (int k = 0; k < VEC; ++k) o.v[k] = (T)(acc[k] * a.scale);
      reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(a.dweight) + (int64_t)token * a.C)[c] = o;
    }
  }
}

// Work-group (piece, 64 columns): where a token's positions start in the piece
// and go on behind it, the sum of its partial sums, in order: each wave a
// contiguous share, then the waves.
template <typename T>
__global__ __launch_bounds__(64 * kJoinWaves) void embed_join_kernel(EmbedGradArgs a) {
  __shared__ float red[kJoinWaves][64];
  __shared__ int ends;
  const int M = *a.count;
  const int64_t piece = blockIdx.x, e0 = piece * a.piece, e1 = e0 + a.piece;
  if (e1 >= M) return;
  const int token = a.list[e1].y;
  if (a.list[e1 - 1].y != token) return;
  if (a.list[e0].y == token && e0 && a.list[e0 - 1].y == token) return;  // starts further ahead
  // The last piece that the token reaches: the first one behind whose next
  // piece starts with another token.
  const int64_t pieces = (M + a.piece - 1) / a.piece;
  if (threadIdx.x == 0) ends = 0x7fffffff;
  __syncthreads();
  int64_t last = 0;
  for (int64_t p = piece + 1;; p += 64 * kJoinWaves) {
    const int64_t q = p + threadIdx.x + 1;  // does piece q start with the token?
    if (q >= pieces || a.list[q * a.piece].y != token) atomicMin(&ends, (int)(q - 1));
    __syncthreads();
    last = ends;
    __syncthreads();
    if (last != 0x7fffffff) break;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t count = last - piece + 1;
  const int64_t share = (count + kJoinWaves - 1) / kJoinWaves;
  const int64_t s0 = wave * share, s1 = min(count, s0 + share);
  const int c = blockIdx.y * 64 + lane;
  float sum = 0.f;
  if (c < a.C) {
#pragma unroll 8
    for (int64_t s = s0; s < s1; ++s)
      sum += a.part[(2 * (piece + s) + (s == 0)) * a.C + c];
  }
  red[wave][lane] = sum;
  __syncthreads();
  if (wave || c >= a.C) return;
  float all = red[0][lane];
#pragma unroll
  for (int w = 1; w < kJoinWaves; ++w) all += red[w][lane];
  static_cast<T*>(a.dweight)[(int64_t)token * a.C + c] = (T)(all * a.scale);
}

template <typename T, int VEC>
hipError_t launch_embed_t(const EmbedArgs& a, hipStream_t stream) {
  const int64_t items = a.N * (a.C / VEC);
  const dim3 grid((unsigned)((items + kEmbThreads - 1) / kEmbThreads));
  hipLaunchKernelGGL((embed_kernel<T, VEC>), grid, dim3(kEmbThreads), 0, stream, a);
  return hipGetLastError();
}

template <typename T, int VEC>
hipError_t launch_grad_t(const EmbedGradArgs& a, hipStream_t stream) {
  const int lds = (kGroupWaves * a.rows_per_group + a.rows_per_group + kGroupWaves) * 4;
  hipLaunchKernelGGL((embed_group_kernel<T, VEC>), dim3(1u << a.group_log2), dim3(kGroupThreads),
                     lds, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.N == 0) return e;
  const int64_t pieces = ((int64_t)a.N + a.piece - 1) / a.piece;
  const int64_t items = pieces * (a.C / VEC);
  hipLaunchKernelGGL((embed_sum_kernel<T, VEC>),
                     dim3((unsigned)((items + kSumThreads - 1) / kSumThreads)), dim3(kSumThreads),
                     0, stream, a);
  e = hipGetLastError();
  if (e != hipSuccess || pieces < 2) return e;
  hipLaunchKernelGGL(embed_join_kernel<T>, dim3((unsigned)pieces, (unsigned)((a.C + 63) / 64)),
                     dim3(64 * kJoinWaves), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

// Work-groups: 512 (two on each CU), more where a group's rows would not fit
// the LDS counters (17 ints a row: 52 KiB); positions a piece: 16.
EmbedPlan embed_plan(int64_t N, int64_t V, int C) {
  EmbedPlan p{};
  p.group_log2 = 9;
  while ((V >> p.group_log2) >= 768) ++p.group_log2;
  p.rows_per_group = (int)((V + (1ll << p.group_log2) - 1) >> p.group_log2);
  p.piece = 16;
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
  if (f32) return vector ? launch_grad_t<float, 4>(a, stream) : launch_grad_t<float, 1>(a, stream);
  return vector ? launch_grad_t<__bf16, 8>(a, stream) : launch_grad_t<__bf16, 1>(a, stream);
}

}  // namespace t2t
