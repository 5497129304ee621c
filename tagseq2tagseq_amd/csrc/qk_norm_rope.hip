// Attention-module prologue with per-head norms: the packed projection rows
// split into heads, each query and key row RMS-normalised and rotated, values
// copied; its gradient; and the same map for new tokens, writing keys and
// values straight into a cache.
//
// For a query or key row x of D values, its weight w (one for all query heads,
// one for all key heads) and position p:
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r,  y = w n,
//   o[i]       = y[i] cos[p][i] + y[i + D/2] sin[p][i]
//   o[i + D/2] = y[i + D/2] cos[p][i] - y[i] sin[p][i]            i < D/2
// and with dy = the transposed rotation of the gradient do, g = dy w:
//   dx = r (g - n mean(g n)),   dw = sum over batch, tokens, heads of dy n.
// All of it in fp32, with one rounding when a result is stored; r is computed
// again in the backward, which reads x anyway.
//
// HBM bound: the forward reads and writes each packed row once; the backward
// reads the three gradients and the query and key part of the row, and writes
// the row's gradient.  A group of LP lanes (D / 16 rounded up to a power of
// two) holds a head row, lane j the values 8j .. 8j + 7 of both halves, so the
// rotation pairs sit in one lane and the mean is log2 LP shuffles.
#include "attn_kernels.h"

namespace t2t {

namespace {

constexpr int kQkThreads = 256;
constexpr int kQkWaves = kQkThreads / 64;

__device__ __forceinline__ void load8(const __bf16* p, float (&x)[8]) {
  const bf16x8 v = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
}

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

__device__ __forceinline__ void store8(__bf16* p, const float (&x)[8]) {
  bf16x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (__bf16)x[e];
  *reinterpret_cast<bf16x8*>(p) = v;
}

__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// Norm weights have any alignment that their type has.
__device__ __forceinline__ void load_weight8(const void* w, bool f32, int i, float (&out)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    out[e] = f32 ? static_cast<const float*>(w)[i + e] : (float)static_cast<const __bf16*>(w)[i + e];
}

__device__ __forceinline__ float group_sum(float x, int LP) {
  for (int off = LP >> 1; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}

// One group of LP lanes per (token, head); heads are the Hq query, Hkv key
// and Hkv value heads of the packed row, in that order.
template <typename T>
__global__ __launch_bounds__(kQkThreads) void qk_norm_rope_kernel(QkNormArgs a) {
  const uint32_t item = blockIdx.x * kQkThreads + threadIdx.x;
  const uint32_t heads = a.Hq + 2 * a.Hkv;
  const uint32_t row = item >> a.lp_log2;
  const uint32_t n = row / heads;
  if (n >= (uint32_t)(a.B * a.T)) return;  // whole groups: the shuffles below stay within one
  const int head = row - n * heads;
  const int b = n / (uint32_t)a.T, t = n - b * a.T;
  const int LP = 1 << a.lp_log2, half = a.D >> 1;
  const int j8 = 8 * (item & (LP - 1));
  const bool in = j8 < half;

  // The position, its cache row where there is a cache, and whether a row of
  // the same position follows (the later one is kept).
  int64_t p = a.pos0 + t;
  bool stored = true;
  if (a.pos) {
    const int64_t* pos = a.pos + b * a.pos_sb;
    p = pos[t];
    for (int u = t + 1; u < a.T; ++u) stored = stored && pos[u] != p;
  }
  const bool known = p >= 0 && p < a.max_pos;

  const int which = head < a.Hq ? 0 : (head < a.Hq + a.Hkv ? 1 : 2);
  const int h = which == 0 ? head : (which == 1 ? head - a.Hq : head - a.Hq - a.Hkv);
  const T* src = static_cast<const T*>(a.packed) + b * a.p_sb + (int64_t)t * a.p_st +
                 (int64_t)head * a.D + j8;
  float x1[8] = {}, x2[8] = {};
  if (in) {
    load8(src, x1);
    load8(src + half, x2);
  }
  if (which < 2) {
    float w1[8] = {}, w2[8] = {}, c[8] = {}, s[8] = {};
    if (in) {
      const void* w = which ? a.kw : a.qw;
      load_weight8(w, a.w_f32, j8, w1);
      load_weight8(w, a.w_f32, half + j8, w2);
      if (known) {
        load8(a.cos + p * half + j8, c);
        load8(a.sin + p * half + j8, s);
      }
    }
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(x1[e], x1[e], fmaf(x2[e], x2[e], ss));
    const float r = rsqrtf(group_sum(ss, LP) / (float)a.D + a.eps);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y1 = x1[e] * r * w1[e], y2 = x2[e] * r * w2[e];
      x1[e] = fmaf(y1, c[e], y2 * s[e]);
      x2[e] = fmaf(y2, c[e], -(y1 * s[e]));
    }
  }
  if (!in) return;
  const TensorView& o = a.ops[which];
  int64_t at = t;
  if (a.append) {
    if (!known) {  // no table row: a query of zeros, nothing into the cache
      if (which) return;
#pragma unroll
      for (int e = 0; e < 8; ++e) x1[e] = x2[e] = 0.f;
    } else if (which) {
      if (!stored) return;
      at = p;
    }
  }
  T* dst = static_cast<T*>(o.data) + b * o.sb + h * o.sh + at * o.st + j8;
  store8(dst, x1);
  store8(dst + half, x2);
}

// Each work-group takes rounds of kQkThreads / LP rows of one kind (query, key
// or value heads, by block index), so that a lane holds the same columns
// throughout and its share of dw stays in registers; per work-group the shares
// are summed by shuffles and through LDS into part[group][D].
template <typename T>
__global__ __launch_bounds__(kQkThreads) void qk_norm_rope_bwd_kernel(QkNormBwdArgs a) {
  __shared__ float red[kQkWaves][2 * 256];
  int which = 0;
  uint32_t group = blockIdx.x;
  while (group >= (uint32_t)a.groups[which]) group -= a.groups[which++];
  const uint32_t H = which ? a.Hkv : a.Hq;
  const int head0 = which == 0 ? 0 : (which == 1 ? a.Hq : a.Hq + a.Hkv);
  const int LP = 1 << a.lp_log2, half = a.D >> 1;
  const int j8 = 8 * (threadIdx.x & (LP - 1));
  const bool in = j8 < half;
  const uint32_t rows = (uint32_t)a.B * a.T * H, per = kQkThreads >> a.lp_log2;
  const TensorView& g = a.ops[which];

  float w1[8] = {}, w2[8] = {}, acc1[8] = {}, acc2[8] = {};
  if (in && which < 2) {
    load_weight8(which ? a.kw : a.qw, a.w_f32, j8, w1);
    load_weight8(which ? a.kw : a.qw, a.w_f32, half + j8, w2);
  }
  for (uint32_t r0 = group * per; r0 < rows; r0 += a.groups[which] * per) {
    const uint32_t row = r0 + (threadIdx.x >> a.lp_log2);
    const bool ok = in && row < rows;
    const uint32_t n = row / H, h = row - n * H;
    const int b = n / (uint32_t)a.T, t = n - b * a.T;
    float d1[8] = {}, d2[8] = {}, x1[8] = {}, x2[8] = {}, c[8] = {}, s[8] = {};
    const int64_t at = b * a.p_sb + (int64_t)t * a.p_st + (int64_t)(head0 + h) * a.D + j8;
    const int64_t to =
        ((int64_t)n * (a.Hq + 2 * a.Hkv) + head0 + h) * a.D + j8;
    if (ok) {
      const T* src = static_cast<const T*>(g.data) + b * g.sb + h * g.sh + (int64_t)t * g.st + j8;
      load8(src, d1);
      load8(src + half, d2);
    }
    if (which < 2) {
      if (ok) {
        const T* x = static_cast<const T*>(a.packed) + at;
        load8(x, x1);
        load8(x + half, x2);
        load8(a.cos + (int64_t)(a.pos0 + t) * half + j8, c);
        load8(a.sin + (int64_t)(a.pos0 + t) * half + j8, s);
      }
      float ss = 0.f, dot = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y1 = fmaf(d1[e], c[e], -(d2[e] * s[e]));
        const float y2 = fmaf(d2[e], c[e], d1[e] * s[e]);
        d1[e] = y1;
        d2[e] = y2;
        ss = fmaf(x1[e], x1[e], fmaf(x2[e], x2[e], ss));
        dot = fmaf(y1 * w1[e], x1[e], fmaf(y2 * w2[e], x2[e], dot));
      }
      ss = group_sum(ss, LP);
      dot = group_sum(dot, LP);
      const float r = rsqrtf(ss / (float)a.D + a.eps);
      const float m = dot * r / (float)a.D;  // mean(g n)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float n1 = x1[e] * r, n2 = x2[e] * r;
        if (ok) {
          acc1[e] = fmaf(d1[e], n1, acc1[e]);
          acc2[e] = fmaf(d2[e], n2, acc2[e]);
        }
        d1[e] = r * (d1[e] * w1[e] - n1 * m);
        d2[e] = r * (d2[e] * w2[e] - n2 * m);
      }
    }
    if (ok) {
      T* dst = static_cast<T*>(a.dpacked) + to;
      store8(dst, d1);
      store8(dst + half, d2);
    }
  }
  if (which == 2) return;
  // The lanes with the same columns: 64 / LP in a wave, then the waves.
  for (int off = LP; off < 64; off <<= 1) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      acc1[e] += __shfl_xor(acc1[e], off, 64);
      acc2[e] += __shfl_xor(acc2[e], off, 64);
    }
  }
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) < LP && in) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      red[wave][j8 + e] = acc1[e];
      red[wave][half + j8 + e] = acc2[e];
    }
  }
  __syncthreads();
  float* part = a.part + ((int64_t)(which ? a.groups[0] : 0) + group) * a.D;
  for (int i = threadIdx.x; i < a.D; i += kQkThreads) {
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < kQkWaves; ++v) sum += red[v][i];
    part[i] = sum;
  }
}

// dw[i] = sum over the work-groups of their shares, in a fixed order: 16 waves
// per 64 columns, wave s summing groups s, s + 16, ..., then the waves.
constexpr int kDwWaves = 16;
__global__ __launch_bounds__(64 * kDwWaves) void qk_norm_dw_kernel(const float* part, int nq,
                                                                   int nk, int D, void* dqw,
                                                                   void* dkw, bool w_f32) {
  __shared__ float red[kDwWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = blockIdx.x * 64 + lane;
  const int first = blockIdx.y ? nq : 0, count = blockIdx.y ? nk : nq;
  float sum = 0.f;
  if (col < D) {
#pragma unroll 8
    for (int g = wave; g < count; g += kDwWaves) sum += part[(int64_t)(first + g) * D + col];
  }
  red[wave][lane] = sum;
  __syncthreads();
  if (wave || col >= D) return;
  float total = 0.f;
#pragma unroll
  for (int v = 0; v < kDwWaves; ++v) total += red[v][lane];
  void* dw = blockIdx.y ? dkw : dqw;
  if (w_f32)
    static_cast<float*>(dw)[col] = total;
  else
    static_cast<__bf16*>(dw)[col] = (__bf16)total;
}

int lanes_log2(int D) {
  int l = 0;
  while ((16 << l) < D) ++l;
  return l;
}

// Work-groups for `rows` head rows: four rounds each, at most 1024.
int groups_of(int64_t rows, int lp_log2) {
  const int64_t per = kQkThreads >> lp_log2;
  const int64_t n = (rows + 4 * per - 1) / (4 * per);
  return (int)(n < 1024 ? n : 1024);
}

}  // namespace

int64_t qk_norm_items(int64_t B, int64_t T, int Hq, int Hkv, int D) {
  return (B * T * (Hq + 2 * (int64_t)Hkv)) << lanes_log2(D);
}

int qk_norm_bwd_groups(int B, int T, int Hq, int Hkv, int D) {
  const int l = lanes_log2(D);
  return groups_of((int64_t)B * T * Hq, l) + groups_of((int64_t)B * T * Hkv, l);
}

hipError_t launch_qk_norm_rope(QkNormArgs a, bool f32, hipStream_t stream) {
  a.lp_log2 = lanes_log2(a.D);
  const int64_t items = qk_norm_items(a.B, a.T, a.Hq, a.Hkv, a.D);
  if (items == 0) return hipSuccess;
  const dim3 grid((unsigned)((items + kQkThreads - 1) / kQkThreads));
  if (f32)
    hipLaunchKernelGGL(qk_norm_rope_kernel<float>, grid, dim3(kQkThreads), 0, stream, a);
  else
    hipLaunchKernelGGL(qk_norm_rope_kernel<__bf16>, grid, dim3(kQkThreads), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_qk_norm_rope_bwd(QkNormBwdArgs a, bool f32, void* dqw, void* dkw,
                                   hipStream_t stream) {
  a.lp_log2 = lanes_log2(a.D);
  const int64_t n = (int64_t)a.B * a.T;
  a.groups[0] = groups_of(n * a.Hq, a.lp_log2);
  a.groups[1] = groups_of(n * a.Hkv, a.lp_log2);
  a.groups[2] = a.groups[1];
  const int total = a.groups[0] + 2 * a.groups[1];
  if (total) {
    if (f32)
      hipLaunchKernelGGL(qk_norm_rope_bwd_kernel<float>, dim3(total), dim3(kQkThreads), 0, stream, a);
    else
      hipLaunchKernelGGL(qk_norm_rope_bwd_kernel<__bf16>, dim3(total), dim3(kQkThreads), 0, stream,
                         a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(qk_norm_dw_kernel, dim3((unsigned)((a.D + 63) / 64), 2), dim3(64 * kDwWaves),
                     0, stream, a.part, a.groups[0], a.groups[1], a.D, dqw, dkw, a.w_f32);
  return hipGetLastError();
}

}  // namespace t2t
