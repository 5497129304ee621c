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
// rotation pairs sit in one lane and the mean is log2 LP shuffles.  A wave takes
// whole tokens -- one, or as many as its groups hold the query heads of --
// and their query, key and value heads one after the other, so that the lanes
// load a token's angles once for all heads.  16384 tokens of 36 heads of 64,
// bf16: 33 us, 4.5 TB/s of the 5.1 of a large copy (one head row a group,
// whatever its token, read the angles with every row: 48 us); the backward, two
// launches, 42 us, 4.8 TB/s.
#include "attn_kernels.h"

namespace t2t {

namespace {

constexpr int kQkThreads = 256;
constexpr int kQkWaves = kQkThreads / 64;
constexpr int kBwdThreads = 256;
constexpr int kBwdWaves = kBwdThreads / 64;
constexpr int kBwdGroups = 1024;  // work-groups of the backward: four on each CU

// Eight values as they are stored.
struct Raw16 { bf16x8 v; };
struct Raw32 { float4 a, b; };
__device__ __forceinline__ Raw16 raw8(const __bf16* p) {
  return {*reinterpret_cast<const bf16x8*>(p)};
}
__device__ __forceinline__ Raw32 raw8(const float* p) {
  return {reinterpret_cast<const float4*>(p)[0], reinterpret_cast<const float4*>(p)[1]};
}
__device__ __forceinline__ void values(const Raw16& r, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (float)r.v[e];
}
__device__ __forceinline__ void values(const Raw32& r, float (&x)[8]) {
  x[0] = r.a.x; x[1] = r.a.y; x[2] = r.a.z; x[3] = r.a.w;
  x[4] = r.b.x; x[5] = r.b.y; x[6] = r.b.z; x[7] = r.b.w;
}
template <typename T>
using RawOf = decltype(raw8(static_cast<const T*>(nullptr)));

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) { values(raw8(p), x); }

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

__device__ __forceinline__ void load_weight8(const void* w, bool f32, int i, float (&out)[8]) {
  if (f32)
    load8(static_cast<const float*>(w) + i, out);
  else
    load8(static_cast<const __bf16*>(w) + i, out);
}

__device__ __forceinline__ float group_sum(float x, int LP) {
  for (int off = LP >> 1; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}

// A lane's place in a wave that works on `tokens` tokens: the token among
// them, the first head of its group, how many heads further the next one is.
struct Place {
  int token, head, step, j8, half;
  bool in;  // the lane has columns
  __device__ Place(int lp_log2, int tokens_log2, int D) {
    const int lane = threadIdx.x & 63, group = lane >> lp_log2;
    const int per = 6 - lp_log2 - tokens_log2;  // log2 of the groups a token
    token = group >> per;
    head = group & ((1 << per) - 1);
    step = 1 << per;
    half = D >> 1;
    j8 = 8 * (lane & ((1 << lp_log2) - 1));
    in = j8 < half;
  }
};

template <typename T>
__global__ __launch_bounds__(kQkThreads, sizeof(T) == 4 ? 3 : 4)
void qk_norm_rope_kernel(QkNormArgs a) {
  const Place at(a.lp_log2, a.tokens_log2, a.D);
  const int LP = 1 << a.lp_log2, half = at.half, j8 = at.j8;
  const int64_t tokens = (int64_t)a.B * a.T;
  const int64_t stride = (int64_t)gridDim.x * kQkWaves << a.tokens_log2;
  int64_t n0 = ((int64_t)blockIdx.x * kQkWaves + (threadIdx.x >> 6)) << a.tokens_log2;
  for (; n0 < tokens; n0 += stride) {
    const uint32_t n = (uint32_t)n0 + at.token;  // (at most 2^31 tokens)
    const bool ok = at.in && n < tokens;
    const int b = n / (uint32_t)a.T, t = n - b * a.T;
    const T* src = static_cast<const T*>(a.packed) + b * a.p_sb + (int64_t)t * a.p_st + j8;

    // The first head row of each kind: all loads in flight at once.
    const int heads[3] = {a.Hq, a.Hkv, a.Hkv};
    RawOf<T> r1[3] = {}, r2[3] = {};
    float c[8] = {}, s[8] = {};
    int first = 0;
#pragma unroll
    for (int w = 0; w < 3; ++w) {
      if (ok && at.head < heads[w]) {
        const T* row = src + (int64_t)(first + at.head) * a.D;
        r1[w] = raw8(row);
        r2[w] = raw8(row + half);
      }
      first += heads[w];
    }
    // The position, and whether a row of the same position follows (the later
    // one is kept).
    int64_t p = a.pos0 + t;
    bool stored = true;
    if (a.pos && ok) {
      const int64_t* pos = a.pos + b * a.pos_sb;
      p = pos[t];
      for (int u = t + 1; u < a.T; ++u) stored = stored && pos[u] != p;
    }
    const bool known = p >= 0 && p < a.max_pos;
    if (ok && known) {
      load8(a.cos + p * half + j8, c);
      load8(a.sin + p * half + j8, s);
    }
    first = 0;
#pragma unroll
    for (int w = 0; w < 3; ++w) {
      float w1[8] = {}, w2[8] = {};
      if (w < 2 && at.in) {
        load_weight8(w ? a.kw : a.qw, a.w_f32, j8, w1);
        load_weight8(w ? a.kw : a.qw, a.w_f32, half + j8, w2);
      }
      for (int h0 = 0; h0 < heads[w]; h0 += at.step) {
        const int h = h0 + at.head;
        const bool row_ok = ok && h < heads[w];
        if (h0) {
          r1[w] = r2[w] = RawOf<T>{};
          if (row_ok) {
            const T* row = src + (int64_t)(first + h) * a.D;
            r1[w] = raw8(row);
            r2[w] = raw8(row + half);
          }
        }
        float x1[8], x2[8];
        values(r1[w], x1);
        values(r2[w], x2);
        if (w < 2) {
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
        if (!row_ok) continue;
        int64_t to = t;
        if (a.append) {
          if (!known) {  // no table row: a query of zeros, nothing into the cache
            if (w) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e) x1[e] = x2[e] = 0.f;
          } else if (w) {
            if (!stored) continue;
            to = p;
          }
        }
        const TensorView& o = a.ops[w];
        T* dst = static_cast<T*>(o.data) + b * o.sb + h * o.sh + to * o.st + j8;
        store8(dst, x1);
        store8(dst + half, x2);
      }
      first += heads[w];
    }
  }
}

// What the backward loads of a head row.
template <typename T>
struct BwdRow {
  RawOf<T> d1, d2, x1, x2;
  uint32_t n, h;  // token, head
  int t;
  bool ok;
};

// Each work-group takes rounds of kBwdThreads / LP rows of one kind (query, key
// or value heads, by block index), so that a lane holds the same columns
// throughout and its share of dw stays in registers; a row's loads are issued
// while the row before is computed.  Per work-group the shares are summed by
// shuffles and through LDS into part[group][D].  (Query and key heads in one
// wave, with the angles loaded once a token: 168 registers, three waves a SIMD,
// 61 us where this takes 41.)
template <typename T, bool Norm>
__device__ __forceinline__ void bwd_rows(const QkNormBwdArgs& a, int which, uint32_t group,
                                         float (&acc1)[8], float (&acc2)[8]) {
  const uint32_t H = which ? a.Hkv : a.Hq, T_ = a.T;
  const int head0 = which == 0 ? 0 : (which == 1 ? a.Hq : a.Hq + a.Hkv);
  const int LP = 1 << a.lp_log2, half = a.D >> 1;
  const int j8 = 8 * (threadIdx.x & (LP - 1));
  const bool in = j8 < half;
  const uint32_t per = kBwdThreads >> a.lp_log2, step = a.groups[which] * per;
  const int64_t rows = (int64_t)a.B * T_ * H;
  const TensorView& g = a.ops[which];
  const auto load = [&](int64_t r0) {
    BwdRow<T> row{};
    const int64_t r = r0 + (threadIdx.x >> a.lp_log2);
    row.ok = in && r < rows;
    if (row.ok) {
      row.n = (uint32_t)(r / H);
      row.h = (uint32_t)(r - (int64_t)row.n * H);
      const uint32_t b = row.n / T_;
      row.t = row.n - b * T_;
      const T* d = static_cast<const T*>(g.data) + b * g.sb + row.h * g.sh + row.t * g.st + j8;
      row.d1 = raw8(d);
      row.d2 = raw8(d + half);
      if (Norm) {
        const T* x = static_cast<const T*>(a.packed) + b * a.p_sb + row.t * a.p_st +
                     (int64_t)(head0 + row.h) * a.D + j8;
        row.x1 = raw8(x);
        row.x2 = raw8(x + half);
      }
    }
    return row;
  };
  float w1[8] = {}, w2[8] = {};
  if (Norm && in) {
    load_weight8(which ? a.kw : a.qw, a.w_f32, j8, w1);
    load_weight8(which ? a.kw : a.qw, a.w_f32, half + j8, w2);
  }
  int64_t r0 = (int64_t)group * per;
  BwdRow<T> next = load(r0);
  for (; r0 < rows; r0 += step) {
    const BwdRow<T> row = next;
    next = load(r0 + step);
    float d1[8], d2[8];
    values(row.d1, d1);
    values(row.d2, d2);
    if (Norm) {
      float x1[8], x2[8], c[8] = {}, s[8] = {};
      values(row.x1, x1);
      values(row.x2, x2);
      if (row.ok) {
        load8(a.cos + (int64_t)(a.pos0 + row.t) * half + j8, c);
        load8(a.sin + (int64_t)(a.pos0 + row.t) * half + j8, s);
      }
      float ss = 0.f, dot = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        ss = fmaf(x1[e], x1[e], fmaf(x2[e], x2[e], ss));
        const float y1 = fmaf(d1[e], c[e], -(d2[e] * s[e]));
        const float y2 = fmaf(d2[e], c[e], d1[e] * s[e]);
        d1[e] = y1;
        d2[e] = y2;
        dot = fmaf(y1 * w1[e], x1[e], fmaf(y2 * w2[e], x2[e], dot));
      }
      ss = group_sum(ss, LP);
      dot = group_sum(dot, LP);
      const float r = rsqrtf(ss / (float)a.D + a.eps);
      const float m = dot * r / (float)a.D;  // mean(g n)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float n1 = x1[e] * r, n2 = x2[e] * r;
        if (row.ok) {  // (0 times the r of no row is not a number at eps = 0)
          acc1[e] = fmaf(d1[e], n1, acc1[e]);
          acc2[e] = fmaf(d2[e], n2, acc2[e]);
        }
        d1[e] = r * (d1[e] * w1[e] - n1 * m);
        d2[e] = r * (d2[e] * w2[e] - n2 * m);
      }
    }
    if (row.ok) {
      T* out = static_cast<T*>(a.dpacked) +
               ((int64_t)row.n * (a.Hq + 2 * a.Hkv) + head0 + row.h) * a.D + j8;
      store8(out, d1);
      store8(out + half, d2);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kBwdThreads, sizeof(T) == 4 ? 3 : 4)
void qk_norm_rope_bwd_kernel(QkNormBwdArgs a) {
  __shared__ float red[kBwdWaves][2 * 256];
  int which = 0;
  uint32_t group = blockIdx.x;
  while (group >= (uint32_t)a.groups[which]) group -= a.groups[which++];
  float acc1[8] = {}, acc2[8] = {};
  if (which == 2) {
    bwd_rows<T, false>(a, which, group, acc1, acc2);
    return;
  }
  bwd_rows<T, true>(a, which, group, acc1, acc2);
  // The lanes with the same columns: 64 / LP in a wave, then the waves.
  const int LP = 1 << a.lp_log2, half = a.D >> 1, wave = threadIdx.x >> 6;
  const int j8 = 8 * (threadIdx.x & (LP - 1));
  for (int off = LP; off < 64; off <<= 1) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      acc1[e] += __shfl_xor(acc1[e], off, 64);
      acc2[e] += __shfl_xor(acc2[e], off, 64);
    }
  }
  if ((threadIdx.x & 63) < LP && j8 < half) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      red[wave][j8 + e] = acc1[e];
      red[wave][half + j8 + e] = acc2[e];
    }
  }
  __syncthreads();
  float* part = a.part + ((int64_t)(which ? a.groups[0] : 0) + group) * a.D;
  for (int i = threadIdx.x; i < a.D; i += kBwdThreads) {
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < kBwdWaves; ++v) sum += red[v][i];
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

// log2 of the tokens a wave takes: as many as its groups hold the query heads of.
int tokens_log2(int lp_log2, int Hq) {
  int l = 0;
  while ((Hq << lp_log2 << (l + 1)) <= 64) ++l;
  return l;
}

// The backward's work-groups for the query, key and value rows: shares of
// kBwdGroups in proportion to their rounds.
void bwd_groups(int64_t tokens, int Hq, int Hkv, int D, int (&groups)[3]) {
  const int64_t per = kBwdThreads >> lanes_log2(D);
  const auto rounds = [&](int64_t heads) { return (tokens * heads + per - 1) / per; };
  const int64_t all = rounds(Hq) + 2 * rounds(Hkv);
  const int64_t each = (all + kBwdGroups - 1) / kBwdGroups;  // rounds a work-group
  for (int w = 0; w < 3; ++w)
    groups[w] = each ? (int)((rounds(w ? Hkv : Hq) + each - 1) / each) : 0;
}

}  // namespace

int qk_norm_bwd_groups(int B, int T, int Hq, int Hkv, int D) {
  int groups[3];
  bwd_groups((int64_t)B * T, Hq, Hkv, D, groups);
  return groups[0] + groups[1];
}

hipError_t launch_qk_norm_rope(QkNormArgs a, bool f32, hipStream_t stream) {
  a.lp_log2 = lanes_log2(a.D);
  a.tokens_log2 = tokens_log2(a.lp_log2, a.Hq);
  const int64_t tokens = (int64_t)a.B * a.T;
  if (tokens == 0) return hipSuccess;
  const int64_t per = (int64_t)kQkWaves << a.tokens_log2, groups = (tokens + per - 1) / per;
  const dim3 grid((unsigned)(groups < 1 << 20 ? groups : 1 << 20));
  if (f32)
    hipLaunchKernelGGL(qk_norm_rope_kernel<float>, grid, dim3(kQkThreads), 0, stream, a);
  else
    hipLaunchKernelGGL(qk_norm_rope_kernel<__bf16>, grid, dim3(kQkThreads), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_qk_norm_rope_bwd(QkNormBwdArgs a, bool f32, void* dqw, void* dkw,
                                   hipStream_t stream) {
  a.lp_log2 = lanes_log2(a.D);
  bwd_groups((int64_t)a.B * a.T, a.Hq, a.Hkv, a.D, a.groups);
  const int total = a.groups[0] + a.groups[1] + a.groups[2];
  if (total) {
    if (f32)
      hipLaunchKernelGGL(qk_norm_rope_bwd_kernel<float>, dim3(total), dim3(kBwdThreads), 0, stream,
                         a);
    else
      hipLaunchKernelGGL(qk_norm_rope_bwd_kernel<__bf16>, dim3(total), dim3(kBwdThreads), 0,
                         stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(qk_norm_dw_kernel, dim3((unsigned)((a.D + 63) / 64), 2), dim3(64 * kDwWaves),
                     0, stream, a.part, a.groups[0], a.groups[1], a.D, dqw, dkw, a.w_f32);
  return hipGetLastError();
}

}  // namespace t2t
