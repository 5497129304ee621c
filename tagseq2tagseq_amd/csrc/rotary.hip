// Attention-module prologue with any rotary form: the packed projection rows
// split into query, key and value heads, the first R dimensions of every query
// and key head rotated, the others and the values copied; and the transpose of
// that map for the backward.
//
// For a head row x of D values at position p, pair i < R / 2 of its first R
// dimensions is (a, b) = (x[i], x[i + R/2]) (half-split) or (x[2i], x[2i + 1])
// (interleaved), and becomes
//   a' = a cos[p][i] + b sin[p][i],   b' = b cos[p][i] - a sin[p][i],
// in fp32 with one rounding; the backward rotates by the negative angle.
// Positions are pos0 + t, or read per token (documents of a packed row count
// from their own starts); one without a table row gives query and key rows of
// zeros, and zeros for their gradient.
//
// HBM bound: each pass reads and writes every packed row once.  A unit is 16
// values of a head row in two runs of 8, both ends of the pairs among them:
// columns (8j .., R/2 + 8j ..) of the rotated part half-split, 16 columns side
// by side otherwise.  U = D / 16 lanes hold a head row; a lane keeps its j, and
// so its eight angles, over all heads of a token, and a wave takes one token
// (or as many as its lanes hold whole), four units' loads in flight a lane
// (two: 39 to 41 us where four take 35 to 37; three: the same as four).  16384
// tokens of 36 heads of 64, bf16: forward 34.7 us, backward 37.4, 4.4 and 4.1 TB/s
// of a large copy's 5.15; 28.9 where the last-level cache holds the input, as
// behind the projection.  Stores that bypass the caches take 29 from memory too,
// and the attention that reads q, k and v next then loses more than that (49.0 to
// 53.2 us at a window of 512): not used.
#include "attn_kernels.h"

namespace t2t {

namespace {

constexpr int kRotThreads = 256;
constexpr int kRotWaves = kRotThreads / 64;
constexpr int kAhead = 4;  // units a lane loads before it stores the first

struct Eight16 { bf16x8 v; };
struct Eight32 { float4 a, b; };
__device__ __forceinline__ Eight16 load_eight(const __bf16* p) {
  return {*reinterpret_cast<const bf16x8*>(p)};
}
__device__ __forceinline__ Eight32 load_eight(const float* p) {
  return {reinterpret_cast<const float4*>(p)[0], reinterpret_cast<const float4*>(p)[1]};
}
__device__ __forceinline__ void store_eight(__bf16* p, const Eight16& r) {
  *reinterpret_cast<bf16x8*>(p) = r.v;
}
__device__ __forceinline__ void store_eight(float* p, const Eight32& r) {
  reinterpret_cast<float4*>(p)[0] = r.a;
  reinterpret_cast<float4*>(p)[1] = r.b;
}
__device__ __forceinline__ void unpack(const Eight16& r, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (float)r.v[e];
}
__device__ __forceinline__ void unpack(const Eight32& r, float (&x)[8]) {
  x[0] = r.a.x; x[1] = r.a.y; x[2] = r.a.z; x[3] = r.a.w;
  x[4] = r.b.x; x[5] = r.b.y; x[6] = r.b.z; x[7] = r.b.w;
}
__device__ __forceinline__ void pack(const float (&x)[8], Eight16& r) {
#pragma unroll
  for (int e = 0; e < 8; ++e) r.v[e] = (__bf16)x[e];
}
__device__ __forceinline__ void pack(const float (&x)[8], Eight32& r) {
  r.a = make_float4(x[0], x[1], x[2], x[3]);
  r.b = make_float4(x[4], x[5], x[6], x[7]);
}
template <typename T>
using EightOf = decltype(load_eight(static_cast<const T*>(nullptr)));

template <bool Inter>
__device__ __forceinline__ void turn(float (&x)[8], float (&y)[8], const float (&c)[8],
                                     const float (&s)[8]) {
  if constexpr (Inter) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float a = x[2 * e], b = x[2 * e + 1], d = y[2 * e], f = y[2 * e + 1];
      x[2 * e] = fmaf(a, c[e], b * s[e]);
      x[2 * e + 1] = fmaf(b, c[e], -(a * s[e]));
      y[2 * e] = fmaf(d, c[4 + e], f * s[4 + e]);
      y[2 * e + 1] = fmaf(f, c[4 + e], -(d * s[4 + e]));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = x[e], b = y[e];
      x[e] = fmaf(a, c[e], b * s[e]);
      y[e] = fmaf(b, c[e], -(a * s[e]));
    }
  }
}

template <typename T, bool Inter, bool Back>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(RotaryArgs a) {
  const int U = a.D >> 4;
  const int lane = threadIdx.x & 63;
  const int group = lane / U, j = lane - group * U;
  const int token = group / a.per_token, head0 = group - token * a.per_token;
  const bool in = token < a.tokens;  // (lanes past the last whole group take none)
  const int heads = a.Hq + 2 * a.Hkv, rotated = a.Hq + a.Hkv;
  const bool turns = 16 * j < a.R;
  const int o1 = !Inter && turns ? 8 * j : 16 * j;
  const int o2 = !Inter && turns ? (a.R >> 1) + 8 * j : 16 * j + 8;
  const int64_t total = (int64_t)a.B * a.T;
  const int64_t stride = (int64_t)gridDim.x * kRotWaves * a.tokens;
  int64_t n0 = ((int64_t)blockIdx.x * kRotWaves + (threadIdx.x >> 6)) * a.tokens;
  for (; n0 < total; n0 += stride) {
    const uint32_t n = (uint32_t)n0 + token;  // (at most 2^31 tokens)
    if (!in || n >= total) continue;
    const int b = n / (uint32_t)a.T, t = n - b * a.T;
    T* row = static_cast<T*>(a.packed) + b * a.p_sb + (int64_t)t * a.p_st;
    // head h of the packed row in its view
    const auto view = [&](int h) {
      const int w = h < a.Hq ? 0 : h < rotated ? 1 : 2;
      const TensorView& o = a.ops[w];
      return static_cast<T*>(o.data) + b * o.sb + (int64_t)t * o.st +
             (h - (w == 0 ? 0 : w == 1 ? a.Hq : rotated)) * o.sh;
    };
    EightOf<T> r1[kAhead], r2[kAhead];
    const auto load = [&](int h0) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int h = h0 + i * a.per_token;
        if (h < heads) {
          const T* src = Back ? view(h) : row + (int64_t)h * a.D;
          r1[i] = load_eight(src + o1);
          r2[i] = load_eight(src + o2);
        }
      }
    };
    load(head0);  // (ahead of the position, which the angles wait for)
    const int64_t p = a.pos ? a.pos[b * a.pos_sb + t] : (int64_t)a.pos0 + t;
    const bool known = p >= 0 && p < a.rows;
    float c[8] = {}, s[8] = {};
    if (turns && known) {
      unpack(load_eight(a.cos + p * (a.R >> 1) + 8 * j), c);
      unpack(load_eight(a.sin + p * (a.R >> 1) + 8 * j), s);
      if constexpr (Back) {
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] = -s[e];
      }
    }
    for (int h0 = head0; h0 < heads; h0 += kAhead * a.per_token) {
      if (h0 != head0) load(h0);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int h = h0 + i * a.per_token;
        if (h >= heads) continue;
        if (h < rotated) {
          float x[8], y[8];
          unpack(r1[i], x);
          unpack(r2[i], y);
          if (turns) turn<Inter>(x, y, c, s);
          if (!known) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = y[e] = 0.f;
          }
          if (turns || !known) {
            pack(x, r1[i]);
            pack(y, r2[i]);
          }
        }
        T* dst = Back ? row + (int64_t)h * a.D : view(h);
        store_eight(dst + o1, r1[i]);
        store_eight(dst + o2, r2[i]);
      }
    }
  }
}

template <typename T, bool Back>
void start(const RotaryArgs& a, unsigned grid, hipStream_t stream) {
  if (a.interleaved)
    hipLaunchKernelGGL((rotary_kernel<T, true, Back>), dim3(grid), dim3(kRotThreads), 0, stream,
                       a);
  else
    hipLaunchKernelGGL((rotary_kernel<T, false, Back>), dim3(grid), dim3(kRotThreads), 0, stream,
                       a);
}

}  // namespace

hipError_t launch_rotary(RotaryArgs a, bool f32, bool backward, hipStream_t stream) {
  const int64_t total = (int64_t)a.B * a.T;
  if (total == 0) return hipSuccess;
  const int heads = a.Hq + 2 * a.Hkv, groups = 64 / (a.D / 16);
  a.tokens = groups > heads ? groups / heads : 1;
  a.per_token = groups / a.tokens;
  const int64_t per = (int64_t)kRotWaves * a.tokens;
  const int64_t blocks = (total + per - 1) / per;
  const unsigned grid = (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20));
  if (f32)
    backward ? start<float, true>(a, grid, stream) : start<float, false>(a, grid, stream);
  else
    backward ? start<__bf16, true>(a, grid, stream) : start<__bf16, false>(a, grid, stream);
  return hipGetLastError();
}

}  // namespace t2t
