// Distillation of a linear head from a teacher's top logits: the loss of each
// row of student logits z (V columns) and its gradient, in one reading of the
// row.  With the teacher's logits t_k at the columns i_k (slots of i_k < 0 are
// empty), temperature T and weight a:
//   p   = softmax over the row's slots of t / T,   q = softmax(z / T)
//   KD  = sum_k p_k (ln p_k - ln q(i_k))            (0 in a row without slots)
//   loss = a T^2 KD + (1 - a) (logsumexp(z) - z[target])
//   dloss/dz_j = a T ([slots] q_j - sum over k with i_k = j of p_k)
//                + (1 - a) (softmax(z)_j - [j = target])
// times the caller's scale.  Rows whose target is ignore_index give loss 0 and
// a zero gradient (their logits are not read); a target outside [0, V) or a
// column i_k >= V gives the loss NaN and a zero gradient.
//
// HBM bound: the row is read once and its gradient written once.  The row
// stays in the registers of a work-group, packed as it was read.  Differences
// z - max are formed first and multiplied then, so that rows of the lowest
// finite values keep their softmax.  Sums are fp32; KD is computed from
//   sum_k w_k ((t_k - max t) - (z(i_k) - max z)) / (T sum w) - ln sum w + ln sum_j
// with w_k = e^((t_k - max t) / T), whose terms are small where the result is.
// The gradient is first written without the teacher's and the target's terms;
// behind a barrier, one thread for each of those columns writes its value
// again, the slots of equal columns added in their order.  The gradient may
// overwrite the logits: everything is read before the barriers ahead of the
// first write.
//
// Addresses: rows start anywhere on their type (V = 50257 columns of bf16 have
// every second row off a 4-byte boundary); 16-byte pieces are read and written
// at that alignment, which global memory instructions allow.
#include "attn_kernels.h"

namespace t2t {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxSlots = kDistillMaxSlots;

template <typename T>
struct Elem;
template <>
struct Elem<__bf16> {
  static constexpr int kVec = 8;
  static constexpr uint32_t kNone = 0xff80ff80u;  // -inf
  struct __attribute__((packed, aligned(2))) Piece { uint32_t w[4]; };
  __device__ static void unpack(const Piece& p, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = __uint_as_float(p.w[e] << 16);
      x[2 * e + 1] = __uint_as_float(p.w[e] & 0xffff0000u);
    }
  }
  __device__ static void pack(const float (&x)[8], Piece& p) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const __bf16 lo = (__bf16)x[2 * e], hi = (__bf16)x[2 * e + 1];
      p.w[e] = (uint32_t)__builtin_bit_cast(uint16_t, lo) |
               ((uint32_t)__builtin_bit_cast(uint16_t, hi) << 16);
    }
  }
};
template <>
struct Elem<float> {
  static constexpr int kVec = 4;
  static constexpr uint32_t kNone = 0xff800000u;
  struct __attribute__((packed, aligned(4))) Piece { uint32_t w[4]; };
  __device__ static void unpack(const Piece& p, float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(p.w[e]);
  }
  __device__ static void pack(const float (&x)[4], Piece& p) {
#pragma unroll
    for (int e = 0; e < 4; ++e) p.w[e] = __float_as_uint(x[e]);
  }
};

// A row of V columns: V / VEC whole pieces, and the columns behind them, which
// the first V % VEC threads hold one each (Tail).
template <typename T>
__device__ __forceinline__ typename Elem<T>::Piece load_piece(const T* row, uint32_t i) {
  // (an unsigned 32-bit offset from the uniform row: one register an address)
  return *reinterpret_cast<const typename Elem<T>::Piece*>(reinterpret_cast<const char*>(row) +
                                                           16 * i);
}

template <typename T>
__device__ __forceinline__ void store_piece(T* row, uint32_t i,
                                            const float (&x)[Elem<T>::kVec]) {
  typename Elem<T>::Piece p;
  Elem<T>::pack(x, p);
  *reinterpret_cast<typename Elem<T>::Piece*>(reinterpret_cast<char*>(row) + 16 * i) = p;
}

template <typename T>
__device__ __forceinline__ int tail_column(int V) {
  const int col = V / Elem<T>::kVec * Elem<T>::kVec + threadIdx.x;
  return col < V ? col : -1;
}

// Combines n values over the work-group, all threads getting the results; red:
// LDS that no earlier call of the same row uses.  The waves' values are combined
// as the lanes' are, lane l taking wave l mod NT / 64's: reading them all in
// every lane would cost 64 registers.
template <int n, bool Max>
__device__ __forceinline__ void combine_lanes(float (&x)[n], int lanes) {
#pragma unroll
  for (int off = lanes / 2; off > 0; off >>= 1)
#pragma unroll
    for (int j = 0; j < n; ++j) {
      const float y = __shfl_xor(x[j], off, 64);
      x[j] = Max ? fmaxf(x[j], y) : x[j] + y;
    }
}

template <int NT, int n, bool Max>
__device__ __forceinline__ void combine(float (&x)[n], float (*red)[n]) {
  combine_lanes<n, Max>(x, 64);
  const int lane = threadIdx.x & 63;
  if (lane == 0)
#pragma unroll
    for (int j = 0; j < n; ++j) red[threadIdx.x >> 6][j] = x[j];
  __syncthreads();
#pragma unroll
  for (int j = 0; j < n; ++j) x[j] = red[lane % (NT / 64)][j];
  combine_lanes<n, Max>(x, NT / 64);
}

// A row's slots in LDS, the target behind them as a slot without mass.
struct Slots {
  int column[kMaxSlots + 1];  // -1: empty
  float t[kMaxSlots + 1];     // the teacher's logit, then its probability
  float z[kMaxSlots + 1];     // the student's logit there
};

// One row of the loss.  Row: how the logits are read (all at once, or twice).
// Two: both softmax(z / T) and softmax(z) are needed.
template <typename T, int NT, bool Two, typename Row>
__device__ __forceinline__ void distill_row(const DistillArgs& a, int64_t row, Row& held,
                                            Slots& s, float (*red_max)[2], float (*red_sum)[4],
                                            int* flags) {
  constexpr int VEC = Elem<T>::kVec;
  const T* z = static_cast<const T*>(a.logits) + row * a.ld;
  T* out = a.grad ? static_cast<T*>(a.grad) + row * a.grad_ld : nullptr;
  const int V = a.V, last = tail_column<T>(V);
  const uint32_t pieces = (uint32_t)V / VEC;
  float tail = -INFINITY;  // no share of the maximum or of a sum
  const auto no_gradient = [&](float loss) {
    if (threadIdx.x == 0 && a.row_loss) a.row_loss[row] = loss;
    if (out) {
      const float zero[VEC] = {};
      for (uint32_t i = threadIdx.x; i < pieces; i += NT) store_piece(out, i, zero);
      if (last >= 0) out[last] = (T)0.f;
    }
    __syncthreads();
  };
  const int64_t target = a.target ? a.target[row] : 0;
  const bool hard = a.alpha < 1.f, soft = a.alpha > 0.f;
  if (a.target && (target == a.ignore_index || target < 0 || target >= V)) {
    no_gradient(target == a.ignore_index ? 0.f : __builtin_nanf(""));
    return;
  }

  held.load(z, pieces);
  if (last >= 0) tail = (float)z[last];
  if (threadIdx.x < 2) flags[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll 1  // (the row's registers are live)
  for (int k = threadIdx.x; k < a.K; k += NT) {
    const int64_t c = a.idx64 ? static_cast<const int64_t*>(a.idx)[row * a.idx_ld + k]
                              : static_cast<const int32_t*>(a.idx)[row * a.idx_ld + k];
    const bool in = c >= 0 && c < V;
    if (c >= V) atomicOr(&flags[0], 1);
    s.column[k] = in ? (int)c : -1;
    const int64_t at = row * a.teacher_ld + k;
    const float t = !in ? -INFINITY
                        : (a.teacher_f32 ? static_cast<const float*>(a.teacher)[at]
                                         : (float)static_cast<const __bf16*>(a.teacher)[at]);
    // (a maximum passes NaN over; slots of -inf alone say nothing)
    if (t != -INFINITY) atomicOr(&flags[1], 1);
    s.t[k] = t;
    s.z[k] = in ? (float)z[c] : 0.f;
  }
  if (threadIdx.x == 0) {
    s.column[a.K] = hard ? (int)target : -1;
    s.t[a.K] = 0.f;
    s.z[a.K] = hard ? (float)z[target] : 0.f;
  }
  __syncthreads();
  const bool bad = soft && flags[0], taught = soft && flags[1];
  if (bad || !(taught || hard)) {
    no_gradient(bad ? __builtin_nanf("") : 0.f);
    return;
  }

  // Maxima of the student's and the teacher's logits.
  float m[2] = {fmaxf(held.max(z, pieces), tail), -INFINITY};
#pragma unroll 1
  for (int k = threadIdx.x; k < a.K; k += NT) m[1] = fmaxf(m[1], s.t[k]);
  combine<NT, 2, true>(m, red_max);
  const float c1 = kLog2e, ct = kLog2e * a.inv_temp;
  const float c = soft ? ct : c1;  // of the only softmax, unless Two

  // Sums: e^((z - m) / T), e^(z - m), the teacher's weights, and KD's terms.
  float sum[4] = {};
  held.template sums<Two>(z, pieces, m[0], c, c1, sum[0], sum[1]);
  if (last >= 0) {
    sum[0] += fast_exp2((tail - m[0]) * c);
    if (Two) sum[1] += fast_exp2((tail - m[0]) * c1);
  }
  if (taught)
#pragma unroll 1
    for (int k = threadIdx.x; k < a.K; k += NT) {
      const float w = s.column[k] < 0 ? 0.f : fast_exp2((s.t[k] - m[1]) * ct);
      if (w != 0.f) {  // (NaN too)
        sum[2] += w;
        sum[3] += w * ((s.t[k] - m[1]) - (s.z[k] - m[0]));
      }
      s.t[k] = w;  // by the thread that reads it here only; by all behind the barrier
    }
  combine<NT, 4, false>(sum, red_sum);
  const float s_hard = Two ? sum[1] : sum[0];

  if (threadIdx.x == 0 && a.row_loss) {
    float loss = 0.f;
    if (taught)
      loss = a.alpha * a.temp * a.temp *
             (sum[3] / sum[2] * a.inv_temp + (__log2f(sum[0]) - __log2f(sum[2])) * kLn2);
    if (hard) loss += (1.f - a.alpha) * (__log2f(s_hard) * kLn2 - (s.z[a.K] - m[0]));
    a.row_loss[row] = loss;
  }
  if (!out) {
    __syncthreads();
    return;
  }

  float scale = a.scale;
  if (a.scale_dev) scale *= *a.scale_dev;
  if (a.g) scale *= a.g[row * a.g_stride];
  const float from_soft = taught ? a.alpha * a.temp * scale : 0.f;
  const float from_hard = hard ? (1.f - a.alpha) * scale : 0.f;
  // Factors of the two exponentials (of the one, with both parts at T = 1).
  const float f0 = Two ? from_soft / sum[0] : (from_soft + from_hard) / sum[0];
  const float f1 = Two ? from_hard / sum[1] : 0.f;
  held.template grads<Two>(z, out, pieces, m[0], c, c1, f0, f1);
  if (last >= 0) {
    float x = fast_exp2((tail - m[0]) * c) * f0;
    if (Two) x = fmaf(fast_exp2((tail - m[0]) * c1), f1, x);
    out[last] = (T)x;
  }
  __syncthreads();

  // The slots' and the target's columns.
  const float per_weight = taught ? from_soft / sum[2] : 0.f;
  for (int k = threadIdx.x; k <= a.K; k += NT) {
    const int col = s.column[k];
    if (col < 0 || (k < a.K && !taught && !(hard && col == s.column[a.K]))) continue;
    float w = 0.f;
    bool first = true;
    for (int j = 0; j <= a.K; ++j)
      if (s.column[j] == col) {
        if (j < k) first = false;
        if (j < a.K && taught) w += s.t[j];
      }
    if (!first) continue;
    const float d = s.z[k] - m[0];
    float x = fast_exp2(d * c) * f0 - w * per_weight;
    if (Two) x += fast_exp2(d * c1) * f1;
    if (hard && col == s.column[a.K]) x -= from_hard;
    out[col] = (T)x;
  }
  __syncthreads();
}

// The row in registers: NP pieces a thread.
template <typename T, int NT, int NP>
struct HeldRow {
  static constexpr int kWaves = NP <= 8 ? 8 : 4;  // a SIMD, for the register budget
  static constexpr int VEC = Elem<T>::kVec;
  typename Elem<T>::Piece q[NP];
  uint32_t first;  // the thread's first piece

  __device__ void load(const T* z, uint32_t pieces) {
    // hidden from the compiler, which would keep every piece's offset
    // from one row to the next
    first = threadIdx.x;
    asm volatile("" : "+v"(first));
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const uint32_t i = first + p * NT;
#pragma unroll
      for (int w = 0; w < 4; ++w) q[p].w[w] = Elem<T>::kNone;
      if (i < pieces) q[p] = load_piece(z, i);
    }
  }
  // Makes the compiler unpack the row anew in each phase instead of keeping
  // every unpacked logit.
  __device__ void phase() {
#pragma unroll
    for (int p = 0; p < NP; ++p)
      asm volatile("" : "+v"(q[p].w[0]), "+v"(q[p].w[1]), "+v"(q[p].w[2]), "+v"(q[p].w[3]));
    asm volatile("" : "+v"(first));
  }
  __device__ float max(const T*, uint32_t) {
    float m = -INFINITY;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      float x[VEC];
      Elem<T>::unpack(q[p], x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) m = fmaxf(m, x[e]);
    }
    phase();
    return m;
  }
  template <bool Two>
  __device__ void sums(const T*, uint32_t, float m, float c, float c1, float& s0, float& s1) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      float x[VEC];
      Elem<T>::unpack(q[p], x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        s0 += fast_exp2((x[e] - m) * c);
        if (Two) s1 += fast_exp2((x[e] - m) * c1);
      }
    }
    phase();
  }
  template <bool Two>
  __device__ void grads(const T*, T* out, uint32_t pieces, float m, float c, float c1, float f0,
                        float f1) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const uint32_t i = first + p * NT;
      float x[VEC];
      Elem<T>::unpack(q[p], x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = x[e] - m;
        x[e] = fast_exp2(d * c) * f0;
        if (Two) x[e] = fmaf(fast_exp2(d * c1), f1, x[e]);
      }
      if (i < pieces) store_piece(out, i, x);
    }
  }
};

// A row wider than the registers hold: read for the maximum, for the sums and
// for the gradient.  In place, a thread's writes follow its own last reading.
template <typename T, int NT>
struct ReadRow {
  static constexpr int kWaves = 8;
  static constexpr int VEC = Elem<T>::kVec;
  __device__ void load(const T*, uint32_t) {}
  __device__ float max(const T* z, uint32_t pieces) {
    float m = -INFINITY;
    for (uint32_t i = threadIdx.x; i < pieces; i += NT) {
      float x[VEC];
      Elem<T>::unpack(load_piece(z, i), x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) m = fmaxf(m, x[e]);
    }
    return m;
  }
  template <bool Two>
  __device__ void sums(const T* z, uint32_t pieces, float m, float c, float c1, float& s0,
                       float& s1) {
    for (uint32_t i = threadIdx.x; i < pieces; i += NT) {
      float x[VEC];
      Elem<T>::unpack(load_piece(z, i), x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        s0 += fast_exp2((x[e] - m) * c);
        if (Two) s1 += fast_exp2((x[e] - m) * c1);
      }
    }
  }
  template <bool Two>
  __device__ void grads(const T* z, T* out, uint32_t pieces, float m, float c, float c1, float f0,
                        float f1) {
    for (uint32_t i = threadIdx.x; i < pieces; i += NT) {
      float x[VEC];
      Elem<T>::unpack(load_piece(z, i), x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = x[e] - m;
        x[e] = fast_exp2(d * c) * f0;
        if (Two) x[e] = fmaf(fast_exp2(d * c1), f1, x[e]);
      }
      store_piece(out, i, x);
    }
  }
};

// Launched for a gradient that stands already (unless_one), every work-group
// ends at once where the incoming gradient is 1.
template <typename T, int NT, bool Two, typename Row>
__global__ __launch_bounds__(NT, Row::kWaves) void distill_kernel(DistillArgs a) {
  __shared__ Slots slots;
  __shared__ float red_max[NT / 64][2], red_sum[NT / 64][4];
  __shared__ int flags[2];
  if (a.unless_one && *a.g == 1.f) return;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    Row row;
    distill_row<T, NT, Two>(a, r, row, slots, red_max, red_sum, flags);
  }
}

constexpr int kOneThreads = 1024;

template <typename V>
__device__ __forceinline__ V wg_total(V x, V* red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  V s = red[0];
#pragma unroll
  for (int w = 1; w < kOneThreads / 64; ++w) s += red[w];
  return s;
}

// out[0] = 1 / max(n, 1), out[1] = 1 / n (NaN for n = 0), n the counted rows.
__global__ __launch_bounds__(kOneThreads) void distill_count_kernel(const int64_t* target,
                                                                    int64_t rows, int64_t ignore,
                                                                    float* out) {
  __shared__ int red[kOneThreads / 64];
  int n = 0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < rows; i += kOneThreads) n += target[i] != ignore;
  n = wg_total(n, red);
  if (threadIdx.x == 0) {
    out[0] = 1.f / (float)(n > 1 ? n : 1);
    out[1] = n ? 1.f / (float)n : __builtin_nanf("");
  }
}

// Sum of the rows' losses in 64 bits and in a fixed order, times the scale.
__global__ __launch_bounds__(kOneThreads) void distill_mean_kernel(const float* row_loss,
                                                                   int64_t rows,
                                                                   const float* scale_dev,
                                                                   float scale, float* loss) {
  __shared__ double red[kOneThreads / 64];
  double s = 0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < rows; i += kOneThreads) s += (double)row_loss[i];
  s = wg_total(s, red);
  if (threadIdx.x == 0) *loss = (float)(s * (double)(scale_dev ? *scale_dev : scale));
}

template <typename T, int NT, typename Row>
hipError_t launch_row(const DistillArgs& a, unsigned grid, hipStream_t stream) {
  if (a.alpha > 0.f && a.alpha < 1.f && a.temp != 1.f)
    hipLaunchKernelGGL((distill_kernel<T, NT, true, Row>), dim3(grid), dim3(NT), 0, stream, a);
  else
    hipLaunchKernelGGL((distill_kernel<T, NT, false, Row>), dim3(grid), dim3(NT), 0, stream, a);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_distill_t(const DistillArgs& a, hipStream_t stream) {
  const int64_t pieces = a.V / Elem<T>::kVec;
  const int64_t most = a.unless_one ? 1024 : 0x7fffffff;
  const unsigned grid = (unsigned)(a.rows < most ? a.rows : most);
#define ROW(NT, NP) return launch_row<T, NT, HeldRow<T, NT, NP>>(a, grid, stream)
  if (pieces <= 256) ROW(256, 1);
  if (pieces <= 512) ROW(256, 2);
  if (pieces <= 1024) ROW(256, 4);
  if (pieces <= 2048) ROW(256, 8);
  if (pieces <= 4096) ROW(1024, 4);
  if (pieces <= 5 * 1024) ROW(1024, 5);
  if (pieces <= 6 * 1024) ROW(1024, 6);
  if (pieces <= 7 * 1024) ROW(1024, 7);
  if (pieces <= 8 * 1024) ROW(1024, 8);
  if (pieces <= 12 * 1024) ROW(1024, 12);
  if (pieces <= 16 * 1024) ROW(1024, 16);
#undef ROW
  return launch_row<T, 1024, ReadRow<T, 1024>>(a, grid, stream);
}

}  // namespace

hipError_t launch_distill_rows(const DistillArgs& a, bool f32, hipStream_t stream) {
  if (a.rows == 0) return hipSuccess;
  return f32 ? launch_distill_t<float>(a, stream) : launch_distill_t<__bf16>(a, stream);
}

hipError_t launch_distill_count(const int64_t* target, int64_t rows, int64_t ignore_index,
                                float* out, hipStream_t stream) {
  hipLaunchKernelGGL(distill_count_kernel, dim3(1), dim3(kOneThreads), 0, stream, target, rows,
                     ignore_index, out);
  return hipGetLastError();
}

hipError_t launch_distill_mean(const float* row_loss, int64_t rows, const float* scale_dev,
                               float scale, float* loss, hipStream_t stream) {
  hipLaunchKernelGGL(distill_mean_kernel, dim3(1), dim3(kOneThreads), 0, stream, row_loss, rows,
                     scale_dev, scale, loss);
  return hipGetLastError();
}

}  // namespace t2t
