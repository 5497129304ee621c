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
// stays in the registers of a work-group, packed as it was read.  An exponential
// is exp2(z c - max c), one fused operation and the instruction; with an integer
// T from 2 to 4, e^(z - max) is a power of e^((z - max) / T).  The rounding of
// max c is a common factor of all exponentials, taken out of the sums' logarithms.
// Rows whose maximum is near the type's largest magnitude (all columns
// masked with the lowest value), where max c would overflow, are read again
// and use (z - max) c.  Sums are fp32; KD is computed from
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

typedef short short2v __attribute__((ext_vector_type(2)));
typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));

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
  // Maximum over pieces on the packed bits.  Values of sign 0 are ordered as
  // signed 16-bit numbers and above all others; only a row without any looks
  // for its smallest unsigned number (a second pass over the registers).
  static constexpr bool kTwoMax = true;
  typedef short2v Max;
  __device__ static Max none() { return Max{-1, -1}; }
  __device__ static void take(const Piece& p, Max& m) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      m = __builtin_elementwise_max(m, __builtin_bit_cast(short2v, p.w[e]));
  }
  __device__ static float half(int bits) { return __uint_as_float((uint32_t)bits << 16); }
  __device__ static float value(Max m) {  // -1 where every value has sign 1
    const int x = m[0] > m[1] ? m[0] : m[1];
    return x < 0 ? -1.f : half(x);
  }
  typedef ushort2v Least;
  __device__ static Least most() { return Least{0xff80, 0xff80}; }
  __device__ static void take_least(const Piece& p, Least& m) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      m = __builtin_elementwise_min(m, __builtin_bit_cast(ushort2v, p.w[e]));
  }
  __device__ static float negative(Least m) { return half(m[0] < m[1] ? m[0] : m[1]); }
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
  static constexpr bool kTwoMax = false;
  typedef float Max;
  __device__ static Max none() { return -INFINITY; }
  __device__ static void take(const Piece& p, Max& m) {
#pragma unroll
    for (int e = 0; e < 4; ++e) m = fmaxf(m, __uint_as_float(p.w[e]));
  }
  __device__ static float value(Max m) { return m; }
  typedef float Least;
  __device__ static Least most() { return -INFINITY; }
  __device__ static void take_least(const Piece&, Least&) {}
  __device__ static float negative(Least m) { return m; }
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

// The exponentials of a row.  P: 1, one softmax; 0, two of unrelated
// temperatures; n >= 2, e^(z - max) is the n-th power of e^((z - max) / T).
// Far: by differences, for maxima whose product with c could overflow.
template <int P, bool Far>
struct Exps {
  float m, c, nm, c1, nm1;
  __device__ Exps(float max, float c_, float c1_)
      : m(max), c(c_), nm(-max * c_), c1(c1_), nm1(-max * c1_) {}
  __device__ float first(float x) const {
    return fast_exp2(Far ? (x - m) * c : fmaf(x, c, nm));
  }
  __device__ float other(float x) const {
    return fast_exp2(Far ? (x - m) * c1 : fmaf(x, c1, nm1));
  }
  __device__ static float power(float e) {  // e^(P - 1), P >= 2
    return P == 2 ? e : P == 3 ? e * e : e * e * e;
  }
  __device__ void sum(float x, float& s0, float& s1) const {
    const float e = first(x);
    s0 += e;
    if (P == 0) s1 += other(x);
    if (P >= 2) s1 = fmaf(power(e), e, s1);
  }
  __device__ float grad(float x, float f0, float f1) const {
    const float e = first(x);
    if (P == 0) return fmaf(other(x), f1, e * f0);
    if (P >= 2) return e * fmaf(power(e), f1, f0);
    return e * f0;
  }
  // log2 of the sums less the common factor 2^(max c - round(max c)).
  __device__ float log2_first(float s0) const {
    return __log2f(s0) - (Far ? 0.f : fmaf(m, c, nm));
  }
  __device__ float log2_other(float s1) const {
    return __log2f(s1) - (Far ? 0.f : P == 0 ? fmaf(m, c1, nm1) : P * fmaf(m, c, nm));
  }
};

struct Shared {
  Slots slots;
  float max[2][16][2], sum[16][4];  // of the waves
  int flags[2];                     // a column >= V; a slot with a say
};

// A row of the loss with everything but its own logits known.
template <typename T>
struct RowAt {
  const T* z;
  T* out;
  uint32_t pieces;
  int last;    // the thread's column behind the pieces, or -1
  float tail;  // its logit
};

template <typename T, int NT, int P, bool Far, typename Row>
__device__ __forceinline__ void finish_row(const DistillArgs& a, int64_t row, const RowAt<T>& at,
                                           Row& held, Shared& sh, float m, float m_teacher,
                                           bool taught, bool hard, float c, float ct) {
  Slots& s = sh.slots;
  const Exps<P, Far> ex(m, c, kLog2e);

  // Sums: e^((z - m) / T), e^(z - m), the teacher's weights, and KD's terms.
  float sum[4] = {};
  held.sums(at, ex, sum[0], sum[1]);
  if (at.last >= 0) ex.sum(at.tail, sum[0], sum[1]);
  if (taught)
#pragma unroll 1
    for (int k = threadIdx.x; k < a.K; k += NT) {
      const float w = s.column[k] < 0 ? 0.f : fast_exp2((s.t[k] - m_teacher) * ct);
      if (w != 0.f) {  // (NaN too)
        sum[2] += w;
        sum[3] += w * ((s.t[k] - m_teacher) - (s.z[k] - m));
      }
      s.t[k] = w;  // by the thread that reads it here only; by all behind the barrier
    }
  combine<NT, 4, false>(sum, sh.sum);

  if (threadIdx.x == 0 && a.row_loss) {
    float loss = 0.f;
    if (taught)
      loss = a.alpha * a.temp * a.temp *
             (sum[3] / sum[2] * a.inv_temp + (ex.log2_first(sum[0]) - __log2f(sum[2])) * kLn2);
    if (hard) {
      const float lse = P == 1 ? ex.log2_first(sum[0]) : ex.log2_other(sum[1]);
      loss += (1.f - a.alpha) * (lse * kLn2 - (s.z[a.K] - m));
    }
    a.row_loss[row] = loss;
  }
  if (!at.out) {
    __syncthreads();
    return;
  }

  float scale = a.scale;
  if (a.scale_dev) scale *= *a.scale_dev;
  if (a.g) scale *= a.g[row * a.g_stride];
  const float from_soft = taught ? a.alpha * a.temp * scale : 0.f;
  const float from_hard = hard ? (1.f - a.alpha) * scale : 0.f;
  // Factors of the two exponentials (of the one, with both parts at T = 1).
  const float f0 = (P == 1 ? from_soft + from_hard : from_soft) / sum[0];
  const float f1 = P == 1 ? 0.f : from_hard / sum[1];
  held.grads(at, ex, f0, f1);
  if (at.last >= 0) at.out[at.last] = (T)ex.grad(at.tail, f0, f1);
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
    float x = ex.grad(s.z[k], f0, f1) - w * per_weight;
    if (hard && col == s.column[a.K]) x -= from_hard;
    at.out[col] = (T)x;
  }
  __syncthreads();
}

// A row wider than the registers hold: read for the maximum, for the sums and
// for the gradient.  In place, a thread's writes follow its own last reading.
template <typename T, int NT>
struct ReadRow {
  static constexpr int kWaves = NT == 1024 ? 8 : 4;
  static constexpr bool kLoop = true;
  static constexpr int VEC = Elem<T>::kVec;
  __device__ void load(const RowAt<T>&) {}
  __device__ float max(const RowAt<T>& at) {
    float m = -INFINITY;
    for (uint32_t i = threadIdx.x; i < at.pieces; i += NT) {
      float x[VEC];
      Elem<T>::unpack(load_piece(at.z, i), x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) m = fmaxf(m, x[e]);
    }
    return m;
  }
  static constexpr bool kTwoMax = false;
  __device__ float least_negative() { return -INFINITY; }
  template <typename E>
  __device__ void sums(const RowAt<T>& at, const E& ex, float& s0, float& s1) {
    for (uint32_t i = threadIdx.x; i < at.pieces; i += NT) {
      float x[VEC];
      Elem<T>::unpack(load_piece(at.z, i), x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) ex.sum(x[e], s0, s1);
    }
  }
  template <typename E>
  __device__ void grads(const RowAt<T>& at, const E& ex, float f0, float f1) {
    for (uint32_t i = threadIdx.x; i < at.pieces; i += NT) {
      float x[VEC];
      Elem<T>::unpack(load_piece(at.z, i), x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[e] = ex.grad(x[e], f0, f1);
      store_piece(at.out, i, x);
    }
  }
};

// The row in registers: NP pieces a thread.  The pieces are worked on one after
// the other (sched_barrier): unpacked all at once, they would spill.
template <typename T, int NT, int NP>
struct HeldRow {
  static constexpr int kWaves = NP <= 7 ? 8 : 4;  // a SIMD, for the register budget
  static constexpr bool kLoop = false;
  static constexpr int VEC = Elem<T>::kVec;
  static constexpr bool kTwoMax = Elem<T>::kTwoMax;
  uint4 q[NP];
  uint32_t first;  // the thread's first piece

  __device__ void load(const RowAt<T>& at) {
    // hidden from the compiler, which would keep every piece's offset
    first = threadIdx.x;
    asm volatile("" : "+v"(first));
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const uint32_t i = first + p * NT;
      // columns past the row: no share of the maximum or of a sum
      constexpr uint32_t none = Elem<T>::kNone;
      q[p] = make_uint4(none, none, none, none);
      if (i < at.pieces) {
        const typename Elem<T>::Piece x = load_piece(at.z, i);
        q[p] = make_uint4(x.w[0], x.w[1], x.w[2], x.w[3]);
      }
    }
  }
  // Makes the compiler unpack the row anew in each phase instead of keeping
  // every unpacked logit.
  __device__ void phase() {
#pragma unroll
    for (int p = 0; p < NP; ++p)
      asm volatile("" : "+v"(q[p].x), "+v"(q[p].y), "+v"(q[p].z), "+v"(q[p].w));
    asm volatile("" : "+v"(first));
  }
  __device__ typename Elem<T>::Piece piece(int p) const {
    return {{q[p].x, q[p].y, q[p].z, q[p].w}};
  }
  __device__ float max(const RowAt<T>&) {
    typename Elem<T>::Max m = Elem<T>::none();
#pragma unroll
    for (int p = 0; p < NP; ++p) Elem<T>::take(piece(p), m);
    phase();
    return Elem<T>::value(m);
  }
  __device__ float least_negative() {
    typename Elem<T>::Least m = Elem<T>::most();
#pragma unroll
    for (int p = 0; p < NP; ++p) Elem<T>::take_least(piece(p), m);
    phase();
    return Elem<T>::negative(m);
  }
  template <typename E>
  __device__ void sums(const RowAt<T>&, const E& ex, float& s0, float& s1) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      float x[VEC];
      Elem<T>::unpack(piece(p), x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) ex.sum(x[e], s0, s1);
      __builtin_amdgcn_sched_barrier(0);
    }
    phase();
  }
  template <typename E>
  __device__ void grads(const RowAt<T>& at, const E& ex, float f0, float f1) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const uint32_t i = first + p * NT;
      float x[VEC];
      Elem<T>::unpack(piece(p), x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[e] = ex.grad(x[e], f0, f1);
      if (i < at.pieces) store_piece(at.out, i, x);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// One row of the loss.  Row: how the logits are read (all at once, or again in
// each phase).
template <typename T, int NT, int P, typename Row>
__device__ __forceinline__ void distill_row(const DistillArgs& a, int64_t row, Shared& sh) {
  constexpr int VEC = Elem<T>::kVec;
  Slots& s = sh.slots;
  const int V = a.V;
  RowAt<T> at;
  at.z = static_cast<const T*>(a.logits) + row * a.ld;
  at.out = a.grad ? static_cast<T*>(a.grad) + row * a.grad_ld : nullptr;
  at.pieces = (uint32_t)V / VEC;
  at.last = tail_column<T>(V);
  at.tail = -INFINITY;
  const auto no_gradient = [&](float loss) {
    if (threadIdx.x == 0 && a.row_loss) a.row_loss[row] = loss;
    if (at.out) {
      const float zero[VEC] = {};
      for (uint32_t i = threadIdx.x; i < at.pieces; i += NT) store_piece(at.out, i, zero);
      if (at.last >= 0) at.out[at.last] = (T)0.f;
    }
    __syncthreads();
  };
  const int64_t target = a.target ? a.target[row] : 0;
  const bool hard = a.alpha < 1.f, soft = a.alpha > 0.f;
  if (a.target && (target == a.ignore_index || target < 0 || target >= V)) {
    no_gradient(target == a.ignore_index ? 0.f : __builtin_nanf(""));
    return;
  }

  const auto column = [&](int k) {
    return a.idx64 ? static_cast<const int64_t*>(a.idx)[row * a.idx_ld + k]
                   : static_cast<const int32_t*>(a.idx)[row * a.idx_ld + k];
  };
  const auto teacher = [&](int k) {
    const int64_t i = row * a.teacher_ld + k;
    return a.teacher_f32 ? static_cast<const float*>(a.teacher)[i]
                         : (float)static_cast<const __bf16*>(a.teacher)[i];
  };
  // The thread's first slot ahead of the row: the student's logit there, loaded
  // behind it, waits for its column alone.
  int64_t c0 = -1;
  float t0 = 0.f;
  if ((int)threadIdx.x < a.K) {
    c0 = column(threadIdx.x);
    t0 = teacher(threadIdx.x);
  }
  Row held;
  held.load(at);
  if (at.last >= 0) at.tail = (float)at.z[at.last];
  if (threadIdx.x < 2) sh.flags[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll 1  // (the row's registers are live)
  for (int k = threadIdx.x; k < a.K; k += NT) {
    const bool ahead = k == (int)threadIdx.x;
    const int64_t c = ahead ? c0 : column(k);
    const bool in = c >= 0 && c < V;
    if (c >= V) atomicOr(&sh.flags[0], 1);
    s.column[k] = in ? (int)c : -1;
    const float t = !in ? -INFINITY : ahead ? t0 : teacher(k);
    // (a maximum passes NaN over; slots of -inf alone say nothing)
    if (t != -INFINITY) atomicOr(&sh.flags[1], 1);
    s.t[k] = t;
    s.z[k] = in ? (float)at.z[c] : 0.f;
  }
  if (threadIdx.x == 0) {
    s.column[a.K] = hard ? (int)target : -1;
    s.t[a.K] = 0.f;
    s.z[a.K] = hard ? (float)at.z[target] : 0.f;
  }

  // Maxima of the student's and the teacher's logits.
  float m[2] = {fmaxf(held.max(at), at.tail), -INFINITY};
#pragma unroll 1
  for (int k = threadIdx.x; k < a.K; k += NT) m[1] = fmaxf(m[1], s.t[k]);
  combine<NT, 2, true>(m, sh.max[0]);  // its barrier also ends the slots
  const bool bad = soft && sh.flags[0], taught = soft && sh.flags[1];
  if (bad || !(taught || hard)) {
    no_gradient(bad ? __builtin_nanf("") : 0.f);
    return;
  }
  if (Row::kTwoMax && m[0] < 0.f) {  // no value of sign 0 among the pieces
    float n[2] = {fmaxf(held.least_negative(), at.tail), -INFINITY};
    combine<NT, 2, true>(n, sh.max[1]);
    m[0] = n[0];
  }
  const float ct = kLog2e * a.inv_temp;
  const float c = soft ? ct : kLog2e;  // of the only softmax, where there is one
  // |max| c below the largest float, for c up to 144
  if (fabsf(m[0]) < 1e36f) {
    finish_row<T, NT, P, false>(a, row, at, held, sh, m[0], m[1], taught, hard, c, ct);
  } else {
    ReadRow<T, NT> again;
    finish_row<T, NT, P, true>(a, row, at, again, sh, m[0], m[1], taught, hard, c, ct);
  }
}

// Launched for a gradient that stands already (unless_one), every work-group
// ends at once where the incoming gradient is 1.
template <typename T, int NT, int P, typename Row>
__global__ __launch_bounds__(NT, Row::kWaves) void distill_kernel(DistillArgs a) {
  __shared__ Shared sh;
  if (a.unless_one && *a.g == 1.f) return;
  if constexpr (Row::kLoop) {
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) distill_row<T, NT, P, Row>(a, r, sh);
  } else {  // (what a loop keeps from one row to the next costs the registers of a piece)
    distill_row<T, NT, P, Row>(a, blockIdx.x, sh);
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
  const bool two = a.alpha > 0.f && a.alpha < 1.f && a.temp != 1.f;
#define EXPS(P) \
  hipLaunchKernelGGL((distill_kernel<T, NT, P, Row>), dim3(grid), dim3(NT), 0, stream, a)
  if (!two) EXPS(1);
  else if (a.temp == 2.f) EXPS(2);
  else if (a.temp == 3.f) EXPS(3);
  else if (a.temp == 4.f) EXPS(4);
  else EXPS(0);
#undef EXPS
  return hipGetLastError();
}

template <typename T>
hipError_t launch_distill_t(const DistillArgs& a, hipStream_t stream) {
  const int64_t pieces = a.V / Elem<T>::kVec;
  // A gradient that stands as a rule: few work-groups, which end at once or
  // read their rows (with the held row's threads, so in its order of additions).
  const int64_t most = 1024;
  const unsigned all = (unsigned)a.rows, few = (unsigned)(a.rows < most ? a.rows : most);
#define READ(NT) return launch_row<T, NT, ReadRow<T, NT>>(a, few, stream)
#define ROW(NT, NP) return launch_row<T, NT, HeldRow<T, NT, NP>>(a, all, stream)
  if (pieces <= 1024) {
    if (a.unless_one) READ(256);
    if (pieces <= 256) ROW(256, 1);
    if (pieces <= 512) ROW(256, 2);
    ROW(256, 4);
  }
  if (pieces <= 2048) {
    if (a.unless_one) READ(512);
    ROW(512, 4);
  }
  if (a.unless_one || pieces > 16 * 1024)
    return launch_row<T, 1024, ReadRow<T, 1024>>(a, a.unless_one ? few : all, stream);
  if (pieces <= 4 * 1024) ROW(1024, 4);
  if (pieces <= 5 * 1024) ROW(1024, 5);
  if (pieces <= 6 * 1024) ROW(1024, 6);
  if (pieces <= 7 * 1024) ROW(1024, 7);
  if (pieces <= 8 * 1024) ROW(1024, 8);
  if (pieces <= 12 * 1024) ROW(1024, 12);
  ROW(1024, 16);
#undef ROW
#undef READ
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
