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
// HBM bound: the row is read once and its gradient written once (8192 rows of 50257
// bf16 columns, 64 slots, with counting and mean: 363 us, 4.5 TB/s of the 5.1 of a
// large copy; 2048 rows without gradient, read from memory: 59 us, 3.5 TB/s; the
// same rows again, from the last-level cache: 47).  The row stays in the registers
// of a work-group, packed as it was read.  An exponential
// is exp2(z c - max c), one fused operation and the instruction; with an integer
// T from 2 to 4, e^(z - max) is a power of e^((z - max) / T).  The rounding of
// max c is a common factor of all exponentials, taken out of the sums' logarithms;
// below |max c| = 2^24 it is at most 2^(1/2), 4 as a fourth power.  Rows whose
// maximum is farther from 0 (all columns masked with a large negative value),
// where that factor would grow past what fp32 holds, are read again and use
// (z - max) c.  Sums are fp32; KD is computed from
//   sum_k w_k ((t_k - max t) - (z(i_k) - max z)) / (T sum w) - ln sum w + ln sum_j
// with w_k = e^((t_k - max t) / T), whose terms are small where the result is.
// The gradient is first written without the teacher's and the target's terms;
// behind a barrier, a thread for each of those columns writes its value again,
// the weights of equal columns added, in their order.  The gradient may
// overwrite the logits: everything is read before the barriers ahead of the
// first write.
//
// Addresses: rows start anywhere on their type (V = 50257 columns of bf16 have
// every second row off a 4-byte boundary); whole pieces start at the row's first
// 16-byte boundary (so the order of a row's additions goes by its address
// modulo 16).  A gradient whose rows lie otherwise is written in pieces
// off that boundary, which global memory instructions allow.
#include "attn_kernels.h"

namespace t2t {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxSlots = kDistillMaxSlots;

typedef float float2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
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
    for (int e = 0; e < 4; ++e)
      p.w[e] = __builtin_bit_cast(
          uint32_t, __builtin_convertvector((float2v{x[2 * e], x[2 * e + 1]}), bf16x2v));
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

// A row of V columns: the columns up to its first 16-byte boundary, whole pieces
// from there (body), and the columns behind them.  The first threads hold one
// of the columns outside the pieces each (`last`).
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

// The exponentials of a row.  P: 1, one softmax; 0, two of unrelated
// temperatures; n >= 2, e^(z - max) is the n-th power of e^((z - max) / T).
// Far: by differences, for maxima whose product with c rounds by more than 1/2.
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

// seen: a bit for every column of a slot (modulo its size: two columns of one
// bit only cost time).  A column that is met twice sends the row to the search
// through `column`; looking for equal columns in every row took 15 % of its time.
constexpr int kSeenWords = 2048;
struct Shared {
  int column[kMaxSlots];  // of the slots; -1: empty
  float w[kMaxSlots];     // their weights
  uint32_t seen[kSeenWords];
  int twice, target_in;   // a bit of `seen` met twice; a slot at the target's column
  float max[2][16][4], sum[16][4];  // of the waves
};

// A row, and what a thread holds of it before the work begins.
template <typename T>
struct RowAt {
  const T* z;
  T* out;
  const T* body;   // the first piece
  T* out_body;
  uint32_t pieces;
  int last;        // the thread's column outside the pieces, or -1
  float tail;      // its logit
  int64_t target;
  int64_t column;  // of the thread's slot; -1: none
  float t;         // the teacher's logit there
};

template <typename T>
__device__ __forceinline__ RowAt<T> row_at(const DistillArgs& a, int64_t row) {
  RowAt<T> at;
  at.z = static_cast<const T*>(a.logits) + row * a.ld;
  at.out = a.grad ? static_cast<T*>(a.grad) + row * a.grad_ld : nullptr;
  const int ahead = min((int)(-reinterpret_cast<uintptr_t>(at.z) & 15) / (int)sizeof(T), a.V);
  at.body = at.z + ahead;
  at.out_body = at.out + ahead;
  at.pieces = (uint32_t)(a.V - ahead) / Elem<T>::kVec;
  const int behind = ahead + at.pieces * Elem<T>::kVec;
  const int i = threadIdx.x, col = i < ahead ? i : behind + i - ahead;
  at.last = col < a.V && (i < ahead || i - ahead < Elem<T>::kVec) ? col : -1;
  at.target = a.target ? a.target[row] : 0;
  at.column = -1;
  at.t = -INFINITY;
  const int k = threadIdx.x;
  if (k < a.K) {
    at.column = a.idx64 ? static_cast<const int64_t*>(a.idx)[row * a.idx_ld + k]
                        : static_cast<const int32_t*>(a.idx)[row * a.idx_ld + k];
    const int64_t slot = row * a.teacher_ld + k;
    at.t = a.teacher_f32 ? static_cast<const float*>(a.teacher)[slot]
                         : (float)static_cast<const __bf16*>(a.teacher)[slot];
  }
  at.tail = at.last >= 0 ? (float)at.z[at.last] : -INFINITY;  // (no share of a sum)
  return at;
}

// A row wider than the registers hold: read for the maximum, for the sums and
// for the gradient.  In place, a thread's writes follow its own last reading.
template <typename T, int NT>
struct ReadRow {
  static constexpr int kWaves = NT == 1024 ? 8 : 4;  // a SIMD, for the register budget
  static constexpr bool kLoop = true;
  static constexpr int VEC = Elem<T>::kVec;
  static constexpr bool kTwoMax = false;
  __device__ void load(const RowAt<T>&) {}
  __device__ float max(const RowAt<T>& at) {
    float m = -INFINITY;
    for (uint32_t i = threadIdx.x; i < at.pieces; i += NT) {
      float x[VEC];
      Elem<T>::unpack(load_piece(at.body, i), x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) m = fmaxf(m, x[e]);
    }
    return m;
  }
  __device__ float least_negative() { return -INFINITY; }
  template <typename E>
  __device__ void sums(const RowAt<T>& at, const E& ex, float& s0, float& s1) {
    for (uint32_t i = threadIdx.x; i < at.pieces; i += NT) {
      float x[VEC];
      Elem<T>::unpack(load_piece(at.body, i), x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) ex.sum(x[e], s0, s1);
    }
  }
  template <typename E>
  __device__ void grads(const RowAt<T>& at, const E& ex, float f0, float f1) {
    for (uint32_t i = threadIdx.x; i < at.pieces; i += NT) {
      float x[VEC];
      Elem<T>::unpack(load_piece(at.body, i), x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[e] = ex.grad(x[e], f0, f1);
      store_piece(at.out_body, i, x);
    }
  }
};

// The row in registers: NP pieces a thread.  The pieces are worked on one after
// the other (sched_barrier): unpacked all at once, they would spill.
template <typename T, int NT, int NP>
struct HeldRow {
  static constexpr int kWaves = NP <= 8 ? 8 : NT < 1024 ? 6 : 4;
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
        const typename Elem<T>::Piece x = load_piece(at.body, i);
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
      if (i < at.pieces) store_piece(at.out_body, i, x);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// The row's sums, its loss and its gradient; m and m_teacher are the maxima.
template <typename T, int NT, int P, bool Far, typename Row>
__device__ __forceinline__ void finish_row(const DistillArgs& a, int64_t row, const RowAt<T>& at,
                                           Row& held, Shared& sh, float z_slot, float z_target,
                                           float m, float m_teacher, bool taught, bool hard,
                                           float c, float ct, float scale) {
  const Exps<P, Far> ex(m, c, kLog2e);
  const int k0 = threadIdx.x;

  // Sums: e^((z - m) / T), e^(z - m), the teacher's weights, and KD's terms.
  float sum[4] = {};
  if (k0 < a.K) {
    const bool in = at.column >= 0;
    const float w = taught && in ? fast_exp2((at.t - m_teacher) * ct) : 0.f;
    if (w != 0.f) {  // (NaN too)
      sum[2] = w;
      sum[3] = w * ((at.t - m_teacher) - (z_slot - m));
    }
    sh.column[k0] = in ? (int)at.column : -1;
    sh.w[k0] = w;
    if (in) {
      const uint32_t bit = (uint32_t)at.column % (32 * kSeenWords);
      if (atomicOr(&sh.seen[bit / 32], 1u << bit % 32) >> bit % 32 & 1) sh.twice = 1;
      if (hard && at.column == at.target) sh.target_in = 1;
    }
  }
  held.sums(at, ex, sum[0], sum[1]);
  if (at.last >= 0) ex.sum(at.tail, sum[0], sum[1]);
  combine<NT, 4, false>(sum, sh.sum);

  if (k0 == 0 && a.row_loss) {
    float loss = 0.f;
    if (taught)
      loss = a.alpha * a.temp * a.temp *
             (sum[3] / sum[2] * a.inv_temp + (ex.log2_first(sum[0]) - __log2f(sum[2])) * kLn2);
    if (hard) {
      const float lse = P == 1 ? ex.log2_first(sum[0]) : ex.log2_other(sum[1]);
      loss += (1.f - a.alpha) * (lse * kLn2 - (z_target - m));
    }
    a.row_loss[row] = loss;
  }
  if (!at.out) return;

  const float from_soft = taught ? a.alpha * a.temp * scale : 0.f;
  const float from_hard = hard ? (1.f - a.alpha) * scale : 0.f;
  // Factors of the two exponentials (of the one, with both parts at T = 1).
  const float f0 = (P == 1 ? from_soft + from_hard : from_soft) / sum[0];
  const float f1 = P == 1 ? 0.f : from_hard / sum[1];
  held.grads(at, ex, f0, f1);
  if (at.last >= 0) at.out[at.last] = (T)ex.grad(at.tail, f0, f1);
  __syncthreads();

  // The slots' columns, each by its first slot, and the target's.
  const float per_weight = taught ? from_soft / sum[2] : 0.f;
  const int64_t target = hard ? at.target : -1;
  if (k0 < a.K && at.column >= 0 && (taught || at.column == target)) {
    float w = sh.w[k0];
    bool first = true;
    if (sh.twice)
      for (int j = 0; j < a.K; ++j)
        if (j != k0 && sh.column[j] == (int)at.column) {
          first = first && j > k0;
          w += sh.w[j];
        }
    if (first) {
      float x = ex.grad(z_slot, f0, f1) - w * per_weight;
      if (at.column == target) x -= from_hard;
      at.out[at.column] = (T)x;
    }
  }
  if (k0 == 0 && hard && !sh.target_in) at.out[target] = (T)(ex.grad(z_target, f0, f1) - from_hard);
}

// One row of the loss.  Row: how the logits are read (all at once, or again in
// each phase).
template <typename T, int NT, int P, typename Row>
__device__ __forceinline__ void distill_row(const DistillArgs& a, int64_t row, const RowAt<T>& at,
                                            Row& held, Shared& sh, float scale) {
  constexpr int VEC = Elem<T>::kVec;
  const int V = a.V;
  const bool hard = a.alpha < 1.f, soft = a.alpha > 0.f;
  const auto no_gradient = [&](float loss) {
    if (threadIdx.x == 0 && a.row_loss) a.row_loss[row] = loss;
    if (at.out) {
      const float zero[VEC] = {};
      for (uint32_t i = threadIdx.x; i < at.pieces; i += NT) store_piece(at.out_body, i, zero);
      if (at.last >= 0) at.out[at.last] = (T)0.f;
    }
  };
  if (a.target && (at.target == a.ignore_index || at.target < 0 || at.target >= V)) {
    no_gradient(at.target == a.ignore_index ? 0.f : __builtin_nanf(""));
    return;
  }
  if (a.K > 0 && at.out)
    for (int i = threadIdx.x; i < kSeenWords; i += NT) sh.seen[i] = 0;
  if (threadIdx.x == 0) sh.twice = sh.target_in = 0;
  const bool in = at.column >= 0 && at.column < V;
  const float z_slot = in ? (float)at.z[at.column] : 0.f;
  const float z_target = hard && threadIdx.x == 0 ? (float)at.z[at.target] : 0.f;

  // Maxima: the student's and the teacher's logits, a column outside the
  // vocabulary, a slot with a say (slots of -inf alone have none; a maximum
  // passes NaN over).
  float m[4] = {fmaxf(held.max(at), at.tail), in ? at.t : -INFINITY, at.column >= V ? 1.f : 0.f,
                in && at.t != -INFINITY ? 1.f : 0.f};
  combine<NT, 4, true>(m, sh.max[0]);
  const bool bad = soft && m[2] != 0.f, taught = soft && m[3] != 0.f;
  if (bad || !(taught || hard)) {
    no_gradient(bad ? __builtin_nanf("") : 0.f);
    return;
  }
  if (Row::kTwoMax && m[0] < 0.f) {  // no value of sign 0 among the pieces
    float n[4] = {fmaxf(held.least_negative(), at.tail)};
    combine<NT, 4, true>(n, sh.max[1]);
    m[0] = n[0];
  }
  const float ct = kLog2e * a.inv_temp;
  const float c = soft ? ct : kLog2e;  // of the only softmax, where there is one
  // Half a step of max c is the exponent of the factor that all exponentials share
  // (of the other softmax's, for P = 0, with its own c).
  if (fabsf(m[0]) * fmaxf(c, kLog2e) < 0x1p24f) {
    finish_row<T, NT, P, false>(a, row, at, held, sh, z_slot, z_target, m[0], m[1], taught, hard,
                                c, ct, scale);
  } else {
    ReadRow<T, NT> again;
    finish_row<T, NT, P, true>(a, row, at, again, sh, z_slot, z_target, m[0], m[1], taught, hard,
                               c, ct, scale);
  }
}

// Launched for a gradient that stands already (unless_one), every work-group
// ends at once where the incoming gradient is 1.
template <typename T, int NT, int P, typename Row>
__global__ __launch_bounds__(NT, Row::kWaves) void distill_kernel(DistillArgs a) {
  __shared__ Shared sh;
  if (a.unless_one && *a.g == 1.f) return;
  const auto one = [&](int64_t row) {
    const RowAt<T> at = row_at<T>(a, row);
    Row held;
    held.load(at);
    const float scale = (a.scale_dev ? a.scale * *a.scale_dev : a.scale) *
                        (a.g ? a.g[row * a.g_stride] : 1.f);
    distill_row<T, NT, P>(a, row, at, held, sh, scale);
  };
  if constexpr (Row::kLoop) {
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
      one(row);
      __syncthreads();  // LDS is the next row's
    }
  } else {  // (what a loop keeps from one row to the next costs the registers of a piece)
    one(blockIdx.x);
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
  const unsigned all = (unsigned)a.rows, few = all < 1024 ? all : 1024;
#define READ(NT) return launch_row<T, NT, ReadRow<T, NT>>(a, few, stream)
#define ROW(NT, NP) return launch_row<T, NT, HeldRow<T, NT, NP>>(a, all, stream)
  // At least a thread a slot.
  // (a gradient that stands as a rule is read, not held, with the threads that
  // hold it: in the same order of additions.  The idle launch takes 5 us; where the
  // incoming gradient is not 1, 8192 rows of 50257 take 626 on top of the forward)
  if (pieces <= 1024 && a.K <= 256) {
    if (a.unless_one) READ(256);
    if (pieces <= 256) ROW(256, 1);
    if (pieces <= 512) ROW(256, 2);
    ROW(256, 4);
  }
  // Rows in as few threads as still hold them: each thread has about 30 registers
  // beside its pieces, and what is left of them is further rows on the CU, whose
  // loads run while another row is computed (8192 rows of 50257: three rows of
  // 512 threads 363 us, two of 1024 372 us; 2048 without gradient 59 and 64 us).
  if (pieces <= 13 * 512 && a.K <= 512) {
    if (a.unless_one) READ(512);
    if (pieces <= 4 * 512) ROW(512, 4);
    if (pieces <= 8 * 512) ROW(512, 8);
    if (pieces <= 10 * 512) ROW(512, 10);
    ROW(512, 13);
  }
  if (a.unless_one || pieces > 16 * 1024) READ(1024);
  if (pieces <= 2 * 1024) ROW(1024, 2);
  if (pieces <= 4 * 1024) ROW(1024, 4);
  if (pieces <= 8 * 1024) ROW(1024, 8);
  if (pieces <= 12 * 1024) ROW(1024, 12);
  ROW(1024, 16);
#undef ROW
#undef READ
}

}  // namespace

// A launch has fewer than 2^32 threads: of more rows than that there are several.
hipError_t launch_distill_rows(const DistillArgs& all, bool f32, hipStream_t stream) {
  constexpr int64_t kRows = 1 << 21;
  const int64_t size = f32 ? 4 : 2;
  for (int64_t r0 = 0; r0 < all.rows; r0 += kRows) {
    DistillArgs a = all;
    const auto from = [r0](auto* p, int64_t bytes) {
      return p ? reinterpret_cast<decltype(p)>(reinterpret_cast<uintptr_t>(p) + r0 * bytes) : p;
    };
    a.rows = all.rows - r0 < kRows ? all.rows - r0 : kRows;
    a.logits = from(a.logits, a.ld * size);
    a.grad = from(a.grad, a.grad_ld * size);
    a.idx = from(a.idx, a.idx_ld * (a.idx64 ? 8 : 4));
    a.teacher = from(a.teacher, a.teacher_ld * (a.teacher_f32 ? 4 : 2));
    a.target = from(a.target, 8);
    a.g = from(a.g, a.g_stride * 4);
    a.row_loss = from(a.row_loss, 4);
    const hipError_t e =
        f32 ? launch_distill_t<float>(a, stream) : launch_distill_t<__bf16>(a, stream);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
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
