// Masked attention of a few new query rows against a key/value cache: the
// decode step of generation.
//
// The reference regenerates every token by rebuilding the mask and running
// the full forward over the whole packed sequence
// (model/generation_loop.py:90-92 -> TS2TSModel.forward_inference,
// model/model.py:214-237) and keeps only the last position's logits.  With
// the keys and values of the unchanged prefix cached, one step needs the
// attention of the new rows only, against every cached key -- an HBM-bound
// gather: each allowed key costs its K and V rows (4 D bytes), each masked
// key only its mask inputs (4 + 8 W bytes), because the mask is evaluated per
// key before any K/V load:
//   allowed(q, j) = j <= pos(q) && (doc[j] == doc(q) ||
//                   OR_w (q_bits[w](q) & kv_bits[w][j]) != 0)
// (the doc_causal / cross_doc_link mask_mod, cross_doc_mask.py:348-357,
// block_mask_creator.py:121-129).
//
// Split-KV.  attn_decode_partial: one work-group per (256-key chunk, kv head,
// batch row) handles all R = G * Tq query rows of the kv head (G query heads
// of the GQA group x Tq new tokens, R <= 8).  A key is read by D/8 adjacent
// lanes, 16 bytes each, so a K or V row is one coalesced run; the lanes of a
// key hold the query rows' matching 8 elements in registers, and the partial
// dot products are summed across them with DPP butterflies.  Pass 1 writes the
// chunk's scores to LDS, pass 2 takes the chunk's row max, weights the V rows
// by exp2(s - max) and sums them across the key groups (DPP, then LDS across
// waves).  The kernel has two dependent memory stages: the keys' mask
// inputs with the query rows, then the K and V rows of the allowed keys.
// Each (row, chunk) leaves (max, sum, unnormalised o[D]) in the
// workspace; attn_decode_combine merges the chunks of a row into o (bf16)
// and the log2-domain LSE.  Fully masked rows give o = 0 and LSE = -inf.
//
// With a sliding window of w positions and s sinks (Win) a key of the row's own
// document is allowed only if pos(q) - j < w or 0 <= j - start(q) < s, start(q)
// = the first position of the row's document; grants are as they were.  The
// chunks are then those of the rows' PieceRange -- without grant words their
// windows and sinks alone, wherever in the cache they are -- and a work-group
// takes every gridDim.x-th of them: 12 heads of 64, a window of 4096 behind
// 32768 positions 8.8 + 3.6 us, where a work-group for every chunk of the cache
// took 11.9 + 7.2.
#include "attn_kernels.h"

namespace t2t {

namespace {

constexpr int kDecThreads = 256;
constexpr int kDecChunk = 256;  // keys per work-group
constexpr int kDecHalf = 128;   // ... of a window, where its chunks are few (launch_both)

struct DecodeArgs {
  TensorView q, k, v;  // q [B][Hq][Tq][D]; k, v [B][Hkv][cap][D]
  const int32_t* key_doc;
  const uint64_t* key_bits;  // [Bm][W][key_stride]
  int64_t key_stride;
  const int32_t* q_pos;      // [Bm][Tq]
  const int32_t* q_doc;
  const uint64_t* q_bits;    // [Bm][W][Tq]
  int Bm, W, B, Hq, Hkv, Tq, Tkv, nch;
  float c;                   // scale * log2(e)
  float* part;               // [B][Hq][Tq][nch][D + 2]
  int window, sinks;         // window 0: none
  const int32_t* q_start;    // [Bm][Tq], or NULL without sinks
  bool half;                 // with a window: chunks of kDecHalf keys, if they fit
};

// Sum over the GL = D/8 lanes of a key group (8 or 16 adjacent, aligned
// lanes): DPP quad_perm [1,0,3,2] and [2,3,0,1] sum each quad, row_half_mirror
// adds the other quad of the 8-lane half row, row_mirror the other half of the
// 16-lane row.  Every lane of the group ends with the group's sum.
template <int GL>
__device__ __forceinline__ float group_sum(float x) {
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xB1, 0xF, 0xF, false));
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x4E, 0xF, 0xF, false));
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x141, 0xF, 0xF, false));
  if constexpr (GL == 16)
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x140, 0xF, 0xF, false));
  return x;
}

// RMAX: compile-time bound on the R query rows (1, 2, 4 or 8), so the common
// single-row step holds 8 + 8 accumulators per lane rather than 64 + 64.
template <int D, int RMAX, bool Win, int Chunk = kDecChunk>
__device__ __forceinline__ void decode_chunk(const DecodeArgs& a, int chunk, int slot) {
  constexpr int GL = D / 8;                    // lanes per key
  constexpr int NKG = kDecThreads / GL;        // key groups per work-group
  constexpr int KPG = Chunk / NKG;             // keys per group
  __shared__ float sc[RMAX][Chunk];            // scores (log2 units)
  __shared__ float red[kDecThreads / 64][RMAX][D];
  __shared__ float rmax[RMAX];
  __shared__ int32_t qpos_s[RMAX], qdoc_s[RMAX], qstart_s[RMAX];
  __shared__ uint64_t qbits_s[kMaxWords][RMAX];

  const int hk = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int dg = tid % GL, kg = tid / GL;
  const int G = a.Hq / a.Hkv;
  const int R = G * a.Tq;
  const int mb = a.Bm > 1 ? b : 0;
  const int j0 = chunk * Chunk;

  const __bf16* kbase = static_cast<const __bf16*>(a.k.data) + b * a.k.sb + hk * a.k.sh + 8 * dg;
  const __bf16* vbase = static_cast<const __bf16*>(a.v.data) + b * a.v.sb + hk * a.v.sh + 8 * dg;
  const int32_t* kdoc = a.key_doc + (size_t)mb * a.key_stride;
  const uint64_t* kbits = a.key_bits + (size_t)mb * a.W * a.key_stride;

  // The keys' doc ids and first grant word depend on nothing else: their
  // loads go out first, with the query rows' and the new rows' mask inputs.
  int dj[KPG];
  uint64_t kw0[KPG];
#pragma unroll
  for (int i = 0; i < KPG; ++i) {
    const int j = j0 + kg + NKG * i;
    dj[i] = j < a.Tkv ? kdoc[j] : 0;
    kw0[i] = (a.W > 0 && j < a.Tkv) ? kbits[j] : 0ull;
  }

  if (tid < a.Tq) {
    qpos_s[tid] = a.q_pos[(size_t)mb * a.Tq + tid];
    qdoc_s[tid] = a.q_doc[(size_t)mb * a.Tq + tid];
    if (Win) qstart_s[tid] = a.q_start ? a.q_start[(size_t)mb * a.Tq + tid] : 0;
    for (int w = 0; w < a.W; ++w)
      qbits_s[w][tid] = a.q_bits[((size_t)mb * a.W + w) * a.Tq + tid];
  }

  // Query rows r = g * Tq + tq (query head hk * G + g), elements 8 dg .. 8 dg + 7.
  float qf[RMAX][8];
#pragma unroll
  for (int r = 0; r < RMAX; ++r) {
    if (r < R) {
      const int g = r / a.Tq, tq = r - g * a.Tq;
      const __bf16* qp = static_cast<const __bf16*>(a.q.data) + b * a.q.sb +
                         (int64_t)(hk * G + g) * a.q.sh + (int64_t)tq * a.q.st + 8 * dg;
      const bf16x8 x = *reinterpret_cast<const bf16x8*>(qp);
#pragma unroll
      for (int e = 0; e < 8; ++e) qf[r][e] = (float)x[e] * a.c;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) qf[r][e] = 0.f;
    }
  }
  __syncthreads();

  // Mask of the group's keys j0 + kg + NKG i: bit tq of allow[i] = allowed for
  // new row tq.  Every load of a stage is issued before any is consumed, so a
  // stage costs one memory latency, not one per key.
  uint32_t allow[KPG];
  {
#pragma unroll
    for (int i = 0; i < KPG; ++i) allow[i] = 0;
    for (int tq = 0; tq < a.Tq; ++tq) {
      const int qd = qdoc_s[tq];
#pragma unroll
      for (int i = 0; i < KPG; ++i) {
        bool own = dj[i] == qd;
        if constexpr (Win) {
          const int64_t j = j0 + kg + NKG * i, at = j - qstart_s[tq];
          own = own && (qpos_s[tq] - j < a.window || (at >= 0 && at < a.sinks));
        }
        allow[i] |= (own ? 1u : 0u) << tq;
      }
    }
    for (int w = 0; w < a.W; ++w) {
      uint64_t kw[KPG];
#pragma unroll
      for (int i = 0; i < KPG; ++i) {
        const int j = j0 + kg + NKG * i;
        kw[i] = w == 0 ? kw0[i] : (j < a.Tkv ? kbits[(size_t)w * a.key_stride + j] : 0ull);
      }
      for (int tq = 0; tq < a.Tq; ++tq) {
        const uint64_t qw = qbits_s[w][tq];
#pragma unroll
        for (int i = 0; i < KPG; ++i) allow[i] |= ((qw & kw[i]) != 0ull ? 1u : 0u) << tq;
      }
    }
#pragma unroll
    for (int i = 0; i < KPG; ++i) {
      const int j = j0 + kg + NKG * i;
      uint32_t causal = 0;
      for (int tq = 0; tq < a.Tq; ++tq) causal |= (j <= qpos_s[tq] ? 1u : 0u) << tq;
      allow[i] = j < a.Tkv ? (allow[i] & causal) : 0u;
    }
  }

  // Pass 1: K and V rows of the allowed keys (both issued here: V depends
  // only on the mask), scores to LDS (-inf where masked).
  bf16x8 vx[KPG];
  {
    bf16x8 kx[KPG];
#pragma unroll
    for (int i = 0; i < KPG; ++i) {
      kx[i] = bf16x8{};
      vx[i] = bf16x8{};
      if (allow[i]) {
        kx[i] = *reinterpret_cast<const bf16x8*>(kbase + (int64_t)(j0 + kg + NKG * i) * a.k.st);
        vx[i] = *reinterpret_cast<const bf16x8*>(vbase + (int64_t)(j0 + kg + NKG * i) * a.v.st);
      }
    }
#pragma unroll
    for (int i = 0; i < KPG; ++i) {
      const int jl = kg + NKG * i;
#pragma unroll
      for (int r = 0; r < RMAX; ++r) {
        if (r < R) {
          float acc = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) acc = fmaf(qf[r][e], (float)kx[i][e], acc);
          // The lanes of a key group hold the same allow[i]; the sum runs on all.
          const float tot = group_sum<GL>(acc);
          if (dg == 0) sc[r][jl] = ((allow[i] >> (r % a.Tq)) & 1u) ? tot : -INFINITY;
        }
      }
    }
  }
  __syncthreads();

  // Chunk row max: wave w reduces rows w, w + 4.
  for (int r = wave; r < R; r += kDecThreads / 64) {
    float m = -INFINITY;
    for (int x = lane; x < Chunk; x += 64) m = fmaxf(m, sc[r][x]);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    if (lane == 0) rmax[r] = m;
  }
  __syncthreads();

  // Pass 2: o[r] = sum_j exp2(s - max) V[j], l[r] = sum_j exp2(s - max).
  float o[RMAX][8], l[RMAX];
#pragma unroll
  for (int r = 0; r < RMAX; ++r) {
    l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[r][e] = 0.f;
  }
  {
#pragma unroll
    for (int i = 0; i < KPG; ++i) {
      const int jl = kg + NKG * i;
#pragma unroll
      for (int r = 0; r < RMAX; ++r) {
        if (r < R) {
          const float sv = sc[r][jl];
          const float pr = sv == -INFINITY ? 0.f : fast_exp2(sv - rmax[r]);
          l[r] += pr;
#pragma unroll
          for (int e = 0; e < 8; ++e) o[r][e] = fmaf(pr, (float)vx[i][e], o[r][e]);
        }
      }
    }
  }
  // Sum over the key groups of a wave (lanes GL apart), then across waves.
#pragma unroll
  for (int r = 0; r < RMAX; ++r) {
    if (r < R) {
#pragma unroll
      for (int off = GL; off < 64; off <<= 1) {
        l[r] += __shfl_xor(l[r], off, 64);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[r][e] += __shfl_xor(o[r][e], off, 64);
      }
      if (lane < GL) {
#pragma unroll
        for (int e = 0; e < 8; ++e) red[wave][r][8 * dg + e] = o[r][e];
      }
    }
  }
  __shared__ float lsum[kDecThreads / 64][RMAX];
  if (lane == 0) {
#pragma unroll
    for (int r = 0; r < RMAX; ++r) lsum[wave][r] = l[r];
  }
  __syncthreads();
  for (int x = tid; x < R * (D + 2); x += kDecThreads) {
    const int r = x / (D + 2), col = x - r * (D + 2);
    const int g = r / a.Tq, tq = r - g * a.Tq;
    float val;
    if (col == 0) {
      val = rmax[r];
    } else if (col == 1) {
      val = 0.f;
      for (int w = 0; w < kDecThreads / 64; ++w) val += lsum[w][r];
    } else {
      val = 0.f;
      for (int w = 0; w < kDecThreads / 64; ++w) val += red[w][r][col - 2];
    }
    const size_t row = ((size_t)b * a.Hq + hk * G + g) * a.Tq + tq;
    a.part[(row * a.nch + slot) * (D + 2) + col] = val;
  }
}

// Chunks of the rows of sequence b (with a window).
template <int Chunk>
__device__ __forceinline__ PieceRange<Chunk> window_chunks(const DecodeArgs& a, int b) {
  const size_t row = (size_t)(a.Bm > 1 ? b : 0) * a.Tq;
  return PieceRange<Chunk>(a.q_pos + row, a.q_start ? a.q_start + row : nullptr, a.Tq, a.Tkv,
                           a.W == 0 ? a.window : 0, a.sinks);
}

// How many of kDecHalf keys; -1: chunks of kDecChunk (the workspace has a slot for
// each of the cache's, which rows far apart can pass in halves).
__device__ __forceinline__ int half_chunks(const DecodeArgs& a, int b) {
  if (!a.half) return -1;
  const int n = window_chunks<kDecHalf>(a, b).count;
  return n <= a.nch ? n : -1;
}

// Half: a.half, whose chunks the kernel has too.
template <int D, int RMAX, bool Win, bool Half>
__global__ __launch_bounds__(kDecThreads) void attn_decode_partial(DecodeArgs a) {
  if constexpr (Win) {
    if constexpr (Half) {
      const int n = half_chunks(a, blockIdx.z);
      if (n >= 0) {
        const auto half = window_chunks<kDecHalf>(a, blockIdx.z);
        for (int i = blockIdx.x; i < n; i += gridDim.x) {
          decode_chunk<D, RMAX, Win, kDecHalf>(a, half.at(i), i);
          __syncthreads();  // (its LDS is the next one's)
        }
        return;
      }
    }
    const auto range = window_chunks<kDecChunk>(a, blockIdx.z);
    for (int i = blockIdx.x; i < range.count; i += gridDim.x) {
      decode_chunk<D, RMAX, Win>(a, range.at(i), i);
      __syncthreads();
    }
  } else {
    decode_chunk<D, RMAX, Win>(a, blockIdx.x, blockIdx.x);
  }
}

// One wave per (new token, query head, batch row).  The chunk maxima load one
// chunk per lane; the weighted sum over chunks then issues its loads
// independently (eight in flight per lane), so the merge costs a few memory
// latencies whatever the chunk count.  With a window, whose chunks are few, the
// first kAhead values go out with the maxima, which they do not wait for (0.3 to
// 1 us of a call; none, or a loss of as much, at the 64 chunks of a 16k cache).
template <int D, bool Win>
__global__ __launch_bounds__(64) void attn_decode_combine(DecodeArgs a, TensorView o,
                                                          float* lse2) {
  constexpr int PER = D / 64;
  constexpr int S = D + 2;
  __shared__ float wsh[64];
  const int tq = blockIdx.x, h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x;
  const size_t row = ((size_t)b * a.Hq + h) * a.Tq + tq;
  const float* pr = a.part + row * a.nch * S;
  int chunks = a.nch;
  if constexpr (Win) {
    chunks = half_chunks(a, b);
    if (chunks < 0) chunks = window_chunks<kDecChunk>(a, b).count;
  }
  constexpr int kAhead = Win ? 32 / PER : 0;
  float ahead[kAhead + 1][PER];
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
#pragma unroll
    for (int e = 0; e < PER; ++e)
      ahead[k][e] = k < chunks ? pr[(size_t)k * S + 2 + lane + 64 * e] : 0.f;
  float M = -INFINITY;
  for (int c = lane; c < chunks; c += 64) M = fmaxf(M, pr[(size_t)c * S]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor(M, off, 64));
  float L = 0.f, acc[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) acc[e] = 0.f;
  if (M != -INFINITY) {
    for (int base = 0; base < chunks; base += 64) {
      const int c = base + lane;
      float w = 0.f;
      if (c < chunks) {
        const float m = pr[(size_t)c * S];
        w = m == -INFINITY ? 0.f : fast_exp2(m - M);
        L += w * pr[(size_t)c * S + 1];
      }
      wsh[lane] = w;
      __syncthreads();
      const int n = min(64, chunks - base);
      int k = 0;
      if (base == 0) {
#pragma unroll
        for (; k < kAhead; ++k)
          if (k < n) {
            const float wk = wsh[k];
#pragma unroll
            for (int e = 0; e < PER; ++e) acc[e] = fmaf(wk, ahead[k][e], acc[e]);
          }
      }
#pragma unroll 8
      for (; k < n; ++k) {
        const float wk = wsh[k];
#pragma unroll
        for (int e = 0; e < PER; ++e)
          acc[e] = fmaf(wk, pr[(size_t)(base + k) * S + 2 + lane + 64 * e], acc[e]);
      }
      __syncthreads();
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) L += __shfl_xor(L, off, 64);
  }
  const float inv = L > 0.f ? 1.f / L : 0.f;
  __bf16* op = static_cast<__bf16*>(o.data) + b * o.sb + h * o.sh + (int64_t)tq * o.st;
#pragma unroll
  for (int e = 0; e < PER; ++e) op[lane + 64 * e] = (__bf16)(acc[e] * inv);
  if (lane == 0) lse2[row] = L > 0.f ? M + log2f(L) : -INFINITY;
}

template <int D, bool Win, bool Half>
void launch_partial(int R, dim3 grid, const DecodeArgs& a, hipStream_t stream) {
  if (R <= 1)
    hipLaunchKernelGGL((attn_decode_partial<D, 1, Win, Half>), grid, dim3(kDecThreads), 0,
                       stream, a);
  else if (R <= 2)
    hipLaunchKernelGGL((attn_decode_partial<D, 2, Win, Half>), grid, dim3(kDecThreads), 0,
                       stream, a);
  else if (R <= 4)
    hipLaunchKernelGGL((attn_decode_partial<D, 4, Win, Half>), grid, dim3(kDecThreads), 0,
                       stream, a);
  else
    hipLaunchKernelGGL((attn_decode_partial<D, 8, Win, Half>), grid, dim3(kDecThreads), 0,
                       stream, a);
}

template <int D>
void launch_both(int R, DecodeArgs& a, const TensorView& o, float* lse2,
                 hipStream_t stream) {
  const dim3 pgrid((unsigned)a.nch, (unsigned)a.Hkv, (unsigned)a.B);
  const dim3 cgrid((unsigned)a.Tq, (unsigned)a.Hq, (unsigned)a.B);
  if (a.window > 0) {
    // a work-group for each chunk that rows next to one another read, which a
    // window or sinks may begin and end inside
    const auto touched = [&](int chunk) -> int64_t {
      if (a.W > 0) return a.nch;
      int64_t n = ((int64_t)a.window + a.Tq + chunk - 2) / chunk + 1;
      if (a.sinks > 0) n += ((int64_t)a.sinks + chunk - 2) / chunk + 1;
      return n;
    };
    // Halves of chunks where whole ones leave a quarter of the CUs without a
    // work-group: the time is then one's chain of loads and products; with more,
    // the halves' sums cost what they save.  us, chunks of 256 / 128 keys: 12
    // heads of 64, windows of 512 (36 work-groups) 10.9 / 9.6, 4096 (216) 12.2 /
    // 12.5, 16000 (768) 21.6 / 25.4; 32 / 8 heads of 128 (24, 144, 512) 24.2 /
    // 18.0, 25.5 / 21.2, 50.9 / 51.4.
    a.half = a.W == 0 && touched(kDecChunk) * a.Hkv * a.B <= 192;
    const int64_t n = touched(a.half ? kDecHalf : kDecChunk);
    const dim3 grid((unsigned)(n < a.nch ? n : a.nch), pgrid.y, pgrid.z);
    a.half ? launch_partial<D, true, true>(R, grid, a, stream)
           : launch_partial<D, true, false>(R, grid, a, stream);
    hipLaunchKernelGGL((attn_decode_combine<D, true>), cgrid, dim3(64), 0, stream, a, o, lse2);
  } else {
    launch_partial<D, false, false>(R, pgrid, a, stream);
    hipLaunchKernelGGL((attn_decode_combine<D, false>), cgrid, dim3(64), 0, stream, a, o, lse2);
  }
}

}  // namespace

int64_t decode_workspace_floats(int B, int Hq, int Tq, int Tkv, int D) {
  const int64_t nch = (Tkv + kDecChunk - 1) / kDecChunk;
  return (int64_t)B * Hq * Tq * (nch > 0 ? nch : 1) * (D + 2);
}

hipError_t launch_attn_decode(const TensorView& q, const TensorView& k, const TensorView& v,
                              const TensorView& o, float* lse2, const int32_t* key_doc,
                              const uint64_t* key_bits, int64_t key_stride, const int32_t* q_pos,
                              const int32_t* q_doc, const uint64_t* q_bits, int Bm, int W,
                              int B, int Hq, int Hkv, int Tq, int Tkv, int D, float scale,
                              int window, int sinks, const int32_t* q_start,
                              float* workspace, hipStream_t stream) {
  DecodeArgs a{q,     k,      v,    key_doc, key_bits, key_stride, q_pos, q_doc,
               q_bits, Bm,    W,    B,       Hq,       Hkv,        Tq,    Tkv,
               (Tkv + kDecChunk - 1) / kDecChunk, scale * kLog2e, workspace,
               window, sinks, q_start, false};
  if (a.nch == 0) a.nch = 1;  // no keys: one chunk that finds nothing
  const int R = (Hq / Hkv) * Tq;
  if (D == 64)
    launch_both<64>(R, a, o, lse2, stream);
  else
    launch_both<128>(R, a, o, lse2, stream);
  return hipGetLastError();
}

}  // namespace t2t
