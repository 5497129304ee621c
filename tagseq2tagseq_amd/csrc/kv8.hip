// A key/value cache held in 8 bits, and the attention of new rows over it.
//
// Keys and values are e4m3 numbers (4 exponent bits, 3 mantissa bits, largest
// 448) times a power of two for each block of 64 positions and head, keys and
// values apart.  Per (batch row, head, block): keys [64][D], values transposed
// [D][64], so that both are read in the order in which the matrix instructions
// take them (below) and a block is one run of memory.
//
// Append (kv8_append).  M tokens go to positions pos .. pos + M - 1; what stands
// behind them is no longer part of the sequence.  A block's scale becomes
//   max(its scale if it holds tokens before pos, 2^ceil(log2(amax / 448)))
// over its new tokens, and the tokens before pos are written again under it
// where it grew: the scale is a power of two, so their codes change in the
// exponent alone (only those that become subnormal lose bits).  Rounding is to
// nearest even, at most 2^-4 of a value or 2^-10 of the scale.  e4m3 rather
// than 8-bit integers because keys have channels of very different sizes: a
// channel 2^-6 of the block's largest value keeps its three bits, where an
// integer would have one left.  A token with a key or value that is not finite
// is stored as NaN keys and zero values: every row that reads it is NaN, no
// other row is touched.  HBM bound for prompts: 16384 tokens of 12 heads of 64
// 16.6 us, 4.5 TB/s of the tokens read and the codes written; one token is a
// launch and its memory latencies in turn, 5.1 us, also where its block's scale
// grows and the codes before it are written again.
//
// Attention (kv8_attend).  One work-group per (chunk of keys, kv head, batch
// row), R = G Tq <= 16 query rows (G query heads a kv head, Tq new tokens), each
// of its 4 to 16 waves on 64-key blocks of its own with a running maximum and sum.
// HBM bound: 2 D bytes a key and kv head.  From eight rows on the products alone
// (R multiply-adds a byte of the 64 a CU makes in a cycle) would take the vector
// units longer than memory takes for the byte, so they go to the matrix unit
// whatever R: S^T = K Q^T and O^T = V^T P^T as 16x16x32 bf16
// (e4m3 numbers are bf16 numbers, exactly, and p is taken as two of them, see
// below).  With A-operand row m of S tile t holding key
// 16 (m / 4) + 4 t + m % 4, lane (g, n) = (l / 16, l % 16) ends up with the
// scores of keys 16 g + 0 .. 15 for row n, which in this order are the B operand
// of the second product, whose A operand is then 16 neighbouring bytes of a row
// of V^T: no shuffle and no LDS between global memory and the products.
// Each (row, chunk) leaves (max, sum, unnormalised o[D]) for kv8_combine.  12
// heads of 64 over 32768 positions: 12.3 + 3.9 us, 4.1 TB/s; 16 sequences of 8192,
// 32 / 8 heads of 128, two tokens: 44 + 4.7 us, 6.1 TB/s (part of it from the
// last-level cache).  Through a window of 512 or 4096 behind the 32768 positions
// 5.9 + 3.5 and 6.6 + 3.3: the chunks are as many as the cache's length asks for,
// most of them without a block.
#include "attn_kernels.h"

namespace t2t {

namespace {

constexpr int kBlk = kKv8Block;

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// ---- append

__device__ __forceinline__ void load_row8(const __bf16* p, float (&x)[8]) {
  const bf16x8 v = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
}
__device__ __forceinline__ void load_row8(const float* p, float (&x)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

// 2^x with x the smallest exponent in [-120, 120] such that amax / 2^x <= 448.
__device__ __forceinline__ float scale_of(float amax) {
  const uint32_t u = __float_as_uint(amax);  // 448 = 1.75 * 2^8
  const int x = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffff) > 0x600000 ? 1 : 0);
  return __uint_as_float((uint32_t)(min(max(x, -120), 120) + 127) << 23);
}

__device__ __forceinline__ uint32_t encode4(const float* x) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
}

// Four codes under a scale that became 1 / r times as large.
__device__ __forceinline__ uint32_t rescale4(uint32_t c, float r) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false);
  const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  const float x[4] = {a.x * r, a.y * r, b.x * r, b.y * r};
  return encode4(x);
}

// grid (blocks that M tokens may touch, Hkv, B).  A work-group owns the block,
// so what it keeps of it can be read, changed and written in 16-byte pieces.
template <typename T, int D>
__global__ __launch_bounds__(256) void kv8_append_kernel(Kv8AppendArgs a) {
  constexpr int kRowPieces = D / 8;                    // 8-value pieces of a token
  constexpr int kPer = kBlk * kRowPieces / 256;        // pieces a thread
  constexpr int kPitch = kBlk + 16;                    // of a staged V^T row
  constexpr int kOut = kBlk * D / 16 / 256;            // 16-byte pieces a thread
  __shared__ __align__(16) uint8_t vs[D * kPitch];
  __shared__ float top[2][4];
  const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
  const int64_t pos = a.pos ? a.pos[b * a.pos_stride] : a.pos0;
  if (pos < 0 || pos > (int64_t)a.capacity - a.M) return;
  const int64_t blk = pos / kBlk + blockIdx.x;
  const int64_t first = blk * kBlk;
  const int lo = (int)(max(pos, first) - first);
  const int hi = (int)(min(pos + a.M, first + kBlk) - first);
  if (lo >= hi) return;
  const int64_t at = ((int64_t)b * a.Hkv + h) * a.blocks + blk;
  uint8_t* kc = a.k_codes + at * kBlk * D;
  uint8_t* vc = a.v_codes + at * kBlk * D;
  const T* k = static_cast<const T*>(a.k.data) + b * a.k.sb + h * a.k.sh;
  const T* v = static_cast<const T*>(a.v.data) + b * a.v.sb + h * a.v.sh;

  // Values are written in 16-byte pieces: tokens t0 .. t0 + 15 of a row of V^T.
  // What the block holds already in those with new and other tokens.
  const bool part = hi - lo < kBlk;
  const auto tokens = [&](int i) { return 16 * ((tid + 256 * i) % (kBlk / 16)); };
  uint4 vold[kOut];
  float kwas = 0.f, vwas = 0.f;
#pragma unroll
  for (int i = 0; i < kOut; ++i) {
    const int t0 = tokens(i);
    vold[i] = make_uint4(0u, 0u, 0u, 0u);
    if (part && t0 < hi && t0 + 16 > lo) vold[i] = reinterpret_cast<const uint4*>(vc)[tid + 256 * i];
  }
  if (lo > 0) {
    kwas = a.k_scale[at];
    vwas = a.v_scale[at];
  }
  float x[kPer][8], y[kPer][8];
  float km = 0.f, vm = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int row = (tid + 256 * i) / kRowPieces, c = 8 * ((tid + 256 * i) % kRowPieces);
    bool finite = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[i][e] = y[i][e] = 0.f;
    if (row >= lo && row < hi) {
      const int64_t t = first + row - pos;
      load_row8(k + t * a.k.st + c, x[i]);
      load_row8(v + t * a.v.st + c, y[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        finite = finite && fabsf(x[i][e]) <= 3.4028234663852886e38f &&
                 fabsf(y[i][e]) <= 3.4028234663852886e38f;
    }
    // (a token's lanes are neighbours in one wave)
    constexpr uint64_t kAll = (1ull << kRowPieces) - 1;
    const int shift = (tid & 63) / kRowPieces * kRowPieces;
    if (((__ballot(finite) >> shift) & kAll) == kAll) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        km = fmaxf(km, fabsf(x[i][e]));
        vm = fmaxf(vm, fabsf(y[i][e]));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[i][e] = __uint_as_float(0x7fc00000u);
        y[i][e] = 0.f;
      }
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    km = fmaxf(km, __shfl_xor(km, off, 64));
    vm = fmaxf(vm, __shfl_xor(vm, off, 64));
  }
  if ((tid & 63) == 0) {
    top[0][tid >> 6] = km;
    top[1][tid >> 6] = vm;
  }
  __syncthreads();
  const float know =
      fmaxf(kwas, scale_of(fmaxf(fmaxf(top[0][0], top[0][1]), fmaxf(top[0][2], top[0][3]))));
  const float vnow =
      fmaxf(vwas, scale_of(fmaxf(fmaxf(top[1][0], top[1][1]), fmaxf(top[1][2], top[1][3]))));
  // (scales are powers of two from 2^-120 to 2^120: exact, and their inverses too)
  const float kr = 1.f / know, vr = 1.f / vnow;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int row = (tid + 256 * i) / kRowPieces, c = 8 * ((tid + 256 * i) % kRowPieces);
    if (row < lo || row >= hi) continue;
    uint32_t kw[2], vw[2];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[i][e] *= kr;
      y[i][e] *= vr;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      kw[e] = encode4(x[i] + 4 * e);
      vw[e] = encode4(y[i] + 4 * e);
    }
    *reinterpret_cast<uint2*>(kc + row * D + c) = make_uint2(kw[0], kw[1]);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      vs[(c + e) * kPitch + row] = (uint8_t)(vw[e >> 2] >> (8 * (e & 3)));
  }
  const float kg = kwas * kr, vg = vwas * vr;  // 1 where the scale stayed
  if (kg != 1.f) {  // (the lo rows before the new ones)
    for (int p = tid; p < lo * (D / 16); p += 256) {
      const uint4 o = reinterpret_cast<const uint4*>(kc)[p];
      reinterpret_cast<uint4*>(kc)[p] =
          make_uint4(rescale4(o.x, kg), rescale4(o.y, kg), rescale4(o.z, kg), rescale4(o.w, kg));
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kOut; ++i) {
    const int p = tid + 256 * i, d = p / (kBlk / 16), t0 = tokens(i);
    const bool some = t0 < hi && t0 + 16 > lo;
    if (!some && (t0 >= hi || vg == 1.f)) continue;
    uint4 n = *reinterpret_cast<const uint4*>(vs + d * kPitch + t0);
    if (part) {
      const uint4 was = some ? vold[i] : reinterpret_cast<const uint4*>(vc)[p];
      const uint32_t o[4] = {was.x, was.y, was.z, was.w};
      uint32_t w[4] = {n.x, n.y, n.z, n.w};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t kept = vg == 1.f ? o[q] : rescale4(o[q], vg);
        uint32_t r = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = t0 + 4 * q + e;
          r |= (t < lo ? kept : t < hi ? w[q] : o[q]) & (0xffu << (8 * e));
        }
        w[q] = r;
      }
      n = make_uint4(w[0], w[1], w[2], w[3]);
    }
    reinterpret_cast<uint4*>(vc)[p] = n;
  }
  if (tid == 0) {
    a.k_scale[at] = know;
    a.v_scale[at] = vnow;
  }
}

// ---- attention

// Combined value of lanes l, l ^ 16, l ^ 32, l ^ 48 (one query row's lanes).
__device__ __forceinline__ float row_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return halves_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float row_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return halves_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// Eight codes as bf16 numbers.
__device__ __forceinline__ bf16x8 decode8(uint32_t a, uint32_t b) {
  const bf16x2 p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)a, 1.f, false);
  const bf16x2 q = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)a, 1.f, true);
  const bf16x2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)b, 1.f, false);
  const bf16x2 s = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)b, 1.f, true);
  return bf16x8{p.x, p.y, q.x, q.y, r.x, r.y, s.x, s.y};
}

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Split: the rows' value sums are taken over p rounded to bf16 and over what
// that rounding left, so that p counts with 16 bits.  Up to eight rows use half
// of the products' 16 columns, and the other half takes the rests (Twice false:
// column n + 8 is row n again); more rows take a second product.
template <int D, bool Twice, int Waves>
__global__ __launch_bounds__(64 * Waves) void kv8_attend_kernel(Kv8AttendArgs a) {
  constexpr int kPieces = D / 64;      // 16-byte pieces of a lane's part of a key
  constexpr int kTiles = D / 16;       // O^T tiles
  __shared__ __align__(16) float osum[Waves][16][D + 4];
  __shared__ float mls[Waves][2][16];
  __shared__ int32_t spos[16], sdoc[16], sstart[16];
  __shared__ uint64_t sbits[kMaxWords][16];
  const int chunk = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, column = lane & 15;
  const int n = Twice ? column : column & 7;  // query row
  const int G = a.Hq / a.Hkv, R = G * a.Tq;
  const int mb = a.Bm > 1 ? b : 0;
  if (tid < a.Tq) {
    spos[tid] = a.q_pos[(size_t)mb * a.Tq + tid];
    sdoc[tid] = a.q_doc[(size_t)mb * a.Tq + tid];
    sstart[tid] = a.q_start ? a.q_start[(size_t)mb * a.Tq + tid] : 0;
    for (int w = 0; w < a.W; ++w) sbits[w][tid] = a.q_bits[((size_t)mb * a.W + w) * a.Tq + tid];
  }
  // query row n = head * Tq + token: its part g of the dimensions
  const int tq_n = n % a.Tq;
  uint4 qraw[2 * kPieces] = {};
  if (n < R) {
    const __bf16* q = static_cast<const __bf16*>(a.q.data) + b * a.q.sb +
                      (int64_t)(hk * G + n / a.Tq) * a.q.sh + (int64_t)tq_n * a.q.st + g * (D / 4);
#pragma unroll
    for (int i = 0; i < 2 * kPieces; ++i) qraw[i] = reinterpret_cast<const uint4*>(q)[i];
  }
  __syncthreads();
  // The blocks that these rows read, in equal shares of whole rounds of the
  // waves.
  const PieceRange<kBlk> range(spos, a.q_start ? sstart : nullptr, a.Tq, a.Tkv,
                               a.W == 0 ? a.window : 0, a.sinks);
  const int share = Waves * ((range.count + Waves * a.chunks - 1) / (Waves * a.chunks));
  const int end = min((chunk + 1) * share, range.count);
  const size_t row0 = ((size_t)b * a.Hq + hk * G) * a.Tq;
  float* pml = a.part + (size_t)a.B * a.Hq * a.Tq * a.chunks * D;
  if (chunk * share >= range.count && a.chunks > 1) {  // no block: no sum either
    if (tid < R) {
      const size_t row = row0 + (size_t)(tid / a.Tq) * a.Tq + tid % a.Tq;
      pml[(row * a.chunks + chunk) * 2] = -INFINITY;
      pml[(row * a.chunks + chunk) * 2 + 1] = 0.f;
    }
    return;
  }
  bf16x8 qf[2 * kPieces];
#pragma unroll
  for (int i = 0; i < 2 * kPieces; ++i) qf[i] = *reinterpret_cast<const bf16x8*>(&qraw[i]);

  const int32_t* kdoc = a.key_doc + (size_t)mb * a.key_stride;
  const uint64_t* kbits = a.key_bits + (size_t)mb * a.W * a.key_stride;
  const int64_t head = ((int64_t)b * a.Hkv + hk) * a.blocks;
  const uint8_t* kc = a.k_codes + head * kBlk * D;
  const uint8_t* vc = a.v_codes + head * kBlk * D;
  const float* kscale = a.k_scale + head;
  const float* vscale = a.v_scale + head;

  f32x4 o[kTiles];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  // (a block's documents are loaded while the one before is worked on: 1 to 5 %
  // of a call)
  const auto doc_of = [&](int v) {
    const int j = range.at(v) * kBlk + lane;
    return v < end && j < a.Tkv ? kdoc[j] : 0;
  };
  int v = chunk * share + wave, next_doc = doc_of(v);
  for (; v < end; v += Waves) {
    const int blk = range.at(v);
    const int j = blk * kBlk + lane;
    const bool in = j < a.Tkv;
    const int jd = next_doc;
    next_doc = doc_of(v + Waves);
    uint64_t mine = 0;  // bit i: key i of the block is allowed for this lane's row
    uint64_t any = 0;
    for (int tq = 0; tq < a.Tq; ++tq) {
      const int64_t p = spos[tq];
      bool ok = jd == sdoc[tq];
      if (a.window > 0) {
        const int64_t s = j - (int64_t)sstart[tq];
        ok = ok && (p - j < a.window || (s >= 0 && s < a.sinks));
      }
      for (int w = 0; w < a.W; ++w)
        ok = ok || (sbits[w][tq] & (in ? kbits[(size_t)w * a.key_stride + j] : 0ull)) != 0ull;
      const uint64_t seen = __ballot(ok && in && j <= p);
      any |= seen;
      if (tq_n == tq) mine = seen;
    }
    if (!any) continue;
    const uint32_t allowed = n < R ? (uint32_t)(mine >> (16 * g)) & 0xffffu : 0u;

    uint4 kraw[4][kPieces], vraw[kTiles];
    const uint8_t* kp = kc + (int64_t)blk * kBlk * D +
                        (16 * (column >> 2) + (column & 3)) * D + g * (D / 4);
    const uint8_t* vp = vc + (int64_t)blk * kBlk * D + column * kBlk + 16 * g;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        kraw[t][i] = *reinterpret_cast<const uint4*>(kp + 4 * t * D + 16 * i);
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
      vraw[i] = *reinterpret_cast<const uint4*>(vp + i * 16 * kBlk);
    const float ks = kscale[blk] * a.c, vs = vscale[blk];
    // Where no row may look there may be anything, NaN codes too, and 0 * NaN is
    // NaN: zeros there.
    if (any != ~0ull) {
      const uint32_t some = (uint32_t)(any >> (16 * g));
      uint32_t keep[4];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        keep[q] = (((some >> (4 * q)) & 0xfu) * 0x204081u & 0x1010101u) * 0xffu;
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
        vraw[i] = make_uint4(vraw[i].x & keep[0], vraw[i].y & keep[1], vraw[i].z & keep[2],
                             vraw[i].w & keep[3]);
    }

    float s[16];
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        acc = mfma16(decode8(kraw[t][i].x, kraw[t][i].y), qf[2 * i], acc);
        acc = mfma16(decode8(kraw[t][i].z, kraw[t][i].w), qf[2 * i + 1], acc);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = 4 * t + i;
        s[e] = (allowed >> e) & 1u ? acc[i] * ks : -INFINITY;
        top = fmaxf(top, s[e]);
      }
    }
    const float now = fmaxf(m, row_max(top));
    // (a row that has seen no key yet: any finite reference, its terms are 0)
    const float ref = now == -INFINITY ? 0.f : now;
    if (__any(now != m)) {
      const float keep = fast_exp2(m - ref);
      l *= keep;
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] *= keep;
      m = now;
    }
    bf16x8 p[2], rest[2];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float x = fast_exp2(s[e] - ref);
      l += x;
      const float y = x * vs;
      const __bf16 hi = (__bf16)y;
      const __bf16 lo = (__bf16)(y - (float)hi);
      p[e >> 3][e & 7] = Twice || column < 8 ? hi : lo;
      if (Twice) rest[e >> 3][e & 7] = lo;
    }
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const bf16x8 v0 = decode8(vraw[i].x, vraw[i].y), v1 = decode8(vraw[i].z, vraw[i].w);
      o[i] = mfma16(v0, p[0], o[i]);
      o[i] = mfma16(v1, p[1], o[i]);
      if (Twice) {
        o[i] = mfma16(v0, rest[0], o[i]);
        o[i] = mfma16(v1, rest[1], o[i]);
      }
    }
  }

  // The waves' sums of a row, joined.  Lane (g, column) holds
  // o[16 i + 4 g + e] of its column.
  l = row_sum(l);
  if (g == 0) {
    mls[wave][0][column] = m;
    mls[wave][1][column] = l;
  }
#pragma unroll
  for (int i = 0; i < kTiles; ++i)
    *reinterpret_cast<f32x4*>(&osum[wave][column][16 * i + 4 * g]) = o[i];
  __syncthreads();
  for (int x = tid; x < R * D; x += 64 * Waves) {
    const int r = x / D, d = x - r * D;
    float M = mls[0][0][r];
#pragma unroll
    for (int w = 1; w < Waves; ++w) M = fmaxf(M, mls[w][0][r]);
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < Waves; ++w) {
      const float f = fast_exp2(mls[w][0][r] - ref);
      L = fmaf(f, mls[w][1][r], L);
      sum = fmaf(f, Twice ? osum[w][r][d] : osum[w][r][d] + osum[w][r + 8][d], sum);
    }
    const int hq = hk * G + r / a.Tq, tq = r % a.Tq;
    const size_t row = ((size_t)b * a.Hq + hq) * a.Tq + tq;
    if (a.chunks == 1) {  // the whole row: no second pass
      // (a sum of NaN is a row's result, one of 0 a row without keys)
      const float inv = L == 0.f ? 0.f : 1.f / L;
      static_cast<__bf16*>(a.o.data)[b * a.o.sb + hq * a.o.sh + (int64_t)tq * a.o.st + d] =
          (__bf16)(sum * inv);
      if (d == 0) a.lse2[row] = L == 0.f ? -INFINITY : M + log2f(L);
    } else {
      a.part[(row * a.chunks + chunk) * D + d] = sum;
      if (d == 0) {
        pml[(row * a.chunks + chunk) * 2] = M;
        pml[(row * a.chunks + chunk) * 2 + 1] = L;
      }
    }
  }
}

// One work-group per (new token, query head, batch row).  A lane holds one
// chunk's (maximum, sum), so that every wave has all weights without LDS; the
// sums are taken D / 4 lanes a chunk, and all of a lane's loads go out before
// any is used: one memory latency whatever the number of chunks.
constexpr int kMaxChunks = 64;

template <int D>
__global__ __launch_bounds__(256) void kv8_combine_kernel(Kv8AttendArgs a) {
  constexpr int kLanes = D / 4, kSlots = 256 / kLanes, kRounds = kMaxChunks / kSlots;
  __shared__ __align__(16) float osh[4][D];
  const int tq = blockIdx.x, hq = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const size_t row = ((size_t)b * a.Hq + hq) * a.Tq + tq;
  const float* part = a.part + row * a.chunks * D;
  const float* ml = a.part + (size_t)a.B * a.Hq * a.Tq * a.chunks * D + row * a.chunks * 2;
  float2 own = make_float2(-INFINITY, 0.f);
  if (lane < a.chunks) own = reinterpret_cast<const float2*>(ml)[lane];
  float4 v[kRounds];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int c = tid / kLanes + i * kSlots;
    v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < a.chunks)
      v[i] = *reinterpret_cast<const float4*>(part + (size_t)c * D + 4 * (tid % kLanes));
  }
  float M = own.x;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor(M, off, 64));
  const float w = fast_exp2(own.x - (M == -INFINITY ? 0.f : M));
  float L = w * own.y;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) L += __shfl_xor(L, off, 64);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const float f = __shfl(w, (tid / kLanes + i * kSlots) & 63, 64);
    if (f != 0.f) {  // (a chunk without a key has left no sums)
      acc.x = fmaf(f, v[i].x, acc.x);
      acc.y = fmaf(f, v[i].y, acc.y);
      acc.z = fmaf(f, v[i].z, acc.z);
      acc.w = fmaf(f, v[i].w, acc.w);
    }
  }
#pragma unroll
  for (int off = kLanes; off < 64; off <<= 1) {
    acc.x += __shfl_xor(acc.x, off, 64);
    acc.y += __shfl_xor(acc.y, off, 64);
    acc.z += __shfl_xor(acc.z, off, 64);
    acc.w += __shfl_xor(acc.w, off, 64);
  }
  if (lane < kLanes) *reinterpret_cast<float4*>(&osh[wave][4 * lane]) = acc;
  __syncthreads();
  if (tid < D) {
    const float sum = (osh[0][tid] + osh[1][tid]) + (osh[2][tid] + osh[3][tid]);
    const float inv = L == 0.f ? 0.f : 1.f / L;
    static_cast<__bf16*>(a.o.data)[b * a.o.sb + hq * a.o.sh + (int64_t)tq * a.o.st + tid] =
        (__bf16)(sum * inv);
  }
  if (tid == 0) a.lse2[row] = L == 0.f ? -INFINITY : M + log2f(L);
}

// Work-groups that the attention aims at: four for each CU, so that one's loads
// run under another's products.
constexpr int kAimGroups = 1024;

// Waves of a work-group that takes a whole row's keys in one pass where each
// wave has one block at most: 12 heads of 64, 512 / 1024 / 2048 keys 5.3 / 6.6 /
// 9.5 us against 6.8 / 6.9 / 6.9 in chunks and two passes (a wave's second block
// costs what the second pass does); 16 x 8 heads of 128, 512 keys 7.2 against 8.9.
template <int D>
constexpr int kWideWaves = D == 64 ? 16 : 8;

bool one_pass(int Tkv, int D) {
  return Tkv <= kBlk * (D == 64 ? kWideWaves<64> : kWideWaves<128>);
}

template <int D, bool Twice>
void start_attend(const Kv8AttendArgs& a, hipStream_t stream) {
  const dim3 grid(a.chunks, a.Hkv, a.B);
  if (one_pass(a.Tkv, D) && a.Tkv > 4 * kBlk)
    hipLaunchKernelGGL((kv8_attend_kernel<D, Twice, kWideWaves<D>>), grid,
                       dim3(64 * kWideWaves<D>), 0, stream, a);
  else
    hipLaunchKernelGGL((kv8_attend_kernel<D, Twice, 4>), grid, dim3(256), 0, stream, a);
}

}  // namespace

// Chunks of a row's keys: as many as fill the aim, at most one for each round of
// the waves' blocks and as many as the second pass has lanes.
int kv8_chunks(int B, int Hkv, int Tkv, int D) {
  if (one_pass(Tkv, D)) return 1;
  const int rounds = (Tkv + 4 * kBlk - 1) / (4 * kBlk);
  const int64_t pairs = (int64_t)B * Hkv;
  const int64_t want = pairs > 0 ? (kAimGroups + pairs - 1) / pairs : 1;
  const int n = (int)(want < kMaxChunks ? want : kMaxChunks);
  return n < rounds ? n : rounds;
}

hipError_t launch_kv8_append(const Kv8AppendArgs& a, bool f32, int D, hipStream_t stream) {
  // from an unknown position M tokens may touch one block more than from a
  // block's start
  const int64_t touched = a.pos ? (a.M + kBlk - 2) / kBlk + 1
                                : (a.pos0 + a.M - 1) / kBlk - a.pos0 / kBlk + 1;
  const dim3 grid((unsigned)touched, a.Hkv, a.B);
  if (f32 && D == 64)
    hipLaunchKernelGGL((kv8_append_kernel<float, 64>), grid, dim3(256), 0, stream, a);
  else if (f32)
    hipLaunchKernelGGL((kv8_append_kernel<float, 128>), grid, dim3(256), 0, stream, a);
  else if (D == 64)
    hipLaunchKernelGGL((kv8_append_kernel<__bf16, 64>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((kv8_append_kernel<__bf16, 128>), grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_kv8_attend(Kv8AttendArgs a, int D, hipStream_t stream) {
  a.chunks = kv8_chunks(a.B, a.Hkv, a.Tkv, D);
  const bool twice = a.Hq / a.Hkv * a.Tq > 8;
  if (D == 64)
    twice ? start_attend<64, true>(a, stream) : start_attend<64, false>(a, stream);
  else
    twice ? start_attend<128, true>(a, stream) : start_attend<128, false>(a, stream);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.chunks == 1) return e;
  const dim3 rows(a.Tq, a.Hq, a.B);
  if (D == 64)
    hipLaunchKernelGGL(kv8_combine_kernel<64>, rows, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(kv8_combine_kernel<128>, rows, dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace t2t
