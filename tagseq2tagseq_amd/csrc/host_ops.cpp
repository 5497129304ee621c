// Host side of the per-layer calls, in C++: output allocation, the argument
// blocks of libt2t_attn.so's C entry points and the launch, on the tensors'
// own device and its current stream.
//
// What bounds it: a layer of a short sequence is host work -- at 512 tokens a
// forward and backward issue about fifty launches whose kernels take 0.26 ms,
// and through ctypes each of these wrappers cost 10 to 25 us (stream and
// device context objects, argument structures, tensor methods).  Here one
// costs 3 to 8 us: B1 H4 T1024 D64 float32 forward 29.7 -> 12.8 us a call,
// bf16 forward + backward at T 1537 156 -> 88, the mask of a 16k row 106 ->
// 64, a layer of 512 x 512 forward + backward 950 -> 750, twelve layers over
// 2048 tokens 3710 -> 2460.  The functions keep nothing from one call to the
// next.
#include <ATen/SavedTensorHooks.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <cmath>
#include <cstdint>
#include <tuple>
#include <vector>

#include "../../include/t2t_attn.h"

namespace {

using at::Tensor;

void* stream_of(const Tensor& t) {
  return at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

void check(int rc, const char* what) {
  TORCH_CHECK(rc == T2T_OK, what, " failed (status ", rc, "): ", t2t_last_error());
}

// The kernels get plain addresses: one of host memory would fault the GPU.
template <typename... Ts>
void need_gpu(const Ts&... t) {
  TORCH_CHECK((t.is_cuda() && ...), "the gfx950 kernels need ROCm GPU tensors");
}

int weight_code(const Tensor& w) {
  TORCH_CHECK(w.scalar_type() == at::kBFloat16 || w.scalar_type() == at::kFloat,
              "weight dtype ", w.scalar_type(), " (bfloat16 or float32)");
  return w.scalar_type() == at::kFloat ? T2T_DTYPE_F32 : T2T_DTYPE_BF16;
}

// The attention kernels' code of q's dtype, which k, v and (backward) out and
// dout share: the kernels read what the code says, whatever the tensors hold.
template <typename... Ts>
int attention_code(const Tensor& q, const Ts&... others) {
  const at::ScalarType t = q.scalar_type();
  TORCH_CHECK_NOT_IMPLEMENTED(t == at::kBFloat16 || t == at::kFloat, "dtype ", t,
                              " is not supported (bfloat16 or float32)");
  TORCH_CHECK_VALUE(((others.scalar_type() == t) && ...), "attention operands differ in dtype");
  return t == at::kFloat ? T2T_DTYPE_F32 : T2T_DTYPE_BF16;
}

// [B, H, T, D] with unit stride along D; a dimension of size 1 is never stepped.
t2t_tensor view4(const Tensor& t) {
  TORCH_CHECK_VALUE(t.dim() == 4, "expected a 4-D [B, H, T, D] tensor, got shape ", t.sizes());
  TORCH_CHECK_VALUE(t.stride(3) == 1, "the head dimension (last) must have unit stride");
  return t2t_tensor{t.data_ptr(), t.size(0) == 1 ? 0 : t.stride(0),
                    t.size(1) == 1 ? 0 : t.stride(1), t.stride(2)};
}

// The rows [N, C] of t's last dimension as the kernels read them: unit column
// stride, row stride a multiple of 8 elements and a 16-byte aligned start;
// anything else is copied (rows that are contiguous but start between two such
// boundaries too, which contiguous() would hand back).
Tensor rows_of(const Tensor& t) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  const bool ok = r.stride(1) == 1 && r.stride(0) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(r.data_ptr()) % 16 == 0;
  return ok ? r : r.clone(at::MemoryFormat::Contiguous);
}

const t2t_block_mask* mask_at(int64_t address) {
  return reinterpret_cast<const t2t_block_mask*>(static_cast<intptr_t>(address));
}

// ---- attention (mask: address of the caller's t2t_block_mask, alive during the call)

// rest: with what rounding left of a bf16 out (else undefined), for attn_bwd
std::tuple<Tensor, Tensor, Tensor> attn_fwd_rest(const Tensor& q, const Tensor& k,
                                                 const Tensor& v, int64_t mask, double scale,
                                                 bool rest) {
  const int dtype = attention_code(q, k, v);
  need_gpu(q, k, v);
  const c10::DeviceGuard guard(q.device());
  const int64_t B = q.size(0), Hq = q.size(1), T = q.size(2), D = q.size(3), Hkv = k.size(1);
  // [B, T, Hq, D] storage seen as [B, Hq, T, D]: the module's output
  // projection then reads token rows without a transpose copy
  Tensor out = at::empty({B, T, Hq, D}, q.options()).transpose(1, 2);
  Tensor lse2 = at::empty({B, Hq, T}, q.options().dtype(at::kFloat));
  const t2t_tensor qs = view4(q), ks = view4(k), vs = view4(v), os = view4(out);
  if (rest && dtype == T2T_DTYPE_BF16) {
    Tensor left = at::empty_like(out);
    const t2t_tensor rs = view4(left);
    check(t2t_attn_fwd_rest(&qs, &ks, &vs, &os, &rs, lse2.data_ptr<float>(), B, Hq, Hkv, T, D,
                            dtype, static_cast<float>(scale), mask_at(mask), stream_of(q)),
          "t2t_attn_fwd_rest");
    return {out, lse2, left};
  }
  check(t2t_attn_fwd(&qs, &ks, &vs, &os, lse2.data_ptr<float>(), B, Hq, Hkv, T, D,
                     dtype, static_cast<float>(scale), mask_at(mask), stream_of(q)),
        "t2t_attn_fwd");
  return {out, lse2, Tensor()};
}

std::tuple<Tensor, Tensor> attn_fwd(const Tensor& q, const Tensor& k, const Tensor& v,
                                    int64_t mask, double scale) {
  auto [out, lse2, none] = attn_fwd_rest(q, k, v, mask, scale, false);
  return {out, lse2};
}

// uneven: t2t_attn_bwd_uneven, or t2t_attn_bwd_rest where no column can be long;
// with rest where the forward has left one
std::tuple<Tensor, Tensor, Tensor> attn_bwd(const Tensor& q, const Tensor& k, const Tensor& v,
                                            const Tensor& out, const Tensor& dout_in,
                                            const Tensor& lse2, int64_t mask, double scale,
                                            bool uneven, const c10::optional<Tensor>& rest) {
  const int dtype = attention_code(q, k, v, out, dout_in);
  need_gpu(q, k, v, out, dout_in, lse2);
  const c10::DeviceGuard guard(q.device());
  const int64_t B = q.size(0), Hq = q.size(1), T = q.size(2), D = q.size(3), Hkv = k.size(1);
  const Tensor dout = dout_in.stride(3) == 1 ? dout_in : dout_in.contiguous();
  Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()),
         dv = at::empty(v.sizes(), v.options());
  Tensor delta = at::empty({B, Hq, T}, q.options().dtype(at::kFloat));
  const t2t_tensor qs = view4(q), ks = view4(k), vs = view4(v), os = view4(out),
                   ds = view4(dout), dqs = view4(dq), dks = view4(dk), dvs = view4(dv);
  if (uneven) {
    t2t_tensor rs{};
    if (rest.has_value()) {
      need_gpu(*rest);
      TORCH_CHECK_VALUE(rest->sizes() == out.sizes() && rest->scalar_type() == out.scalar_type(),
                        "rest ", rest->sizes(), " ", rest->scalar_type(), " is not out's");
      rs = view4(*rest);
    }
    const t2t_tensor* left = rest.has_value() ? &rs : nullptr;
    if (t2t_attn_bwd_uneven_pieces(B, Hq, Hkv, T, D, dtype) == 1) {
      check(t2t_attn_bwd_rest(&qs, &ks, &vs, &os, left, &ds, lse2.data_ptr<float>(),
                              delta.data_ptr<float>(), &dqs, &dks, &dvs, B, Hq, Hkv, T, D, dtype,
                              static_cast<float>(scale), mask_at(mask), stream_of(q)),
            "t2t_attn_bwd_rest");
      return {dq, dk, dv};
    }
    const int64_t bytes = t2t_attn_bwd_uneven_workspace(B, Hkv, T, D, dtype);
    Tensor ws = at::empty({bytes / 4}, delta.options());
    check(t2t_attn_bwd_uneven(&qs, &ks, &vs, &os, left, &ds, lse2.data_ptr<float>(),
                              delta.data_ptr<float>(), &dqs, &dks, &dvs, B, Hq, Hkv, T, D, dtype,
                              static_cast<float>(scale), mask_at(mask), ws.data_ptr(), bytes,
                              stream_of(q)),
          "t2t_attn_bwd_uneven");
    return {dq, dk, dv};
  }
  check(t2t_attn_bwd(&qs, &ks, &vs, &os, &ds, lse2.data_ptr<float>(), delta.data_ptr<float>(),
                     &dqs, &dks, &dvs, B, Hq, Hkv, T, D, dtype,
                     static_cast<float>(scale), mask_at(mask), stream_of(q)),
        "t2t_attn_bwd");
  return {dq, dk, dv};
}

// ---- RMS normalisation

std::tuple<Tensor, Tensor> rms_norm(const Tensor& x, const Tensor& weight, double eps) {
  need_gpu(x, weight);
  const c10::DeviceGuard guard(x.device());
  const int64_t C = x.size(-1);
  const Tensor xr = rows_of(x), w = weight.contiguous();
  const int64_t N = xr.size(0);
  Tensor y = at::empty(x.sizes(), x.options());
  Tensor rstd = at::empty({N}, x.options().dtype(at::kFloat));
  check(t2t_rms_norm(xr.data_ptr(), xr.stride(0), w.data_ptr(), weight_code(w), y.data_ptr(), C,
                     rstd.data_ptr<float>(), N, C, static_cast<float>(eps), stream_of(x)),
        "t2t_rms_norm");
  return {y, rstd};
}

std::tuple<Tensor, Tensor> rms_norm_backward(const Tensor& dy, const Tensor& x,
                                             const Tensor& weight, const Tensor& rstd) {
  need_gpu(dy, x, weight, rstd);
  const c10::DeviceGuard guard(x.device());
  const int64_t C = x.size(-1);
  const Tensor xr = rows_of(x), dyr = rows_of(dy), w = weight.contiguous();
  const int64_t N = xr.size(0);
  Tensor dx = at::empty(x.sizes(), x.options());
  Tensor dw = at::empty(w.sizes(), w.options());
  const int64_t bytes = t2t_rms_norm_backward_workspace(N, C);
  Tensor ws = at::empty({std::max<int64_t>(1, bytes / 4)}, x.options().dtype(at::kFloat));
  check(t2t_rms_norm_backward(dyr.data_ptr(), dyr.stride(0), xr.data_ptr(), xr.stride(0),
                              w.data_ptr(), weight_code(w), rstd.data_ptr<float>(), dx.data_ptr(),
                              C, dw.data_ptr(), ws.data_ptr(), ws.numel() * 4, N, C,
                              stream_of(x)),
        "t2t_rms_norm_backward");
  return {dx, dw};
}

// ---- QKV split + rotary embedding

std::tuple<Tensor, Tensor, Tensor> qkv_rope(const Tensor& qkv_in, const Tensor& cos_in,
                                            const Tensor& sin_in, int64_t heads, int64_t pos0) {
  TORCH_CHECK_VALUE(qkv_in.dim() == 3, "qkv must be [B, T, 3 C], got shape ", qkv_in.sizes());
  TORCH_CHECK_VALUE(heads > 0, "num_heads=", heads, " must be positive");
  TORCH_CHECK_VALUE(qkv_in.size(2) % (3 * heads) == 0, "last dim ", qkv_in.size(2),
                    " is not 3 * num_heads * head_dim (num_heads=", heads, ")");
  TORCH_CHECK_NOT_IMPLEMENTED(qkv_in.scalar_type() == at::kBFloat16, "qkv dtype ",
                              qkv_in.scalar_type(), " is not supported (bfloat16 only)");
  need_gpu(qkv_in, cos_in, sin_in);
  const c10::DeviceGuard guard(qkv_in.device());
  const Tensor qkv = qkv_in.stride(2) == 1 ? qkv_in : qkv_in.contiguous();
  const Tensor cos = cos_in.contiguous(), sin = sin_in.contiguous();
  const int64_t B = qkv.size(0), T = qkv.size(1), D = qkv.size(2) / (3 * heads);
  Tensor q = at::empty({B, heads, T, D}, qkv.options()), k = at::empty_like(q),
         v = at::empty_like(q);
  const t2t_tensor qs{q.data_ptr(), q.stride(0), q.stride(1), q.stride(2)},
      ks{k.data_ptr(), k.stride(0), k.stride(1), k.stride(2)},
      vs{v.data_ptr(), v.stride(0), v.stride(1), v.stride(2)};
  check(t2t_qkv_rope(qkv.data_ptr(), qkv.stride(0), qkv.stride(1), B, T, heads, D,
                     cos.data_ptr<float>(), sin.data_ptr<float>(), cos.size(0), pos0, &qs, &ks,
                     &vs, stream_of(qkv)),
        "t2t_qkv_rope");
  return {q, k, v};
}

Tensor qkv_rope_backward(const Tensor& dq_in, const Tensor& dk_in, const Tensor& dv_in,
                         const Tensor& cos_in, const Tensor& sin_in, int64_t pos0) {
  for (const Tensor* t : {&dq_in, &dk_in, &dv_in})
    TORCH_CHECK_VALUE(t->dim() == 4, "expected a 4-D [B, H, T, D] gradient, got shape ",
                      t->sizes());
  need_gpu(dq_in, dk_in, dv_in, cos_in, sin_in);
  const c10::DeviceGuard guard(dq_in.device());
  const int64_t B = dq_in.size(0), H = dq_in.size(1), T = dq_in.size(2), D = dq_in.size(3);
  const Tensor dq = dq_in.stride(3) == 1 ? dq_in : dq_in.contiguous();
  const Tensor dk = dk_in.stride(3) == 1 ? dk_in : dk_in.contiguous();
  const Tensor dv = dv_in.stride(3) == 1 ? dv_in : dv_in.contiguous();
  const Tensor cos = cos_in.contiguous(), sin = sin_in.contiguous();
  Tensor dqkv = at::empty({B, T, 3 * H * D}, dq.options());
  const t2t_tensor qs{dq.data_ptr(), dq.stride(0), dq.stride(1), dq.stride(2)},
      ks{dk.data_ptr(), dk.stride(0), dk.stride(1), dk.stride(2)},
      vs{dv.data_ptr(), dv.stride(0), dv.stride(1), dv.stride(2)};
  check(t2t_qkv_rope_backward(&qs, &ks, &vs, cos.data_ptr<float>(), sin.data_ptr<float>(),
                              cos.size(0), pos0, B, T, H, D, dqkv.data_ptr(), dqkv.stride(0),
                              dqkv.stride(1), stream_of(dq)),
        "t2t_qkv_rope_backward");
  return dqkv;
}

// ---- QKV split + norms of queries and keys + rotary embedding

// bfloat16 or float32 rows as the kernels read them: unit stride along the
// last dimension, the other strides (of dimensions that are stepped) and the
// start on 16-byte boundaries; anything else is copied.
Tensor vector_rows(const Tensor& t) {
  const int64_t align = 16 / t.element_size();
  bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t d = 0; d + 1 < t.dim(); ++d)
    ok = ok && (t.size(d) == 1 || (t.stride(d) >= 0 && t.stride(d) % align == 0));
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

t2t_tensor heads_of(const Tensor& t) {
  const auto stride = [&](int d) { return t.size(d) == 1 ? 0 : t.stride(d); };
  return t2t_tensor{t.data_ptr(), stride(0), stride(1), stride(2)};
}

// What the three calls below take, checked: the packed rows (copied where the
// kernels cannot read them), weights and tables.
struct QkNorm {
  Tensor qkv, qw, kw, cos, sin;
  int64_t B, T, H, Hkv, D, sb, st;
  int code, wcode;
  QkNorm(const Tensor& qkv_in, const Tensor& qw_in, const Tensor& kw_in, const Tensor& cos_in,
         const Tensor& sin_in, int64_t heads, int64_t kv_heads, double eps) {
    TORCH_CHECK_VALUE(qkv_in.dim() == 3, "qkv must be [B, T, (H + 2 Hkv) D], got shape ",
                      qkv_in.sizes());
    TORCH_CHECK_VALUE(heads > 0 && kv_heads > 0, "num_heads=", heads, " and num_kv_heads=",
                      kv_heads, " must be positive");
    H = heads;
    Hkv = kv_heads;
    // (as a quotient: twice a huge count would not fit)
    TORCH_CHECK_VALUE(H <= qkv_in.size(2) && Hkv <= qkv_in.size(2) &&
                          qkv_in.size(2) % (H + 2 * Hkv) == 0,
                      "last dim ", qkv_in.size(2), " is not (num_heads + 2 num_kv_heads) * "
                      "head_dim (num_heads=", H, ", num_kv_heads=", Hkv, ")");
    TORCH_CHECK_NOT_IMPLEMENTED(
        qkv_in.scalar_type() == at::kBFloat16 || qkv_in.scalar_type() == at::kFloat, "qkv dtype ",
        qkv_in.scalar_type(), " is not supported (bfloat16 or float32)");
    D = qkv_in.size(2) / (H + 2 * Hkv);
    TORCH_CHECK_VALUE(qw_in.dim() == 1 && qw_in.size(0) == D && kw_in.sizes() == qw_in.sizes(),
                      "q_weight ", qw_in.sizes(), " and k_weight ", kw_in.sizes(),
                      " must be [head_dim] = [", D, "]");
    TORCH_CHECK_VALUE(qw_in.scalar_type() == kw_in.scalar_type(),
                      "q_weight and k_weight differ in dtype");
    TORCH_CHECK_VALUE(cos_in.dim() == 2 && cos_in.size(1) * 2 == D &&
                          sin_in.sizes() == cos_in.sizes() &&
                          cos_in.scalar_type() == at::kFloat &&
                          sin_in.scalar_type() == at::kFloat,
                      "cos ", cos_in.sizes(), " and sin ", sin_in.sizes(),
                      " must be float32 [rows, head_dim / 2]");
    TORCH_CHECK_VALUE(eps >= 0 && std::isfinite(eps), "eps=", eps);
    need_gpu(qkv_in, qw_in, kw_in, cos_in, sin_in);
    for (const Tensor* t : {&qw_in, &kw_in, &cos_in, &sin_in})
      TORCH_CHECK_VALUE(t->device() == qkv_in.device(), "operands on different devices");
    const c10::DeviceGuard guard(qkv_in.device());
    code = qkv_in.scalar_type() == at::kFloat ? T2T_DTYPE_F32 : T2T_DTYPE_BF16;
    wcode = weight_code(qw_in);
    qkv = vector_rows(qkv_in);
    qw = vector_rows(qw_in.contiguous());
    kw = vector_rows(kw_in.contiguous());
    cos = vector_rows(cos_in.contiguous());
    sin = vector_rows(sin_in.contiguous());
    B = qkv.size(0);
    T = qkv.size(1);
    sb = B == 1 ? 0 : qkv.stride(0);
    st = T == 1 ? 0 : qkv.stride(1);
    TORCH_CHECK_VALUE(B <= INT32_MAX && T <= INT32_MAX && H <= INT32_MAX && D <= INT32_MAX,
                      "qkv ", qkv.sizes(), " is too large");
  }
  int64_t rows() const { return std::min<int64_t>(cos.size(0), INT32_MAX); }
  int64_t first(int64_t pos0) const {
    TORCH_CHECK_VALUE(pos0 >= 0 && pos0 <= rows() && pos0 + T <= rows(), "positions ", pos0,
                      " .. ", pos0 + T - 1, " exceed the ", rows(), " table rows");
    return pos0;
  }
};

std::tuple<Tensor, Tensor, Tensor> qk_norm_rope(const Tensor& qkv_in, const Tensor& q_weight,
                                                const Tensor& k_weight, const Tensor& cos_in,
                                                const Tensor& sin_in, int64_t heads,
                                                int64_t kv_heads, int64_t pos0, double eps) {
  const QkNorm a(qkv_in, q_weight, k_weight, cos_in, sin_in, heads, kv_heads, eps);
  const c10::DeviceGuard guard(a.qkv.device());
  a.first(pos0);
  Tensor q = at::empty({a.B, a.H, a.T, a.D}, a.qkv.options()),
         k = at::empty({a.B, a.Hkv, a.T, a.D}, a.qkv.options()), v = at::empty_like(k);
  const t2t_tensor qs = heads_of(q), ks = heads_of(k), vs = heads_of(v);
  check(t2t_qk_norm_rope(a.qkv.data_ptr(), a.sb, a.st, a.B, a.T, a.H, a.Hkv, a.D, a.code,
                         a.qw.data_ptr(), a.kw.data_ptr(), a.wcode, static_cast<float>(eps),
                         a.cos.data_ptr<float>(), a.sin.data_ptr<float>(), a.rows(), pos0, &qs,
                         &ks, &vs, stream_of(a.qkv)),
        "t2t_qk_norm_rope");
  return {q, k, v};
}

std::tuple<Tensor, Tensor, Tensor> qk_norm_rope_backward(
    const Tensor& dq_in, const Tensor& dk_in, const Tensor& dv_in, const Tensor& qkv_in,
    const Tensor& q_weight, const Tensor& k_weight, const Tensor& cos_in, const Tensor& sin_in,
    int64_t heads, int64_t kv_heads, int64_t pos0, double eps) {
  const QkNorm a(qkv_in, q_weight, k_weight, cos_in, sin_in, heads, kv_heads, eps);
  const c10::DeviceGuard guard(a.qkv.device());
  a.first(pos0);
  need_gpu(dq_in, dk_in, dv_in);
  const std::vector<int64_t> qshape{a.B, a.H, a.T, a.D}, kshape{a.B, a.Hkv, a.T, a.D};
  TORCH_CHECK_VALUE(dq_in.sizes() == at::IntArrayRef(qshape) &&
                        dk_in.sizes() == at::IntArrayRef(kshape) &&
                        dv_in.sizes() == at::IntArrayRef(kshape),
                    "gradients ", dq_in.sizes(), ", ", dk_in.sizes(), ", ", dv_in.sizes(),
                    " do not fit qkv ", qkv_in.sizes());
  for (const Tensor* t : {&dq_in, &dk_in, &dv_in})
    TORCH_CHECK_VALUE(t->scalar_type() == a.qkv.scalar_type() && t->device() == a.qkv.device(),
                      "gradients differ from qkv in dtype or device");
  const Tensor dq = vector_rows(dq_in), dk = vector_rows(dk_in), dv = vector_rows(dv_in);
  Tensor dqkv = at::empty(a.qkv.sizes(), a.qkv.options());
  Tensor dqw = at::empty_like(a.qw), dkw = at::empty_like(a.kw);
  const int64_t bytes = t2t_qk_norm_rope_backward_workspace(a.B, a.T, a.H, a.Hkv, a.D);
  Tensor ws = at::empty({std::max<int64_t>(1, bytes / 4)}, a.cos.options());
  const t2t_tensor qs = heads_of(dq), ks = heads_of(dk), vs = heads_of(dv);
  check(t2t_qk_norm_rope_backward(&qs, &ks, &vs, a.qkv.data_ptr(), a.sb, a.st, a.B, a.T, a.H,
                                  a.Hkv, a.D, a.code, a.qw.data_ptr(), a.kw.data_ptr(), a.wcode,
                                  static_cast<float>(eps), a.cos.data_ptr<float>(),
                                  a.sin.data_ptr<float>(), a.rows(), pos0, dqkv.data_ptr(),
                                  dqw.data_ptr(), dkw.data_ptr(), ws.data_ptr(), ws.numel() * 4,
                                  stream_of(a.qkv)),
        "t2t_qk_norm_rope_backward");
  return {dqkv, dqw, dkw};
}

// pos: int64 [M] or [B, M] on the device, or undefined for pos0 + m.
Tensor qk_norm_rope_append(const Tensor& qkv_in, const Tensor& q_weight, const Tensor& k_weight,
                           const Tensor& cos_in, const Tensor& sin_in, int64_t heads,
                           const c10::optional<Tensor>& pos_in, int64_t pos0,
                           const Tensor& k_cache, const Tensor& v_cache, double eps) {
  TORCH_CHECK_VALUE(k_cache.dim() == 4 && k_cache.sizes() == v_cache.sizes(), "caches ",
                    k_cache.sizes(), " and ", v_cache.sizes(),
                    " must both be [B, Hkv, capacity, D]");
  const QkNorm a(qkv_in, q_weight, k_weight, cos_in, sin_in, heads, k_cache.size(1), eps);
  const c10::DeviceGuard guard(a.qkv.device());
  TORCH_CHECK_VALUE(k_cache.size(0) == a.B && k_cache.size(3) == a.D, "caches ", k_cache.sizes(),
                    " do not fit qkv ", qkv_in.sizes(), " of ", heads, " query heads");
  for (const Tensor* t : {&k_cache, &v_cache}) {
    need_gpu(*t);
    TORCH_CHECK_VALUE(t->scalar_type() == a.qkv.scalar_type() && t->device() == a.qkv.device(),
                      "the caches differ from qkv in dtype or device");
    // written in place, so not copied
    TORCH_CHECK_VALUE(t->stride(3) == 1 || t->numel() == 0,
                      "the cache rows must have unit stride");
  }
  const int64_t cap = std::min<int64_t>(k_cache.size(2), INT32_MAX);
  Tensor pos;
  int64_t pos_sb = 0;
  if (pos_in.has_value()) {
    TORCH_CHECK_VALUE(pos_in->is_cuda() && pos_in->device() == a.qkv.device() &&
                          pos_in->scalar_type() == at::kLong,
                      "pos must be an int64 tensor on qkv's device");
    const bool each = pos_in->dim() == 2;
    TORCH_CHECK_VALUE((pos_in->dim() == 1 && pos_in->size(0) == a.T) ||
                          (each && pos_in->size(0) == a.B && pos_in->size(1) == a.T),
                      "pos ", pos_in->sizes(), " must be [", a.T, "] or [", a.B, ", ", a.T, "]");
    pos = pos_in->contiguous();
    pos_sb = each ? a.T : 0;
  } else {
    TORCH_CHECK_VALUE(pos0 >= 0 && pos0 <= std::min(cap, a.rows()) &&
                          pos0 + a.T <= std::min(cap, a.rows()),
                      "positions ", pos0, " .. ", pos0 + a.T - 1, " exceed the ", a.rows(),
                      " table rows or the ", cap, " cache rows");
  }
  Tensor q = at::empty({a.B, a.H, a.T, a.D}, a.qkv.options());
  const auto cache = [](const Tensor& t) {
    t2t_tensor s = heads_of(t);
    s.stride_t = t.stride(2);
    return s;
  };
  const t2t_tensor qs = heads_of(q), ks = cache(k_cache), vs = cache(v_cache);
  check(t2t_qk_norm_rope_append(a.qkv.data_ptr(), a.sb, a.st, a.B, a.T, a.H, a.Hkv, a.D, a.code,
                                a.qw.data_ptr(), a.kw.data_ptr(), a.wcode,
                                static_cast<float>(eps), a.cos.data_ptr<float>(),
                                a.sin.data_ptr<float>(), a.rows(),
                                pos.defined() ? pos.data_ptr<int64_t>() : nullptr, pos_sb,
                                pos.defined() ? 0 : pos0, &qs, &ks, &vs, cap, stream_of(a.qkv)),
        "t2t_qk_norm_rope_append");
  // written in place, which graphs that saved the caches have to see (inference
  // tensors have no versions)
  for (const Tensor* t : {&k_cache, &v_cache})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return q;
}

// ---- QKV split + any rotary form

// What both directions take, checked: tables, head counts and positions (pos:
// int64 [T] or [B, T] on the device, or undefined for pos0 + t).
struct Rotary {
  Tensor cos, sin, pos;
  int64_t B = 0, T = 0, H = 0, Hkv = 0, D = 0, R = 0, pos_sb = 0;
  int code = 0;
  Rotary(const Tensor& rows, int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads,
         int64_t head_dim, const Tensor& cos_in, const Tensor& sin_in,
         const c10::optional<Tensor>& pos_in, int64_t pos0)
      : B(batch), T(tokens), H(heads), Hkv(kv_heads), D(head_dim) {
    TORCH_CHECK_NOT_IMPLEMENTED(
        rows.scalar_type() == at::kBFloat16 || rows.scalar_type() == at::kFloat, "dtype ",
        rows.scalar_type(), " is not supported (bfloat16 or float32)");
    code = rows.scalar_type() == at::kFloat ? T2T_DTYPE_F32 : T2T_DTYPE_BF16;
    TORCH_CHECK_VALUE(cos_in.dim() == 2 && sin_in.sizes() == cos_in.sizes() &&
                          cos_in.size(1) >= 1 && cos_in.size(1) <= D / 2 &&
                          cos_in.scalar_type() == at::kFloat &&
                          sin_in.scalar_type() == at::kFloat,
                      "cos ", cos_in.sizes(), " and sin ", sin_in.sizes(),
                      " must be float32 [rows, R / 2] with R at most head_dim=", D);
    need_gpu(rows, cos_in, sin_in);
    TORCH_CHECK_VALUE(cos_in.device() == rows.device() && sin_in.device() == rows.device(),
                      "operands on different devices");
    const c10::DeviceGuard guard(rows.device());
    cos = vector_rows(cos_in.contiguous());
    sin = vector_rows(sin_in.contiguous());
    R = 2 * cos.size(1);
    TORCH_CHECK_VALUE(B <= INT32_MAX && T <= INT32_MAX && H <= INT32_MAX && D <= INT32_MAX,
                      "rows ", rows.sizes(), " are too large");
    if (pos_in.has_value()) {
      TORCH_CHECK_VALUE(pos_in->is_cuda() && pos_in->device() == rows.device() &&
                            pos_in->scalar_type() == at::kLong,
                        "pos must be an int64 tensor on the rows' device");
      const bool each = pos_in->dim() == 2;
      TORCH_CHECK_VALUE((pos_in->dim() == 1 && pos_in->size(0) == T) ||
                            (each && pos_in->size(0) == B && pos_in->size(1) == T),
                        "pos ", pos_in->sizes(), " must be [", T, "] or [", B, ", ", T, "]");
      pos = pos_in->contiguous();
      pos_sb = each ? T : 0;
    } else {
      TORCH_CHECK_VALUE(pos0 >= 0 && pos0 <= rows_() && pos0 + T <= rows_(), "positions ", pos0,
                        " .. ", pos0 + T - 1, " exceed the ", rows_(), " table rows");
    }
  }
  int64_t rows_() const { return std::min<int64_t>(cos.size(0), INT32_MAX); }
  const int64_t* positions() const {
    return pos.defined() && pos.numel() ? pos.data_ptr<int64_t>() : nullptr;
  }
};

std::tuple<Tensor, Tensor, Tensor> qkv_rotary(const Tensor& qkv_in, const Tensor& cos_in,
                                              const Tensor& sin_in, int64_t heads,
                                              int64_t kv_heads,
                                              const c10::optional<Tensor>& pos_in, int64_t pos0,
                                              bool interleaved) {
  TORCH_CHECK_VALUE(qkv_in.dim() == 3, "qkv must be [B, T, (H + 2 Hkv) D], got shape ",
                    qkv_in.sizes());
  TORCH_CHECK_VALUE(heads > 0 && kv_heads > 0, "num_heads=", heads, " and num_kv_heads=", kv_heads,
                    " must be positive");
  // (as a quotient: twice a huge count would not fit)
  TORCH_CHECK_VALUE(heads <= qkv_in.size(2) && kv_heads <= qkv_in.size(2) &&
                        qkv_in.size(2) % (heads + 2 * kv_heads) == 0,
                    "last dim ", qkv_in.size(2), " is not (num_heads + 2 num_kv_heads) * "
                    "head_dim (num_heads=", heads, ", num_kv_heads=", kv_heads, ")");
  const Rotary a(qkv_in, qkv_in.size(0), qkv_in.size(1), heads, kv_heads,
                 qkv_in.size(2) / (heads + 2 * kv_heads), cos_in, sin_in, pos_in, pos0);
  const c10::DeviceGuard guard(qkv_in.device());
  const Tensor qkv = vector_rows(qkv_in);
  Tensor q = at::empty({a.B, a.H, a.T, a.D}, qkv.options()),
         k = at::empty({a.B, a.Hkv, a.T, a.D}, qkv.options()), v = at::empty_like(k);
  if (q.numel() == 0) return {q, k, v};
  const t2t_tensor qs = heads_of(q), ks = heads_of(k), vs = heads_of(v);
  check(t2t_qkv_rotary(qkv.data_ptr(), a.B == 1 ? 0 : qkv.stride(0), a.T == 1 ? 0 : qkv.stride(1),
                       a.B, a.T, a.H, a.Hkv, a.D, a.R, interleaved, a.code,
                       a.cos.data_ptr<float>(), a.sin.data_ptr<float>(), a.rows_(), a.positions(),
                       a.pos_sb, pos0, &qs, &ks, &vs, stream_of(qkv)),
        "t2t_qkv_rotary");
  return {q, k, v};
}

Tensor qkv_rotary_backward(const Tensor& dq_in, const Tensor& dk_in, const Tensor& dv_in,
                           const Tensor& cos_in, const Tensor& sin_in,
                           const c10::optional<Tensor>& pos_in, int64_t pos0, bool interleaved) {
  TORCH_CHECK_VALUE(dq_in.dim() == 4 && dk_in.dim() == 4 && dk_in.sizes() == dv_in.sizes() &&
                        dk_in.size(0) == dq_in.size(0) &&
                        dk_in.sizes().slice(2) == dq_in.sizes().slice(2),
                    "gradients ", dq_in.sizes(), ", ", dk_in.sizes(), ", ", dv_in.sizes(),
                    " must be [B, H, T, D] and twice [B, Hkv, T, D]");
  need_gpu(dq_in, dk_in, dv_in);
  for (const Tensor* t : {&dk_in, &dv_in})
    TORCH_CHECK_VALUE(t->scalar_type() == dq_in.scalar_type() && t->device() == dq_in.device(),
                      "the gradients differ in dtype or device");
  const Rotary a(dq_in, dq_in.size(0), dq_in.size(2), dq_in.size(1), dk_in.size(1), dq_in.size(3),
                 cos_in, sin_in, pos_in, pos0);
  const c10::DeviceGuard guard(dq_in.device());
  const Tensor dq = vector_rows(dq_in), dk = vector_rows(dk_in), dv = vector_rows(dv_in);
  Tensor dqkv = at::empty({a.B, a.T, (a.H + 2 * a.Hkv) * a.D}, dq.options());
  if (dqkv.numel() == 0) return dqkv;
  const t2t_tensor qs = heads_of(dq), ks = heads_of(dk), vs = heads_of(dv);
  check(t2t_qkv_rotary_backward(&qs, &ks, &vs, dqkv.data_ptr(), dqkv.stride(0), dqkv.stride(1),
                                a.B, a.T, a.H, a.Hkv, a.D, a.R, interleaved, a.code,
                                a.cos.data_ptr<float>(), a.sin.data_ptr<float>(), a.rows_(),
                                a.positions(), a.pos_sb, pos0, stream_of(dq)),
        "t2t_qkv_rotary_backward");
  return dqkv;
}

// ---- decode step

// Mask inputs of Tq new rows a sequence over a cache, checked.
struct RowMask {
  int64_t Bm, W, cap;
  const Tensor &key_doc, &q_pos, &q_doc;
  const c10::optional<Tensor>&key_bits, &q_bits, &q_start;
  RowMask(const Tensor& q, int64_t B, int64_t Tq, const Tensor& key_doc_in,
          const c10::optional<Tensor>& key_bits_in, const Tensor& q_pos_in,
          const Tensor& q_doc_in, const c10::optional<Tensor>& q_bits_in, int64_t sinks,
          const c10::optional<Tensor>& q_start_in)
      : key_doc(key_doc_in), q_pos(q_pos_in), q_doc(q_doc_in), key_bits(key_bits_in),
        q_bits(q_bits_in), q_start(q_start_in) {
    W = key_bits.has_value() && key_bits->dim() == 3 ? key_bits->size(1) : 0;
    TORCH_CHECK_VALUE(q_bits.has_value() == key_bits.has_value() &&
                          (!q_bits.has_value() || (q_bits->dim() == 3 && q_bits->size(1) == W)),
                      "q_bits and key_bits must both be given with the same word count (they go "
                      "together)");
    TORCH_CHECK_VALUE((sinks > 0) == q_start.has_value(), "q_start goes with sinks");
    TORCH_CHECK_VALUE(key_doc.dim() == 2, "key_doc ", key_doc.sizes(), " must be [Bm, cap]");
    Bm = key_doc.size(0);
    cap = key_doc.size(1);
    TORCH_CHECK_VALUE(Bm == 1 || Bm == B, "mask batch ", Bm, " does not broadcast to B=", B);
    TORCH_CHECK_NOT_IMPLEMENTED(W <= T2T_MAX_WORDS, W, " grant words exceed ", T2T_MAX_WORDS);
    const std::vector<int64_t> rows{Bm, Tq}, keys{Bm, cap}, kw{Bm, W, cap}, qw{Bm, W, Tq};
    take(q, key_doc, at::kInt, keys, "key_doc");
    take(q, q_pos, at::kInt, rows, "q_pos");
    take(q, q_doc, at::kInt, rows, "q_doc");
    if (q_start.has_value()) take(q, *q_start, at::kInt, rows, "q_start");
    if (key_bits.has_value()) {
      take(q, *key_bits, at::kLong, kw, "key_bits");
      take(q, *q_bits, at::kLong, qw, "q_bits");
    }
  }
  static void take(const Tensor& q, const Tensor& t, at::ScalarType type, at::IntArrayRef shape,
                   const char* name) {
    TORCH_CHECK_VALUE(t.scalar_type() == type && t.is_contiguous() && t.sizes() == shape, name,
                      " must be contiguous ", type, " ", shape, ", not ", t.scalar_type(), " ",
                      t.sizes());
    TORCH_CHECK(t.device() == q.device(), name, " must be on q's device, the GPU ", q.device());
  }
  static const uint64_t* bits(const c10::optional<Tensor>& t) {
    return t.has_value() && t->numel() ? static_cast<const uint64_t*>(t->data_ptr()) : nullptr;
  }
  const int32_t* start() const {
    return q_start.has_value() ? q_start->data_ptr<int32_t>() : nullptr;
  }
};

// window 0: none
std::tuple<Tensor, Tensor> attn_decode(
    const Tensor& q_in, const Tensor& k, const Tensor& v, int64_t n_keys, const Tensor& key_doc,
    const c10::optional<Tensor>& key_bits, const Tensor& q_pos, const Tensor& q_doc,
    const c10::optional<Tensor>& q_bits, double scale, const c10::optional<Tensor>& out,
    int64_t window, int64_t sinks, const c10::optional<Tensor>& q_start) {
  TORCH_CHECK_NOT_IMPLEMENTED(q_in.scalar_type() == at::kBFloat16 &&
                                  k.scalar_type() == at::kBFloat16 &&
                                  v.scalar_type() == at::kBFloat16,
                              "bfloat16 only");
  TORCH_CHECK(q_in.is_cuda() && k.is_cuda() && v.is_cuda(),
              "the decode kernel needs ROCm GPU tensors");
  TORCH_CHECK(k.device() == q_in.device() && v.device() == q_in.device(),
              "the caches must be on q's device, ", q_in.device());
  TORCH_CHECK_VALUE(q_in.dim() == 4 && k.dim() == 4, "q ", q_in.sizes(), " and the caches ",
                    k.sizes(), " must be 4-D");
  const int64_t B = q_in.size(0), Hq = q_in.size(1), Tq = q_in.size(2), D = q_in.size(3);
  const RowMask m(q_in, B, Tq, key_doc, key_bits, q_pos, q_doc, q_bits, sinks, q_start);
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && k.size(0) == B && k.size(3) == D, "caches ",
                    k.sizes(), " / ", v.sizes(), " do not fit q ", q_in.sizes());
  TORCH_CHECK_VALUE(n_keys >= 0 && n_keys <= std::min(m.cap, k.size(2)), "n_keys=", n_keys,
                    " exceeds the cache (", k.size(2), " rows, ", m.cap, " mask slots)");
  const c10::DeviceGuard guard(q_in.device());
  const Tensor q = q_in.stride(3) == 1 ? q_in : q_in.contiguous();
  Tensor o = out.has_value() ? *out : at::empty({B, Hq, Tq, D}, q.options());
  if (out.has_value())
    TORCH_CHECK_VALUE(o.sizes() == q.sizes() && o.scalar_type() == at::kBFloat16 &&
                          o.device() == q.device(),
                      "out ", o.sizes(), " must be bfloat16 of q's shape and on its device");
  Tensor lse2 = at::empty({B, Hq, Tq}, q.options().dtype(at::kFloat));
  Tensor ws = at::empty({t2t_attn_decode_workspace(B, Hq, Tq, n_keys, D) / 4}, lse2.options());
  const t2t_tensor qs = view4(q), ks = view4(k), vs = view4(v), os = view4(o);
  const int32_t *doc = key_doc.data_ptr<int32_t>(), *pos = q_pos.data_ptr<int32_t>(),
                *qd = q_doc.data_ptr<int32_t>();
  const float c = static_cast<float>(scale);
  const int rc =
      window == 0
          ? t2t_attn_decode(&qs, &ks, &vs, &os, lse2.data_ptr<float>(), doc, m.bits(key_bits),
                            m.cap, pos, qd, m.bits(q_bits), m.Bm, m.W, B, Hq, k.size(1), Tq,
                            n_keys, D, T2T_DTYPE_BF16, c, ws.data_ptr(), ws.numel() * 4,
                            stream_of(q))
          : t2t_attn_decode_window(&qs, &ks, &vs, &os, lse2.data_ptr<float>(), doc,
                                   m.bits(key_bits), m.cap, pos, qd, m.bits(q_bits), m.Bm, m.W, B,
                                   Hq, k.size(1), Tq, n_keys, D, T2T_DTYPE_BF16, c,
                                   std::min<int64_t>(window, INT32_MAX),
                                   std::min<int64_t>(sinks, INT32_MAX), m.start(), ws.data_ptr(),
                                   ws.numel() * 4, stream_of(q));
  check(rc, "t2t_attn_decode");
  return {o, lse2};
}

// ---- 8-bit key/value cache

// Codes and scales of a cache, checked against the heads they are used with.
// They are read and written in place, so never copied.
struct Kv8 {
  int64_t B, Hkv, blocks, D;
  Kv8(const Tensor& k_codes, const Tensor& v_codes, const Tensor& k_scale, const Tensor& v_scale,
      const Tensor& like) {
    TORCH_CHECK_VALUE(k_codes.dim() == 5 && k_codes.size(3) == T2T_KV8_BLOCK &&
                          v_codes.dim() == 5 && v_codes.size(4) == T2T_KV8_BLOCK &&
                          v_codes.size(3) == k_codes.size(4) &&
                          v_codes.sizes().slice(0, 3) == k_codes.sizes().slice(0, 3),
                      "codes ", k_codes.sizes(), " and ", v_codes.sizes(), " must be [B, Hkv, "
                      "blocks, ", T2T_KV8_BLOCK, ", D] and [B, Hkv, blocks, D, ", T2T_KV8_BLOCK,
                      "]");
    TORCH_CHECK_VALUE(k_scale.sizes() == k_codes.sizes().slice(0, 3) &&
                          v_scale.sizes() == k_scale.sizes(),
                      "scales ", k_scale.sizes(), " and ", v_scale.sizes(),
                      " must be [B, Hkv, blocks]");
    TORCH_CHECK_VALUE(k_codes.scalar_type() == at::kFloat8_e4m3fn &&
                          v_codes.scalar_type() == at::kFloat8_e4m3fn &&
                          k_scale.scalar_type() == at::kFloat &&
                          v_scale.scalar_type() == at::kFloat,
                      "codes must be float8_e4m3fn and scales float32");
    need_gpu(like, k_codes, v_codes, k_scale, v_scale);
    for (const Tensor* t : {&k_codes, &v_codes, &k_scale, &v_scale})
      TORCH_CHECK_VALUE(t->is_contiguous() && t->device() == like.device(),
                        "codes and scales must be contiguous and on the heads' device");
    B = k_codes.size(0);
    Hkv = k_codes.size(1);
    blocks = k_codes.size(2);
    D = k_codes.size(4);
    TORCH_CHECK_NOT_IMPLEMENTED(D == 64 || D == 128, "head dim ", D, " is not supported (64 or "
                                "128)");
    TORCH_CHECK_VALUE(B <= INT32_MAX && Hkv <= INT32_MAX && blocks <= INT32_MAX / 64 - 16,
                      "codes ", k_codes.sizes(), " are too large");
  }
};

// pos: int64, one value or one a sequence, on the device, or undefined for pos0.
void kv8_append(const Tensor& k_in, const Tensor& v_in, const c10::optional<Tensor>& pos_in,
                int64_t pos0, const Tensor& k_codes, const Tensor& v_codes, const Tensor& k_scale,
                const Tensor& v_scale, int64_t capacity) {
  const Kv8 c(k_codes, v_codes, k_scale, v_scale, k_in);
  TORCH_CHECK_VALUE(k_in.dim() == 4 && k_in.sizes() == v_in.sizes() && k_in.size(0) == c.B &&
                        k_in.size(1) == c.Hkv && k_in.size(3) == c.D,
                    "k ", k_in.sizes(), " and v ", v_in.sizes(), " must be [B, Hkv, M, D] of "
                    "codes ", k_codes.sizes());
  TORCH_CHECK_NOT_IMPLEMENTED(
      k_in.scalar_type() == at::kBFloat16 || k_in.scalar_type() == at::kFloat, "dtype ",
      k_in.scalar_type(), " is not supported (bfloat16 or float32)");
  need_gpu(v_in);
  TORCH_CHECK_VALUE(v_in.scalar_type() == k_in.scalar_type() && v_in.device() == k_in.device(),
                    "k and v differ in dtype or device");
  if (capacity < 0) capacity = c.blocks * T2T_KV8_BLOCK;
  TORCH_CHECK_VALUE(capacity <= c.blocks * T2T_KV8_BLOCK, "capacity=", capacity, " exceeds the ",
                    c.blocks, " blocks");
  const c10::DeviceGuard guard(k_in.device());
  const int64_t M = k_in.size(2);
  Tensor pos;
  if (pos_in.has_value()) {
    TORCH_CHECK_VALUE(pos_in->is_cuda() && pos_in->device() == k_in.device() &&
                          pos_in->scalar_type() == at::kLong,
                      "pos must be an int64 tensor on the heads' device");
    TORCH_CHECK_VALUE(pos_in->dim() <= 1 && (pos_in->numel() == 1 || pos_in->numel() == c.B),
                      "pos ", pos_in->sizes(), " must be one position, or one for each of ", c.B,
                      " sequences");
    TORCH_CHECK_VALUE(M <= capacity, M, " tokens exceed capacity=", capacity);
    pos = pos_in->contiguous();
  } else {
    TORCH_CHECK_VALUE(pos0 >= 0 && pos0 <= capacity - M, "positions ", pos0, " .. ",
                      pos0 + M - 1, " exceed capacity=", capacity);
  }
  if (k_in.numel() == 0) return;
  const Tensor k = vector_rows(k_in), v = vector_rows(v_in);
  const t2t_tensor ks = heads_of(k), vs = heads_of(v);
  check(t2t_kv8_append(&ks, &vs, c.B, c.Hkv, M, c.D,
                       k.scalar_type() == at::kFloat ? T2T_DTYPE_F32 : T2T_DTYPE_BF16,
                       pos.defined() ? pos.data_ptr<int64_t>() : nullptr,
                       pos.defined() && pos.numel() > 1 ? 1 : 0, pos.defined() ? 0 : pos0,
                       k_codes.data_ptr(), v_codes.data_ptr(), k_scale.data_ptr<float>(),
                       v_scale.data_ptr<float>(), c.blocks, capacity, stream_of(k)),
        "t2t_kv8_append");
  // written in place, which graphs that saved the cache have to see (inference
  // tensors have no versions)
  for (const Tensor* t : {&k_codes, &v_codes, &k_scale, &v_scale})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

std::tuple<Tensor, Tensor> kv8_attend(
    const Tensor& q_in, const Tensor& k_codes, const Tensor& v_codes, const Tensor& k_scale,
    const Tensor& v_scale, int64_t n_keys, const Tensor& key_doc,
    const c10::optional<Tensor>& key_bits, const Tensor& q_pos, const Tensor& q_doc,
    const c10::optional<Tensor>& q_bits, double scale, int64_t window, int64_t sinks,
    const c10::optional<Tensor>& q_start) {
  const Kv8 c(k_codes, v_codes, k_scale, v_scale, q_in);
  TORCH_CHECK_NOT_IMPLEMENTED(q_in.scalar_type() == at::kBFloat16, "q dtype ", q_in.scalar_type(),
                              " is not supported (bfloat16)");
  TORCH_CHECK_VALUE(q_in.dim() == 4 && q_in.size(0) == c.B && q_in.size(3) == c.D && c.Hkv > 0 &&
                        q_in.size(1) % c.Hkv == 0,
                    "q ", q_in.sizes(), " must be [B, Hq, Tq, D] of codes ", k_codes.sizes(),
                    ", Hq a multiple of Hkv");
  const int64_t Hq = q_in.size(1), Tq = q_in.size(2);
  TORCH_CHECK_NOT_IMPLEMENTED(Hq / c.Hkv * Tq <= T2T_KV8_MAX_ROWS, "(Hq / Hkv) * Tq = ",
                              Hq / c.Hkv * Tq, " query rows per kv head exceeds ",
                              T2T_KV8_MAX_ROWS);
  const RowMask m(q_in, c.B, Tq, key_doc, key_bits, q_pos, q_doc, q_bits, sinks, q_start);
  TORCH_CHECK_VALUE(n_keys >= 0 && n_keys <= m.cap && n_keys <= c.blocks * T2T_KV8_BLOCK,
                    "n_keys=", n_keys, " exceeds the cache (", c.blocks * T2T_KV8_BLOCK,
                    " positions, ", m.cap, " mask slots)");
  TORCH_CHECK_VALUE(scale > 0 && std::isfinite(scale), "scale=", scale, " must be positive and "
                    "finite");
  const c10::DeviceGuard guard(q_in.device());
  const Tensor q = vector_rows(q_in);
  Tensor o = at::empty({c.B, Hq, Tq, c.D}, q.options());
  Tensor lse2 = at::empty({c.B, Hq, Tq}, q.options().dtype(at::kFloat));
  if (o.numel() == 0) return {o, lse2};
  const int64_t bytes = t2t_kv8_attend_workspace(c.B, Hq, c.Hkv, Tq, n_keys, c.D);
  Tensor ws = at::empty({bytes / 4}, lse2.options());
  const t2t_tensor qs = heads_of(q), os = heads_of(o);
  check(t2t_kv8_attend(&qs, k_codes.data_ptr(), v_codes.data_ptr(), k_scale.data_ptr<float>(),
                       v_scale.data_ptr<float>(), c.blocks, &os, lse2.data_ptr<float>(),
                       key_doc.data_ptr<int32_t>(), m.bits(key_bits), m.cap,
                       q_pos.data_ptr<int32_t>(), q_doc.data_ptr<int32_t>(), m.bits(q_bits), m.Bm,
                       m.W, c.B, Hq, c.Hkv, Tq, n_keys, c.D, T2T_DTYPE_BF16,
                       static_cast<float>(scale), std::min<int64_t>(window, INT32_MAX),
                       std::min<int64_t>(sinks, INT32_MAX), m.start(), ws.data_ptr(),
                       ws.numel() * 4, stream_of(q)),
        "t2t_kv8_attend");
  return {o, lse2};
}

// ---- scaled embedding

int embed_code(const Tensor& w) {
  TORCH_CHECK_NOT_IMPLEMENTED(w.scalar_type() == at::kBFloat16 || w.scalar_type() == at::kFloat,
                              "weight dtype ", w.scalar_type(),
                              " is not supported (bfloat16 or float32)");
  return w.scalar_type() == at::kFloat ? T2T_DTYPE_F32 : T2T_DTYPE_BF16;
}

Tensor embed_ids(const Tensor& tokens) {
  TORCH_CHECK_VALUE(tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt,
                    "tokens must be int64 or int32, not ", tokens.scalar_type());
  return tokens.to(at::kLong).contiguous();
}

// (before a count of columns is handed on as 32 bits)
void need_columns(int64_t C) {
  TORCH_CHECK_NOT_IMPLEMENTED(C <= INT32_MAX, "rows of ", C, " columns are not supported");
}

Tensor embedding(const Tensor& tokens, const Tensor& weight, double scale) {
  TORCH_CHECK_VALUE(weight.dim() == 2, "weight must be [V, C], got shape ", weight.sizes());
  const int code = embed_code(weight);
  need_gpu(tokens, weight);
  TORCH_CHECK_VALUE(tokens.device() == weight.device(), "tokens and weight on different devices");
  const c10::DeviceGuard guard(weight.device());
  const Tensor ids = embed_ids(tokens);
  const int64_t V = weight.size(0), C = weight.size(1);
  need_columns(C);
  const bool rows = (weight.stride(1) == 1 || C == 1) && weight.stride(0) >= C;
  const Tensor w = rows ? weight : weight.contiguous();
  std::vector<int64_t> shape = tokens.sizes().vec();
  shape.push_back(C);
  Tensor out = at::empty(shape, weight.options());
  if (out.numel())
    check(t2t_embedding(ids.data_ptr<int64_t>(), ids.numel(), w.data_ptr(),
                        V == 1 ? C : w.stride(0), V, static_cast<int32_t>(C), code,
                        static_cast<float>(scale), out.data_ptr(), stream_of(weight)),
          "t2t_embedding");
  return out;
}

// dy [..., C] of the tokens; the gradient [V, C] of dy's dtype.
Tensor embedding_backward(const Tensor& tokens, const Tensor& dy_in, int64_t V, double scale,
                          int64_t padding) {
  const int code = embed_code(dy_in);
  need_gpu(tokens, dy_in);
  TORCH_CHECK_VALUE(tokens.device() == dy_in.device(), "tokens and gradient on different devices");
  const c10::DeviceGuard guard(dy_in.device());
  const Tensor ids = embed_ids(tokens);
  const int64_t C = dy_in.size(-1), N = ids.numel();
  need_columns(C);
  TORCH_CHECK_VALUE(dy_in.numel() == N * C, "gradient ", dy_in.sizes(), " does not fit tokens ",
                    tokens.sizes());
  Tensor dw = at::empty({V, C}, dy_in.options());
  if (dw.numel() == 0) return dw;
  Tensor dy = dy_in.dim() == 2 ? dy_in : dy_in.reshape({N, C});
  if (dy.stride(1) != 1) dy = dy.contiguous();
  Tensor ws = at::empty({t2t_embedding_backward_workspace(N, V, C)},
                        dy.options().dtype(at::kByte));
  check(t2t_embedding_backward(ids.data_ptr<int64_t>(), N, dy.data_ptr(),
                               N == 1 ? C : dy.stride(0), V, static_cast<int32_t>(C), code,
                               static_cast<float>(scale), padding, dw.data_ptr(), ws.data_ptr(),
                               ws.numel(), stream_of(dy)),
        "t2t_embedding_backward");
  return dw;
}

// ---- distillation loss

int float_code(const Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat,
                              what, " dtype ", t.scalar_type(),
                              " is not supported (bfloat16 or float32)");
  return t.scalar_type() == at::kFloat ? T2T_DTYPE_F32 : T2T_DTYPE_BF16;
}

// The last dimension's rows with unit stride and a row stride of at least
// their length.
Tensor plain_rows(const Tensor& t) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  const bool ok = (r.stride(1) == 1 || r.size(1) == 1) &&
                  (r.size(0) == 1 || r.stride(0) >= r.size(1));
  return ok ? r : r.clone(at::MemoryFormat::Contiguous);
}

// What the distillation calls take, checked; reduction: 0 none, 1 sum, 2 mean.
struct Distill {
  Tensor z, idx, teacher, target;
  std::vector<int64_t> shape;  // of the logits
  int64_t rows = 0, V = 0, K = 0, ignore = 0;
  int code = 0, teacher_code = 0;
  double temp = 1, alpha = 1;
  Distill(const Tensor& logits, const Tensor& idx_in, const Tensor& teacher_in,
          const c10::optional<Tensor>& target_in, double temperature, double alpha_in,
          int64_t ignore_index)
      : ignore(ignore_index), temp(temperature), alpha(alpha_in) {
    TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1 && logits.size(-1) <= INT32_MAX,
                      "logits must be [..., V], got shape ", logits.sizes());
    TORCH_CHECK_VALUE(idx_in.sizes() == teacher_in.sizes() && idx_in.dim() == logits.dim() &&
                          idx_in.sizes().slice(0, idx_in.dim() - 1) ==
                              logits.sizes().slice(0, logits.dim() - 1),
                      "teacher_idx ", idx_in.sizes(), " and teacher_logits ", teacher_in.sizes(),
                      " must be [..., K] of logits ", logits.sizes());
    TORCH_CHECK_NOT_IMPLEMENTED(idx_in.size(-1) <= T2T_DISTILL_MAX_SLOTS, "K=", idx_in.size(-1),
                                " slots a row; at most ", T2T_DISTILL_MAX_SLOTS);
    TORCH_CHECK_VALUE(idx_in.scalar_type() == at::kLong || idx_in.scalar_type() == at::kInt,
                      "teacher_idx must be int64 or int32, not ", idx_in.scalar_type());
    TORCH_CHECK_VALUE(temp >= 0.01 && temp <= 100, "temperature=", temp,
                      " must be in [0.01, 100]");
    TORCH_CHECK_VALUE(alpha >= 0 && alpha <= 1, "alpha=", alpha, " must be in [0, 1]");
    TORCH_CHECK_VALUE(alpha == 1 || target_in.has_value(), "alpha below 1 needs targets");
    code = float_code(logits, "logits");
    teacher_code = float_code(teacher_in, "teacher_logits");
    need_gpu(logits, idx_in, teacher_in);
    TORCH_CHECK_VALUE(idx_in.device() == logits.device() && teacher_in.device() == logits.device(),
                      "logits and teacher on different devices");
    shape = logits.sizes().vec();
    V = logits.size(-1);
    rows = logits.numel() / V;
    K = idx_in.size(-1);
    const c10::DeviceGuard guard(logits.device());
    if (target_in.has_value()) {
      TORCH_CHECK_VALUE(target_in->sizes() == logits.sizes().slice(0, logits.dim() - 1) &&
                            (target_in->scalar_type() == at::kLong ||
                             target_in->scalar_type() == at::kInt),
                        "targets ", target_in->sizes(), " must be int64 or int32 ids of logits ",
                        logits.sizes());
      need_gpu(*target_in);
      TORCH_CHECK_VALUE(target_in->device() == logits.device(),
                        "logits and targets on different devices");
      target = target_in->to(at::kLong).contiguous().view({-1});
    }
    if (rows == 0) return;
    z = plain_rows(logits);
    if (K > 0) {
      idx = plain_rows(idx_in);
      teacher = plain_rows(teacher_in);
    }
  }
  // One launch over the rows; any of the outputs may be undefined.  grad: rows
  // of stride grad_ld, the logits themselves among them.
  void launch(const Tensor& row_loss, const Tensor& grad, int64_t grad_ld, double scale,
              const Tensor& scale_dev, const Tensor& g, bool unless_one) const {
    if (rows == 0) return;
    const auto ptr = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    check(t2t_distill_rows(
              z.data_ptr(), step(z), rows, static_cast<int32_t>(V), code, ptr(idx),
              idx.defined() && idx.scalar_type() == at::kInt ? 4 : 8, step(idx), ptr(teacher),
              teacher_code, step(teacher), static_cast<int32_t>(K),
              static_cast<const int64_t*>(ptr(target)), ignore, static_cast<float>(temp),
              static_cast<float>(alpha), static_cast<float>(scale),
              static_cast<const float*>(ptr(scale_dev)), static_cast<const float*>(ptr(g)),
              g.defined() && g.numel() > 1 ? 1 : 0, unless_one,
              static_cast<float*>(ptr(row_loss)), ptr(grad), grad_ld, stream_of(z)),
          "t2t_distill_rows");
  }
  static int64_t step(const Tensor& t) {
    return !t.defined() ? 0 : t.size(0) == 1 ? t.size(1) : t.stride(0);
  }
};

// (loss, gradient for an incoming gradient of 1, [1 / max(n, 1), 1 / n]); the
// second only when asked for, and never for the rows' own losses.
std::tuple<Tensor, Tensor, Tensor> distill_loss(
    const Tensor& logits, const Tensor& idx, const Tensor& teacher,
    const c10::optional<Tensor>& target, double temperature, double alpha, int64_t ignore_index,
    int64_t reduction, bool with_grad) {
  const Distill a(logits, idx, teacher, target, temperature, alpha, ignore_index);
  const c10::DeviceGuard guard(logits.device());
  const auto f32 = logits.options().dtype(at::kFloat);
  Tensor row_loss = at::empty(logits.sizes().slice(0, logits.dim() - 1), f32);
  if (reduction == 0) {
    a.launch(row_loss, Tensor(), a.V, 1.0, Tensor(), Tensor(), false);
    return {row_loss, Tensor(), Tensor()};
  }
  Tensor inv;
  double scale = 1.0;
  if (reduction == 2) {
    if (a.target.defined()) {
      inv = at::empty({2}, f32);
      check(t2t_distill_count(a.target.data_ptr<int64_t>(), a.rows, ignore_index,
                              inv.data_ptr<float>(), stream_of(logits)),
            "t2t_distill_count");
    } else {
      scale = a.rows ? 1.0 / static_cast<double>(a.rows) : NAN;
    }
  }
  Tensor grad = with_grad ? at::empty(a.shape, logits.options()) : Tensor();
  a.launch(row_loss, grad, a.V, scale, inv, Tensor(), false);
  Tensor loss = at::empty({}, f32);
  check(t2t_distill_mean(row_loss.data_ptr<float>(), a.rows,
                         inv.defined() ? inv.data_ptr<float>() + 1 : nullptr,
                         static_cast<float>(scale), loss.data_ptr<float>(), stream_of(logits)),
        "t2t_distill_mean");
  return {loss, grad, inv};
}

// The logits' gradient for the incoming gradient g (one value, or one a row for
// reduction 0).  kept: the gradient of distill_loss, which stands where g is 1
// and is written again where it is not.
Tensor distill_loss_backward(const Tensor& g_in, const Tensor& logits, const Tensor& idx,
                             const Tensor& teacher, const c10::optional<Tensor>& target,
                             double temperature, double alpha, int64_t ignore_index,
                             int64_t reduction, const c10::optional<Tensor>& inv_in,
                             const c10::optional<Tensor>& kept) {
  const Distill a(logits, idx, teacher, target, temperature, alpha, ignore_index);
  need_gpu(g_in);
  const c10::DeviceGuard guard(logits.device());
  TORCH_CHECK_VALUE(g_in.scalar_type() == at::kFloat && g_in.device() == logits.device() &&
                        g_in.numel() == (reduction == 0 ? a.rows : 1),
                    "gradient ", g_in.sizes(), " ", g_in.scalar_type(), " does not fit the loss");
  const Tensor g = g_in.contiguous();
  Tensor inv = inv_in.has_value() ? *inv_in : Tensor();
  double scale = 1.0;
  if (reduction == 2 && !inv.defined()) {
    if (a.target.defined()) {
      inv = at::empty({2}, g.options());
      check(t2t_distill_count(a.target.data_ptr<int64_t>(), a.rows, ignore_index,
                              inv.data_ptr<float>(), stream_of(logits)),
            "t2t_distill_count");
    } else if (a.rows) {
      scale = 1.0 / static_cast<double>(a.rows);
    }
  }
  Tensor grad = kept.has_value() ? *kept : at::empty(a.shape, logits.options());
  a.launch(Tensor(), grad, a.V, scale, inv, g, kept.has_value());
  return grad;
}

// Over chunk rows of a head's logits: the gradient in place of the logits.
void distill_rows_(const Tensor& logits, const Tensor& idx, const Tensor& teacher,
                   const c10::optional<Tensor>& target, double temperature, double alpha,
                   int64_t ignore_index, const c10::optional<Tensor>& inv, double scale,
                   const Tensor& row_loss, bool with_grad) {
  const Distill a(logits, idx, teacher, target, temperature, alpha, ignore_index);
  const c10::DeviceGuard guard(logits.device());
  TORCH_CHECK(logits.dim() == 2 && (a.rows == 0 || a.z.data_ptr() == logits.data_ptr()) &&
                  row_loss.is_cuda() && row_loss.scalar_type() == at::kFloat &&
                  row_loss.is_contiguous() && row_loss.numel() == a.rows,
              "logits of unit stride [rows, V] and float32 row losses [rows]");
  if (a.rows)
    a.launch(row_loss, with_grad ? a.z : Tensor(), Distill::step(a.z), scale,
             inv.has_value() ? *inv : Tensor(), Tensor(), false);
}

// [1 / max(n, 1), 1 / n] of the targets, n the counted ones.
Tensor distill_count(const Tensor& target, int64_t ignore_index) {
  need_gpu(target);
  TORCH_CHECK_VALUE(target.scalar_type() == at::kLong && target.is_contiguous(),
                    "targets must be contiguous int64");
  const c10::DeviceGuard guard(target.device());
  Tensor inv = at::empty({2}, target.options().dtype(at::kFloat));
  check(t2t_distill_count(target.data_ptr<int64_t>(), target.numel(), ignore_index,
                          inv.data_ptr<float>(), stream_of(target)),
        "t2t_distill_count");
  return inv;
}

// scale (inv[1] where given) times the sum of row losses.
Tensor distill_mean(const Tensor& row_loss, const c10::optional<Tensor>& inv, double scale) {
  need_gpu(row_loss);
  TORCH_CHECK_VALUE(row_loss.scalar_type() == at::kFloat && row_loss.is_contiguous(),
                    "row losses must be contiguous float32");
  const c10::DeviceGuard guard(row_loss.device());
  Tensor loss = at::empty({}, row_loss.options());
  check(t2t_distill_mean(row_loss.data_ptr<float>(), row_loss.numel(),
                         inv.has_value() ? inv->data_ptr<float>() + 1 : nullptr,
                         static_cast<float>(scale), loss.data_ptr<float>(), stream_of(row_loss)),
        "t2t_distill_mean");
  return loss;
}

// ---- SwiGLU

std::tuple<Tensor, Tensor> swiglu(const Tensor& gu) {
  need_gpu(gu);
  const c10::DeviceGuard guard(gu.device());
  const Tensor g2 = rows_of(gu);
  const int64_t N = g2.size(0), H = g2.size(1) / 2;
  std::vector<int64_t> shape = gu.sizes().vec();
  shape.back() = H;
  Tensor h = at::empty(shape, gu.options());
  check(t2t_swiglu(g2.data_ptr(), g2.stride(0), h.data_ptr(), H, N, H, stream_of(gu)),
        "t2t_swiglu");
  return {h, g2};
}

Tensor swiglu_backward(const Tensor& g2, const Tensor& dh, at::IntArrayRef shape) {
  need_gpu(g2, dh);
  const c10::DeviceGuard guard(g2.device());
  const int64_t N = g2.size(0), H = g2.size(1) / 2;
  const Tensor d2 = rows_of(dh);
  Tensor dgu = at::empty(shape, g2.options());
  check(t2t_swiglu_backward(g2.data_ptr(), g2.stride(0), d2.data_ptr(), d2.stride(0),
                            dgu.data_ptr(), 2 * H, N, H, stream_of(g2)),
        "t2t_swiglu_backward");
  return dgu;
}

// ---- linear map of token rows: x W^T, or x W (transposed)

Tensor linear(const Tensor& x, const Tensor& w, bool transposed) {
  need_gpu(x, w);
  const c10::DeviceGuard guard(x.device());
  const Tensor x2 = rows_of(x), w2 = rows_of(w);
  const int64_t M = x2.size(0), K = x2.size(1), N = w2.size(transposed ? 1 : 0);
  TORCH_CHECK(w2.size(transposed ? 0 : 1) == K, "weight ", w.sizes(), " does not take rows of ", K);
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = N;
  Tensor y = at::empty(shape, x.options());
  check(t2t_linear(x2.data_ptr(), x2.stride(0), w2.data_ptr(), w2.stride(0), transposed,
                   y.data_ptr(), N, M, N, K, stream_of(x)),
        "t2t_linear");
  return y;
}

// ---- weight gradient dY^T X

Tensor wgrad(const Tensor& dy, const Tensor& x, at::ScalarType out_dtype) {
  need_gpu(dy, x);
  const c10::DeviceGuard guard(x.device());
  const Tensor d2 = rows_of(dy), x2 = rows_of(x);
  const int64_t K = d2.size(0), M = d2.size(1), N = x2.size(1);
  Tensor ws = at::empty({t2t_wgrad_workspace(M, N, K)}, x.options().dtype(at::kByte));
  Tensor out = at::empty({M, N}, x.options().dtype(out_dtype));
  check(t2t_wgrad(d2.data_ptr(), d2.stride(0), x2.data_ptr(), x2.stride(0), out.data_ptr(),
                  out_dtype == at::kFloat ? T2T_DTYPE_F32 : T2T_DTYPE_BF16, M, N, K,
                  ws.data_ptr(), ws.numel(), stream_of(x)),
        "t2t_wgrad");
  return out;
}

// ---- mask metadata

// The tables of t2t_mask_meta for doc [Bm, T] (int32) and words [Bm, W, T]
// (int64), in the order tile_class, the 13 tables of t2t_block_mask.  The
// index tables are views of one allocation; the bitmaps, which dwarf them,
// are their own.
// window 0: none; sinks add t2t_doc_starts of doc behind the tables.
std::vector<Tensor> mask_meta_window(const Tensor& doc, const Tensor& q_bits,
                                     const Tensor& kv_bits, int64_t window, int64_t sinks,
                                     int64_t stream_in) {
  need_gpu(doc, q_bits, kv_bits);
  void* const stream = reinterpret_cast<void*>(static_cast<intptr_t>(stream_in));
  const c10::DeviceGuard guard(doc.device());
  const int64_t Bm = doc.size(0), T = doc.size(1), W = q_bits.size(1);
  const int64_t nt = (T + T2T_TILE - 1) / T2T_TILE;
  const auto i32 = doc.options().dtype(at::kInt);
  const int64_t row = Bm * nt, grid = Bm * nt * nt;
  const auto padded = [](int64_t n) { return (n + 15) / 16 * 16; };  // 64-byte starts
  Tensor pool = at::empty({7 * padded(row) + 5 * padded(grid)}, i32);
  int64_t at_ = 0;
  const auto take = [&](at::IntArrayRef shape, int64_t n) {
    Tensor t = at::as_strided(pool, shape, c10::contiguous_strides(shape), at_);
    at_ += padded(n);
    return t;
  };
  std::vector<Tensor> t;
  t.reserve(14);
  t.push_back(at::empty({Bm, nt, nt}, doc.options().dtype(at::kChar)));
  for (int i = 0; i < 4; ++i) {  // kv, full_kv, q, full_q
    t.push_back(take({Bm, 1, nt}, row));
    t.push_back(take({Bm, 1, nt, nt}, grid));
  }
  t.push_back(take({Bm, nt}, row));       // row_order
  t.push_back(take({Bm, nt}, row));       // col_order
  t.push_back(take({Bm, nt}, row));       // kv_bits_off
  t.push_back(take({Bm, nt, nt}, grid));  // q_bits_slot
  const int64_t slots = std::max<int64_t>(1, Bm * nt * (nt + 1) / 2);
  t.push_back(at::empty({slots, 2, T2T_TILE, 4}, i32));
  const auto ptr = [&](int i) { return static_cast<int32_t*>(t[i].data_ptr()); };
  t2t_block_mask m{};
  m.mask_batch = Bm;
  m.num_tiles = nt;
  m.kv_num = ptr(1); m.kv_idx = ptr(2); m.full_kv_num = ptr(3); m.full_kv_idx = ptr(4);
  m.q_num = ptr(5); m.q_idx = ptr(6); m.full_q_num = ptr(7); m.full_q_idx = ptr(8);
  m.row_order = ptr(9); m.col_order = ptr(10); m.kv_bits_off = ptr(11); m.q_bits_slot = ptr(12);
  m.tile_bits = static_cast<uint32_t*>(t[13].data_ptr());
  m.tile_bits_slots = slots;
  const int32_t* d = static_cast<const int32_t*>(doc.data_ptr());
  const uint64_t* qb = W ? static_cast<const uint64_t*>(q_bits.data_ptr()) : nullptr;
  const uint64_t* kb = W ? static_cast<const uint64_t*>(kv_bits.data_ptr()) : nullptr;
  int8_t* cls = static_cast<int8_t*>(t[0].data_ptr());
  if (window == 0) {
    check(t2t_mask_meta(d, qb, kb, Bm, T, W, cls, &m, stream), "t2t_mask_meta");
    return t;
  }
  const int32_t* start = nullptr;
  if (sinks > 0) {
    t.push_back(at::empty({Bm, T}, i32));
    start = ptr(14);
    check(t2t_doc_starts(d, Bm, T, ptr(14), stream), "t2t_doc_starts");
  }
  check(t2t_mask_meta_window(d, qb, kb, start, Bm, T, W, std::min<int64_t>(window, INT32_MAX),
                             std::min<int64_t>(sinks, INT32_MAX), cls, &m, stream),
        "t2t_mask_meta_window");
  return t;
}

std::vector<Tensor> mask_meta(const Tensor& doc, const Tensor& q_bits, const Tensor& kv_bits,
                              int64_t stream) {
  return mask_meta_window(doc, q_bits, kv_bits, 0, 0, stream);
}

// First token of each token's document, int32 of doc's shape [B, T].
Tensor doc_starts(const Tensor& doc) {
  need_gpu(doc);
  TORCH_CHECK_VALUE(doc.dim() == 2 && doc.scalar_type() == at::kInt && doc.is_contiguous(),
                    "doc must be contiguous int32 [B, T]");
  const c10::DeviceGuard guard(doc.device());
  Tensor start = at::empty_like(doc);
  check(t2t_doc_starts(static_cast<const int32_t*>(doc.data_ptr()), doc.size(0), doc.size(1),
                       static_cast<int32_t*>(start.data_ptr()), stream_of(doc)),
        "t2t_doc_starts");
  return start;
}

// doc [B, T] and, when words > 0, q / kv words [B, words, T] (else undefined)
// from the device-resident lists (int32): spans at 0, grants at `grants`,
// the counts at `counts`, and link rows (uint64) at `links` (-1: none).
std::vector<Tensor> token_inputs(const Tensor& lists, int64_t grants, int64_t counts,
                                 int64_t links, int64_t B, int64_t T, int64_t words,
                                 int64_t max_spans, int64_t max_grants, bool has_grants,
                                 const std::vector<Tensor>& out) {
  TORCH_CHECK(out.empty() || words == 0 || out.size() == 3,
              "doc, q_bits and kv_bits are needed to overwrite ", words, " words a token");
  need_gpu(lists);
  const c10::DeviceGuard guard(lists.device());
  std::vector<Tensor> t = out;
  for (const Tensor& o : t) need_gpu(o);
  if (t.empty()) {
    t.push_back(at::empty({B, T}, lists.options()));
    if (words > 0)
      for (int i = 0; i < 2; ++i)
        t.push_back(at::empty({B, words, T}, lists.options().dtype(at::kLong)));
  }
  const int32_t* base = static_cast<const int32_t*>(lists.data_ptr());
  check(t2t_token_inputs(base, base + counts, max_spans, has_grants ? base + grants : nullptr,
                         has_grants ? base + counts + B : nullptr, max_grants,
                         links >= 0 ? reinterpret_cast<const uint64_t*>(base + links) : nullptr,
                         B, T, words, static_cast<int32_t*>(t[0].data_ptr()),
                         words > 0 ? static_cast<uint64_t*>(t[1].data_ptr()) : nullptr,
                         words > 0 ? static_cast<uint64_t*>(t[2].data_ptr()) : nullptr,
                         stream_of(lists)),
        "t2t_token_inputs");
  return t;
}

// ---- the same calls recorded by autograd, from C++
//
// A call that only autograd watches (plain() below) is recorded here: a Python
// autograd.Function costs its own host time forward, and backward a switch to
// the engine's thread that waits for the interpreter.

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Results of a backward that itself has no gradient: an error where one is asked for.
variable_list once(variable_list grads, const char* what) {
  if (!c10::GradMode::is_enabled()) return grads;
  return torch::autograd::DelayedError(std::string(what) + " is differentiable once",
                                       static_cast<int64_t>(grads.size()))(std::move(grads));
}

// The mask's 13 tables (in t2t_block_mask's order) as the kernels take them.
t2t_block_mask mask_of(const std::vector<Tensor>& t) {
  TORCH_CHECK_VALUE(t.size() == 13, "a mask has 13 tables, not ", t.size());
  need_gpu(t[0]);
  const auto ptr = [&](int i) { return static_cast<int32_t*>(t[i].data_ptr()); };
  t2t_block_mask m{};
  m.mask_batch = t[0].size(0);
  m.num_tiles = t[0].size(-1);
  m.kv_num = ptr(0); m.kv_idx = ptr(1); m.full_kv_num = ptr(2); m.full_kv_idx = ptr(3);
  m.q_num = ptr(4); m.q_idx = ptr(5); m.full_q_num = ptr(6); m.full_q_idx = ptr(7);
  m.row_order = ptr(8); m.col_order = ptr(9); m.kv_bits_off = ptr(10); m.q_bits_slot = ptr(11);
  m.tile_bits = static_cast<uint32_t*>(t[12].data_ptr());
  m.tile_bits_slots = t[12].size(0);
  return m;
}

// (the tables are the mask's own, which no one writes to: kept, not saved)
struct AttentionAd : torch::autograd::Function<AttentionAd> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k,
                               const Tensor& v, const std::vector<Tensor>& tables, double scale,
                               bool uneven) {
    const t2t_block_mask m = mask_of(tables);
    auto [out, lse2, rest] =
        attn_fwd_rest(q, k, v, static_cast<int64_t>(reinterpret_cast<intptr_t>(&m)), scale, uneven);
    ctx->save_for_backward({q, k, v, out, lse2, rest});
    ctx->saved_data["tables"] = tables;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["uneven"] = uneven;
    ctx->mark_non_differentiable({lse2});
    return {out, lse2};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list t = ctx->get_saved_variables();
    const t2t_block_mask m = mask_of(ctx->saved_data["tables"].toTensorVector());
    auto [dq, dk, dv] = attn_bwd(t[0], t[1], t[2], t[3], g[0], t[4],
                                 static_cast<int64_t>(reinterpret_cast<intptr_t>(&m)),
                                 ctx->saved_data["scale"].toDouble(),
                                 ctx->saved_data["uneven"].toBool(),
                                 t[5].defined() ? c10::make_optional(t[5]) : c10::nullopt);
    variable_list d = once({dq, dk, dv}, "masked attention");
    d.resize(6);
    return d;
  }
};

std::tuple<Tensor, Tensor> attn_ad(const Tensor& q, const Tensor& k, const Tensor& v,
                                   const std::vector<Tensor>& tables, double scale, bool uneven) {
  variable_list o = AttentionAd::apply(q, k, v, tables, scale, uneven);
  return {o[0], o[1]};
}

struct QkNormAd : torch::autograd::Function<QkNormAd> {
  static variable_list forward(AutogradContext* ctx, const Tensor& qkv, const Tensor& qw,
                               const Tensor& kw, const Tensor& cos, const Tensor& sin,
                               int64_t heads, int64_t kv_heads, int64_t pos0, double eps) {
    ctx->save_for_backward({qkv, qw, kw, cos, sin});
    ctx->saved_data["n"] = std::vector<int64_t>{heads, kv_heads, pos0};
    ctx->saved_data["eps"] = eps;
    auto [q, k, v] = qk_norm_rope(qkv, qw, kw, cos, sin, heads, kv_heads, pos0, eps);
    return {q, k, v};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list t = ctx->get_saved_variables();
    const std::vector<int64_t> n = ctx->saved_data["n"].toIntVector();
    auto [dqkv, dqw, dkw] = qk_norm_rope_backward(g[0], g[1], g[2], t[0], t[1], t[2], t[3], t[4],
                                                  n[0], n[1], n[2],
                                                  ctx->saved_data["eps"].toDouble());
    variable_list d = once({dqkv, dqw, dkw}, "qk_norm_rope");
    d.resize(9);
    return d;
  }
};

std::tuple<Tensor, Tensor, Tensor> qk_norm_rope_ad(const Tensor& qkv, const Tensor& qw,
                                                   const Tensor& kw, const Tensor& cos,
                                                   const Tensor& sin, int64_t heads,
                                                   int64_t kv_heads, int64_t pos0, double eps) {
  variable_list o = QkNormAd::apply(qkv, qw, kw, cos, sin, heads, kv_heads, pos0, eps);
  return {o[0], o[1], o[2]};
}

// The rotation is linear, so each direction's gradient is the other one, and
// both may be differentiated again.
struct RotaryAd {
  using Pos = c10::optional<Tensor>;
  static void keep(AutogradContext* ctx, const Tensor& cos, const Tensor& sin, const Pos& pos,
                   std::vector<int64_t> n) {
    ctx->save_for_backward({cos, sin, pos.has_value() ? *pos : Tensor()});
    ctx->saved_data["n"] = std::move(n);
  }
  struct Kept {
    variable_list t;
    std::vector<int64_t> n;  // heads, kv_heads, pos0, interleaved
    Pos pos;
    explicit Kept(AutogradContext* ctx)
        : t(ctx->get_saved_variables()), n(ctx->saved_data["n"].toIntVector()) {
      if (t[2].defined()) pos = t[2];
    }
  };
  struct Forward : torch::autograd::Function<Forward> {
    static variable_list forward(AutogradContext* ctx, const Tensor& qkv, const Tensor& cos,
                                 const Tensor& sin, int64_t heads, int64_t kv_heads,
                                 const Pos& pos, int64_t pos0, bool interleaved) {
      keep(ctx, cos, sin, pos, {heads, kv_heads, pos0, interleaved});
      auto [q, k, v] = qkv_rotary(qkv, cos, sin, heads, kv_heads, pos, pos0, interleaved);
      return {q, k, v};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
      const Kept a(ctx);
      variable_list d(8);
      d[0] = c10::GradMode::is_enabled()
                 ? Backward::apply(g[0], g[1], g[2], a.t[0], a.t[1], a.pos, a.n[0], a.n[1], a.n[2],
                                   a.n[3] != 0)
                 : qkv_rotary_backward(g[0], g[1], g[2], a.t[0], a.t[1], a.pos, a.n[2],
                                       a.n[3] != 0);
      return d;
    }
  };
  struct Backward : torch::autograd::Function<Backward> {
    static Tensor forward(AutogradContext* ctx, const Tensor& dq, const Tensor& dk,
                          const Tensor& dv, const Tensor& cos, const Tensor& sin, const Pos& pos,
                          int64_t heads, int64_t kv_heads, int64_t pos0, bool interleaved) {
      keep(ctx, cos, sin, pos, {heads, kv_heads, pos0, interleaved});
      return qkv_rotary_backward(dq, dk, dv, cos, sin, pos, pos0, interleaved);
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
      const Kept a(ctx);
      variable_list d =
          Forward::apply(g[0], a.t[0], a.t[1], a.n[0], a.n[1], a.pos, a.n[2], a.n[3] != 0);
      d.resize(10);
      return d;
    }
  };
};

std::tuple<Tensor, Tensor, Tensor> qkv_rotary_ad(const Tensor& qkv, const Tensor& cos,
                                                 const Tensor& sin, int64_t heads,
                                                 int64_t kv_heads,
                                                 const c10::optional<Tensor>& pos, int64_t pos0,
                                                 bool interleaved) {
  variable_list o =
      RotaryAd::Forward::apply(qkv, cos, sin, heads, kv_heads, pos, pos0, interleaved);
  return {o[0], o[1], o[2]};
}

struct EmbeddingAd : torch::autograd::Function<EmbeddingAd> {
  static Tensor forward(AutogradContext* ctx, const Tensor& tokens, const Tensor& weight,
                        double scale, int64_t padding) {
    ctx->save_for_backward({tokens});
    ctx->saved_data["n"] = std::vector<int64_t>{weight.size(0), padding};
    ctx->saved_data["scale"] = scale;
    return embedding(tokens, weight, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const std::vector<int64_t> n = ctx->saved_data["n"].toIntVector();
    variable_list d = once({embedding_backward(ctx->get_saved_variables()[0], g[0], n[0],
                                               ctx->saved_data["scale"].toDouble(), n[1])},
                           "embedding");
    return {Tensor(), d[0], Tensor(), Tensor()};
  }
};

Tensor embedding_ad(const Tensor& tokens, const Tensor& weight, double scale, int64_t padding) {
  return EmbeddingAd::apply(tokens, weight, scale, padding);
}

// Whether hooks take what a graph saves: a recomputed region's, which drops it,
// or a user's, which moves it elsewhere.
bool saved_tensors_hooked() {
  return !at::SavedTensorDefaultHooks::get_tls_state().stack.empty();
}

// A sum or mean is differentiated with an incoming gradient of 1 as a rule, so
// the forward's pass over the logits writes its gradient.  Kept beside what the
// graph saves, it would stay where hooks take the rest away, so it is then left
// to the backward.
struct DistillAd : torch::autograd::Function<DistillAd> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& idx,
                        const Tensor& teacher, const c10::optional<Tensor>& target,
                        double temperature, double alpha, int64_t ignore_index,
                        int64_t reduction) {
    auto [loss, grad, inv] =
        distill_loss(logits, idx, teacher, target, temperature, alpha, ignore_index, reduction,
                     reduction != 0 && logits.requires_grad() && !saved_tensors_hooked());
    ctx->save_for_backward({logits, idx, teacher, target.has_value() ? *target : Tensor(), inv});
    ctx->saved_data["x"] = std::vector<double>{temperature, alpha};
    ctx->saved_data["n"] = std::vector<int64_t>{ignore_index, reduction};
    if (grad.defined()) ctx->saved_data["kept"] = grad;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto given = [](const Tensor& t) {
      return t.defined() ? c10::optional<Tensor>(t) : c10::nullopt;
    };
    const variable_list t = ctx->get_saved_variables();
    const std::vector<double> x = ctx->saved_data["x"].toDoubleVector();
    const std::vector<int64_t> n = ctx->saved_data["n"].toIntVector();
    c10::optional<Tensor> kept;  // handed over: a second backward computes its own
    const auto at = ctx->saved_data.find("kept");
    if (at != ctx->saved_data.end()) {
      kept = at->second.toTensor();
      ctx->saved_data.erase(at);
    }
    variable_list d = once({distill_loss_backward(g[0], t[0], t[1], t[2], given(t[3]), x[0], x[1],
                                                  n[0], n[1], given(t[4]), kept)},
                           "distill_loss");
    d.resize(8);
    return d;
  }
};

Tensor distill_loss_ad(const Tensor& logits, const Tensor& idx, const Tensor& teacher,
                       const c10::optional<Tensor>& target, double temperature, double alpha,
                       int64_t ignore_index, int64_t reduction) {
  return DistillAd::apply(logits, idx, teacher, target, temperature, alpha, ignore_index,
                          reduction);
}

// ---- what may be watching a call

// Nothing but the caller sees the call, and the tensors are what their
// addresses say: no tracer, dispatch mode or function transform is active,
// and every argument is a torch.Tensor or Parameter itself (not a subclass)
// with plain memory of its own (not batched, nested, sparse or lazily
// negated).  A kernel called on addresses would be missing from a trace, and
// its output in it is the empty allocation.
bool plain_call(PyObject* const* args, Py_ssize_t n, bool recorded_counts) {
  constexpr c10::DispatchKeySet kIndirect{
      c10::DispatchKey::Batched,    c10::DispatchKey::FuncTorchBatched,
      c10::DispatchKey::Python,     c10::DispatchKey::NestedTensor,
      c10::DispatchKey::Negative,   c10::DispatchKey::Conjugate,
      c10::DispatchKey::ZeroTensor, c10::DispatchKey::Functionalize};
  if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::any_modes_set() ||
      c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode))
    return false;
  const bool grad = recorded_counts && c10::GradMode::is_enabled();
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (!THPVariable_CheckExact(args[i])) return false;
    const Tensor& t = THPVariable_Unpack(args[i]);
    if (t.key_set().has_any(kIndirect) || t.layout() != at::kStrided || !t.has_storage() ||
        (grad && t.requires_grad()))
      return false;
  }
  return true;
}

PyObject* plain(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return PyBool_FromLong(plain_call(args, n, false));
}

PyObject* unwatched(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return PyBool_FromLong(plain_call(args, n, true));
}

PyMethodDef kPredicates[] = {
    {"plain", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(plain)), METH_FASTCALL,
     "plain(*tensors): nothing but the caller sees a call on them"},
    {"unwatched", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(unwatched)),
     METH_FASTCALL, "plain(*tensors), and no graph records it"},
    {nullptr, nullptr, 0, nullptr}};

int64_t current_stream(int64_t device) {
  return reinterpret_cast<int64_t>(
      at::hip::getCurrentHIPStreamMasqueradingAsCUDA(static_cast<c10::DeviceIndex>(device))
          .stream());
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  // a launch may wait on a full queue, an allocation on the device: other
  // Python threads run meanwhile
  const auto no_gil = py::call_guard<py::gil_scoped_release>();
  m.def("attn_fwd", &attn_fwd, no_gil);
  m.def("attn_fwd_rest", &attn_fwd_rest, no_gil);
  m.def("attn_bwd", &attn_bwd, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("out"),
        py::arg("dout"), py::arg("lse2"), py::arg("mask"), py::arg("scale"),
        py::arg("uneven") = false, py::arg("rest") = py::none(), no_gil);
  m.def("rms_norm", &rms_norm, no_gil);
  m.def("rms_norm_backward", &rms_norm_backward, no_gil);
  m.def("qkv_rope", &qkv_rope, no_gil);
  m.def("qkv_rope_backward", &qkv_rope_backward, no_gil);
  m.def("qk_norm_rope", &qk_norm_rope, no_gil);
  m.def("qk_norm_rope_backward", &qk_norm_rope_backward, no_gil);
  m.def("qk_norm_rope_append", &qk_norm_rope_append, no_gil);
  m.def("qk_norm_rope_ad", &qk_norm_rope_ad, no_gil);
  m.def("qkv_rotary", &qkv_rotary, no_gil);
  m.def("qkv_rotary_backward", &qkv_rotary_backward, no_gil);
  m.def("qkv_rotary_ad", &qkv_rotary_ad, no_gil);
  m.def("attn_ad", &attn_ad, no_gil);
  m.def("attn_decode", &attn_decode, no_gil);
  m.def("kv8_append", &kv8_append, no_gil);
  m.def("kv8_attend", &kv8_attend, no_gil);
  m.def("embedding_ad", &embedding_ad, no_gil);
  m.def("distill_loss_ad", &distill_loss_ad, no_gil);
  m.def("embedding", &embedding, no_gil);
  m.def("embedding_backward", &embedding_backward, no_gil);
  m.def("distill_loss", &distill_loss, no_gil);
  m.def("distill_loss_backward", &distill_loss_backward, no_gil);
  m.def("distill_rows_", &distill_rows_, no_gil);
  m.def("saved_tensors_hooked", &saved_tensors_hooked);
  m.def("distill_count", &distill_count, no_gil);
  m.def("distill_mean", &distill_mean, no_gil);
  m.def("swiglu", &swiglu, no_gil);
  m.def("swiglu_backward",
        [](const Tensor& g2, const Tensor& dh, const std::vector<int64_t>& shape) {
          return swiglu_backward(g2, dh, shape);
        }, no_gil);
  m.def("linear", &linear, no_gil);
  m.def("wgrad", [](const Tensor& dy, const Tensor& x, bool f32) {
    return wgrad(dy, x, f32 ? at::kFloat : at::kBFloat16);
  }, no_gil);
  m.def("mask_meta", &mask_meta, no_gil);
  m.def("mask_meta_window", &mask_meta_window, no_gil);
  m.def("doc_starts", &doc_starts, no_gil);
  m.def("token_inputs", &token_inputs, no_gil);
  m.def("current_stream", &current_stream);
  if (PyModule_AddFunctions(m.ptr(), kPredicates) != 0) throw py::error_already_set();
}
