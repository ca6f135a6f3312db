// Host side of the operators around attention for PyTorch tensors: argument checks, allocation, the calls of the
// C ABI (include/tattn.h) and autograd.
//
// tattn.attention does this in Python through ctypes. Here the device part of a call is often a few
// microseconds (one token's heads, one token over a short cache), and a training step's autograd through
// Python costs more than its kernels: qk_norm_rope of one token took 21 us a call and 173 us forward and
// backward that way. Nothing in this file touches device memory; it is built against the installed
// PyTorch into tattn/_torch_ext.so and finds libtattn_b200.so beside it.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <cmath>
#include <limits>
#include <optional>
#include <vector>

#include "../../include/tattn.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kGroupDims = 64;  // head dims that share a scale and a minimum in the 4-bit cache

// ------------------------------------------------------------------------------------------ helpers
// A refused argument is a ValueError.
#define CHECK_VALUE(condition, ...) \
  do {                              \
    if (!(condition)) throw pybind11::value_error(c10::str(__VA_ARGS__)); \
  } while (false)

// A library status as an error. With the GIL (a direct call): tattn._lib.TattnError; in an autograd worker: a
// RuntimeError of the same text.
void check_status(const char* fn, int rc) {
  if (rc == TATTN_OK) return;
  if (PyGILState_Check()) pybind11::module_::import("tattn._lib").attr("check")(fn, rc);
  TORCH_CHECK(false, fn, " failed with status ", rc, ": ", tattn_status_string(rc));
}

void require_cuda(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "tattn_b200 runs only on CUDA sm_100 devices (got a tensor on ", t.device(),
              "); there is no CPU path");
}

bool head_dim_ok(int64_t d) { return d == 16 || d == 32 || d == 64 || d == 128; }
bool dtype_ok(const Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kFloat; }
int code(const Tensor& t) { return t.scalar_type() == at::kHalf ? TATTN_F16 : TATTN_F32; }
int clamp_int(int64_t x) { return int(std::min<int64_t>(x, std::numeric_limits<int>::max())); }
int dim(const Tensor& t, int i) {
  CHECK_VALUE(t.size(i) <= std::numeric_limits<int>::max(), "dimension ", i, " of ", t.sizes(), " is too large");
  return int(t.size(i));
}
bool aligned16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// Can the last dimension's rows be read 16 bytes at a time?
bool rows16_ok(const Tensor& t) {
  if (t.stride(-1) != 1 || !aligned16(t)) return false;
  const int64_t unit = 16 / t.element_size();
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) % unit != 0) return false;
  return true;
}
Tensor dense16(const Tensor& t) {
  Tensor c = t.contiguous();
  return aligned16(c) ? c : c.clone();
}
Tensor rows16(const Tensor& t) { return rows16_ok(t) ? t : dense16(t); }
// In place if the fp16 kernels' TMA can address it, else a dense copy.
Tensor tma_ready(const Tensor& t) {
  return tattn_layout_ok(t.data_ptr(), t.strides().data(), dim(t, 0), dim(t, 1), dim(t, 2), dim(t, 3)) ? t : dense16(t);
}
// A tensor for results, dense in the order of t's dimensions where that leaves 16-byte rows.
Tensor like(const Tensor& t) {
  Tensor out = at::empty_like(t);
  return rows16_ok(out) ? out : at::empty(t.sizes(), t.options());
}

struct Strides {
  int64_t s[26];
  int n = 0;
  void add(const Tensor& t) {
    for (int64_t x : t.strides()) s[n++] = x;
  }
  void add(int64_t a, int64_t b) {
    s[n++] = a;
    s[n++] = b;
  }
};

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
Tensor bytes(int64_t size, const Tensor& like) { return at::empty({size}, like.options().dtype(at::kByte)); }
void* ptr(const std::optional<Tensor>& t) { return t.has_value() ? t->data_ptr() : nullptr; }

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->requires_grad()) return true;
  return false;
}
// None of the operators carries forward-mode derivatives: a result without a tangent would say that it is zero.
void refuse_forward_mode(const char* fn, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), fn, " has no forward-mode derivatives");
}
// A backward that can be differentiated once: its results raise when differentiated again.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  std::vector<int> at;
  variable_list in;
  for (size_t i = 0; i < grads.size(); ++i)
    if (grads[i].defined()) {
      at.push_back(int(i));
      in.push_back(grads[i].detach().requires_grad_());
    }
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with once_differentiable", int(in.size()));
  variable_list out = (*error)(std::move(in));
  for (size_t i = 0; i < at.size(); ++i) grads[at[i]] = out[i];
  return grads;
}

// ------------------------------------------------------------------------- head norms with rotation
void check_norm_rope(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, const Tensor& cos,
                     const Tensor& sin, const std::optional<Tensor>& positions) {
  CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && q.size(0) == k.size(0) && q.size(2) == k.size(2) && q.size(3) == k.size(3),
                    "expected q [batch, heads, seq, dim] and k [batch, kv_heads, seq, dim]; got ", q.sizes(), ", ", k.sizes());
  const int64_t b = q.size(0), n = q.size(2), d = q.size(3);
  CHECK_VALUE(q.size(1) > 0 && k.size(1) > 0, "q and k need at least one head; got ", q.sizes(), ", ", k.sizes());
  CHECK_VALUE(head_dim_ok(d), "head dim must be 16, 32, 64 or 128, got ", d);
  CHECK_VALUE(k.scalar_type() == q.scalar_type() && dtype_ok(q), "q, k must share dtype float16 or float32, got ",
                    q.scalar_type(), ", ", k.scalar_type());
  CHECK_VALUE(wq.dim() == 1 && wk.dim() == 1 && wq.size(0) == d && wk.size(0) == d, "weights must have shape [", d,
                    "]; got ", wq.sizes(), ", ", wk.sizes());
  CHECK_VALUE(wk.scalar_type() == wq.scalar_type() && (wq.scalar_type() == q.scalar_type() || wq.scalar_type() == at::kFloat),
                    "weights must share q's dtype or float32; got ", wq.scalar_type(), ", ", wk.scalar_type());
  CHECK_VALUE(cos.dim() == 2 && cos.size(1) == d / 2 && sin.sizes() == cos.sizes(),
                    "cos and sin must have shape [positions, ", d / 2, "]; got ", cos.sizes(), ", ", sin.sizes());
  CHECK_VALUE(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat, "cos and sin must be float32; got ",
                    cos.scalar_type(), ", ", sin.scalar_type());
  if (!positions.has_value()) {
    CHECK_VALUE(cos.size(0) >= n, "the tables hold ", cos.size(0), " positions, fewer than the ", n, " tokens");
  } else {
    const Tensor& p = *positions;
    const bool shape = (p.dim() == 1 && p.size(0) == n) || (p.dim() == 2 && p.size(0) == b && p.size(1) == n);
    CHECK_VALUE(p.scalar_type() == at::kInt && shape, "positions must be int32 [", n, "] or [", b, ", ", n, "]; got ",
                      p.scalar_type(), " ", p.sizes());
    CHECK_VALUE(cos.size(0) > 0 || b * n == 0, "the tables hold no positions");
    CHECK_VALUE(p.device() == q.device(), "all tensors must be on one device, got ", q.device(), " and ", p.device());
  }
  TORCH_CHECK(!wants_grad({&cos, &sin}), "cos and sin get no gradients; detach them");
  refuse_forward_mode("qk_norm_rope", {&q, &k, &wq, &wk, &cos, &sin});
  for (const Tensor* t : {&k, &wq, &wk, &cos, &sin})
    CHECK_VALUE(t->device() == q.device(), "all tensors must be on one device, got ", q.device(), " and ", t->device());
  require_cuda(q);
}

void add_positions(Strides& st, const std::optional<Tensor>& p) {
  if (!p.has_value()) return st.add(0, 0);
  p->dim() == 1 ? st.add(0, p->stride(0)) : st.add(p->stride(0), p->stride(1));
}

std::tuple<Tensor, Tensor> norm_rope_forward(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk,
                                             const Tensor& cos, const Tensor& sin, const std::optional<Tensor>& positions,
                                             double eps, bool interleaved) {
  Tensor q_out = like(q), k_out = like(k);
  Strides st;
  st.add(q);
  st.add(k);
  st.add(q_out);
  st.add(k_out);
  add_positions(st, positions);
  const c10::cuda::CUDAGuard guard(q.device());
  check_status("tattn_qk_norm_rope",
               tattn_qk_norm_rope(q.data_ptr(), k.data_ptr(), wq.data_ptr(), wk.data_ptr(), q_out.data_ptr(), k_out.data_ptr(),
                                  cos.data_ptr<float>(), sin.data_ptr<float>(), static_cast<const int32_t*>(ptr(positions)), st.s,
                                  dim(q, 0), dim(q, 1), dim(k, 1), dim(q, 2), dim(q, 3), dim(cos, 0), code(q), code(wq),
                                  float(eps), interleaved, stream_of(q)));
  return {q_out, k_out};
}

struct QkNormRope : torch::autograd::Function<QkNormRope> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk,
                               const Tensor& cos, const Tensor& sin, const std::optional<Tensor>& positions, double eps,
                               bool interleaved) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({q, k, wq, wk, cos, sin, positions.has_value() ? *positions : Tensor()});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    auto [q_out, k_out] = norm_rope_forward(q, k, wq, wk, cos, sin, positions, eps, interleaved);
    return {q_out, k_out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(9);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const variable_list saved = ctx->get_saved_variables();
      const Tensor &q = saved[0], &k = saved[1], &wq = saved[2], &wk = saved[3], &cos = saved[4], &sin = saved[5];
      const std::optional<Tensor> positions = saved[6].defined() ? std::optional<Tensor>(saved[6]) : std::nullopt;
      const Tensor gq = rows16(grads[0].defined() ? grads[0] : at::zeros_like(q));
      const Tensor gk = rows16(grads[1].defined() ? grads[1] : at::zeros_like(k));
      Tensor dq = like(q), dk = like(k), dwq = at::empty_like(wq), dwk = at::empty_like(wk);
      Strides st;
      st.add(q);
      st.add(k);
      st.add(gq);
      st.add(gk);
      st.add(dq);
      st.add(dk);
      add_positions(st, positions);
      const c10::cuda::CUDAGuard guard(q.device());
      const Tensor ws = bytes(tattn_qk_norm_rope_bwd_workspace_bytes(dim(q, 3)), q);
      check_status("tattn_qk_norm_rope_bwd",
                   tattn_qk_norm_rope_bwd(q.data_ptr(), k.data_ptr(), wq.data_ptr(), wk.data_ptr(), gq.data_ptr(), gk.data_ptr(),
                                          dq.data_ptr(), dk.data_ptr(), dwq.data_ptr(), dwk.data_ptr(), cos.data_ptr<float>(),
                                          sin.data_ptr<float>(), static_cast<const int32_t*>(ptr(positions)), ws.data_ptr(), st.s,
                                          dim(q, 0), dim(q, 1), dim(k, 1), dim(q, 2), dim(q, 3), dim(cos, 0), code(q), code(wq),
                                          float(ctx->saved_data["eps"].toDouble()), ctx->saved_data["interleaved"].toBool(),
                                          stream_of(q)));
      out[0] = dq;
      out[1] = dk;
      out[2] = dwq;
      out[3] = dwk;
    }
    return once(std::move(out));
  }
};

std::tuple<Tensor, Tensor> qk_norm_rope(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, const Tensor& cos,
                                        const Tensor& sin, const std::optional<Tensor>& positions, double eps, bool interleaved) {
  check_norm_rope(q, k, wq, wk, cos, sin, positions);
  const Tensor q_ = rows16(q), k_ = rows16(k), wq_ = dense16(wq), wk_ = dense16(wk), cos_ = dense16(cos), sin_ = dense16(sin);
  if (!wants_grad({&q, &k, &wq, &wk})) return norm_rope_forward(q_, k_, wq_, wk_, cos_, sin_, positions, eps, interleaved);
  variable_list out = QkNormRope::apply(q_, k_, wq_, wk_, cos_, sin_, positions, eps, interleaved);
  return {out[0], out[1]};
}

// --------------------------------------------------------------------------------- window attention
void check_heads(const Tensor& q, const Tensor& k, const Tensor& v) {
  CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && v.sizes() == k.sizes(),
                    "expected q [batch, heads, seq, dim] and k, v of equal shape [batch, kv_heads, kv_seq, dim]; got ", q.sizes(),
                    ", ", k.sizes(), ", ", v.sizes());
  CHECK_VALUE(k.size(0) == q.size(0) && k.size(3) == q.size(3), "q and k must agree in batch and head dim; got ", q.sizes(),
                    ", ", k.sizes());
  CHECK_VALUE(k.size(1) > 0 && q.size(1) % k.size(1) == 0, "query heads must be a multiple of key/value heads; got ",
                    q.size(1), " and ", k.size(1));
  CHECK_VALUE(k.device() == q.device() && v.device() == q.device(), "q, k, v must be on one device, got ", q.device(), ", ",
                    k.device(), ", ", v.device());
  CHECK_VALUE(head_dim_ok(q.size(3)), "head dim must be 16, 32, 64 or 128, got ", q.size(3));
  CHECK_VALUE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() && dtype_ok(q),
                    "q, k, v must share dtype float16 or float32, got ", q.scalar_type(), ", ", k.scalar_type(), ", ",
                    v.scalar_type());
}
void check_window(const std::optional<int64_t>& window, int64_t sinks) {
  CHECK_VALUE(!window.has_value() || *window >= 1, "window must be at least 1, got ", window.value_or(0));
  CHECK_VALUE(sinks >= 0, "sinks must not be negative, got ", sinks);
}
double scale_of(const std::optional<double>& sm_scale, const Tensor& q) {
  return sm_scale.has_value() ? *sm_scale : 1.0 / std::sqrt(double(q.size(3)));
}

// (O like q, M fp32 [Z, H, Nq]) of checked tensors and, in fp16 with `rest`, what rounding took off O, for a
// backward pass (else an undefined tensor).
std::tuple<Tensor, Tensor, Tensor> window_forward_rest(const Tensor& q0, const Tensor& k0, const Tensor& v0, int64_t window,
                                                       int64_t sinks, double scale, bool rest) {
  const bool half = q0.scalar_type() == at::kHalf;
  const Tensor q = half ? tma_ready(q0) : q0, k = half ? tma_ready(k0) : k0, v = half ? tma_ready(v0) : v0;
  Tensor o = like(q), m = at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat)), o_rest;
  if (rest && half) o_rest = at::empty(q.sizes(), q.options().dtype(at::kByte), at::MemoryFormat::Contiguous);
  Strides st;
  st.add(q);
  st.add(k);
  st.add(v);
  st.add(o);
  const c10::cuda::CUDAGuard guard(q.device());
  check_status("tattn_window_fwd",
               tattn_window_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), m.data_ptr<float>(),
                                o_rest.defined() ? o_rest.data_ptr() : nullptr, st.s, dim(q, 0), dim(q, 1), dim(k, 1),
                                dim(q, 2), dim(k, 2), dim(q, 3), code(q), clamp_int(window),
                                clamp_int(sinks), float(scale), stream_of(q)));
  return {o, m, o_rest};
}
std::tuple<Tensor, Tensor> window_forward(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks,
                                          double scale) {
  const auto [o, m, rest] = window_forward_rest(q, k, v, window, sinks, scale, false);
  return {o, m};
}

// Dense (dq, dk, dv); rest: the forward's, or undefined.
std::tuple<Tensor, Tensor, Tensor> window_backward_rest(const Tensor& q0, const Tensor& k0, const Tensor& v0, const Tensor& o0,
                                                        const Tensor& m, const Tensor& rest, const Tensor& do0,
                                                        int64_t window, int64_t sinks, double scale) {
  const bool half = q0.scalar_type() == at::kHalf;
  const Tensor dout = do0.to(q0.scalar_type());
  const Tensor q = half ? tma_ready(q0) : q0, k = half ? tma_ready(k0) : k0, v = half ? tma_ready(v0) : v0;
  const Tensor o = half ? tma_ready(o0) : dense16(o0), g = half ? tma_ready(dout) : dense16(dout);
  const int z = dim(q, 0), h = dim(q, 1), hk = dim(k, 1), n = dim(q, 2), nk = dim(k, 2), d = dim(q, 3);
  const int w = clamp_int(window), s = clamp_int(sinks);
  Tensor delta = at::empty({z, h, n}, q.options().dtype(at::kFloat));
  Tensor dq = at::empty({z, h, n, d}, q.options()), dk = at::empty({z, hk, nk, d}, q.options());
  Tensor dv = at::empty({z, hk, nk, d}, q.options());
  Strides st;
  st.add(q);
  st.add(k);
  st.add(v);
  st.add(o);
  st.add(g);
  const c10::cuda::CUDAGuard guard(q.device());
  const Tensor ws = bytes(std::max<int64_t>(0, tattn_window_bwd_workspace_bytes(z, h, hk, n, nk, d, code(q), w, s)), q);
  check_status("tattn_window_bwd",
               tattn_window_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), g.data_ptr(), dq.data_ptr(),
                                dk.data_ptr(), dv.data_ptr(), m.data_ptr<float>(), rest.defined() ? rest.data_ptr() : nullptr,
                                delta.data_ptr<float>(), ws.data_ptr(), st.s, z, h, hk, n, nk, d, code(q), w, s, float(scale), stream_of(q)));
  return {dq, dk, dv};
}
std::tuple<Tensor, Tensor, Tensor> window_backward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o,
                                                   const Tensor& m, const Tensor& dout, int64_t window, int64_t sinks,
                                                   double scale) {
  return window_backward_rest(q, k, v, o, m, Tensor(), dout, window, sinks, scale);
}

struct WindowAttention : torch::autograd::Function<WindowAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks,
                        double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [o, m, rest] = window_forward_rest(q, k, v, window, sinks, scale, true);
    ctx->save_for_backward({q, k, v, o, m, rest});
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    ctx->saved_data["scale"] = scale;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(6);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const variable_list s = ctx->get_saved_variables();
      std::tie(out[0], out[1], out[2]) =
          window_backward_rest(s[0], s[1], s[2], s[3], s[4], s[5], grads[0], ctx->saved_data["window"].toInt(),
                          ctx->saved_data["sinks"].toInt(), ctx->saved_data["scale"].toDouble());
    }
    return once(std::move(out));
  }
};

Tensor window_attention(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks,
                        const std::optional<double>& sm_scale) {
  check_heads(q, k, v);
  check_window(window, sinks);
  CHECK_VALUE(k.size(2) >= q.size(2), "the queries are the last of the keys' sequence; got ", q.size(2), " queries, ",
                    k.size(2), " keys");
  refuse_forward_mode("window_attention", {&q, &k, &v});
  require_cuda(q);
  if (!wants_grad({&q, &k, &v})) return std::get<0>(window_forward(q, k, v, window, sinks, scale_of(sm_scale, q)));
  return WindowAttention::apply(q, k, v, window, sinks, scale_of(sm_scale, q));
}

// ------------------------------------------------------------------------- single tokens over a cache
// inputs: q, and the keys and values that may need gradients.
void check_token(std::initializer_list<const Tensor*> inputs, const Tensor& lengths, const std::optional<int64_t>& window,
                 int64_t sinks) {
  const Tensor& q = **inputs.begin();
  CHECK_VALUE(q.size(2) == 1, "q holds one token of each sequence; got ", q.sizes());
  CHECK_VALUE(lengths.scalar_type() == at::kInt && lengths.dim() == 1 && lengths.size(0) == q.size(0),
                    "lengths must be int32 [", q.size(0), "]; got ", lengths.scalar_type(), " ", lengths.sizes());
  CHECK_VALUE(lengths.device() == q.device(), "lengths must be on q's device, got ", lengths.device());
  TORCH_CHECK(!wants_grad(inputs), "attention over a cache has no backward pass; use window_attention, or torch.no_grad()");
  check_window(window, sinks);
}

Tensor decode_attention(const Tensor& q0, const Tensor& k, const Tensor& v, const Tensor& lengths0,
                        const std::optional<int64_t>& window, int64_t sinks, const std::optional<double>& sm_scale) {
  check_heads(q0, k, v);
  check_token({&q0, &k, &v}, lengths0, window, sinks);
  refuse_forward_mode("decode_attention", {&q0, &k, &v});
  require_cuda(q0);
  CHECK_VALUE(rows16_ok(k) && rows16_ok(v),
                    "k and v need contiguous, 16-byte aligned rows: a cache is read in place, never copied");
  const Tensor q = rows16(q0), lengths = lengths0.contiguous();
  Tensor o = like(q);
  if (o.numel() == 0) return o;
  const int z = dim(q, 0), h = dim(q, 1), hk = dim(k, 1), cap = dim(k, 2), d = dim(q, 3);
  const int w = clamp_int(window.value_or(0)), s = clamp_int(sinks);
  Strides st;
  st.add(q);
  st.add(k);
  st.add(v);
  st.add(o);
  const c10::cuda::CUDAGuard guard(q.device());
  const int64_t size = tattn_decode_workspace_bytes(z, h, hk, cap, d, code(q), w, s);
  const Tensor ws = size > 0 ? bytes(size, q) : Tensor();
  check_status("tattn_decode",
               tattn_decode(q.data_ptr(), k.data_ptr(), v.data_ptr(), lengths.data_ptr<int>(), o.data_ptr(),
                            size > 0 ? ws.data_ptr() : nullptr, st.s, z, h, hk, cap, d, code(q), w, s,
                            float(scale_of(sm_scale, q)), stream_of(q)));
  return o;
}

// ------------------------------------------------------------------------------------- 4-bit cache
// The cache's tensors, as tattn.Int4Cache holds them.
void int4_check(const Tensor& kc, const Tensor& kp, const Tensor& vc, const Tensor& vp) {
  CHECK_VALUE(kc.dim() == 4 && (kc.size(3) == 32 || kc.size(3) == 64),
                    "codes must be [batch, kv_heads, capacity, dim / 2] for dim 64 or 128; got ", kc.sizes());
  const std::vector<int64_t> params = {kc.size(0), kc.size(1), kc.size(2), kc.size(3) * 2 / kGroupDims, 2};
  CHECK_VALUE(vc.sizes() == kc.sizes() && kp.sizes() == params && vp.sizes() == params, "expected codes ", kc.sizes(),
                    " and params ", params, "; got ", vc.sizes(), ", ", kp.sizes(), ", ", vp.sizes());
  for (const Tensor* t : {&kc, &kp, &vc, &vp}) {
    const bool is_code = t == &kc || t == &vc;
    CHECK_VALUE(t->scalar_type() == (is_code ? at::kByte : at::kHalf) && t->device() == kc.device(),
                      "codes must be uint8 and params float16 on one device; got ", t->scalar_type(), " on ", t->device());
    CHECK_VALUE(t->is_contiguous() && aligned16(*t), "the cache's tensors must be contiguous and 16-byte aligned");
  }
}

std::optional<Tensor> check_index(const char* name, const std::optional<Tensor>& t, const Tensor& kc) {
  if (!t.has_value()) return std::nullopt;
  CHECK_VALUE(t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == kc.size(0) && t->device() == kc.device(), name,
                    " must be int32 [", kc.size(0), "] on ", kc.device(), "; got ", t->scalar_type(), " ", t->sizes(), " on ",
                    t->device());
  return t->contiguous();
}

void int4_append(const Tensor& kc, const Tensor& kp, const Tensor& vc, const Tensor& vp, const Tensor& k0, const Tensor& v0,
                 const std::optional<Tensor>& start0, const std::optional<Tensor>& counts0) {
  const int64_t d = kc.size(3) * 2;
  CHECK_VALUE(k0.dim() == 4 && k0.size(0) == kc.size(0) && k0.size(1) == kc.size(1) && k0.size(3) == d &&
                        v0.sizes() == k0.sizes(),
                    "expected k, v [", kc.size(0), ", ", kc.size(1), ", seq, ", d, "]; got ", k0.sizes(), ", ", v0.sizes());
  CHECK_VALUE(k0.scalar_type() == at::kHalf && v0.scalar_type() == at::kHalf, "k, v must be float16, got ",
                    k0.scalar_type(), ", ", v0.scalar_type());
  CHECK_VALUE(k0.device() == kc.device() && v0.device() == kc.device(), "k, v and the cache must be on one device, got ",
                    k0.device(), ", ", v0.device());
  const std::optional<Tensor> start = check_index("start", start0, kc), counts = check_index("counts", counts0, kc);
  TORCH_CHECK(!wants_grad({&k0, &v0}), "the cache carries no gradients; detach k and v, or use torch.no_grad()");
  refuse_forward_mode("Int4Cache.append", {&k0, &v0});
  require_cuda(k0);
  const Tensor k = rows16(k0), v = rows16(v0);
  Strides st;
  st.add(k);
  st.add(v);
  const c10::cuda::CUDAGuard guard(k.device());
  check_status("tattn_int4_append",
               tattn_int4_append(k.data_ptr(), v.data_ptr(), kc.data_ptr(), kp.data_ptr(), vc.data_ptr(), vp.data_ptr(),
                                 static_cast<const int32_t*>(ptr(start)), static_cast<const int32_t*>(ptr(counts)), st.s, dim(kc, 0),
                                 dim(kc, 1), dim(k, 2), dim(kc, 2), int(d), stream_of(k)));
}

std::tuple<Tensor, Tensor> int4_read(const Tensor& kc, const Tensor& kp, const Tensor& vc, const Tensor& vp, int64_t count,
                                     const std::optional<Tensor>& start0) {
  CHECK_VALUE(count >= 0, "count must not be negative, got ", count);
  const std::optional<Tensor> start = check_index("start", start0, kc);
  require_cuda(kc);
  const std::vector<int64_t> shape = {kc.size(0), kc.size(1), count, kc.size(3) * 2};
  Tensor k = at::empty(shape, kp.options()), v = at::empty(shape, kp.options());
  const c10::cuda::CUDAGuard guard(k.device());
  check_status("tattn_int4_read", tattn_int4_read(kc.data_ptr(), kp.data_ptr(), vc.data_ptr(), vp.data_ptr(),
                                                  static_cast<const int32_t*>(ptr(start)), k.data_ptr(), v.data_ptr(), dim(kc, 0),
                                                  dim(kc, 1), dim(k, 2), dim(kc, 2), dim(k, 3), stream_of(k)));
  return {k, v};
}

Tensor int4_attend(const Tensor& kc, const Tensor& kp, const Tensor& vc, const Tensor& vp, const Tensor& q0,
                   const Tensor& lengths0, const std::optional<int64_t>& window, int64_t sinks,
                   const std::optional<double>& sm_scale) {
  const int64_t d = kc.size(3) * 2;
  CHECK_VALUE(q0.dim() == 4 && q0.size(0) == kc.size(0) && q0.size(3) == d, "expected q [", kc.size(0), ", heads, 1, ", d,
                    "]; got ", q0.sizes());
  CHECK_VALUE(q0.size(1) > 0 && kc.size(1) > 0 && q0.size(1) % kc.size(1) == 0,
                    "query heads must be a multiple of key/value heads; got ", q0.size(1), " and ", kc.size(1));
  CHECK_VALUE(q0.scalar_type() == at::kHalf, "q must be float16, got ", q0.scalar_type());
  CHECK_VALUE(q0.device() == kc.device(), "q and the cache must be on one device, got ", q0.device(), ", ", kc.device());
  check_token({&q0}, lengths0, window, sinks);
  refuse_forward_mode("Int4Cache.attend", {&q0});
  require_cuda(q0);
  const Tensor q = rows16(q0), lengths = lengths0.contiguous();
  Tensor o = like(q);
  if (o.numel() == 0) return o;
  const int z = dim(q, 0), h = dim(q, 1), hk = dim(kc, 1), cap = dim(kc, 2);
  const int w = clamp_int(window.value_or(0)), s = clamp_int(sinks);
  Strides st;
  st.add(q);
  st.add(o);
  const c10::cuda::CUDAGuard guard(q.device());
  const int64_t size = tattn_int4_decode_workspace_bytes(z, h, hk, cap, int(d), w, s);
  const Tensor ws = size > 0 ? bytes(size, q) : Tensor();
  check_status("tattn_int4_decode",
               tattn_int4_decode(q.data_ptr(), kc.data_ptr(), kp.data_ptr(), vc.data_ptr(), vp.data_ptr(), lengths.data_ptr<int>(),
                                 o.data_ptr(), size > 0 ? ws.data_ptr() : nullptr, st.s, z, h, hk, cap, int(d), w, s,
                                 float(scale_of(sm_scale, q)), stream_of(q)));
  return o;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("abi_version", &tattn_abi_version);
  m.def("qk_norm_rope", &qk_norm_rope);
  m.def("window_attention", &window_attention);
  m.def("window_forward", &window_forward);
  m.def("window_backward", &window_backward);
  m.def("decode_attention", &decode_attention);
  m.def("int4_check", &int4_check);
  m.def("int4_append", &int4_append);
  m.def("int4_read", &int4_read);
  m.def("int4_attend", &int4_attend);
}
