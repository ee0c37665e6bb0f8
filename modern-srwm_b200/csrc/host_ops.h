// Selective scan, causal convolution, root-mean-square norm and clipping by the gradients' norm, with autograd.
#pragma once
#include <algorithm>
#include <unordered_set>
#include <vector>

#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/variable.h>

#include "host_common.h"

namespace host {

// [N, L, X] rows that the kernels read as they are: innermost dense, any other strides.
inline bool rows_ok(const Tensor& t) { return t.size(2) == 1 || t.stride(2) == 1; }
inline srwm_b200_rows rows(const Tensor& t) {
  if (!t.defined()) return {nullptr, 0, 0};
  return {const_cast<void*>(t.const_data_ptr()), t.stride(0), t.stride(1)};
}
// [N, L, S] or [N, L, G, S]
inline bool bc_ok(const Tensor& t) { return t.size(t.dim() - 1) == 1 || t.stride(t.dim() - 1) == 1; }
inline srwm_b200_seq bc_rows(const Tensor& t) {
  return {const_cast<void*>(t.const_data_ptr()), t.stride(0), t.dim() == 4 ? t.stride(2) : 0, t.stride(1)};
}
// Uninitialised, in the memory order of the input view
inline Tensor rows_like(const Tensor& t) {
  if (t.is_non_overlapping_and_dense()) return at::empty_like(t);
  auto sizes = t.sizes().vec();
  if (t.stride(0) >= t.stride(1)) return at::empty(sizes, t.options());
  std::swap(sizes[0], sizes[1]);
  return at::empty(sizes, t.options()).transpose(0, 1);
}
inline bool dense_f32(const Tensor& t, at::IntArrayRef shape) {
  return t.is_cuda() && t.scalar_type() == at::kFloat && t.sizes() == shape && t.is_contiguous() &&
         reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
}
inline const float* floats_of(const Tensor& t) { return t.defined() ? static_cast<const float*>(t.const_data_ptr()) : nullptr; }
inline float* floats_in(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }
inline Tensor opt(const std::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }
inline std::optional<Tensor> opt(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
inline Tensor saved_any(const Tensor& t) { return !t.defined() || (t.dim() ? t.stride(t.dim() - 1) == 1 : true) ? t : dense(t); }
// Gradient of an output as rows; zeros where it takes no part
inline Tensor grad_or_zeros(const Tensor& g, const Tensor& like) {
  if (!g.defined()) return at::zeros_like(like);
  const Tensor r = g.scalar_type() == like.scalar_type() ? g : g.to(like.scalar_type());
  return rows_ok(r) ? r : r.contiguous();
}
inline bool done_ok(const Tensor& done, const Tensor& x) {
  return !done.defined() || (done.device() == x.device() && (done.scalar_type() == at::kBool || done.scalar_type() == at::kByte) &&
                             done.dim() == 2 && done.size(0) == x.size(0) && done.size(1) == x.size(1));
}
inline bool io_rows(const Tensor& t) { return t.is_cuda() && t.dim() == 3 && io_ok(t) && t.numel() > 0 && rows_ok(t); }
inline bool fits_int(const Tensor& t) {
  for (const int64_t n : t.sizes())
    if (n > 0x7fffffff) return false;
  return true;
}

// Rows that can be written in place: no two of [N, L] share a value
inline bool rows_apart(const Tensor& t) {
  const int a = t.stride(0) >= t.stride(1) ? 0 : 1, b = 1 - a;      // the rows further apart, and the others
  return (t.size(b) == 1 || t.stride(b) >= t.size(2)) && (t.size(a) == 1 || t.stride(a) >= (t.size(b) == 1 ? 0 : t.stride(b) * (t.size(b) - 1)) + t.size(2));
}
// ---- selective scan ----

struct ScanIn {
  Tensor u, delta, A, B, C, D, z, bias, state, done;
  bool softplus;
};
inline bool scan_ok(const ScanIn& s) {
  const Tensor& u = s.u;
  if (!io_rows(u) || !fits_int(u)) return false;
  const int64_t N = u.size(0), L = u.size(1), D = u.size(2);
  for (const Tensor* t : {&s.delta, &s.z})
    if (t->defined() && (t->device() != u.device() || t->scalar_type() != u.scalar_type() || t->sizes() != u.sizes() || !rows_ok(*t)))
      return false;
  if (!s.delta.defined() || s.A.dim() != 2 || !head_dim_ok(s.A.size(1))) return false;
  const int64_t S = s.A.size(1);
  if (!dense_f32(s.A, {D, S}) || s.A.device() != u.device()) return false;
  for (const Tensor* t : {&s.B, &s.C}) {
    if (t->device() != u.device() || t->scalar_type() != u.scalar_type() || (t->dim() != 3 && t->dim() != 4)) return false;
    if (t->sizes() != s.B.sizes() || t->size(0) != N || t->size(1) != L || t->size(-1) != S || !bc_ok(*t)) return false;
    if (t->dim() == 4 && (t->size(2) == 0 || D % t->size(2))) return false;
  }
  for (const Tensor* t : {&s.D, &s.bias})
    if (t->defined() && (t->device() != u.device() || t->scalar_type() != at::kFloat || t->dim() != 1 || t->size(0) != D || !t->is_contiguous()))
      return false;
  if (s.state.defined() && (!dense_f32(s.state, {N, D, S}) || s.state.device() != u.device())) return false;
  return done_ok(s.done, u);
}
inline void scan_args(const ScanIn& s, srwm_b200_scan_args& a) {
  a.N = s.u.size(0); a.L = s.u.size(1); a.D = s.u.size(2); a.S = s.A.size(1);
  a.G = s.B.dim() == 4 ? s.B.size(2) : 1;
  a.io_dtype = io_code(s.u);
  a.softplus = s.softplus;
  a.u = rows(s.u); a.delta = rows(s.delta); a.z = rows(s.z);
  a.B = bc_rows(s.B); a.C = bc_rows(s.C);
  a.A = floats_of(s.A); a.skip = floats_of(s.D); a.delta_bias = floats_of(s.bias); a.state_in = floats_of(s.state);
  if (s.done.defined()) {
    a.done = static_cast<const uint8_t*>(s.done.const_data_ptr());
    a.done_stride_n = s.done.stride(0);
    a.done_stride_l = s.done.stride(1);
  }
}
inline variable_list scan_forward(const ScanIn& s, bool inplace, Tensor* checkpoints) {
  c10::cuda::CUDAGuard guard(s.u.device());
  srwm_b200_scan_args a = {};
  scan_args(s, a);
  Tensor y = rows_like(s.u), state = inplace ? s.state : floats(s.u, {a.N, a.D, a.S}), scratch;
  a.y = rows(y);
  a.state_out = floats_in(state);
  if (checkpoints) {
    *checkpoints = floats(s.u, {api().srwm_b200_scan_checkpoint_floats(a.N, a.L, a.D, a.S)});
    a.checkpoints = floats_in(*checkpoints);
  }
  if (const int64_t need = api().srwm_b200_scan_scratch_bytes(a.N, a.L, a.D, a.S, a.G)) {
    scratch = floats(s.u, {need / 4});
    a.scratch = scratch.data_ptr();
    a.scratch_bytes = need;
  }
  if (inplace) state.unsafeGetTensorImpl()->bump_version();
  check(api().srwm_b200_scan_forward(&a, stream_of(s.u)), "scan_forward");
  return {y, state};
}

struct Scan : torch::autograd::Function<Scan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C,
                               const std::optional<Tensor>& D, const std::optional<Tensor>& z, const std::optional<Tensor>& bias,
                               const std::optional<Tensor>& state, const std::optional<Tensor>& done, bool softplus) {
    const ScanIn s = {u, delta, A, B, C, opt(D), opt(z), opt(bias), opt(state), opt(done), softplus};
    Tensor ckpt;
    variable_list r = scan_forward(s, false, &ckpt);
    ctx->save_for_backward({u, delta, A, B, C, s.D, s.z, s.bias, s.done, ckpt});
    ctx->saved_data["softplus"] = softplus;
    ctx->saved_data["state"] = state.has_value();
    ctx->set_materialize_grads(false);
    return r;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto t = ctx->get_saved_variables();
    c10::cuda::CUDAGuard guard(t[0].device());
    const ScanIn s = {saved_any(t[0]), saved_any(t[1]), dense(t[2]), saved_any(t[3]), saved_any(t[4]),
                      t[5].defined() ? dense(t[5]) : t[5], saved_any(t[6]), t[7].defined() ? dense(t[7]) : t[7], Tensor(), t[8],
                      ctx->saved_data["softplus"].toBool()};
    const Tensor ckpt = dense(t[9]);
    srwm_b200_scan_args a = {};
    scan_args(s, a);
    const Tensor dy = grad_or_zeros(g[0], s.u);
    const Tensor dstate = g[1].defined() ? dense(g[1].to(at::kFloat)) : Tensor();
    Tensor du = rows_like(s.u), dd = rows_like(s.delta), dz, dB = rows_like(s.B), dC = rows_like(s.C), dA = at::empty_like(s.A), dD, db, dh0;
    if (s.z.defined()) dz = rows_like(s.z);
    if (s.D.defined()) dD = at::empty_like(s.D);
    if (s.bias.defined()) db = at::empty_like(s.bias);
    // (edges are counted without the arguments that were not given)
    const size_t state_edge = 5 + s.D.defined() + s.z.defined() + s.bias.defined();
    if (ctx->saved_data["state"].toBool() && ctx->needs_input_grad(state_edge)) dh0 = floats(s.u, {a.N, a.D, a.S});
    a.checkpoints = floats_in(ckpt);
    const int64_t need = api().srwm_b200_scan_backward_scratch_bytes(a.N, a.L, a.D, a.S, a.G);
    Tensor scratch = floats(s.u, {need / 4});
    a.scratch = scratch.data_ptr();
    a.scratch_bytes = need;
    srwm_b200_scan_grads o = {};
    o.dy = rows(dy); o.dstate_out = floats_of(dstate);
    o.du = rows(du); o.ddelta = rows(dd); o.dz = rows(dz);
    o.dB = bc_rows(dB); o.dC = bc_rows(dC);
    o.dA = floats_in(dA); o.dskip = floats_in(dD); o.ddelta_bias = floats_in(db); o.dstate_in = floats_in(dh0);
    check(api().srwm_b200_scan_backward(&a, &o, stream_of(s.u)), "scan_backward");
    return {du, dd, dA, dB, dC, dD, dz, db, dh0, Tensor(), Tensor()};
  }
};

// ---- causal convolution ----

struct ConvIn {
  Tensor x, w, bias, state, done;
  bool silu;
};
inline bool conv_ok(const ConvIn& s) {
  const Tensor& x = s.x;
  if (!io_rows(x) || !fits_int(x)) return false;
  const int64_t N = x.size(0), D = x.size(2);
  if (s.w.device() != x.device() || s.w.scalar_type() != at::kFloat || s.w.dim() != 2 || s.w.size(0) != D || !s.w.is_contiguous()) return false;
  const int64_t K = s.w.size(1);
  if (K < 2 || K > 4) return false;
  if (s.bias.defined() && (s.bias.device() != x.device() || s.bias.scalar_type() != at::kFloat || s.bias.dim() != 1 || s.bias.size(0) != D ||
                           !s.bias.is_contiguous()))
    return false;
  if (s.state.defined() && (s.state.device() != x.device() || s.state.scalar_type() != x.scalar_type() || s.state.dim() != 3 ||
                            s.state.size(0) != N || s.state.size(1) != K - 1 || s.state.size(2) != D || !rows_ok(s.state)))
    return false;
  return done_ok(s.done, x);
}
inline void conv_args(const ConvIn& s, srwm_b200_conv_args& a) {
  a.N = s.x.size(0); a.L = s.x.size(1); a.D = s.x.size(2); a.K = s.w.size(1);
  a.io_dtype = io_code(s.x);
  a.silu = s.silu;
  a.x = rows(s.x); a.w = floats_of(s.w); a.bias = floats_of(s.bias); a.state_in = rows(s.state);
  if (s.done.defined()) {
    a.done = static_cast<const uint8_t*>(s.done.const_data_ptr());
    a.done_stride_n = s.done.stride(0);
    a.done_stride_l = s.done.stride(1);
  }
}
inline variable_list conv_forward(const ConvIn& s, bool inplace) {
  c10::cuda::CUDAGuard guard(s.x.device());
  srwm_b200_conv_args a = {};
  conv_args(s, a);
  Tensor y = rows_like(s.x);
  const bool direct = inplace && a.L <= 16;      // (longer calls write the state while it is still read)
  Tensor state = direct ? s.state : at::empty({a.N, a.K - 1, a.D}, s.x.options());
  a.y = rows(y);
  a.state_out = rows(state);
  if (inplace) s.state.unsafeGetTensorImpl()->bump_version();
  check(api().srwm_b200_conv_forward(&a, stream_of(s.x)), "conv_forward");
  if (inplace && !direct) {
    s.state.detach().copy_(state);
    state = s.state;
  }
  return {y, state};
}

struct Conv : torch::autograd::Function<Conv> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const std::optional<Tensor>& bias,
                               const std::optional<Tensor>& state, const std::optional<Tensor>& done, bool silu) {
    const ConvIn s = {x, w, opt(bias), opt(state), opt(done), silu};
    variable_list r = conv_forward(s, false);
    ctx->save_for_backward({x, w, s.bias, s.state, s.done});
    ctx->saved_data["silu"] = silu;
    ctx->set_materialize_grads(false);
    return r;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto t = ctx->get_saved_variables();
    c10::cuda::CUDAGuard guard(t[0].device());
    const ConvIn s = {saved_any(t[0]), t[1].contiguous(), t[2].defined() ? t[2].contiguous() : t[2], saved_any(t[3]), t[4],
                      ctx->saved_data["silu"].toBool()};
    srwm_b200_conv_args a = {};
    conv_args(s, a);
    const Tensor dy = grad_or_zeros(g[0], s.x);
    Tensor dsT;
    if (g[1].defined()) {
      dsT = g[1].to(s.x.scalar_type());
      if (!rows_ok(dsT)) dsT = dsT.contiguous();
    }
    Tensor dx = rows_like(s.x), dw = at::empty_like(s.w), db, ds0;
    if (s.bias.defined()) db = at::empty_like(s.bias);
    if (s.state.defined() && ctx->needs_input_grad(2 + s.bias.defined())) ds0 = at::empty({a.N, a.K - 1, a.D}, s.x.options());
    const int64_t need = api().srwm_b200_conv_scratch_bytes(a.N, a.L, a.D, a.K);
    Tensor scratch = floats(s.x, {need / 4});
    srwm_b200_conv_grads o = {};
    o.dy = rows(dy); o.dstate_out = rows(dsT); o.dx = rows(dx); o.dstate_in = rows(ds0);
    o.dw = floats_in(dw); o.dbias = floats_in(db);
    o.scratch = scratch.data_ptr();
    o.scratch_bytes = need;
    check(api().srwm_b200_conv_backward(&a, &o, stream_of(s.x)), "conv_backward");
    return {dx, dw, db, ds0, Tensor(), Tensor()};
  }
};

// ---- root-mean-square norm ----

// Rows of D values at one distance from each other (leading dimensions that fold into one)
inline bool row_stride(const Tensor& t, int64_t* stride) {
  const int64_t n = t.dim();
  if (t.size(n - 1) > 1 && t.stride(n - 1) != 1) return false;
  *stride = t.size(n - 1);
  int64_t next = -1;      // distance of the rows of the dimensions seen, as a whole
  for (int64_t d = n - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (next < 0) *stride = t.stride(d);
    else if (t.stride(d) != next) return false;
    next = t.stride(d) * t.size(d);
  }
  return true;
}
inline bool rms_ok(const Tensor& x, const Tensor& w, const Tensor& res) {
  int64_t s;
  if (!x.is_cuda() || !io_ok(x) || x.dim() < 1 || x.numel() == 0 || !row_stride(x, &s)) return false;
  const int64_t D = x.size(-1);
  if (D > 8192 || w.device() != x.device() || w.scalar_type() != at::kFloat || w.dim() != 1 || w.size(0) != D || !w.is_contiguous()) return false;
  return !res.defined() || (res.device() == x.device() && res.scalar_type() == x.scalar_type() && res.sizes() == x.sizes() && row_stride(res, &s));
}
// y, (the sum), (the scales)
inline variable_list rms_forward(const Tensor& x, const Tensor& w, const Tensor& res, double eps, bool fp8, Tensor* rstd) {
  c10::cuda::CUDAGuard guard(x.device());
  srwm_b200_rms_args a = {};
  a.D = x.size(-1);
  a.rows = x.numel() / a.D;
  a.io_dtype = io_code(x);
  a.eps = (float)eps;
  a.x = x.const_data_ptr();
  row_stride(x, &a.x_stride);
  a.w = floats_of(w);
  variable_list r;
  r.push_back(at::empty(x.sizes(), fp8 ? x.options().dtype(at::kFloat8_e4m3fn) : x.options()));
  a.y = r[0].data_ptr();
  if (fp8) {
    auto shape = x.sizes().vec();
    shape.back() = 1;
    r.push_back(floats(x, shape));
    a.scale = floats_in(r.back());
  }
  if (res.defined()) {
    a.residual = res.const_data_ptr();
    row_stride(res, &a.residual_stride);
    r.push_back(at::empty(x.sizes(), x.options()));
    a.sum = r.back().data_ptr();
  }
  if (rstd) {
    *rstd = floats(x, {a.rows});
    a.rstd = floats_in(*rstd);
  }
  check(api().srwm_b200_rms_forward(&a, stream_of(x)), "rms_forward");
  return r;
}
struct Rms : torch::autograd::Function<Rms> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const std::optional<Tensor>& res, double eps) {
    Tensor rstd;
    variable_list r = rms_forward(x, w, opt(res), eps, false, &rstd);
    ctx->save_for_backward({res.has_value() ? r[1] : x, w, rstd});
    ctx->saved_data["res"] = res.has_value();
    ctx->set_materialize_grads(false);
    return r;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto t = ctx->get_saved_variables();
    c10::cuda::CUDAGuard guard(t[0].device());
    const bool has_res = ctx->saved_data["res"].toBool();
    srwm_b200_rms_grads a = {};
    auto as_rows = [&](const Tensor& v, int64_t* stride) {
      Tensor r = v.scalar_type() == t[0].scalar_type() ? v : v.to(t[0].scalar_type());
      if (!row_stride(r, stride)) {
        r = r.contiguous();
        row_stride(r, stride);
      }
      return r;
    };
    const Tensor sum = as_rows(t[0], &a.sum_stride), w = t[1].contiguous(), rstd = t[2].contiguous();
    const Tensor dy = as_rows(g[0].defined() ? g[0] : at::zeros_like(sum), &a.dy_stride);
    Tensor dsum;
    if (has_res && g[1].defined()) dsum = as_rows(g[1], &a.dsum_stride);
    a.D = sum.size(-1);
    a.rows = sum.numel() / a.D;
    a.io_dtype = io_code(sum);
    Tensor dx = at::empty(sum.sizes(), sum.options()), dw = at::empty_like(w);
    const int64_t need = api().srwm_b200_rms_scratch_bytes(a.rows, a.D);
    Tensor scratch = floats(sum, {need / 4});
    a.sum = sum.const_data_ptr(); a.dy = dy.const_data_ptr();
    a.dsum = dsum.defined() ? dsum.const_data_ptr() : nullptr;
    a.w = floats_of(w); a.rstd = floats_of(rstd);
    a.dx = dx.data_ptr(); a.dw = floats_in(dw);
    a.scratch = scratch.data_ptr();
    a.scratch_bytes = need;
    check(api().srwm_b200_rms_backward(&a, stream_of(sum)), "rms_backward");
    return {dx, dw, has_res ? dx : Tensor(), Tensor()};
  }
};

// ---- captures ----

// A leaf's gradient is gathered on the stream on which a graph first used the leaf.  Where that graph still lives and the stream is
// the default one, a backward pass under capture would draw the default stream into the capture, which ends the process; said
// here instead, while the forward pass is captured.  The leaves are those of the call and those that this capture has made its
// arguments of (casts, projections), up to operators of this file, which have asked already.
inline void check_capture(std::initializer_list<const Tensor*> ts) {
  using torch::autograd::Node;
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  auto refuse = [](Node& gathers) {
    const auto stream = gathers.stream();
    TORCH_CHECK(!stream || *stream != c10::cuda::getDefaultCUDAStream(stream->device_index()).unwrap(),
                "a leaf of this call belongs to an autograd graph that was built on the default stream and is still alive: drop its "
                "outputs (a loss, a carried state) before a training step is captured");
  };
  std::vector<Node*> open;
  std::unordered_set<Node*> seen;
  auto reach = [&](Node* n) {
    if (n && seen.insert(n).second) open.push_back(n);
  };
  for (const Tensor* t : ts) {
    if (!t->defined() || !t->requires_grad()) continue;
    if (!t->is_leaf()) reach(t->grad_fn().get());
    else if (const auto sum = torch::autograd::impl::try_get_grad_accumulator(*t)) refuse(*sum);
  }
  while (!open.empty()) {
    Node* n = open.back();
    open.pop_back();
    if (dynamic_cast<torch::autograd::CppNode<Scan>*>(n) || dynamic_cast<torch::autograd::CppNode<Conv>*>(n) ||
        dynamic_cast<torch::autograd::CppNode<Rms>*>(n))
      continue;
    const auto stream = n->stream();
    if (dynamic_cast<torch::autograd::AccumulateGrad*>(n)) refuse(*n);
    else if (!stream || *stream == c10::cuda::getCurrentCUDAStream(stream->device_index()).unwrap())
      for (const auto& e : n->next_edges()) reach(e.function.get());      // (what was there before the capture is not its business)
  }
}

// ---- norm over many tensors, clipping ----

// Values of one device that lie dense (in any order) and, where they are to be written, apart from each other
inline bool grads_ok(const std::vector<Tensor>& ts, bool written) {
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;
  if (written) spans.reserve(ts.size());
  for (const Tensor& t : ts) {
    if (!t.is_cuda() || t.device() != ts[0].device() || !io_ok(t) || t.layout() != at::kStrided || !t.is_non_overlapping_and_dense()) return false;
    const uintptr_t p = reinterpret_cast<uintptr_t>(t.const_data_ptr());
    if (written && t.numel() > 0) spans.emplace_back(p, p + t.numel() * t.element_size());
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].first < spans[i - 1].second) return false;
  return true;
}
// max_norm < 0: the norm alone
inline Tensor grads_norm(const std::vector<Tensor>& ts, double max_norm) {
  c10::cuda::CUDAGuard guard(ts[0].device());
  std::vector<srwm_b200_tensor> list;
  list.reserve(ts.size());
  for (const Tensor& t : ts) {
    if (max_norm >= 0) t.unsafeGetTensorImpl()->bump_version();
    list.push_back({const_cast<void*>(t.const_data_ptr()), t.numel(), io_code(t), 0});
  }
  const int64_t need = api().srwm_b200_grads_scratch_bytes(list.data(), (int32_t)list.size());
  Tensor norm = floats(ts[0], {}), scratch = floats(ts[0], {need / 4});
  if (max_norm < 0)
    check(api().srwm_b200_grads_norm(list.data(), (int32_t)list.size(), floats_in(norm), scratch.data_ptr(), need, stream_of(ts[0])), "grads_norm");
  else
    check(api().srwm_b200_grads_clip(list.data(), (int32_t)list.size(), (float)max_norm, floats_in(norm), scratch.data_ptr(), need,
                                     stream_of(ts[0])),
          "grads_clip");
  return norm;
}

}  // namespace host
