// Module `attention_cuda`: cross entropy of a linear layer without kept logits, twice differentiable.
#include "ext_common.h"

#include <ATen/Context.h>

#include <limits>

namespace ext {

namespace {

struct LossArgs { int64_t ignore_index, reduction; };

attn_lce_shape_t loss_shape(const torch::Tensor& x, const torch::Tensor& w, const LossArgs& a) {
  attn_lce_shape_t s{};
  s.n = (int32_t)x.size(0);
  s.d = (int32_t)x.size(1);
  s.V = (int32_t)w.size(0);
  s.dtype = dtype_code(x);
  s.reduction = (int32_t)a.reduction;
  s.ignore_index = a.ignore_index;
  return s;
}

void check_loss(const torch::Tensor& x, const torch::Tensor& w, const torch::Tensor& targets) {
  TORCH_CHECK(x.is_cuda() && w.is_cuda() && targets.is_cuda(), "x, weight and targets must be CUDA tensors");
  TORCH_CHECK(x.device() == w.device() && x.device() == targets.device(), "x, weight and targets must be on one device");
  TORCH_CHECK(x.dim() == 2 && w.dim() == 2 && x.size(1) == w.size(1), "x must be [..., d] and weight [V, d]");
  TORCH_CHECK(x.scalar_type() == w.scalar_type(), "x and weight must have the same dtype");
  TORCH_CHECK(targets.dim() == 1 && targets.size(0) == x.size(0), "targets must have the shape of x without its last axis");
  TORCH_CHECK(targets.scalar_type() == at::kLong, "targets must be int64");
  TORCH_CHECK(x.size(0) <= (1 << 30) && w.size(0) <= (1 << 30) && x.size(1) <= (1 << 20), "x or weight is too large");
  TORCH_CHECK(w.size(0) > 0 && w.size(1) > 0, "weight must not be empty");
}

// {output, lse, counted}
variable_list loss_forward(const torch::Tensor& x_in, const torch::Tensor& w_in, const torch::Tensor& targets_in, const LossArgs& a) {
  check_loss(x_in, w_in, targets_in);
  c10::cuda::CUDAGuard guard(x_in.device());
  raise_if_earlier_call_timed_out(x_in.device().index());
  const torch::Tensor x = dense(x_in), w = dense(w_in), targets = targets_in.contiguous();
  const attn_lce_shape_t s = loss_shape(x, w, a);
  auto losses = fresh({x.size(0)}, at::kFloat, x);
  auto lse = fresh({x.size(0)}, at::kFloat, x);
  auto value = a.reduction == ATTN_REDUCE_NONE ? losses : fresh(at::IntArrayRef{}, at::kFloat, x);
  auto counted = fresh(at::IntArrayRef{}, at::kFloat, x);
  auto scratch = fresh({(int64_t)attn_b200_linear_ce_forward_scratch_bytes(&s)}, at::kByte, x);
  check_rc(attn_b200_linear_ce_forward(&s, x.data_ptr(), w.data_ptr(), targets.data_ptr<int64_t>(), losses.data_ptr<float>(), lse.data_ptr<float>(),
                                       value.data_ptr<float>(), counted.data_ptr<float>(), scratch.data_ptr(), at::cuda::getCurrentCUDAStream().stream()),
           "linear_cross_entropy");
  return {value, lse, counted};
}

// {dx, dw}, undefined where not wanted
variable_list loss_backward(const torch::Tensor& g_in, const torch::Tensor& x_in, const torch::Tensor& w_in, const torch::Tensor& targets_in,
                            const torch::Tensor& lse, const torch::Tensor& counted_rows, const LossArgs& a, bool want_dx, bool want_dw) {
  variable_list r(2);
  if (!want_dx && !want_dw) return r;
  c10::cuda::CUDAGuard guard(x_in.device());
  raise_if_earlier_call_timed_out(x_in.device().index());
  const torch::Tensor x = dense(x_in), w = dense(w_in), targets = targets_in.contiguous(), g = g_in.to(at::kFloat).contiguous();
  const attn_lce_shape_t s = loss_shape(x, w, a);
  if (want_dx) r[0] = fresh_like(x);
  if (want_dw) r[1] = fresh_like(w);
  auto scratch = fresh({(int64_t)attn_b200_linear_ce_backward_scratch_bytes(&s, want_dx, want_dw)}, at::kByte, x);
  check_rc(attn_b200_linear_ce_backward(&s, x.data_ptr(), w.data_ptr(), targets.data_ptr<int64_t>(), lse.data_ptr<float>(), g.data_ptr<float>(),
                                        counted_rows.data_ptr<float>(), want_dx ? r[0].data_ptr() : nullptr, want_dw ? r[1].data_ptr() : nullptr,
                                        scratch.data_ptr(), at::cuda::getCurrentCUDAStream().stream()),
           "linear_cross_entropy backward");
  return r;
}

// Second backward, out of ordinary operations over pieces of the rows: with tangents u on dx and v on dw, T = u W^T + x v^T,
// P = exp(z - lse), c the rows' factors, r_i = sum_j P_ij T_ij:
//   to c_i: r_i - T_i,y      H = c P (T - r), G = c (P - onehot)      to x: H W + G v      to W: H^T x + G^T u
// Products of half types are summed and kept in float; H and G are rounded to the input type, in bf16 relative to the largest factor (one that
// all rows share would be rounded in the same direction everywhere), in fp16 to their own largest elements (its range).
variable_list loss_double_backward(const torch::Tensor& u_in, const torch::Tensor& v_in, const torch::Tensor& g, const torch::Tensor& x,
                                   const torch::Tensor& w, const torch::Tensor& targets, const torch::Tensor& lse, const torch::Tensor& counted_rows,
                                   const LossArgs& a) {
  at::AutoGradMode off(false);
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t n = x.size(0), V = w.size(0);
  // a target that is no class: taken out of the sums, and not a number in the end
  const torch::Tensor classes = targets.clamp(0, V - 1), named = targets != a.ignore_index, wrong = named & (classes != targets), counted = named ^ wrong;
  torch::Tensor c = g.to(at::kFloat);
  if (a.reduction == ATTN_REDUCE_MEAN) c = c / counted_rows;
  c = torch::where(counted, c.expand({n}), torch::zeros({}, c.options()));
  torch::Tensor gx = torch::zeros_like(x), gw = torch::zeros(w.sizes(), w.options().dtype(at::kFloat)), gc = torch::zeros({n}, c.options());
  const bool half = x.scalar_type() != at::kFloat;
  // Whatever the process allows its own products: TF32 operands would leave P = exp(z - lse), of logits in full float, without a sum of 1, and half
  // products that may be summed in fp16 have no float result.  The guard speaks for cuBLAS alone; where cuBLASLt is preferred, float goes through double.
  // Autocast would round the operands of float products.
  const c10::impl::ExcludeDispatchKeyGuard as_they_are(c10::autocast_dispatch_keyset);
  const at::NoTF32Guard full_float;
  auto& context = at::globalContext();
  const at::ScalarType wide = !half ? at::kDouble : at::kFloat;
  const bool widen = half ? x.scalar_type() == at::kHalf && context.allowFP16AccumulationCuBLAS() : context.blasPreferredBackend() != at::BlasBackend::Cublas;
  auto mm = [&](const torch::Tensor& p, const torch::Tensor& q) {
    if (widen) return at::mm(p.to(wide), q.to(wide)).to(at::kFloat);
    return half ? at::mm(p, q, at::kFloat) : at::mm(p, q);
  };
  auto unit = [&](const torch::Tensor& t, float largest) {
    const torch::Tensor top = t.numel() > 0 ? t.abs().amax() : torch::zeros({}, t.options());
    return torch::where((top > 0) & (top < std::numeric_limits<float>::infinity()), largest / top, torch::ones({}, top.options()));
  };
  const torch::Tensor common = x.scalar_type() == at::kBFloat16 ? unit(c, 1.f) : torch::ones({}, c.options());
  const int64_t step = std::max<int64_t>(1, std::min<int64_t>(n, (int64_t(1) << 28) / V));
  for (int64_t i = 0; i < n; i += step) {
    const int64_t e = std::min(n, i + step);
    const torch::Tensor mask = counted.slice(0, i, e).unsqueeze(1), zero = torch::zeros({}, c.options());
    auto rows = [&](const torch::Tensor& t) { return torch::where(mask, t.slice(0, i, e), torch::zeros({}, t.options())); };
    const torch::Tensor xs = rows(x), us = u_in.defined() ? rows(u_in) : torch::Tensor(), cs = c.slice(0, i, e).unsqueeze(1);
    const torch::Tensor y = classes.slice(0, i, e).unsqueeze(1);
    torch::Tensor P = torch::exp(mm(xs, w.t()) - lse.slice(0, i, e).unsqueeze(1));
    torch::Tensor T = us.defined() ? mm(us, w.t()) : torch::zeros_like(P);
    if (v_in.defined()) T.add_(mm(xs, v_in.t()));
    const torch::Tensor r = (P * T).sum(1, true);
    gc.slice(0, i, e).copy_(torch::where(mask, r - T.gather(1, y), zero).squeeze(1));
    torch::Tensor H = T.sub_(r).mul_(P).mul_(cs);
    torch::Tensor G = P.scatter_add_(1, y, torch::full({}, -1.f, P.options()).expand_as(y)).mul_(cs);
    H = torch::where(mask, H, zero);
    G = torch::where(mask, G, zero);
    const bool fp16 = x.scalar_type() == at::kHalf;
    const torch::Tensor sh = fp16 ? unit(H, 32768.f) : common, sg = fp16 ? unit(G, 32768.f) : common;
    const torch::Tensor Ht = (H * sh).to(x.scalar_type()), Gt = (G * sg).to(x.scalar_type());
    torch::Tensor to_x = mm(Ht, w) / sh;
    if (v_in.defined()) to_x.add_(mm(Gt, v_in) / sg);
    gx.slice(0, i, e).copy_(to_x);
    gw.add_(mm(Ht.t(), xs) / sh);
    if (us.defined()) gw.add_(mm(Gt.t(), us) / sg);
  }
  // as in the first backward: the row's, and all that is summed over it
  const double nan = std::numeric_limits<double>::quiet_NaN();
  gx.masked_fill_(wrong.unsqueeze(1), nan);
  gw.masked_fill_(wrong.any(), nan);
  gc.masked_fill_(wrong, nan);
  torch::Tensor gg;
  if (a.reduction == ATTN_REDUCE_NONE) gg = gc;
  else if (a.reduction == ATTN_REDUCE_SUM) gg = gc.sum();
  else gg = gc.sum() / counted_rows;
  return {gg.to(g.scalar_type()), gx, gw.to(w.scalar_type())};
}

void save_args(AutogradContext* ctx, int64_t ignore_index, int64_t reduction) {
  ctx->set_materialize_grads(false);
  ctx->saved_data["ignore_index"] = ignore_index;
  ctx->saved_data["reduction"] = reduction;
}
LossArgs saved_args(AutogradContext* ctx) { return {ctx->saved_data["ignore_index"].toInt(), ctx->saved_data["reduction"].toInt()}; }

struct LinearCrossEntropyBackward : public torch::autograd::Function<LinearCrossEntropyBackward> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& g, const torch::Tensor& x, const torch::Tensor& w,
                               const torch::Tensor& targets, const torch::Tensor& lse, const torch::Tensor& counted_rows, int64_t ignore_index,
                               int64_t reduction) {
    save_args(ctx, ignore_index, reduction);
    ctx->save_for_backward({g, x, w, targets, lse, counted_rows});
    return loss_backward(g, x, w, targets, lse, counted_rows, {ignore_index, reduction}, true, true);
  }

  static variable_list backward(AutogradContext* ctx, variable_list t) {
    variable_list out(8);      // g, x, w, targets, lse, counted_rows, ignore_index, reduction
    if (!t[0].defined() && !t[1].defined()) return out;
    TORCH_CHECK(!at::GradMode::is_enabled(), "linear_cross_entropy has no third derivative: call the second backward without create_graph");
    const variable_list s = ctx->get_saved_variables();
    variable_list r = loss_double_backward(t[0], t[1], s[0], s[1], s[2], s[3], s[4], s[5], saved_args(ctx));
    for (int i = 0; i < 3; ++i) out[i] = std::move(r[i]);
    return out;
  }
};

struct LinearCrossEntropy : public torch::autograd::Function<LinearCrossEntropy> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& w, const torch::Tensor& targets,
                               int64_t ignore_index, int64_t reduction) {
    variable_list r = loss_forward(x, w, targets, {ignore_index, reduction});
    save_args(ctx, ignore_index, reduction);
    ctx->save_for_backward({x, w, targets, r[1], r[2]});
    return r[0];
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(5);      // x, w, targets, ignore_index, reduction
    if (!g[0].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    const LossArgs a = saved_args(ctx);
    TORCH_CHECK(!has_tangent({&g[0], &s[0], &s[1]}), "linear_cross_entropy has no forward-mode derivative");
    variable_list r = at::GradMode::is_enabled()
                          ? LinearCrossEntropyBackward::apply(g[0], s[0], s[1], s[2], s[3], s[4], a.ignore_index, a.reduction)
                          : loss_backward(g[0], s[0], s[1], s[2], s[3], s[4], a, ctx->needs_input_grad(0), ctx->needs_input_grad(1));
    for (int i = 0; i < 2; ++i) out[i] = std::move(r[i]);
    return out;
  }
};

torch::Tensor linear_cross_entropy(const torch::Tensor& x, const torch::Tensor& weight, const torch::Tensor& targets, int64_t ignore_index,
                                   int64_t reduction) {
  refuse_transforms({&x, &weight}, "linear_cross_entropy");
  TORCH_CHECK(reduction >= ATTN_REDUCE_NONE && reduction <= ATTN_REDUCE_MEAN, "reduction unknown");
  if (!wants_graph({&x, &weight})) return loss_forward(x, weight, targets, {ignore_index, reduction})[0];
  return LinearCrossEntropy::apply(x, weight, targets, ignore_index, reduction);
}

}  // namespace

void register_loss(pybind11::module& m) {
  m.def("linear_cross_entropy", &linear_cross_entropy, "cross entropy of x weight^T without kept logits, twice differentiable",
        py::arg("x"), py::arg("weight"), py::arg("targets"), py::arg("ignore_index") = -100, py::arg("reduction") = 2,
        py::call_guard<py::gil_scoped_release>());
}

}  // namespace ext
