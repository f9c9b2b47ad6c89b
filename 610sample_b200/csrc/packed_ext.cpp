// Module `attention_cuda`, packed batches: the plan, attention with its two backward passes.  The autograd
// functions are written in C++ as flash_attention's (attention_ext.cpp); there is no Python form behind
// them, so tracing, forward-mode tangents and functorch transforms are refused.
#include "ext_common.h"

#include <ATen/cuda/CUDAGraphsUtils.cuh>

#include <limits>

namespace ext {

namespace {

int64_t window_of(const c10::optional<int64_t>& window_size) {
  if (!window_size.has_value()) return std::numeric_limits<int32_t>::max();
  TORCH_CHECK(*window_size >= 0, "window_size must be >= 0, or None");
  return std::min<int64_t>(*window_size, std::numeric_limits<int32_t>::max());
}

void check_packed(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& plan, int64_t n_seq) {
  TORCH_CHECK(q.is_cuda() && k.is_cuda() && v.is_cuda(), "q, k and v must be CUDA tensors");
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.dim() == 3, "q, k, v must be [n_tok, heads, D]");
  TORCH_CHECK(k.sizes() == v.sizes(), "k and v must have the same shape");
  TORCH_CHECK(q.size(0) == k.size(0) && q.size(2) == k.size(2), "q and k must agree in n_tok and D");
  TORCH_CHECK(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(), "q, k, v must have the same dtype");
  TORCH_CHECK(q.device() == k.device() && q.device() == v.device(), "q, k, v must be on one device");
  TORCH_CHECK(q.size(0) <= (1 << 30), "n_tok must be at most 2^30");
  TORCH_CHECK(k.size(1) > 0 && q.size(1) > 0 && q.size(1) % k.size(1) == 0 && q.size(1) <= (1 << 24),
              "the heads of q must be a positive multiple of those of k (got ", q.size(1), " and ", k.size(1), ")");
  TORCH_CHECK(plan.is_cuda() && plan.device() == q.device() && plan.scalar_type() == at::kInt && plan.is_contiguous(),
              "plan must be a plan made by packed_plan on the device of q");
  TORCH_CHECK(n_seq >= 0 && n_seq <= (1 << 30) && plan.numel() == (int64_t)attn_b200_packed_plan_ints((int32_t)q.size(0), (int32_t)n_seq),
              "the plan is not one for ", q.size(0), " rows");
}

// As the kernels take it: for f16 / bf16 any strides that a tensor map can have, else a dense copy.
torch::Tensor strided(const torch::Tensor& t) {
  if (t.scalar_type() == at::kFloat || t.numel() == 0) return dense(t);
  auto fits = [&](int dim) { return t.size(dim) == 1 || (t.stride(dim) > 0 && t.stride(dim) % 8 == 0 && t.stride(dim) < (1LL << 39)); };
  const bool ok = t.stride(2) == 1 && t.size(2) % 8 == 0 && fits(0) && fits(1) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  return ok ? t : dense(t);
}

attn_packed_shape_t packed_shape(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor* dO, int64_t n_seq,
                                 int64_t window) {
  attn_packed_shape_t s{};
  s.n_tok = (int32_t)q.size(0);
  s.n_seq = (int32_t)n_seq;
  s.q_heads = (int32_t)q.size(1);
  s.kv_heads = (int32_t)k.size(1);
  s.D = (int32_t)q.size(2);
  s.window_size = (int32_t)window;
  s.dtype = dtype_code(q);
  const torch::Tensor* in[4] = {&q, &k, &v, dO != nullptr ? dO : &q};
  for (int i = 0; i < 4; ++i) {      // an axis of one element may have any stride
    s.head_stride[i] = in[i]->size(1) == 1 ? in[i]->size(2) : in[i]->stride(1);
    s.row_stride[i] = in[i]->size(0) == 1 ? in[i]->size(1) * in[i]->size(2) : in[i]->stride(0);
  }
  return s;
}

variable_list packed_forward(const torch::Tensor& q_in, const torch::Tensor& k_in, const torch::Tensor& v_in, const torch::Tensor& plan,
                             int64_t n_seq, int64_t window) {
  check_packed(q_in, k_in, v_in, plan, n_seq);
  c10::cuda::CUDAGuard guard(q_in.device());
  raise_if_earlier_call_timed_out(q_in.device().index());
  const torch::Tensor q = strided(q_in), k = strided(k_in), v = strided(v_in);
  const attn_packed_shape_t s = packed_shape(q, k, v, nullptr, n_seq, window);
  auto O = fresh(q.sizes(), q.scalar_type(), q);
  auto L = fresh({q.size(1), q.size(0)}, at::kFloat, q);
  check_rc(attn_b200_packed_forward(&s, plan.data_ptr<int32_t>(), q.data_ptr(), k.data_ptr(), v.data_ptr(), O.data_ptr(), L.data_ptr<float>(),
                                    at::cuda::getCurrentCUDAStream().stream()),
           "packed_attention");
  return {O, L};
}

variable_list packed_backward(const torch::Tensor& dO_in, const torch::Tensor& q_in, const torch::Tensor& k_in, const torch::Tensor& v_in,
                              const torch::Tensor& O, const torch::Tensor& L, const torch::Tensor& plan, int64_t n_seq, int64_t window) {
  check_packed(q_in, k_in, v_in, plan, n_seq);
  TORCH_CHECK(dO_in.sizes() == q_in.sizes() && dO_in.scalar_type() == q_in.scalar_type() && dO_in.device() == q_in.device(),
              "the gradient of packed_attention's result must be like it");
  c10::cuda::CUDAGuard guard(q_in.device());
  raise_if_earlier_call_timed_out(q_in.device().index());
  const torch::Tensor q = strided(q_in), k = strided(k_in), v = strided(v_in), dO = strided(dO_in);
  const attn_packed_shape_t s = packed_shape(q, k, v, &dO, n_seq, window);
  auto dQ = fresh(q.sizes(), q.scalar_type(), q);
  auto dK = fresh(k.sizes(), k.scalar_type(), k);
  auto dV = fresh(v.sizes(), v.scalar_type(), v);
  auto scratch = fresh({q.size(0) * q.size(1) + 4}, at::kFloat, q);
  check_rc(attn_b200_packed_backward(&s, plan.data_ptr<int32_t>(), dO.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), O.data_ptr(),
                                     L.data_ptr<float>(), dQ.data_ptr(), dK.data_ptr(), dV.data_ptr(), scratch.data_ptr<float>(),
                                     at::cuda::getCurrentCUDAStream().stream()),
           "packed_attention backward");
  return {dQ, dK, dV};
}

// Second backward: the sequences as rows of a padded batch, through the double-backward kernels of flash_attention.  A
// padded row has zeros everywhere and comes behind its sequence's rows, which do not see it, so it adds nothing.  The longest
// sequence's length is read from the plan unless the caller has given it, which waits for the device.
variable_list packed_double_backward(const torch::Tensor& g_dq, const torch::Tensor& g_dk, const torch::Tensor& g_dv, const torch::Tensor& dO,
                                     const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& O,
                                     const torch::Tensor& L, const torch::Tensor& plan, int64_t n_seq, int64_t window, int64_t max_seqlen) {
  at::AutoGradMode off(false);
  c10::cuda::CUDAGuard guard(q.device());
  const int64_t n_tok = q.size(0), Hq = q.size(1), Hkv = k.size(1), group = Hq / Hkv;
  variable_list zero{torch::zeros_like(q), torch::zeros_like(q), torch::zeros_like(k), torch::zeros_like(v)};
  if (n_tok == 0 || n_seq == 0) return zero;
  if (max_seqlen < 0) {
    TORCH_CHECK(at::cuda::currentStreamCaptureStatusMayInitCtx() == at::cuda::CaptureStatus::None,
                "the second derivative of packed_attention needs packed_plan(..., max_seqlen=...) while a graph is being captured");
    max_seqlen = plan[1].item<int32_t>();
  }
  const int64_t width = std::min(max_seqlen, n_tok);
  if (width == 0) return zero;
  const torch::Tensor ends = plan.slice(0, plan.numel() - 2 * n_seq, plan.numel() - n_seq).to(at::kLong);
  const torch::Tensor starts = torch::cat({plan.slice(0, 4, 5).to(at::kLong), ends.slice(0, 0, n_seq - 1)});
  const torch::Tensor at = starts.unsqueeze(1) + torch::arange(width, ends.options()).unsqueeze(0);      // [n_seq, width]
  const torch::Tensor in = at < ends.unsqueeze(1);
  const torch::Tensor from = torch::where(in, at, torch::zeros_like(at)).reshape({-1});
  const torch::Tensor in4 = in.view({n_seq, width, 1, 1});
  // [n_tok, H, D] -> [n_seq, Hq, width, D]
  auto pad = [&](const torch::Tensor& t) {
    torch::Tensor p = t.index_select(0, from).view({n_seq, width, t.size(1), t.size(2)});
    p = torch::where(in4, p, torch::zeros({}, p.options())).permute({0, 2, 1, 3});
    return t.size(1) == Hq ? p.contiguous() : p.unsqueeze(2).expand({n_seq, Hkv, group, width, t.size(2)}).reshape({n_seq, Hq, width, t.size(2)});
  };
  const torch::Tensor Lp = torch::where(in.view({n_seq, 1, width}), L.index_select(1, from).view({Hq, n_seq, width}).permute({1, 0, 2}),
                                        torch::zeros({}, L.options())).contiguous();
  const int seen = (int)std::min<int64_t>(window, std::numeric_limits<int32_t>::max());
  const variable_list r = v7_double_backward_cuda(pad(g_dq), pad(g_dk), pad(g_dv), pad(dO), pad(q), pad(k), pad(v), pad(O), Lp, seen, 0, 0, 0);
  // a row of no sequence is where every padded row goes, and gets zeros
  const torch::Tensor to = torch::where(in, at, torch::full_like(at, n_tok)).reshape({-1});
  auto unpad = [&](const torch::Tensor& t, const torch::Tensor& like) {
    torch::Tensor p = t;
    if (like.size(1) != Hq) p = p.view({n_seq, Hkv, group, width, like.size(2)}).to(at::kFloat).sum(2).to(like.scalar_type());
    p = p.permute({0, 2, 1, 3}).reshape({n_seq * width, like.size(1), like.size(2)});
    torch::Tensor out = torch::zeros({n_tok + 1, like.size(1), like.size(2)}, like.options());
    out.index_copy_(0, to, p);
    return out.slice(0, 0, n_tok);
  };
  return {unpad(r[0], q), unpad(r[1], q), unpad(r[2], k), unpad(r[3], v)};
}

struct PackedAttentionBackward : public torch::autograd::Function<PackedAttentionBackward> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& dO, const torch::Tensor& q, const torch::Tensor& k,
                               const torch::Tensor& v, const torch::Tensor& O, const torch::Tensor& L, const torch::Tensor& plan, int64_t n_seq,
                               int64_t window, int64_t max_seqlen) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({dO, q, k, v, O, L, plan});
    ctx->saved_data["n_seq"] = n_seq;
    ctx->saved_data["window"] = window;
    ctx->saved_data["max_seqlen"] = max_seqlen;
    return packed_backward(dO, q, k, v, O, L, plan, n_seq, window);
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(10);
    if (!g[0].defined() && !g[1].defined() && !g[2].defined()) return out;
    TORCH_CHECK(!at::GradMode::is_enabled(), "packed_attention has no third derivative: call the second backward without create_graph");
    const variable_list s = ctx->get_saved_variables();
    auto tangent = [](const torch::Tensor& t, const torch::Tensor& like) { return t.defined() ? t : torch::zeros_like(like); };
    variable_list r = packed_double_backward(tangent(g[0], s[1]), tangent(g[1], s[2]), tangent(g[2], s[3]), s[0], s[1], s[2], s[3], s[4], s[5],
                                             s[6], ctx->saved_data["n_seq"].toInt(), ctx->saved_data["window"].toInt(),
                                             ctx->saved_data["max_seqlen"].toInt());
    for (int i = 0; i < 4; ++i) out[i] = std::move(r[i]);
    return out;
  }
};

struct PackedAttention : public torch::autograd::Function<PackedAttention> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
                               const torch::Tensor& plan, int64_t n_seq, int64_t window, int64_t max_seqlen) {
    variable_list r = packed_forward(q, k, v, plan, n_seq, window);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({q, k, v, r[0], r[1], plan});
    ctx->saved_data["n_seq"] = n_seq;
    ctx->saved_data["window"] = window;
    ctx->saved_data["max_seqlen"] = max_seqlen;
    return r[0];
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(7);
    if (!g[0].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    const int64_t n_seq = ctx->saved_data["n_seq"].toInt(), window = ctx->saved_data["window"].toInt();
    TORCH_CHECK(!has_tangent({&g[0], &s[0], &s[1], &s[2]}), "packed_attention has no forward-mode derivative");
    variable_list r = at::GradMode::is_enabled()
                          ? PackedAttentionBackward::apply(g[0], s[0], s[1], s[2], s[3].detach(), s[4], s[5], n_seq, window,
                                                           ctx->saved_data["max_seqlen"].toInt())
                          : packed_backward(g[0], s[0], s[1], s[2], s[3], s[4], s[5], n_seq, window);
    for (int i = 0; i < 3; ++i) out[i] = std::move(r[i]);
    return out;
  }
};

torch::Tensor packed_plan(const torch::Tensor& cu_seqlens, int64_t n_tok) {
  TORCH_CHECK(cu_seqlens.is_cuda() && cu_seqlens.dim() == 1 && cu_seqlens.numel() >= 1, "cu_seqlens must be a CUDA tensor of n_seq + 1 offsets");
  TORCH_CHECK(cu_seqlens.scalar_type() == at::kInt || cu_seqlens.scalar_type() == at::kLong, "cu_seqlens must be int32 or int64");
  TORCH_CHECK(n_tok >= 0 && n_tok <= (1 << 30), "n_tok must be in [0, 2^30]");
  TORCH_CHECK(cu_seqlens.numel() - 1 <= (1 << 30), "too many sequences");
  c10::cuda::CUDAGuard guard(cu_seqlens.device());
  const int32_t n_seq = (int32_t)(cu_seqlens.numel() - 1);
  torch::Tensor cu = cu_seqlens;
  if (cu.scalar_type() == at::kLong) cu = cu.clamp(0, n_tok).to(at::kInt);
  cu = cu.contiguous();
  torch::Tensor plan = fresh({(int64_t)attn_b200_packed_plan_ints((int32_t)n_tok, n_seq)}, at::kInt, cu);
  check_rc(attn_b200_packed_plan(cu.data_ptr<int32_t>(), (int32_t)n_tok, n_seq, plan.data_ptr<int32_t>(),
                                 at::cuda::getCurrentCUDAStream().stream()),
           "packed_plan");
  return plan;
}

torch::Tensor packed_attention(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& plan, int64_t n_tok,
                               int64_t n_seq, c10::optional<int64_t> window_size, c10::optional<int64_t> max_seqlen) {
  refuse_transforms({&q, &k, &v}, "packed_attention");
  TORCH_CHECK(q.dim() != 3 || q.size(0) == n_tok, "the plan is one for ", n_tok, " rows, q has ", q.size(0));
  const int64_t window = window_of(window_size);
  if (!wants_graph({&q, &k, &v})) return packed_forward(q, k, v, plan, n_seq, window)[0];
  return PackedAttention::apply(q, k, v, plan, n_seq, window, max_seqlen.value_or(-1));
}

}  // namespace

void register_packed(pybind11::module& m) {
  m.def("packed_plan", &packed_plan, "the plan of a packed batch, int32", py::arg("cu_seqlens"), py::arg("n_tok"),
        py::call_guard<py::gil_scoped_release>());
  m.def("packed_attention", &packed_attention, "causal attention within the sequences of a packed batch, grouped heads, twice differentiable -> O",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("plan"), py::arg("n_tok"), py::arg("n_seq"), py::arg("window_size") = py::none(),
        py::arg("max_seqlen") = py::none(), py::call_guard<py::gil_scoped_release>());
}

}  // namespace ext
