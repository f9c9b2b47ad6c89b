// Module `attention_cuda`, packed batches: the plan, attention with its two backward passes.  The autograd
// functions are written in C++ as flash_attention's (attention_ext.cpp); there is no Python form behind
// them, so tracing, forward-mode tangents and functorch transforms are refused.
#include "ext_common.h"

#include <ATen/cuda/CUDAGraphsUtils.cuh>

#include <algorithm>
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

// The sequences that one call of the second backward takes, each padded to `width` rows.
struct PaddedGroup { torch::Tensor starts, ends; int64_t width; };

// No call has more than `most` padded rows (or one sequence).  Without lengths from the host every sequence counts as one of `width`.  With them sequences
// whose lengths are within a factor of two go together, and then those of the next shorter group with them where the rows that this adds cost less than a
// call: 450 us of the host.  In us, for one element (row, head and column) of one padded tensor: 1.1e-4 and 1.7e-8 times the width in half types, 2.1e-4 and
// 6.3e-7 times the width in float (fitted to batches of 300 to 16000 rows in 5 to 60 sequences in one call, 0.5 to 19 ms, within 0.1).
// 12 heads of 64, bf16, one call / a call for every factor of two / this rule, in us: 1000 rows in 20 sequences 684 / 2 218 / 676;
// 4000 in 20 2 029 / 2 244 / 1 383; 16000 in 20 10 655 / 2 941 / 2 881.
std::vector<PaddedGroup> padded_groups(const torch::Tensor& starts, const torch::Tensor& ends, const std::vector<int64_t>& lens, int64_t width, int64_t most,
                                       int64_t row_elements, bool half) {
  const int64_t n_seq = ends.size(0);
  std::vector<PaddedGroup> groups;
  if (lens.empty()) {
    const int64_t each = std::max<int64_t>(1, most / width);
    for (int64_t i = 0; i < n_seq; i += each) groups.push_back({starts.slice(0, i, std::min(n_seq, i + each)), ends.slice(0, i, std::min(n_seq, i + each)), width});
    return groups;
  }
  std::vector<int64_t> order;
  for (int64_t i = 0; i < n_seq; ++i)
    if (lens[i] > 0) order.push_back(i);
  std::stable_sort(order.begin(), order.end(), [&](int64_t a, int64_t b) { return lens[a] > lens[b]; });
  const int64_t count = (int64_t)order.size();
  std::vector<int64_t> first;      // of every group, in `order`
  for (int64_t i = 0, e; i < count; i = e) {
    const int64_t longest = lens[order[i]];
    first.push_back(i);
    for (e = i + 1; e < count && 2 * lens[order[e]] >= longest && (e + 1 - i) * longest <= most; ++e) { }
  }
  auto cost = [&](int64_t n, int64_t w) { return (double)(n * w * row_elements) * (half ? 1.1e-4 + 1.7e-8 * w : 2.1e-4 + 6.3e-7 * w); };
  for (size_t g = first.size() - 1, behind = (size_t)count; g > 0; --g) {      // [first[g], behind) and the group before it
    const int64_t w = lens[order[first[g]]], wider = lens[order[first[g - 1]]], n = (int64_t)behind - first[g];
    if (((int64_t)behind - first[g - 1]) * wider <= most && cost(n, wider) - cost(n, w) < 450.) first.erase(first.begin() + g);
    else behind = (size_t)first[g];
  }
  if (first.size() == 1 && count == n_seq) return {{starts, ends, width}};
  const torch::Tensor by_length = torch::tensor(order, torch::kLong).to(ends.device());
  for (size_t g = 0; g < first.size(); ++g) {
    const torch::Tensor which = by_length.slice(0, first[g], g + 1 < first.size() ? first[g + 1] : count);
    groups.push_back({starts.index_select(0, which), ends.index_select(0, which), lens[order[first[g]]]});
  }
  return groups;
}

// Second backward: the sequences as rows of padded batches, through the double-backward kernels of flash_attention.  A
// padded row has zeros everywhere and comes behind its sequence's rows, which do not see it, so it adds nothing.  The lengths are
// read from the plan unless the caller has given the longest one, which waits for the device.
variable_list packed_double_backward(const torch::Tensor& g_dq, const torch::Tensor& g_dk, const torch::Tensor& g_dv, const torch::Tensor& dO,
                                     const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& O,
                                     const torch::Tensor& L, const torch::Tensor& plan, int64_t n_seq, int64_t window, int64_t max_seqlen) {
  at::AutoGradMode off(false);
  c10::cuda::CUDAGuard guard(q.device());
  const int64_t n_tok = q.size(0), Hq = q.size(1), Hkv = k.size(1), group = Hq / Hkv;
  // a row more than the result's, where every padded row goes
  auto fresh_zeros = [&](const torch::Tensor& like) { return torch::zeros({n_tok + 1, like.size(1), like.size(2)}, like.options()); };
  const variable_list out{fresh_zeros(q), fresh_zeros(q), fresh_zeros(k), fresh_zeros(v)};
  auto results = [&]() {
    variable_list r;
    for (const torch::Tensor& t : out) r.push_back(t.slice(0, 0, n_tok));
    return r;
  };
  if (n_tok == 0 || n_seq == 0 || max_seqlen == 0) return results();
  // bounded as in the kernels: what is no plan (the memory of one that a captured graph has yet to make) must not index outside of the rows
  const torch::Tensor ends = plan.slice(0, plan.numel() - 2 * n_seq, plan.numel() - n_seq).to(at::kLong).clamp_(0, n_tok);
  const torch::Tensor starts = torch::cat({plan.slice(0, 4, 5).to(at::kLong).clamp_(0, n_tok), ends.slice(0, 0, n_seq - 1)});
  std::vector<int64_t> lens;
  int64_t longest = max_seqlen;
  if (max_seqlen < 0) {
    TORCH_CHECK(at::cuda::currentStreamCaptureStatusMayInitCtx() == at::cuda::CaptureStatus::None,
                "the second derivative of packed_attention needs packed_plan(..., max_seqlen=...) while a graph is being captured");
    const torch::Tensor host = (ends - starts).cpu();
    lens.assign(host.data_ptr<int64_t>(), host.data_ptr<int64_t>() + n_seq);
    longest = *std::max_element(lens.begin(), lens.end());
    if (longest <= 0) return results();
  }
  // at most twice the batch's rows, or 128 MB of a tensor, in a call: memory goes with the batch
  const int64_t row_elements = Hq * q.size(2), most = std::max<int64_t>(2 * n_tok, (int64_t(128) << 20) / (row_elements * (int64_t)q.element_size()));
  for (const PaddedGroup& part : padded_groups(starts, ends, lens, std::min(longest, n_tok), most, row_elements, q.scalar_type() != at::kFloat)) {
    const int64_t n = part.ends.size(0), width = part.width;
    const torch::Tensor at = part.starts.unsqueeze(1) + torch::arange(width, ends.options()).unsqueeze(0);      // [n, width]
    const torch::Tensor in = at < part.ends.unsqueeze(1);
    const torch::Tensor from = torch::where(in, at, torch::zeros_like(at)).reshape({-1});
    const torch::Tensor in4 = in.view({n, width, 1, 1});
    // [n_tok, H, D] -> [n, Hq, width, D]
    auto pad = [&](const torch::Tensor& t) {
      torch::Tensor p = t.index_select(0, from).view({n, width, t.size(1), t.size(2)});
      p = torch::where(in4, p, torch::zeros({}, p.options())).permute({0, 2, 1, 3});
      return t.size(1) == Hq ? p.contiguous() : p.unsqueeze(2).expand({n, Hkv, group, width, t.size(2)}).reshape({n, Hq, width, t.size(2)});
    };
    const torch::Tensor Lp = torch::where(in.view({n, 1, width}), L.index_select(1, from).view({Hq, n, width}).permute({1, 0, 2}),
                                          torch::zeros({}, L.options())).contiguous();
    const int seen = (int)std::min<int64_t>(window, std::numeric_limits<int32_t>::max());
    const variable_list r = v7_double_backward_cuda(pad(g_dq), pad(g_dk), pad(g_dv), pad(dO), pad(q), pad(k), pad(v), pad(O), Lp, seen, 0, 0, 0);
    const torch::Tensor to = torch::where(in, at, torch::full_like(at, n_tok)).reshape({-1});
    for (int i = 0; i < 4; ++i) {
      torch::Tensor p = r[i];
      const int64_t heads = out[i].size(1), D = out[i].size(2);
      if (heads != Hq) p = p.view({n, Hkv, group, width, D}).to(at::kFloat).sum(2).to(out[i].scalar_type());
      out[i].index_copy_(0, to, p.permute({0, 2, 1, 3}).reshape({n * width, heads, D}));
    }
  }
  // a given length that is too small would leave rows out of the sums without a word
  if (max_seqlen > 0 && max_seqlen < n_tok) {
    const torch::Tensor longer = plan.select(0, 1) > max_seqlen;
    for (torch::Tensor t : out) t.masked_fill_(longer, std::numeric_limits<double>::quiet_NaN());
  }
  return results();
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

// ---- norm and rotation of q and k ---------------------------------------------------------------

struct RopeArgs { std::vector<int64_t> sections; double eps; };

torch::Tensor or_none(const torch::Tensor& w) { return w.numel() > 0 ? w : torch::Tensor(); }

void check_rope(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& qw, const torch::Tensor& kw, const torch::Tensor& freqs,
                const torch::Tensor& positions, const RopeArgs& a) {
  TORCH_CHECK(q.is_cuda() && k.is_cuda() && freqs.is_cuda() && positions.is_cuda(), "q, k, freqs and positions must be CUDA tensors");
  TORCH_CHECK(q.device() == k.device() && q.device() == freqs.device() && q.device() == positions.device(), "all tensors must be on one device");
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3, "q and k must be [n_tok, heads, D]");
  TORCH_CHECK(q.size(0) == k.size(0) && q.size(2) == k.size(2), "q and k must agree in n_tok and D");
  TORCH_CHECK(q.scalar_type() == k.scalar_type(), "q and k must have the same dtype");
  TORCH_CHECK(q.size(0) <= (1 << 30) && q.size(1) <= (1 << 20) && k.size(1) <= (1 << 20), "q or k is too large");
  for (const torch::Tensor* w : {&qw, &kw}) {
    if (!w->defined()) continue;
    TORCH_CHECK(w->is_cuda() && w->device() == q.device() && w->dim() == 1 && w->size(0) == q.size(2), "a weight must be a CUDA tensor [D]");
    TORCH_CHECK(w->scalar_type() == q.scalar_type() || w->scalar_type() == at::kFloat, "a weight must have the dtype of q and k, or be float32");
  }
  TORCH_CHECK(freqs.scalar_type() == at::kFloat && freqs.dim() == 3 && freqs.size(2) == 2 && freqs.size(1) * 2 == q.size(2) && freqs.size(0) <= (1 << 30),
              "freqs must be float32 [rows, D / 2, 2]");
  TORCH_CHECK(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong, "positions must be int32 or int64");
  TORCH_CHECK((positions.dim() == 1 || positions.dim() == 2) && positions.size(-1) == q.size(0), "positions must be [n_tok] or [axes, n_tok]");
  TORCH_CHECK((int64_t)a.sections.size() == (positions.dim() == 1 ? 1 : positions.size(0)) && a.sections.size() <= 4,
              "sections must name the pairs of every axis of positions, at most 4");
}

// rows whose elements lie side by side
torch::Tensor with_dense_rows(const torch::Tensor& t) { return t.stride(2) == 1 || t.size(2) == 1 ? t : t.contiguous(); }

attn_rope_shape_t rope_shape(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& qw, const torch::Tensor& kw, const torch::Tensor& freqs,
                             const torch::Tensor& positions, const RopeArgs& a) {
  attn_rope_shape_t s{};
  s.n_tok = (int32_t)q.size(0);
  s.q_heads = (int32_t)q.size(1);
  s.k_heads = (int32_t)k.size(1);
  s.D = (int32_t)q.size(2);
  s.dtype = dtype_code(q);
  s.table_rows = (int32_t)freqs.size(0);
  s.axes = (int32_t)a.sections.size();
  s.positions64 = positions.scalar_type() == at::kLong;
  for (size_t i = 0; i < a.sections.size(); ++i) s.section[i] = (int32_t)std::min<int64_t>(a.sections[i], 1 << 20);
  s.weight_float[0] = qw.defined() && qw.scalar_type() == at::kFloat;
  s.weight_float[1] = kw.defined() && kw.scalar_type() == at::kFloat;
  s.eps = (float)a.eps;
  s.axis_stride = positions.dim() == 2 ? positions.stride(0) : 0;
  s.row_stride[0] = q.stride(0); s.head_stride[0] = q.stride(1);
  s.row_stride[1] = k.stride(0); s.head_stride[1] = k.stride(1);
  return s;
}

void* ptr_or_null(const torch::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

variable_list rope_forward(const torch::Tensor& q_in, const torch::Tensor& k_in, const torch::Tensor& qw_in, const torch::Tensor& kw_in,
                           const torch::Tensor& freqs_in, const torch::Tensor& positions_in, const RopeArgs& a) {
  check_rope(q_in, k_in, qw_in, kw_in, freqs_in, positions_in, a);
  c10::cuda::CUDAGuard guard(q_in.device());
  const torch::Tensor q = with_dense_rows(q_in), k = with_dense_rows(k_in), freqs = freqs_in.contiguous();
  const torch::Tensor positions = positions_in.size(-1) > 1 && positions_in.stride(-1) != 1 ? positions_in.contiguous() : positions_in;
  const torch::Tensor qw = qw_in.defined() ? qw_in.contiguous() : qw_in, kw = kw_in.defined() ? kw_in.contiguous() : kw_in;
  const attn_rope_shape_t s = rope_shape(q, k, qw, kw, freqs, positions, a);
  variable_list out{fresh(q.sizes(), q.scalar_type(), q), fresh(k.sizes(), k.scalar_type(), k)};
  check_rc(attn_b200_packed_qk_norm_rope(&s, q.data_ptr(), k.data_ptr(), ptr_or_null(qw), ptr_or_null(kw), freqs.data_ptr<float>(), positions.data_ptr(),
                                         out[0].data_ptr(), out[1].data_ptr(), at::cuda::getCurrentCUDAStream().stream()),
           "packed_qk_norm_rope");
  return out;
}

// {gq, gk, gq_weight, gk_weight}; a weight's is undefined without it or where it is not wanted
variable_list rope_backward(const torch::Tensor& gq_in, const torch::Tensor& gk_in, const torch::Tensor& q_in, const torch::Tensor& k_in,
                            const torch::Tensor& qw_in, const torch::Tensor& kw_in, const torch::Tensor& freqs_in, const torch::Tensor& positions_in,
                            const RopeArgs& a, bool want_qw, bool want_kw) {
  c10::cuda::CUDAGuard guard(q_in.device());
  const torch::Tensor q = with_dense_rows(q_in), k = with_dense_rows(k_in), freqs = freqs_in.contiguous();
  const torch::Tensor positions = positions_in.size(-1) > 1 && positions_in.stride(-1) != 1 ? positions_in.contiguous() : positions_in;
  const torch::Tensor qw = qw_in.defined() ? qw_in.contiguous() : qw_in, kw = kw_in.defined() ? kw_in.contiguous() : kw_in;
  auto gradient = [](const torch::Tensor& g, const torch::Tensor& like) {
    TORCH_CHECK(!g.defined() || (g.sizes() == like.sizes() && g.scalar_type() == like.scalar_type() && g.device() == like.device()),
                "the gradients of packed_qk_norm_rope's results must be like them");
    return g.defined() ? with_dense_rows(g) : torch::zeros(like.sizes(), like.options());
  };
  const torch::Tensor gq = gradient(gq_in, q), gk = gradient(gk_in, k);
  attn_rope_shape_t s = rope_shape(q, k, qw, kw, freqs, positions, a);
  s.g_row_stride[0] = gq.stride(0); s.g_head_stride[0] = gq.stride(1);
  s.g_row_stride[1] = gk.stride(0); s.g_head_stride[1] = gk.stride(1);
  variable_list out{fresh(q.sizes(), q.scalar_type(), q), fresh(k.sizes(), k.scalar_type(), k), torch::Tensor(), torch::Tensor()};
  if (want_qw && qw.defined()) out[2] = fresh(qw.sizes(), qw.scalar_type(), qw);
  if (want_kw && kw.defined()) out[3] = fresh(kw.sizes(), kw.scalar_type(), kw);
  torch::Tensor scratch;
  if (out[2].defined() || out[3].defined())
    scratch = fresh({(int64_t)(attn_b200_packed_qk_norm_rope_backward_scratch_bytes(&s) / sizeof(float)) + 4}, at::kFloat, q);
  check_rc(attn_b200_packed_qk_norm_rope_backward(&s, q.data_ptr(), k.data_ptr(), ptr_or_null(qw), ptr_or_null(kw), freqs.data_ptr<float>(),
                                                  positions.data_ptr(), gq.data_ptr(), gk.data_ptr(), out[0].data_ptr(), out[1].data_ptr(),
                                                  ptr_or_null(out[2]), ptr_or_null(out[3]), static_cast<float*>(ptr_or_null(scratch)),
                                                  at::cuda::getCurrentCUDAStream().stream()),
           "packed_qk_norm_rope backward");
  return out;
}

// The same out of ordinary operations, for the second backward.
torch::Tensor rope_angles(const torch::Tensor& freqs, const torch::Tensor& positions, const RopeArgs& a) {
  const torch::Tensor nan = torch::full({}, std::numeric_limits<float>::quiet_NaN(), freqs.options());
  if (freqs.size(0) == 0) return nan.expand({positions.size(-1), 1, freqs.size(1), 2});
  std::vector<torch::Tensor> parts;
  int64_t first = 0;
  for (size_t i = 0; i < a.sections.size(); ++i) {
    const torch::Tensor p = (positions.dim() == 2 ? positions.select(0, (int64_t)i) : positions).to(at::kLong);
    const torch::Tensor in = (p >= 0) & (p < freqs.size(0));
    const torch::Tensor t = freqs.slice(1, first, first + a.sections[i]).index_select(0, torch::where(in, p, torch::zeros_like(p)));
    parts.push_back(torch::where(in.view({-1, 1, 1}), t, nan));
    first += a.sections[i];
  }
  return torch::cat(parts, 1).unsqueeze(1);      // [n_tok, 1, D / 2, 2]
}

torch::Tensor rope_formula(const torch::Tensor& x, const torch::Tensor& w, const torch::Tensor& angles, double eps) {
  torch::Tensor y = x.to(at::kFloat);
  if (w.defined()) y = y * torch::rsqrt(y.pow(2).mean({-1}, true) + eps) * w.to(at::kFloat);
  const torch::Tensor pair = y.reshape({x.size(0), x.size(1), x.size(2) / 2, 2});
  const torch::Tensor u = pair.select(-1, 0), v = pair.select(-1, 1), c = angles.select(-1, 0), s = angles.select(-1, 1);
  return torch::stack({u * c - v * s, u * s + v * c}, -1).reshape(x.sizes()).to(x.scalar_type());
}

void save_rope(AutogradContext* ctx, const std::vector<int64_t>& sections, double eps) {
  ctx->set_materialize_grads(false);
  ctx->saved_data["sections"] = sections;
  ctx->saved_data["eps"] = eps;
}
RopeArgs saved_rope(AutogradContext* ctx) { return {ctx->saved_data["sections"].toIntVector(), ctx->saved_data["eps"].toDouble()}; }

struct PackedQKNormRopeBackward : public torch::autograd::Function<PackedQKNormRopeBackward> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& gq, const torch::Tensor& gk, const torch::Tensor& q, const torch::Tensor& k,
                               const torch::Tensor& qw, const torch::Tensor& kw, const torch::Tensor& freqs, const torch::Tensor& positions,
                               std::vector<int64_t> sections, double eps) {
    save_rope(ctx, sections, eps);
    ctx->save_for_backward({gq, gk, q, k, qw, kw, freqs, positions});
    variable_list r = rope_backward(gq, gk, q, k, or_none(qw), or_none(kw), freqs, positions, {sections, eps}, true, true);
    for (int i = 2; i < 4; ++i)
      if (!r[i].defined()) r[i] = fresh({0}, at::kFloat, q);
    return r;
  }

  static variable_list backward(AutogradContext* ctx, variable_list tangents) {
    variable_list out(10);      // gq, gk, q, k, qw, kw, freqs, positions, sections, eps
    const variable_list s = ctx->get_saved_variables();
    const RopeArgs a = saved_rope(ctx);
    const bool keep_graph = at::GradMode::is_enabled();
    at::AutoGradMode on(true);
    const torch::Tensor angles = rope_angles(s[6], s[7], a).detach();
    // aliases of the inputs, so that the derivatives are partial ones even where the inputs depend on one another
    auto alias = [&](const torch::Tensor& t) { return keep_graph && t.requires_grad() ? t.view_as(t) : t.detach().requires_grad_(true); };
    for (int side = 0; side < 2; ++side) {
      // a row without a gradient that is not a number, or whose position is outside of the table, gives 0 here too
      const torch::Tensor still = (s[side].detach() == 0).all(-1, true);
      const torch::Tensor dead = still & s[2 + side].detach().isfinite().all(-1, true).logical_not();
      const torch::Tensor turn = torch::where(still.unsqueeze(-1) & angles.isnan(), torch::zeros({}, angles.options()), angles);
      const torch::Tensor g = alias(s[side]), x = alias(s[2 + side]), kept = torch::where(dead, torch::zeros({}, x.options()), x);
      variable_list first_wrt{x}, wrt{g, x};
      torch::Tensor w;
      if (s[4 + side].numel() > 0) {
        w = alias(s[4 + side]);
        first_wrt.push_back(w);
        wrt.push_back(w);
      }
      const variable_list first = torch::autograd::grad({rope_formula(kept, w, turn, a.eps)}, first_wrt, {g}, true, true);
      variable_list of, with;
      for (size_t i = 0; i < first.size(); ++i) {
        const torch::Tensor& t = tangents[i == 0 ? side : 2 + side];
        if (t.defined()) { of.push_back(first[i]); with.push_back(t); }
      }
      if (of.empty()) continue;
      const variable_list r = torch::autograd::grad(of, wrt, with, true, keep_graph, true);
      out[side] = r[0];
      out[2 + side] = r[1];
      if (w.defined()) out[4 + side] = r[2];
    }
    return out;
  }
};

struct PackedQKNormRope : public torch::autograd::Function<PackedQKNormRope> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& qw, const torch::Tensor& kw,
                               const torch::Tensor& freqs, const torch::Tensor& positions, std::vector<int64_t> sections, double eps) {
    variable_list r = rope_forward(q, k, or_none(qw), or_none(kw), freqs, positions, {sections, eps});
    save_rope(ctx, sections, eps);
    ctx->save_for_backward({q, k, qw, kw, freqs, positions});
    return r;
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(8);      // q, k, qw, kw, freqs, positions, sections, eps
    if (!g[0].defined() && !g[1].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    const RopeArgs a = saved_rope(ctx);
    TORCH_CHECK(!has_tangent({&g[0], &g[1], &s[0], &s[1], &s[2], &s[3]}), "packed_qk_norm_rope has no forward-mode derivative");
    variable_list r;
    if (at::GradMode::is_enabled()) {
      auto whole = [](const torch::Tensor& t, const torch::Tensor& like) { return t.defined() ? t : torch::zeros(like.sizes(), like.options()); };
      r = PackedQKNormRopeBackward::apply(whole(g[0], s[0]), whole(g[1], s[1]), s[0], s[1], s[2], s[3], s[4], s[5], a.sections, a.eps);
      for (int i = 2; i < 4; ++i)
        if (s[i].numel() == 0) r[i] = torch::Tensor();
    } else {
      r = rope_backward(g[0], g[1], s[0], s[1], or_none(s[2]), or_none(s[3]), s[4], s[5], a, ctx->needs_input_grad(2), ctx->needs_input_grad(3));
    }
    for (int i = 0; i < 4; ++i) out[i] = std::move(r[i]);
    return out;
  }
};

variable_list packed_qk_norm_rope(const torch::Tensor& q, const torch::Tensor& k, c10::optional<torch::Tensor> q_weight,
                                  c10::optional<torch::Tensor> k_weight, const torch::Tensor& freqs, const torch::Tensor& positions,
                                  std::vector<int64_t> sections, double eps) {
  const torch::Tensor qw = q_weight.value_or(torch::Tensor()), kw = k_weight.value_or(torch::Tensor());
  refuse_transforms({&q, &k, &qw, &kw, &freqs}, "packed_qk_norm_rope");
  TORCH_CHECK(!freqs.requires_grad(), "packed_qk_norm_rope has no gradient of freqs");
  TORCH_CHECK(q.dim() != 3 || q.size(2) > 0, "D must be positive");
  if (!wants_graph({&q, &k, &qw, &kw})) return rope_forward(q, k, qw, kw, freqs, positions, {sections, eps});
  check_rope(q, k, qw, kw, freqs, positions, {sections, eps});
  const torch::Tensor none = qw.defined() && kw.defined() ? torch::Tensor() : fresh({0}, q.scalar_type(), q);
  return PackedQKNormRope::apply(q, k, qw.defined() ? qw : none, kw.defined() ? kw : none, freqs, positions, sections, eps);
}

}  // namespace

void register_packed(pybind11::module& m) {
  m.def("packed_plan", &packed_plan, "the plan of a packed batch, int32", py::arg("cu_seqlens"), py::arg("n_tok"),
        py::call_guard<py::gil_scoped_release>());
  m.def("packed_attention", &packed_attention, "causal attention within the sequences of a packed batch, grouped heads, twice differentiable -> O",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("plan"), py::arg("n_tok"), py::arg("n_seq"), py::arg("window_size") = py::none(),
        py::arg("max_seqlen") = py::none(), py::call_guard<py::gil_scoped_release>());
  m.def("packed_qk_norm_rope", &packed_qk_norm_rope, "RMS norm of q and k per head and rotation by per-token positions, twice differentiable -> [q, k]",
        py::arg("q"), py::arg("k"), py::arg("q_weight"), py::arg("k_weight"), py::arg("freqs"), py::arg("positions"), py::arg("sections"),
        py::arg("eps") = 1e-6, py::call_guard<py::gil_scoped_release>());
}

}  // namespace ext
