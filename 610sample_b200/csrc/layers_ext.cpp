// Module `attention_cuda`: a decoder layer's operators between its attention calls, twice differentiable: layer norm, linear layers with bias,
// activation and residual, gated feed-forward blocks.
#include "ext_common.h"

namespace ext {

namespace {

// A matrix as the kernels take it: columns dense; for half types rows a multiple of 8 elements apart from a 16-byte aligned base.  What is not so is
// copied, with padded rows.
struct Matrix {
  torch::Tensor t;
  int64_t ld = 0;
  const void* data() const { return t.data_ptr(); }
};

torch::Tensor padded(int64_t rows, int64_t cols, const torch::Tensor& like, at::ScalarType type) {
  const int64_t pitch = type == at::kFloat ? cols : (cols + 7) / 8 * 8;
  torch::Tensor t = fresh({rows, pitch}, type, like);
  return pitch == cols ? t : t.narrow(1, 0, cols);
}

int64_t columns_of(const torch::Tensor& t) { return t.size(t.dim() - 1); }

// a matrix whose columns are dense, into another one
void copy_rows(const torch::Tensor& from, int64_t from_ld, const torch::Tensor& to, int64_t to_ld) {
  check_rc(attn_b200_copy_rows(from.data_ptr(), from_ld, to.data_ptr(), to_ld, (int32_t)from.size(0), (int32_t)from.size(1), dtype_code(from),
                               at::cuda::getCurrentCUDAStream().stream()),
           "copy");
}

Matrix matrix(const torch::Tensor& t_in, bool any_rows = false) {
  const int64_t cols = columns_of(t_in), rows = cols > 0 ? t_in.numel() / cols : 0;
  torch::Tensor t = t_in.dim() == 2 ? t_in : t_in.reshape({rows, cols});
  if (t.is_neg()) t = t.resolve_neg();      // a negation that has not been carried out yet (the imaginary part of a conjugate)
  const bool half = t.scalar_type() != at::kFloat;
  const int64_t ld = rows > 1 ? t.stride(0) : (cols + 7) / 8 * 8;      // one row: any distance
  const bool dense_rows = (cols <= 1 || t.stride(1) == 1) && ld >= cols;
  if (t.numel() > 0 && dense_rows && (any_rows || !half || (ld % 8 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0))) return {t, ld};
  torch::Tensor copy = any_rows ? fresh({rows, cols}, t.scalar_type(), t) : padded(rows, cols, t, t.scalar_type());
  const int64_t pitch = any_rows || !half ? cols : (cols + 7) / 8 * 8;
  if (dense_rows && t.numel() > 0) copy_rows(t, ld, copy, pitch);
  else copy.copy_(t);
  return {copy, rows > 1 ? pitch : (cols + 7) / 8 * 8};
}

// a vector as the kernels take it
torch::Tensor packed(const torch::Tensor& t) { return t.defined() ? t.resolve_neg().contiguous() : t; }

// The copy that `matrix` made of a tensor, for the backward to read again; nothing where it made none
torch::Tensor copied(const Matrix& m, const torch::Tensor& from) { return m.t.is_alias_of(from) ? torch::Tensor() : m.t; }
const torch::Tensor& either(const torch::Tensor& copy, const torch::Tensor& from) { return copy.defined() ? copy : from; }

Matrix result(int64_t rows, int64_t cols, const torch::Tensor& like, at::ScalarType type) {
  return {padded(rows, cols, like, type), type == at::kFloat ? cols : (cols + 7) / 8 * 8};
}
Matrix result(int64_t rows, int64_t cols, const torch::Tensor& like) { return result(rows, cols, like, like.scalar_type()); }
// A result as the caller gets it: of its own, not a view that autograd knows of, which could not be changed in place behind a custom function
torch::Tensor handed(const Matrix& m, at::IntArrayRef sizes) {
  if (m.t.is_contiguous()) {
    if (m.t.sizes() == sizes && !m.t.is_view()) return m.t;
    at::AutoDispatchBelowADInplaceOrView untracked;
    return m.t.view(sizes);
  }
  const torch::Tensor t = fresh(sizes, m.t.scalar_type(), m.t);
  copy_rows(m.t, m.ld, t, m.t.size(1));
  return t;
}

// What a gated product keeps (attn_products_t): of half types z and u in rows of whole sectors, and a plane of bytes
struct KeptPlanes {
  Matrix z, u;
  torch::Tensor low;
  int64_t ld_low = 0;
};
KeptPlanes kept_planes(int64_t rows, int64_t cols, const torch::Tensor& like) {
  if (like.scalar_type() == at::kFloat) return {result(rows, cols, like), result(rows, cols, like), torch::Tensor(), 0};
  const int64_t pitch = (cols + 15) / 16 * 16, bytes = (cols + 31) / 32 * 32;
  auto plane = [&] { return Matrix{fresh({rows, pitch}, like.scalar_type(), like), pitch}; };
  return {plane(), plane(), fresh({rows, bytes}, at::kByte, like), bytes};
}
KeptPlanes kept_planes(const torch::Tensor& z, const torch::Tensor& u, const torch::Tensor& low) {
  return {{z, z.size(1)}, {u, u.size(1)}, low, low.defined() ? low.size(1) : 0};
}

std::vector<int64_t> with_columns(const torch::Tensor& x, int64_t cols) {
  std::vector<int64_t> sizes = x.sizes().vec();
  sizes.back() = cols;
  return sizes;
}

struct Pair { const Matrix *a, *b; };

// One call of attn_b200_products, put together result by result
struct Products {
  attn_products_t c{};
  torch::Tensor like;

  Products(const torch::Tensor& t, int form, int kind = ATTN_PRODUCT_PLAIN, int64_t activation = ATTN_ACT_NONE) : like(t) {
    c.dtype = dtype_code(t);
    c.form = form;
    c.kind = kind;
    c.activation = (int32_t)activation;
  }
  Products& add(const Matrix& out, int64_t rows, int64_t cols, int64_t k, std::initializer_list<Pair> pairs) {
    attn_product_t& p = c.product[c.count++];
    p.rows = (int32_t)rows; p.cols = (int32_t)cols; p.k = (int32_t)k;
    for (const Pair& q : pairs) {
      if (q.a == nullptr || q.b == nullptr || !q.a->t.defined() || !q.b->t.defined()) continue;
      p.pair[p.pairs++] = {q.a->data(), q.b->data(), q.a->ld, q.b->ld};
    }
    p.out = out.t.data_ptr();
    p.ldo = out.ld;
    return *this;
  }
  Products& bias(const torch::Tensor& b) {
    if (b.defined()) c.bias = b.data_ptr();
    return *this;
  }
  Products& residual(const Matrix& r) {
    if (r.t.defined()) { c.residual = r.data(); c.ld_residual = r.ld; }
    return *this;
  }
  Products& kept(int i, const Matrix& m) {
    if (m.t.defined()) { c.kept[i] = const_cast<void*>(m.data()); c.ld_kept[i] = m.ld; }
    return *this;
  }
  Products& kept(const KeptPlanes& k) {
    if (!k.z.t.defined()) return *this;
    kept(0, k.z).kept(1, k.u);
    if (k.low.defined()) { c.kept_low = k.low.data_ptr(); c.ld_low = k.ld_low; }
    return *this;
  }
  void run(const char* what) {
    if (c.count == 0) return;
    const int64_t bytes = (int64_t)attn_b200_products_scratch_bytes(&c);
    torch::Tensor scratch;
    if (bytes > 0) scratch = fresh({bytes}, at::kByte, like);
    check_rc(attn_b200_products(&c, bytes > 0 ? scratch.data_ptr() : nullptr, at::cuda::getCurrentCUDAStream().stream()), what);
  }
};

struct Elements {
  attn_elements_t e{};
  torch::Tensor like;

  Elements(const torch::Tensor& t, int64_t n, int64_t m, int pass, int64_t activation) : like(t) {
    e.n = (int32_t)n; e.m = (int32_t)m;
    e.dtype = dtype_code(t);
    e.activation = (int32_t)activation;
    e.pass = pass;
  }
  Elements& in(int i, const Matrix& m) {
    if (m.t.defined()) { e.in[i] = m.data(); e.ld_in[i] = m.ld; }
    return *this;
  }
  Elements& kept(int i, const KeptPlanes& k) {
    if (k.low.defined()) { e.kept_low = k.low.data_ptr(); e.ld_low = k.ld_low; }
    return in(i, k.z).in(i + 1, k.u);
  }
  Elements& out(int i, const Matrix& m) {
    e.out[i] = m.t.data_ptr();
    e.ld_out[i] = m.ld;
    return *this;
  }
  void run(const torch::Tensor& sum, const char* what) {
    torch::Tensor scratch;
    if (sum.defined()) {
      e.sum = sum.data_ptr();
      scratch = fresh({(int64_t)attn_b200_elements_scratch_bytes(&e)}, at::kByte, like);
    }
    check_rc(attn_b200_elements(&e, sum.defined() ? scratch.data_ptr() : nullptr, at::cuda::getCurrentCUDAStream().stream()), what);
  }
};

void check_tensors(std::initializer_list<std::pair<const torch::Tensor*, const char*>> all, const torch::Tensor& x) {
  for (const auto& [t, name] : all) {
    if (!t->defined()) continue;
    TORCH_CHECK(t->is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t->device() == x.device(), name, " must be on x's device");
    TORCH_CHECK(t->scalar_type() == x.scalar_type(), name, " must have the dtype of x (", x.scalar_type(), "), got ", t->scalar_type());
  }
}
void check_sizes(const torch::Tensor& x) {
  TORCH_CHECK(x.dim() >= 1, "x must have at least one axis");
  TORCH_CHECK(columns_of(x) > 0, "x must have columns");
  TORCH_CHECK(x.numel() / columns_of(x) <= (1 << 30) && columns_of(x) <= (1 << 28), "x is too large");
}
void check_activation(int64_t a) { TORCH_CHECK(a >= ATTN_ACT_NONE && a <= ATTN_ACT_GELU_TANH, "activation unknown"); }
// An input that there may not be.  The autograd functions count those that there are only, in needs_input_grad and among their results.
typedef c10::optional<torch::Tensor> Maybe;
torch::Tensor or_nothing(const Maybe& t) { return t.has_value() ? *t : torch::Tensor(); }
Maybe maybe(const torch::Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }

void begin_call(const torch::Tensor& x) { raise_if_earlier_call_timed_out(x.device().index()); }

// ---- linear -----------------------------------------------------------------------------------------

void check_linear(const torch::Tensor& x, const torch::Tensor& w, const torch::Tensor& b, const torch::Tensor& r) {
  check_tensors({{&x, "x"}, {&w, "weight"}, {&b, "bias"}, {&r, "residual"}}, x);
  dtype_code(x);
  check_sizes(x);
  TORCH_CHECK(w.dim() == 2 && w.size(1) == columns_of(x), "weight must be [m, k] for x of [..., k]");
  TORCH_CHECK(w.size(0) > 0 && w.size(0) <= (1 << 28), "weight must have rows, 2^28 at most");
  TORCH_CHECK(!b.defined() || (b.dim() == 1 && b.size(0) == w.size(0)), "bias must be [m]");
  TORCH_CHECK(!r.defined() || r.sizes() == at::IntArrayRef(with_columns(x, w.size(0))), "residual must have the shape of the result");
}

// {y, z, copies of x and w}; z, what the activation is applied to, where it is to be kept
variable_list linear_forward(const torch::Tensor& x_in, const torch::Tensor& w_in, const torch::Tensor& b_in, const torch::Tensor& r_in,
                             int64_t activation, bool keep) {
  c10::cuda::CUDAGuard guard(x_in.device());
  begin_call(x_in);
  const int64_t k = columns_of(x_in), m = w_in.size(0), n = x_in.numel() / k;
  const Matrix x = matrix(x_in), w = matrix(w_in), y = result(n, m, x_in);
  Matrix r, z;
  if (r_in.defined()) r = matrix(r_in);
  if (keep) z = result(n, m, x_in, x_in.scalar_type() == at::kFloat ? at::kFloat : at::kHalf);
  const torch::Tensor b = packed(b_in);
  Products(x_in, ATTN_FORM_NT, ATTN_PRODUCT_PLAIN, activation).add(y, n, m, k, {{&x, &w}}).bias(b).residual(r).kept(0, z).run("linear");
  return {handed(y, with_columns(x_in, m)), z.t, copied(x, x_in), copied(w, w_in)};
}

// {dx, dw, db}, undefined where not wanted.  x_copy, w_copy: the forward's, where it made any
variable_list linear_backward(const torch::Tensor& g_in, const torch::Tensor& x_in, const torch::Tensor& w_in, const torch::Tensor& z_in,
                              int64_t activation, bool want_x, bool want_w, bool want_b, const torch::Tensor& x_copy = {}, const torch::Tensor& w_copy = {}) {
  variable_list out(3);
  if (!want_x && !want_w && !want_b) return out;
  c10::cuda::CUDAGuard guard(x_in.device());
  begin_call(x_in);
  const int64_t k = columns_of(x_in), m = w_in.size(0), n = x_in.numel() / k;
  const Matrix g = matrix(g_in);
  Matrix dz = g;
  if (want_b) out[2] = fresh({m}, x_in.scalar_type(), x_in);
  if (activation != ATTN_ACT_NONE) {
    dz = result(n, m, x_in);
    Elements(x_in, n, m, ATTN_ELEMENTS_FIRST, activation).in(0, g).in(1, matrix(z_in)).out(0, dz).run(out[2], "linear backward");
  } else if (want_b) {
    Elements(x_in, n, m, ATTN_ELEMENTS_FIRST, activation).in(0, g).run(out[2], "linear backward");
  }
  if (want_x) {
    const Matrix w = matrix(either(w_copy, w_in)), dx = result(n, k, x_in);
    Products(x_in, ATTN_FORM_NN).add(dx, n, k, m, {{&dz, &w}}).run("linear backward");
    out[0] = handed(dx, x_in.sizes());
  }
  if (want_w) {
    const Matrix x = matrix(either(x_copy, x_in)), dw = result(m, k, x_in);
    Products(x_in, ATTN_FORM_TN).add(dw, m, k, n, {{&dz, &x}}).run("linear backward");
    out[1] = handed(dw, w_in.sizes());
  }
  return out;
}

// Second backward.  With the cotangents (u, uw, ub) of (dx, dw, db), t = u w^T + x uw^T + ub is the tangent of z along them and <g a'(z), t> what is
// differentiated:  to g: t a'(z);  s = g a''(z) t, dz = g a'(z):  to x: s w + dz uw;  to w: s^T x + dz^T u;  to b: the sum of s.
// t and s are rounded to the inputs' type, as gradients between two layers are.
variable_list linear_second(const torch::Tensor& u_in, const torch::Tensor& uw_in, const torch::Tensor& ub_in, const torch::Tensor& g_in,
                            const torch::Tensor& x_in, const torch::Tensor& w_in, const torch::Tensor& z_in, int64_t activation, bool want_b) {
  c10::cuda::CUDAGuard guard(x_in.device());
  begin_call(x_in);
  const int64_t k = columns_of(x_in), m = w_in.size(0), n = x_in.numel() / k;
  const Matrix x = matrix(x_in), w = matrix(w_in), g = matrix(g_in);
  Matrix u, uw, t;
  if (u_in.defined()) u = matrix(u_in);
  if (uw_in.defined()) uw = matrix(uw_in);
  const torch::Tensor ub = packed(ub_in);
  if (u_in.defined() || uw_in.defined()) {
    t = result(n, m, x_in);
    Products(x_in, ATTN_FORM_NT).add(t, n, m, k, {{&u, &w}, {&x, &uw}}).bias(ub).run("linear second backward");
  } else {
    t = result(n, m, x_in);      // in memory of its own: without an activation it is a gradient
    t.t.copy_(ub.unsqueeze(0).expand({n, m}));
  }
  variable_list out(4);      // g, x, w, b
  Matrix dz = g, s;
  if (activation == ATTN_ACT_NONE) {
    out[0] = handed(t, g_in.sizes());
  } else {
    const Matrix gg = result(n, m, x_in);
    dz = result(n, m, x_in);
    s = result(n, m, x_in);
    if (want_b) out[3] = fresh({m}, x_in.scalar_type(), x_in);
    Elements(x_in, n, m, ATTN_ELEMENTS_SECOND, activation).in(0, g).in(1, matrix(z_in)).in(2, t).out(0, gg).out(1, s).out(2, dz)
        .run(out[3], "linear second backward");
    out[0] = handed(gg, g_in.sizes());
  }
  if (s.t.defined() || uw_in.defined()) {
    const Matrix gx = result(n, k, x_in);
    Products(x_in, ATTN_FORM_NN).add(gx, n, k, m, {{&s, &w}, {&dz, &uw}}).run("linear second backward");
    out[1] = handed(gx, x_in.sizes());
  }
  if (s.t.defined() || u_in.defined()) {
    const Matrix gw = result(m, k, x_in);
    Products(x_in, ATTN_FORM_TN).add(gw, m, k, n, {{&s, &x}, {&dz, &u}}).run("linear second backward");
    out[2] = handed(gw, w_in.sizes());
  }
  return out;
}

struct LinearBackward : public torch::autograd::Function<LinearBackward> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& g, const torch::Tensor& x, const torch::Tensor& w, const Maybe& b_in,
                               const Maybe& z_in, int64_t activation) {
    const torch::Tensor b = or_nothing(b_in), z = or_nothing(z_in);
    ctx->set_materialize_grads(false);
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["bias"] = b.defined();
    ctx->save_for_backward({g, x, w, z});
    variable_list out = linear_backward(g, x, w, z, activation, true, true, b.defined());
    if (!b.defined()) out.pop_back();
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list t) {
    variable_list out(6);      // g, x, w, b, z, activation
    const bool bias = ctx->saved_data["bias"].toBool();
    if (!bias) t.emplace_back();
    if (!t[0].defined() && !t[1].defined() && !t[2].defined()) return out;
    TORCH_CHECK(!at::GradMode::is_enabled(), "linear has no third derivative: call the second backward without create_graph");
    const variable_list s = ctx->get_saved_variables();
    variable_list r = linear_second(t[0], t[1], t[2], s[0], s[1], s[2], s[3], ctx->saved_data["activation"].toInt(), bias);
    for (int i = 0; i < 4; ++i) out[i] = std::move(r[i]);
    return out;
  }
};

struct Linear : public torch::autograd::Function<Linear> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& w, const Maybe& b_in, const Maybe& r_in,
                               int64_t activation) {
    const torch::Tensor b = or_nothing(b_in), r = or_nothing(r_in);
    variable_list out = linear_forward(x, w, b, r, activation, activation != ATTN_ACT_NONE);
    ctx->set_materialize_grads(false);
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["residual"] = r.defined();
    ctx->save_for_backward({x, w, b, out[1], out[2], out[3]});
    return out[0];
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(5);      // x, w, b, residual, activation
    if (!g[0].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    const int64_t activation = ctx->saved_data["activation"].toInt();
    TORCH_CHECK(!has_tangent({&g[0], &s[0], &s[1], &s[2]}), "linear has no forward-mode derivative");
    variable_list r = at::GradMode::is_enabled()
                          ? LinearBackward::apply(g[0], s[0], s[1], maybe(s[2]), maybe(s[3]), activation)
                          : linear_backward(g[0], s[0], s[1], s[3], activation, ctx->needs_input_grad(0), ctx->needs_input_grad(1),
                                            s[2].defined() && ctx->needs_input_grad(2), s[4], s[5]);
    for (size_t i = 0; i < r.size(); ++i) out[i] = std::move(r[i]);
    if (ctx->saved_data["residual"].toBool()) out[3] = g[0];
    return out;
  }
};

torch::Tensor linear(const torch::Tensor& x, const torch::Tensor& weight, const Maybe& bias,
                     const Maybe& residual, int64_t activation) {
  const torch::Tensor b = or_nothing(bias), r = or_nothing(residual);
  refuse_transforms({&x, &weight, &b, &r}, "linear");
  check_activation(activation);
  check_linear(x, weight, b, r);
  if (!wants_graph({&x, &weight, &b, &r})) return linear_forward(x, weight, b, r, activation, false)[0];
  return Linear::apply(x, weight, maybe(b), maybe(r), activation);
}

// ---- gated feed-forward block -------------------------------------------------------------------------

void check_gated(const torch::Tensor& x, const torch::Tensor& wg, const torch::Tensor& wu, const torch::Tensor& wd, const torch::Tensor& r) {
  check_tensors({{&x, "x"}, {&wg, "w_gate"}, {&wu, "w_up"}, {&wd, "w_down"}, {&r, "residual"}}, x);
  dtype_code(x);
  check_sizes(x);
  TORCH_CHECK(wg.dim() == 2 && wg.size(1) == columns_of(x) && wu.sizes() == wg.sizes(), "w_gate and w_up must be [f, d] for x of [..., d]");
  TORCH_CHECK(wd.dim() == 2 && wd.size(1) == wg.size(0), "w_down must be [m, f]");
  TORCH_CHECK(wg.size(0) > 0 && wg.size(0) <= (1 << 28) && wd.size(0) > 0 && wd.size(0) <= (1 << 28), "the weights must have rows, 2^28 at most");
  TORCH_CHECK(!r.defined() || r.sizes() == at::IntArrayRef(with_columns(x, wd.size(0))), "residual must have the shape of the result");
}

// {y, z, u, their lower bits, h, copies of x, wg, wu, wd}; z = x wg^T and u = x wu^T where they are to be kept, h = a(z) u
variable_list gated_forward(const torch::Tensor& x_in, const torch::Tensor& wg_in, const torch::Tensor& wu_in, const torch::Tensor& wd_in,
                            const torch::Tensor& r_in, int64_t activation, bool keep) {
  c10::cuda::CUDAGuard guard(x_in.device());
  begin_call(x_in);
  const int64_t d = columns_of(x_in), n = x_in.numel() / d, f = wg_in.size(0), m = wd_in.size(0);
  const Matrix x = matrix(x_in), wg = matrix(wg_in), wu = matrix(wu_in), wd = matrix(wd_in), h = result(n, f, x_in), y = result(n, m, x_in);
  Matrix r;
  KeptPlanes kept;
  if (r_in.defined()) r = matrix(r_in);
  if (keep) kept = kept_planes(n, f, x_in);
  Products inner(x_in, ATTN_FORM_NT, ATTN_PRODUCT_GATED, activation);
  inner.add(h, n, f, d, {{&x, &wg}}).kept(kept);
  inner.c.b2 = wu.data();
  inner.c.ldb2 = wu.ld;
  inner.run("gated_feed_forward");
  Products(x_in, ATTN_FORM_NT).add(y, n, m, f, {{&h, &wd}}).residual(r).run("gated_feed_forward");
  return {handed(y, with_columns(x_in, m)), kept.z.t, kept.u.t, kept.low, h.t, copied(x, x_in), copied(wg, wg_in), copied(wu, wu_in), copied(wd, wd_in)};
}

// {dx, dwg, dwu, dwd}, undefined where not wanted; copies: the forward's of x, wg, wu, wd, or none.  The gradient of h exists in the product's epilogue only, where it becomes those of z and u.
variable_list gated_backward(const torch::Tensor& g_in, const torch::Tensor& x_in, const torch::Tensor& wg_in, const torch::Tensor& wu_in,
                             const torch::Tensor& wd_in, const KeptPlanes& kept, const torch::Tensor& h_in,
                             int64_t activation, bool want_x, bool want_g, bool want_u, bool want_d, const variable_list& copies = variable_list(4)) {
  variable_list out(4);
  if (!want_x && !want_g && !want_u && !want_d) return out;
  c10::cuda::CUDAGuard guard(x_in.device());
  begin_call(x_in);
  const int64_t d = columns_of(x_in), n = x_in.numel() / d, f = wg_in.size(0), m = wd_in.size(0);
  const Matrix g = matrix(g_in), x = matrix(either(copies[0], x_in));
  Matrix dz, du;
  if (want_x || want_g || want_u) {
    const Matrix wd = matrix(either(copies[3], wd_in));
    dz = result(n, f, x_in);
    du = result(n, f, x_in);
    Products inner(x_in, ATTN_FORM_NN, ATTN_PRODUCT_GATED_GRAD, activation);
    inner.add(dz, n, f, m, {{&g, &wd}}).kept(kept);
    inner.c.out2 = du.t.data_ptr();
    inner.c.ldo2 = du.ld;
    inner.run("gated_feed_forward backward");
  }
  if (want_x) {
    const Matrix wg = matrix(either(copies[1], wg_in)), wu = matrix(either(copies[2], wu_in)), dx = result(n, d, x_in);
    Products(x_in, ATTN_FORM_NN).add(dx, n, d, f, {{&dz, &wg}, {&du, &wu}}).run("gated_feed_forward backward");
    out[0] = handed(dx, x_in.sizes());
  }
  Products weights(x_in, ATTN_FORM_TN);
  Matrix dwg, dwu, dwd;
  const Matrix h = matrix(h_in);
  if (want_g) weights.add(dwg = result(f, d, x_in), f, d, n, {{&dz, &x}});
  if (want_u) weights.add(dwu = result(f, d, x_in), f, d, n, {{&du, &x}});
  if (want_d) weights.add(dwd = result(m, f, x_in), m, f, n, {{&g, &h}});
  weights.run("gated_feed_forward backward");
  if (want_g) out[1] = handed(dwg, wg_in.sizes());
  if (want_u) out[2] = handed(dwu, wu_in.sizes());
  if (want_d) out[3] = handed(dwd, wd_in.sizes());
  return out;
}

// Second backward, with the cotangents (ux, ug, uu, ud) of (dx, dwg, dwu, dwd): tangents zt = ux wg^T + x ug^T, ut = ux wu^T + x uu^T and
// ht = a' zt u + a ut, and <g, ht wd^T + h ud^T> is what is differentiated.  With gh = g wd and gh2 = g ud
//   ez = gh a' u, eu = gh a (those of zt, ut);  dz = gh (a'' zt u + a' ut) + gh2 a' u, du = gh a' zt + gh2 a (those of z, u):
//   to g: ht wd^T + h ud^T     to x: dz wg + du wu + ez ug + eu uu     to wg: dz^T x + ez^T ux     to wu: du^T x + eu^T ux     to wd: g^T ht
variable_list gated_second(variable_list t, const torch::Tensor& g_in, const torch::Tensor& x_in, const torch::Tensor& wg_in, const torch::Tensor& wu_in,
                           const torch::Tensor& wd_in, const KeptPlanes& kept, const torch::Tensor& h_in, int64_t activation) {
  c10::cuda::CUDAGuard guard(x_in.device());
  begin_call(x_in);
  const char* what = "gated_feed_forward second backward";
  const int64_t d = columns_of(x_in), n = x_in.numel() / d, f = wg_in.size(0), m = wd_in.size(0);
  const Matrix g = matrix(g_in), x = matrix(x_in), wg = matrix(wg_in), wu = matrix(wu_in), wd = matrix(wd_in), h = matrix(h_in);
  Matrix ux, ug, uu, ud, gh2;
  if (t[0].defined()) ux = matrix(t[0]);
  if (t[1].defined()) ug = matrix(t[1]);
  if (t[2].defined()) uu = matrix(t[2]);
  if (t[3].defined()) ud = matrix(t[3]);
  auto tangent = [&](const Matrix& w, const Matrix& uw) {
    const Matrix r = result(n, f, x_in);
    if (!ux.t.defined() && !uw.t.defined()) r.t.zero_();
    else Products(x_in, ATTN_FORM_NT).add(r, n, f, d, {{&ux, &w}, {&x, &uw}}).run(what);
    return r;
  };
  const Matrix zt = tangent(wg, ug), ut = tangent(wu, uu), gh = result(n, f, x_in);
  Products(x_in, ATTN_FORM_NN).add(gh, n, f, m, {{&g, &wd}}).run(what);
  if (ud.t.defined()) {
    gh2 = result(n, f, x_in);
    Products(x_in, ATTN_FORM_NN).add(gh2, n, f, m, {{&g, &ud}}).run(what);
  }
  const Matrix ht = result(n, f, x_in), ez = result(n, f, x_in), eu = result(n, f, x_in), dz = result(n, f, x_in), du = result(n, f, x_in);
  Elements(x_in, n, f, ATTN_ELEMENTS_GATED_SECOND, activation).in(0, gh).kept(1, kept).in(3, zt).in(4, ut).in(5, gh2)
      .out(0, ht).out(1, ez).out(2, eu).out(3, dz).out(4, du).run(torch::Tensor(), what);
  const Matrix gg = result(n, m, x_in), gx = result(n, d, x_in), gwg = result(f, d, x_in), gwu = result(f, d, x_in), gwd = result(m, f, x_in);
  Products(x_in, ATTN_FORM_NT).add(gg, n, m, f, {{&ht, &wd}, {&h, &ud}}).run(what);
  Products(x_in, ATTN_FORM_NN).add(gx, n, d, f, {{&dz, &wg}, {&du, &wu}, {&ez, &ug}, {&eu, &uu}}).run(what);
  Products(x_in, ATTN_FORM_TN).add(gwg, f, d, n, {{&dz, &x}, {&ez, &ux}}).add(gwu, f, d, n, {{&du, &x}, {&eu, &ux}}).add(gwd, m, f, n, {{&g, &ht}}).run(what);
  return {handed(gg, g_in.sizes()), handed(gx, x_in.sizes()), handed(gwg, wg_in.sizes()), handed(gwu, wu_in.sizes()), handed(gwd, wd_in.sizes())};
}

struct GatedBackward : public torch::autograd::Function<GatedBackward> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& g, const torch::Tensor& x, const torch::Tensor& wg, const torch::Tensor& wu,
                               const torch::Tensor& wd, const torch::Tensor& z, const torch::Tensor& u, const Maybe& low_in, const torch::Tensor& h,
                               int64_t activation) {
    const torch::Tensor low = or_nothing(low_in);
    ctx->set_materialize_grads(false);
    ctx->saved_data["activation"] = activation;
    ctx->save_for_backward({g, x, wg, wu, wd, z, u, low, h});
    return gated_backward(g, x, wg, wu, wd, kept_planes(z, u, low), h, activation, true, true, true, true);
  }

  static variable_list backward(AutogradContext* ctx, variable_list t) {
    variable_list out(10);      // g, x, wg, wu, wd, z, u, low, h, activation
    if (!t[0].defined() && !t[1].defined() && !t[2].defined() && !t[3].defined()) return out;
    TORCH_CHECK(!at::GradMode::is_enabled(), "gated_feed_forward has no third derivative: call the second backward without create_graph");
    const variable_list s = ctx->get_saved_variables();
    variable_list r = gated_second(t, s[0], s[1], s[2], s[3], s[4], kept_planes(s[5], s[6], s[7]), s[8], ctx->saved_data["activation"].toInt());
    for (int i = 0; i < 5; ++i) out[i] = std::move(r[i]);
    return out;
  }
};

struct Gated : public torch::autograd::Function<Gated> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& wg, const torch::Tensor& wu, const torch::Tensor& wd,
                               const Maybe& r_in, int64_t activation) {
    const torch::Tensor r = or_nothing(r_in);
    variable_list out = gated_forward(x, wg, wu, wd, r, activation, true);
    ctx->set_materialize_grads(false);
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["residual"] = r.defined();
    ctx->save_for_backward({x, wg, wu, wd, out[1], out[2], out[3], out[4], out[5], out[6], out[7], out[8]});
    return out[0];
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(6);      // x, wg, wu, wd, residual, activation
    if (!g[0].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    const int64_t activation = ctx->saved_data["activation"].toInt();
    TORCH_CHECK(!has_tangent({&g[0], &s[0], &s[1], &s[2], &s[3]}), "gated_feed_forward has no forward-mode derivative");
    variable_list r = at::GradMode::is_enabled()
                          ? GatedBackward::apply(g[0], s[0], s[1], s[2], s[3], s[4], s[5], maybe(s[6]), s[7], activation)
                          : gated_backward(g[0], s[0], s[1], s[2], s[3], kept_planes(s[4], s[5], s[6]), s[7], activation, ctx->needs_input_grad(0), ctx->needs_input_grad(1),
                                           ctx->needs_input_grad(2), ctx->needs_input_grad(3), {s[8], s[9], s[10], s[11]});
    for (int i = 0; i < 4; ++i) out[i] = std::move(r[i]);
    if (ctx->saved_data["residual"].toBool()) out[4] = g[0];
    return out;
  }
};

torch::Tensor gated_feed_forward(const torch::Tensor& x, const torch::Tensor& w_gate, const torch::Tensor& w_up, const torch::Tensor& w_down,
                                 const Maybe& residual, int64_t activation) {
  const torch::Tensor r = or_nothing(residual);
  refuse_transforms({&x, &w_gate, &w_up, &w_down, &r}, "gated_feed_forward");
  check_activation(activation);
  check_gated(x, w_gate, w_up, w_down, r);
  if (!wants_graph({&x, &w_gate, &w_up, &w_down, &r})) return gated_forward(x, w_gate, w_up, w_down, r, activation, false)[0];
  return Gated::apply(x, w_gate, w_up, w_down, maybe(r), activation);
}

// ---- layer norm -----------------------------------------------------------------------------------------

void check_norm(const torch::Tensor& x, const torch::Tensor& w, const torch::Tensor& b) {
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
  dtype_code(x);
  check_sizes(x);
  TORCH_CHECK(columns_of(x) <= 32768, "x may have 32768 columns at most");
  for (const torch::Tensor* p : {&w, &b}) {
    if (!p->defined()) continue;
    TORCH_CHECK(p->is_cuda() && p->device() == x.device(), "weight and bias must be on x's device");
    TORCH_CHECK(p->dim() == 1 && p->size(0) == columns_of(x), "weight and bias must be [d] for x of [..., d]");
    TORCH_CHECK(p->scalar_type() == x.scalar_type() || p->scalar_type() == at::kFloat, "weight and bias must have the dtype of x or float32");
  }
  TORCH_CHECK(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(), "weight and bias must have one dtype");
}

// the parameters' type; that of x where there are none
at::ScalarType param_type(const torch::Tensor& x, const torch::Tensor& w, const torch::Tensor& b) {
  return w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : x.scalar_type();
}
attn_norm_shape_t norm_shape(const torch::Tensor& x, const Matrix& m, at::ScalarType params, double eps) {
  attn_norm_shape_t s{};
  s.d = (int32_t)columns_of(x);
  s.n = (int32_t)(x.numel() / s.d);
  s.dtype = dtype_code(x);
  s.param_float = params == at::kFloat && s.dtype != ATTN_F32;
  s.eps = (float)eps;
  s.ldx = m.ld;
  return s;
}
const void* pointer(const torch::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* target(const torch::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// {y, mean, rstd}; the last two where they are to be kept
variable_list norm_forward(const torch::Tensor& x_in, const torch::Tensor& w_in, const torch::Tensor& b_in, double eps, bool keep) {
  c10::cuda::CUDAGuard guard(x_in.device());
  begin_call(x_in);
  const Matrix x = matrix(x_in, true);
  const torch::Tensor w = packed(w_in), b = packed(b_in);
  const attn_norm_shape_t s = norm_shape(x_in, x, param_type(x_in, w_in, b_in), eps);
  const torch::Tensor y = fresh(x_in.sizes(), x_in.scalar_type(), x_in);
  torch::Tensor mean, rstd;
  if (keep) {
    mean = fresh({s.n}, at::kFloat, x_in);
    rstd = fresh({s.n}, at::kFloat, x_in);
  }
  check_rc(attn_b200_layer_norm(&s, x.data(), pointer(w), pointer(b), y.data_ptr(), static_cast<float*>(target(mean)), static_cast<float*>(target(rstd)),
                                at::cuda::getCurrentCUDAStream().stream()),
           "layer_norm");
  return {y, mean, rstd};
}

// {dx, dw, db}, undefined where not wanted
variable_list norm_backward(const torch::Tensor& g_in, const torch::Tensor& x_in, const torch::Tensor& w_in, const torch::Tensor& mean,
                            const torch::Tensor& rstd, at::ScalarType params, double eps, bool want_x, bool want_w, bool want_b) {
  variable_list out(3);
  if (!want_x && !want_w && !want_b) return out;
  c10::cuda::CUDAGuard guard(x_in.device());
  begin_call(x_in);
  const Matrix x = matrix(x_in, true), g = matrix(g_in, true);
  const torch::Tensor w = packed(w_in);
  attn_norm_shape_t s = norm_shape(x_in, x, params, eps);
  s.ldg = g.ld;
  torch::Tensor scratch;
  if (want_x) out[0] = fresh(x_in.sizes(), x_in.scalar_type(), x_in);
  if (want_w) out[1] = fresh({s.d}, params, x_in);
  if (want_b) out[2] = fresh({s.d}, params, x_in);
  if (want_w || want_b) scratch = fresh({(int64_t)attn_b200_layer_norm_backward_scratch_bytes(&s)}, at::kByte, x_in);
  check_rc(attn_b200_layer_norm_backward(&s, x.data(), pointer(w), g.data(), mean.data_ptr<float>(), rstd.data_ptr<float>(), target(out[0]), target(out[1]),
                                         target(out[2]), target(scratch), at::cuda::getCurrentCUDAStream().stream()),
           "layer_norm backward");
  return out;
}

// {gg, gx, gw}
variable_list norm_second(const torch::Tensor& u_in, const torch::Tensor& uw_in, const torch::Tensor& ub_in, const torch::Tensor& g_in,
                          const torch::Tensor& x_in, const torch::Tensor& w_in, const torch::Tensor& mean, const torch::Tensor& rstd, at::ScalarType params,
                          double eps) {
  c10::cuda::CUDAGuard guard(x_in.device());
  begin_call(x_in);
  const Matrix x = matrix(x_in, true), g = matrix(g_in, true);
  Matrix u;
  if (u_in.defined()) u = matrix(u_in, true);
  const torch::Tensor w = packed(w_in), uw = packed(uw_in), ub = packed(ub_in);
  attn_norm_shape_t s = norm_shape(x_in, x, params, eps);
  s.ldg = g.ld;
  s.ldu = u.ld;
  variable_list out(3);
  out[0] = fresh(g_in.sizes(), x_in.scalar_type(), x_in);
  out[1] = fresh(x_in.sizes(), x_in.scalar_type(), x_in);
  torch::Tensor scratch;
  if (w_in.defined()) {
    out[2] = fresh({s.d}, params, x_in);
    scratch = fresh({(int64_t)attn_b200_layer_norm_backward_scratch_bytes(&s)}, at::kByte, x_in);
  }
  check_rc(attn_b200_layer_norm_second_backward(&s, x.data(), pointer(w), g.data(), mean.data_ptr<float>(), rstd.data_ptr<float>(),
                                                u.t.defined() ? u.data() : nullptr, pointer(uw), pointer(ub), out[0].data_ptr(), out[1].data_ptr(),
                                                target(out[2]), target(scratch), at::cuda::getCurrentCUDAStream().stream()),
           "layer_norm second backward");
  return out;
}

struct LayerNormBackward : public torch::autograd::Function<LayerNormBackward> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& g, const torch::Tensor& x, const Maybe& w_in, const Maybe& b_in,
                               const torch::Tensor& mean, const torch::Tensor& rstd, int64_t params, double eps) {
    const torch::Tensor w = or_nothing(w_in), b = or_nothing(b_in);
    ctx->set_materialize_grads(false);
    ctx->saved_data["params"] = params;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["weight"] = w.defined();
    ctx->saved_data["bias"] = b.defined();
    ctx->save_for_backward({g, x, w, mean, rstd});
    variable_list r = norm_backward(g, x, w, mean, rstd, (at::ScalarType)params, eps, true, w.defined(), b.defined()), out = {r[0]};
    if (w.defined()) out.push_back(r[1]);
    if (b.defined()) out.push_back(r[2]);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list t) {
    variable_list out(8);      // g, x, w, b, mean, rstd, params, eps
    size_t next = 1;
    const torch::Tensor uw = ctx->saved_data["weight"].toBool() ? t[next++] : torch::Tensor();
    const torch::Tensor ub = ctx->saved_data["bias"].toBool() ? t[next++] : torch::Tensor();
    if (!t[0].defined() && !uw.defined() && !ub.defined()) return out;
    TORCH_CHECK(!at::GradMode::is_enabled(), "layer_norm has no third derivative: call the second backward without create_graph");
    const variable_list s = ctx->get_saved_variables();
    variable_list r = norm_second(t[0], uw, ub, s[0], s[1], s[2], s[3], s[4], (at::ScalarType)ctx->saved_data["params"].toInt(), ctx->saved_data["eps"].toDouble());
    for (int i = 0; i < 3; ++i) out[i] = std::move(r[i]);
    return out;
  }
};

struct LayerNorm : public torch::autograd::Function<LayerNorm> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& x, const Maybe& w_in, const Maybe& b_in, double eps) {
    const torch::Tensor w = or_nothing(w_in), b = or_nothing(b_in);
    variable_list out = norm_forward(x, w, b, eps, true);
    ctx->set_materialize_grads(false);
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["params"] = (int64_t)param_type(x, w, b);
    ctx->save_for_backward({x, w, b, out[1], out[2]});
    return out[0];
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(4);      // x, w, b, eps
    if (!g[0].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    const int64_t params = ctx->saved_data["params"].toInt();
    const double eps = ctx->saved_data["eps"].toDouble();
    const bool w = s[1].defined(), b = s[2].defined();
    TORCH_CHECK(!has_tangent({&g[0], &s[0], &s[1], &s[2]}), "layer_norm has no forward-mode derivative");
    if (!at::GradMode::is_enabled()) {
      variable_list r = norm_backward(g[0], s[0], s[1], s[3], s[4], (at::ScalarType)params, eps, ctx->needs_input_grad(0), w && ctx->needs_input_grad(1),
                                      b && ctx->needs_input_grad(w ? 2 : 1));
      for (int i = 0; i < 3; ++i) out[i] = std::move(r[i]);
      return out;
    }
    variable_list r = LayerNormBackward::apply(g[0], s[0], maybe(s[1]), maybe(s[2]), s[3], s[4], params, eps);
    size_t next = 0;
    out[0] = r[next++];
    if (w) out[1] = r[next++];
    if (b) out[2] = r[next++];
    return out;
  }
};

torch::Tensor layer_norm(const torch::Tensor& x, const Maybe& weight, const Maybe& bias, double eps) {
  const torch::Tensor w = or_nothing(weight), b = or_nothing(bias);
  refuse_transforms({&x, &w, &b}, "layer_norm");
  check_norm(x, w, b);
  if (!wants_graph({&x, &w, &b})) return norm_forward(x, w, b, eps, false)[0];
  return LayerNorm::apply(x, maybe(w), maybe(b), eps);
}

}  // namespace

void register_layers(pybind11::module& m) {
  m.def("layer_norm", &layer_norm, "layer norm over the last axis, twice differentiable", py::arg("x"), py::arg("weight") = py::none(),
        py::arg("bias") = py::none(), py::arg("eps") = 1e-5, py::call_guard<py::gil_scoped_release>());
  m.def("linear", &linear, "activation(x weight^T + bias) + residual, twice differentiable", py::arg("x"), py::arg("weight"), py::arg("bias") = py::none(),
        py::arg("residual") = py::none(), py::arg("activation") = 0, py::call_guard<py::gil_scoped_release>());
  m.def("gated_feed_forward", &gated_feed_forward, "(activation(x w_gate^T) * (x w_up^T)) w_down^T + residual, twice differentiable", py::arg("x"),
        py::arg("w_gate"), py::arg("w_up"), py::arg("w_down"), py::arg("residual") = py::none(), py::arg("activation") = 1,
        py::call_guard<py::gil_scoped_release>());
}

}  // namespace ext
