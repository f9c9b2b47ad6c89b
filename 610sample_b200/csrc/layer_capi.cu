// C ABI of a layer's operators (include/attn_b200.h): argument checks, launches.
#include "capi_common.h"
#include "layer_launch.h"
#include "layer_norm.cuh"

namespace {

using namespace attn;
using namespace attn::layer;
using capi::aligned16;
using capi::fail;

constexpr int kMostRows = 1 << 30;

bool known_type(int dtype) { return dtype == ATTN_F16 || dtype == ATTN_BF16 || dtype == ATTN_F32; }
int size_of(int dtype) { return dtype == ATTN_F32 ? 4 : 2; }

// a matrix of a product: on the tensor cores what a tensor map takes
int check_matrix(const char* name, const void* p, int64_t ld, int cols, int dtype) {
  if (p == nullptr) return fail(ATTN_EINVAL, "%s is null", name);
  if (ld < cols || ld > (int64_t(1) << 36)) return fail(ATTN_EINVAL, "%s: rows are %lld elements apart, and %d long", name, (long long)ld, cols);
  if (dtype == ATTN_F32) {
    if (reinterpret_cast<uintptr_t>(p) % 4 != 0) return fail(ATTN_EINVAL, "%s is not 4-byte aligned", name);
  } else if (!aligned16(p) || ld % 8 != 0) {
    return fail(ATTN_EINVAL, "%s: half types need a 16-byte aligned base and rows a multiple of 8 elements apart", name);
  }
  return ATTN_OK;
}

int check_rows(const char* name, const void* p, int64_t ld, int m, int dtype) {
  if (p == nullptr) return fail(ATTN_EINVAL, "%s is null", name);
  if (ld < m || ld > (int64_t(1) << 36)) return fail(ATTN_EINVAL, "%s: rows are %lld elements apart, and %d long", name, (long long)ld, m);
  if (reinterpret_cast<uintptr_t>(p) % size_of(dtype) != 0) return fail(ATTN_EINVAL, "%s is not aligned", name);
  return ATTN_OK;
}

int check_low(const void* p, int64_t ld, int cols) {
  if (p == nullptr || reinterpret_cast<uintptr_t>(p) % 32 != 0 || ld % 32 != 0 || ld < cols || ld > (int64_t(1) << 36))
    return fail(ATTN_EINVAL, "kept_low: 32-byte aligned rows of at least %d bytes are needed", cols);
  return ATTN_OK;
}

int check_products(const attn_products_t* c, bool pointers) {
  if (c == nullptr) return fail(ATTN_EINVAL, "call is null");
  if (!known_type(c->dtype)) return fail(ATTN_EUNSUPPORTED, "dtype %d: expected ATTN_F16, ATTN_BF16 or ATTN_F32", c->dtype);
  if (c->form < ATTN_FORM_NT || c->form > ATTN_FORM_TN) return fail(ATTN_EINVAL, "form %d unknown", c->form);
  if (c->kind < ATTN_PRODUCT_PLAIN || c->kind > ATTN_PRODUCT_GATED_GRAD) return fail(ATTN_EINVAL, "kind %d unknown", c->kind);
  if (c->activation < ATTN_ACT_NONE || c->activation > ATTN_ACT_GELU_TANH) return fail(ATTN_EINVAL, "activation %d unknown", c->activation);
  if (c->count < 1 || c->count > ATTN_PRODUCT_COUNT) return fail(ATTN_EINVAL, "count must be in [1, %d] (got %d)", ATTN_PRODUCT_COUNT, c->count);
  int factors = 0;
  for (int i = 0; i < c->count; ++i) {
    const attn_product_t& p = c->product[i];
    if (p.rows < 0 || p.cols < 0 || p.k < 0 || p.rows > kMostRows || p.cols > kMostRows || p.k > kMostRows)
      return fail(ATTN_EINVAL, "rows, cols and k must be in [0, 2^30] (got %d, %d, %d)", p.rows, p.cols, p.k);
    if (p.pairs < 1 || p.pairs > ATTN_PRODUCT_PAIRS) return fail(ATTN_EINVAL, "pairs must be in [1, %d] (got %d)", ATTN_PRODUCT_PAIRS, p.pairs);
    if ((long long)p.k * p.pairs > kMostRows) return fail(ATTN_EINVAL, "k is too large for so many pairs");
    factors += p.pairs;
  }
  if (factors > kMaxFactors) return fail(ATTN_EINVAL, "more than %d pairs in all", kMaxFactors);
  const bool plain = c->kind == ATTN_PRODUCT_PLAIN;
  if (plain && c->form != ATTN_FORM_NT && c->kept[0] != nullptr) return fail(ATTN_EINVAL, "z is kept in the form NT only");
  if (c->count > 1 && (!plain || c->bias != nullptr || c->residual != nullptr || c->kept[0] != nullptr || c->activation != ATTN_ACT_NONE))
    return fail(ATTN_EINVAL, "a call of several results takes nothing behind them");
  const attn_product_t& first = c->product[0];
  if (c->kind == ATTN_PRODUCT_GATED && (c->form != ATTN_FORM_NT || first.pairs != 1)) return fail(ATTN_EINVAL, "a gated product is of form NT, with one pair");
  if (c->kind == ATTN_PRODUCT_GATED_GRAD && c->form != ATTN_FORM_NN) return fail(ATTN_EINVAL, "a gated gradient is of form NN");
  if (!plain && (c->bias != nullptr || c->residual != nullptr)) return fail(ATTN_EINVAL, "bias and residual go with plain products");
  if (c->kind == ATTN_PRODUCT_GATED && (c->kept[0] == nullptr) != (c->kept[1] == nullptr)) return fail(ATTN_EINVAL, "z and u are kept together");
  // a result without a sum is 0 only where nothing follows
  if (first.k == 0 && first.rows > 0 && first.cols > 0 &&
      (!plain || c->bias != nullptr || c->residual != nullptr || c->kept[0] != nullptr || c->activation != ATTN_ACT_NONE))
    return fail(ATTN_EINVAL, "k must be at least 1 (got 0)");
  if (!pointers) return ATTN_OK;
  for (int i = 0; i < c->count; ++i) {
    const attn_product_t& p = c->product[i];
    if (p.rows == 0 || p.cols == 0) continue;
    int rc = check_matrix("out", p.out, p.ldo, p.cols, c->dtype);
    if (rc != ATTN_OK) return rc;
    for (int q = 0; q < p.pairs && p.k > 0; ++q) {
      rc = check_matrix("a", p.pair[q].a, p.pair[q].lda, c->form == ATTN_FORM_TN ? p.rows : p.k, c->dtype);
      if (rc == ATTN_OK) rc = check_matrix("b", p.pair[q].b, p.pair[q].ldb, c->form == ATTN_FORM_NT ? p.k : p.cols, c->dtype);
      if (rc != ATTN_OK) return rc;
    }
  }
  if (first.rows == 0 || first.cols == 0) return ATTN_OK;
  int rc = ATTN_OK;
  if (c->bias != nullptr && reinterpret_cast<uintptr_t>(c->bias) % size_of(c->dtype) != 0) rc = fail(ATTN_EINVAL, "bias is not aligned");
  if (rc == ATTN_OK && c->residual != nullptr) rc = check_rows("residual", c->residual, c->ld_residual, first.cols, c->dtype);
  if (rc == ATTN_OK && c->kind == ATTN_PRODUCT_GATED) rc = check_matrix("b2", c->b2, c->ldb2, first.k, c->dtype);
  const bool both = c->kind == ATTN_PRODUCT_GATED_GRAD || (c->kind == ATTN_PRODUCT_GATED && c->kept[0] != nullptr);
  for (int q = 0; q < 2 && rc == ATTN_OK; ++q)
    if (both || (plain && q == 0 && c->kept[0] != nullptr))  rc = check_matrix("kept", c->kept[q], c->ld_kept[q], first.cols, c->dtype);
  if (rc == ATTN_OK && c->kind == ATTN_PRODUCT_GATED_GRAD) rc = check_matrix("out2", c->out2, c->ldo2, first.cols, c->dtype);
  if (rc == ATTN_OK && both && c->dtype != ATTN_F32) rc = check_low(c->kept_low, c->ld_low, first.cols);
  return rc;
}

size_t parts_bytes(const attn_products_t& c) { return c.dtype == ATTN_F32 ? simt_parts_bytes(c) : few_rows(c) ? 0 : tc_parts_bytes(c); }

int inputs_of(int pass, int act) { return pass == ATTN_ELEMENTS_FIRST ? (act == ATTN_ACT_NONE ? 1 : 2) : pass == ATTN_ELEMENTS_SECOND ? 3 : 5; }
int outputs_of(int pass, int act) { return pass == ATTN_ELEMENTS_FIRST ? (act == ATTN_ACT_NONE ? 0 : 1) : pass == ATTN_ELEMENTS_SECOND ? 3 : 5; }

int check_elements(const attn_elements_t* e, bool pointers) {
  if (e == nullptr) return fail(ATTN_EINVAL, "call is null");
  if (!known_type(e->dtype)) return fail(ATTN_EUNSUPPORTED, "dtype %d: expected ATTN_F16, ATTN_BF16 or ATTN_F32", e->dtype);
  if (e->pass < ATTN_ELEMENTS_FIRST || e->pass > ATTN_ELEMENTS_GATED_SECOND) return fail(ATTN_EINVAL, "pass %d unknown", e->pass);
  if (e->activation < ATTN_ACT_NONE || e->activation > ATTN_ACT_GELU_TANH) return fail(ATTN_EINVAL, "activation %d unknown", e->activation);
  if (e->n < 0 || e->m < 0 || e->n > kMostRows || e->m > kMostRows) return fail(ATTN_EINVAL, "n and m must be in [0, 2^30] (got %d, %d)", e->n, e->m);
  if (e->sum != nullptr && e->pass == ATTN_ELEMENTS_GATED_SECOND) return fail(ATTN_EINVAL, "this pass has no sum");
  if (!pointers || e->n == 0 || e->m == 0) return ATTN_OK;
  const int in = inputs_of(e->pass, e->activation), out = outputs_of(e->pass, e->activation);
  int rc = ATTN_OK;
  for (int i = 0; i < 6 && rc == ATTN_OK; ++i)
    if (i < in || (e->pass == ATTN_ELEMENTS_GATED_SECOND && e->in[i] != nullptr)) rc = check_rows("an input", e->in[i], e->ld_in[i], e->m, e->dtype);
  for (int i = 0; i < out && rc == ATTN_OK; ++i) rc = check_rows("a result", e->out[i], e->ld_out[i], e->m, e->dtype);
  if (rc == ATTN_OK && e->pass == ATTN_ELEMENTS_GATED_SECOND && e->dtype != ATTN_F32) rc = check_low(e->kept_low, e->ld_low, e->m);
  return rc;
}

int check_norm(const attn_norm_shape_t* s) {
  if (s == nullptr) return fail(ATTN_EINVAL, "shape is null");
  if (!known_type(s->dtype)) return fail(ATTN_EUNSUPPORTED, "dtype %d: expected ATTN_F16, ATTN_BF16 or ATTN_F32", s->dtype);
  if (s->n < 0 || s->n > kMostRows) return fail(ATTN_EINVAL, "n must be in [0, 2^30] (got %d)", s->n);
  if (s->d < 1 || s->d > 32768) return fail(ATTN_EINVAL, "d must be in [1, 32768] (got %d)", s->d);
  return ATTN_OK;
}

unsigned groups_of(const NormPlan& p) { return p.tpr >= kNormThreads ? 1u : p.tpr == 96 ? 3u : (unsigned)(kNormThreads / p.tpr); }
// rows of a backward pass go to so many CTAs, which each leave a row of partial sums
unsigned backward_ctas(const attn_norm_shape_t* s, const NormPlan& p) {
  const unsigned want = ((unsigned)s->n + groups_of(p) - 1) / groups_of(p), most = p.tpr > kNormThreads ? kSms : 2 * kSms;      // that run at a time
  return want < most ? want : most;
}

NormArgs norm_args(const attn_norm_shape_t* s, const void* x, const void* w) {
  NormArgs a = {};
  a.n = s->n; a.d = s->d;
  a.param_float = s->param_float != 0;
  a.eps = s->eps;
  a.x = x; a.w = w;
  a.ldx = s->ldx; a.ldg = s->ldg; a.ldu = s->ldu;
  return a;
}
bool wide_rows(const attn_norm_shape_t* s, const void* p, int64_t ld) { return p == nullptr || (aligned16(p) && ld * size_of(s->dtype) % 16 == 0); }
bool wide_norm(const attn_norm_shape_t* s, std::initializer_list<const void*> dense) {
  bool wide = s->d % 8 == 0;
  for (const void* p : dense) wide = wide && (p == nullptr || aligned16(p));
  return wide;
}

}  // namespace

extern "C" {

size_t attn_b200_products_scratch_bytes(const attn_products_t* call) { return check_products(call, false) == ATTN_OK ? parts_bytes(*call) : 0; }

int attn_b200_products(const attn_products_t* call, void* scratch, void* stream) {
  int rc = check_products(call, true);
  if (rc != ATTN_OK) return rc;
  const size_t bytes = parts_bytes(*call);
  if (bytes > 0 && (scratch == nullptr || !aligned16(scratch))) return fail(ATTN_EINVAL, "scratch is null or not 16-byte aligned");
  unsigned int* status = nullptr;
  rc = capi::begin(&status);
  if (rc != ATTN_OK) return rc;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  const char* why = nullptr;
  int launches = 0;
  const size_t size = size_of(call->dtype);
  for (int i = 0; i < call->count && e == cudaSuccess; ++i) {      // sums of nothing
    const attn_product_t& p = call->product[i];
    if (p.k == 0 && p.rows > 0 && p.cols > 0) e = cudaMemset2DAsync(p.out, p.ldo * size, 0, p.cols * size, p.rows, cs);
  }
  if (e == cudaSuccess) {
    float* const parts = static_cast<float*>(scratch);
    e = call->dtype == ATTN_F32 ? simt_products(*call, parts, cs, &launches)
        : few_rows(*call)       ? few_products(*call, cs, &launches)
                                : tc_products(*call, parts, status, cs, &launches, &why);
  }
  return capi::done(e, "products launch failed", why, launches);
}

size_t attn_b200_elements_scratch_bytes(const attn_elements_t* e) {
  return check_elements(e, false) == ATTN_OK ? (size_t)element_chunks(e->n, e->m) * e->m * sizeof(float) : 0;
}

int attn_b200_elements(const attn_elements_t* e, void* scratch, void* stream) {
  int rc = check_elements(e, true);
  if (rc != ATTN_OK) return rc;
  unsigned int* status = nullptr;
  rc = capi::begin(&status);
  if (rc != ATTN_OK) return rc;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  cudaError_t err = cudaSuccess;
  int launches = 0;
  if (e->m > 0 && e->n == 0 && e->sum != nullptr) err = cudaMemsetAsync(e->sum, 0, (size_t)e->m * size_of(e->dtype), cs);
  if (e->m > 0 && e->n > 0) {
    if (e->sum != nullptr && (scratch == nullptr || !aligned16(scratch))) return fail(ATTN_EINVAL, "scratch is null or not 16-byte aligned");
    if (e->sum == nullptr && outputs_of(e->pass, e->activation) == 0) return capi::done(cudaSuccess, "", nullptr, 0);
    ElementArgs a = {};
    a.n = e->n; a.m = e->m;
    const int in = inputs_of(e->pass, e->activation), out = outputs_of(e->pass, e->activation);
    for (int i = 0; i < 6; ++i)
      if (i < in || e->pass == ATTN_ELEMENTS_GATED_SECOND) { a.in[i] = e->in[i]; a.ld_in[i] = e->ld_in[i]; }
    for (int i = 0; i < out; ++i) { a.out[i] = e->out[i]; a.ld_out[i] = e->ld_out[i]; }
    a.low = e->kept_low;
    a.ld_low = e->ld_low;
    a.partial = e->sum != nullptr ? static_cast<float*>(scratch) : nullptr;
    err = launch_elementwise(a, e->pass, e->activation, e->dtype, cs);
    ++launches;
    if (e->sum != nullptr && err == cudaSuccess) {
      err = launch_sum_rows(a.partial, element_chunks(e->n, e->m), 1, e->m, e->dtype, e->sum, nullptr, cs);
      ++launches;
    }
  }
  return capi::done(err, "elements launch failed", nullptr, launches);
}

int attn_b200_copy_rows(const void* src, int64_t lds, void* dst, int64_t ldd, int32_t rows, int32_t cols, int32_t dtype, void* stream) {
  if (!known_type(dtype)) return fail(ATTN_EUNSUPPORTED, "dtype %d: expected ATTN_F16, ATTN_BF16 or ATTN_F32", dtype);
  if (rows < 0 || cols < 0 || rows > kMostRows || cols > kMostRows) return fail(ATTN_EINVAL, "rows and cols must be in [0, 2^30] (got %d, %d)", rows, cols);
  int rc = ATTN_OK;
  if (rows > 0 && cols > 0) {
    rc = check_rows("src", src, lds, cols, dtype);
    if (rc == ATTN_OK) rc = check_rows("dst", dst, ldd, cols, dtype);
  }
  if (rc != ATTN_OK) return rc;
  unsigned int* status = nullptr;
  rc = capi::begin(&status);
  if (rc != ATTN_OK) return rc;
  if (rows == 0 || cols == 0) return capi::done(cudaSuccess, "", nullptr, 0);
  return capi::done(launch_copy_rows(src, lds, dst, ldd, rows, cols, size_of(dtype), static_cast<cudaStream_t>(stream)), "copy launch failed", nullptr, 1);
}

int attn_b200_layer_norm(const attn_norm_shape_t* s, const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, void* stream) {
  int rc = check_norm(s);
  if (rc != ATTN_OK) return rc;
  if (s->n > 0) rc = check_rows("x", x, s->ldx, s->d, s->dtype);
  if (rc == ATTN_OK && s->n > 0) rc = check_rows("y", y, s->d, s->d, s->dtype);
  if (rc != ATTN_OK) return rc;
  if ((mean == nullptr) != (rstd == nullptr)) return fail(ATTN_EINVAL, "mean and rstd go together");
  unsigned int* status = nullptr;
  rc = capi::begin(&status);
  if (rc != ATTN_OK) return rc;
  if (s->n == 0) return capi::done(cudaSuccess, "", nullptr, 0);
  const NormPlan p = plan_norm(s->d, wide_norm(s, {w, b, y}) && wide_rows(s, x, s->ldx), false);
  NormArgs a = norm_args(s, x, w);
  a.b = b;
  a.y = y;
  a.mean = mean; a.rstd = rstd;
  const unsigned ctas = ((unsigned)s->n + groups_of(p) - 1) / groups_of(p);
  return capi::done(launch_norm_forward(p, a, s->dtype, ctas, static_cast<cudaStream_t>(stream)), "layer norm launch failed", nullptr, 1);
}

size_t attn_b200_layer_norm_backward_scratch_bytes(const attn_norm_shape_t* s) {
  if (check_norm(s) != ATTN_OK) return 0;
  return (size_t)backward_ctas(s, plan_norm(s->d, true, true)) * 2 * s->d * sizeof(float);
}

static int norm_backward(const attn_norm_shape_t* s, NormArgs a, bool wide, int order, void* sum0, void* sum1, void* scratch, void* stream) {
  unsigned int* status = nullptr;
  const int rc = capi::begin(&status);
  if (rc != ATTN_OK) return rc;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const bool sums = sum0 != nullptr || sum1 != nullptr;
  const int type = s->param_float ? ATTN_F32 : s->dtype;
  cudaError_t e = cudaSuccess;
  if (s->n == 0) {
    for (void* p : {sum0, sum1})
      if (p != nullptr && e == cudaSuccess) e = cudaMemsetAsync(p, 0, (size_t)s->d * size_of(type), cs);
    return capi::done(e, "memset failed", nullptr, 0);
  }
  const NormPlan p = plan_norm(s->d, wide, true);
  const unsigned ctas = backward_ctas(s, p);
  a.partial = sums ? static_cast<float*>(scratch) : nullptr;
  e = order == 1 ? launch_norm_first(p, a, s->dtype, ctas, cs) : launch_norm_second(p, a, s->dtype, ctas, cs);
  if (sums && e == cudaSuccess) e = launch_sum_rows(a.partial, (int)ctas, order == 1 ? 2 : 1, s->d, type, sum0, sum1, cs);
  return capi::done(e, "layer norm launch failed", nullptr, sums ? 2 : 1);
}

static int check_norm_backward(const attn_norm_shape_t* s, const void* x, const void* g, const float* mean, const float* rstd, bool sums, const void* scratch) {
  int rc = check_norm(s);
  if (rc != ATTN_OK || s->n == 0) return rc;
  rc = check_rows("x", x, s->ldx, s->d, s->dtype);
  if (rc == ATTN_OK) rc = check_rows("g", g, s->ldg, s->d, s->dtype);
  if (rc != ATTN_OK) return rc;
  if (mean == nullptr || rstd == nullptr) return fail(ATTN_EINVAL, "mean or rstd is null");
  if (sums && (scratch == nullptr || !aligned16(scratch))) return fail(ATTN_EINVAL, "scratch is null or not 16-byte aligned");
  return ATTN_OK;
}

int attn_b200_layer_norm_backward(const attn_norm_shape_t* s, const void* x, const void* w, const void* g, const float* mean, const float* rstd,
                                  void* dx, void* dw, void* db, void* scratch, void* stream) {
  const int rc = check_norm_backward(s, x, g, mean, rstd, dw != nullptr || db != nullptr, scratch);
  if (rc != ATTN_OK) return rc;
  if (s->n > 0 && dx == nullptr && dw == nullptr && db == nullptr) return fail(ATTN_EINVAL, "no gradient is asked for");
  NormArgs a = norm_args(s, x, w);
  a.g = g;
  a.gx = dx;
  a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
  return norm_backward(s, a, wide_norm(s, {w, dx}) && wide_rows(s, x, s->ldx) && wide_rows(s, g, s->ldg), 1, dw, db, scratch, stream);
}

int attn_b200_layer_norm_second_backward(const attn_norm_shape_t* s, const void* x, const void* w, const void* g, const float* mean, const float* rstd,
                                         const void* u, const void* uw, const void* ub, void* gg, void* gx, void* gw, void* scratch, void* stream) {
  int rc = check_norm_backward(s, x, g, mean, rstd, gw != nullptr, scratch);
  if (rc == ATTN_OK && u != nullptr && s->n > 0) rc = check_rows("u", u, s->ldu, s->d, s->dtype);
  if (rc != ATTN_OK) return rc;
  if (s->n > 0 && gg == nullptr && gx == nullptr && gw == nullptr) return fail(ATTN_EINVAL, "no gradient is asked for");
  NormArgs a = norm_args(s, x, w);
  a.g = g;
  a.u = u; a.uw = uw; a.ub = ub;
  a.y = gg; a.gx = gx;
  a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
  const bool wide = wide_norm(s, {w, uw, ub, gg, gx}) && wide_rows(s, x, s->ldx) && wide_rows(s, g, s->ldg) && wide_rows(s, u, s->ldu);
  return norm_backward(s, a, wide, 2, gw, nullptr, scratch, stream);
}

}  // extern "C"
