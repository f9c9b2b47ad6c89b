// C ABI of the linear cross entropy (include/attn_b200.h): argument checks, the plan of the backward's pieces, launches.
#include "attn_common.cuh"
#include "capi_common.h"
#include "lce_launch.h"

namespace {

using namespace attn;
using namespace attn::lce;
using capi::aligned16;
using capi::fail;

int check_shape(const attn_lce_shape_t* s) {
  if (s == nullptr) return fail(ATTN_EINVAL, "shape is null");
  if (s->dtype != ATTN_F16 && s->dtype != ATTN_BF16 && s->dtype != ATTN_F32)
    return fail(ATTN_EUNSUPPORTED, "dtype %d: expected ATTN_F16, ATTN_BF16 or ATTN_F32", s->dtype);
  if (s->n < 0 || s->n > (1 << 30)) return fail(ATTN_EINVAL, "n must be in [0, 2^30] (got %d)", s->n);
  if (s->d <= 0 || s->d > (1 << 20)) return fail(ATTN_EINVAL, "d must be in [1, 2^20] (got %d)", s->d);
  if (s->V <= 0 || s->V > (1 << 30)) return fail(ATTN_EINVAL, "V must be in [1, 2^30] (got %d)", s->V);
  if (s->reduction < RED_NONE || s->reduction > RED_MEAN) return fail(ATTN_EINVAL, "reduction %d unknown", s->reduction);
  return ATTN_OK;
}

// half types whose rows a tensor map takes
bool on_tensor_cores(const attn_lce_shape_t* s) { return s->dtype != ATTN_F32 && s->d % 8 == 0; }

size_t up(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

// G, the gradient with respect to the logits, exists for a piece of the vocabulary at a time.  Larger pieces make fewer and fuller
// products (dW's tiles are rows of the piece) and fewer passes over dx's float sums: 16384 x 768 x 32000 takes 3.74 ms with 68 MB, 3.14 with
// 135, 2.83 with 206, 2.76 with 256, 2.70 with 420, 2.66 with 560 (4099 x 2048 x 100003: 5.79, 5.54, 5.40, 5.42, 5.34, 5.33).  So 512 MB, pieces
// of equal size, whole tiles.
constexpr long long kPieceBytes = 512ll << 20;

struct BackwardPlan {
  bool tc;
  int cols, pieces;               // columns of a piece (the last may have fewer)
  int dx_splits;                  // CUDA cores: most shares of k of any piece
  size_t coef, scale, G, x, acc_dx, acc_dw, parts, total;      // offsets in bytes
};

int piece_cols(const BackwardPlan& b, const attn_lce_shape_t* s, int i) { return i + 1 < b.pieces ? b.cols : s->V - (b.pieces - 1) * b.cols; }

BackwardPlan plan_backward(const attn_lce_shape_t* s, bool dx, bool dw) {
  BackwardPlan b;
  b.tc = on_tensor_cores(s);
  const long long size = s->dtype == ATTN_F32 ? 4 : 2, g_size = b.tc ? 2 : 4, n = s->n > 0 ? s->n : 1;
  long long most = kPieceBytes / (n * g_size) / 256 * 256;
  if (most < 1024) most = 1024;
  long long pieces = (s->V + most - 1) / most;
  const long long cols = ((s->V + pieces - 1) / pieces + 255) / 256 * 256;
  pieces = (s->V + cols - 1) / cols;
  b.cols = (int)(cols < s->V ? cols : s->V);
  b.pieces = (int)pieces;
  b.dx_splits = b.tc ? 1 : simt_splits(n, s->d, b.cols);      // the first piece's, the longest in k
  size_t dw_floats = 0, parts = 0;
  for (int i = 0; i < b.pieces; i += b.pieces > 1 ? b.pieces - 1 : 1) {      // all but the last are alike
    const int c = piece_cols(b, s, i);
    if (b.tc) {
      for (const size_t bytes : {dx ? tc_parts_bytes(n, s->d, c) : 0, dw ? tc_parts_bytes(c, s->d, n) : 0}) parts = bytes > parts ? bytes : parts;
    } else {
      const int sp = simt_splits(c, s->d, n);
      if (sp > 1 && (size_t)sp * c * s->d > dw_floats) dw_floats = (size_t)sp * c * s->d;
    }
  }
  size_t at = 0;
  auto take = [&](size_t bytes) { const size_t here = at; at += up(bytes); return here; };
  b.coef = take((size_t)n * 4);
  b.scale = take(16);
  b.G = take((size_t)n * ((b.cols + 7) / 8 * 8) * g_size);
  b.x = take(dw ? (size_t)n * s->d * size : 0);
  b.acc_dx = take(dx && (b.pieces > 1 || b.dx_splits > 1) ? (size_t)b.dx_splits * n * s->d * 4 : 0);
  b.acc_dw = take(dw ? dw_floats * 4 : 0);
  b.parts = take(parts);
  b.total = at;
  return b;
}

#define REQUIRE(p)                                                                          \
  do {                                                                                      \
    if ((p) == nullptr) return fail(ATTN_EINVAL, #p " is null");                            \
    if (!aligned16(p)) return fail(ATTN_EINVAL, #p " is not 16-byte aligned");              \
  } while (0)

Problem make_problem(const attn_lce_shape_t* s, const void* x, const void* w, const int64_t* targets) {
  Problem p;
  p.n = s->n; p.d = s->d; p.V = s->V;
  p.dtype = s->dtype;
  p.ignore_index = s->ignore_index;
  p.x = x; p.w = w;
  p.targets = targets;
  p.status = nullptr;
  return p;
}

struct ForwardScratch { size_t partial, logit, total; int tiles; };
ForwardScratch plan_forward(const attn_lce_shape_t* s) {
  ForwardScratch f;
  f.tiles = on_tensor_cores(s) ? tc_tiles(s->V) : simt_tiles(s->V);
  f.partial = 0;
  f.logit = up((size_t)f.tiles * s->n * sizeof(Partial));
  f.total = f.logit + up((size_t)s->n * 4);
  return f;
}

}  // namespace

extern "C" {

size_t attn_b200_linear_ce_forward_scratch_bytes(const attn_lce_shape_t* s) { return check_shape(s) == ATTN_OK ? plan_forward(s).total : 0; }

size_t attn_b200_linear_ce_backward_scratch_bytes(const attn_lce_shape_t* s, int32_t want_dx, int32_t want_dw) {
  return check_shape(s) == ATTN_OK ? plan_backward(s, want_dx != 0, want_dw != 0).total : 0;
}

int attn_b200_linear_ce_forward(const attn_lce_shape_t* shape, const void* x, const void* w, const int64_t* targets, float* loss, float* lse,
                                float* value, float* counted, void* scratch, void* stream) {
  int rc = check_shape(shape);
  if (rc != ATTN_OK) return rc;
  if (shape->reduction != RED_NONE && (value == nullptr || counted == nullptr)) return fail(ATTN_EINVAL, "value or counted is null");
  if (shape->n > 0) {
    REQUIRE(x); REQUIRE(w); REQUIRE(scratch);
    if (targets == nullptr || loss == nullptr || lse == nullptr) return fail(ATTN_EINVAL, "targets, loss or lse is null");
    if (reinterpret_cast<uintptr_t>(targets) % 8 != 0) return fail(ATTN_EINVAL, "targets is not 8-byte aligned");
  }
  Problem p = make_problem(shape, x, w, targets);
  if (p.n == 0 && shape->reduction == RED_NONE) return capi::done(cudaSuccess, "", nullptr, 0);
  rc = capi::begin(&p.status);
  if (rc != ATTN_OK) return rc;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  const char* why = nullptr;
  int launches = 0;
  if (p.n > 0) {
    const ForwardScratch f = plan_forward(shape);
    char* base = static_cast<char*>(scratch);
    const Scores sc{reinterpret_cast<Partial*>(base + f.partial), reinterpret_cast<float*>(base + f.logit), f.tiles};
    if (on_tensor_cores(shape)) {
      e = tc_scores(p, sc, cs, &launches, &why);
    } else {
      e = simt_scores(p, sc, cs);
      ++launches;
    }
    if (e == cudaSuccess) e = launch_finish(p, sc, loss, lse, cs);
    ++launches;
  }
  if (e == cudaSuccess && shape->reduction != RED_NONE) {
    e = launch_total(p, loss, shape->reduction, value, counted, cs);
    ++launches;
  }
  return capi::done(e, "linear cross entropy launch failed", why, launches);
}

int attn_b200_linear_ce_backward(const attn_lce_shape_t* shape, const void* x, const void* w, const int64_t* targets, const float* lse,
                                 const float* grad, const float* counted, void* dx, void* dw, void* scratch, void* stream) {
  int rc = check_shape(shape);
  if (rc != ATTN_OK) return rc;
  if (dx == nullptr && dw == nullptr) return fail(ATTN_EINVAL, "neither gradient is asked for");
  if (dx != nullptr && !aligned16(dx)) return fail(ATTN_EINVAL, "dx is not 16-byte aligned");
  if (dw != nullptr && !aligned16(dw)) return fail(ATTN_EINVAL, "dw is not 16-byte aligned");
  Problem p = make_problem(shape, x, w, targets);
  if (p.n > 0) {
    REQUIRE(x); REQUIRE(w); REQUIRE(scratch);
    if (targets == nullptr || lse == nullptr || grad == nullptr) return fail(ATTN_EINVAL, "targets, lse or grad is null");
    if (reinterpret_cast<uintptr_t>(targets) % 8 != 0) return fail(ATTN_EINVAL, "targets is not 8-byte aligned");
    if (shape->reduction == RED_MEAN && counted == nullptr) return fail(ATTN_EINVAL, "counted is null");
  }
  rc = capi::begin(&p.status);
  if (rc != ATTN_OK) return rc;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const size_t size = shape->dtype == ATTN_F32 ? 4 : 2;
  if (p.n == 0) return capi::done(dw == nullptr ? cudaSuccess : cudaMemsetAsync(dw, 0, size * p.V * p.d, cs), "memset failed", nullptr, 0);
  const BackwardPlan b = plan_backward(shape, dx != nullptr, dw != nullptr);
  char* base = static_cast<char*>(scratch);
  const Coefficients c{reinterpret_cast<float*>(base + b.coef), reinterpret_cast<float*>(base + b.scale)};
  float* const acc_dx = reinterpret_cast<float*>(base + b.acc_dx);
  float* const acc_dw = reinterpret_cast<float*>(base + b.acc_dw);
  void* const G = base + b.G;
  const char* why = nullptr;
  int launches = 0;
  cudaError_t e = cudaSuccess;
  auto then = [&](auto&& launch) {
    if (e != cudaSuccess) return;
    e = launch();
    ++launches;
  };
  then([&] { return launch_coefficients(p, grad, counted, shape->reduction, c, cs); });
  if (dw != nullptr) then([&] { return launch_counted_rows(p, base + b.x, cs); });
  for (int i = 0; i < b.pieces; ++i) {
    Piece piece;
    piece.first = i * b.cols;
    piece.cols = piece_cols(b, shape, i);
    piece.ld = (b.cols + 7) / 8 * 8;
    piece.is_first = i == 0;
    piece.is_last = i + 1 == b.pieces;
    if (b.tc) {
      float* const parts = reinterpret_cast<float*>(base + b.parts);
      if (e == cudaSuccess) e = tc_piece_grad(p, piece, lse, c, G, cs, &launches, &why);
      if (dw != nullptr && e == cudaSuccess) e = tc_piece_dw(p, piece, c, G, base + b.x, parts, dw, cs, &launches, &why);
      if (dx != nullptr && e == cudaSuccess) e = tc_piece_dx(p, piece, c, G, parts, acc_dx, dx, cs, &launches, &why);
      continue;
    }
    then([&] { return simt_piece_grad(p, piece, lse, c, (float*)G, cs); });
    if (dw != nullptr) {
      const int sp = simt_splits(piece.cols, p.d, p.n);
      then([&] { return simt_piece_dw(p, piece, c, (const float*)G, base + b.x, sp, acc_dw, dw, cs); });
      if (sp > 1)
        then([&] { return launch_sum_splits(acc_dw, sp, (long long)piece.cols * p.d, c.scale, static_cast<char*>(dw) + size * piece.first * p.d, p.dtype, cs); });
    }
    if (dx != nullptr) {
      int sp = simt_splits(p.n, p.d, piece.cols);
      if (sp > b.dx_splits) sp = b.dx_splits;
      then([&] { return simt_piece_dx(p, piece, c, (const float*)G, sp, b.dx_splits > 1, acc_dx, dx, cs); });
    }
  }
  if (dx != nullptr && b.dx_splits > 1)
    then([&] { return launch_sum_splits(acc_dx, b.dx_splits, (long long)p.n * p.d, c.scale, dx, p.dtype, cs); });
  return capi::done(e, "linear cross entropy launch failed", why, launches);
}

}  // extern "C"
