// C ABI of the packed-batch attention (include/attn_b200.h): argument checks and dispatch.
#include "capi_common.h"
#include "packed_launch.h"

#include <cmath>
#include <cstring>

namespace {

using namespace attn;
using capi::aligned16;
using capi::fail;

constexpr int kMaxRows = 1 << 30;

int check_shape(const attn_packed_shape_t* s) {
  if (s == nullptr) return fail(ATTN_EINVAL, "shape is null");
  if (s->dtype != ATTN_F16 && s->dtype != ATTN_BF16 && s->dtype != ATTN_F32)
    return fail(ATTN_EUNSUPPORTED, "dtype %d: expected ATTN_F16, ATTN_BF16 or ATTN_F32", s->dtype);
  if (s->n_tok < 0 || s->n_tok > kMaxRows) return fail(ATTN_EINVAL, "n_tok must be in [0, 2^30] (got %d)", s->n_tok);
  if (s->n_seq < 0 || s->n_seq > kMaxRows) return fail(ATTN_EINVAL, "n_seq must be in [0, 2^30] (got %d)", s->n_seq);
  if (s->kv_heads <= 0 || s->q_heads <= 0 || s->q_heads % s->kv_heads != 0)
    return fail(ATTN_EINVAL, "q_heads must be a positive multiple of kv_heads (got %d and %d)", s->q_heads, s->kv_heads);
  if (s->D <= 0 || s->D % 16 != 0) return fail(ATTN_EINVAL, "D must be a positive multiple of 16 (got %d)", s->D);
  if (s->D > 128) return fail(ATTN_EUNSUPPORTED, "unsupported head dimension D=%d (maximum 128)", s->D);
  if (s->window_size < 0) return fail(ATTN_EINVAL, "window_size must be >= 0");
  const long long units = plan_tiles(s->n_tok, s->n_seq) * s->q_heads * (s->dtype == ATTN_F32 ? 4 : 1);
  if (units > 0x7fffffffLL) return fail(ATTN_ETOOLARGE, "n_tok, n_seq and q_heads make %lld tiles", units);
  return ATTN_OK;
}

PackedGeometry make_geometry(const attn_packed_shape_t* s, const int32_t* plan) {
  PackedGeometry g;
  g.BH = s->q_heads;
  g.N_q = g.N_kv = s->n_tok;
  g.D = s->D;
  g.qi_base = g.ki_base = 0;
  g.window = s->window_size > (1 << 30) ? (1 << 30) : s->window_size;
  g.mask_mode = 0;
  g.head_group = 1;
  g.beside = 0;
  g.split = 1;
  g.scale = 1.0f / sqrtf((float)s->D);
  g.scale_log2e = g.scale * kLog2e;
  g.cap = (int)plan_tiles(s->n_tok, s->n_seq);
  g.row_tiles = reinterpret_cast<const PackedTile*>(plan + kPlanHeader);
  g.col_tiles = g.row_tiles + g.cap;
  g.pair_tiles = g.col_tiles + g.cap;
  g.pair_cap = (int)plan_pairs(s->n_tok, s->n_seq);
  g.q_heads = s->q_heads;
  g.kv_heads = s->kv_heads;
  g.n_seq = s->n_seq;
  g.group = s->q_heads / s->kv_heads;
  return g;
}

PackedLayout make_layout(const attn_packed_shape_t* s) {
  PackedLayout lay;
  for (int i = 0; i < PI_COUNT; ++i) lay.of[i] = PackedStrides{s->row_stride[i], s->head_stride[i]};
  return lay;
}

// the inputs' strides: dense in the fp32 family, multiples of 16 bytes that a tensor map takes else
int check_strides(const attn_packed_shape_t* s, int inputs) {
  for (int i = 0; i < inputs; ++i) {
    const long long heads = i == PI_K || i == PI_V ? s->kv_heads : s->q_heads;
    if (s->dtype == ATTN_F32) {
      if (s->row_stride[i] != heads * s->D || s->head_stride[i] != s->D) return fail(ATTN_EUNSUPPORTED, "float32 inputs must be dense [n_tok, heads, D]");
    } else if (s->row_stride[i] <= 0 || s->head_stride[i] <= 0 || s->row_stride[i] % 8 != 0 || s->head_stride[i] % 8 != 0 ||
               s->row_stride[i] >= (1LL << 39) || s->head_stride[i] >= (1LL << 39)) {
      return fail(ATTN_EINVAL, "strides must be positive multiples of 8 elements below 2^39");
    }
  }
  return ATTN_OK;
}

#define REQUIRE(p)                                                                          \
  do {                                                                                      \
    if ((p) == nullptr) return fail(ATTN_EINVAL, #p " is null");                            \
    if (!aligned16(p)) return fail(ATTN_EINVAL, #p " is not 16-byte aligned");              \
  } while (0)

int run(int op, const attn_packed_shape_t* s, const int32_t* plan, Tensors& t, void* stream) {
  const int rc = capi::begin(&t.status);
  if (rc != ATTN_OK) return rc;
  const PackedGeometry g = make_geometry(s, plan);
  const char* why = nullptr;
  int launches = 0;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const cudaError_t e = s->dtype == ATTN_F32 ? launch_packed_simt(op, g, t, cs, &launches)
                                             : launch_packed_tc(op, s->dtype, g, t, make_layout(s), cs, &launches, &why);
  return capi::done(e, "packed attention launch failed", why, launches);
}

}  // namespace

extern "C" {

size_t attn_b200_packed_plan_ints(int32_t n_tok, int32_t n_seq) {
  if (n_tok < 0 || n_seq < 0 || n_tok > kMaxRows || n_seq > kMaxRows) return 0;
  return (size_t)plan_ints(n_tok, n_seq);
}

int attn_b200_packed_plan(const int32_t* cu_seqlens, int32_t n_tok, int32_t n_seq, int32_t* plan, void* stream) {
  if (n_tok < 0 || n_seq < 0 || n_tok > kMaxRows || n_seq > kMaxRows) return fail(ATTN_EINVAL, "n_tok and n_seq must be in [0, 2^30]");
  if (plan_tiles(n_tok, n_seq) > 0x7fffffffLL) return fail(ATTN_ETOOLARGE, "too many tiles");
  if (cu_seqlens == nullptr || (reinterpret_cast<uintptr_t>(cu_seqlens) & 3u) != 0) return fail(ATTN_EINVAL, "cu_seqlens is null or misaligned");
  REQUIRE(plan);
  unsigned int* status = nullptr;
  const int rc = capi::begin(&status);
  if (rc != ATTN_OK) return rc;
  return capi::done(launch_packed_plan(cu_seqlens, plan, n_tok, n_seq, static_cast<cudaStream_t>(stream)), "plan launch failed", nullptr, 1);
}

int attn_b200_packed_forward(const attn_packed_shape_t* shape, const int32_t* plan, const void* Q, const void* K, const void* V, void* O,
                             float* L, void* stream) {
  int rc = check_shape(shape);
  if (rc == ATTN_OK) rc = check_strides(shape, 3);
  if (rc != ATTN_OK) return rc;
  if (shape->n_tok == 0) return capi::done(cudaSuccess, "", nullptr, 0);
  REQUIRE(plan); REQUIRE(Q); REQUIRE(K); REQUIRE(V); REQUIRE(O);
  if (L == nullptr) return fail(ATTN_EINVAL, "L is null");
  Tensors t;
  memset(&t, 0, sizeof(t));
  t.Q = Q; t.K = K; t.V = V; t.out_O = O; t.out_L = L;
  return run(OP_FORWARD, shape, plan, t, stream);
}

size_t attn_b200_packed_backward_scratch_bytes(const attn_packed_shape_t* s) {
  if (s == nullptr || s->n_tok < 0 || s->q_heads < 0) return 0;
  return sizeof(float) * (size_t)s->n_tok * s->q_heads;
}

int attn_b200_packed_backward(const attn_packed_shape_t* shape, const int32_t* plan, const void* dO, const void* Q, const void* K,
                              const void* V, const void* O, const float* L, void* dQ, void* dK, void* dV, float* scratch, void* stream) {
  int rc = check_shape(shape);
  if (rc == ATTN_OK) rc = check_strides(shape, 4);
  if (rc != ATTN_OK) return rc;
  if (shape->n_tok == 0) return capi::done(cudaSuccess, "", nullptr, 0);
  REQUIRE(plan); REQUIRE(dO); REQUIRE(Q); REQUIRE(K); REQUIRE(V); REQUIRE(O); REQUIRE(dQ); REQUIRE(dK); REQUIRE(dV);
  if (L == nullptr || scratch == nullptr) return fail(ATTN_EINVAL, "L or scratch is null");
  Tensors t;
  memset(&t, 0, sizeof(t));
  t.dO = dO; t.Q = Q; t.K = K; t.V = V; t.O = O; t.L = L;
  t.out_dQ = dQ; t.out_dK = dK; t.out_dV = dV;
  t.Dv = scratch;
  return run(OP_BACKWARD, shape, plan, t, stream);
}

}  // extern "C"
