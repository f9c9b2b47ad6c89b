// Norm and rotation of Q and K rows of a packed batch, in one pass over both: per (token, head) RMS normalisation with a learned weight,
// then rotation of the pairs (x[2i], x[2i + 1]) by the table's angle for pair i at the token's position.  Positions are given
// per token, on one or several axes (time, height, width); `section` says which pairs turn with which axis.
//
//   n = x r, r = (mean(x^2) + eps)^-1/2, y = n w, out = rotation(y)
//   gy = rotation^T(g), gw = sum gy n, gx = r gy w - x (r^3 / D) sum_k gy_k w_k x_k           (no weight: no norm, gx = gy)
//
// Everything in fp32 from the loads to the one rounding of a result.  Bound by HBM: x is read and the result written once, in
// the backward x and g are read and gx written.  A group of 8 (D <= 64) or 16 lanes owns a token, a lane eight consecutive elements (one
// 16-byte access for the half types); the group walks over four heads of its token with their loads in flight, and fetches the
// angles, which all heads share, once.  q and k are read where they lie in the projection's result.  The weights' gradients are
// summed per lane over all a CTA walks through, then across the CTA, then over the CTAs by a second launch, in a fixed order.
// 30011 rows, 40 heads of 128, three axes, fp16: forward 117 us (5.3 TB/s), backward 191 (4.8): 24 warps an SM issue in 62 and 70 % of the
// cycles and else wait for loads.  float32, 16384 rows, 24 heads of 64: 40 us (5.0 TB/s) and 62 (4.9).  Packed fp32 instructions took the backward from 202 to 197 (replayed graphs), but the forward from 119 to 127; not kept.
#include "capi_common.h"
#include "attn_common.cuh"
#include "tc_common.cuh"

#include <cstring>

namespace attn {
namespace rope {

using tc::from_l2;

constexpr int kThreads = 256, kMaxAxes = 4;
constexpr int kForwardHeads = 4, kBackwardHeads = 2;      // of a batch

struct Side {                    // q or k
  const void *x, *g, *w;         // w: null for no norm
  void* out;                     // forward: the result; backward: gx; dense [n_tok, heads, D]
  long long row, head;           // strides of x in elements
  long long g_row, g_head;       // and of g
  int heads, w_float;            // w_float: the weight is float32 beside half-precision rows
};

struct Args {
  Side side[2];
  const float* table;            // [table_rows][D / 2][cos, sin]
  const void* positions;         // [axes][n_tok]
  long long axis_stride;
  int positions64;
  int table_rows, n_tok, D, axes;
  int section_end[kMaxAxes];     // pairs [section_end[a - 1], section_end[a]) turn with axis a
  float eps;
};

template <typename T> __device__ __forceinline__ void widen8(const uint4& q, float (&v)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f;
    if constexpr (tc::Pack<T>::kIsBf16) f = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    else f = tc::Pack<T>::unpack(w[i]);
    v[2 * i] = f.x; v[2 * i + 1] = f.y;
  }
}

// eight consecutive elements as they lie in memory (raw), and as floats
template <typename T> struct Eight {
  uint4 q;
  __device__ __forceinline__ void zero() { q = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void load(const T* p) { q = from_l2(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void load_some(const T* p, int n) {
    zero();
    const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
    uint32_t w[4] = {};
    for (int i = 0; i < n; ++i) w[i >> 1] |= (uint32_t)s[i] << (16 * (i & 1));
    q = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const { widen8<T>(q, v); }
  static __device__ __forceinline__ void store(T* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(tc::Pack<T>::pack(v[0], v[1]), tc::Pack<T>::pack(v[2], v[3]), tc::Pack<T>::pack(v[4], v[5]), tc::Pack<T>::pack(v[6], v[7]));
  }
};
template <> struct Eight<float> {
  float4 a, b;
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void load(const float* p) { a = from_l2(reinterpret_cast<const float4*>(p)); b = from_l2(reinterpret_cast<const float4*>(p) + 1); }
  __device__ __forceinline__ void load_some(const float* p, int n) {
    float v[8] = {};
    for (int i = 0; i < n; ++i) v[i] = p[i];
    a = make_float4(v[0], v[1], v[2], v[3]);
    b = make_float4(v[4], v[5], v[6], v[7]);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const { v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w; }
  static __device__ __forceinline__ void store(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
};

// WIDE: D and the strides are multiples of 8 and everything is 16-byte aligned; else element by element, `n` of them
template <typename T, bool WIDE> __device__ __forceinline__ void load8(Eight<T>& e, const T* p, int n) {
  if constexpr (WIDE) e.load(p);
  else e.load_some(p, n);
}
template <typename T, bool WIDE> __device__ __forceinline__ void store8(T* p, const float (&v)[8], int n) {
  if constexpr (WIDE) Eight<T>::store(p, v);
  else
    for (int i = 0; i < n; ++i) p[i] = Elem<T>::from_float(v[i]);
}

// this lane's eight weights; 1 where there is no norm
template <typename T, bool WIDE>
__device__ __forceinline__ void load_weight(const Side& s, int col, int n, float (&w)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = 1.f;
  if (s.w == nullptr || n <= 0) return;
  if (s.w_float) {
    const float* p = static_cast<const float*>(s.w) + col;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) w[e] = p[e];
  } else if (WIDE) {
    Eight<T> e;
    e.load(static_cast<const T*>(s.w) + col);
    e.get(w);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) w[e] = Elem<T>::to_float(static_cast<const T*>(s.w)[col + e]);
  }
}

// (cos, sin) of this lane's four pairs; not a number for a position outside of the table
__device__ __forceinline__ void load_angles(const Args& a, int tok, int pair0, int pairs, float2 (&cs)[4]) {
  if (a.axes == 1) {
    const long long pos = a.positions64 ? from_l2(static_cast<const long long*>(a.positions) + tok) : from_l2(static_cast<const int*>(a.positions) + tok);
    const bool in = pos >= 0 && pos < a.table_rows;
    const float2* row = reinterpret_cast<const float2*>(a.table) + (in ? pos : 0) * pairs + pair0;
#pragma unroll
    for (int i = 0; i < 4; ++i) cs[i] = in && pair0 + i < pairs ? from_l2(row + i) : make_float2(NAN, NAN);
    return;
  }
  int axis = 0, row = -1, row_axis = -1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    cs[i] = make_float2(NAN, NAN);
    const int p = pair0 + i;
    if (p >= pairs) continue;
    while (axis + 1 < a.axes && p >= a.section_end[axis]) ++axis;
    if (axis != row_axis) {
      const long long at = axis * a.axis_stride + tok;
      const long long pos = a.positions64 ? from_l2(static_cast<const long long*>(a.positions) + at) : from_l2(static_cast<const int*>(a.positions) + at);
      row = pos >= 0 && pos < a.table_rows ? (int)pos : -1;
      row_axis = axis;
    }
    if (row >= 0) cs[i] = from_l2(reinterpret_cast<const float2*>(a.table) + (size_t)row * pairs + p);
  }
}

template <int G> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Heads are taken a few at a time, those of q first: a batch's side, its first head and how many heads it has.
struct Batch { int which, h0, heads; };
template <int H>
__device__ __forceinline__ Batch batch_at(const Args& a, int b) {
  const int q_batches = (a.side[0].heads + H - 1) / H, which = b >= q_batches;
  const int h0 = (which ? b - q_batches : b) * H;
  return {which, h0, min(H, a.side[which].heads - h0)};
}
__host__ __device__ inline int batches_of(long long q_heads, long long k_heads, int H) { return (int)((q_heads + H - 1) / H + (k_heads + H - 1) / H); }

// A group of G lanes owns a token and walks over its share of the batches, the next one on its way meanwhile; the angles are
// fetched once.  `shares` CTAs have the same tokens.
template <typename T, int G, bool WIDE>
__global__ void __launch_bounds__(kThreads)
forward_kernel(const __grid_constant__ Args a, const int shares) {
  tc::pdl_wait();
  tc::pdl_trigger();
  const int share = (int)(blockIdx.x % (unsigned)shares), batches = batches_of(a.side[0].heads, a.side[1].heads, kForwardHeads);
  const int first = (int)((long long)batches * share / shares), last = (int)((long long)batches * (share + 1) / shares);
  const int sub = threadIdx.x % G, col = sub * 8, n = min(8, a.D - col);
  const int tok = (int)(blockIdx.x / (unsigned)shares) * (kThreads / G) + threadIdx.x / G;
  const bool on = tok < a.n_tok && n > 0;      // the shuffles need every lane of a warp
  const float inv_d = 1.f / (float)a.D;
  auto load = [&](const Batch& b, Eight<T> (&raw)[kForwardHeads]) {
    const Side& s = a.side[b.which];
    const T* p = static_cast<const T*>(s.x) + tok * s.row + b.h0 * s.head + col;
#pragma unroll
    for (int i = 0; i < kForwardHeads; ++i) {
      raw[i].zero();
      if (on && i < b.heads) load8<T, WIDE>(raw[i], p + i * s.head, n);
    }
  };
  Batch cur = batch_at<kForwardHeads>(a, first);
  Eight<T> raw[kForwardHeads], next[kForwardHeads];
  load(cur, raw);
  float2 cs[4] = {};
  if (on) load_angles(a, tok, sub * 4, a.D >> 1, cs);
  int side = -1;
  float w[8];
  for (int b = first; b < last; ++b) {
    const Batch now = cur;
    const bool more = b + 1 < last;
    if (more) {
      cur = batch_at<kForwardHeads>(a, b + 1);
      load(cur, next);
    }
    const Side& s = a.side[now.which];
    if (now.which != side) {
      side = now.which;
      load_weight<T, WIDE>(s, col, on ? n : 0, w);
    }
    const bool norm = s.w != nullptr;      // uniform over the CTA
    T* out = static_cast<T*>(s.out) + ((size_t)tok * s.heads + now.h0) * a.D + col;
#pragma unroll
    for (int i = 0; i < kForwardHeads; ++i) {
      float v[8];
      raw[i].get(v);
      if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(v[e], v[e], ss);
        const float r = rsqrtf(fmaf(group_sum<G>(ss), inv_d, a.eps));
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= r * w[e];
      }
      if (on && i < now.heads) {
        float o[8];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          o[2 * p] = v[2 * p] * cs[p].x - v[2 * p + 1] * cs[p].y;
          o[2 * p + 1] = v[2 * p] * cs[p].y + v[2 * p + 1] * cs[p].x;
        }
        store8<T, WIDE>(out + (size_t)i * a.D, o, n);
      }
    }
    if (more) {
#pragma unroll
      for (int i = 0; i < kForwardHeads; ++i) raw[i] = next[i];
    }
  }
}

// The tasks, tokens x shares of the batches, are dealt to the CTAs in turn.
template <typename T, int G, bool WIDE>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 3 : 2)
backward_kernel(const __grid_constant__ Args a, const int shares, float* partial) {      // partial: [2][CTAs][D], null where no weight's gradient is wanted
  constexpr int kTok = kThreads / G;
  __shared__ __align__(16) float sums[kThreads * 8];
  tc::pdl_wait();
  tc::pdl_trigger();
  const int sub = threadIdx.x % G, col = sub * 8, n = min(8, a.D - col), batches = batches_of(a.side[0].heads, a.side[1].heads, kBackwardHeads);
  const unsigned tasks = (unsigned)((a.n_tok + kTok - 1) / kTok) * (unsigned)shares;
  const float inv_d = 1.f / (float)a.D;
  float w[8], acc[2][8] = {};
  int side = -1;
  for (unsigned task = blockIdx.x; task < tasks; task += gridDim.x) {
    const int share = (int)(task % (unsigned)shares), tok = (int)(task / (unsigned)shares) * kTok + threadIdx.x / G;
    const int first = (int)((long long)batches * share / shares), last = (int)((long long)batches * (share + 1) / shares);
    const bool on = tok < a.n_tok && n > 0;
    float2 cs[4] = {};
    for (int b = first; b < last; ++b) {
      const Batch now = batch_at<kBackwardHeads>(a, b);
      const Side& s = a.side[now.which];
      const bool norm = s.w != nullptr;
      Eight<T> rx[kBackwardHeads], rg[kBackwardHeads];
      {
        const T* px = static_cast<const T*>(s.x) + tok * s.row + now.h0 * s.head + col;
        const T* pg = static_cast<const T*>(s.g) + tok * s.g_row + now.h0 * s.g_head + col;
#pragma unroll
        for (int i = 0; i < kBackwardHeads; ++i) {
          rx[i].zero();
          rg[i].zero();
          if (on && i < now.heads) {
            load8<T, WIDE>(rg[i], pg + i * s.g_head, n);
            if (norm) load8<T, WIDE>(rx[i], px + i * s.head, n);
          }
        }
      }
      if (b == first && on) load_angles(a, tok, sub * 4, a.D >> 1, cs);
      if (now.which != side) {
        side = now.which;
        load_weight<T, WIDE>(s, col, n, w);
      }
      T* out = static_cast<T*>(s.out) + ((size_t)tok * s.heads + now.h0) * a.D + col;
#pragma unroll
      for (int i = 0; i < kBackwardHeads; ++i) {
        float gv[8], xv[8], gy[8];
        rg[i].get(gv);
        rx[i].get(xv);
        // a row whose gradient is 0 gives 0, also where the row (of no sequence, say) is infinite or not a number, or its
        // position is outside of the table
        bool any = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) any |= gv[e] != 0.f;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          gy[2 * p] = gv[2 * p] * cs[p].x + gv[2 * p + 1] * cs[p].y;
          gy[2 * p + 1] = gv[2 * p + 1] * cs[p].x - gv[2 * p] * cs[p].y;
        }
        if (norm) {      // uniform: every lane takes part in the shuffles
          float ss = 0.f, dot = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            ss = fmaf(xv[e], xv[e], ss);
            if (WIDE || e < n) dot = fmaf(gy[e] * w[e], xv[e], dot);      // pairs beyond D have no angle
          }
          ss = group_sum<G>(ss);
          dot = group_sum<G>(dot);
          const unsigned lanes = __ballot_sync(0xffffffffu, any);
          any = ((lanes >> ((threadIdx.x & 31) / G * G)) & ((1u << G) - 1u)) != 0u;
          if (on && i < now.heads && any) {
            const float r = rsqrtf(fmaf(ss, inv_d, a.eps)), k = r * r * r * inv_d * dot;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float add = (WIDE || e < n) ? gy[e] * (xv[e] * r) : 0.f;
              if (now.which) acc[1][e] += add; else acc[0][e] += add;
              gy[e] = r * gy[e] * w[e] - k * xv[e];
            }
          }
        }
        if (!any) {
#pragma unroll
          for (int e = 0; e < 8; ++e) gy[e] = 0.f;
        }
        if (on && i < now.heads) store8<T, WIDE>(out + (size_t)i * a.D, gy, n);
      }
    }
  }
  if (partial == nullptr) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
    float4* mine = reinterpret_cast<float4*>(sums + (threadIdx.x / G) * (8 * G) + col);
    mine[0] = make_float4(acc[which][0], acc[which][1], acc[which][2], acc[which][3]);
    mine[1] = make_float4(acc[which][4], acc[which][5], acc[which][6], acc[which][7]);
    __syncthreads();
    if (threadIdx.x < a.D) {
      float t = 0.f;
#pragma unroll 8
      for (int i = 0; i < kTok; ++i) t += sums[i * (8 * G) + threadIdx.x];
      partial[((size_t)which * gridDim.x + blockIdx.x) * a.D + threadIdx.x] = t;
    }
  }
}

// gw[c] = sum of the rows of `partial`: 32 columns per CTA, 32 interleaved row sums per column; blockIdx.y: q, k
template <typename T>
__global__ void __launch_bounds__(1024)
weight_grad_kernel(const float* partial, void* gw0, void* gw1, int rows, int D, int float0, int float1) {
  __shared__ float sums[32][33];
  tc::pdl_wait();
  tc::pdl_trigger();
  void* gw = blockIdx.y ? gw1 : gw0;
  if (gw == nullptr) return;
  const int c = blockIdx.x * 32 + threadIdx.x % 32, r0 = threadIdx.x / 32;
  float s = 0.f;
  if (c < D)
#pragma unroll 4
    for (int r = r0; r < rows; r += 32) s += from_l2(partial + ((size_t)blockIdx.y * rows + r) * D + c);
  sums[r0][threadIdx.x % 32] = s;
  __syncthreads();
  s = sums[threadIdx.x % 32][r0];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int at = blockIdx.x * 32 + r0;
  if (threadIdx.x % 32 != 0 || at >= D) return;
  if (blockIdx.y ? float1 : float0) static_cast<float*>(gw)[at] = s;
  else static_cast<T*>(gw)[at] = Elem<T>::from_float(s);
}

static long long token_blocks(long long n_tok, int D) {
  const long long per = kThreads / (D <= 64 ? 8 : 16);
  return (n_tok + per - 1) / per;
}
// into how many shares a token's batches go, so that there are about `want` CTAs or tasks
static int shares_of(long long blocks, int batches, long long want) {
  const long long s = (want + blocks - 1) / blocks;
  return s < 1 ? 1 : s < batches ? (int)s : batches;
}

// backward: three CTAs on each SM, four tasks for each of them where there are so many
constexpr int kBackwardCtas = 3 * kSms;
static int backward_shares(long long n_tok, long long q_heads, long long k_heads, int D) {
  return shares_of(token_blocks(n_tok, D), batches_of(q_heads, k_heads, kBackwardHeads), 4 * kBackwardCtas);
}
static unsigned backward_ctas(long long n_tok, long long q_heads, long long k_heads, int D) {
  const long long tasks = token_blocks(n_tok, D) * backward_shares(n_tok, q_heads, k_heads, D);
  return (unsigned)(tasks < kBackwardCtas ? tasks : kBackwardCtas);
}

static bool wide(const Args& a, int size, bool backward) {
  if (a.D % 8 != 0) return false;
  auto off = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; };
  const int unit = 16 / size;      // elements of 16 bytes
  for (const Side& s : a.side) {
    if (s.heads == 0) continue;
    if (off(s.x) || off(s.out) || off(s.w) || s.row % unit || s.head % unit) return false;
    if (backward && (off(s.g) || s.g_row % unit || s.g_head % unit)) return false;
  }
  return true;
}

template <typename T>
static cudaError_t launch_forward(const Args& a, cudaStream_t s) {
  const int G = a.D <= 64 ? 8 : 16;
  const long long blocks = token_blocks(a.n_tok, a.D);
  const int shares = shares_of(blocks, batches_of(a.side[0].heads, a.side[1].heads, kForwardHeads), 8 * kSms);
  if (blocks * shares > 0x7fffffffLL) return cudaErrorInvalidValue;
  const bool w = wide(a, sizeof(T), false);
  auto kern = G == 8 ? (w ? forward_kernel<T, 8, true> : forward_kernel<T, 8, false>) : (w ? forward_kernel<T, 16, true> : forward_kernel<T, 16, false>);
  return tc::launch_pdl(kern, (unsigned)(blocks * shares), kThreads, 0, s, a, shares);
}

template <typename T>
static cudaError_t launch_backward(const Args& a, void* const (&gw)[2], float* partial, cudaStream_t s, int* launches) {
  const unsigned ctas = backward_ctas(a.n_tok, a.side[0].heads, a.side[1].heads, a.D);
  const bool w = wide(a, sizeof(T), true);
  auto kern = a.D <= 64 ? (w ? backward_kernel<T, 8, true> : backward_kernel<T, 8, false>) : (w ? backward_kernel<T, 16, true> : backward_kernel<T, 16, false>);
  const bool any = gw[0] != nullptr || gw[1] != nullptr;
  *launches = 1;
  cudaError_t e = tc::launch_pdl(kern, ctas, kThreads, 0, s, a, backward_shares(a.n_tok, a.side[0].heads, a.side[1].heads, a.D),
                                 any ? partial : nullptr);
  if (e != cudaSuccess || !any) return e;
  *launches = 2;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.D + 31) / 32, 2);
  cfg.blockDim = dim3(1024);
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, weight_grad_kernel<T>, (const float*)partial, gw[0], gw[1], (int)ctas, a.D, a.side[0].w_float, a.side[1].w_float);
}

}  // namespace rope
}  // namespace attn

namespace {

using namespace attn;
using namespace attn::rope;
using capi::fail;

int check(const attn_rope_shape_t* s) {
  if (s == nullptr) return fail(ATTN_EINVAL, "shape is null");
  if (s->dtype != ATTN_F16 && s->dtype != ATTN_BF16 && s->dtype != ATTN_F32)
    return fail(ATTN_EUNSUPPORTED, "dtype %d: expected ATTN_F16, ATTN_BF16 or ATTN_F32", s->dtype);
  if (s->n_tok < 0 || s->n_tok > (1 << 30)) return fail(ATTN_EINVAL, "n_tok must be in [0, 2^30] (got %d)", s->n_tok);
  if (s->q_heads < 0 || s->k_heads < 0 || s->q_heads > (1 << 20) || s->k_heads > (1 << 20)) return fail(ATTN_EINVAL, "heads must be in [0, 2^20]");
  if (s->D <= 0 || s->D % 2 != 0 || s->D > 128) return fail(ATTN_EINVAL, "D must be even, in [2, 128] (got %d)", s->D);
  if (s->table_rows < 0) return fail(ATTN_EINVAL, "table_rows must be >= 0");
  if (s->axes < 1 || s->axes > kMaxAxes) return fail(ATTN_EINVAL, "axes must be in [1, %d] (got %d)", kMaxAxes, s->axes);
  long long pairs = 0;
  for (int i = 0; i < s->axes; ++i) {
    if (s->section[i] < 0) return fail(ATTN_EINVAL, "a section must not be negative");
    pairs += s->section[i];
  }
  if (pairs != s->D / 2) return fail(ATTN_EINVAL, "the sections must sum to D / 2 = %d (got %lld)", s->D / 2, pairs);
  // the grid, and the element offsets of the task lists
  if (((long long)s->n_tok + 15) / 16 * ((s->q_heads + 3) / 4 + (s->k_heads + 3) / 4) > 0x7fffffffLL) return fail(ATTN_ETOOLARGE, "n_tok and the heads make too many tiles");
  return ATTN_OK;
}

int fill(Args& a, const attn_rope_shape_t* s, const float* table, const void* positions, const void* const (&x)[2], const void* const (&g)[2],
         const void* const (&w)[2], void* const (&out)[2], bool backward) {
  memset(&a, 0, sizeof(a));
  if ((table == nullptr && s->table_rows > 0) || positions == nullptr) return fail(ATTN_EINVAL, "freqs or positions is null");
  if (reinterpret_cast<uintptr_t>(table) % 8 != 0) return fail(ATTN_EINVAL, "freqs is not 8-byte aligned");
  if (reinterpret_cast<uintptr_t>(positions) % (s->positions64 ? 8 : 4) != 0) return fail(ATTN_EINVAL, "positions is misaligned");
  const uintptr_t size = s->dtype == ATTN_F32 ? 4 : 2;
  for (int i = 0; i < 2; ++i) {
    Side& d = a.side[i];
    d.heads = i ? s->k_heads : s->q_heads;
    if (d.heads == 0) continue;
    if (x[i] == nullptr || out[i] == nullptr || (backward && g[i] == nullptr)) return fail(ATTN_EINVAL, "a tensor of q or k is null");
    for (const void* p : {x[i], (const void*)out[i], g[i]})
      if (reinterpret_cast<uintptr_t>(p) % size != 0) return fail(ATTN_EINVAL, "a tensor of q or k is misaligned");
    d.w_float = s->weight_float[i] != 0;
    if (reinterpret_cast<uintptr_t>(w[i]) % (d.w_float ? 4 : size) != 0) return fail(ATTN_EINVAL, "a weight is misaligned");
    d.x = x[i]; d.g = g[i]; d.w = w[i]; d.out = out[i];
    d.row = s->row_stride[i]; d.head = s->head_stride[i];
    d.g_row = s->g_row_stride[i]; d.g_head = s->g_head_stride[i];
  }
  a.table = table;
  a.positions = positions;
  a.axis_stride = s->axis_stride;
  a.positions64 = s->positions64;
  a.table_rows = s->table_rows;
  a.n_tok = s->n_tok;
  a.D = s->D;
  a.axes = s->axes;
  int end = 0;
  for (int i = 0; i < s->axes; ++i) a.section_end[i] = end += s->section[i];
  a.eps = s->eps;
  return ATTN_OK;
}

#define BY_TYPE(f, ...) (shape->dtype == ATTN_F16 ? f<__half>(__VA_ARGS__) : shape->dtype == ATTN_BF16 ? f<__nv_bfloat16>(__VA_ARGS__) : f<float>(__VA_ARGS__))

}  // namespace

extern "C" {

int attn_b200_packed_qk_norm_rope(const attn_rope_shape_t* shape, const void* q, const void* k, const void* q_weight, const void* k_weight,
                                  const float* freqs, const void* positions, void* q_out, void* k_out, void* stream) {
  int rc = check(shape);
  if (rc != ATTN_OK) return rc;
  if (shape->n_tok == 0 || shape->q_heads + shape->k_heads == 0) return capi::done(cudaSuccess, "", nullptr, 0);
  Args a;
  rc = fill(a, shape, freqs, positions, {q, k}, {nullptr, nullptr}, {q_weight, k_weight}, {q_out, k_out}, false);
  if (rc != ATTN_OK) return rc;
  unsigned int* status = nullptr;
  rc = capi::begin(&status);
  if (rc != ATTN_OK) return rc;
  return capi::done(BY_TYPE(launch_forward, a, static_cast<cudaStream_t>(stream)), "packed_qk_norm_rope launch failed", nullptr, 1);
}

size_t attn_b200_packed_qk_norm_rope_backward_scratch_bytes(const attn_rope_shape_t* s) {
  if (check(s) != ATTN_OK) return 0;
  return 2 * sizeof(float) * backward_ctas(s->n_tok, s->q_heads, s->k_heads, s->D) * (size_t)s->D;
}

int attn_b200_packed_qk_norm_rope_backward(const attn_rope_shape_t* shape, const void* q, const void* k, const void* q_weight, const void* k_weight,
                                           const float* freqs, const void* positions, const void* gq_out, const void* gk_out, void* gq, void* gk,
                                           void* gq_weight, void* gk_weight, float* scratch, void* stream) {
  int rc = check(shape);
  if (rc != ATTN_OK) return rc;
  if ((gq_weight != nullptr && q_weight == nullptr) || (gk_weight != nullptr && k_weight == nullptr))
    return fail(ATTN_EINVAL, "the gradient of a weight that is not there");
  if ((gq_weight != nullptr || gk_weight != nullptr) && scratch == nullptr) return fail(ATTN_EINVAL, "scratch is null");
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  unsigned int* status = nullptr;
  void* const gw[2] = {shape->q_heads > 0 ? gq_weight : nullptr, shape->k_heads > 0 ? gk_weight : nullptr};
  if (shape->n_tok == 0 || shape->q_heads + shape->k_heads == 0 || (gw[0] != gq_weight) || (gw[1] != gk_weight)) {
    // a weight that no row used
    rc = capi::begin(&status);
    if (rc != ATTN_OK) return rc;
    cudaError_t e = cudaSuccess;
    for (int i = 0; i < 2; ++i) {
      void* p = i ? gk_weight : gq_weight;
      if (p != nullptr && e == cudaSuccess && (shape->n_tok == 0 || gw[i] == nullptr))
        e = cudaMemsetAsync(p, 0, (size_t)shape->D * (shape->dtype == ATTN_F32 || shape->weight_float[i] ? 4 : 2), cs);
    }
    if (e != cudaSuccess || shape->n_tok == 0 || shape->q_heads + shape->k_heads == 0) return capi::done(e, "memset failed", nullptr, 0);
  }
  Args a;
  rc = fill(a, shape, freqs, positions, {q, k}, {gq_out, gk_out}, {q_weight, k_weight}, {gq, gk}, true);
  if (rc != ATTN_OK) return rc;
  rc = capi::begin(&status);
  if (rc != ATTN_OK) return rc;
  int launches = 0;
  const cudaError_t e = BY_TYPE(launch_backward, a, gw, scratch, cs, &launches);
  return capi::done(e, "packed_qk_norm_rope backward launch failed", nullptr, launches);
}

}  // extern "C"
