// Layer norm of rows, y = (x - mean) r w + b with r = 1 / sqrt(variance + eps), and its two backward passes, in fp32, each result rounded once.
//
//   first    c = g w:  dx = r (c - m(c) - xh m(c xh)),  dw = sum g xh,  db = sum g            (xh = (x - mean) r, m: mean over the row)
//   second   along tangents (u, uw, ub) of (x, w, b), P = r (u - m(u) - xh m(u xh)) is the tangent of xh:
//            to g: w P + uw xh + ub        to w: sum g P
//            to x: r (q - m(q) - xh m(q xh)) - r^2 xh (m(c u) - m(c) m(u) - m(c xh) m(u xh)),  q = g uw - r (c m(u xh) + u m(c xh))
//            m(q) and m(q xh) follow from the means of c, u, g uw and their products with xh, so one round of sums over the row does
//
// Every pass reads its rows once: a row stays in the registers of a group of 32 to 1024 threads, so that the variance is that of the centred row.  Sums over the rows
// stay in registers while a group goes from row to row, its next row on the way; a kernel behind adds what the CTAs have, in order.
//
// 16384 x 768 bf16 (ncu, cold): forward 15 to 17 us (50 MB: 8 us at the copy rate), dx with dw and db 20 to 23 (75 MB) and 7 to 9, second 72 (126 MB) and 8; 8195 x 4096 f16:
// 32 to 35, 45 to 48 and 8 to 10, 145 (336 MB) and 8.  The forward issues in 64 % of its cycles: a row's warps load and unpack w and b for every row, and the arithmetic is
// scalar.  The backward passes wait, for loads and the sums over a row, with two CTAs an SM or one.  The kernel behind has 48 CTAs at 768 columns, whose threads add ten
// of 296 rows each.  Above 8192 columns the backward's registers spill.
#pragma once

#include "attn_common.cuh"
#include "layer_launch.h"
#include "tc_common.cuh"

namespace attn {
namespace layer {

using tc::from_l2;

constexpr int kNormThreads = 256;

struct NormArgs {
  int n, d;
  bool param_float;
  float eps;
  const void *x, *w, *b, *g, *u, *uw, *ub;
  void *y, *gx;
  float *mean, *rstd;
  float* partial;                // [CTAs][sums][d]
  long long ldx, ldg, ldu;
};

// How a row lies in a group: `tpr` threads with `vectors` times eight elements each; wide: with 16-byte loads.  The fewest threads that hold it in
// 32 elements each; in the backward passes, which keep sums and the next row beside it, in 16 up to 16384, and three warps for 768 and a little
// less (dx and dw of 8195 x 4096 f16 with 32 elements each took 58 us, of 16384 x 768 bf16 with 24 43 to 56: one CTA an SM, or spills).
struct NormPlan { int tpr, vectors; bool wide; };
inline NormPlan plan_norm(int d, bool wide, bool backward) {
  const int vectors = (d + 7) / 8;
  if (!backward) {
    const int tpr = vectors <= 128 ? 32 : vectors <= 512 ? 128 : vectors <= 2048 ? 512 : 1024;
    return {tpr, (vectors + tpr - 1) / tpr, wide};
  }
  if (vectors <= 64) return {32, (vectors + 31) / 32, wide};
  if (vectors <= 96) return {96, 1, wide};
  int tpr = 64;
  while (tpr < 1024 && vectors > 2 * tpr) tpr *= 2;
  return {tpr, vectors > 2 * tpr ? 4 : 2, wide};
}

// Eight elements of a row at a time.  WIDE: in sequence, with 16-byte loads; else one by one, neighbouring threads on neighbouring elements, for any
// width and alignment.
template <typename T, int TPR, bool WIDE>
struct Lanes {
  static __device__ __forceinline__ int column(int t, int v, int e) { return WIDE ? (v * TPR + t) * 8 + e : (v * 8 + e) * TPR + t; }
  static __device__ __forceinline__ bool inside(int t, int v, int e, int d) { return column(t, v, WIDE ? 0 : e) < d; }      // WIDE: d is a multiple of 8
  static constexpr int kWords = sizeof(T) == 4 ? 8 : 4;
  struct Raw { uint32_t w[WIDE ? kWords : 8]; };

  static __device__ __forceinline__ Raw load(const T* row, int t, int v, int d) {
    Raw r;
    if constexpr (WIDE) {
      if (inside(t, v, 0, d)) {
        const uint4* p = reinterpret_cast<const uint4*>(row + column(t, v, 0));
#pragma unroll
        for (int q = 0; q < kWords / 4; ++q) {
          const uint4 a = from_l2(p + q);
          r.w[4 * q] = a.x; r.w[4 * q + 1] = a.y; r.w[4 * q + 2] = a.z; r.w[4 * q + 3] = a.w;
        }
      } else {
#pragma unroll
        for (int q = 0; q < kWords; ++q) r.w[q] = 0u;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) r.w[e] = inside(t, v, e, d) ? __float_as_uint(Elem<T>::to_float(row[column(t, v, e)])) : 0u;
    }
    return r;
  }
  static __device__ __forceinline__ void values(const Raw& r, float (&f)[8]) {
    if constexpr (WIDE && sizeof(T) == 2) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 a = tc::Pack<T>::unpack(r.w[e]);
        f[2 * e] = a.x; f[2 * e + 1] = a.y;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(r.w[e]);
    }
  }
  static __device__ __forceinline__ void store(T* row, int t, int v, int d, const float (&f)[8]) {
    if constexpr (WIDE) {
      if (!inside(t, v, 0, d)) return;
      uint4* p = reinterpret_cast<uint4*>(row + column(t, v, 0));
      if constexpr (sizeof(T) == 4) {
        p[0] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
        p[1] = make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7]));
      } else {
        p[0] = make_uint4(tc::Pack<T>::pack(f[0], f[1]), tc::Pack<T>::pack(f[2], f[3]), tc::Pack<T>::pack(f[4], f[5]), tc::Pack<T>::pack(f[6], f[7]));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (inside(t, v, e, d)) row[column(t, v, e)] = Elem<T>::from_float(f[e]);
    }
  }
};
// a parameter's (or its tangent's) elements of the same columns, float or of the rows' type; `fill` where there is none
template <typename L, typename T, bool WIDE>
__device__ __forceinline__ void parameter(const void* p, bool is_float, int t, int v, int d, float fill, float (&f)[8]) {
  if (p == nullptr) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = fill;
    return;
  }
  if (WIDE && !L::inside(t, v, 0, d)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = 0.f;
    return;
  }
  if (sizeof(T) == 4 || is_float) {
    const float* at = static_cast<const float*>(p);
    if constexpr (WIDE) {
      const float4 a = reinterpret_cast<const float4*>(at + L::column(t, v, 0))[0], b = reinterpret_cast<const float4*>(at + L::column(t, v, 0))[1];
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = L::inside(t, v, e, d) ? at[L::column(t, v, e)] : 0.f;
    }
  } else if constexpr (sizeof(T) == 2) {
    const T* at = static_cast<const T*>(p);
    if constexpr (WIDE) {
      const uint4 a = *reinterpret_cast<const uint4*>(at + L::column(t, v, 0));
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 b = tc::Pack<T>::unpack(w[e]);
        f[2 * e] = b.x; f[2 * e + 1] = b.y;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = L::inside(t, v, e, d) ? Elem<T>::to_float(at[L::column(t, v, e)]) : 0.f;
    }
  }
}

// Sums over the TPR threads of a group, all of which call it.  `turn` alternates between two places in shared memory.
template <int TPR, int THREADS, int K>
__device__ __forceinline__ void group_sum(float (&v)[K], float* shared, int& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if constexpr (TPR > 32) {
    constexpr int kWarps = THREADS / 32, kMine = TPR / 32;
    float* s = shared + turn * K * kWarps;
    turn ^= 1;
    const int warp = threadIdx.x >> 5, first = warp / kMine * kMine;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) s[k * kWarps + warp] = v[k];
    tc::named_barrier_sync(1 + first / kMine, TPR);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kMine; ++w) sum += s[k * kWarps + first + w];
      v[k] = sum;
    }
  }
}
template <int TPR> constexpr int kThreadsOf = TPR > kNormThreads ? TPR : TPR == 96 ? 288 : kNormThreads;

template <typename T, int TPR, int V, bool WIDE>
__global__ void __launch_bounds__(kThreadsOf<TPR>, 1)
norm_forward_kernel(const NormArgs a) {
  constexpr int kThreads = kThreadsOf<TPR>;
  __shared__ float sums[2 * (kThreads / 32)];
  typedef Lanes<T, TPR, WIDE> L;
  tc::pdl_wait();
  tc::pdl_trigger();
  const int t = threadIdx.x % TPR;
  const long long row = blockIdx.x * (long long)(kThreads / TPR) + threadIdx.x / TPR;
  const bool in = row < a.n;
  const T* x = static_cast<const T*>(a.x) + (in ? row : 0) * a.ldx;
  float f[V][8], s[1] = {0.f};
#pragma unroll
  for (int v = 0; v < V; ++v) L::values(L::load(x, t, v, a.d), f[v]);
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int e = 0; e < 8; ++e) s[0] += f[v][e];      // 0 outside
  int turn = 0;
  const float over = 1.f / (float)a.d;
  group_sum<TPR, kThreads>(s, sums, turn);
  const float mean = s[0] * over;
  s[0] = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      f[v][e] = L::inside(t, v, e, a.d) ? f[v][e] - mean : 0.f;
      s[0] = fmaf(f[v][e], f[v][e], s[0]);
    }
  group_sum<TPR, kThreads>(s, sums, turn);
  const float r = 1.f / sqrtf(s[0] * over + a.eps);
  if (!in) return;
  if (t == 0 && a.mean != nullptr) { a.mean[row] = mean; a.rstd[row] = r; }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float w[8], b[8];
    parameter<L, T, WIDE>(a.w, a.param_float, t, v, a.d, 1.f, w);
    parameter<L, T, WIDE>(a.b, a.param_float, t, v, a.d, 0.f, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[v][e] = fmaf(f[v][e] * r, w[e], b[e]);
    L::store(static_cast<T*>(a.y) + row * a.d, t, v, a.d, f[v]);
  }
}

// ORDER 1: dx, sums dw and db.  ORDER 2: the gradients of g and x, sum dw.
template <typename T, int TPR, int V, bool WIDE, int ORDER>
__global__ void __launch_bounds__(kThreadsOf<TPR>, ORDER == 1 && TPR <= kNormThreads ? 2 : 1)
norm_backward_kernel(const NormArgs a) {
  constexpr int kThreads = kThreadsOf<TPR>, kGroups = kThreads / TPR, kSums = ORDER == 1 ? 2 : 1, kMeans = ORDER == 1 ? 2 : 7;
  __shared__ float sums[2 * kMeans * (kThreads / 32)];
  typedef Lanes<T, TPR, WIDE> L;
  tc::pdl_wait();
  tc::pdl_trigger();
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const long long stride = (long long)gridDim.x * kGroups;
  float total[kSums][V][8];
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) total[k][v][e] = 0.f;
  int turn = 0;
  const float over = 1.f / (float)a.d;
  // a row stays as it was read: what follows from it is computed before the sums over the row and again behind them, in fewer registers
  struct Row { typename L::Raw x[V], g[V], u[ORDER == 2 ? V : 1]; float mean, r; };
  auto fetch = [&](Row& row, long long at) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      row.x[v] = L::load(static_cast<const T*>(a.x) + at * a.ldx, t, v, a.d);
      row.g[v] = L::load(static_cast<const T*>(a.g) + at * a.ldg, t, v, a.d);
      if constexpr (ORDER == 2)
        row.u[v] = a.u == nullptr ? typename L::Raw{} : L::load(static_cast<const T*>(a.u) + at * a.ldu, t, v, a.d);
    }
    row.mean = from_l2(a.mean + at);
    row.r = from_l2(a.rstd + at);
  };
  auto normed = [&](const Row& row, int v, float (&xh)[8]) {
    L::values(row.x[v], xh);
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float2 h = __fmul2_rn(__fadd2_rn(make_float2(xh[e], xh[e + 1]), make_float2(-row.mean, -row.mean)), make_float2(row.r, row.r));
      xh[e] = h.x; xh[e + 1] = h.y;
    }
  };
  auto as_read = [](typename L::Raw& raw) {      // keeps the compiler from holding on to the values instead
#pragma unroll
    for (int i = 0; i < (int)(sizeof(raw.w) / 4); ++i) asm volatile("" : "+r"(raw.w[i]));
  };
  // w in fp32, for as many threads as fill their registers with sums over the rows
  constexpr bool kSharedW = TPR <= 512;
  __shared__ __align__(16) float weight[kSharedW ? TPR * V * 8 : 4];
  if constexpr (kSharedW) {
    for (int i = threadIdx.x; i < TPR * V; i += kThreads) {
      float w[8];
      parameter<L, T, WIDE>(a.w, a.param_float, i % TPR, i / TPR, a.d, 1.f, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) weight[(i / TPR) * TPR * 8 + (e >> 2) * TPR * 4 + (i % TPR) * 4 + (e & 3)] = w[e];
    }
    __syncthreads();
  }
  auto weight_of = [&](int v, float (&w)[8]) {
    if constexpr (kSharedW) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4 q = *reinterpret_cast<const float4*>(&weight[v * TPR * 8 + h * TPR * 4 + t * 4]);
        w[4 * h] = q.x; w[4 * h + 1] = q.y; w[4 * h + 2] = q.z; w[4 * h + 3] = q.w;
      }
    } else {
      parameter<L, T, WIDE>(a.w, a.param_float, t, v, a.d, 1.f, w);
    }
  };
  Row next;
  const long long first = blockIdx.x * (long long)kGroups + group;
  if (first < a.n) fetch(next, first);
  for (long long at = first; at < a.n; at += stride) {
    Row row = next;
    if (at + stride < a.n) fetch(next, at + stride);
    float m[kMeans];
#pragma unroll
    for (int k = 0; k < kMeans; ++k) m[k] = 0.f;
    [[maybe_unused]] float2 m0 = make_float2(0.f, 0.f), m1 = m0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float xh[8], g[8], w[8];      // g and u are 0 outside of the row, and everything is a multiple of them
      normed(row, v, xh);
      L::values(row.g[v], g);
      weight_of(v, w);
      if constexpr (ORDER == 1) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float2 gg = make_float2(g[e], g[e + 1]), h = make_float2(xh[e], xh[e + 1]), c = __fmul2_rn(gg, make_float2(w[e], w[e + 1]));
          m0 = __fadd2_rn(m0, c);
          m1 = __ffma2_rn(c, h, m1);
          const float2 t0 = __ffma2_rn(gg, h, make_float2(total[0][v][e], total[0][v][e + 1])), t1 = __fadd2_rn(gg, make_float2(total[1][v][e], total[1][v][e + 1]));
          total[0][v][e] = t0.x; total[0][v][e + 1] = t0.y;
          total[1][v][e] = t1.x; total[1][v][e + 1] = t1.y;
        }
      } else {
        float uw[8], u[8];
        parameter<L, T, WIDE>(a.uw, a.param_float, t, v, a.d, 0.f, uw);
        L::values(row.u[v], u);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float c = g[e] * w[e], q = g[e] * uw[e];
          m[0] += c;
          m[1] = fmaf(c, xh[e], m[1]);
          m[2] += u[e];
          m[3] = fmaf(u[e], xh[e], m[3]);
          m[4] = fmaf(c, u[e], m[4]);
          m[5] += q;
          m[6] = fmaf(q, xh[e], m[6]);
        }
      }
    }
    if constexpr (ORDER == 1) {
      m[0] = m0.x + m0.y;
      m[1] = m1.x + m1.y;
    }
    group_sum<TPR, kThreads>(m, sums, turn);
#pragma unroll
    for (int k = 0; k < kMeans; ++k) m[k] *= over;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      as_read(row.x[v]);
      as_read(row.g[v]);
      if constexpr (ORDER == 2) as_read(row.u[v]);
    }
    const float r = row.r;
    if constexpr (ORDER == 1) {
      if (a.gx != nullptr) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float xh[8], g[8], w[8];
          normed(row, v, xh);
          L::values(row.g[v], g);
          weight_of(v, w);
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            float2 c = __ffma2_rn(make_float2(g[e], g[e + 1]), make_float2(w[e], w[e + 1]), make_float2(-m[0], -m[0]));
            c = __fmul2_rn(__ffma2_rn(make_float2(xh[e], xh[e + 1]), make_float2(-m[1], -m[1]), c), make_float2(r, r));
            g[e] = c.x; g[e + 1] = c.y;
          }
          L::store(static_cast<T*>(a.gx) + at * a.d, t, v, a.d, g);
        }
      }
    } else {
      const float mc = m[0], mch = m[1], mu = m[2], muh = m[3];
      const float mq = m[5] - r * (mc * muh + mu * mch), mqh = m[6] - 2.f * r * mch * muh, turned = r * r * (m[4] - mc * mu - mch * muh);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float xh[8], g[8], u[8], w[8], uw[8], ub[8], gg[8], gx[8];
        normed(row, v, xh);
        L::values(row.g[v], g);
        L::values(row.u[v], u);
        weight_of(v, w);
        parameter<L, T, WIDE>(a.uw, a.param_float, t, v, a.d, 0.f, uw);
        parameter<L, T, WIDE>(a.ub, a.param_float, t, v, a.d, 0.f, ub);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float h = xh[e], P = r * (u[e] - mu - h * muh);
          gg[e] = fmaf(w[e], P, fmaf(uw[e], h, ub[e]));
          const float q = fmaf(-r, g[e] * w[e] * muh + u[e] * mch, g[e] * uw[e]);
          gx[e] = r * (q - mq - h * mqh) - h * turned;
          total[0][v][e] = fmaf(g[e], P, total[0][v][e]);
        }
        if (a.y != nullptr) L::store(static_cast<T*>(a.y) + at * a.d, t, v, a.d, gg);
        if (a.gx != nullptr) L::store(static_cast<T*>(a.gx) + at * a.d, t, v, a.d, gx);
      }
    }
  }
  if (a.partial == nullptr) return;
  // the CTA's groups, one after the other, into its row of the partial sums
  __shared__ __align__(16) float joined[kGroups > 1 ? kSums * TPR * V * 8 : 4];
  float* out = a.partial + (size_t)blockIdx.x * kSums * a.d;
  for (int q = kGroups - 1; q >= 0; --q) {
    if (group == q)
#pragma unroll
      for (int k = 0; k < kSums; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float s = total[k][v][e];
            const int at = ((k * V + v) * 8 + e) * TPR + t;
            if (q < kGroups - 1) s += joined[at];
            if (q > 0) joined[at] = s;
            else if (L::inside(t, v, e, a.d)) out[(size_t)k * a.d + L::column(t, v, e)] = s;
          }
    __syncthreads();
  }
}

// ---- host ---------------------------------------------------------------------------------------
template <typename T, int TPR, int V, bool WIDE, int ORDER>
inline cudaError_t launch_norm(const NormArgs& a, unsigned ctas, cudaStream_t stream) {
  if constexpr (ORDER == 0) return tc::launch_pdl(norm_forward_kernel<T, TPR, V, WIDE>, ctas, (unsigned)kThreadsOf<TPR>, 0, stream, a);
  else return tc::launch_pdl(norm_backward_kernel<T, TPR, V, WIDE, ORDER>, ctas, (unsigned)kThreadsOf<TPR>, 0, stream, a);
}
template <typename T, bool WIDE, int ORDER>
inline cudaError_t launch_plan(const NormPlan& p, const NormArgs& a, unsigned ctas, cudaStream_t stream) {
  if (p.tpr == 32) {
    if (p.vectors == 1) return launch_norm<T, 32, 1, WIDE, ORDER>(a, ctas, stream);
    if (p.vectors == 2) return launch_norm<T, 32, 2, WIDE, ORDER>(a, ctas, stream);
  }
  if constexpr (ORDER == 0) {
    if (p.tpr == 32 && p.vectors == 3) return launch_norm<T, 32, 3, WIDE, 0>(a, ctas, stream);
    if (p.tpr == 32) return launch_norm<T, 32, 4, WIDE, 0>(a, ctas, stream);
    if (p.tpr == 128) return p.vectors == 2   ? launch_norm<T, 128, 2, WIDE, 0>(a, ctas, stream)
                             : p.vectors == 3 ? launch_norm<T, 128, 3, WIDE, 0>(a, ctas, stream)
                                              : launch_norm<T, 128, 4, WIDE, 0>(a, ctas, stream);
    if (p.tpr == 512) return p.vectors == 2 ? launch_norm<T, 512, 2, WIDE, 0>(a, ctas, stream) : launch_norm<T, 512, 4, WIDE, 0>(a, ctas, stream);
    return launch_norm<T, 1024, 4, WIDE, 0>(a, ctas, stream);
  } else {
    switch (p.tpr) {
      case 96: return launch_norm<T, 96, 1, WIDE, ORDER>(a, ctas, stream);
      case 64: return launch_norm<T, 64, 2, WIDE, ORDER>(a, ctas, stream);
      case 128: return launch_norm<T, 128, 2, WIDE, ORDER>(a, ctas, stream);
      case 256: return launch_norm<T, 256, 2, WIDE, ORDER>(a, ctas, stream);
      case 512: return launch_norm<T, 512, 2, WIDE, ORDER>(a, ctas, stream);
      default: return p.vectors == 2 ? launch_norm<T, 1024, 2, WIDE, ORDER>(a, ctas, stream) : launch_norm<T, 1024, 4, WIDE, ORDER>(a, ctas, stream);
    }
  }
}
template <int ORDER>
inline cudaError_t launch_typed(const NormPlan& p, const NormArgs& a, int dtype, unsigned ctas, cudaStream_t stream) {
  if (dtype == ATTN_F16) return p.wide ? launch_plan<__half, true, ORDER>(p, a, ctas, stream) : launch_plan<__half, false, ORDER>(p, a, ctas, stream);
  if (dtype == ATTN_BF16) return p.wide ? launch_plan<__nv_bfloat16, true, ORDER>(p, a, ctas, stream) : launch_plan<__nv_bfloat16, false, ORDER>(p, a, ctas, stream);
  return p.wide ? launch_plan<float, true, ORDER>(p, a, ctas, stream) : launch_plan<float, false, ORDER>(p, a, ctas, stream);
}

cudaError_t launch_norm_forward(const NormPlan& p, const NormArgs& a, int dtype, unsigned ctas, cudaStream_t stream);
cudaError_t launch_norm_first(const NormPlan& p, const NormArgs& a, int dtype, unsigned ctas, cudaStream_t stream);
cudaError_t launch_norm_second(const NormPlan& p, const NormArgs& a, int dtype, unsigned ctas, cudaStream_t stream);

}  // namespace layer
}  // namespace attn
