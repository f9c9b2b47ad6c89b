// Row kernels of the linear cross entropy: the loss from the product's partial maxima and sums, the gradient's row factors, the
// copy of x without the rows that do not count, the sum over shares of k.
#include "attn_common.cuh"
#include "lce_launch.h"
#include "tc_common.cuh"

namespace attn {
namespace lce {

using tc::from_l2;

// 0: ignored; 1: counts; 2: no such class, so its loss is not a number
__device__ __forceinline__ int row_kind(int64_t y, long long ignore_index, int V) {
  return y == ignore_index ? 0 : y >= 0 && y < V ? 1 : 2;
}
__device__ __forceinline__ int64_t target_of(const int64_t* targets, int i) { return from_l2(reinterpret_cast<const long long*>(targets) + i); }

// ---- loss ---------------------------------------------------------------------------------------
// 32 rows of a CTA, 16 threads a row, each a sixteenth of the column tiles (coalesced along the rows); one read of the partials,
// 8 bytes per row and tile: 16384 x 125, 16 MB, 13 to 15 us.
constexpr int kRowGroups = 16;

__global__ void __launch_bounds__(32 * kRowGroups)
finish_kernel(const Partial* partial, const float* target_logit, const int64_t* targets, float* loss, float* lse, int n, int V, int tiles,
              long long ignore_index) {
  __shared__ float ms[kRowGroups][32], ls[kRowGroups][32];
  tc::pdl_wait();
  tc::pdl_trigger();
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, r = blockIdx.x * 32 + x;
  float m = -INFINITY, part = 0.f;
  if (r < n)
#pragma unroll 8
    for (int t = y; t < tiles; t += kRowGroups) {
      const float2 v = from_l2(reinterpret_cast<const float2*>(partial) + (size_t)t * n + r);
      const float m_new = fmaxf(m, v.x);
      part = part * (m == m_new ? 1.f : exp2f(m - m_new)) + v.y * (v.x == m_new ? 1.f : exp2f(v.x - m_new));
      m = m_new;
    }
  ms[y][x] = m;
  ls[y][x] = part;
  __syncthreads();
  if (y != 0 || r >= n) return;
  float top = ms[0][x];
  for (int i = 1; i < kRowGroups; ++i) top = fmaxf(top, ms[i][x]);
  float sum = 0.f;
  for (int i = 0; i < kRowGroups; ++i) sum += ls[i][x] * (ms[i][x] == top ? 1.f : exp2f(ms[i][x] - top));
  const float over = log2f(sum);
  lse[r] = (float)(((double)top + over) / kLog2e);      // maxima are multiples of kLog2e: a row of one logit gives that logit
  const int kind = row_kind(target_of(targets, r), ignore_index, V);
  float l = kind == 0 ? 0.f : NAN;
  if (kind == 1) {      // not lse - z: where the target has nearly all of the sum, that would be the rounding of lse.  Below 0 only by rounding
    l = (fmaf(-from_l2(target_logit + r), kLog2e, top) + over) * kLn2;
    if (l < 0.f) l = 0.f;
  }
  loss[r] = l;
}

cudaError_t launch_finish(const Problem& p, const Scores& s, float* loss, float* lse, cudaStream_t stream) {
  return tc::launch_pdl(finish_kernel, (unsigned)((p.n + 31) / 32), 32 * kRowGroups, 0, stream, s.partial, s.target_logit, p.targets, loss, lse, p.n,
                        p.V, s.tiles, p.ignore_index);
}

// Sum over a CTA of 1024 threads, in a fixed order.
template <typename V>
__device__ __forceinline__ V block_sum(V v, V* shared) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = shared[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  return v;
}

// in 64 bits: a sum of tens of thousands of losses in 32 would lose the last digits of the mean
__global__ void __launch_bounds__(1024)
total_kernel(const float* loss, const int64_t* targets, float* value, float* counted, int n, int reduction, long long ignore_index) {
  __shared__ double sums[32];
  tc::pdl_wait();
  tc::pdl_trigger();
  double s = 0.0, count = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += 1024) {
    s += from_l2(loss + i);
    count += target_of(targets, i) != ignore_index ? 1.0 : 0.0;
  }
  s = block_sum(s, sums);
  count = block_sum(count, sums);
  if (threadIdx.x == 0) {
    *value = (float)(reduction == RED_MEAN ? s / count : s);      // a mean over no rows is 0 / 0
    *counted = (float)count;
  }
}

cudaError_t launch_total(const Problem& p, const float* loss, int reduction, float* value, float* counted, cudaStream_t stream) {
  return tc::launch_pdl(total_kernel, 1u, 1024u, 0, stream, loss, p.targets, value, counted, p.n, reduction, p.ignore_index);
}

// ---- gradient's row factors -----------------------------------------------------------------------
// G is rounded to the input type before its products, so the factors are taken relative to the largest one, and the results are multiplied
// back.  Where all rows have the same factor c, as in a mean, it is then exactly 1: c (P - 1), at every row's target, would be off by the
// same share of up to half a step for all rows, which sums do not average out (bf16, 16384 x 768 x 32000: gradients 3.8e-3 from 64 bits in the
// 2-norm).  In fp16 a factor of 1 / n and probabilities of 1e-5 would also leave its normal range (6e-5): there the largest one is 2^15 (then
// |G| <= 2^15 < 65504, and what is 2^29 below the largest factor is still normal).  G is kept in float for float.
__global__ void __launch_bounds__(1024)
coefficients_kernel(const float* grad, const float* counted, const int64_t* targets, float* coef, float* scale, int n, int V, int reduction,
                    float largest, long long ignore_index) {
  __shared__ float tops[32];
  tc::pdl_wait();
  tc::pdl_trigger();
  const float common = reduction == RED_NONE ? 0.f : reduction == RED_MEAN ? from_l2(grad) / from_l2(counted) : from_l2(grad);
  auto factor = [&](int i) {
    const int kind = row_kind(target_of(targets, i), ignore_index, V);
    return kind == 0 ? 0.f : kind == 1 ? (reduction == RED_NONE ? from_l2(grad + i) : common) : NAN;
  };
  float unit = 1.f, times = 1.f;
  if (largest > 0.f) {      // every CTA looks for the largest factor where rows have their own
    float top = 0.f;
    if (reduction == RED_NONE) {
#pragma unroll 4
      for (int i = threadIdx.x; i < n; i += 1024) top = fmaxf(top, fabsf(factor(i)));
    } else {
      top = fabsf(common);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int i = 0; i < 32; ++i) top = fmaxf(top, tops[i]);
    if (top > 0.f && top < INFINITY) { unit = top; times = largest; }
  }
#pragma unroll 4
  for (int i = blockIdx.x * 1024 + threadIdx.x; i < n; i += gridDim.x * 1024) coef[i] = factor(i) / unit * times;
  if (blockIdx.x == 0 && threadIdx.x == 0) *scale = unit / times;
}

cudaError_t launch_coefficients(const Problem& p, const float* grad, const float* counted, int reduction, const Coefficients& c, cudaStream_t stream) {
  const unsigned ctas = (unsigned)((p.n + 1023) / 1024 < kSms ? (p.n + 1023) / 1024 : kSms);
  const float largest = p.dtype == 0 ? 32768.f : p.dtype == 1 ? 1.f : 0.f;
  return tc::launch_pdl(coefficients_kernel, ctas, 1024u, 0, stream, grad, counted, p.targets, c.coef, c.scale, p.n, p.V, reduction, largest,
                        p.ignore_index);
}

// ---- x with zeros in the rows that do not count ----------------------------------------------------
// dW sums over the rows, where a factor of 0 does not keep an inf or NaN of an ignored row (padding, say) out.  U: 16 bytes, or one element.
template <typename U>
__global__ void __launch_bounds__(256)
counted_rows_kernel(const U* x, U* dst, const int64_t* targets, int n, int width, long long ignore_index) {
  tc::pdl_wait();
  tc::pdl_trigger();
  const long long total = (long long)n * width;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    U v = {};
    if (target_of(targets, (int)(i / width)) != ignore_index) v = from_l2(x + i);
    dst[i] = v;
  }
}

cudaError_t launch_counted_rows(const Problem& p, void* dst, cudaStream_t stream) {
  const int size = p.dtype == 2 ? 4 : 2;
  const long long bytes = (long long)p.d * size, total = bytes % 16 == 0 ? p.n * (bytes / 16) : (long long)p.n * p.d;
  const long long want = (total + 255) / 256;
  const unsigned ctas = (unsigned)(want < 16 * kSms ? want : 16 * kSms);
  const bool aligned = bytes % 16 == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && reinterpret_cast<uintptr_t>(dst) % 16 == 0;
  if (aligned) return tc::launch_pdl(counted_rows_kernel<uint4>, ctas, 256u, 0, stream, (const uint4*)p.x, (uint4*)dst, p.targets, p.n, (int)(bytes / 16), p.ignore_index);
  if (size == 4) return tc::launch_pdl(counted_rows_kernel<float>, ctas, 256u, 0, stream, (const float*)p.x, (float*)dst, p.targets, p.n, p.d, p.ignore_index);
  return tc::launch_pdl(counted_rows_kernel<unsigned short>, ctas, 256u, 0, stream, (const unsigned short*)p.x, (unsigned short*)dst, p.targets, p.n,
                        p.d, p.ignore_index);
}

// ---- sum over the shares of k ----------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256)
sum_splits_kernel(const float* acc, int splits, long long count, const float* scale, T* result) {
  tc::pdl_wait();
  tc::pdl_trigger();
  const float mul = from_l2(scale);
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < count; i += gridDim.x * 256ll) {
    float v = 0.f;
#pragma unroll 8
    for (int s = 0; s < splits; ++s) v += from_l2(acc + s * count + i);
    result[i] = Elem<T>::from_float(v * mul);
  }
}

cudaError_t launch_sum_splits(const float* acc, int splits, long long count, const float* scale, void* result, int dtype, cudaStream_t stream) {
  const long long want = (count + 255) / 256;
  const unsigned ctas = (unsigned)(want < 16 * kSms ? want : 16 * kSms);
  if (dtype == 0) return tc::launch_pdl(sum_splits_kernel<__half>, ctas, 256u, 0, stream, acc, splits, count, scale, (__half*)result);
  if (dtype == 1) return tc::launch_pdl(sum_splits_kernel<__nv_bfloat16>, ctas, 256u, 0, stream, acc, splits, count, scale, (__nv_bfloat16*)result);
  return tc::launch_pdl(sum_splits_kernel<float>, ctas, 256u, 0, stream, acc, splits, count, scale, (float*)result);
}

}  // namespace lce
}  // namespace attn
