// Matrix products of few rows (single tokens, small batches) with a weight, half types: out[r, j] = sum_k a[r, k] b[j, k] for up to 32 rows, with what follows
// (product_tc.cu).  Bound by reading the weight once: a tile of 256 x 256 would leave most SMs idle and its rows empty.
//
// A CTA has 16 rows of the weight (of Wg and of Wu in a gated product), its warps share k in blocks of 32.  A thread reads 16 bytes of two rows of
// the weight and of one row of `a` straight into the fragments of two m16n8k16 products, whose order of k does not matter as long as both operands have
// the same.  Four blocks of a warp are on their way at once.  The warps' sums meet in shared memory, in order.
//
// One row, bf16, in a graph of many calls on weights from HBM: 768 -> 2304 2.6 us, 2048 -> 5504 6.6, 5504 -> 2048 7.2 (9.7 with eight warps), 4096 -> 14336 25.6 (4.6 TB/s; the copy
// rate takes 17.9).  Short of it by how CTAs fill the SMs: 5504 -> 2048 is 128 CTAs for 148 SMs, a gated 2048 -> 5504 (13 us) 344 CTAs of 114 registers, two to an SM, 1.16
// waves.  Eight blocks on their way were 7.7 at 2048 -> 5504, with fewer CTAs an SM.
#include "activation.cuh"
#include "layer_launch.h"
#include "tc_common.cuh"

namespace attn {
namespace layer {

using namespace tc;

// What a CTA has: 16 rows of a weight, 16 of either weight of a gated product, 32 of a weight
enum Few { ONE = 0, GATE = 1, TWO = 2 };

struct FewArgs {
  int rows, cols, k, act;
  const void *a, *b, *b2;
  long long lda, ldb, ldb2;
  const void *bias, *residual;
  long long ld_residual;
  void* out;
  long long ldo;
  void* kept[2];
  long long ld_kept[2];
  void* low;
  long long ld_low;
};

template <typename T>
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (Pack<T>::kIsBf16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// eight elements of a row from k, zeros behind its end
__device__ __forceinline__ uint4 few_load(const uint16_t* row, bool in, int k, int k_end) {
  if (!in || k >= k_end) return make_uint4(0u, 0u, 0u, 0u);
  if (k + 8 <= k_end) return from_l2(reinterpret_cast<const uint4*>(row + k));
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = (k + 2 * e < k_end ? (uint32_t)row[k + 2 * e] : 0u) | (k + 2 * e + 1 < k_end ? (uint32_t)row[k + 2 * e + 1] << 16 : 0u);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T, int FEW, int NB, int kFewWarps>
__global__ void __launch_bounds__(32 * kFewWarps)
product_few_kernel(const __grid_constant__ FewArgs g) {
  constexpr bool kGate = FEW == GATE;
  constexpr int kWeights = FEW == ONE ? 1 : 2, kRows = 8 * NB, kAtOnce = 4;
  __shared__ float sums[kWeights][kFewWarps][kRows][17];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = lane >> 2, t = lane & 3;
  const int j0 = (int)blockIdx.x * (FEW == TWO ? 32 : 16);
  const uint16_t *w[kWeights][2], *x[NB];
  bool in_w[kWeights][2], in_x[NB];
#pragma unroll
  for (int i = 0; i < kWeights; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int j = j0 + group + 8 * h + (FEW == TWO ? 16 * i : 0);
      in_w[i][h] = j < g.cols;
      w[i][h] = static_cast<const uint16_t*>(kGate && i == 1 ? g.b2 : g.b) + (in_w[i][h] ? j : 0) * (kGate && i == 1 ? g.ldb2 : g.ldb);
    }
#pragma unroll
  for (int q = 0; q < NB; ++q) {
    const int r = 8 * q + group;
    in_x[q] = r < g.rows;
    x[q] = static_cast<const uint16_t*>(g.a) + (in_x[q] ? r : 0) * g.lda;
  }
  float acc[kWeights][NB][4];
#pragma unroll
  for (int i = 0; i < kWeights; ++i)
#pragma unroll
    for (int q = 0; q < NB; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][q][e] = 0.f;
  for (int k0 = warp * 32; k0 < g.k; k0 += 32 * kFewWarps * kAtOnce) {
    uint4 wv[kAtOnce][kWeights][2], xv[kAtOnce][NB];
#pragma unroll
    for (int s = 0; s < kAtOnce; ++s) {
      const int k = k0 + s * 32 * kFewWarps + 8 * t;
#pragma unroll
      for (int i = 0; i < kWeights; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) wv[s][i][h] = few_load(w[i][h], in_w[i][h], k, g.k);
#pragma unroll
      for (int q = 0; q < NB; ++q) xv[s][q] = few_load(x[q], in_x[q], k, g.k);
    }
#pragma unroll
    for (int s = 0; s < kAtOnce; ++s)
#pragma unroll
      for (int i = 0; i < kWeights; ++i)
#pragma unroll
        for (int q = 0; q < NB; ++q) {
          const uint4 &a = wv[s][i][0], &b = wv[s][i][1], &c = xv[s][q];
          mma_16x8x16<T>(acc[i][q], a.x, b.x, a.y, b.y, c.x, c.y);
          mma_16x8x16<T>(acc[i][q], a.z, b.z, a.w, b.w, c.z, c.w);
        }
  }
#pragma unroll
  for (int i = 0; i < kWeights; ++i)
#pragma unroll
    for (int q = 0; q < NB; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[i][warp][8 * q + 2 * t + (e & 1)][group + 8 * (e >> 1)] = acc[i][q][e];
  __syncthreads();
  constexpr int kOut = FEW == TWO ? 32 : 16;
  for (int i = threadIdx.x; i < kRows * kOut; i += 32 * kFewWarps) {
    const int r = i / kOut, c = i % 16, half = FEW == TWO ? i / 16 % 2 : 0, j = j0 + 16 * half + c;
    if (r >= g.rows || j >= g.cols) continue;
    float z = 0.f, u = 0.f;
#pragma unroll
    for (int s = 0; s < kFewWarps; ++s) {
      z += sums[half][s][r][c];
      if constexpr (kGate) u += sums[kWeights - 1][s][r][c];
    }
    if (!kGate && g.bias != nullptr) z += Elem<T>::to_float(static_cast<const T*>(g.bias)[j]);
    if (g.kept[0] != nullptr) {
      if constexpr (kGate) {
        const uint32_t cz = Kept<T>::code(z), cu = Kept<T>::code(u);
        static_cast<uint16_t*>(g.kept[0])[r * g.ld_kept[0] + j] = (uint16_t)(cz >> 16);
        static_cast<uint16_t*>(g.kept[1])[r * g.ld_kept[1] + j] = (uint16_t)(cu >> 16);
        static_cast<uint8_t*>(g.low)[r * g.ld_low + j] = (uint8_t)((cz >> 12 & 0xfu) | (cu >> 8 & 0xf0u));
      } else {
        static_cast<uint16_t*>(g.kept[0])[r * g.ld_kept[0] + j] = (uint16_t)pack_argument(z, z);
      }
    }
    float y = z;
    with_activation(g.act, [&](auto act) {
      float2 a, d;
      activate2<decltype(act)::value, false>(make_float2(z, z), a, d);
      y = a.x;
    });
    if constexpr (kGate) y *= u;
    else if (g.residual != nullptr) y += Elem<T>::to_float(static_cast<const T*>(g.residual)[r * g.ld_residual + j]);
    static_cast<T*>(g.out)[r * g.ldo + j] = Elem<T>::from_float(y);
  }
}

// Up to 16 rows always; up to 32 against a weight of up to 20 million elements, or two of a gated product of 12 million together.  The rows are read by every CTA,
// so more of them cost more here, and nothing in tiles, where the number of tiles decides.  Both forms timed in graphs, us here / in tiles (k -> columns, bf16, weights from HBM):
//                            1 row          16 rows        17 rows        32 rows
//   plain   768 ->  2304    2.6 /  8.4     2.9 /  8.6     3.5 /  8.6     3.9 /  8.6
//          2048 ->  5504    6.6 / 15.9    11.2 / 14.9    12.5 / 14.9    14.3 / 15.0      11.3 million
//          4096 ->  4096   10.2 / 21.2    12.6 / 19.9    14.6 / 19.9    16.5 / 20.0      16.8
//          4096 ->  6144   11.8 / 25.6    19.5 / 22.4    21.7 / 22.2    24.8 / 22.4      25.2
//          4096 -> 14336   25.6 / 40.3    30.7 / 29.0    52.2 / 29.0    53.9 / 29.4      58.7
//   gated  2048 ->  2048    5.6 / 14.5     6.8 / 14.4     8.5 / 14.3     8.8 / 14.4       8.4, both weights
//          2048 ->  2752    7.3 / 15.6     8.6 / 14.6    14.9 / 14.6    15.5 / 14.6      11.3
//          2048 ->  5504   13.0 / 23.0    16.1 / 19.6    22.4 / 19.3    23.1 / 16.1      22.5
//          4096 -> 14336   43.1 / 68.1    49.7 / 52.2    88.1 / 52.2    90.1 / 52.7     117
bool few_rows(const attn_products_t& c) {
  const attn_product_t& p = c.product[0];
  const long long most = c.kind == ATTN_PRODUCT_GATED ? 6000000 : 20000000;      // elements of a weight
  return c.form == ATTN_FORM_NT && c.kind != ATTN_PRODUCT_GATED_GRAD && c.count == 1 && p.pairs == 1 && p.rows > 0 && p.cols > 0 && p.k > 0 &&
         (p.rows <= 16 || (p.rows <= 32 && (long long)p.cols * p.k <= most));
}

template <typename T, int FEW, int WARPS>
static cudaError_t launch(const FewArgs& a, cudaStream_t stream) {
  constexpr int kOut = FEW == TWO ? 32 : 16;
  const unsigned ctas = ((unsigned)a.cols + kOut - 1) / kOut, threads = 32 * WARPS;
  if (a.rows <= 8) return launch_pdl(product_few_kernel<T, FEW, 1, WARPS>, ctas, threads, 0, stream, a);
  if (a.rows <= 16) return launch_pdl(product_few_kernel<T, FEW, 2, WARPS>, ctas, threads, 0, stream, a);
  return launch_pdl(product_few_kernel<T, FEW, 4, WARPS>, ctas, threads, 0, stream, a);
}
// Sixteen warps where that leaves no SM more than two CTAs and k is long enough for them; 32 rows of the weight where there are CTAs enough, which
// read the rows of `a` half as often
template <typename T>
static cudaError_t launch_shape(const FewArgs& a, bool gate, cudaStream_t stream) {
  if (gate) return launch<T, GATE, 8>(a, stream);
  if (a.cols >= 16 * 4 * kSms) return launch<T, TWO, 8>(a, stream);
  if (a.cols <= 16 * 2 * kSms && a.k >= 1024) return launch<T, ONE, 16>(a, stream);
  return launch<T, ONE, 8>(a, stream);
}

cudaError_t few_products(const attn_products_t& c, cudaStream_t stream, int* launches) {
  const attn_product_t& p = c.product[0];
  FewArgs a = {};
  a.rows = p.rows; a.cols = p.cols; a.k = p.k;
  a.act = c.activation;
  a.a = p.pair[0].a; a.b = p.pair[0].b; a.b2 = c.b2;
  a.lda = p.pair[0].lda; a.ldb = p.pair[0].ldb; a.ldb2 = c.ldb2;
  a.bias = c.bias; a.residual = c.residual; a.ld_residual = c.ld_residual;
  a.out = p.out; a.ldo = p.ldo;
  for (int q = 0; q < 2; ++q) { a.kept[q] = c.kept[q]; a.ld_kept[q] = c.ld_kept[q]; }
  a.low = c.kept_low; a.ld_low = c.ld_low;
  ++*launches;
  const bool gate = c.kind == ATTN_PRODUCT_GATED;
  return c.dtype == ATTN_BF16 ? launch_shape<__nv_bfloat16>(a, gate, stream) : launch_shape<__half>(a, gate, stream);
}

}  // namespace layer
}  // namespace attn
