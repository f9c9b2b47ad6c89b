// Matrix products on the CUDA cores, float32, with what follows them (product_tc.cu has the same for half types): everything is computed and kept in
// fp32.  Tiles of 128 x 128 (simt_product.cuh); a gated product's tile is 64 columns, its B 64 rows of Wg and the same rows of Wu, so that a thread's
// columns j and 64 + j are z and u of one element.  Where the tiles are few, a plain product is shared out along k and a kernel behind adds the parts
// in order and does the epilogue.  These are the sizes of debugging and gradient checks; bound by how many CTAs there are.
#include "activation.cuh"
#include "layer_launch.h"
#include "simt_product.cuh"

namespace attn {
namespace layer {

using namespace simt;

struct SimtResult {
  int rows, cols, k, pairs;
  int m_tiles, tile_end;
  Operand<float> a[kMaxPairs], b[kMaxPairs];
  float* out;
  long long ldo;
};
struct SimtArgs {
  SimtResult result[kMaxProducts];
  int results, tiles, act;
  int splits, split_blocks;      // of the blocks of all pairs, one pair behind the other
  float* parts;                  // [splits][tiles][128][128]
  const float *bias, *residual;
  long long ld_residual;
  Operand<float> b2;
  float* kept[2];
  long long ld_kept[2];
  float* out2;
  long long ldo2;
};

__device__ __forceinline__ int simt_result_of(const SimtArgs& g, int t) {
  int p = 0;
  while (p + 1 < g.results && t >= g.result[p].tile_end) ++p;
  return p;
}

// a plain result's element
template <int ACT>
__device__ __forceinline__ void finish(const SimtArgs& g, const SimtResult& s, int r, int c, float v) {
  if (g.bias != nullptr) v += g.bias[c];
  if (g.kept[0] != nullptr) g.kept[0][r * g.ld_kept[0] + c] = v;
  float a, d1, d2;
  activate<ACT, true, 0>(v, a, d1, d2);
  if (g.residual != nullptr) a += g.residual[r * g.ld_residual + c];
  s.out[r * s.ldo + c] = a;
}

template <int KIND>
__global__ void __launch_bounds__(256)
product_simt_kernel(const __grid_constant__ SimtArgs g) {
  __shared__ __align__(16) float as[2][kBlock * kPitch], bs[2][kBlock * kPitch];
  tc::pdl_wait();
  tc::pdl_trigger();
  constexpr bool kGate = KIND == ATTN_PRODUCT_GATED;
  constexpr int kCols = kGate ? kTile / 2 : kTile;
  const int t = (int)blockIdx.x, split = (int)blockIdx.y, p = simt_result_of(g, t);
  const SimtResult& s = g.result[p];
  const int local = t - (p == 0 ? 0 : g.result[p - 1].tile_end), nt = local / s.m_tiles, r0 = (local - nt * s.m_tiles) * kTile, c0 = nt * kCols;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  float2 sum[8][4];
  clear(sum);
  int buf = 0;
  const int blocks = (s.k + kBlock - 1) / kBlock;
  const int first = split * g.split_blocks, last = min(first + g.split_blocks, blocks * s.pairs);
  for (int q = 0; q < s.pairs; ++q) {
    const int k_begin = max(first - q * blocks, 0) * kBlock, k_end = min(min(last - q * blocks, blocks) * kBlock, s.k);
    if (k_begin >= k_end) continue;      // uniform
    const Operand<float>&a = s.a[q], &b = s.b[q];
    const bool ka = a.sk == 1, kb = b.sk == 1;
    auto bring_b = [&](int k0, float (&v)[8]) {
      if constexpr (kGate) {      // rows 0 to 63 of the block from Wg, the others from Wu
        const bool up = (kb ? threadIdx.x >> 1 : (threadIdx.x & 15) * 8) >= kCols;
        fetch(up ? g.b2 : b, up ? c0 - kCols : c0, k0, up ? s.cols : min(s.cols, c0 + kCols), k_end, v, kb);
      } else {
        fetch(b, c0, k0, s.cols, k_end, v, kb);
      }
    };
    accumulate(as, bs, buf, k_begin, k_end, [&](int k0, float (&v)[8]) { fetch(a, r0, k0, s.rows, k_end, v, ka); }, bring_b, ka, kb, sum);
  }
  float acc[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) { acc[i][2 * j] = sum[i][j].x; acc[i][2 * j + 1] = sum[i][j].y; }
  if (KIND == ATTN_PRODUCT_PLAIN && g.splits > 1) {
    float* at = g.parts + (((size_t)split * g.tiles + t) * kTile + ty * 8) * kTile;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<float4*>(at + i * kTile + 64 * h + tx * 4) = make_float4(acc[i][4 * h], acc[i][4 * h + 1], acc[i][4 * h + 2], acc[i][4 * h + 3]);
    return;
  }
  with_activation(g.act, [&](auto act) {
    constexpr int kAct = decltype(act)::value;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = r0 + ty * 8 + i;
      if (r >= s.rows) continue;
#pragma unroll
      for (int j = 0; j < (kGate ? 4 : 8); ++j) {
        const int c = c0 + (j >> 2) * 64 + tx * 4 + (j & 3);
        if (c >= s.cols) continue;
        [[maybe_unused]] float a, d1, d2;
        if constexpr (kGate) {
          const float z = acc[i][j], u = acc[i][4 + (j & 3)];
          if (g.kept[0] != nullptr) {
            g.kept[0][r * g.ld_kept[0] + c] = z;
            g.kept[1][r * g.ld_kept[1] + c] = u;
          }
          activate<kAct, true, 0>(z, a, d1, d2);
          s.out[r * s.ldo + c] = a * u;
        } else if constexpr (KIND == ATTN_PRODUCT_GATED_GRAD) {
          const float u = g.kept[1][r * g.ld_kept[1] + c];
          activate<kAct, true, 1>(g.kept[0][r * g.ld_kept[0] + c], a, d1, d2);
          s.out[r * s.ldo + c] = acc[i][j] * d1 * u;
          g.out2[r * g.ldo2 + c] = acc[i][j] * a;
        } else {
          finish<kAct>(g, s, r, c, acc[i][j]);
        }
      }
    }
  });
}

// a CTA has 16 rows of a tile
__global__ void __launch_bounds__(256)
join_simt_kernel(const __grid_constant__ SimtArgs g) {
  tc::pdl_wait();
  tc::pdl_trigger();
  const int t = (int)(blockIdx.x >> 3), p = simt_result_of(g, t);
  const SimtResult& s = g.result[p];
  const int local = t - (p == 0 ? 0 : g.result[p - 1].tile_end), nt = local / s.m_tiles, mt = local - nt * s.m_tiles;
  const int col = threadIdx.x & 127, c = nt * kTile + col;
  if (c >= s.cols) return;
  with_activation(g.act, [&](auto act) {
#pragma unroll 2
    for (int i = threadIdx.x >> 7; i < 16; i += 2) {
      const int row = (int)(blockIdx.x & 7) * 16 + i, r = mt * kTile + row;
      if (r >= s.rows) break;
      float v = 0.f;
#pragma unroll 8
      for (int q = 0; q < g.splits; ++q) v += from_l2(g.parts + (((size_t)q * g.tiles + t) * kTile + row) * kTile + col);
      finish<decltype(act)::value>(g, s, r, c, v);
    }
  });
}

// ---- host ---------------------------------------------------------------------------------------
// two CTAs an SM, at least 64 in k a share
static bool plan(const attn_products_t& c, SimtArgs& g) {
  const long long tile_cols = c.kind == ATTN_PRODUCT_GATED ? kTile / 2 : kTile;
  long long tiles = 0, blocks = 0;
  bool equal = true;
  g.results = 0;
  for (int i = 0; i < c.count; ++i) {
    const attn_product_t& p = c.product[i];
    if (p.rows == 0 || p.cols == 0 || p.k == 0) continue;
    SimtResult& s = g.result[g.results++];
    s.rows = p.rows; s.cols = p.cols; s.k = p.k; s.pairs = p.pairs;
    s.m_tiles = (int)(((long long)p.rows + kTile - 1) / kTile);
    tiles += s.m_tiles * ((p.cols + tile_cols - 1) / tile_cols);
    if (tiles > 0x7fffffff / 8) return false;
    s.tile_end = (int)tiles;
    const long long own = ((long long)p.k + kBlock - 1) / kBlock * p.pairs;
    equal = equal && (blocks == 0 || own == blocks);
    if (own > blocks) blocks = own;
  }
  if (blocks > 0x7fffffff) return false;
  g.tiles = (int)tiles;
  long long splits = 1;
  if (c.kind == ATTN_PRODUCT_PLAIN && equal && tiles > 0) {
    splits = 2 * kSms / tiles;
    if (splits > blocks / 4) splits = blocks / 4;
    if (splits > 256) splits = 256;
    if (splits < 1) splits = 1;
  }
  const long long each = blocks > 0 ? (blocks + splits - 1) / splits : 0;
  g.splits = each > 0 ? (int)((blocks + each - 1) / each) : 1;
  g.split_blocks = (int)each;
  return true;
}

size_t simt_parts_bytes(const attn_products_t& c) {
  SimtArgs g = {};
  return plan(c, g) && g.splits > 1 ? (size_t)g.splits * g.tiles * kTile * kTile * sizeof(float) : 0;
}

cudaError_t simt_products(const attn_products_t& c, float* parts, cudaStream_t stream, int* launches) {
  SimtArgs g = {};
  if (!plan(c, g)) return cudaErrorInvalidValue;
  if (g.results == 0) return cudaSuccess;
  int i = 0;
  for (int n = 0; n < c.count; ++n) {
    const attn_product_t& p = c.product[n];
    if (p.rows == 0 || p.cols == 0 || p.k == 0) continue;
    SimtResult& s = g.result[i++];
    for (int q = 0; q < p.pairs; ++q) {
      s.a[q] = c.form == ATTN_FORM_TN ? columns_of<float>(p.pair[q].a, p.pair[q].lda) : rows_of<float>(p.pair[q].a, p.pair[q].lda);
      s.b[q] = c.form == ATTN_FORM_NT ? rows_of<float>(p.pair[q].b, p.pair[q].ldb) : columns_of<float>(p.pair[q].b, p.pair[q].ldb);
    }
    s.out = static_cast<float*>(p.out);
    s.ldo = p.ldo;
  }
  g.act = c.activation;
  g.parts = parts;
  g.bias = static_cast<const float*>(c.bias);
  g.residual = static_cast<const float*>(c.residual);
  g.ld_residual = c.ld_residual;
  if (c.kind == ATTN_PRODUCT_GATED) g.b2 = rows_of<float>(c.b2, c.ldb2);
  for (int q = 0; q < 2; ++q) {
    g.kept[q] = static_cast<float*>(c.kept[q]);
    g.ld_kept[q] = c.ld_kept[q];
  }
  g.out2 = static_cast<float*>(c.out2);
  g.ldo2 = c.ldo2;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)g.tiles, (unsigned)g.splits);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaError_t e = c.kind == ATTN_PRODUCT_GATED        ? cudaLaunchKernelEx(&cfg, product_simt_kernel<ATTN_PRODUCT_GATED>, g)
                  : c.kind == ATTN_PRODUCT_GATED_GRAD ? cudaLaunchKernelEx(&cfg, product_simt_kernel<ATTN_PRODUCT_GATED_GRAD>, g)
                                                      : cudaLaunchKernelEx(&cfg, product_simt_kernel<ATTN_PRODUCT_PLAIN>, g);
  ++*launches;
  if (g.splits > 1 && e == cudaSuccess) {
    e = tc::launch_pdl(join_simt_kernel, (unsigned)g.tiles * 8, 256u, 0, stream, g);
    ++*launches;
  }
  return e;
}

}  // namespace layer
}  // namespace attn
