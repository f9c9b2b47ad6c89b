// Matrix products on the CUDA cores, float32, with what follows them (product_tc.cu has the same for half types): everything is computed and kept in
// fp32.  Tiles of 128 x 128 (simt_product.cuh), or of 64 x 64, 4 x 4 a thread, where the larger ones are few; a gated product's tile has half as many
// columns, its B that many rows of Wg and the same rows of Wu, so that a thread's columns of either half are z and u of one element.  Where the tiles are still
// few, a plain product is shared out along k and a kernel behind adds the parts in order and does the epilogue.  These are the sizes of debugging and gradient
// checks; bound by how many CTAs there are: 333 x 200 -> 515 14 us in 54 CTAs, 700 x 400 -> 900 37, 4096 x 1024 -> 1024 241 (36 TFLOP/s).
#include "activation.cuh"
#include "layer_launch.h"
#include "simt_product.cuh"

namespace attn {
namespace layer {

using namespace simt;

constexpr int kSmallTile = 64, kSmallBlock = 32, kSmallPitch = kSmallTile + 4;
template <int TILE> constexpr int kBlockOf = TILE == kTile ? kBlock : kSmallBlock;

// The small tile's eight elements of a [64][32] block of an operand, and its product: as fetch, put and accumulate of the large one.  Blocks of 32, since with
// few CTAs a block takes as long as its loads: 333 x 200 -> 515 14.4 us in blocks of 16.
__device__ __forceinline__ void fetch_small(const Operand<float>& o, int i0, int k0, int n_i, int n_k, float (&v)[8], bool k_dense) {
  const int t = threadIdx.x, i = i0 + (k_dense ? t >> 2 : (t & 7) * 8), k = k0 + (k_dense ? (t & 3) * 8 : t >> 3);
  const float* p = o.p + i * o.si + k * o.sk;
  if (o.wide && (k_dense ? i < n_i && k + 8 <= n_k : k < n_k && i + 8 <= n_i)) {
    const float4 a = from_l2(reinterpret_cast<const float4*>(p)), b = from_l2(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (k_dense ? i < n_i && k + e < n_k : k < n_k && i + e < n_i) ? p[e] : 0.f;
}
__device__ __forceinline__ void put_small(float* s, const float (&v)[8], bool k_dense) {
  const int t = threadIdx.x;
  if (k_dense) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s[((t & 3) * 8 + e) * kSmallPitch + (t >> 2)] = v[e];
  } else {
    float4* at = reinterpret_cast<float4*>(s + (t >> 3) * kSmallPitch + (t & 7) * 8);
    at[0] = make_float4(v[0], v[1], v[2], v[3]);
    at[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}
template <typename BringA, typename BringB>
__device__ __forceinline__ void accumulate_small(float (&as)[2][kSmallBlock * kSmallPitch], float (&bs)[2][kSmallBlock * kSmallPitch], int& buf, int k_begin, int k_end,
                                                 BringA bring_a, BringB bring_b, bool ka, bool kb, float2 (&sum)[4][2]) {
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  float va[8], vb[8];
  bring_a(k_begin, va);
  bring_b(k_begin, vb);
  for (int k0 = k_begin; k0 < k_end; k0 += kSmallBlock, buf ^= 1) {
    put_small(as[buf], va, ka);
    put_small(bs[buf], vb, kb);
    __syncthreads();
    if (k0 + kSmallBlock < k_end) {
      bring_a(k0 + kSmallBlock, va);
      bring_b(k0 + kSmallBlock, vb);
    }
#pragma unroll 16
    for (int k = 0; k < kSmallBlock; ++k) {
      const float4 a = *reinterpret_cast<const float4*>(&as[buf][k * kSmallPitch + ty * 4]);
      const float2 b[2] = {*reinterpret_cast<const float2*>(&bs[buf][k * kSmallPitch + tx * 2]), *reinterpret_cast<const float2*>(&bs[buf][k * kSmallPitch + 32 + tx * 2])};
      const float r[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) sum[i][j] = __ffma2_rn(make_float2(r[i], r[i]), b[j], sum[i][j]);
    }
  }
}

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
  int tile;                      // 128 or 64
  float* parts;                  // [splits][tiles][tile][tile]
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

template <int KIND, int TILE>
__global__ void __launch_bounds__(256, TILE == kTile ? 1 : 2)
product_simt_kernel(const __grid_constant__ SimtArgs g) {
  constexpr int R = TILE / 16, kHalf = TILE / 2, C = R / 2;      // a thread's rows, and columns of either half
  __shared__ __align__(16) float as[2][kBlockOf<TILE> * (TILE + 4)], bs[2][kBlockOf<TILE> * (TILE + 4)];
  tc::pdl_wait();
  tc::pdl_trigger();
  constexpr bool kGate = KIND == ATTN_PRODUCT_GATED;
  constexpr int kCols = kGate ? kHalf : TILE;
  const int t = (int)blockIdx.x, split = (int)blockIdx.y, p = simt_result_of(g, t);
  const SimtResult& s = g.result[p];
  const int local = t - (p == 0 ? 0 : g.result[p - 1].tile_end), nt = local / s.m_tiles, r0 = (local - nt * s.m_tiles) * TILE, c0 = nt * kCols;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  float2 sum[R][C];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < C; ++j) sum[i][j] = make_float2(0.f, 0.f);
  int buf = 0;
  constexpr int kB = kBlockOf<TILE>;
  const int blocks = (s.k + kB - 1) / kB;
  const int first = split * g.split_blocks, last = min(first + g.split_blocks, blocks * s.pairs);
  for (int q = 0; q < s.pairs; ++q) {
    const int k_begin = max(first - q * blocks, 0) * kB, k_end = min(min(last - q * blocks, blocks) * kB, s.k);
    if (k_begin >= k_end) continue;      // uniform
    const Operand<float>&a = s.a[q], &b = s.b[q];
    const bool ka = a.sk == 1, kb = b.sk == 1;
    auto bring = [&](const Operand<float>& o, int i0, int k0, int n_i, float (&v)[8], bool dense) {
      if constexpr (TILE == kTile) fetch(o, i0, k0, n_i, k_end, v, dense);
      else fetch_small(o, i0, k0, n_i, k_end, v, dense);
    };
    auto bring_a = [&](int k0, float (&v)[8]) { bring(a, r0, k0, s.rows, v, ka); };
    auto bring_b = [&](int k0, float (&v)[8]) {
      if constexpr (kGate) {      // the first half of the block's rows from Wg, the others from Wu
        const bool up = (TILE == kTile ? (kb ? threadIdx.x >> 1 : (threadIdx.x & 15) * 8) : (kb ? threadIdx.x >> 2 : (threadIdx.x & 7) * 8)) >= kCols;
        bring(up ? g.b2 : b, up ? c0 - kCols : c0, k0, up ? s.cols : min(s.cols, c0 + kCols), v, kb);
      } else {
        bring(b, c0, k0, s.cols, v, kb);
      }
    };
    if constexpr (TILE == kTile) accumulate(as, bs, buf, k_begin, k_end, bring_a, bring_b, ka, kb, sum);
    else accumulate_small(as, bs, buf, k_begin, k_end, bring_a, bring_b, ka, kb, sum);
  }
  float acc[R][R];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < C; ++j) { acc[i][2 * j] = sum[i][j].x; acc[i][2 * j + 1] = sum[i][j].y; }
  if (KIND == ATTN_PRODUCT_PLAIN && g.splits > 1) {
    float* at = g.parts + (((size_t)split * g.tiles + t) * TILE + ty * R) * TILE;
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < R; j += 2) *reinterpret_cast<float2*>(at + i * TILE + j / C * kHalf + tx * C + j % C) = make_float2(acc[i][j], acc[i][j + 1]);
    return;
  }
  with_activation(g.act, [&](auto act) {
    constexpr int kAct = decltype(act)::value;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int r = r0 + ty * R + i;
      if (r >= s.rows) continue;
#pragma unroll
      for (int j = 0; j < (kGate ? C : R); ++j) {
        const int c = c0 + j / C * kHalf + tx * C + j % C;
        if (c >= s.cols) continue;
        [[maybe_unused]] float a, d1, d2;
        if constexpr (kGate) {
          const float z = acc[i][j], u = acc[i][C + j % C];
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

// a CTA has 256 elements of a tile
__global__ void __launch_bounds__(256)
join_simt_kernel(const __grid_constant__ SimtArgs g) {
  tc::pdl_wait();
  tc::pdl_trigger();
  const int shift = g.tile == kTile ? 7 : 6, per_tile = 2 * shift - 8, t = (int)(blockIdx.x >> per_tile), p = simt_result_of(g, t);
  const int i = (int)(blockIdx.x - ((unsigned)t << per_tile)) * 256 + (int)threadIdx.x;
  const SimtResult& s = g.result[p];
  const int local = t - (p == 0 ? 0 : g.result[p - 1].tile_end), nt = local / s.m_tiles, mt = local - nt * s.m_tiles;
  const int r = (mt << shift) + (i >> shift), c = (nt << shift) + (i & (g.tile - 1));
  if (r >= s.rows || c >= s.cols) return;
  float v = 0.f;
#pragma unroll 8
  for (int q = 0; q < g.splits; ++q) v += from_l2(g.parts + (((size_t)q * g.tiles + t) << 2 * shift) + i);
  with_activation(g.act, [&](auto act) { finish<decltype(act)::value>(g, s, r, c, v); });
}

// ---- host ---------------------------------------------------------------------------------------
// Tiles of 128 where they fill the GPU once, else of 64; then shares of k, two CTAs an SM and at least 128 in k a share, below which
// the launch that adds them costs more.
static bool plan(const attn_products_t& c, SimtArgs& g) {
  long long tiles = 0, blocks = 0;
  bool equal = true;
  for (g.tile = kTile;; g.tile = kSmallTile) {
    equal = true;
    const long long tile_cols = c.kind == ATTN_PRODUCT_GATED ? g.tile / 2 : g.tile;
    g.results = 0;
    tiles = blocks = 0;
    for (int i = 0; i < c.count; ++i) {
      const attn_product_t& p = c.product[i];
      if (p.rows == 0 || p.cols == 0 || p.k == 0) continue;
      SimtResult& s = g.result[g.results++];
      s.rows = p.rows; s.cols = p.cols; s.k = p.k; s.pairs = p.pairs;
      s.m_tiles = (int)(((long long)p.rows + g.tile - 1) / g.tile);
      tiles += s.m_tiles * ((p.cols + tile_cols - 1) / tile_cols);
      if (tiles > 0x7fffffff / 64) return false;
      s.tile_end = (int)tiles;
      const long long block = g.tile == kTile ? kBlock : kSmallBlock, own = (p.k + block - 1) / block * p.pairs;
      equal = equal && (blocks == 0 || own == blocks);
      if (own > blocks) blocks = own;
    }
    if (g.tile == kSmallTile || tiles >= kSms) break;
  }
  if (blocks > 0x7fffffff) return false;
  g.tiles = (int)tiles;
  long long splits = 1;
  if (c.kind == ATTN_PRODUCT_PLAIN && equal && tiles > 0) {
    splits = 2 * kSms / tiles;
    if (splits > blocks / (g.tile == kTile ? 8 : 4)) splits = blocks / (g.tile == kTile ? 8 : 4);
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
  return plan(c, g) && g.splits > 1 ? (size_t)g.splits * g.tiles * g.tile * g.tile * sizeof(float) : 0;
}

template <int TILE>
static cudaError_t launch_kind(const cudaLaunchConfig_t& cfg, int kind, const SimtArgs& g) {
  if (kind == ATTN_PRODUCT_GATED) return cudaLaunchKernelEx(&cfg, product_simt_kernel<ATTN_PRODUCT_GATED, TILE>, g);
  if (kind == ATTN_PRODUCT_GATED_GRAD) return cudaLaunchKernelEx(&cfg, product_simt_kernel<ATTN_PRODUCT_GATED_GRAD, TILE>, g);
  return cudaLaunchKernelEx(&cfg, product_simt_kernel<ATTN_PRODUCT_PLAIN, TILE>, g);
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
  cudaError_t e = g.tile == kTile ? launch_kind<kTile>(cfg, c.kind, g) : launch_kind<kSmallTile>(cfg, c.kind, g);
  ++*launches;
  if (g.splits > 1 && e == cudaSuccess) {
    e = tc::launch_pdl(join_simt_kernel, (unsigned)(g.tiles * (g.tile * g.tile / 256)), 256u, 0, stream, g);
    ++*launches;
  }
  return e;
}

}  // namespace layer
}  // namespace attn
