// The matrix products of the linear cross entropy on the tensor cores (f16/bf16, sm_100a): one persistent kernel, four uses.
//
//   use    A                      B                     result of a tile
//   LSE    x [n, d]               W [V, d]              per row: maximum, sum of exponentials; the target's logit
//   GRAD   x [n, d]               W [piece, d]          G = coef (exp(z - lse) - onehot), rounded to the input type
//   DX     G [n, piece]           W [piece, d], read by columns    dx (float between pieces)
//   DW     G [n, piece], by columns   x [n, d], by columns         dW rows of the piece
//
// A pair of CTAs (a cluster) owns a tile of 256 rows x 256 columns: either holds 128 rows of A and half of B's columns, one
// tcgen05.mma.cta_group::2 reads both.  A single CTA's 128 x 256 tile would stream 96 bytes per clock from L2 and read 96 more from
// shared memory for the product, above either's rate; the pair needs 64 of each.  A warp
// loads through a ring of six stages of 64 in k, one (in rank 0) issues the products, eight finish a tile from tensor memory while
// the next one accumulates in the other half of it.  The order of the tiles runs along the axis of the smaller operand first, so
// that the larger one is read from HBM once and the smaller one stays in L2.
//
// DX and DW have few tiles with long sums: dW of a piece of 8192 classes x 768 from 16384 rows is 96 tiles of 256 blocks of k for 74 pairs, two
// rounds, 65 % busy.  There the tiles of the last round are each shared out along k among several pairs (plan_shares), and a small kernel behind
// adds the parts in order (join_kernel).  Whole rounds stay as they are: pairs that are at the same place in k read the same rows of G and x from
// L2; equal, contiguous shares of all blocks left no pair idle, but took dW's product from 178 to 168 us only (that size), and dx's from
// 146 to between 167 and 187, since G then came from HBM several times.
//
// 16384 x 768 x 32000, bf16, each by itself: LSE 490 to 517 us (1 600 TFLOP/s, tensor pipe 87 % active); for a piece of 16128 classes GRAD 295 to 321
// (1 320, 68 %: it writes 475 MB), DW 250 to 275 (1 550, 83 %), DX 240 to 264 (1 610, 87 %), join 12 each.  In a loop the board is at its power limit.
//
// Logits are as exact as the tensor cores' own sums, which lose a little toward 0 with every block of k: 6e-7 of a logit at d = 768 and 2.1e-6 at 2048 (a
// library's product the same), 3e-7 and 1e-6 of the loss; the CUDA cores' 1e-8.
#include "lce_launch.h"
#include "tc_common.cuh"

#include <cstdio>
#include <mutex>

namespace attn {
namespace lce {

using namespace tc;

enum Use { LSE = 0, GRAD = 1, DX = 2, DW = 3 };

constexpr int kTileM = 256, kTileN = 256, kBlockK = 64;
constexpr int kHalfN = kTileN / 2;                             // columns of B in one CTA, and of a result in one half of its epilogue
constexpr int kStages = 6;
constexpr uint32_t kOperandBytes = 128 * 128;                  // 128 rows (or columns) of 64 in k, of A or of B, in one CTA
constexpr uint32_t kStageBytes = 2 * kOperandBytes;
constexpr uint32_t kStagingBytes = 128 * 128;                  // [128 rows][64 columns] of a result, for either half of the epilogue
constexpr int kEpilogueWarps = 8, kLoadWarp = 8, kIssueWarp = 9, kThreads = 320;
constexpr int KLCE = 32;                                       // kernel id inside device status codes: 32 + use

struct Control {
  uint64_t full[kStages], empty[kStages];      // full: rank 0's counts both CTAs' loads
  uint64_t acc_full[2], acc_empty[2];          // acc_empty: rank 0's counts both CTAs' warps
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
};
constexpr uint32_t kContentBytes = kStages * kStageBytes + 2 * kStagingBytes + sizeof(Control);
constexpr uint32_t kSmemBytes = kContentBytes + 1024;
static_assert(kSmemBytes <= 232448, "shared memory");

struct GemmMaps { CUtensorMap a, b, out; };

struct GemmArgs {
  int m_tiles, n_tiles, k_blocks;
  int rows, cols;                // of the result
  int m_fast;                    // tiles in sequence along the rows
  // LSE, GRAD
  const int64_t* targets;
  int first_col;                 // vocabulary index of column 0
  Partial* partial;
  float* target_logit;
  const float *lse, *coef;
  // DX, DW
  float* acc;                    // DX: [rows, cols], where there are several pieces
  int acc_in, acc_out;           // add it; leave the sum there instead of in the result
  const float* scale;
  int full, rest, splits, split_blocks;      // tiles taken whole; the others, each in `splits` shares of `split_blocks` blocks of k
  float* parts;                  // [rest x splits][2 CTAs][128][256], where there are several shares
  unsigned int* status;
};

template <typename T, int USE>
__global__ void __launch_bounds__(kThreads, 1)
lce_gemm_kernel(const __grid_constant__ GemmMaps maps, const GemmArgs g) {
  constexpr bool kByColumns = USE == DX || USE == DW;            // B, and in DW A, is read along its rows as k
  constexpr int KCODE = KLCE + USE;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t staging = smem_base + kStages * kStageBytes;
  Control* ctl = reinterpret_cast<Control*>(smem_raw + (smem_base - smem_u32(smem_raw)) + kStages * kStageBytes + 2 * kStagingBytes);
  float2* halves = reinterpret_cast<float2*>(smem_raw + (staging - smem_u32(smem_raw)));      // LSE, [2][128]: the upper half's (m, l)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  auto bar_full = [&](int s) { return smem_u32(&ctl->full[s]); };
  auto bar_empty = [&](int s) { return smem_u32(&ctl->empty[s]); };
  auto bar_acc_full = [&](int b) { return smem_u32(&ctl->acc_full[b]); };
  auto bar_acc_empty = [&](int b) { return smem_u32(&ctl->acc_empty[b]); };

  if (warp == kLoadWarp && lane == 0) {
    tma_prefetch_desc(&maps.a);
    tma_prefetch_desc(&maps.b);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full(s), 1);
      mbar_init(bar_empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_acc_full(b), 1);
      mbar_init(bar_acc_empty(b), 2 * kEpilogueWarps);
    }
    ctl->abort_flag = 0u;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == kIssueWarp) tmem_alloc_pair(smem_u32(&ctl->tmem_base), 512);
  tc_fence_before_sync();
  cluster_barrier();
  tc_fence_after_sync();
  const uint32_t tmem_base = ctl->tmem_base;
  volatile uint32_t* abort_flag = &ctl->abort_flag;
  pdl_wait();
  pdl_trigger();

  // what the pairs work on in turn: the tiles taken whole, then the shares of the others, all first shares first
  const int items = g.full + g.rest * g.splits;
  auto item_at = [&](int i, int& t, int& first_block, int& blocks) {
    t = i;
    first_block = 0;
    blocks = g.k_blocks;
    if (kByColumns && i >= g.full) {
      const int split = (i - g.full) / g.rest;
      t = i - split * g.rest;
      first_block = split * g.split_blocks;
      blocks = min(g.split_blocks, g.k_blocks - first_block);
    }
  };
  auto tile_at = [&](int t, int& mt, int& nt) {
    if (g.m_fast) { nt = t / g.m_tiles; mt = t - nt * g.m_tiles; }
    else { mt = t / g.n_tiles; nt = t - mt * g.n_tiles; }
  };

  if (warp == kLoadWarp) {
    if (lane == 0) {
      bool ok = true;
      int it = 0;
      for (int item = pair; item < items && ok; item += pairs) {
        int t, mt, nt, first_block, blocks;
        item_at(item, t, first_block, blocks);
        tile_at(t, mt, nt);
        const int m0 = mt * kTileM + (int)rank * 128, n0 = nt * kTileN + (int)rank * kHalfN;
        for (int kb = 0; kb < blocks; ++kb, ++it) {
          const int s = it % kStages;
          if (it >= kStages) {
            ok = mbar_wait(bar_empty(s), ((it / kStages) & 1) ^ 1, abort_flag, g.status, wait_code(KCODE, 1));
            if (!ok) break;
          }
          if (rank == 0) mbar_arrive_expect_tx(bar_full(s), 2 * kStageBytes);
          const uint32_t bar = map_rank(bar_full(s), 0), a = smem_base + s * kStageBytes, b = a + kOperandBytes;
          const int k0 = (first_block + kb) * kBlockK;
          if constexpr (USE == DW) {
            for (int i = 0; i < 2; ++i) tma_load_2d_pair(a + i * 8192, &maps.a, m0 + 64 * i, k0, bar);
          } else {
            tma_load_2d_pair(a, &maps.a, k0, m0, bar);
          }
          if constexpr (kByColumns) {
            for (int i = 0; i < 2; ++i) tma_load_2d_pair(b + i * 8192, &maps.b, n0 + 64 * i, k0, bar);
          } else {
            tma_load_2d_pair(b, &maps.b, k0, n0, bar);
          }
        }
      }
      // every product that reads this CTA's stages has completed, and told this CTA so, before it leaves
      for (int j = it > kStages ? it - kStages : 0; j < it && ok; ++j)
        ok = mbar_wait(bar_empty(j % kStages), (j / kStages) & 1, abort_flag, g.status, wait_code(KCODE, 5));
      if (!ok) {   // give copies already in flight a bounded chance to land before the CTA exits
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) { }
      }
    }
  } else if (warp == kIssueWarp) {
    if (rank == 0) {
      const uint32_t idesc = make_idesc(kTileM, kTileN, Pack<T>::kIsBf16, USE == DW ? 1 : 0, kByColumns ? 1 : 0);
      bool ok = true;
      int it = 0, i = 0;
      for (int item = pair; item < items && ok; item += pairs, ++i) {
        int t, first_block, blocks;
        item_at(item, t, first_block, blocks);
        const int buf = i & 1;
        if (i >= 2) {
          ok = __all_sync(0xffffffffu, mbar_wait(bar_acc_empty(buf), ((i >> 1) & 1) ^ 1, abort_flag, g.status, wait_code(KCODE, 2)));
          if (!ok) break;
          tc_fence_after_sync();
        }
        const uint32_t acc = tmem_base + (uint32_t)buf * 256u;
        for (int kb = 0; kb < blocks; ++kb, ++it) {
          const int s = it % kStages;
          ok = __all_sync(0xffffffffu, mbar_wait(bar_full(s), (it / kStages) & 1, abort_flag, g.status, wait_code(KCODE, 3)));
          if (!ok) break;
          tc_fence_after_sync();
          const uint32_t a = smem_base + s * kStageBytes, b = a + kOperandBytes;
          // rows along k: blocks of 64 rows (or columns) 8 KB apart, a step of 16 in k is 16 rows; else 32 bytes within a row
          const uint64_t da = smem_desc_sw128(a, USE == DW ? 8192 : 16, 1024), db = smem_desc_sw128(b, kByColumns ? 8192 : 16, 1024);
          constexpr uint64_t step_a = (USE == DW ? 2048 : 32) >> 4, step_b = (kByColumns ? 2048 : 32) >> 4;
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) mma_ss_pair(acc, da + ks * step_a, db + ks * step_b, idesc, (kb | ks) != 0);
            mma_commit_pair(bar_empty(s));
            if (kb + 1 == blocks) mma_commit_pair(bar_acc_full(buf));
          }
          __syncwarp();
        }
      }
    }
  } else {
    const int quarter = warp & 3, half = warp >> 2;
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t tile_smem = staging + (uint32_t)half * kStagingBytes;
    float scale = 1.f;
    if constexpr (kByColumns) scale = from_l2(g.scale);
    bool ok = true;
    int i = 0;
    for (int item = pair; item < items && ok; item += pairs, ++i) {
      int t, mt, nt, first_block, blocks;
      item_at(item, t, first_block, blocks);
      tile_at(t, mt, nt);
      const int buf = i & 1, r0 = mt * kTileM + (int)rank * 128, r = r0 + row;
      const int col0 = nt * kTileN + half * kHalfN;      // this half's first column
      const uint32_t acc = lane_addr + (uint32_t)buf * 256u + (uint32_t)(half * kHalfN);
      const bool in = r < g.rows;
      int target = -1;                                     // column of this row's target, counted from col0
      float lse = 0.f, coef = 0.f;
      if constexpr (USE == LSE || USE == GRAD) {
        if (in) {
          const int64_t y = from_l2(reinterpret_cast<const long long*>(g.targets) + r) - g.first_col - col0;
          if (y >= 0 && y < kHalfN) target = (int)y;
          if constexpr (USE == GRAD) { lse = from_l2(g.lse + r); coef = from_l2(g.coef + r); }
        }
      }
      // the eight warps go on, or give up, together: the barriers below need all of them
      ok = named_barrier_all(1, 32 * kEpilogueWarps, mbar_wait(bar_acc_full(buf), (i >> 1) & 1, abort_flag, g.status, wait_code(KCODE, 4)));
      if (!ok) break;
      tc_fence_after_sync();
      auto release = [&]() {                               // the accumulator is in registers
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_rank(bar_acc_empty(buf), 0));
      };

      if constexpr (USE == LSE) {
        float m = -INFINITY, l = 0.f;
        const int left = g.cols - col0;                    // valid columns of this half, where less than kHalfN
        for (int c = 0; c < kHalfN; c += 16) {
          uint32_t v[16];
          tmem_ld16(acc + c, v);
          tmem_ld_wait(v);
          if (c >= left) continue;                         // uniform
          float z[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) z[e] = c + e < left ? __uint_as_float(v[e]) : -INFINITY;
          if (__any_sync(0xffffffffu, (uint32_t)(target - c) < 16u)) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (target == c + e) g.target_logit[r] = z[e];
          }
          float mx = z[0];
#pragma unroll
          for (int e = 1; e < 16; ++e) mx = fmaxf(mx, z[e]);
          const float m_new = fmaxf(m, mx * kLog2e), ref = m_new == -INFINITY ? 0.f : m_new;      // logits of -inf alone: every term 0
          float sum = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) sum += ex2(fmaf(z[e], kLog2e, -ref));
          l = fmaf(l, m == -INFINITY ? 0.f : ex2(m - m_new), sum);
          m = m_new;
        }
        release();
        if (half == 1) halves[buf * 128 + row] = make_float2(m, l);
        named_barrier_sync(2, 32 * kEpilogueWarps);
        if (half == 0 && in) {
          const float2 o = halves[buf * 128 + row];
          const float m_all = fmaxf(m, o.x);
          const float l_all = fmaf(l, m == -INFINITY ? 0.f : ex2(m - m_all), o.y * (o.x == -INFINITY ? 0.f : ex2(o.x - m_all)));
          g.partial[(size_t)nt * g.rows + r] = Partial{m_all, l_all};
        }
      } else {
        const bool to_acc = USE == DX && g.acc_out;
        const bool part = kByColumns && item >= g.full && g.splits > 1;      // a share of a tile
        float* part_row = nullptr;
        if (part) part_row = g.parts + (((size_t)(item - g.full) * 2 + rank) * 128 + row) * 256 + half * 128;
#pragma unroll 1
        for (int c = 0; c < 128; c += 64) {
          uint32_t v[4][16];
#pragma unroll
          for (int q = 0; q < 4; ++q) tmem_ld16(acc + c + 16 * q, v[q]);
#pragma unroll
          for (int q = 0; q < 4; ++q) tmem_ld_wait(v[q]);
          if (c == 64) release();
          const int col = col0 + c;
          if (col >= g.cols) continue;                     // uniform
          float f[64];
#pragma unroll
          for (int e = 0; e < 64; ++e) f[e] = __uint_as_float(v[e >> 4][e & 15]);
          if constexpr (USE == GRAD) {
            // a row that does not count has a factor of 0 and G = 0, whatever its logits are
#pragma unroll
            for (int e = 0; e < 64; e += 2) {      // the difference first: exact where a row is sure of a class, so that P is 1 there
              const float2 t = __fmul2_rn(__fadd2_rn(make_float2(f[e], f[e + 1]), make_float2(-lse, -lse)), make_float2(kLog2e, kLog2e));
              const float2 p = __fmul2_rn(make_float2(ex2(t.x), ex2(t.y)), make_float2(coef, coef));
              f[e] = coef == 0.f ? 0.f : p.x;
              f[e + 1] = coef == 0.f ? 0.f : p.y;
            }
            if (__any_sync(0xffffffffu, (uint32_t)(target - c) < 64u)) {
#pragma unroll
              for (int e = 0; e < 64; ++e)
                if (target == c + e) f[e] -= coef;
            }
          } else {
            if (part) {
              float4* at = reinterpret_cast<float4*>(part_row + c);
#pragma unroll
              for (int q = 0; q < 16; ++q) __stcg(at + q, make_float4(f[4 * q], f[4 * q + 1], f[4 * q + 2], f[4 * q + 3]));
            } else if (USE == DX && (g.acc_in || to_acc) && in) {
              float4* at = reinterpret_cast<float4*>(g.acc + (size_t)r * g.cols + col);
#pragma unroll
              for (int q = 0; q < 16; ++q)
                if (col + 4 * q < g.cols) {                // cols is a multiple of 8
                  if (g.acc_in) {
                    const float4 x = __ldcg(at + q);
                    f[4 * q] += x.x; f[4 * q + 1] += x.y; f[4 * q + 2] += x.z; f[4 * q + 3] += x.w;
                  }
                  if (to_acc) __stcg(at + q, make_float4(f[4 * q], f[4 * q + 1], f[4 * q + 2], f[4 * q + 3]));
                }
            }
#pragma unroll
            for (int e = 0; e < 64; ++e) f[e] *= scale;
          }
          if (!to_acc && !part) {
            // through shared memory; the store before must have read it
            if (quarter == 0 && lane == 0) bulk_wait_group_read_all();
            named_barrier_sync(3 + half, 128);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t w[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) w[e] = Pack<T>::pack(f[16 * q + 2 * e], f[16 * q + 2 * e + 1]);
              store_op16(tile_smem, row, 16 * q, w);
            }
            fence_proxy_async_smem();
            named_barrier_sync(3 + half, 128);
            if (quarter == 0 && lane == 0) {
              tma_store_2d(&maps.out, tile_smem, col, r0);
              bulk_commit_group();
            }
          }
        }
      }
    }
    if (quarter == 0 && lane == 0) bulk_wait_group_read_all();
  }
  tc_fence_before_sync();
  cluster_barrier();      // no barrier or tensor memory of a CTA is used by the other one any more
  if (warp == kIssueWarp) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// The tiles in several shares.  A CTA has eight rows of one CTA's half of a tile; the parts are read once.
template <typename T>
__global__ void __launch_bounds__(256)
join_kernel(const GemmArgs g, T* out) {
  pdl_wait();
  pdl_trigger();
  const int tile = (int)(blockIdx.x >> 5), t = g.full + tile, rank = (int)(blockIdx.x >> 4) & 1, row0 = (int)(blockIdx.x & 15) * 8;
  int mt, nt;
  if (g.m_fast) { nt = t / g.m_tiles; mt = t - nt * g.m_tiles; }
  else { mt = t / g.n_tiles; nt = t - mt * g.n_tiles; }
  const float scale = from_l2(g.scale);
#pragma unroll
  for (int i = threadIdx.x; i < 8 * 64; i += 256) {
    const int row = row0 + (i >> 6), c = (i & 63) * 4, r = mt * kTileM + rank * 128 + row, col = nt * kTileN + c;
    if (r >= g.rows || col >= g.cols) continue;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int q = 0; q < g.splits; ++q) {
      const float4 x = from_l2(reinterpret_cast<const float4*>(g.parts + (((size_t)(q * g.rest + tile) * 2 + rank) * 128 + row) * 256 + c));
      v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
    }
    float4* acc = reinterpret_cast<float4*>(g.acc + (size_t)r * g.cols + col);
    if (g.acc_in) {
      const float4 x = from_l2(acc);
      v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
    }
    if (g.acc_out) *acc = v;
    else *reinterpret_cast<uint2*>(out + (size_t)r * g.cols + col) = make_uint2(Pack<T>::pack(v.x * scale, v.y * scale), Pack<T>::pack(v.z * scale, v.w * scale));
  }
}

// ---- host ---------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// [rows][cols] with `ld` elements from row to row, boxes of 64 columns x `box_rows`; outside of it loads give zeros and stores nothing
static bool encode(CUtensorMap* map, const void* p, bool bf16, long long rows, long long cols, long long ld, int box_rows) {
  const EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return false;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(p), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static int blocks_of(long long k) { return (int)((k + kBlockK - 1) / kBlockK); }
static long long tiles_of(long long rows, long long cols) { return (rows + kTileM - 1) / kTileM * ((cols + kTileN - 1) / kTileN); }

// DX and DW: the tiles of the last, part-filled round in shares along k, where that is shorter.  In blocks of k (0.28 us): a round of the shares takes
// split_blocks; shared tiles cost the launch behind them, 20, and a quarter of a block for every part that is written and read.  At least 8 blocks a share.
struct SharePlan { int full, rest, splits, split_blocks; };
static SharePlan plan_shares(long long rows, long long cols, long long k) {
  const int pairs = kSms / 2, tiles = (int)tiles_of(rows, cols), blocks = blocks_of(k);
  SharePlan best{tiles, 0, 1, blocks};
  const int rest = tiles % pairs;
  float least = (float)blocks;
  for (int s = 2; rest > 0 && rest * s <= 2 * pairs && blocks / s >= 8; ++s) {
    const int each = (blocks + s - 1) / s, shares = (blocks + each - 1) / each;      // none without blocks
    const float cost = (float)each * ((rest * shares + pairs - 1) / pairs) + 20.f + 0.25f * rest * shares;
    if (cost < least) {
      least = cost;
      best = SharePlan{tiles - rest, rest, shares, each};
    }
  }
  return best;
}
size_t tc_parts_bytes(long long rows, long long cols, long long k) {
  const SharePlan s = plan_shares(rows, cols, k);
  return s.splits > 1 ? (size_t)s.rest * s.splits * kTileM * kTileN * sizeof(float) : 0;
}

template <int USE>
static cudaError_t launch_use(const GemmMaps& maps, GemmArgs g, int dtype, long long k, void* out, cudaStream_t stream, int* launches) {
  g.m_tiles = (g.rows + kTileM - 1) / kTileM;
  g.n_tiles = (g.cols + kTileN - 1) / kTileN;
  g.k_blocks = blocks_of(k);
  g.m_fast = g.rows < g.cols;      // A, of `rows` rows, is the smaller operand
  const long long tiles = (long long)g.m_tiles * g.n_tiles;
  if (tiles > 0x3fffffffLL) return cudaErrorInvalidValue;
  SharePlan plan{(int)tiles, 0, 1, g.k_blocks};
  if (USE == DX || USE == DW) plan = plan_shares(g.rows, g.cols, k);
  g.full = plan.full; g.rest = plan.rest; g.splits = plan.splits; g.split_blocks = plan.split_blocks;
  const int items = g.full + g.rest * g.splits, pairs = items < kSms / 2 ? items : kSms / 2;
  static std::atomic<unsigned long long> smem_set[2];
  auto kern = dtype == 1 ? lce_gemm_kernel<__nv_bfloat16, USE> : lce_gemm_kernel<__half, USE>;
  cudaError_t e = set_smem_once(kern, kSmemBytes, smem_set[dtype == 1]);
  if (e == cudaSuccess) e = launch_pdl_cluster(kern, (unsigned)pairs * 2, kThreads, kSmemBytes, 2, stream, maps, g);
  ++*launches;
  if (g.splits > 1 && e == cudaSuccess) {
    const unsigned ctas = (unsigned)g.rest * 32;
    e = dtype == 1 ? launch_pdl(join_kernel<__nv_bfloat16>, ctas, 256u, 0, stream, g, (__nv_bfloat16*)out)
                   : launch_pdl(join_kernel<__half>, ctas, 256u, 0, stream, g, (__half*)out);
    ++*launches;
  }
  return e;
}

static const char* const kMapError = "cuTensorMapEncodeTiled refused a tensor";

int tc_tiles(int V) { return (V + kTileN - 1) / kTileN; }

cudaError_t tc_scores(const Problem& p, const Scores& s, cudaStream_t stream, int* launches, const char** err) {
  GemmMaps maps;
  GemmArgs g = {};
  const bool bf = p.dtype == 1;
  if (!encode(&maps.a, p.x, bf, p.n, p.d, p.d, 128) || !encode(&maps.b, p.w, bf, p.V, p.d, p.d, kHalfN)) {
    *err = kMapError;
    return cudaErrorInvalidValue;
  }
  maps.out = maps.a;      // not used
  g.rows = p.n; g.cols = p.V;
  g.targets = p.targets;
  g.partial = s.partial;
  g.target_logit = s.target_logit;
  g.status = p.status;
  return launch_use<LSE>(maps, g, p.dtype, p.d, nullptr, stream, launches);
}

cudaError_t tc_piece_grad(const Problem& p, const Piece& piece, const float* lse, const Coefficients& c, void* G, cudaStream_t stream, int* launches,
                          const char** err) {
  GemmMaps maps;
  GemmArgs g = {};
  const bool bf = p.dtype == 1;
  const void* w = static_cast<const uint16_t*>(p.w) + (size_t)piece.first * p.d;
  if (!encode(&maps.a, p.x, bf, p.n, p.d, p.d, 128) || !encode(&maps.b, w, bf, piece.cols, p.d, p.d, 128) ||
      !encode(&maps.out, G, bf, p.n, piece.cols, piece.ld, 128)) {
    *err = kMapError;
    return cudaErrorInvalidValue;
  }
  g.rows = p.n; g.cols = piece.cols;
  g.targets = p.targets;
  g.first_col = piece.first;
  g.lse = lse;
  g.coef = c.coef;
  g.status = p.status;
  return launch_use<GRAD>(maps, g, p.dtype, p.d, nullptr, stream, launches);
}

cudaError_t tc_piece_dx(const Problem& p, const Piece& piece, const Coefficients& c, const void* G, float* parts, float* acc, void* dx,
                        cudaStream_t stream, int* launches, const char** err) {
  GemmMaps maps;
  GemmArgs g = {};
  const bool bf = p.dtype == 1;
  const void* w = static_cast<const uint16_t*>(p.w) + (size_t)piece.first * p.d;
  if (!encode(&maps.a, G, bf, p.n, piece.cols, piece.ld, 128) || !encode(&maps.b, w, bf, piece.cols, p.d, p.d, 64) ||
      !encode(&maps.out, dx, bf, p.n, p.d, p.d, 128)) {
    *err = kMapError;
    return cudaErrorInvalidValue;
  }
  g.rows = p.n; g.cols = p.d;
  g.parts = parts;
  g.acc = acc;
  g.acc_in = !piece.is_first;
  g.acc_out = !piece.is_last;
  g.scale = c.scale;
  g.status = p.status;
  return launch_use<DX>(maps, g, p.dtype, piece.cols, dx, stream, launches);
}

cudaError_t tc_piece_dw(const Problem& p, const Piece& piece, const Coefficients& c, const void* G, const void* x, float* parts, void* dw,
                        cudaStream_t stream, int* launches, const char** err) {
  GemmMaps maps;
  GemmArgs g = {};
  const bool bf = p.dtype == 1;
  void* out = static_cast<uint16_t*>(dw) + (size_t)piece.first * p.d;
  if (!encode(&maps.a, G, bf, p.n, piece.cols, piece.ld, 64) || !encode(&maps.b, x, bf, p.n, p.d, p.d, 64) ||
      !encode(&maps.out, out, bf, piece.cols, p.d, p.d, 128)) {
    *err = kMapError;
    return cudaErrorInvalidValue;
  }
  g.rows = piece.cols; g.cols = p.d;
  g.parts = parts;
  g.scale = c.scale;
  g.status = p.status;
  return launch_use<DW>(maps, g, p.dtype, p.n, out, stream, launches);
}

}  // namespace lce
}  // namespace attn
