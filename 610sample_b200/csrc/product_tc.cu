// Matrix products on the tensor cores (f16/bf16, sm_100a) with what follows them in their epilogue: one persistent kernel.
//
//   form   A                      B
//   NT     [rows, k]              [cols, k]
//   NN     [rows, k]              [k, cols], read by columns
//   TN     [k, rows], by columns  [k, cols], by columns
//
// A pair of CTAs (a cluster) owns a tile of 256 x 256: either holds 128 rows of A and half of B's columns, and one tcgen05.mma.cta_group::2
// reads both.  A warp loads through a ring of stages of 64 in k, one (in rank 0) issues the products, eight finish a tile from tensor memory
// while the next one accumulates in the other half of it.  A result is the sum of up to four products, one behind the other along k.
//
// kind    what the eight warps do with a tile, 64 columns at a time in 16 KB of shared memory per buffer and half of the warps
// PLAIN   z = sum + bias, activation, residual.  The residual is loaded into the buffer that the result leaves from
// KEEP    the same with z kept
// GATED   128 columns: CTA 0 holds rows of Wg as its half of B and CTA 1 the same rows of Wu, so that columns j and 128 + j of the accumulator are z and u
// KEPT    the same with z and u kept (three buffers)
// GRAD    z and u are loaded into the buffers that their gradients leave from
// A buffer's next input is asked for as soon as its last result has been read, so it is on its way while the next tile accumulates.
//
// The tiles of several results are one list, so that three small ones (the weights' gradients of a gated block at 16384 x 768 x 2048: 24 tiles each
// of 256 blocks of k) fill the 74 pairs once.  Where the last round of tiles stays short of them, its tiles are shared out along k and a small kernel behind adds
// the parts in order and does the epilogue (PLAIN and KEEP).
#include "activation.cuh"
#include "layer_launch.h"
#include "product_common.cuh"
#include "tc_common.cuh"

namespace attn {
namespace layer {

using namespace tc;
using namespace product;

enum Kind { PLAIN = 0, KEEP = 1, GATED = 2, KEPT = 3, GRAD = 4 };

constexpr int kHalfN = kTileN / 2;
constexpr uint32_t kOperandBytes = 128 * 128;                  // 128 rows (or columns) of 64 in k, of A or of B, in one CTA
constexpr uint32_t kStageBytes = 2 * kOperandBytes;
constexpr uint32_t kBufferBytes = 128 * 128;                   // [128 rows][64 columns] of a result or an input
constexpr int kEpilogueWarps = 8, kLoadWarp = 8, kIssueWarp = 9, kThreads = 320;
constexpr int KPRODUCT = 40;                                   // kernel id inside device status codes: 40 + kind

template <int KIND> constexpr int kBuffersOf = KIND == KEPT ? 3 : KIND == KEEP || KIND == GRAD ? 2 : 1;
template <int KIND> constexpr int kStagesOf = 7 - kBuffersOf<KIND>;

template <int STAGES>
struct Control {
  uint64_t full[STAGES], empty[STAGES];        // full: rank 0's counts both CTAs' loads
  uint64_t acc_full[2], acc_empty[2];          // acc_empty: rank 0's counts both CTAs' warps
  uint64_t in_full[2];                         // inputs of the epilogue, by half
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
};
template <int KIND> constexpr uint32_t smem_bytes() {
  return kStagesOf<KIND> * kStageBytes + 2 * kBuffersOf<KIND> * kBufferBytes + sizeof(Control<kStagesOf<KIND>>) + 1024;
}
static_assert(smem_bytes<PLAIN>() <= 232448 && smem_bytes<KEEP>() <= 232448 && smem_bytes<KEPT>() <= 232448, "shared memory");

struct Maps {
  CUtensorMap a[kMaxFactors], b[kMaxFactors];
  CUtensorMap out[kMaxProducts];
  CUtensorMap side[2];           // PLAIN, KEEP: residual, z.  KEPT, GRAD: z, u
  CUtensorMap out2;              // GRAD
};

struct Result {
  int rows, cols;
  int m_tiles, n_tiles, m_fast;  // m_fast: tiles in sequence along the rows
  int tile_end;                  // in the list of all tiles
  int first_factor, factor_blocks, blocks;      // blocks of k of one product of the sum, and of all of them
  void* out;
  long long ldo;
};
struct ProductArgs {
  Result result[kMaxProducts];
  int results, act;
  int full, rest, splits, split_blocks;      // tiles taken whole; the others, each in `splits` shares of `split_blocks` blocks of k
  float* parts;                  // [rest x splits][2 CTAs][128][256], where there are several shares
  const void *bias, *residual;
  long long ld_residual;
  void* z;
  long long ld_z;
  unsigned int* status;
};

struct Item { int t, first_block, blocks; bool part; };
__device__ __forceinline__ int result_of(const ProductArgs& g, int t) {
  int p = 0;
  while (p + 1 < g.results && t >= g.result[p].tile_end) ++p;
  return p;
}
__device__ __forceinline__ Item item_at(const ProductArgs& g, int i) {
  if (i < g.full || g.splits == 1) return {i, 0, g.result[result_of(g, i)].blocks, false};
  const int split = (i - g.full) / g.rest, first = split * g.split_blocks, t = i - split * g.rest;
  return {t, first, min(g.split_blocks, g.result[0].blocks - first), true};      // results that share tiles have as many blocks each
}
__device__ __forceinline__ void tile_at(const Result& r, int tiles_before, int t, int& mt, int& nt) {
  t -= tiles_before;
  if (r.m_fast) { nt = t / r.m_tiles; mt = t - nt * r.m_tiles; }
  else { mt = t / r.n_tiles; nt = t - mt * r.n_tiles; }
}
__device__ __forceinline__ int tiles_before(const ProductArgs& g, int p) { return p == 0 ? 0 : g.result[p - 1].tile_end; }

// bias[col .. col + 16) in fp32; zeros outside
template <typename T>
__device__ __forceinline__ void bias16(const void* bias, int col, int cols, float (&b)[16]) {
  const T* p = static_cast<const T*>(bias) + col;
  if (col + 16 <= cols && reinterpret_cast<uintptr_t>(bias) % 16 == 0) {      // col is a multiple of 16
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[q];
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = Pack<T>::unpack(w[e]);
        b[8 * q + 2 * e] = f.x; b[8 * q + 2 * e + 1] = f.y;
      }
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) b[e] = col + e < cols ? Elem<T>::to_float(p[e]) : 0.f;
}

template <typename T>
__device__ __forceinline__ void unpack16(const uint32_t (&w)[8], float (&f)[16]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float2 v = Pack<T>::unpack(w[e]);
    f[2 * e] = v.x; f[2 * e + 1] = v.y;
  }
}
template <typename T>
__device__ __forceinline__ void put16(uint32_t buffer, int row, int col, const float (&f)[16]) {
  uint32_t w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = Pack<T>::pack(f[2 * e], f[2 * e + 1]);
  store_op16(buffer, row, col, w);
}
template <typename T>
__device__ __forceinline__ void keep16(uint32_t buffer, int row, int col, const float (&f)[16]) {
  float v[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] = within<T>(f[e]);
  put16<T>(buffer, row, col, v);
}

template <typename T, int FORM, int KIND>
__global__ void __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ Maps maps, const __grid_constant__ ProductArgs g) {
  constexpr int kStages = kStagesOf<KIND>, kBuffers = kBuffersOf<KIND>;
  constexpr bool kAByColumns = FORM == ATTN_FORM_TN, kBByColumns = FORM != ATTN_FORM_NT, kGate = KIND == GATED || KIND == KEPT;
  constexpr int kChunks = kGate ? 1 : 2;                         // of 64 columns of a result, for either half
  constexpr int KCODE = KPRODUCT + KIND;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t buffers = smem_base + kStages * kStageBytes;
  typedef Control<kStages> Ctl;
  Ctl* ctl = reinterpret_cast<Ctl*>(smem_raw + (smem_base - smem_u32(smem_raw)) + kStages * kStageBytes + 2 * kBuffers * kBufferBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  auto bar_full = [&](int s) { return smem_u32(&ctl->full[s]); };
  auto bar_empty = [&](int s) { return smem_u32(&ctl->empty[s]); };
  auto bar_acc_full = [&](int b) { return smem_u32(&ctl->acc_full[b]); };
  auto bar_acc_empty = [&](int b) { return smem_u32(&ctl->acc_empty[b]); };
  auto bar_in_full = [&](int h) { return smem_u32(&ctl->in_full[h]); };

  if (warp == kLoadWarp && lane == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full(s), 1);
      mbar_init(bar_empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_acc_full(b), 1);
      mbar_init(bar_acc_empty(b), 2 * kEpilogueWarps);
      mbar_init(bar_in_full(b), 1);
    }
    ctl->abort_flag = 0u;
    fence_barrier_init();
    fence_proxy_async_smem();
    tma_prefetch_desc(&maps.a[0]);
    tma_prefetch_desc(&maps.b[0]);
  }
  if (warp == kIssueWarp) tmem_alloc_pair(smem_u32(&ctl->tmem_base), 512);
  tc_fence_before_sync();
  cluster_barrier();
  tc_fence_after_sync();
  const uint32_t tmem_base = ctl->tmem_base;
  volatile uint32_t* abort_flag = &ctl->abort_flag;
  pdl_wait();
  pdl_trigger();

  const int items = g.full + g.rest * g.splits;

  if (warp == kLoadWarp) {
    if (lane == 0) {
      bool ok = true;
      int it = 0;
      for (int i = pair; i < items && ok; i += pairs) {
        const Item item = item_at(g, i);
        const int p = result_of(g, item.t);
        const Result& r = g.result[p];
        int mt, nt;
        tile_at(r, tiles_before(g, p), item.t, mt, nt);
        const int m0 = mt * kTileM + (int)rank * 128, n0 = kGate ? nt * kHalfN : nt * kTileN + (int)rank * kHalfN;
        int factor = item.first_block / r.factor_blocks, kb = item.first_block - factor * r.factor_blocks;
        for (int left = item.blocks; left > 0; --left, ++it) {
          const int s = it % kStages;
          if (it >= kStages) {
            ok = mbar_wait(bar_empty(s), ((it / kStages) & 1) ^ 1, abort_flag, g.status, wait_code(KCODE, 1));
            if (!ok) break;
          }
          if (rank == 0) mbar_arrive_expect_tx(bar_full(s), 2 * kStageBytes);
          const uint32_t bar = map_rank(bar_full(s), 0), a = smem_base + s * kStageBytes, b = a + kOperandBytes;
          const CUtensorMap* ma = &maps.a[r.first_factor + factor];
          const CUtensorMap* mb = &maps.b[kGate ? (int)rank : r.first_factor + factor];
          const int k0 = kb * kBlockK;
          if constexpr (kAByColumns) {
            for (int j = 0; j < 2; ++j) tma_load_2d_pair(a + j * 8192, ma, m0 + 64 * j, k0, bar);
          } else {
            tma_load_2d_pair(a, ma, k0, m0, bar);
          }
          if constexpr (kBByColumns) {
            for (int j = 0; j < 2; ++j) tma_load_2d_pair(b + j * 8192, mb, n0 + 64 * j, k0, bar);
          } else {
            tma_load_2d_pair(b, mb, k0, n0, bar);
          }
          if (++kb == r.factor_blocks) { kb = 0; ++factor; }
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
      const uint32_t idesc = make_idesc(kTileM, kTileN, Pack<T>::kIsBf16, kAByColumns ? 1 : 0, kBByColumns ? 1 : 0);
      bool ok = true;
      int it = 0, n = 0;
      for (int i = pair; i < items && ok; i += pairs, ++n) {
        const int blocks = item_at(g, i).blocks, buf = n & 1;
        if (n >= 2) {
          ok = __all_sync(0xffffffffu, mbar_wait(bar_acc_empty(buf), ((n >> 1) & 1) ^ 1, abort_flag, g.status, wait_code(KCODE, 2)));
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
          // by columns: blocks of 64 rows (or columns) 8 KB apart, a step of 16 in k is 16 rows; else 32 bytes within a row
          const uint64_t da = smem_desc_sw128(a, kAByColumns ? 8192 : 16, 1024), db = smem_desc_sw128(b, kBByColumns ? 8192 : 16, 1024);
          constexpr uint64_t step_a = (kAByColumns ? 2048 : 32) >> 4, step_b = (kBByColumns ? 2048 : 32) >> 4;
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
    const bool leader = quarter == 0 && lane == 0;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t buf0 = buffers + (uint32_t)(half * kBuffers) * kBufferBytes, buf1 = buf0 + kBufferBytes, buf2 = buf1 + kBufferBytes;
    const bool inputs = KIND == GRAD || ((KIND == PLAIN || KIND == KEEP) && g.residual != nullptr);
    // the leader: inputs of chunk c of item i, where there is such an item and it is a whole tile (the join kernel finishes the others).  Boxes may
    // lie outside of the tensor, and are zeros there
    auto ask = [&](int i, int c) {
      if (i >= items) return;
      const Item item = item_at(g, i);
      if (item.part) return;
      const int p = result_of(g, item.t);
      int mt, nt;
      tile_at(g.result[p], tiles_before(g, p), item.t, mt, nt);
      const int r0 = mt * kTileM + (int)rank * 128, col = nt * kTileN + half * kHalfN + 64 * c;
      const uint32_t bar = map_rank(bar_in_full(half), rank);
      mbar_arrive_expect_tx(bar_in_full(half), (KIND == GRAD ? 2 : 1) * kBufferBytes);
      tma_load_2d_pair(buf0, &maps.side[0], col, r0, bar);
      if constexpr (KIND == GRAD) tma_load_2d_pair(buf1, &maps.side[1], col, r0, bar);
    };
    if (inputs && leader) ask(pair, 0);
    // A wait for inputs that gives up is this half's alone: it goes on, with what is there, to the next tile, where all warps hear of it
    bool ok = true, alive = true;
    int n = 0, asked = 0;                                  // asked: chunks with inputs so far
    for (int i = pair; i < items && ok; i += pairs, ++n) {
      const Item item = item_at(g, i);
      const int p = result_of(g, item.t);
      const Result& r = g.result[p];
      int mt, nt;
      tile_at(r, tiles_before(g, p), item.t, mt, nt);
      const int buf = n & 1, r0 = mt * kTileM + (int)rank * 128;
      // this half's first column, of the result and of the accumulator
      const int col0 = kGate ? nt * kHalfN + half * 64 : nt * kTileN + half * kHalfN;
      const uint32_t acc = lane_addr + (uint32_t)buf * 256u + (uint32_t)(kGate ? half * 64 : half * kHalfN);
      // the eight warps go on, or give up, together: the barriers below need all of them
      ok = named_barrier_all(1, 32 * kEpilogueWarps, mbar_wait(bar_acc_full(buf), (n >> 1) & 1, abort_flag, g.status, wait_code(KCODE, 4)) && alive);
      if (!ok) break;
      tc_fence_after_sync();
      auto release = [&]() {                               // the accumulator is in registers
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_rank(bar_acc_empty(buf), 0));
      };
      float* part_row = nullptr;
      if (item.part) part_row = g.parts + (((size_t)(i - g.full) * 2 + rank) * 128 + row) * 256 + half * kHalfN;

#pragma unroll 1
      for (int c = 0; c < kChunks; ++c) {
        const int col = col0 + 64 * c;
        const bool in = col < r.cols;                      // uniform
        if (!item.part) {
          // the buffers: the stores before have read them, and the inputs are there
          if (inputs) {
            const bool there = mbar_wait(bar_in_full(half), asked & 1, abort_flag, g.status, wait_code(KCODE, 6));
            alive = named_barrier_all(3 + half, 128, there) && alive;
            ++asked;
          } else {
            if (leader) bulk_wait_group_read_all();
            named_barrier_sync(3 + half, 128);
          }
        }
#pragma unroll
        for (int s = 0; s < 64; s += 32) {
          uint32_t v[32], v2[32];
          tmem_ld32(acc + 64 * c + s, v);
          if constexpr (kGate) tmem_ld32(acc + 128 + s, v2);
          tmem_ld_wait32(v);
          if constexpr (kGate) tmem_ld_wait32(v2);
          if (c + 1 == kChunks && s == 32) release();
          if (!in) continue;
          if (item.part) {
            float4* at = reinterpret_cast<float4*>(part_row + 64 * c + s);
#pragma unroll
            for (int q = 0; q < 8; ++q)
              __stcg(at + q, make_float4(__uint_as_float(v[4 * q]), __uint_as_float(v[4 * q + 1]), __uint_as_float(v[4 * q + 2]), __uint_as_float(v[4 * q + 3])));
            continue;
          }
#pragma unroll
          for (int q = 0; q < 32; q += 16) {
            float f[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) f[e] = __uint_as_float(v[q + e]);
            if constexpr (kGate) {
              float u[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) u[e] = __uint_as_float(v2[q + e]);
              if constexpr (KIND == KEPT) {
                keep16<T>(buf1, row, s + q, f);
                keep16<T>(buf2, row, s + q, u);
              }
              with_activation(g.act, [&](auto act) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  float a, d1, d2;
                  activate<decltype(act)::value, false, 0>(f[e], a, d1, d2);
                  f[e] = a * u[e];
                }
              });
              put16<T>(buf0, row, s + q, f);
            } else if constexpr (KIND == GRAD) {
              uint32_t wz[8], wu[8];
              load_op16(buf0, row, s + q, wz);
              load_op16(buf1, row, s + q, wu);
              float z[16], u[16];
              unpack16<T>(wz, z);
              unpack16<T>(wu, u);
              with_activation(g.act, [&](auto act) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  float a, d1, d2;
                  activate<decltype(act)::value, false, 1>(z[e], a, d1, d2);
                  z[e] = f[e] * d1 * u[e];
                  u[e] = f[e] * a;
                }
              });
              put16<T>(buf0, row, s + q, z);
              put16<T>(buf1, row, s + q, u);
            } else {
              if (g.bias != nullptr) {
                float b[16];
                bias16<T>(g.bias, col + s + q, r.cols, b);
#pragma unroll
                for (int e = 0; e < 16; ++e) f[e] += b[e];
              }
              if constexpr (KIND == KEEP) keep16<T>(buf1, row, s + q, f);
              if (g.act != ACT_NONE)
                with_activation(g.act, [&](auto act) {
#pragma unroll
                  for (int e = 0; e < 16; ++e) {
                    float d1, d2;
                    activate<decltype(act)::value, false, 0>(f[e], f[e], d1, d2);
                  }
                });
              if (inputs) {
                uint32_t w[8];
                float x[16];
                load_op16(buf0, row, s + q, w);
                unpack16<T>(w, x);
#pragma unroll
                for (int e = 0; e < 16; ++e) f[e] += x[e];
              }
              put16<T>(buf0, row, s + q, f);
            }
          }
        }
        if (item.part) continue;
        fence_proxy_async_smem();
        named_barrier_sync(3 + half, 128);
        if (leader) {
          if (in) {
            tma_store_2d(&maps.out[p], buf0, col, r0);
            if constexpr (KIND == KEEP) tma_store_2d(&maps.side[1], buf1, col, r0);
            if constexpr (KIND == KEPT) {
              tma_store_2d(&maps.side[0], buf1, col, r0);
              tma_store_2d(&maps.side[1], buf2, col, r0);
            }
            if constexpr (KIND == GRAD) tma_store_2d(&maps.out2, buf1, col, r0);
            bulk_commit_group();
          }
          if (inputs) {
            bulk_wait_group_read_all();
            if (c + 1 < kChunks) ask(i, c + 1);
            else ask(i + pairs, 0);
          }
        }
      }
    }
    if (leader) {
      if (!ok || !alive) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) { }
      }
      bulk_wait_group_read_all();
    }
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
join_kernel(const __grid_constant__ ProductArgs g) {
  pdl_wait();
  pdl_trigger();
  const int tile = (int)(blockIdx.x >> 5), t = g.full + tile, rank = (int)(blockIdx.x >> 4) & 1, row0 = (int)(blockIdx.x & 15) * 8;
  const int p = result_of(g, t);
  const Result& res = g.result[p];
  int mt, nt;
  tile_at(res, tiles_before(g, p), t, mt, nt);
#pragma unroll
  for (int i = threadIdx.x; i < 8 * 64; i += 256) {
    const int row = row0 + (i >> 6), c = (i & 63) * 4, r = mt * kTileM + rank * 128 + row, col = nt * kTileN + c;
    if (r >= res.rows || col >= res.cols) continue;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int q = 0; q < g.splits; ++q) {
      const float4 x = from_l2(reinterpret_cast<const float4*>(g.parts + (((size_t)(q * g.rest + tile) * 2 + rank) * 128 + row) * 256 + c));
      v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
    }
    // rows start at 16 bytes and col is a multiple of 4
    const int width = min(4, res.cols - col);
    auto pack = [](const float (&f)[4]) { return make_uint2(Pack<T>::pack(f[0], f[1]), Pack<T>::pack(f[2], f[3])); };
    auto put = [&](void* base, long long ld, const float (&f)[4]) {
      T* at = static_cast<T*>(base) + r * ld + col;
      if (width == 4) *reinterpret_cast<uint2*>(at) = pack(f);
      else
        for (int e = 0; e < width; ++e) at[e] = Elem<T>::from_float(f[e]);
    };
    if (g.bias != nullptr)
      for (int e = 0; e < width; ++e) v[e] += Elem<T>::to_float(static_cast<const T*>(g.bias)[col + e]);
    if (g.z != nullptr) {
      float k[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) k[e] = within<T>(v[e]);
      put(g.z, g.ld_z, k);
    }
    with_activation(g.act, [&](auto act) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float d1, d2;
        activate<decltype(act)::value, false, 0>(v[e], v[e], d1, d2);
      }
    });
    if (g.residual != nullptr)
      for (int e = 0; e < width; ++e) v[e] += Elem<T>::to_float(static_cast<const T*>(g.residual)[r * g.ld_residual + col + e]);
    put(res.out, res.ldo, v);
  }
}

// ---- host ---------------------------------------------------------------------------------------
static int kind_of(const attn_products_t& c) {
  if (c.kind == ATTN_PRODUCT_GATED) return c.kept[0] != nullptr ? KEPT : GATED;
  if (c.kind == ATTN_PRODUCT_GATED_GRAD) return GRAD;
  return c.kept[0] != nullptr ? KEEP : PLAIN;
}

// Results, tiles and shares of a call; results without rows, columns or k have no tiles
static long long plan(const attn_products_t& c, ProductArgs& g) {
  const int kind = kind_of(c), tile_n = kind == GATED || kind == KEPT ? kHalfN : kTileN;
  long long tiles = 0;
  bool equal = true;
  int factors = 0;
  g.results = 0;
  for (int i = 0; i < c.count; ++i) {
    const attn_product_t& p = c.product[i];
    if (p.rows == 0 || p.cols == 0 || p.k == 0) continue;
    Result& r = g.result[g.results];
    r.rows = p.rows; r.cols = p.cols;
    r.m_tiles = (int)(((long long)p.rows + kTileM - 1) / kTileM);
    r.n_tiles = (int)(((long long)p.cols + tile_n - 1) / tile_n);
    r.m_fast = p.rows < p.cols;      // A, of `rows` rows, is the smaller operand
    r.first_factor = factors;
    r.factor_blocks = blocks_of(p.k);
    r.blocks = r.factor_blocks * p.pairs;
    r.out = p.out;
    r.ldo = p.ldo;
    factors += p.pairs;
    tiles += (long long)r.m_tiles * r.n_tiles;
    if (tiles > 0x3fffffffLL) return -1;
    r.tile_end = (int)tiles;
    equal = equal && r.blocks == g.result[0].blocks;
    ++g.results;
  }
  SharePlan s{(int)tiles, 0, 1, 0};
  if (tiles > 0 && equal && (kind == PLAIN || kind == KEEP)) s = plan_shares((int)tiles, g.result[0].blocks);
  g.full = s.full; g.rest = s.rest; g.splits = s.splits; g.split_blocks = s.split_blocks;
  return tiles;
}

size_t tc_parts_bytes(const attn_products_t& c) {
  ProductArgs g = {};
  if (plan(c, g) < 0) return 0;
  return g.splits > 1 ? (size_t)g.rest * g.splits * kTileM * kTileN * sizeof(float) : 0;
}

template <typename T, int FORM, int KIND>
static cudaError_t launch(const Maps& maps, const ProductArgs& g, cudaStream_t stream, int* launches) {
  static std::atomic<unsigned long long> smem_set;
  const int items = g.full + g.rest * g.splits, pairs = items < kSms / 2 ? items : kSms / 2;
  cudaError_t e = set_smem_once(product_kernel<T, FORM, KIND>, smem_bytes<KIND>(), smem_set);
  if (e == cudaSuccess) e = launch_pdl_cluster(product_kernel<T, FORM, KIND>, (unsigned)pairs * 2, kThreads, smem_bytes<KIND>(), 2, stream, maps, g);
  ++*launches;
  if (g.splits > 1 && e == cudaSuccess) {
    e = launch_pdl(join_kernel<T>, (unsigned)g.rest * 32, 256u, 0, stream, g);
    ++*launches;
  }
  return e;
}

template <typename T>
static cudaError_t launch_type(int form, int kind, const Maps& maps, const ProductArgs& g, cudaStream_t stream, int* launches) {
  if (kind == GATED) return launch<T, ATTN_FORM_NT, GATED>(maps, g, stream, launches);
  if (kind == KEPT) return launch<T, ATTN_FORM_NT, KEPT>(maps, g, stream, launches);
  if (kind == GRAD) return launch<T, ATTN_FORM_NN, GRAD>(maps, g, stream, launches);
  if (kind == KEEP) return launch<T, ATTN_FORM_NT, KEEP>(maps, g, stream, launches);
  if (form == ATTN_FORM_NT) return launch<T, ATTN_FORM_NT, PLAIN>(maps, g, stream, launches);
  if (form == ATTN_FORM_NN) return launch<T, ATTN_FORM_NN, PLAIN>(maps, g, stream, launches);
  return launch<T, ATTN_FORM_TN, PLAIN>(maps, g, stream, launches);
}

cudaError_t tc_products(const attn_products_t& c, float* parts, unsigned int* status, cudaStream_t stream, int* launches, const char** why) {
  Maps maps;
  ProductArgs g = {};
  const int kind = kind_of(c);
  const bool bf = c.dtype == ATTN_BF16;
  if (plan(c, g) < 0) return cudaErrorInvalidValue;
  if (g.results == 0) return cudaSuccess;
  bool ok = true;
  int factor = 0, result = 0;
  for (int i = 0; i < c.count; ++i) {
    const attn_product_t& p = c.product[i];
    if (p.rows == 0 || p.cols == 0 || p.k == 0) continue;
    for (int q = 0; q < p.pairs; ++q, ++factor) {
      const attn_factors_t& f = p.pair[q];
      ok = ok && (c.form == ATTN_FORM_TN ? encode(&maps.a[factor], f.a, bf, p.k, p.rows, f.lda, 64) : encode(&maps.a[factor], f.a, bf, p.rows, p.k, f.lda, 128));
      ok = ok && (c.form == ATTN_FORM_NT ? encode(&maps.b[factor], f.b, bf, p.cols, p.k, f.ldb, 128) : encode(&maps.b[factor], f.b, bf, p.k, p.cols, f.ldb, 64));
    }
    ok = ok && encode(&maps.out[result++], p.out, bf, p.rows, p.cols, p.ldo, 128);
  }
  const attn_product_t& p = c.product[0];
  auto side = [&](CUtensorMap* map, const void* at, int64_t ld) { ok = ok && encode(map, at, bf, p.rows, p.cols, ld, 128); };
  if (kind == PLAIN || kind == KEEP) {
    if (c.residual != nullptr) side(&maps.side[0], c.residual, c.ld_residual);
    if (kind == KEEP) side(&maps.side[1], c.kept[0], c.ld_kept[0]);
  } else {
    if (kind != GRAD) ok = ok && encode(&maps.b[1], c.b2, bf, p.cols, p.k, c.ldb2, 128);
    if (kind != GATED)
      for (int q = 0; q < 2; ++q) side(&maps.side[q], c.kept[q], c.ld_kept[q]);
    if (kind == GRAD) side(&maps.out2, c.out2, c.ldo2);
  }
  if (!ok) {
    *why = "cuTensorMapEncodeTiled refused a tensor";
    return cudaErrorInvalidValue;
  }
  g.act = c.activation;
  g.parts = parts;
  g.bias = c.bias;
  g.residual = c.residual;
  g.ld_residual = c.ld_residual;
  g.z = kind == KEEP ? c.kept[0] : nullptr;
  g.ld_z = c.ld_kept[0];
  g.status = status;
  return bf ? launch_type<__nv_bfloat16>(c.form, kind, maps, g, stream, launches) : launch_type<__half>(c.form, kind, maps, g, stream, launches);
}

}  // namespace layer
}  // namespace attn
