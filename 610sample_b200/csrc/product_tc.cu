// Matrix products on the tensor cores (f16/bf16, sm_100a) with what follows them in their epilogue: one persistent kernel.
//
//   form   A                      B
//   NT     [rows, k]              [cols, k]
//   NN     [rows, k]              [k, cols], read by columns
//   TN     [k, rows], by columns  [k, cols], by columns
//
// A pair of CTAs (a cluster) owns a tile of 256 x 256: either holds 128 rows of A and half of B's columns, and one tcgen05.mma.cta_group::2
// reads both.  A warp loads through a ring of stages of 64 in k, one (in rank 0) issues the products, sixteen finish a tile from tensor memory
// while the next one accumulates in the other half of it.  A result is the sum of up to four products, one behind the other along k.
//
// kind    what the sixteen warps do with a tile
// PLAIN   z = sum + bias, activation, residual; z is kept or not
// GATED   128 columns: CTA 0 holds rows of Wg as its half of B and CTA 1 the same rows of Wu, so that columns j and 128 + j of the accumulator are z and u,
//         which are kept or not
// GRAD    reads z and u, and leaves their gradients
// A warp has 32 rows and a quarter of the columns, a thread one of the rows, 16 columns at a time.  Results leave through shared memory by TMA, 4 KB of each
// warp's own, so that no warp waits for another one.  Stored from registers, 32 rows to an instruction, they take 70 cycles of the shared memory's
// pipe each, which the products read their operands through (with z kept 64 us, 16384 x 768 x 2048).  In GRAD z and u come by TMA, 32 columns at a time for each
// four warps, and their gradients leave from where they lay: loads of 32 rows to an instruction are 32 requests, of which an SM has too few in flight.
//
// The tiles of several results are one list, so that three small ones (the weights' gradients of a gated block at 16384 x 768 x 2048: 24 tiles each
// of 256 blocks of k) fill the 74 pairs once.  Where the last round of tiles stays short of them, its tiles are shared out along k and a small kernel behind adds
// the parts in order and does the epilogue (PLAIN and KEEP).
//
// 16384 rows, 768 wide, 2048 inner, bf16, each by itself (ncu, cold, over boards): PLAIN with gelu and z kept 53 to 60 us, without either 44; NN 42 to 47, of two pairs 72 to 80;
// TN 41 to 46 and 7 to join, three results 93 to 107 (1 450 to 1 640 TFLOP/s, tensor pipe 77 to 84 % active); GATED 72, with z and u kept 86 to 94 (178 MB written); GRAD 72 to 79 (201 MB
// read, 94 written).  At the peak rate the operands come in at 64 bytes a clock and go out at 64, all that an SM's shared memory carries: with 12 blocks of k to a tile, what the
// epilogue stages there is the difference between these and the 31 and 63 us of the tensor cores.  With 64 blocks (16384 x 4096 -> 2048) 177 us, 1 556 TFLOP/s.
#include "activation.cuh"
#include "layer_launch.h"
#include "product_common.cuh"
#include "tc_common.cuh"

namespace attn {
namespace layer {

using namespace tc;
using namespace product;

enum Kind { PLAIN = 0, GATED = 1, GRAD = 2 };

constexpr int kHalfN = kTileN / 2;
constexpr uint32_t kOperandBytes = 128 * 128;                  // 128 rows (or columns) of 64 in k, of A or of B, in one CTA
constexpr uint32_t kStageBytes = 2 * kOperandBytes;
constexpr int kEpilogueWarps = 16, kLoadWarp = 16, kIssueWarp = 17, kThreads = 576;
constexpr int KPRODUCT = 40;                                   // kernel id inside device status codes: 40 + kind

template <int KIND> constexpr int kStagesOf = KIND == GRAD ? 4 : 5;
constexpr int kParts = kEpilogueWarps / 4;
constexpr uint32_t kStagingBytes = 4096;                       // of a warp, for results on their way out (not GRAD)
// z, u and their lower bits, [128 rows][32 columns], for each part
constexpr uint32_t kPlaneBytes = 128 * 64, kLowBytes = 128 * 32, kInputBytes = 2 * kPlaneBytes + kLowBytes;

template <int KIND> constexpr uint32_t kSideOf = KIND == GRAD ? kParts * kInputBytes : kEpilogueWarps * kStagingBytes;

template <int STAGES>
struct Control {
  uint64_t full[STAGES], empty[STAGES];        // full: rank 0's counts both CTAs' loads
  uint64_t acc_full[2], acc_empty[2];          // acc_empty: rank 0's counts both CTAs' warps
  uint64_t in_full[kParts];                    // GRAD
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
};
template <int KIND> constexpr uint32_t kSmemOf = kStagesOf<KIND> * kStageBytes + kSideOf<KIND> + sizeof(Control<kStagesOf<KIND>>) + 1024;
static_assert(kSmemOf<PLAIN> <= 232448 && kSmemOf<GRAD> <= 232448, "shared memory");

// side: z (PLAIN); z, u and their lower bits (GATED, and GRAD, which loads them)
struct Maps { CUtensorMap a[kMaxFactors], b[kMaxFactors], out[kMaxProducts], side[3]; };

// rows `ld` elements apart; wide: runs of 16 elements start at 32 bytes (2), at 16 (1), or anywhere (0)
struct Rows {
  void* p;
  long long ld;
  int wide;
};
struct Result {
  int rows, cols;
  int m_tiles, n_tiles, m_fast;  // m_fast: tiles in sequence along the rows
  int tile_end;                  // in the list of all tiles
  int first_factor, factor_blocks, blocks;      // blocks of k of one product of the sum, and of all of them
  Rows out;
};
struct ProductArgs {
  Result result[kMaxProducts];
  int results, act;
  int full, rest, splits, split_blocks;      // tiles taken whole; the others, each in `splits` shares of `split_blocks` blocks of k
  float* parts;                  // [rest x splits][2 CTAs][128][256], where there are several shares
  const void* bias;
  Rows residual, kept;           // kept: z of PLAIN; of GATED, whether z and u are
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

// 16 elements of a row, `left` of which are inside
template <typename T>
__device__ __forceinline__ void get16(const Rows& t, long long row, int col, int left, uint32_t (&w)[8]) {
  const T* p = static_cast<const T*>(t.p) + row * t.ld + col;
  if (left >= 16 && t.wide == 2) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p)
                 : "memory");
  } else if (left >= 16 && t.wide == 1) {
    const uint4 a = reinterpret_cast<const uint4*>(p)[0], b = reinterpret_cast<const uint4*>(p)[1];
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = (2 * e < left ? (uint32_t)h[2 * e] : 0u) | (2 * e + 1 < left ? (uint32_t)h[2 * e + 1] << 16 : 0u);
  }
}
__device__ __forceinline__ void load_shared16(uint32_t at, uint32_t* w) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
}

__device__ __forceinline__ void store_shared16(uint32_t at, uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w0), "r"(w1), "r"(w2), "r"(w3) : "memory");
}
// 16-byte chunk `c` of a row in a tile of rows of 64 bytes and of 32, in the swizzle of that width
__device__ __forceinline__ uint32_t sw64(int row, int c) { return (uint32_t)row * 64u + ((uint32_t)(c ^ (row >> 1 & 3)) << 4); }
__device__ __forceinline__ uint32_t sw32(int row, int c) { return (uint32_t)row * 32u + ((uint32_t)(c ^ (row >> 2 & 1)) << 4); }
// 16 elements of a row: of 64 columns, or of 32
__device__ __forceinline__ void stage16(uint32_t tile, bool of64, int row, int col, const uint32_t (&w)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    store_shared16(tile + (of64 ? sw128_offset(row, col + 8 * h) : sw64(row, (col >> 3) + h)), w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]);
}

// bias[col .. col + 16), packed; `left` of them are inside
template <typename T>
__device__ __forceinline__ void bias16(const void* bias, int col, int left, uint32_t (&w)[8]) {
  get16<T>(Rows{const_cast<void*>(bias), 0, reinterpret_cast<uintptr_t>(bias) % 16 == 0 ? 1 : 0}, 0, col, left, w);
}

template <typename T, int FORM, int KIND>
__global__ void __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ Maps maps, const __grid_constant__ ProductArgs g) {
  constexpr bool kAByColumns = FORM == ATTN_FORM_TN, kBByColumns = FORM != ATTN_FORM_NT, kGate = KIND == GATED;
  constexpr int kColumns = kGate ? 32 : 64;                      // of a result, for each warp
  constexpr int KCODE = KPRODUCT + KIND, kStages = kStagesOf<KIND>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t side = smem_base + kStages * kStageBytes;
  typedef Control<kStages> Ctl;
  Ctl* ctl = reinterpret_cast<Ctl*>(smem_raw + (smem_base - smem_u32(smem_raw)) + kStages * kStageBytes + kSideOf<KIND>);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  auto bar_full = [&](int s) { return smem_u32(&ctl->full[s]); };
  auto bar_empty = [&](int s) { return smem_u32(&ctl->empty[s]); };
  auto bar_acc_full = [&](int b) { return smem_u32(&ctl->acc_full[b]); };
  auto bar_acc_empty = [&](int b) { return smem_u32(&ctl->acc_empty[b]); };

  if (warp == kLoadWarp && lane == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full(s), 1);
      mbar_init(bar_empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_acc_full(b), 1);
      mbar_init(bar_acc_empty(b), 2 * kEpilogueWarps);
    }
    for (int q = 0; q < kParts; ++q) mbar_init(smem_u32(&ctl->in_full[q]), 1);
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
    const int quarter = warp & 3, part = warp >> 2;          // of the rows, and of the columns
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const bool residual = KIND == PLAIN && g.residual.p != nullptr, keep = KIND != GRAD && g.kept.p != nullptr;
    // GRAD: one thread of a part asks for the inputs of 32 columns of an item.  Boxes may lie outside of the planes, and are zeros there
    const uint32_t in_z = side + part * kInputBytes, in_u = in_z + kPlaneBytes, in_low = in_u + kPlaneBytes, bar_in = smem_u32(&ctl->in_full[part]);
    auto fetch = [&](int i, int c) {
      if (i >= items) return;
      const Item item = item_at(g, i);
      int mt, nt;
      tile_at(g.result[0], 0, item.t, mt, nt);
      const int col = nt * kTileN + part * kColumns + c, r0 = mt * kTileM + (int)rank * 128;
      const uint32_t bar = map_rank(bar_in, rank);
      mbar_arrive_expect_tx(bar_in, kInputBytes);
      tma_load_2d_pair(in_z, &maps.side[0], col, r0, bar);
      tma_load_2d_pair(in_u, &maps.side[1], col, r0, bar);
      tma_load_2d_pair(in_low, &maps.side[2], col, r0, bar);
    };
    // what the warp has written to its staging leaves it
    const uint32_t staging = side + (uint32_t)warp * kStagingBytes;
    auto leave = [&](auto&& store, bool inside) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0 && inside) {
        store();
        bulk_commit_group();
      }
    };
    const bool leader = quarter == 0 && lane == 0;
    if (KIND == GRAD && leader) fetch(pair, 0);
    // GRAD: the four warps of a part meet, so they go on or give up together; a wait for inputs that gives up goes on to the next tile, where all hear of it
    bool ok = true, alive = true;
    int n = 0, fetched = 0;
    for (int i = pair; i < items && ok; i += pairs, ++n) {
      const Item item = item_at(g, i);
      const int p = result_of(g, item.t);
      const Result& r = g.result[p];
      int mt, nt;
      tile_at(r, tiles_before(g, p), item.t, mt, nt);
      const int buf = n & 1;
      const int r0 = mt * kTileM + (int)rank * 128 + quarter * 32;      // the warp's first row
      const long long at = r0 + lane;
      const bool in = at < r.rows;
      const int col0 = (kGate ? nt * kHalfN : nt * kTileN) + part * kColumns;      // the warp's first column
      const uint32_t acc = lane_addr + (uint32_t)buf * 256u + (uint32_t)(part * kColumns);
      // the residual of the next two runs of 16 columns; each is asked for anew once it has been used
      uint32_t next[2][KIND == PLAIN ? 8 : 1];
      auto ask = [&](int c, int q) {
        const int col = col0 + c + 16 * q, left = r.cols - col;
        if constexpr (KIND == PLAIN)
          if (residual && in && !item.part && left > 0) get16<T>(g.residual, at, col, left, next[q]);
      };
      ask(0, 0);
      ask(0, 1);
      ok = mbar_wait(bar_acc_full(buf), (n >> 1) & 1, abort_flag, g.status, wait_code(KCODE, 4));
      ok = KIND == GRAD ? named_barrier_all(1 + part, 128, ok && alive) : (bool)__all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after_sync();
      float* part_row = nullptr;
      if (item.part) part_row = g.parts + (((size_t)(i - g.full) * 2 + rank) * 128 + row) * 256 + part * kColumns;

#pragma unroll 1
      for (int c = 0; c < kColumns; c += 32) {
        uint32_t low[KIND == PLAIN ? 1 : 8], hs[KIND == GATED ? 16 : 1];
        if constexpr (KIND == GRAD) {
          alive = mbar_wait(bar_in, fetched & 1, abort_flag, g.status, wait_code(KCODE, 6)) && alive;
          ++fetched;
#pragma unroll
          for (int e = 0; e < 2; ++e) load_shared16(in_low + sw32(row, e), &low[4 * e]);
        } else if (c == 0 || keep) {                       // the staging: what left it last has been read
          if (lane == 0) bulk_wait_group_read_all();
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          __syncwarp();
          uint32_t v[16], v2[kGate ? 16 : 1];
          tmem_ld16(acc + c + 16 * q, v);
          if constexpr (kGate) tmem_ld16(acc + 128 + c + 16 * q, v2);
          tmem_ld_wait(v);
          if constexpr (kGate) tmem_ld_wait(v2);
          if (c + 32 == kColumns && q == 1) {              // the accumulator is in registers
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_local(map_rank(bar_acc_empty(buf), 0));
          }
          const int col = col0 + c + 16 * q, left = r.cols - col;
          if (left <= 0) continue;                         // uniform
          if (KIND == PLAIN && item.part) {
            float4* to = reinterpret_cast<float4*>(part_row + c + 16 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              __stcg(to + e, make_float4(__uint_as_float(v[4 * e]), __uint_as_float(v[4 * e + 1]), __uint_as_float(v[4 * e + 2]), __uint_as_float(v[4 * e + 3])));
            continue;
          }
          float2 f[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = make_float2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1]));
          uint32_t w[8];
          if constexpr (kGate) {
            float2 u[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = make_float2(__uint_as_float(v2[2 * e]), __uint_as_float(v2[2 * e + 1]));
            if (keep) {
              uint32_t wu[8];
#pragma unroll
              for (int e = 0; e < 8; e += 2) {
                const uint32_t cz[4] = {Kept<T>::code(f[e].x), Kept<T>::code(f[e].y), Kept<T>::code(f[e + 1].x), Kept<T>::code(f[e + 1].y)};
                const uint32_t cu[4] = {Kept<T>::code(u[e].x), Kept<T>::code(u[e].y), Kept<T>::code(u[e + 1].x), Kept<T>::code(u[e + 1].y)};
                w[e] = kept_high(cz[0], cz[1]);
                w[e + 1] = kept_high(cz[2], cz[3]);
                wu[e] = kept_high(cu[0], cu[1]);
                wu[e + 1] = kept_high(cu[2], cu[3]);
                low[4 * q + (e >> 1)] = kept_low(cz, cu);
              }
              stage16(staging, false, lane, 16 * q, w);
              stage16(staging + 2048, false, lane, 16 * q, wu);
            }
            with_activation(g.act, [&](auto act) {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                float2 a, d;
                activate2<decltype(act)::value, false>(f[e], a, d);
                f[e] = __fmul2_rn(a, u[e]);
              }
            });
#pragma unroll
            for (int e = 0; e < 8; ++e) hs[8 * q + e] = Pack<T>::pack(f[e].x, f[e].y);
          } else if constexpr (KIND == GRAD) {
            uint32_t wu[8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              load_shared16(in_z + sw64(row, 2 * q + h), &w[4 * h]);
              load_shared16(in_u + sw64(row, 2 * q + h), &wu[4 * h]);
            }
            with_activation(g.act, [&](auto act) {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const uint32_t hz = w[e], hu = wu[e], nz = kept_z(low[4 * q + (e >> 1)]), nu = kept_u(low[4 * q + (e >> 1)]);
                const float2 z = (e & 1) ? make_float2(Kept<T>::value(kept_code<2>(hz, nz)), Kept<T>::value(kept_code<3>(hz, nz)))
                                         : make_float2(Kept<T>::value(kept_code<0>(hz, nz)), Kept<T>::value(kept_code<1>(hz, nz)));
                const float2 u = (e & 1) ? make_float2(Kept<T>::value(kept_code<2>(hu, nu)), Kept<T>::value(kept_code<3>(hu, nu)))
                                         : make_float2(Kept<T>::value(kept_code<0>(hu, nu)), Kept<T>::value(kept_code<1>(hu, nu)));
                float2 a, d;
                activate2<decltype(act)::value, true>(z, a, d);
                a = __fmul2_rn(f[e], a);
                f[e] = __fmul2_rn(__fmul2_rn(f[e], d), u);
                w[e] = Pack<T>::pack(f[e].x, f[e].y);
                wu[e] = Pack<T>::pack(a.x, a.y);
              }
            });
            stage16(in_z, false, row, 16 * q, w);
            stage16(in_u, false, row, 16 * q, wu);
          } else {
            if (g.bias != nullptr) {
              uint32_t b[8];
              bias16<T>(g.bias, col, left, b);
#pragma unroll
              for (int e = 0; e < 8; ++e) f[e] = __fadd2_rn(f[e], Pack<T>::unpack(b[e]));
            }
            if (keep) {
#pragma unroll
              for (int e = 0; e < 8; ++e) w[e] = pack_argument(f[e].x, f[e].y);
              stage16(staging + 2048, false, lane, 16 * q, w);
            }
            if (g.act != ACT_NONE)
              with_activation(g.act, [&](auto act) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  float2 d;
                  activate2<decltype(act)::value, false>(f[e], f[e], d);
                }
              });
            if (residual) {
#pragma unroll
              for (int e = 0; e < 8; ++e) f[e] = __fadd2_rn(f[e], Pack<T>::unpack(next[q][e]));
              if (c + 32 < kColumns) ask(c + 32, q);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = Pack<T>::pack(f[e].x, f[e].y);
            stage16(staging, !keep, lane, (keep ? 0 : c) + 16 * q, w);
          }
        }
        if constexpr (KIND == GRAD) {
          fence_proxy_async_smem();
          alive = named_barrier_all(1 + part, 128, alive);
          if (leader) {
            if (col0 + c < r.cols) {                       // rows of the whole part: quarter 0's first one
              tma_store_2d(&maps.out[0], in_z, col0 + c, r0);
              tma_store_2d(&maps.out[1], in_u, col0 + c, r0);
              bulk_commit_group();
              bulk_wait_group_read_all();
            }
            if (c + 32 < kColumns) fetch(i, c + 32);
            else fetch(i + pairs, 0);
          }
          continue;
        }
        if (item.part || r0 >= r.rows) continue;           // uniform
        if constexpr (kGate) {
          const int col = col0 + c;
          if (keep) {
            leave([&] {
              tma_store_2d(&maps.side[0], staging, col, r0);
              tma_store_2d(&maps.side[1], staging + 2048, col, r0);
            }, col < r.cols);
            if (lane == 0) bulk_wait_group_read_all();
            __syncwarp();
#pragma unroll
            for (int h = 0; h < 2; ++h) store_shared16(staging + 2048 + sw32(lane, h), low[4 * h], low[4 * h + 1], low[4 * h + 2], low[4 * h + 3]);
          }
#pragma unroll
          for (int h = 0; h < 4; ++h) store_shared16(staging + sw64(lane, h), hs[4 * h], hs[4 * h + 1], hs[4 * h + 2], hs[4 * h + 3]);
          leave([&] {
            tma_store_2d(&maps.out[0], staging, col, r0);
            if (keep) tma_store_2d(&maps.side[2], staging + 2048, col, r0);
          }, col < r.cols);
        } else if (keep) {
          leave([&] {
            tma_store_2d(&maps.out[0], staging, col0 + c, r0);
            tma_store_2d(&maps.side[0], staging + 2048, col0 + c, r0);
          }, col0 + c < r.cols);
        } else if (c + 32 == kColumns) {
          leave([&] { tma_store_2d(&maps.out[p], staging, col0, r0); }, col0 < r.cols);
        }
      }
    }
    if (lane == 0) bulk_wait_group_read_all();
    if (!alive) {      // inputs that are still on their way: a bounded chance to land before the CTA exits
      const long long t0 = clock64();
      while (clock64() - t0 < 2000000LL) { }
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
    const int width = min(4, res.cols - col);      // col is a multiple of 4
    auto put = [&](const Rows& to, uint32_t w0, uint32_t w1) {
      uint16_t* p = static_cast<uint16_t*>(to.p) + r * to.ld + col;
      if (width == 4 && to.wide > 0) *reinterpret_cast<uint2*>(p) = make_uint2(w0, w1);
      else
        for (int e = 0; e < width; ++e) p[e] = (uint16_t)((e < 2 ? w0 : w1) >> (16 * (e & 1)));
    };
    if (g.bias != nullptr)
      for (int e = 0; e < width; ++e) v[e] += Elem<T>::to_float(static_cast<const T*>(g.bias)[col + e]);
    if (g.kept.p != nullptr) put(g.kept, pack_argument(v[0], v[1]), pack_argument(v[2], v[3]));
    with_activation(g.act, [&](auto act) {
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        float2 a, d;
        activate2<decltype(act)::value, false>(make_float2(v[e], v[e + 1]), a, d);
        v[e] = a.x; v[e + 1] = a.y;
      }
    });
    if (g.residual.p != nullptr)
      for (int e = 0; e < width; ++e) v[e] += Elem<T>::to_float(static_cast<const T*>(g.residual.p)[r * g.residual.ld + col + e]);
    put(res.out, Pack<T>::pack(v[0], v[1]), Pack<T>::pack(v[2], v[3]));
  }
}

// ---- host ---------------------------------------------------------------------------------------
static Rows rows_of(const void* p, int64_t ld) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * 2);
  return {const_cast<void*>(p), ld, a % 32 == 0 ? 2 : a % 16 == 0 ? 1 : 0};
}

// a matrix of `size` bytes an element, boxes of 32 columns
static bool encode_plane(CUtensorMap* map, const void* p, int size, long long rows, long long cols, long long ld, int box_rows) {
  const EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return false;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)(ld * size)};
  cuuint32_t box[2] = {32, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, size == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(p), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, size == 1 ? CU_TENSOR_MAP_SWIZZLE_32B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Results, tiles and shares of a call; results without rows, columns or k have no tiles
static long long plan(const attn_products_t& c, ProductArgs& g) {
  const int tile_n = c.kind == ATTN_PRODUCT_GATED ? kHalfN : kTileN;
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
    r.out = rows_of(p.out, p.ldo);
    factors += p.pairs;
    tiles += (long long)r.m_tiles * r.n_tiles;
    if (tiles > 0x3fffffffLL) return -1;
    r.tile_end = (int)tiles;
    equal = equal && r.blocks == g.result[0].blocks;
    ++g.results;
  }
  SharePlan s{(int)tiles, 0, 1, 0};
  if (tiles > 0 && equal && c.kind == ATTN_PRODUCT_PLAIN) s = plan_shares((int)tiles, g.result[0].blocks);
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
  cudaError_t e = set_smem_once(product_kernel<T, FORM, KIND>, kSmemOf<KIND>, smem_set);
  if (e == cudaSuccess) e = launch_pdl_cluster(product_kernel<T, FORM, KIND>, (unsigned)pairs * 2, kThreads, kSmemOf<KIND>, 2, stream, maps, g);
  ++*launches;
  if (g.splits > 1 && e == cudaSuccess) {
    e = launch_pdl(join_kernel<T>, (unsigned)g.rest * 32, 256u, 0, stream, g);
    ++*launches;
  }
  return e;
}

template <typename T>
static cudaError_t launch_type(const attn_products_t& c, const Maps& maps, const ProductArgs& g, cudaStream_t stream, int* launches) {
  if (c.kind == ATTN_PRODUCT_GATED) return launch<T, ATTN_FORM_NT, GATED>(maps, g, stream, launches);
  if (c.kind == ATTN_PRODUCT_GATED_GRAD) return launch<T, ATTN_FORM_NN, GRAD>(maps, g, stream, launches);
  if (c.form == ATTN_FORM_NT) return launch<T, ATTN_FORM_NT, PLAIN>(maps, g, stream, launches);
  if (c.form == ATTN_FORM_NN) return launch<T, ATTN_FORM_NN, PLAIN>(maps, g, stream, launches);
  return launch<T, ATTN_FORM_TN, PLAIN>(maps, g, stream, launches);
}

cudaError_t tc_products(const attn_products_t& c, float* parts, unsigned int* status, cudaStream_t stream, int* launches, const char** why) {
  Maps maps;
  ProductArgs g = {};
  const bool bf = c.dtype == ATTN_BF16;
  if (plan(c, g) < 0) return cudaErrorInvalidValue;
  if (g.results == 0) return cudaSuccess;
  bool ok = true;
  int factor = 0, result = 0;
  const bool keep = c.kept[0] != nullptr, of64 = c.kind == ATTN_PRODUCT_PLAIN && !keep;      // how results are staged
  const int box_rows = c.kind == ATTN_PRODUCT_GATED_GRAD ? 128 : 32;
  for (int i = 0; i < c.count; ++i) {
    const attn_product_t& p = c.product[i];
    if (p.rows == 0 || p.cols == 0 || p.k == 0) continue;
    ok = ok && (of64 ? encode(&maps.out[result], p.out, bf, p.rows, p.cols, p.ldo, 32) : encode_plane(&maps.out[result], p.out, 2, p.rows, p.cols, p.ldo, box_rows));
    ++result;
    for (int q = 0; q < p.pairs; ++q, ++factor) {
      const attn_factors_t& f = p.pair[q];
      ok = ok && (c.form == ATTN_FORM_TN ? encode(&maps.a[factor], f.a, bf, p.k, p.rows, f.lda, 64) : encode(&maps.a[factor], f.a, bf, p.rows, p.k, f.lda, 128));
      ok = ok && (c.form == ATTN_FORM_NT ? encode(&maps.b[factor], f.b, bf, p.cols, p.k, f.ldb, 128) : encode(&maps.b[factor], f.b, bf, p.k, p.cols, f.ldb, 64));
    }
  }
  const attn_product_t& p = c.product[0];
  if (c.kind == ATTN_PRODUCT_GATED) ok = ok && encode(&maps.b[1], c.b2, bf, p.cols, p.k, c.ldb2, 128);
  if (keep) {
    const int planes = c.kind == ATTN_PRODUCT_PLAIN ? 1 : 2;
    for (int q = 0; q < planes; ++q) ok = ok && encode_plane(&maps.side[q], c.kept[q], 2, p.rows, p.cols, c.ld_kept[q], box_rows);
    if (planes == 2) ok = ok && encode_plane(&maps.side[2], c.kept_low, 1, p.rows, p.cols, c.ld_low, box_rows);
  }
  if (c.kind == ATTN_PRODUCT_GATED_GRAD) ok = ok && encode_plane(&maps.out[1], c.out2, 2, p.rows, p.cols, c.ldo2, box_rows);
  if (!ok) {
    *why = "cuTensorMapEncodeTiled refused a tensor";
    return cudaErrorInvalidValue;
  }
  g.act = c.activation;
  g.parts = parts;
  g.bias = c.bias;
  g.residual = rows_of(c.residual, c.ld_residual);
  g.kept = rows_of(c.kept[0], c.ld_kept[0]);
  g.status = status;
  return bf ? launch_type<__nv_bfloat16>(c, maps, g, stream, launches) : launch_type<__half>(c, maps, g, stream, launches);
}

}  // namespace layer
}  // namespace attn
