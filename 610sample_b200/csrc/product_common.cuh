// What the tensor-core products share on the host: tensor maps of matrices, and how the tiles of a part-filled last round are shared out.
#pragma once

#include "attn_common.cuh"

#include <cuda.h>
#include <mutex>

namespace attn {
namespace product {

constexpr int kTileM = 256, kTileN = 256, kBlockK = 64;       // of a pair of CTAs

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiledFn encode_fn() {
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
inline bool encode(CUtensorMap* map, const void* p, bool bf16, long long rows, long long cols, long long ld, int box_rows) {
  const EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return false;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(p), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

inline int blocks_of(long long k) { return (int)((k + kBlockK - 1) / kBlockK); }

// The tiles of the last, part-filled round in shares along k, where that is shorter.  In blocks of k (0.28 us): a round of the shares takes
// split_blocks; shared tiles cost the launch behind them, 20, and a quarter of a block for every part that is written and read.  At least 8 blocks a share.
struct SharePlan { int full, rest, splits, split_blocks; };
inline SharePlan plan_shares(int tiles, int blocks) {
  const int pairs = kSms / 2;
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

}  // namespace product
}  // namespace attn
