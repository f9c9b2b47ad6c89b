// Packed batches: sequences of different lengths laid end to end on one axis of n_tok rows, tensors
// [n_tok, heads, D], `group` query heads for every key/value head, causal attention within a sequence.
//
// A plan, made on the device from the sequences' offsets (packed_plan.cu), lists the stationary tiles of a
// batch: up to 128 rows of ONE sequence each, so that a sequence's result depends neither on what lies
// beside it (also where that is infinite or not a number) nor on where it lies in the batch; but which kernels a batch
// takes goes by its size and mean length, and with them the order of sums: a sequence by itself may differ in the last bits.  Rows of no
// sequence are listed too; they get zeros.  Short sequences pay for that with part-filled tiles: tiles of 128
// consecutive rows over several sequences would need up to 128 / length times fewer of them, but mix the rows of
// two sequences in one product, where 0 * inf and 0 * NaN of a neighbour's masked keys reach the sums.
// The entries are sorted by the length of a tile's stream, longest first, once for query tiles, once for key tiles and
// once for pairs of query tiles (256 rows).  Kernels bound every entry on reading it: a plan that is not one gives wrong results, but no
// access outside of the tensors.
#pragma once

#include "attn_common.cuh"

namespace attn {

constexpr int kPlanRows = 128;      // rows of a stationary tile
constexpr int kPlanHeader = 8;      // ints: tiles, longest sequence, n_tok, n_seq, 4 unused

// rows [row0, min(row0 + 128, end)), in the list of pairs 256, of the sequence [begin, end); begin < 0: rows of no sequence; row0 < 0: unused entry
struct alignas(16) PackedTile { int row0, begin, end, unused; };

// Entries of either list: a sequence's last tile and the gaps in front and behind take one more each than
// n_tok / 128.
__host__ __device__ inline long long plan_tiles(long long n_tok, long long n_seq) { return n_tok / kPlanRows + n_seq + 2; }

__host__ __device__ inline long long plan_pairs(long long n_tok, long long n_seq) { return n_tok / (2 * kPlanRows) + n_seq + 2; }

// A plan: header | query tiles | key tiles | pairs | row behind each sequence, and its tiles so far (n_seq ints each)
inline long long plan_ints(long long n_tok, long long n_seq) {
  return kPlanHeader + 8 * plan_tiles(n_tok, n_seq) + 4 * plan_pairs(n_tok, n_seq) + 2 * n_seq;
}

struct PackedGeometry : Geometry {
  static constexpr bool kPacked = true;
  const PackedTile* row_tiles;
  const PackedTile* col_tiles;
  const PackedTile* pair_tiles;
  int cap, pair_cap;        // entries of either list, and of that of the pairs
  int group;                // query heads per key/value head
  int q_heads, kv_heads, n_seq;
};

// what the kernels that serve both kinds of geometry ask for; a plain one has its heads on both sides alike
__device__ __forceinline__ int kv_plane_of(const Geometry&, int bh) { return bh; }
__device__ __forceinline__ int kv_plane_of(const PackedGeometry& g, int bh) { return bh / g.group; }
__device__ __forceinline__ int packed_cap(const Geometry&) { return 0; }
__device__ __forceinline__ int packed_cap(const PackedGeometry& g) { return g.cap; }

// Heads of a group of the CTAs' order (Geometry::head_group): all of them where the streamed tensors of all heads, of `bytes`, fit L2 together
// with the rest, so that the longest streams of all heads come first; else as many as 16 MB hold.  Groups of four of twelve heads left the SMs idle for
// 18 % of the forward's and 13 to 17 % of the backward's time (16384 rows in 19 sequences, 12 heads of 64).
// So do a few CTAs, whose longest ones decide (8192 rows in 7 sequences, 32 and 8 heads of 128, dK/dV: 584 CTAs, 281 us, 365 head by head).
inline int packed_head_group(const PackedGeometry& g, long long ctas, long long bytes) {
  if (ctas < 8 * kSms || bytes <= (64ll << 20)) return g.BH;
  const long long n = (16ll << 20) * g.BH / bytes;
  return n < 1 ? 1 : n < g.BH ? (int)n : g.BH;
}

// What a CTA works on: rows [r0, row_end) of its sequence against the streamed rows [lo, hi); lo == hi: none.
struct PackedWork { int r0, row_end, begin, end, lo, hi; };

__device__ __forceinline__ bool packed_work(const PackedGeometry& g, bool col, int rank, PackedWork& w) {
  const int4 e = __ldcg(reinterpret_cast<const int4*>((col ? g.col_tiles : g.row_tiles) + rank));
  if (e.x < 0 || e.x >= g.N_q) return false;
  w.r0 = e.x;
  w.end = min(max(e.z, e.x + 1), g.N_q);
  w.begin = min(e.y, e.x);
  w.row_end = min(w.r0 + kPlanRows, w.end);
  if (w.begin < 0) {
    w.begin = 0;
    w.lo = w.hi = w.r0;
  } else if (col) {      // queries that see the first to the last of these keys
    w.lo = w.r0;
    w.hi = (int)min((long long)w.end, (long long)w.row_end - 1 + g.window);
  } else {
    w.lo = max(w.begin, w.r0 - g.window + 1);
    w.hi = w.row_end;
  }
  if (w.hi < w.lo) w.hi = w.lo;
  return true;
}

// the streamed rows [lo, hi) that stationary row i sees, none for a row behind the tile's
__device__ __forceinline__ void packed_row_range(const PackedGeometry& g, const PackedWork& w, bool col, int i, int& lo, int& hi) {
  lo = hi = 0;
  if (i >= w.row_end || w.lo == w.hi) return;
  if (col) { lo = i; hi = (int)min((long long)w.end, (long long)i + g.window); }
  else { lo = max(w.begin, i - g.window + 1); hi = i + 1; }
  if (hi < lo) hi = lo;
}

}  // namespace attn
