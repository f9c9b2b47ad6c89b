// The order in which the issuing warps of the paired forward (packed_fwd.cu) take the items of its ring and issue their products.  No CUDA:
// tests/host/packed_order.cpp walks through it on the CPU.
//
// The ring holds K(0), V(0), K(1), V(1), ...: item i is K (even) or V (odd) of streamed tile i / 2.  Items are loads of their own, on barriers of their
// own, and complete in any order: that K(j + 1) has arrived says nothing of V(j).
#pragma once

#ifdef __CUDACC__
#define ATTN_ORDER __device__ __forceinline__
#else
#define ATTN_ORDER inline
#endif

namespace attn {

// Streamed tiles [from(x), to(x)) of `tiles` belong to row tile x: A (0), B (1).
struct ProductOrder {
  int to_a, from_b, to_b, tiles;
  ATTN_ORDER int from(int x) const { return x == 0 ? 0 : from_b; }
  ATTN_ORDER int to(int x) const { return x == 0 ? to_a : to_b; }
  ATTN_ORDER bool on(int x, int j) const { return j >= from(x) && j < to(x); }
};

// An item that a warp has waited for is not asked for again (a satisfied wait takes some 90 clocks).  Every warp asks for the items of a kind in
// turn, so the last one of either kind says which those are.
struct Arrivals {
  int k = -1, v = -1;
  template <typename Wait> ATTN_ORDER bool operator()(int i, Wait&& wait) {
    if (i <= ((i & 1) ? v : k)) return true;
    if (i & 1) v = i; else k = i;
    return wait(i);
  }
};

// What a warp does, each false once a wait has given up:
//   arrived(i)             item i is there
//   skip(i)                gives back an item that no product of this warp reads
//   free(x, j)             the scores of tile j are in registers
//   scores(x, j, release)  S(j), of K(j); release: this warp's last product of the item
//   outputs(x, j, release) O += P(j) V(j), when P(j) is there
// A warp for row tile x alone: the next scores as soon as these are in registers.
template <typename Skip, typename Free, typename Scores, typename Outputs>
ATTN_ORDER bool issue_one_row_tile(const ProductOrder& o, int x, Skip&& skip, Free&& free, Scores&& scores, Outputs&& outputs) {
  const int from = o.from(x), to = o.to(x), behind = from > to ? from : to;
  bool ok = true;
  for (int i = 0; i < 2 * from && ok; ++i) ok = skip(i);
  if (to > from && ok) ok = scores(x, from, true);
  for (int j = from; j < to && ok; ++j) {
    if (j + 1 < to) ok = free(x, j) && scores(x, j + 1, true);
    ok = ok && outputs(x, j, true);
  }
  for (int i = 2 * behind; i < 2 * o.tiles && ok; ++i) ok = skip(i);
  return ok;
}

// One warp for both, so that one tile's products run while the other one's scores are exponentiated: P lies over the scores, and the
// next ones come right behind the product that reads it.  Every tile of the stream belongs to A, to B or to both.
template <typename Arrived, typename Scores, typename Outputs>
ATTN_ORDER bool issue_both_row_tiles(const ProductOrder& o, Arrived&& arrived, Scores&& scores, Outputs&& outputs) {
  bool ok = true;
  if (o.on(0, 0)) ok = scores(0, 0, !o.on(1, 0));
  if (ok && o.on(1, 0)) ok = scores(1, 0, true);
  for (int j = 0; j < o.tiles && ok; ++j) {
    const bool next = j + 1 < o.tiles;
    ok = arrived(2 * j + 1) && (!next || arrived(2 * j + 2));      // while P is still being made
    if (ok && o.on(0, j)) ok = outputs(0, j, !o.on(1, j));
    if (ok && next && o.on(0, j + 1)) ok = scores(0, j + 1, !o.on(1, j + 1));
    if (ok && o.on(1, j)) ok = outputs(1, j, true);
    if (ok && next && o.on(1, j + 1)) ok = scores(1, j + 1, true);
  }
  return ok;
}

// The streamed tiles of `keys` keys of either row tile of a pair, for rows [r0, row_end), up to 256, that see keys from lo on.
ATTN_ORDER ProductOrder pair_order(int r0, int row_end, int lo, int window, int keys) {
  const int tiles = (row_end - lo + keys - 1) / keys, last_a = row_end < r0 + 128 ? row_end : r0 + 128;
  const long long first_b = (long long)r0 + 128 - window + 1;
  ProductOrder o;
  o.tiles = tiles;
  o.to_a = (last_a - lo + keys - 1) / keys;
  o.from_b = first_b > lo ? (int)((first_b - lo) / keys) : 0;
  o.to_b = row_end > r0 + 128 ? tiles : 0;
  return o;
}

}  // namespace attn
