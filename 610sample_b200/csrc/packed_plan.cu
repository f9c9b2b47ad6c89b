// The plan of a packed batch (packed_geometry.cuh) from the sequences' offsets cu_seqlens[n_seq + 1], in one launch of
// one CTA.  Offsets are taken as they come: each is cut to [0, n_tok] and to no less than those before it, so that the
// sequences never overlap.
//   pass 1  running maximum of the offsets and running count of tiles, 1024 sequences at a time, kept in the plan
//   pass 2  histograms of the tiles (both lists have the same one) and of the pairs by the length of their stream, in tiles
//   pass 3  every tile to its place, longest streams first
// Made once per batch and shared by all layers and both directions, so what counts is that it is one short launch: 5 to 9 us.
#include "packed_geometry.cuh"
#include "packed_launch.h"
#include "tc_common.cuh"

namespace attn {

constexpr int kPlanThreads = 1024;
constexpr int kPlanBins = 2048;      // stream lengths told apart; longer ones share bins

// inclusive scan over the CTA, `op` associative
template <typename Op>
__device__ __forceinline__ int block_scan(int v, int* warp_sums, Op op, int identity) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = op(v, u);
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  int before = identity;
  for (int i = 0; i < warp; ++i) before = op(before, warp_sums[i]);
  return op(before, v);
}

__global__ void __launch_bounds__(kPlanThreads)
packed_plan_kernel(const int* cu, int* plan, int n_tok, int n_seq) {
  __shared__ int warp_sums[32], place[kPlanBins], pair_place[kPlanBins], shared_max, shared_longest;
  const int cap = (int)plan_tiles(n_tok, n_seq), pair_cap = (int)plan_pairs(n_tok, n_seq);
  PackedTile* const rows = reinterpret_cast<PackedTile*>(plan + kPlanHeader);
  PackedTile* const cols = rows + cap;
  PackedTile* const pairs = cols + cap;
  int* const ends = reinterpret_cast<int*>(pairs + pair_cap);      // row behind sequence i
  int* const counts = ends + n_seq;                           // tiles of the sequences up to and with i
  const int tid = threadIdx.x;
  // streams of up to cap tiles fall into the bins `shift` apart
  int shift = 0;
  while ((n_tok / kPlanRows >> shift) >= kPlanBins - 1) ++shift;
  for (int i = tid; i < kPlanBins; i += kPlanThreads) place[i] = pair_place[i] = 0;
  if (tid == 0) shared_longest = 0;
  auto cut = [&](int v) { return min(max(v, 0), n_tok); };
  const int first = cut(cu[0]);
  int last = first, tiles = 0;
  for (int i0 = 0; i0 < n_seq; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int m = block_scan(i < n_seq ? cut(cu[i + 1]) : 0, warp_sums, [](int a, int b) { return max(a, b); }, 0);
    m = max(m, last);
    if (i < n_seq) ends[i] = m;
    __syncthreads();
    const int begin = i < n_seq ? (i == 0 ? first : ends[i - 1]) : 0;
    const int mine = i < n_seq ? m - begin : 0;
    const int c = block_scan((mine + kPlanRows - 1) / kPlanRows, warp_sums, [](int a, int b) { return a + b; }, 0) + tiles;
    if (i < n_seq) counts[i] = c;
    if (mine > 0) atomicMax(&shared_longest, mine);
    __syncthreads();
    if (tid == kPlanThreads - 1) { shared_max = m; warp_sums[0] = c; }
    __syncthreads();
    last = shared_max;
    tiles = warp_sums[0];
    __syncthreads();
  }
  const int front = (first + kPlanRows - 1) / kPlanRows, back = (n_tok - last + kPlanRows - 1) / kPlanRows;
  // a tile by its number over all sequences: sequence, its rows, number within it and tiles of the sequence
  auto find = [&](int t, int& begin, int& end, int& k, int& n) {
    int a = 0, b = n_seq - 1;
    while (a < b) {
      const int mid = (a + b) >> 1;
      if (counts[mid] > t) b = mid; else a = mid + 1;
    }
    begin = a == 0 ? first : ends[a - 1];
    end = ends[a];
    const int before = a == 0 ? 0 : counts[a - 1];
    k = t - before;
    n = counts[a] - before;
  };
  // the tile number k of n has a stream of k + 1 tiles, as a tile of keys one of n - k: the same numbers for both lists
  for (int t = tid; t < tiles; t += kPlanThreads) {
    int begin, end, k, n;
    find(t, begin, end, k, n);
    atomicAdd(&place[kPlanBins - 1 - (k >> shift)], 1);
    if (k % 2 == 0) atomicAdd(&pair_place[kPlanBins - 1 - (k >> shift)], 1);
  }
  __syncthreads();
  for (int which = 0; which < 2; ++which) {
    int* const bins = which ? pair_place : place;
    const int a = bins[2 * tid], b = bins[2 * tid + 1];
    const int through = block_scan(a + b, warp_sums, [](int x, int y) { return x + y; }, 0);
    bins[2 * tid] = through - a - b;
    bins[2 * tid + 1] = through - b;
    if (which && tid == kPlanThreads - 1) shared_max = through;
  }
  __syncthreads();
  const int pair_count = shared_max;
  for (int t = tid; t < tiles; t += kPlanThreads) {
    int begin, end, k, n;
    find(t, begin, end, k, n);
    const int at = atomicAdd(&place[kPlanBins - 1 - (k >> shift)], 1);
    rows[at] = PackedTile{begin + k * kPlanRows, begin, end, 0};
    cols[at] = PackedTile{begin + (n - 1 - k) * kPlanRows, begin, end, 0};
    if (k % 2 == 0) pairs[atomicAdd(&pair_place[kPlanBins - 1 - (k >> shift)], 1)] = PackedTile{begin + k * kPlanRows, begin, end, 0};
  }
  for (int t = tid; t < cap - tiles; t += kPlanThreads) {
    PackedTile e{-1, -1, -1, 0};
    if (t < front) e = PackedTile{t * kPlanRows, -1, first, 0};
    else if (t < front + back) e = PackedTile{last + (t - front) * kPlanRows, -1, n_tok, 0};
    rows[tiles + t] = e;
    cols[tiles + t] = e;
  }
  const int pair_front = (front + 1) / 2, pair_back = (back + 1) / 2;
  for (int t = tid; t < pair_cap - pair_count; t += kPlanThreads) {
    PackedTile e{-1, -1, -1, 0};
    if (t < pair_front) e = PackedTile{t * 2 * kPlanRows, -1, first, 0};
    else if (t < pair_front + pair_back) e = PackedTile{last + (t - pair_front) * 2 * kPlanRows, -1, n_tok, 0};
    pairs[pair_count + t] = e;
  }
  if (tid == 0) {
    plan[0] = tiles; plan[1] = shared_longest; plan[2] = n_tok; plan[3] = n_seq;
    plan[4] = first; plan[5] = last; plan[6] = plan[7] = 0;
  }
}

cudaError_t launch_packed_plan(const int* cu_seqlens, int* plan, int n_tok, int n_seq, cudaStream_t s) {
  static_assert(kPlanBins == 2 * kPlanThreads, "a thread scans two bins");
  packed_plan_kernel<<<1, kPlanThreads, 0, s>>>(cu_seqlens, plan, n_tok, n_seq);
  return cudaGetLastError();
}

}  // namespace attn
