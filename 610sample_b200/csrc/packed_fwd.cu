// Forward attention over a packed batch on sm_100a (f16/bf16): O and L of 256 query rows of one sequence and head per CTA, against
// tiles of 128 keys, in one pass with an online softmax.
//
// The rows are two tiles, A and B, of 128, each with math warps, scores S (128 columns of tensor memory) and an O of its own.  Both read
// the same K and V tiles, so every byte brought into shared memory is used for 256 rows.  m is a reference, not the maximum: a
// row's first visible tile sets it, a later one moves it only where its maximum is more than 2^8 above, and then the row's own threads multiply
// its O in tensor memory by 2^(m_old - m_new).  The largest P of a row is then at most 2^8, exactly representable; sums are in fp32.
//
// D > 64: a thread owns a row, P lies over the first 64 columns of the scores it came from, and one warp issues all products, in the order
//     S_A(0) S_B(0) | O_A += P_A(0) V(0), S_A(1), O_B += P_B(0) V(0), S_B(1) | ...
// so that one tile's products run while the other one's scores are exponentiated.  The products of a thread execute in the order of
// issue: S(j + 1) may be issued right behind the P V that still reads P(j) from the same columns, and a math warp that sees S(j + 1)
// complete knows P V of j complete too, which is all that rescaling O needs.
// D <= 64: there is room for P beside S, so the next scores come as soon as these are in registers; a warp for either row tile issues
// its products.  What counts then is to keep the special-function unit busy (8 clocks for a warp's exponentials: 2 048 for 256 x 128 scores),
// which one warp of a tile on each scheduler does to 60 % and two do better: two threads a row, half of the columns each, which agree on
// the row's reference through shared memory.  The order of the issuing warps is in packed_order.h.
//
// One sequence of 8192, 16 heads, causal: D = 128 (4 key heads) 239 us, 1 151 TFLOP/s, 70 % of the measured peak (single tiles 252); D = 64 177 us,
// 778 TFLOP/s, the special-function unit 70 % busy (201).  Tried on the way, beside 231 and 196 us of another board with one thread a row and one
// issuing warp: P handed over in halves 257 and 220; two issuing warps and halves 310 and 198 (both tiles then wait for the tensor pipe, and
// then exponentiate, at the same time); exponentials strictly in turn 241 and 211; a quarter or half of them by polynomial on the FMA pipe no
// faster and 257 and 224; 208 registers a thread 239 and 201; two threads a row 247 and 186.
#include "packed_launch.h"
#include "packed_order.h"
#include "tc_common.cuh"

namespace attn {
namespace tc {

namespace {

constexpr int KPF = 21;                                       // kernel id inside device status codes
constexpr int kKeys = 128;                                    // keys of a streamed tile
constexpr uint32_t kAtomBytes = 128 * 128;                    // [128 rows][64 halves]
constexpr int kMaxSlots = 10;

struct Control2 {
  uint64_t q_full;
  uint64_t slot_full[kMaxSlots], slot_empty[kMaxSlots];       // K(0), V(0), K(1), V(1), ... in turn
  uint64_t ragged_full[2];                                    // the last K and V tile, where rows of them are to be cleared
  uint64_t s_full[2], s_free[2], p_full[2], pv_done[2], acc_done[2];      // by tile A, B
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
};

template <int DT>
struct Cfg2 {
  static constexpr int kAtoms = DT / 64;
  // math threads of a row, each with its share of the columns, and the other warps: loads, products (for either row tile at DT = 64)
  static constexpr int kHalves = DT == 64 ? 2 : 1, kCols = kKeys / kHalves;
  static constexpr int kTileWarps = 4 * kHalves, kTileThreads = 32 * kTileWarps;
  static constexpr int kLoadWarp = 2 * kTileWarps, kIssueWarp = kLoadWarp + 1;
  static constexpr int kThreads = DT == 64 ? 640 : 320;
  static constexpr uint32_t kTileBytes = kAtoms * kAtomBytes;                       // 128 rows of Q, K or V
  // P of its own beside S and O fits tensor memory at DT = 64 only
  static constexpr bool kOwnP = DT == 64;
  // a row's maxima, later its sums, of either half of its columns: [2 in turn][2 halves][128] for either row tile
  static constexpr uint32_t kExchange = kHalves == 2 ? 2 * 2 * 128 * 4 : 0;
  static constexpr uint32_t kAux = 512 + 2 * kExchange;
  static constexpr uint32_t kSlack = 1024;                                          // for the alignment of the base
  static constexpr int kFit = (int)((232448 - kSlack - kAux - 2 * kTileBytes) / kTileBytes);
  static constexpr int kSlots = kFit < kMaxSlots ? kFit : kMaxSlots;
  static constexpr uint32_t kContentBytes = (2 + kSlots) * kTileBytes + kAux;
  static constexpr uint32_t kSmemBytes = kContentBytes + kSlack;
  // tensor memory: S of tile x at 128 x, O at kO + DT x, P over S or in columns of its own
  static constexpr int kO = 256, kP = kOwnP ? 384 : 0, kPStride = kOwnP ? 64 : 128;
  static_assert(sizeof(Control2) <= 512 && kSlots >= 4, "shared memory");
};

template <int DT, typename T>
__global__ void __launch_bounds__(Cfg2<DT>::kThreads, 1)
packed_fwd_kernel(const __grid_constant__ TmaMaps maps, const PackedGeometry g, const Tensors t) {
  using CF = Cfg2<DT>;
  constexpr int kSlots = CF::kSlots, kAtoms = CF::kAtoms, kHalves = CF::kHalves, kCols = CF::kCols;
  constexpr int kLoadWarp = CF::kLoadWarp, kIssueWarp = CF::kIssueWarp, kThreads = CF::kThreads, kTileThreads = CF::kTileThreads;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t ring = smem_base + 2 * CF::kTileBytes;
  Control2* ctl = reinterpret_cast<Control2*>(smem_raw + (smem_base - smem_u32(smem_raw)) + (2 + kSlots) * CF::kTileBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  {
    uint32_t dyn_size;
    asm("mov.u32 %0, %%dynamic_smem_size;" : "=r"(dyn_size));
    if (smem_base - smem_u32(smem_raw) + CF::kContentBytes > dyn_size) {   // uniform over the CTA
      if (threadIdx.x == 0 && t.status != nullptr) atomicCAS(t.status, 0u, wait_code(KPF, 15));
      return;
    }
  }

  pdl_wait();          // the plan may be the work of the kernel before
  pdl_trigger();
  int head, rank;
  tile_to_head_and_rank(g, blockIdx.x, g.pair_cap, head, rank);
  const int4 entry = from_l2(reinterpret_cast<const int4*>(g.pair_tiles + rank));
  const int r0 = entry.x;
  if (r0 < 0 || r0 >= g.N_q) return;
  const int end = min(max(entry.z, r0 + 1), g.N_q), row_end = min(r0 + 256, end), begin = min(entry.y, r0);
  const int lo = begin < 0 ? r0 : max(begin, r0 - g.window + 1);
  if (begin < 0 || g.window == 0) {      // rows of no sequence, or that see nothing
    store_packed_rows<true>(t.out_O, 0u, r0, row_end, head, g.q_heads, g.D, kThreads);
    if (threadIdx.x < 256 && r0 + (int)threadIdx.x < row_end) t.out_L[(size_t)head * g.N_q + r0 + threadIdx.x] = -INFINITY;
    return;
  }
  // B may have no rows, and with a window its first keys come later
  const ProductOrder order = pair_order(r0, row_end, lo, g.window, kKeys);
  const int tiles = order.tiles;

  auto bar_slot_full = [&](int s) { return smem_u32(&ctl->slot_full[s]); };
  auto bar_slot_empty = [&](int s) { return smem_u32(&ctl->slot_empty[s]); };
  const uint32_t bar_q = smem_u32(&ctl->q_full);
  if (warp == kLoadWarp && lane == 0) {
    mbar_init(bar_q, 1);
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(bar_slot_full(s), 1);
      mbar_init(bar_slot_empty(s), CF::kOwnP ? 2 : 1);      // issuing warps
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(smem_u32(&ctl->ragged_full[x]), 1);
      mbar_init(smem_u32(&ctl->s_full[x]), 1);
      mbar_init(smem_u32(&ctl->s_free[x]), CF::kTileWarps);
      mbar_init(smem_u32(&ctl->p_full[x]), CF::kTileWarps);
      mbar_init(smem_u32(&ctl->pv_done[x]), 1);
      mbar_init(smem_u32(&ctl->acc_done[x]), 1);
    }
    ctl->abort_flag = 0u;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  const int kv_head = head / g.group, last_rows = (row_end - lo) % kKeys;
  // item i of the ring: K (even) or V (odd) of tile i / 2
  auto request = [&](int i) {
    const int s = i % kSlots, j = i >> 1;
    const uint32_t bar = last_rows != 0 && j + 1 == tiles ? smem_u32(&ctl->ragged_full[i & 1]) : bar_slot_full(s);
    mbar_arrive_expect_tx(bar, CF::kTileBytes);
#pragma unroll
    for (int a = 0; a < kAtoms; ++a)
      tma_load_3d(ring + s * CF::kTileBytes + a * kAtomBytes, &maps.m[(i & 1) ? T_V : T_K], a * 64, lo + j * kKeys, kv_head, bar);
  };
  if (warp == kLoadWarp && lane == 0) {
    const int q_tiles = order.to(1) > 0 ? 2 : 1;
    mbar_arrive_expect_tx(bar_q, q_tiles * CF::kTileBytes);
    for (int x = 0; x < q_tiles; ++x)
#pragma unroll
      for (int a = 0; a < kAtoms; ++a)
        tma_load_3d(smem_base + x * CF::kTileBytes + a * kAtomBytes, &maps.m[T_Q], a * 64, r0 + 128 * x, head, bar_q);
    request(0);
  }
  if (warp == kIssueWarp) tmem_alloc(smem_u32(&ctl->tmem_base), 512);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = ctl->tmem_base;
  volatile uint32_t* abort_flag = &ctl->abort_flag;
  auto wait = [&](uint32_t bar, uint32_t parity, int id) {      // a whole warp
    return (bool)__all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, t.status, wait_code(KPF, id)));
  };

  // 640 threads: the launch gives every one 96 registers; the 16 math warps take 104, the others 64 (5 x 96 = 4 x 104 + 64)
  if (warp >= kLoadWarp) {
    if constexpr (kThreads == 640) registers_down<64>();
  if (warp == kLoadWarp) {
    bool ok = true;
    for (int i = 1; i < 2 * tiles && ok; ++i) {
      if (i >= kSlots) ok = wait(bar_slot_empty(i % kSlots), ((i / kSlots) & 1) ^ 1, 1);
      if (ok && lane == 0) request(i);
      __syncwarp();
    }
    // the rows behind the range in the last two tiles (tc_common.cuh); no tile before them waits for this
    if (last_rows != 0)
      for (int h = 0; h < 2 && ok; ++h) {
        ok = wait(smem_u32(&ctl->ragged_full[h]), 0, 2);
        if (!ok) break;
        const int s = (2 * (tiles - 1) + h) % kSlots;
        const uint32_t tile = ring + s * CF::kTileBytes;
        for (int a = 0; a < kAtoms; ++a)
          for (int c = lane; c < (kKeys - last_rows) * 8; c += 32)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + a * kAtomBytes + last_rows * 128 + c * 16), "r"(0u) : "memory");
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_slot_full(s));
      }
    if (!ok) {   // give copies already in flight a bounded chance to land before the CTA exits
      const long long t0 = clock64();
      while (clock64() - t0 < 2000000LL) { }
    }
  } else if (warp == kIssueWarp || (CF::kOwnP && warp == kIssueWarp + 1)) {
    with_k_steps<DT>(g.D, [&](auto k_steps) {
      constexpr int kSteps = decltype(k_steps)::value, KS = kSteps > 0 ? kSteps : DT / 16;
      const int ks_n = kSteps > 0 ? KS : g.D >> 4;
      constexpr uint32_t idesc_s = make_idesc(128, kKeys, Pack<T>::kIsBf16, 0, 0);
      const uint32_t idesc_o = make_idesc(128, g.D, Pack<T>::kIsBf16, 0, 1);
      auto step = [](int ks) { return (uint64_t)(((ks >> 2) * kAtomBytes + (ks & 3) * 32) >> 4); };
      Arrivals known;
      auto arrived = [&](int i) { return known(i, [&](int n) { return wait(bar_slot_full(n % kSlots), (n / kSlots) & 1, 3); }); };
      // an item that a row tile does not use: its slot is given back all the same
      auto skip = [&](int i) {
        const bool here = arrived(i);
        if (here && lane == 0) mbar_arrive(bar_slot_empty(i % kSlots));
        return here;
      };
      // `release`: no other product of this warp reads the item
      auto scores = [&](int x, int j, bool release) {
        if (!arrived(2 * j)) return false;
        tc_fence_after_sync();
        const int s = (2 * j) % kSlots;
        const uint64_t dq = smem_desc_sw128(smem_base + x * CF::kTileBytes, 16, 1024), dk = smem_desc_sw128(ring + s * CF::kTileBytes, 16, 1024);
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
            if (ks < ks_n) mma_ss(tmem_base + 128 * x, dq + step(ks), dk + step(ks), idesc_s, ks > 0);
          mma_commit(smem_u32(&ctl->s_full[x]));
          if (release) mma_commit(bar_slot_empty(s));
        }
        __syncwarp();
        return true;
      };
      auto outputs = [&](int x, int j, bool release) {
        if (!arrived(2 * j + 1) || !wait(smem_u32(&ctl->p_full[x]), (j - order.from(x)) & 1, 5 + x)) return false;
        tc_fence_after_sync();
        const int s = (2 * j + 1) % kSlots;
        const uint64_t dv = smem_desc_sw128(ring + s * CF::kTileBytes, kAtomBytes, 1024);
        const uint32_t o_tmem = tmem_base + CF::kO + DT * x, p_tmem = tmem_base + CF::kP + CF::kPStride * x;
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < kKeys / 16; ++ks)
            mma_ts(o_tmem, p_tmem + 8 * ks, dv + (uint64_t)((ks * 2048) >> 4), idesc_o, j > order.from(x) || ks > 0);
          if (CF::kOwnP) mma_commit(smem_u32(&ctl->pv_done[x]));
          if (j + 1 == order.to(x)) mma_commit(smem_u32(&ctl->acc_done[x]));
          if (release) mma_commit(bar_slot_empty(s));
        }
        __syncwarp();
        return true;
      };
      if (!wait(bar_q, 0, 4)) return;
      if constexpr (CF::kOwnP) {
        auto free = [&](int x, int j) { return wait(smem_u32(&ctl->s_free[x]), (j - order.from(x)) & 1, 9); };
        issue_one_row_tile(order, warp - kIssueWarp, skip, free, scores, outputs);
      } else {
        issue_both_row_tiles(order, arrived, scores, outputs);
      }
    });
  }
  } else {
    if constexpr (kThreads == 640) registers_up<104>();
    const int x = warp / CF::kTileWarps, half = kHalves == 2 ? (warp >> 2) & 1 : 0, quarter = warp & 3, row = quarter * 32 + lane, i = r0 + 128 * x + row;
    const int from = order.from(x), to = order.to(x);
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_addr = lane_addr + 128 * x + kCols * half, o_addr = lane_addr + CF::kO + DT * x + DT / kHalves * half;
    const uint32_t p_addr = lane_addr + CF::kP + CF::kPStride * x + kCols / 2 * half;
    float* const exchange = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(ctl) + 512 + x * CF::kExchange);      // [turns][2 halves][128]
    // keys [vlo, vhi) are visible to this row
    const bool in = i < row_end;
    const int vlo = in ? max(begin, i - g.window + 1) : 0, vhi = in ? max(i + 1, vlo) : 0;
    const uint32_t vspan = (uint32_t)(vhi - vlo);
    float m_ref = -INFINITY, l_sum = 0.f;      // l_sum: of this half of the columns
    bool ok = true;
    const float2 sc2 = make_float2(g.scale_log2e, g.scale_log2e);
    for (int j = from; j < to; ++j) {
      ok = wait(smem_u32(&ctl->s_full[x]), (j - from) & 1, 7);
      tc_fence_after_sync();
      uint32_t s_[kCols / 32][32];
#pragma unroll
      for (int c = 0; c < kCols / 32; ++c) tmem_ld32(s_addr + 32 * c, s_[c]);
#pragma unroll
      for (int c = 0; c < kCols / 32; ++c) tmem_ld_wait32(s_[c]);
      const int j0 = lo + j * kKeys + kCols * half;
      if (__any_sync(0xffffffffu, !(j0 >= vlo && j0 + kCols <= vhi))) {
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((uint32_t)(j0 + 32 * c + e - vlo) < vspan)) s_[c][e] = 0xff800000u;   // -inf
      }
      float mx;
      {
        float m4[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {      // four chains, three scores to an instruction
          constexpr int kEach = kCols / 4;
          auto v = [&](int e) { return __uint_as_float(s_[(kEach * c + e) >> 5][(kEach * c + e) & 31]); };
          m4[c] = max3(v(0), v(1), v(2));
#pragma unroll
          for (int e = 3; e < kEach - 1; e += 2) m4[c] = max3(m4[c], v(e), v(e + 1));
          m4[c] = fmaxf(m4[c], v(kEach - 1));
        }
        mx = fmaxf(max3(m4[0], m4[1], m4[2]), m4[3]);
      }
      if constexpr (kHalves == 2) {      // a row has one reference for both halves of its columns
        float* const slot = exchange + ((j - from) & 1) * 256;
        slot[half * 128 + row] = mx;
        ok = named_barrier_all(1 + x, kTileThreads, ok);      // the warps of a row tile go on, or give up, together
        if (ok) mx = fmaxf(mx, slot[(half ^ 1) * 128 + row]);
      }
      if (!ok) break;
      mx *= g.scale_log2e;
      if constexpr (CF::kOwnP) {
        tc_fence_before_sync();
        if (lane == 0) mbar_arrive(smem_u32(&ctl->s_free[x]));      // the scores of the next tile may come
        // P V of the tile before: where P has its own columns, scores that are complete do not tell
        if (j > from) {
          ok = wait(smem_u32(&ctl->pv_done[x]), (j - from - 1) & 1, 10);
          tc_fence_after_sync();
        }
      }
      const bool grow = mx > m_ref + 8.f || (m_ref == -INFINITY && mx > -INFINITY);
      if (__any_sync(0xffffffffu, grow)) {
        const float m_new = grow ? mx : m_ref, f = m_ref == -INFINITY ? 0.f : ex2(m_ref - m_new);      // 1 for the rows that do not move
        l_sum *= f;
        m_ref = m_new;
        if (j > from) {
#pragma unroll
          for (int c = 0; c < DT / kHalves / 16; ++c) {
            if (DT / kHalves * half + 16 * c >= g.D) break;
            uint32_t o_[16];
            tmem_ld16(o_addr + 16 * c, o_);
            tmem_ld_wait(o_);
#pragma unroll
            for (int e = 0; e < 16; ++e) o_[e] = __float_as_uint(__uint_as_float(o_[e]) * f);
            tmem_st16(o_addr + 16 * c, o_);
          }
        }
      }
      const float nm = m_ref == -INFINITY ? 0.f : -m_ref;      // no visible key yet: every score is -inf, every p 0
      const float2 nm2 = make_float2(nm, nm);
      float2 sum_a = make_float2(0.f, 0.f), sum_b = make_float2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < kCols / 32; ++c) {
        uint32_t kp[16];
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float2 xa = __ffma2_rn(make_float2(__uint_as_float(s_[c][e]), __uint_as_float(s_[c][e + 1])), sc2, nm2);
          const float2 xb = __ffma2_rn(make_float2(__uint_as_float(s_[c][e + 2]), __uint_as_float(s_[c][e + 3])), sc2, nm2);
          const float2 pa = make_float2(ex2(xa.x), ex2(xa.y)), pb = make_float2(ex2(xb.x), ex2(xb.y));
          sum_a = __fadd2_rn(sum_a, pa);
          sum_b = __fadd2_rn(sum_b, pb);
          kp[e >> 1] = Pack<T>::pack(pa.x, pa.y);
          kp[(e >> 1) + 1] = Pack<T>::pack(pb.x, pb.y);
        }
        tmem_st16(p_addr + 16 * c, kp);
      }
      l_sum += (sum_a.x + sum_a.y) + (sum_b.x + sum_b.y);
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl->p_full[x]));
    }
    if (to > from) {
      float* const slot = exchange + ((to - from) & 1) * 256;
      if constexpr (kHalves == 2) slot[half * 128 + row] = l_sum;
      ok = named_barrier_all(1 + x, kTileThreads, ok && mbar_wait(smem_u32(&ctl->acc_done[x]), 0, abort_flag, t.status, wait_code(KPF, 8)));
      tc_fence_after_sync();
      if (ok) {
        const float l = kHalves == 2 ? slot[row] + slot[128 + row] : l_sum;
        const bool nan_row = l != l;      // a visible score that is not a number goes on to the result
        const float inv = nan_row ? l : l > 0.f ? 1.f / l : 0.f;
        if (in && half == 0) t.out_L[(size_t)head * g.N_q + i] = nan_row ? l : l > 0.f ? (m_ref + log2f(l)) * kLn2 : -INFINITY;
        // through the shared memory of this tile's Q, which every score product has read
        const uint32_t out = smem_base + x * CF::kTileBytes;
#pragma unroll
        for (int c = 0; c < DT / kHalves / 16; ++c) {
          const int col = DT / kHalves * half + 16 * c;
          if (col >= g.D) break;     // padding columns
          uint32_t o_[16], w[8];
          tmem_ld16(o_addr + 16 * c, o_);
          tmem_ld_wait(o_);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            // an empty row's O was never a number of its own
            const float v0 = inv == 0.f ? 0.f : __uint_as_float(o_[2 * e]) * inv, v1 = inv == 0.f ? 0.f : __uint_as_float(o_[2 * e + 1]) * inv;
            w[e] = Pack<T>::pack(v0, v1);
          }
          if (in) store_op16(out + (uint32_t)(col >> 6) * kAtomBytes, row, col & 63, w);
        }
        const int rows = min(row_end - (r0 + 128 * x), 128);
        if (rows < 128) {
          named_barrier_sync(1 + x, kTileThreads);
          const int chunks = g.D >> 3;
          for (int k = threadIdx.x % kTileThreads; k < rows * chunks; k += kTileThreads) {
            const int r = k / chunks, c = k - r * chunks;
            uint4 v;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                         : "r"(out + (uint32_t)(c >> 3) * kAtomBytes + sw128_offset(r, (c & 7) * 8)) : "memory");
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(t.out_O) + ((size_t)(r0 + 128 * x + r) * g.q_heads + head) * g.D + c * 8) = v;
          }
        } else {
          fence_proxy_async_smem();
          named_barrier_sync(1 + x, kTileThreads);
          if (threadIdx.x % kTileThreads == 0) {
            for (int a = 0; a * 64 < g.D; ++a) tma_store_3d(&maps.out[TO_O], out + a * kAtomBytes, a * 64, r0 + 128 * x, head);
            bulk_commit_group();
            bulk_wait_group_read_all();
          }
        }
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == kIssueWarp) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512);
  }
}

template <int DT, typename T>
cudaError_t launch_one(const TmaMaps& maps, const PackedGeometry& g_in, const Tensors& t, cudaStream_t s) {
  using CF = Cfg2<DT>;
  PackedGeometry g = g_in;
  g.BH = g.q_heads;
  const long long ctas = (long long)g.BH * g.pair_cap;
  if (ctas > 0x7fffffffLL) return cudaErrorInvalidValue;
  g.head_group = packed_head_group(g, ctas, 2ll * g.kv_heads * g.N_kv * g.D * 2);
  static std::atomic<unsigned long long> smem_set{0};
  auto kern = packed_fwd_kernel<DT, T>;
  const cudaError_t e = set_smem_once(kern, CF::kSmemBytes, smem_set);
  return e != cudaSuccess ? e : launch_pdl(kern, (unsigned)ctas, CF::kThreads, CF::kSmemBytes, s, maps, g, t);
}

}  // namespace

cudaError_t launch_packed_fwd_pairs(int is_bf16, const TmaMaps& maps, const PackedGeometry& g, const Tensors& t, cudaStream_t s) {
  if (g.D <= 64) return is_bf16 ? launch_one<64, __nv_bfloat16>(maps, g, t, s) : launch_one<64, __half>(maps, g, t, s);
  return is_bf16 ? launch_one<128, __nv_bfloat16>(maps, g, t, s) : launch_one<128, __half>(maps, g, t, s);
}

}  // namespace tc
}  // namespace attn
