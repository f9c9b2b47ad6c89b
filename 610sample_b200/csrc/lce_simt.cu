// The matrix products of the linear cross entropy on the CUDA cores, for float32 and for what the tensor-core kernel does not take
// (widths that are no multiple of 8).  The same four uses as there (lce_tc.cu); G is kept in float.  All arithmetic is in fp32.
// A CTA of 256 threads computes 128 x 128 results, 8 x 8 a thread, over blocks of 16 in k that go through shared memory, the next one
// on its way into registers meanwhile.  A thread brings eight elements of either operand, along whichever axis is dense, with 16-byte loads
// where that axis' extent and the addresses allow it.  At 333 x 200 x 5003 the launches with gradients, nine of 80 to 290 CTAs, take 151 us.  The four
// products, 9 us each at the FMA pipe's rate, take 32 to 38: one CTA of eight warps an SM issues in 37 % of the cycles (packed multiply-adds, of two
// cycles, in 25 %) and else waits for shared memory or the next block, and the SMs are idle for a quarter of the time at either end.  With many tiles,
// 2048 x 770 x 32000 in bf16, the forward takes 3.25 ms, 31 TFLOP/s, and with gradients 14.6.
#include "attn_common.cuh"
#include "lce_launch.h"
#include "tc_common.cuh"

namespace attn {
namespace lce {

using tc::from_l2;

enum Use { LSE = 0, GRAD = 1, DX = 2, DW = 3 };
constexpr int kTile = 128, kBlock = 16, kPitch = kTile + 4;

// element (i, k) of an operand at p[i * si + k * sk]; one of the strides is 1
template <typename T> struct Operand { const T* p; long long si, sk; int wide; };      // wide: runs of eight are 16-byte aligned

struct SimtArgs {
  int rows, cols, k;
  int splits, split_k;           // DX, DW: shares of k
  int first_col, tiles;
  long long tiles_m;
  const int64_t* targets;
  Partial* partial;
  float* target_logit;
  const float *lse, *coef;
  float* G;                      // GRAD: [rows, ld]
  long long ld;
  float* acc;
  int acc_in, acc_out;
  const float* scale;
};

// The eight elements of a [128][16] block that this thread brings: along k of row t / 2, or along i at k = t / 16.
template <typename T>
__device__ __forceinline__ void fetch(const Operand<T>& o, int i0, int k0, int n_i, int n_k, float (&v)[8], bool k_dense) {
  const int t = threadIdx.x, i = i0 + (k_dense ? t >> 1 : (t & 15) * 8), k = k0 + (k_dense ? (t & 1) * 8 : t >> 4);
  const T* p = o.p + i * o.si + k * o.sk;
  if (o.wide && (k_dense ? i < n_i && k + 8 <= n_k : k < n_k && i + 8 <= n_i)) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = from_l2(reinterpret_cast<const float4*>(p)), b = from_l2(reinterpret_cast<const float4*>(p) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 q = from_l2(reinterpret_cast<const uint4*>(p));
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = tc::Pack<T>::unpack(w[e]);
        v[2 * e] = f.x; v[2 * e + 1] = f.y;
      }
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const bool in = k_dense ? i < n_i && k + e < n_k : k < n_k && i + e < n_i;
    v[e] = in ? Elem<T>::to_float(p[e]) : 0.f;
  }
}
__device__ __forceinline__ void put(float* s, const float (&v)[8], bool k_dense) {
  const int t = threadIdx.x;
  if (k_dense) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s[((t & 1) * 8 + e) * kPitch + (t >> 1)] = v[e];
  } else {
    float4* at = reinterpret_cast<float4*>(s + (t >> 4) * kPitch + (t & 15) * 8);
    at[0] = make_float4(v[0], v[1], v[2], v[3]);
    at[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}

template <int USE, typename TA, typename TB, typename T>
__global__ void __launch_bounds__(256)
lce_simt_kernel(const Operand<TA> A, const Operand<TB> B, const SimtArgs g, T* out) {
  __shared__ __align__(16) float as[2][kBlock * kPitch], bs[2][kBlock * kPitch];
  tc::pdl_wait();
  tc::pdl_trigger();
  const int nt = (int)(blockIdx.x / g.tiles_m), r0 = (int)(blockIdx.x - nt * g.tiles_m) * kTile, c0 = nt * kTile, split = blockIdx.y;
  const int k_begin = split * g.split_k, k_end = min(g.k, k_begin + g.split_k);
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;      // rows ty * 8 + i, columns tx * 4 + j and 64 + tx * 4 + j
  const bool ka = A.sk == 1, kb = B.sk == 1;
  float2 sum[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[i][j] = make_float2(0.f, 0.f);
  float va[8], vb[8];
  fetch(A, r0, k_begin, g.rows, k_end, va, ka);
  fetch(B, c0, k_begin, g.cols, k_end, vb, kb);
  int buf = 0;
  for (int k0 = k_begin; k0 < k_end; k0 += kBlock, buf ^= 1) {
    put(as[buf], va, ka);
    put(bs[buf], vb, kb);
    __syncthreads();
    if (k0 + kBlock < k_end) {
      fetch(A, r0, k0 + kBlock, g.rows, k_end, va, ka);
      fetch(B, c0, k0 + kBlock, g.cols, k_end, vb, kb);
    }
#pragma unroll
    for (int k = 0; k < kBlock; ++k) {
      float a[8];
      *reinterpret_cast<float4*>(a) = *reinterpret_cast<const float4*>(&as[buf][k * kPitch + ty * 8]);
      *reinterpret_cast<float4*>(a + 4) = *reinterpret_cast<const float4*>(&as[buf][k * kPitch + ty * 8 + 4]);
      const float4 b0 = *reinterpret_cast<const float4*>(&bs[buf][k * kPitch + tx * 4]), b1 = *reinterpret_cast<const float4*>(&bs[buf][k * kPitch + 64 + tx * 4]);
      const float2 b[4] = {make_float2(b0.x, b0.y), make_float2(b0.z, b0.w), make_float2(b1.x, b1.y), make_float2(b1.z, b1.w)};
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[i][j] = __ffma2_rn(make_float2(a[i], a[i]), b[j], sum[i][j]);
    }
  }
  float acc[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) { acc[i][2 * j] = sum[i][j].x; acc[i][2 * j + 1] = sum[i][j].y; }
  auto col_of = [&](int j) { return c0 + (j >> 2) * 64 + tx * 4 + (j & 3); };
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + ty * 8 + i;
    const bool in = r < g.rows;
    if constexpr (USE == LSE) {
      const int64_t target = in ? from_l2(reinterpret_cast<const long long*>(g.targets) + r) : -1;
      float m = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (col_of(j) >= g.cols) acc[i][j] = -INFINITY;
        else if (in && target == col_of(j)) g.target_logit[r] = acc[i][j];
        m = fmaxf(m, acc[i][j] * kLog2e);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));      // the 16 threads of a row
      const float ref = m == -INFINITY ? 0.f : m;      // logits of -inf alone: every term 0
      float l = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) l += exp2f(fmaf(acc[i][j], kLog2e, -ref));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      if (in && tx == 0) g.partial[(size_t)nt * g.rows + r] = Partial{m, l};
    } else if (in) {
      if constexpr (USE == GRAD) {
        const int64_t target = from_l2(reinterpret_cast<const long long*>(g.targets) + r) - g.first_col;
        const float lse = from_l2(g.lse + r), coef = from_l2(g.coef + r);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = col_of(j);
          if (c < g.cols) g.G[r * g.ld + c] = coef == 0.f ? 0.f : (expf(acc[i][j] - lse) - (target == c ? 1.f : 0.f)) * coef;
        }
      } else {
        const float scale = from_l2(g.scale);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = col_of(j);
          if (c >= g.cols) continue;
          float* at = g.acc + ((size_t)split * g.rows + r) * g.cols + c;
          float v = acc[i][j];
          if (g.acc_in) v += from_l2(at);
          if (g.acc_out) *at = v;
          else out[(size_t)r * g.cols + c] = Elem<T>::from_float(v * scale);
        }
      }
    }
  }
}

// a share of k: whole blocks, so that runs of eight that are aligned in the first share are so in every one
static long long share_of(long long k, long long splits) { return ((k + splits - 1) / splits + kBlock - 1) / kBlock * kBlock; }

template <int USE, typename TA, typename TB, typename T>
static cudaError_t launch_use(const Operand<TA>& A, const Operand<TB>& B, SimtArgs g, T* out, cudaStream_t stream) {
  g.tiles_m = (g.rows + kTile - 1) / kTile;
  const long long tiles = g.tiles_m * ((g.cols + kTile - 1) / kTile);
  if (g.splits < 1) g.splits = 1;
  g.split_k = (int)share_of(g.k, g.splits);
  if (tiles > 0x7fffffffLL || g.splits > 65535) return cudaErrorInvalidValue;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)tiles, (unsigned)g.splits);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, lce_simt_kernel<USE, TA, TB, T>, A, B, g, out);
}

int simt_tiles(int V) { return (V + kTile - 1) / kTile; }

// two CTAs an SM, at least 64 in k a share
int simt_splits(long long rows, long long cols, long long k) {
  const long long tiles = ((rows + kTile - 1) / kTile) * ((cols + kTile - 1) / kTile);
  long long s = 2 * kSms / tiles;
  if (s > k / 64) s = k / 64;
  if (s > 256) s = 256;
  if (s < 2) return 1;
  const long long each = share_of(k, s);
  return (int)((k + each - 1) / each);
}

static int wide(const void* p, long long ld, int size) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * size % 16 == 0; }
template <typename T> static Operand<T> rows_of(const void* p, long long ld) { return {static_cast<const T*>(p), ld, 1, wide(p, ld, sizeof(T))}; }
template <typename T> static Operand<T> columns_of(const void* p, long long ld) { return {static_cast<const T*>(p), 1, ld, wide(p, ld, sizeof(T))}; }

template <typename T>
static cudaError_t scores(const Problem& p, const Scores& s, cudaStream_t stream) {
  SimtArgs g = {};
  g.rows = p.n; g.cols = p.V; g.k = p.d;
  g.targets = p.targets;
  g.partial = s.partial;
  g.target_logit = s.target_logit;
  return launch_use<LSE>(rows_of<T>(p.x, p.d), rows_of<T>(p.w, p.d), g, (T*)nullptr, stream);
}

template <typename T>
static cudaError_t piece_grad(const Problem& p, const Piece& piece, const float* lse, const Coefficients& c, float* G, cudaStream_t stream) {
  SimtArgs g = {};
  g.rows = p.n; g.cols = piece.cols; g.k = p.d;
  g.targets = p.targets;
  g.first_col = piece.first;
  g.lse = lse;
  g.coef = c.coef;
  g.G = G;
  g.ld = piece.ld;
  return launch_use<GRAD>(rows_of<T>(p.x, p.d), rows_of<T>(static_cast<const T*>(p.w) + (size_t)piece.first * p.d, p.d), g, (T*)nullptr, stream);
}

template <typename T>
static cudaError_t piece_dx(const Problem& p, const Piece& piece, const Coefficients& c, const float* G, int splits, bool keep, float* acc, void* dx,
                            cudaStream_t stream) {
  SimtArgs g = {};
  g.rows = p.n; g.cols = p.d; g.k = piece.cols;
  g.splits = splits;
  g.acc = acc;
  g.acc_in = !piece.is_first;
  g.acc_out = !piece.is_last || keep;
  g.scale = c.scale;
  return launch_use<DX>(rows_of<float>(G, piece.ld), columns_of<T>(static_cast<const T*>(p.w) + (size_t)piece.first * p.d, p.d), g, (T*)dx, stream);
}

template <typename T>
static cudaError_t piece_dw(const Problem& p, const Piece& piece, const Coefficients& c, const float* G, const void* x, int splits, float* acc,
                            void* dw, cudaStream_t stream) {
  SimtArgs g = {};
  g.rows = piece.cols; g.cols = p.d; g.k = p.n;
  g.splits = splits;
  g.acc = acc;
  g.acc_out = splits > 1;
  g.scale = c.scale;
  return launch_use<DW>(columns_of<float>(G, piece.ld), columns_of<T>(x, p.d), g, static_cast<T*>(dw) + (size_t)piece.first * p.d, stream);
}

#define BY_TYPE(f, ...) (p.dtype == 0 ? f<__half>(__VA_ARGS__) : p.dtype == 1 ? f<__nv_bfloat16>(__VA_ARGS__) : f<float>(__VA_ARGS__))

cudaError_t simt_scores(const Problem& p, const Scores& s, cudaStream_t stream) { return BY_TYPE(scores, p, s, stream); }
cudaError_t simt_piece_grad(const Problem& p, const Piece& piece, const float* lse, const Coefficients& c, float* G, cudaStream_t stream) {
  return BY_TYPE(piece_grad, p, piece, lse, c, G, stream);
}
cudaError_t simt_piece_dx(const Problem& p, const Piece& piece, const Coefficients& c, const float* G, int splits, bool keep, float* acc, void* dx,
                          cudaStream_t stream) {
  return BY_TYPE(piece_dx, p, piece, c, G, splits, keep, acc, dx, stream);
}
cudaError_t simt_piece_dw(const Problem& p, const Piece& piece, const Coefficients& c, const float* G, const void* x, int splits, float* acc,
                          void* dw, cudaStream_t stream) {
  return BY_TYPE(piece_dw, p, piece, c, G, x, splits, acc, dw, stream);
}

}  // namespace lce
}  // namespace attn
