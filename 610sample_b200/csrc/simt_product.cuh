// Tiles of matrix products on the CUDA cores, in fp32: a CTA of 256 threads computes 128 x 128 results, 8 x 8 a thread, over blocks of 16 in k
// that go through shared memory, the next one on its way into registers meanwhile.  A thread brings eight elements of either operand, along whichever
// axis is dense, with 16-byte loads where that axis' extent and the addresses allow it.
#pragma once

#include "attn_common.cuh"
#include "tc_common.cuh"

namespace attn {
namespace simt {

using tc::from_l2;

constexpr int kTile = 128, kBlock = 16, kPitch = kTile + 4;

// element (i, k) of an operand at p[i * si + k * sk]; one of the strides is 1
template <typename T> struct Operand { const T* p; long long si, sk; int wide; };      // wide: runs of eight are 16-byte aligned

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

// sum += the product of A's and B's [128][k_begin, k_end), which bring_a(k0, v) and bring_b fetch; `buf` goes on from call to call.
// Rows of the thread: (t / 16) * 8 + i; columns: (t % 16) * 4 + j, and 64 more.
template <typename BringA, typename BringB>
__device__ __forceinline__ void accumulate(float (&as)[2][kBlock * kPitch], float (&bs)[2][kBlock * kPitch], int& buf, int k_begin, int k_end,
                                           BringA bring_a, BringB bring_b, bool ka, bool kb, float2 (&sum)[8][4]) {
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  float va[8], vb[8];
  bring_a(k_begin, va);
  bring_b(k_begin, vb);
  for (int k0 = k_begin; k0 < k_end; k0 += kBlock, buf ^= 1) {
    put(as[buf], va, ka);
    put(bs[buf], vb, kb);
    __syncthreads();
    if (k0 + kBlock < k_end) {
      bring_a(k0 + kBlock, va);
      bring_b(k0 + kBlock, vb);
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
}
__device__ __forceinline__ void clear(float2 (&sum)[8][4]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[i][j] = make_float2(0.f, 0.f);
}

// a share of k: whole blocks, so that runs of eight that are aligned in the first share are so in every one
inline long long share_of(long long k, long long splits) { return ((k + splits - 1) / splits + kBlock - 1) / kBlock * kBlock; }

inline int wide(const void* p, long long ld, int size) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * size % 16 == 0; }
template <typename T> inline Operand<T> rows_of(const void* p, long long ld) { return {static_cast<const T*>(p), ld, 1, wide(p, ld, sizeof(T))}; }
template <typename T> inline Operand<T> columns_of(const void* p, long long ld) { return {static_cast<const T*>(p), 1, ld, wide(p, ld, sizeof(T))}; }


}  // namespace simt
}  // namespace attn
