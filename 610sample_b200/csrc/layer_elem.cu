// Elementwise passes of the layers' backward passes, each one read of its inputs and one write of its results, and sums over rows.
//
//   activation     dz = g a'(z), and the bias' gradient, the sum of dz over the rows (of g without an activation)
//   second         along the tangent t of z: to g  t a'(z),  s = g a''(z) t, and dz again; the sum of s over the rows
//   gated second   h = a(z) u along the tangents (zt, ut), with gh the gradient of h and gh2 the part of h's own gradient that the tangent of Wd makes:
//                  ht = a' zt u + a ut,  ez = gh a' u,  eu = gh a,  dz = gh (a'' zt u + a' ut) + gh2 a' u,  du = gh a' zt + gh2 a
//
// A CTA of 256 threads has 256 columns, eight to a thread (neighbouring threads' in sequence with 16-byte accesses, or one by one where widths or
// addresses do not allow that), and a run of rows, eight at a time.  In the first pass a thread has several rows on their way: with an activation four of half types (two:
// 45 us) and two of float32, without one twice as many; the others have two.  16384 x 2048 bf16 (ncu, cold): the first pass with gelu and the bias' gradient, 201 MB, 36 to 38 us
// (5.4 TB/s) and 6 for the sums over the runs; the second, 403 MB, 72; of a gated block, 772 MB, 150.
#include "activation.cuh"
#include "layer_launch.h"

namespace attn {
namespace layer {

using tc::from_l2;

constexpr int kElemCols = 256;

template <typename T, bool WIDE>
struct Columns {
  static __device__ __forceinline__ int at(int c0, int e) { return WIDE ? c0 + (int)(threadIdx.x & 31) * 8 + e : c0 + e * 32 + (int)(threadIdx.x & 31); }
  // the same in two steps, so that several rows can be on their way at once
  struct Raw { uint32_t w[WIDE && sizeof(T) == 2 ? 4 : 8]; };
  static __device__ __forceinline__ Raw fetch(const void* p, long long ld, int r, int c0, int m) {
    Raw raw;
    if constexpr (WIDE && sizeof(T) == 2) {
      const uint4 a = at(c0, 0) < m ? from_l2(reinterpret_cast<const uint4*>(static_cast<const T*>(p) + r * ld + at(c0, 0))) : make_uint4(0u, 0u, 0u, 0u);
      raw.w[0] = a.x; raw.w[1] = a.y; raw.w[2] = a.z; raw.w[3] = a.w;
    } else {
      float f[8];
      load(p, ld, r, c0, m, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) raw.w[e] = __float_as_uint(f[e]);
    }
    return raw;
  }
  static __device__ __forceinline__ void values(const Raw& raw, float (&f)[8]) {
    if constexpr (WIDE && sizeof(T) == 2) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 b = tc::Pack<T>::unpack(raw.w[e]);
        f[2 * e] = b.x; f[2 * e + 1] = b.y;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(raw.w[e]);
    }
  }
  static __device__ __forceinline__ void load(const void* p, long long ld, int r, int c0, int m, float (&f)[8]) {
    const T* row = static_cast<const T*>(p) + r * ld;
    if constexpr (WIDE) {      // m is a multiple of 8
      if (at(c0, 0) >= m) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = 0.f;
      } else if constexpr (sizeof(T) == 4) {
        const float4 a = from_l2(reinterpret_cast<const float4*>(row + at(c0, 0))), b = from_l2(reinterpret_cast<const float4*>(row + at(c0, 0)) + 1);
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
      } else {
        const uint4 a = from_l2(reinterpret_cast<const uint4*>(row + at(c0, 0)));
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 b = tc::Pack<T>::unpack(w[e]);
          f[2 * e] = b.x; f[2 * e + 1] = b.y;
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = at(c0, e) < m ? Elem<T>::to_float(row[at(c0, e)]) : 0.f;
    }
  }
  // z and u as a gated product keeps them, whose upper halves have been loaded as if they were values of the type
  static __device__ __forceinline__ void with_low(const void* low, long long ld, int r, int c0, int m, float (&z)[8], float (&u)[8]) {
    const uint8_t* row = static_cast<const uint8_t*>(low) + r * ld;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t b = at(c0, e) < m ? row[at(c0, e)] : 0u;
      z[e] = Kept<T>::value(kept_code<0>(bits(z[e]), kept_z(b)));
      u[e] = Kept<T>::value(kept_code<0>(bits(u[e]), kept_u(b)));
    }
  }
  static __device__ __forceinline__ uint32_t bits(float v) {
    const T h = Elem<T>::from_float(v);
    return *reinterpret_cast<const uint16_t*>(&h);
  }
  static __device__ __forceinline__ void store(void* p, long long ld, int r, int c0, int m, const float (&f)[8]) {
    T* row = static_cast<T*>(p) + r * ld;
    if constexpr (WIDE) {
      if (at(c0, 0) >= m) return;
      if constexpr (sizeof(T) == 4) {
        float4* q = reinterpret_cast<float4*>(row + at(c0, 0));
        q[0] = make_float4(f[0], f[1], f[2], f[3]);
        q[1] = make_float4(f[4], f[5], f[6], f[7]);
      } else {
        *reinterpret_cast<uint4*>(row + at(c0, 0)) =
            make_uint4(tc::Pack<T>::pack(f[0], f[1]), tc::Pack<T>::pack(f[2], f[3]), tc::Pack<T>::pack(f[4], f[5]), tc::Pack<T>::pack(f[6], f[7]));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (at(c0, e) < m) row[at(c0, e)] = Elem<T>::from_float(f[e]);
    }
  }
};

template <typename T, int PASS, int ACT, bool WIDE>
__global__ void __launch_bounds__(256)
elementwise_kernel(const __grid_constant__ ElementArgs a) {
  constexpr bool kPrecise = sizeof(T) == 4;
  typedef Columns<T, WIDE> C;
  typedef Columns<typename ArgumentOf<T>::type, WIDE> Z;      // z of a plain product
  __shared__ float sums[8][kElemCols];
  tc::pdl_wait();
  tc::pdl_trigger();
  const int c0 = (int)blockIdx.x * kElemCols, group = threadIdx.x >> 5;
  const long long first = (long long)blockIdx.y * a.chunk;
  const int end = (int)(first + a.chunk < a.n ? first + a.chunk : a.n);
  float sum[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[e] = 0.f;
  auto load = [&](int i, int r, float (&f)[8]) { C::load(a.in[i], a.ld_in[i], r, c0, a.m, f); };
  auto store = [&](int i, int r, const float (&f)[8]) { C::store(a.out[i], a.ld_out[i], r, c0, a.m, f); };
  if constexpr (PASS == PASS_FIRST) {
    constexpr int kRows = (sizeof(T) == 2 ? 4 : 2) * (ACT == ACT_NONE ? 2 : 1);      // of a thread, on their way at once
    for (int r0 = (int)first + group; r0 < end; r0 += 8 * kRows) {
      typename C::Raw rg[kRows];
      typename Z::Raw rz[ACT != ACT_NONE ? kRows : 1];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int r = min(r0 + 8 * i, end - 1);
        rg[i] = C::fetch(a.in[0], a.ld_in[0], r, c0, a.m);
        if constexpr (ACT != ACT_NONE) rz[i] = Z::fetch(a.in[1], a.ld_in[1], r, c0, a.m);
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int r = r0 + 8 * i;
        if (r >= end) break;      // uniform within a warp
        float g[8];
        C::values(rg[i], g);
        if constexpr (ACT != ACT_NONE) {
          float z[8];
          Z::values(rz[i], z);
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            if constexpr (kPrecise) {
              float v, d1, d2;
              activate<ACT, true, 1>(z[e], v, d1, d2);
              g[e] *= d1;
              activate<ACT, true, 1>(z[e + 1], v, d1, d2);
              g[e + 1] *= d1;
            } else {
              float2 v, d;
              activate2<ACT, true>(make_float2(z[e], z[e + 1]), v, d);
              g[e] *= d.x;
              g[e + 1] *= d.y;
            }
          }
          store(0, r, g);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += g[e];
      }
    }
  } else
#pragma unroll 2
  for (int r = (int)first + group; r < end; r += 8) {
    float g[8], z[8];
    load(0, r, g);
    if constexpr (PASS == PASS_SECOND) {
      float t[8], gg[8], s[8];
      Z::load(a.in[1], a.ld_in[1], r, c0, a.m, z);
      load(2, r, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v, d1, d2;
        activate<ACT, kPrecise, 2>(z[e], v, d1, d2);
        gg[e] = t[e] * d1;
        s[e] = g[e] * d2 * t[e];
        g[e] *= d1;
        sum[e] += s[e];
      }
      store(0, r, gg);
      store(1, r, s);
      store(2, r, g);
    } else {
      float u[8], zt[8], ut[8], gh2[8], ht[8], ez[8], eu[8], dz[8], du[8];
      load(1, r, z);
      load(2, r, u);
      if constexpr (!kPrecise) C::with_low(a.low, a.ld_low, r, c0, a.m, z, u);
      load(3, r, zt);
      load(4, r, ut);
      if (a.in[5] != nullptr) load(5, r, gh2);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v, d1, d2;
        activate<ACT, kPrecise, 2>(z[e], v, d1, d2);
        const float own = a.in[5] != nullptr ? gh2[e] : 0.f;
        ht[e] = fmaf(d1 * zt[e], u[e], v * ut[e]);
        ez[e] = g[e] * d1 * u[e];
        eu[e] = g[e] * v;
        dz[e] = fmaf(g[e], fmaf(d2 * zt[e], u[e], d1 * ut[e]), own * d1 * u[e]);
        du[e] = fmaf(g[e], d1 * zt[e], own * v);
      }
      store(0, r, ht);
      store(1, r, ez);
      store(2, r, eu);
      store(3, r, dz);
      store(4, r, du);
    }
  }
  if (a.partial == nullptr) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) sums[group][C::at(0, e)] = sum[e];
  __syncthreads();
  const int c = c0 + (int)threadIdx.x;
  if (c >= a.m) return;
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) v += sums[i][threadIdx.x];
  a.partial[(size_t)blockIdx.y * a.m + c] = v;
}

// column sums: out[k][c] = sum over the rows of partial [rows][kinds][d], in order; a CTA has 32 columns of one kind
template <typename P>
__global__ void __launch_bounds__(1024)
sum_rows_kernel(const float* partial, int rows, int kinds, int d, P* out0, P* out1) {
  __shared__ float s[32][32];
  tc::pdl_wait();
  tc::pdl_trigger();
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + x, k = blockIdx.y;
  float v = 0.f;
  if (c < d)
#pragma unroll 10
    for (int i = y; i < rows; i += 32) v += from_l2(partial + ((size_t)i * kinds + k) * d + c);
  s[y][x] = v;
  __syncthreads();
  if (y != 0 || c >= d) return;
#pragma unroll
  for (int i = 1; i < 32; ++i) v += s[i][x];
  P* out = k == 0 ? out0 : out1;
  if (out != nullptr) out[c] = Elem<P>::from_float(v);
}

cudaError_t launch_sum_rows(const float* partial, int rows, int kinds, int d, int dtype, void* out0, void* out1, cudaStream_t stream) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((d + 31) / 32), (unsigned)kinds);
  cfg.blockDim = dim3(1024);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (dtype == ATTN_F16) return cudaLaunchKernelEx(&cfg, sum_rows_kernel<__half>, partial, rows, kinds, d, (__half*)out0, (__half*)out1);
  if (dtype == ATTN_BF16) return cudaLaunchKernelEx(&cfg, sum_rows_kernel<__nv_bfloat16>, partial, rows, kinds, d, (__nv_bfloat16*)out0, (__nv_bfloat16*)out1);
  return cudaLaunchKernelEx(&cfg, sum_rows_kernel<float>, partial, rows, kinds, d, (float*)out0, (float*)out1);
}


// Rows into rows of another pitch, for widths that the tensor cores' loads do not take as they are: one element of `sizeof(U)` bytes at a time, neighbouring
// threads on neighbouring elements.  The ten copies of a gated block's pass of odd widths took
// the host 80 us as tensor operations, about 55 so.  I: unsigned where all elements have one.
template <typename U, typename I>
__global__ void __launch_bounds__(256)
copy_rows_kernel(const U* src, long long lds, U* dst, long long ldd, I total, I cols) {
  tc::pdl_wait();
  tc::pdl_trigger();
  const I step = (I)gridDim.x * 256;
#pragma unroll 4
  for (I i = (I)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
    const I r = i / cols, c = i - r * cols;
    dst[(long long)r * ldd + c] = src[(long long)r * lds + c];
  }
}

template <typename U>
static cudaError_t copy_rows(const void* src, long long lds, void* dst, long long ldd, int rows, int cols, cudaStream_t stream) {
  const unsigned long long total = (unsigned long long)rows * cols, want = (total + 1023) / 1024;
  const unsigned ctas = (unsigned)(want < 16 * kSms ? want : 16 * kSms);
  if (total < (1ull << 31))      // a step beyond the last element stays below 2^32
    return tc::launch_pdl(copy_rows_kernel<U, unsigned>, ctas, 256u, 0, stream, (const U*)src, lds, (U*)dst, ldd, (unsigned)total, (unsigned)cols);
  return tc::launch_pdl(copy_rows_kernel<U, unsigned long long>, ctas, 256u, 0, stream, (const U*)src, lds, (U*)dst, ldd, total, (unsigned long long)cols);
}
cudaError_t launch_copy_rows(const void* src, long long lds, void* dst, long long ldd, int rows, int cols, int size, cudaStream_t stream) {
  return size == 2 ? copy_rows<uint16_t>(src, lds, dst, ldd, rows, cols, stream) : copy_rows<uint32_t>(src, lds, dst, ldd, rows, cols, stream);
}

// ---- host ---------------------------------------------------------------------------------------
// Runs of rows: as many as make six CTAs an SM, 64 rows each at least.  The first pass in half types has 54 registers (without an activation) or 64 (gelu), and four
// CTAs run on an SM: 888 of them (16384 x 2048) are 1.5 waves
int element_chunks(int n, int m) {
  const long long tiles = ((long long)m + kElemCols - 1) / kElemCols;
  if (tiles == 0) return 1;
  long long chunks = (6 * kSms + tiles - 1) / tiles;
  if (chunks > (n + 63) / 64) chunks = (n + 63) / 64;
  return chunks < 1 ? 1 : (int)chunks;
}

template <typename T, int PASS, int ACT>
static cudaError_t launch(const ElementArgs& a, bool wide, unsigned chunks, cudaStream_t stream) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.m + kElemCols - 1) / kElemCols), chunks);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return wide ? cudaLaunchKernelEx(&cfg, elementwise_kernel<T, PASS, ACT, true>, a) : cudaLaunchKernelEx(&cfg, elementwise_kernel<T, PASS, ACT, false>, a);
}
template <typename T, int PASS>
static cudaError_t launch_act(const ElementArgs& a, int act, bool wide, unsigned chunks, cudaStream_t stream) {
  if (act == ACT_SILU) return launch<T, PASS, ACT_SILU>(a, wide, chunks, stream);
  if (act == ACT_GELU) return launch<T, PASS, ACT_GELU>(a, wide, chunks, stream);
  if (act == ACT_GELU_TANH) return launch<T, PASS, ACT_GELU_TANH>(a, wide, chunks, stream);
  return launch<T, PASS, ACT_NONE>(a, wide, chunks, stream);
}
template <typename T>
static cudaError_t launch_pass(const ElementArgs& a, int pass, int act, bool wide, unsigned chunks, cudaStream_t stream) {
  if (pass == PASS_FIRST) return launch_act<T, PASS_FIRST>(a, act, wide, chunks, stream);
  if (pass == PASS_SECOND) return launch_act<T, PASS_SECOND>(a, act, wide, chunks, stream);
  return launch_act<T, PASS_GATED_SECOND>(a, act, wide, chunks, stream);
}

cudaError_t launch_elementwise(ElementArgs a, int pass, int act, int dtype, cudaStream_t stream) {
  const int chunks = element_chunks(a.n, a.m), size = dtype == ATTN_F32 ? 4 : 2;
  a.chunk = (a.n + chunks - 1) / chunks;
  bool wide = a.m % 8 == 0;
  auto look = [&](const void* p, long long ld) { wide = wide && reinterpret_cast<uintptr_t>(p) % 16 == 0 && (p == nullptr || ld * size % 16 == 0); };
  for (int i = 0; i < 6; ++i) look(a.in[i], a.ld_in[i]);
  for (int i = 0; i < 5; ++i) look(a.out[i], a.ld_out[i]);
  if (dtype == ATTN_F16) return launch_pass<__half>(a, pass, act, wide, (unsigned)chunks, stream);
  if (dtype == ATTN_BF16) return launch_pass<__nv_bfloat16>(a, pass, act, wide, (unsigned)chunks, stream);
  return launch_pass<float>(a, pass, act, wide, (unsigned)chunks, stream);
}

}  // namespace layer
}  // namespace attn
