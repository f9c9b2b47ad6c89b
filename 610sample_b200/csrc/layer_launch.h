// Operators of a decoder layer between its attention calls.  Interface between the C ABI (layer_capi.cu) and the kernel files.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "attn_b200.h"

namespace attn {
namespace layer {

constexpr int kMaxPairs = ATTN_PRODUCT_PAIRS, kMaxProducts = ATTN_PRODUCT_COUNT, kMaxFactors = 6;

// matrix products on the tensor cores (product_tc.cu): f16 / bf16.  parts: tc_parts_bytes
size_t tc_parts_bytes(const attn_products_t& c);
cudaError_t tc_products(const attn_products_t& c, float* parts, unsigned int* status, cudaStream_t stream, int* launches, const char** why);
// few rows against a weight (product_few.cu): f16 / bf16, what few_rows says
bool few_rows(const attn_products_t& c);
cudaError_t few_products(const attn_products_t& c, cudaStream_t stream, int* launches);
// on the CUDA cores (product_simt.cu): float32
size_t simt_parts_bytes(const attn_products_t& c);
cudaError_t simt_products(const attn_products_t& c, float* parts, cudaStream_t stream, int* launches);

// elementwise passes (layer_elem.cu).  in: g, z | g, z, t | gh, z, u, zt, ut, gh2; out: dz | gg, s, dz | ht, ez, eu, dz, du (`gh2` may be null).
// partial: [element_chunks][m] floats, the sums over runs of rows of dz | s, where wanted
enum Pass { PASS_FIRST = ATTN_ELEMENTS_FIRST, PASS_SECOND = ATTN_ELEMENTS_SECOND, PASS_GATED_SECOND = ATTN_ELEMENTS_GATED_SECOND };
struct ElementArgs {
  int n, m;
  int chunk;                     // rows of a run, filled in by the launch
  const void* in[6];
  long long ld_in[6];
  const void* low;               // the lower bits of z and u, half types of PASS_GATED_SECOND
  long long ld_low;
  void* out[5];
  long long ld_out[5];
  float* partial;
};
int element_chunks(int n, int m);
cudaError_t launch_elementwise(ElementArgs a, int pass, int act, int dtype, cudaStream_t stream);
// dst[r][c] = src[r][c], elements of 2 or 4 bytes
cudaError_t launch_copy_rows(const void* src, long long lds, void* dst, long long ldd, int rows, int cols, int size, cudaStream_t stream);
// out_k[c] = sum over the rows of partial [rows][kinds][d], in order; one or two kinds
cudaError_t launch_sum_rows(const float* partial, int rows, int kinds, int d, int dtype, void* out0, void* out1, cudaStream_t stream);

}  // namespace layer
}  // namespace attn
