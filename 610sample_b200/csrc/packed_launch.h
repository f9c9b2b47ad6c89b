// Internal launcher interface of the packed-batch kernels, between the C ABI (packed_capi.cu) and the kernel files.
#pragma once
#include "attn_launch.h"
#include "packed_geometry.cuh"

namespace attn {

// Elements from row to row and from head to head of the inputs; outputs are dense [n_tok, heads, D].
struct PackedStrides { long long row, head; };
enum PackedInput { PI_Q = 0, PI_K, PI_V, PI_dO, PI_COUNT };
struct PackedLayout { PackedStrides of[PI_COUNT]; };

cudaError_t launch_packed_plan(const int* cu_seqlens, int* plan, int n_tok, int n_seq, cudaStream_t s);

// f16 / bf16 on the tensor cores; inputs 16-byte aligned with strides that are multiples of 8 elements
cudaError_t launch_packed_tc(int op, int dtype, const PackedGeometry& g, const Tensors& t, const PackedLayout& lay, cudaStream_t s,
                             int* launches, const char** err);
// float32 on the CUDA cores; dense inputs
cudaError_t launch_packed_simt(int op, const PackedGeometry& g, const Tensors& t, cudaStream_t s, int* launches);

}  // namespace attn
