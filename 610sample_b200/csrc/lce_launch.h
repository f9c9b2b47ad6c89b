// Cross entropy of a linear layer's outputs: z = x W^T, loss_i = log sum_j exp(z_ij) - z_i,y(i), and its gradients
//   G_ij = c_i (exp(z_ij - lse_i) - [j = y(i)]),  dx = G W,  dW = G^T x
// without ever holding z.  Interface between the C ABI (lce_capi.cu) and the kernel files.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace attn {
namespace lce {

struct Problem {
  int n, d, V;                    // rows of x, width, rows of W
  int dtype;
  long long ignore_index;
  const void *x, *w;              // dense [n, d], [V, d]
  const int64_t* targets;         // [n]
  unsigned int* status;
};

// One value per row and column tile of the forward: maximum (in units of log 2) and sum of 2^(z log2 e - maximum)
struct Partial { float m, l; };

// What the forward's product leaves for the row kernel: partial [tiles][n]; the logit of every row's target
struct Scores {
  Partial* partial;
  float* target_logit;
  int tiles;
};

enum Reduction { RED_NONE = 0, RED_SUM = 1, RED_MEAN = 2 };

// The gradient's row factors: G is formed with coef[i] (0 for rows that do not count), results are multiplied by *scale.
struct Coefficients { float* coef; float* scale; };

// row kernels (lce_rows.cu)
cudaError_t launch_finish(const Problem& p, const Scores& s, float* loss, float* lse, cudaStream_t stream);
// *value = sum or mean over the rows that count, *counted = their number
cudaError_t launch_total(const Problem& p, const float* loss, int reduction, float* value, float* counted, cudaStream_t stream);
// grad: [n] (RED_NONE) or one value; counted: as launch_total left it (RED_MEAN)
cudaError_t launch_coefficients(const Problem& p, const float* grad, const float* counted, int reduction, const Coefficients& c, cudaStream_t stream);
// dst = x with zeros in the rows that do not count
cudaError_t launch_counted_rows(const Problem& p, void* dst, cudaStream_t stream);

// pieces of the vocabulary in the backward
struct Piece { int first, cols, ld; bool is_first, is_last; };

// result = *scale x the sum of `splits` planes of `count` values, in order
cudaError_t launch_sum_splits(const float* acc, int splits, long long count, const float* scale, void* result, int dtype, cudaStream_t stream);

// tensor cores: f16 / bf16, d a multiple of 8, 16-byte aligned tensors; G in the input type.  acc [n, d] floats, where there are several
// pieces; parts: tc_parts_bytes of a product's rows, columns and length in k.  x is launch_counted_rows' copy in dW.  `launches` is added to.
int tc_tiles(int V);
size_t tc_parts_bytes(long long rows, long long cols, long long k);
cudaError_t tc_scores(const Problem& p, const Scores& s, cudaStream_t stream, int* launches, const char** err);
cudaError_t tc_piece_grad(const Problem& p, const Piece& piece, const float* lse, const Coefficients& c, void* G, cudaStream_t stream, int* launches,
                          const char** err);
cudaError_t tc_piece_dx(const Problem& p, const Piece& piece, const Coefficients& c, const void* G, float* parts, float* acc, void* dx,
                        cudaStream_t stream, int* launches, const char** err);
cudaError_t tc_piece_dw(const Problem& p, const Piece& piece, const Coefficients& c, const void* G, const void* x, float* parts, void* dw,
                        cudaStream_t stream, int* launches, const char** err);

// dx: acc [splits][n, d] floats, where there are several pieces or splits; `keep` leaves the sum there after the last piece.
// dW: acc [splits][piece, d], likewise.
// CUDA cores: every type and size; G in float
int simt_tiles(int V);
int simt_splits(long long rows, long long cols, long long k);
cudaError_t simt_scores(const Problem& p, const Scores& s, cudaStream_t stream);
cudaError_t simt_piece_grad(const Problem& p, const Piece& piece, const float* lse, const Coefficients& c, float* G, cudaStream_t stream);
cudaError_t simt_piece_dx(const Problem& p, const Piece& piece, const Coefficients& c, const float* G, int splits, bool keep, float* acc, void* dx,
                          cudaStream_t stream);
cudaError_t simt_piece_dw(const Problem& p, const Piece& piece, const Coefficients& c, const float* G, const void* x, int splits, float* acc,
                          void* dw, cudaStream_t stream);

}  // namespace lce
}  // namespace attn
