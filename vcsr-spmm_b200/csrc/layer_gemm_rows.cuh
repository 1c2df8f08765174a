// layer_gemm_rows.cuh — the products whose epilogue works along an output row (gated
// pairs of columns, 8-bit operands with a scale for each block of 128): layer_gemm_rows.cu.
#pragma once
#include "layer_gemm.cuh"

namespace vcsr {
namespace layer {

// The values of k, and the rows of w, that share a scale.
constexpr int kScaleBlock = 128;

// out[i, j] over k of x (M x K) and w, both stored along k, bases and pitches multiples of
// 16 bytes, K > 0.
//   gated:  w is 2N x K; act(g) u of its sums with row j of w (g) and row N + j (u);
//           e.bias and e.col_scale have 2N values, e.pre 2N columns.
//   blocks: w is N x K; the sum of each kScaleBlock values of k is multiplied by x_scale
//           [i, block] and w_scale[j / kScaleBlock, block].
struct RowsGemm {
  int64_t M, N, K;
  const void *x, *w;
  int64_t ldx, ldw;
  int dtype;
  Epilogue e;
  const float *x_scale, *w_scale;
  int64_t ldxs, ldws;
};
vcsr_status launch_gated_tc(const RowsGemm &g, cudaStream_t st);
vcsr_status launch_blocks_tc(const RowsGemm &g, cudaStream_t st);
vcsr_status take_wait_error_rows(int *word);

}  // namespace layer
}  // namespace vcsr
