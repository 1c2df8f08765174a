// layer_gemm.cuh — the products behind vcsr_linear and its gradient:
//   out[i, j] = epilogue(sum_k A(i, k) B(j, k))
// for operands stored along k or along their own index, with the epilogue's
// mathematics.
#pragma once
#include "layer_common.cuh"

namespace vcsr {
namespace layer {

// An operand (rows x K values of a type): element (r, k) lies at r * ld + k,
// or at k * ld + r where `transposed`.
struct Operand {
  const void *p;
  int64_t ld;
  bool transposed;
};

struct Epilogue {
  const float *row_scale, *col_scale;  // multiply the sum; NULL = 1
  const void *bias;                    // per column j
  const void *residual;
  void *out;
  void *pre;  // the value before the activation
  int64_t ldr, ldo, ldp;
  int act, type;  // type of bias, residual, out and pre
};

struct Gemm {
  int64_t M, N, K;
  Operand a, b;
  int dtype;
  Epilogue e;
};

__device__ __forceinline__ float activate(int act, float z) {
  if (act == VCSR_ACT_RELU) return z < 0.0f ? 0.0f : z;  // a NaN stays
  if (act == VCSR_ACT_GELU) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
  if (act == VCSR_ACT_SILU) return z / (1.0f + expf(-z));
  return z;
}

__device__ __forceinline__ float activate_slope(int act, float z) {
  if (act == VCSR_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  if (act == VCSR_ACT_GELU)
    return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) +
           z * 0.39894228040143268f * expf(-0.5f * z * z);
  if (act == VCSR_ACT_SILU) {
    const float s = 1.0f / (1.0f + expf(-z));
    return s * (1.0f + z * (1.0f - s));
  }
  return 1.0f;
}

// On the FP32 units: any operands.
vcsr_status launch_gemm_simt(const Gemm &g, cudaStream_t st);
// On the tensor cores: 16-bit operands, and 8-bit ones stored along k, whose
// bases and pitches are multiples of 16 bytes (tc_aligned); K > 0.
vcsr_status launch_gemm_tc(const Gemm &g, cudaStream_t st);
bool tc_aligned(const void *p, int64_t ld, int dtype);

}  // namespace layer
}  // namespace vcsr
