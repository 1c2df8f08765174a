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

// Activations and their slopes.  FP32 results take CUDA's erf, exp and division;
// 16-bit ones (FAST) forms that are right to well below their last place in a
// third of the instructions: exp and quotient by the hardware's approximations,
// and Phi by Abramowitz and Stegun 7.1.26, erfc(x) = (a1 t + ... + a5 t^5) exp(-x^2)
// with t = 1 / (1 + 0.3275911 x), |error| <= 1.5e-7, for x = |z| / sqrt(2).

// Phi(-|z|), and exp(-z^2 / 2) on the way.
__device__ __forceinline__ float lower_tail(float z, float *gauss) {
  const float t = __fdividef(1.0f, fmaf(0.3275911f * 0.70710678f, fabsf(z), 1.0f));
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  *gauss = __expf(-0.5f * z * z);
  return 0.5f * p * t * *gauss;
}

template <bool FAST>
__device__ __forceinline__ float activate(int act, float z) {
  if (act == VCSR_ACT_RELU) return z < 0.0f ? 0.0f : z;  // a NaN stays
  if (act == VCSR_ACT_GELU) {
    if constexpr (FAST) {
      float g;
      const float q = lower_tail(z, &g);
      return z * (z < 0.0f ? q : 1.0f - q);
    }
    return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
  }
  if (act == VCSR_ACT_SILU)
    return FAST ? __fdividef(z, 1.0f + __expf(-z)) : z / (1.0f + expf(-z));
  return z;
}

template <bool FAST>
__device__ __forceinline__ float activate_slope(int act, float z) {
  if (act == VCSR_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  if (act == VCSR_ACT_GELU) {
    if constexpr (FAST) {
      float g;
      const float q = lower_tail(z, &g);
      return fmaf(z * 0.39894228040143268f, g, z < 0.0f ? q : 1.0f - q);
    }
    return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) +
           z * 0.39894228040143268f * expf(-0.5f * z * z);
  }
  if (act == VCSR_ACT_SILU) {
    const float s = FAST ? __fdividef(1.0f, 1.0f + __expf(-z)) : 1.0f / (1.0f + expf(-z));
    return s * (1.0f + z * (1.0f - s));
  }
  return 1.0f;
}

// On the tensor cores: operands whose bases and pitches are multiples of 16 bytes
// (tc_aligned); K > 0.  16-bit operands, and 8-bit ones stored along k; FP32 ones.
vcsr_status launch_gemm_tc(const Gemm &g, cudaStream_t st);
vcsr_status launch_gemm_f32(const Gemm &g, cudaStream_t st);
bool tc_aligned(const void *p, int64_t ld, int dtype);
vcsr_status take_wait_error_f32(int *word);

}  // namespace layer
}  // namespace vcsr
