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
// 16-bit ones (FAST) forms that are off by at most 2^-13 of themselves (a quarter of
// float16's half place, down to values of 1e-35, which may become zero) in a third of the
// instructions: exp and quotient by the hardware's approximations, and Phi, as in
// Abramowitz and Stegun 7.1.26, by erfc(x) = (a1 t + ... + a6 t^6) exp(-x^2) with
// t = 1 / (1 + 0.4126667 x), x = |z| / sqrt(2).  Their five coefficients bound the
// absolute error alone, and gelu of a negative z is that tail: 1e-2 of it at z = -8, over a
// bfloat16 place.  These six were fitted (linear programming on x up to 9.6) to both: 7e-5
// of the tail and 2e-7.

// Phi(-|z|) of two values, and exp(-z^2 / 2) on the way.
__device__ __forceinline__ float2 lower_tails(float2 z, float2 *gauss) {
  auto both = [](float v) { return make_float2(v, v); };
  const float2 d = __ffma2_rn(make_float2(fabsf(z.x), fabsf(z.y)), both(0.4126667f * 0.70710678f), both(1.0f));
  float2 t, e;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t.x) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t.y) : "f"(d.y));
  // half of each coefficient
  float2 p = __ffma2_rn(t, both(-0.5f * 0.17410895f), both(0.5f * 0.54500295f));
  p = __ffma2_rn(p, t, both(-0.5f * 0.15675931f));
  p = __ffma2_rn(p, t, both(0.5f * 0.34406872f));
  p = __ffma2_rn(p, t, both(0.5f * 0.20700936f));
  p = __ffma2_rn(p, t, both(0.5f * 0.23478712f));
  const float2 s = __fmul2_rn(__fmul2_rn(z, z), both(-0.5f * 1.44269504f));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(s.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(s.y));
  *gauss = e;
  return __fmul2_rn(__fmul2_rn(p, t), e);
}
// z Phi(z) = max(z, 0) - |z| Phi(-|z|); the second term is long gone at |z| = 64
__device__ __forceinline__ float2 gelu_pair(float2 z) {
  float2 g;
  const float2 q = lower_tails(z, &g);
  return __ffma2_rn(make_float2(-fminf(fabsf(z.x), 64.0f), -fminf(fabsf(z.y), 64.0f)), q,
                    make_float2(fmaxf(z.x, 0.0f), fmaxf(z.y, 0.0f)));
}
__device__ __forceinline__ float2 gelu_slope_pair(float2 z) {
  float2 g;
  const float2 q = lower_tails(z, &g);
  const float2 phi = make_float2(z.x < 0.0f ? q.x : 1.0f - q.x, z.y < 0.0f ? q.y : 1.0f - q.y);
  return __ffma2_rn(__fmul2_rn(z, make_float2(0.39894228f, 0.39894228f)), g, phi);
}

template <bool FAST>
__device__ __forceinline__ float activate(int act, float z) {
  if (act == VCSR_ACT_RELU) return z < 0.0f ? 0.0f : z;  // a NaN stays
  if (act == VCSR_ACT_GELU) {
    if constexpr (FAST) return gelu_pair(make_float2(z, z)).x;
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
    if constexpr (FAST) return gelu_slope_pair(make_float2(z, z)).x;
    return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) +
           z * 0.39894228040143268f * expf(-0.5f * z * z);
  }
  if (act == VCSR_ACT_SILU) {
    const float s = FAST ? __fdividef(1.0f, 1.0f + __expf(-z)) : 1.0f / (1.0f + expf(-z));
    return s * (1.0f + z * (1.0f - s));
  }
  return 1.0f;
}

// o[j] *= the slope at z[j], N values, the branch outside the loop.
template <int N, bool FAST>
__device__ __forceinline__ void times_slopes(int act, const float *z, float *o) {
  if (act == VCSR_ACT_GELU && FAST && N % 2 == 0) {
#pragma unroll
    for (int j = 0; j + 1 < N; j += 2) {
      const float2 s = gelu_slope_pair(make_float2(z[j], z[j + 1]));
      o[j] *= s.x;
      o[j + 1] *= s.y;
    }
  } else if (act == VCSR_ACT_GELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] *= activate_slope<FAST>(VCSR_ACT_GELU, z[j]);
  } else if (act == VCSR_ACT_SILU) {
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] *= activate_slope<FAST>(VCSR_ACT_SILU, z[j]);
  } else if (act == VCSR_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] *= activate_slope<FAST>(VCSR_ACT_RELU, z[j]);
  }
}

// On the tensor cores: operands whose bases and pitches are multiples of 16 bytes
// (tc_aligned); K > 0.  16-bit operands, and 8-bit ones stored along k; FP32 ones.
vcsr_status launch_gemm_tc(const Gemm &g, cudaStream_t st);
// Two of them (16-bit), in one launch where that is expected to be faster; those without
// an output (e.out NULL) are left out.
vcsr_status launch_gemms_tc(const Gemm &g0, const Gemm &g1, cudaStream_t st);
vcsr_status launch_gemm_f32(const Gemm &g, cudaStream_t st);
bool tc_aligned(const void *p, int64_t ld, int dtype);
vcsr_status take_wait_error_f32(int *word);

}  // namespace layer
}  // namespace vcsr
