// layer_common.cuh — element types and vector access shared by the dense
// layer operators (layer_norm.cu, layer_adamw.cu, layer_linear.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "common.h"

namespace vcsr {
namespace layer {

inline size_t type_size(int t) { return t == VCSR_F32 ? 4 : t == VCSR_E4M3 ? 1 : 2; }
inline bool is_float16_or_32(int t) { return t == VCSR_F32 || t == VCSR_BF16 || t == VCSR_F16; }
inline bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; }

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
// To nearest even: the one rounding of a 16-bit result.
template <class T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half narrow<__half>(float v) {
  return __float2half_rn(v);
}

// N values of type T moved as one access of N * sizeof(T) bytes (a power of
// two up to 16; 32 bytes take two).
template <int BYTES>
struct Raw;
template <>
struct Raw<2> {
  using type = uint16_t;
};
template <>
struct Raw<4> {
  using type = uint32_t;
};
template <>
struct Raw<8> {
  using type = uint2;
};
template <>
struct Raw<16> {
  using type = uint4;
};
template <>
struct Raw<1> {
  using type = uint8_t;
};

template <class T, int N>
struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Vec {
  T v[N];
};

template <class T, int N>
__device__ __forceinline__ Vec<T, N> load_vec(const T *p) {
  Vec<T, N> out;
  constexpr int kBytes = sizeof(T) * N;
  if constexpr (kBytes > 16) {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i)
      reinterpret_cast<uint4 *>(out.v)[i] = reinterpret_cast<const uint4 *>(p)[i];
  } else {
    using R = typename Raw<kBytes>::type;
    *reinterpret_cast<R *>(out.v) = *reinterpret_cast<const R *>(p);
  }
  return out;
}

template <class T, int N>
__device__ __forceinline__ void store_vec(T *p, const Vec<T, N> &x) {
  constexpr int kBytes = sizeof(T) * N;
  if constexpr (kBytes > 16) {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i)
      reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(x.v)[i];
  } else {
    using R = typename Raw<kBytes>::type;
    *reinterpret_cast<R *>(p) = *reinterpret_cast<const R *>(x.v);
  }
}

// N values at p, of a type chosen at run time, as FP32.
template <int N>
__device__ __forceinline__ void load_as_float(const void *p, int type, int64_t at, float *out) {
  if (type == VCSR_F32) {
    const Vec<float, N> x = load_vec<float, N>(static_cast<const float *>(p) + at);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = x.v[i];
  } else if (type == VCSR_BF16) {
    const Vec<__nv_bfloat16, N> x =
        load_vec<__nv_bfloat16, N>(static_cast<const __nv_bfloat16 *>(p) + at);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = widen(x.v[i]);
  } else {
    const Vec<__half, N> x = load_vec<__half, N>(static_cast<const __half *>(p) + at);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = widen(x.v[i]);
  }
}

// N values rounded to T, two per conversion where T has 16 bits.
template <class T, int N>
__device__ __forceinline__ Vec<T, N> narrow_vec(const float *x) {
  Vec<T, N> o;
  if constexpr (sizeof(T) == 2 && N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      if constexpr (std::is_same_v<T, __half>)
        *reinterpret_cast<__half2 *>(o.v + i) = __floats2half2_rn(x[i], x[i + 1]);
      else
        *reinterpret_cast<__nv_bfloat162 *>(o.v + i) = __floats2bfloat162_rn(x[i], x[i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) o.v[i] = narrow<T>(x[i]);
  }
  return o;
}

template <class T, int N>
__device__ __forceinline__ void store_narrow(T *p, const float *x) {
  store_vec<T, N>(p, narrow_vec<T, N>(x));
}

// f(T{}) for the element type named by `type`, which is F32, BF16 or F16.
template <class F>
__device__ __forceinline__ void with_type(int type, F &&f) {
  if (type == VCSR_F32)
    f(float{});
  else if (type == VCSR_BF16)
    f(__nv_bfloat16{});
  else
    f(__half{});
}

// The e4m3 code of a value, to nearest even, magnitudes past 448 stored as
// 448 (a NaN stays one).
__device__ __forceinline__ uint8_t e4m3_code(float v) {
  return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float e4m3_value(uint8_t c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

template <int N>
__device__ __forceinline__ void store_codes(uint8_t *p, const float *x) {
  if constexpr (N % 2 == 0) {
    Vec<uint16_t, N / 2> o;
#pragma unroll
    for (int i = 0; i < N; i += 2)
      o.v[i / 2] = __nv_cvt_float2_to_fp8x2(make_float2(x[i], x[i + 1]), __NV_SATFINITE, __NV_E4M3);
    store_vec<uint16_t, N / 2>(reinterpret_cast<uint16_t *>(p), o);
  } else {
    Vec<uint8_t, N> o;
#pragma unroll
    for (int i = 0; i < N; ++i) o.v[i] = e4m3_code(x[i]);
    store_vec<uint8_t, N>(p, o);
  }
}

// The larger of two magnitudes, NaN where one is: a scale made from it shows that its
// values are not all finite.
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// N values stored in a type chosen at run time.
template <int N>
__device__ __forceinline__ void store_as(void *p, int type, int64_t at, const float *x) {
  if (type == VCSR_F32)
    store_narrow<float, N>(static_cast<float *>(p) + at, x);
  else if (type == VCSR_BF16)
    store_narrow<__nv_bfloat16, N>(static_cast<__nv_bfloat16 *>(p) + at, x);
  else if (type == VCSR_F16)
    store_narrow<__half, N>(static_cast<__half *>(p) + at, x);
  else
    store_codes<N>(static_cast<uint8_t *>(p) + at, x);
}

// The scale of e4m3 codes for values up to `top` in magnitude, and the
// quotient value / scale correctly rounded without a division per value: with
// y = 1/b correctly rounded and q = a y, the remainder r = a - q b is exact in
// one FMA and q + r y is a / b rounded to nearest (Markstein 1990).  Scales
// below 2^-108 are first raised, since their reciprocal overflows FP32.
struct CodeScale {
  float scale, raise, divisor, inverse;
  template <bool RAISED>
  __device__ __forceinline__ float2 quotients(float2 x) const {
    auto both = [](float v) { return make_float2(v, v); };
    const float2 a = RAISED ? __fmul2_rn(x, both(raise)) : x, q = __fmul2_rn(a, both(inverse));
    return __ffma2_rn(__ffma2_rn(make_float2(-q.x, -q.y), both(divisor), a), both(inverse), q);
  }
  __device__ __forceinline__ float quotient(float x) const { return quotients<true>(make_float2(x, x)).x; }
};
__device__ __forceinline__ CodeScale code_scale(float top) {
  CodeScale s;
  s.scale = top * (1.0f / 448.0f);
  s.raise = top < 1e-30f ? 0x1p64f : 1.0f;
  s.divisor = s.scale > 0.0f ? s.scale * s.raise : 1.0f;
  s.inverse = 1.0f / s.divisor;
  return s;
}

// out[c] = the sum of `count` FP32 partial rows of `dim` values, for the 32 columns of
// `group`, by a block of 256 threads: in order within each of 8 slices of the rows, the
// slices then added in order.
__device__ __forceinline__ void column_sum_block(const float *partial, int count, int64_t dim, void *out,
                                                 int dtype, int64_t group, float (*part)[33]) {
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int64_t c = group * 32 + lane;
  float sum = 0.0f;
  if (c < dim) {
    const int per = (count + 7) / 8, lo = slice * per, hi = min(count, lo + per);
#pragma unroll 8
    for (int p = lo; p < hi; ++p) sum += partial[(int64_t)p * dim + c];
  }
  part[slice][lane] = sum;
  __syncthreads();
  if (slice == 0 && c < dim) {
    float total = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) total += part[k][lane];
    store_as<1>(out, dtype, c, &total);
  }
}

// Shared host checks (layer_norm.cu).  check_matrix: a pointer
// (NULL only where optional) aligned to its type, and a pitch that holds a
// row.
vcsr_status check_matrix(const char *name, const void *p, int64_t ld, int64_t dim, int type,
                         bool optional);

// SMs of the current device, and a kernel's dynamic shared memory limit raised to
// `bytes`: asked of the runtime once per device (and kernel), since each question
// costs a good part of a microsecond of every call otherwise (layer_norm.cu).
int sm_count();
vcsr_status allow_shared(const void *kernel, size_t bytes);

}  // namespace layer
}  // namespace vcsr
