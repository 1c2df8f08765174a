// layer_block.cu — 8-bit (e4m3) operands with an FP32 scale for each block of 128 values:
// made from rows (1 x 128) or from weights (128 x 128), turned back into values, and their
// product (the kernels are in layer_gemm_rows.cu).
//
// Making codes is bound by HBM: a block's values stay in registers between its largest
// magnitude and their codes, so x is read once.  scale is the largest magnitude times 1/448
// and a code x / scale, each rounded once to nearest (CodeScale gives correctly rounded
// quotients), so codes are those of the same formula in any IEEE arithmetic.
#include <algorithm>

#include "layer_gemm_rows.cuh"
#include "layer_linear.cuh"

namespace vcsr {
namespace layer {
namespace {

constexpr int kLanes = 16, kPer = kScaleBlock / kLanes;  // that hold 128 values, and how many each

// A lane's 8 values of a block of columns of a row (n of them in the row), zeros beyond.
template <class T, bool VEC>
__device__ __forceinline__ void block_load(const T *p, int n, float *out) {
  if (VEC && n >= kPer) {
    const Vec<T, kPer> v = load_vec<T, kPer>(p);
#pragma unroll
    for (int j = 0; j < kPer; ++j) out[j] = widen(v.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) out[j] = j < n ? widen(p[j]) : 0.0f;
  }
}
template <bool VEC>
__device__ __forceinline__ void block_store(uint8_t *p, int n, const CodeScale &c, const float *x) {
  float q[kPer];
#pragma unroll
  for (int j = 0; j < kPer; j += 2) {
    const float2 y = c.quotients<true>(make_float2(x[j], x[j + 1]));
    q[j] = y.x;
    q[j + 1] = y.y;
  }
  if (VEC && n >= kPer) {
    store_codes<kPer>(p, q);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (j < n) p[j] = e4m3_code(q[j]);
  }
}
__device__ __forceinline__ float block_top(const float *x) {
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < kPer; ++j) top = max_or_nan(top, fabsf(x[j]));
  return top;
}

// Blocks of 1 x 128: 16 lanes each.
template <class T, bool VEC>
__global__ void __launch_bounds__(256)
    quantize_rows_kernel(const T *x, int64_t ldx, uint8_t *codes, int64_t ldc, float *scale, int64_t lds, int64_t rows,
                         int64_t dim) {
  const int64_t across = (dim + kScaleBlock - 1) / kScaleBlock, total = rows * across;
  const int lane = threadIdx.x % kLanes;
  // both halves of a warp take the same number of turns
  for (int64_t i = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes; i - (threadIdx.x / kLanes & 1) < total;
       i += (int64_t)gridDim.x * (256 / kLanes)) {
    const bool live = i < total;
    const int64_t r = live ? i / across : 0, b = live ? i - r * across : 0, c = b * kScaleBlock + lane * kPer;
    const int n = live ? (int)max((int64_t)0, min((int64_t)kPer, dim - c)) : 0;
    float v[kPer];
    block_load<T, VEC>(x + r * ldx + c, n, v);
    float top = block_top(v);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o /= 2) top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    const CodeScale s = code_scale(top);
    block_store<VEC>(codes + r * ldc + c, n, s, v);
    if (live && lane == 0) scale[r * lds + b] = s.scale;
  }
}

// Blocks of 128 x 128: 256 threads each, 16 rows at a time.
template <class T, bool VEC>
__global__ void __launch_bounds__(256)
    quantize_tiles_kernel(const T *x, int64_t ldx, uint8_t *codes, int64_t ldc, float *scale, int64_t lds, int64_t rows,
                          int64_t dim) {
  __shared__ float tops[8];
  const int lane = threadIdx.x % kLanes, sub = threadIdx.x / kLanes;
  constexpr int kAtOnce = 256 / kLanes, kTurns = kScaleBlock / kAtOnce;
  const int64_t c = (int64_t)blockIdx.x * kScaleBlock + lane * kPer, r0 = (int64_t)blockIdx.y * kScaleBlock + sub;
  const int n = (int)max((int64_t)0, min((int64_t)kPer, dim - c));
  float v[kTurns][kPer], top = 0.0f;
#pragma unroll
  for (int k = 0; k < kTurns; ++k) {
    const int64_t r = r0 + k * kAtOnce;
    block_load<T, VEC>(x + r * ldx + c, r < rows ? n : 0, v[k]);
    top = max_or_nan(top, block_top(v[k]));
  }
#pragma unroll
  for (int o = 16; o > 0; o /= 2) top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 8; ++k) top = max_or_nan(top, tops[k]);
  const CodeScale s = code_scale(top);
#pragma unroll
  for (int k = 0; k < kTurns; ++k) {
    const int64_t r = r0 + k * kAtOnce;
    block_store<VEC>(codes + r * ldc + c, r < rows ? n : 0, s, v[k]);
  }
  if (threadIdx.x == 0) scale[blockIdx.y * lds + blockIdx.x] = s.scale;
}

// V values from codes, a divisor of 128.
template <int V>
__global__ void __launch_bounds__(256)
    dequantize_blocks_kernel(const uint8_t *codes, int64_t ldc, const float *scale, int64_t lds, int64_t rows,
                             int64_t dim, int block_rows, void *out, int64_t ldo, int dtype) {
  const int64_t per_row = dim / V, total = rows * per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per_row, c = (i - r * per_row) * V;
    const Vec<uint8_t, V> q = load_vec<uint8_t, V>(codes + r * ldc + c);
    const float s = scale[(block_rows == 1 ? r : r / kScaleBlock) * lds + c / kScaleBlock];
    float o[V];
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = e4m3_value(q.v[j]) * s;
    store_as<V>(out, dtype, r * ldo + c, o);
  }
}

// ------------------------------------------------------------------ host

vcsr_status check_blocks(int64_t rows, int64_t dim, int block_rows) {
  if (rows < 0 || dim < 0) return fail(VCSR_ERR_INVALID, "negative size");
  if (block_rows != 1 && block_rows != kScaleBlock)
    return fail(VCSR_ERR_UNSUPPORTED, "blocks of %d rows (1 or %d)", block_rows, kScaleBlock);
  if (rows > 0x7fffffffll || dim > 0x7fffffffll) return fail(VCSR_ERR_RANGE, "a size above 2^31 - 1");
  return VCSR_OK;
}

template <class T>
vcsr_status launch_quantize(const void *from, int64_t ldx, int64_t rows, int64_t dim, int block_rows, void *to,
                            int64_t ldc, float *scale, int64_t lds, cudaStream_t st) {
  const T *x = static_cast<const T *>(from);
  uint8_t *codes = static_cast<uint8_t *>(to);
  const bool vec = aligned(x, 16) && ldx * (int64_t)sizeof(T) % 16 == 0 && aligned(codes, kPer) && ldc % kPer == 0;
  if (block_rows == 1) {
    const int64_t total = rows * ceil_div(dim, kScaleBlock);
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(total, 256 / kLanes), (int64_t)sm_count() * 32);
    if (vec)
      quantize_rows_kernel<T, true><<<grid, 256, 0, st>>>(x, ldx, codes, ldc, scale, lds, rows, dim);
    else
      quantize_rows_kernel<T, false><<<grid, 256, 0, st>>>(x, ldx, codes, ldc, scale, lds, rows, dim);
    return VCSR_OK;
  }
  if (ceil_div(rows, kScaleBlock) > 65535) return fail(VCSR_ERR_RANGE, "more than 65535 blocks of rows");
  const dim3 grid((unsigned)ceil_div(dim, kScaleBlock), (unsigned)ceil_div(rows, kScaleBlock));
  if (vec)
    quantize_tiles_kernel<T, true><<<grid, 256, 0, st>>>(x, ldx, codes, ldc, scale, lds, rows, dim);
  else
    quantize_tiles_kernel<T, false><<<grid, 256, 0, st>>>(x, ldx, codes, ldc, scale, lds, rows, dim);
  return VCSR_OK;
}

vcsr_status quantize(const void *x, int64_t ldx, int64_t rows, int64_t dim, int x_dtype, int block_rows, void *codes,
                     int64_t ldc, float *scale, int64_t lds, cudaStream_t st) {
  VCSR_TRY(check_blocks(rows, dim, block_rows));
  if (!is_float16_or_32(x_dtype)) return fail(VCSR_ERR_UNSUPPORTED, "x type %d", x_dtype);
  if (rows == 0 || dim == 0) return VCSR_OK;
  VCSR_TRY(check_matrix("x", x, ldx, dim, x_dtype, false));
  VCSR_TRY(check_matrix("codes", codes, ldc, dim, VCSR_E4M3, false));
  VCSR_TRY(check_matrix("scale", scale, lds, ceil_div(dim, kScaleBlock), VCSR_F32, false));
  vcsr_status done;
  if (x_dtype == VCSR_F32)
    done = launch_quantize<float>(x, ldx, rows, dim, block_rows, codes, ldc, scale, lds, st);
  else if (x_dtype == VCSR_BF16)
    done = launch_quantize<__nv_bfloat16>(x, ldx, rows, dim, block_rows, codes, ldc, scale, lds, st);
  else
    done = launch_quantize<__half>(x, ldx, rows, dim, block_rows, codes, ldc, scale, lds, st);
  VCSR_TRY(done);
  VCSR_CUDA(cudaGetLastError());
  return VCSR_OK;
}

vcsr_status dequantize(const void *codes, int64_t ldc, const float *scale, int64_t lds, int64_t rows, int64_t dim,
                       int block_rows, void *out, int64_t ldo, int out_dtype, cudaStream_t st) {
  VCSR_TRY(check_blocks(rows, dim, block_rows));
  if (!is_float16_or_32(out_dtype)) return fail(VCSR_ERR_UNSUPPORTED, "out type %d", out_dtype);
  if (rows == 0 || dim == 0) return VCSR_OK;
  VCSR_TRY(check_matrix("codes", codes, ldc, dim, VCSR_E4M3, false));
  VCSR_TRY(check_matrix("scale", scale, lds, ceil_div(dim, kScaleBlock), VCSR_F32, false));
  VCSR_TRY(check_matrix("out", out, ldo, dim, out_dtype, false));
  const uint8_t *c = static_cast<const uint8_t *>(codes);
  auto fits = [&](int v) {
    return dim % v == 0 && ldc % v == 0 && aligned(c, v) && aligned(out, 16) && ldo * (int64_t)type_size(out_dtype) % 16 == 0;
  };
  const int v = fits(16) ? 16 : fits(4) ? 4 : 1;
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(rows * (dim / v), 256), (int64_t)sm_count() * 16);
  if (v == 16)
    dequantize_blocks_kernel<16><<<grid, 256, 0, st>>>(c, ldc, scale, lds, rows, dim, block_rows, out, ldo, out_dtype);
  else if (v == 4)
    dequantize_blocks_kernel<4><<<grid, 256, 0, st>>>(c, ldc, scale, lds, rows, dim, block_rows, out, ldo, out_dtype);
  else
    dequantize_blocks_kernel<1><<<grid, 256, 0, st>>>(c, ldc, scale, lds, rows, dim, block_rows, out, ldo, out_dtype);
  VCSR_CUDA(cudaGetLastError());
  return VCSR_OK;
}

size_t block_linear_workspace(const vcsr_block_linear_args *a) {
  if (a->M <= 0 || a->N <= 0 || a->K <= 0) return 0;
  return packed(a->x, a->ldx, a->M, a->K, VCSR_E4M3).bytes + packed(a->w, a->ldw, a->N, a->K, VCSR_E4M3).bytes;
}

vcsr_status block_linear(const vcsr_block_linear_args *a, cudaStream_t st) {
  if (!a) return fail(VCSR_ERR_INVALID, "no arguments");
  VCSR_TRY(check_sizes(a->M, a->N, a->K));
  if (!is_float16_or_32(a->out_dtype)) return fail(VCSR_ERR_UNSUPPORTED, "output type %d", a->out_dtype);
  if (a->act < VCSR_ACT_NONE || a->act > VCSR_ACT_SILU)
    return fail(VCSR_ERR_UNSUPPORTED, "activation %d", a->act);
  if (a->M == 0 || a->N == 0) return VCSR_OK;
  const int64_t blocks = ceil_div(a->K, kScaleBlock);
  if (a->K > 0) {
    VCSR_TRY(check_matrix("x", a->x, a->ldx, a->K, VCSR_E4M3, false));
    VCSR_TRY(check_matrix("w", a->w, a->ldw, a->K, VCSR_E4M3, false));
    VCSR_TRY(check_matrix("x_scale", a->x_scale, a->ldxs, blocks, VCSR_F32, false));
    VCSR_TRY(check_matrix("w_scale", a->w_scale, a->ldws, blocks, VCSR_F32, false));
  }
  VCSR_TRY(check_matrix("bias", a->bias, a->N, a->N, a->out_dtype, true));
  VCSR_TRY(check_matrix("residual", a->residual, a->ldr, a->N, a->out_dtype, true));
  VCSR_TRY(check_matrix("y", a->y, a->ldy, a->N, a->out_dtype, false));
  const Epilogue e{nullptr, nullptr, a->bias, a->residual, a->y, nullptr, a->ldr, a->ldy, 0, a->act, a->out_dtype};
  if (a->K == 0) return launch_gemm({a->M, a->N, 0, {}, {}, VCSR_E4M3, e}, st);
  const Packed px = packed(a->x, a->ldx, a->M, a->K, VCSR_E4M3), pw = packed(a->w, a->ldw, a->N, a->K, VCSR_E4M3);
  VCSR_TRY(check_workspace(a->workspace, a->workspace_bytes, block_linear_workspace(a)));
  Prepare before(a->workspace);
  RowsGemm g{};
  g.M = a->M;
  g.N = a->N;
  g.K = a->K;
  g.x = before.matrix(px, a->x, a->ldx, a->M, a->K, VCSR_E4M3);
  g.w = before.matrix(pw, a->w, a->ldw, a->N, a->K, VCSR_E4M3);
  VCSR_TRY(before.run(VCSR_E4M3, st));
  g.ldx = px.ld;
  g.ldw = pw.ld;
  g.dtype = VCSR_E4M3;
  g.e = e;
  g.x_scale = a->x_scale;
  g.w_scale = a->w_scale;
  g.ldxs = a->ldxs;
  g.ldws = a->ldws;
  return launch_blocks_tc(g, st);
}

}  // namespace
}  // namespace layer
}  // namespace vcsr

extern "C" {

vcsr_status vcsr_block_quantize(const void *x, int64_t ldx, int64_t rows, int64_t dim, int x_dtype, int block_rows,
                                void *codes, int64_t ldc, float *scale, int64_t lds, vcsr_stream_t stream) {
  vcsr::clear_error();
  return vcsr::no_throw([&] {
    return vcsr::layer::quantize(x, ldx, rows, dim, x_dtype, block_rows, codes, ldc, scale, lds, (cudaStream_t)stream);
  });
}

vcsr_status vcsr_block_dequantize(const void *codes, int64_t ldc, const float *scale, int64_t lds, int64_t rows,
                                  int64_t dim, int block_rows, void *out, int64_t ldo, int out_dtype,
                                  vcsr_stream_t stream) {
  vcsr::clear_error();
  return vcsr::no_throw([&] {
    return vcsr::layer::dequantize(codes, ldc, scale, lds, rows, dim, block_rows, out, ldo, out_dtype,
                                   (cudaStream_t)stream);
  });
}

vcsr_status vcsr_block_linear(const vcsr_block_linear_args *a, vcsr_stream_t stream) {
  vcsr::clear_error();
  return vcsr::no_throw([&] { return vcsr::layer::block_linear(a, (cudaStream_t)stream); });
}

size_t vcsr_block_linear_workspace(const vcsr_block_linear_args *a) {
  return a ? vcsr::layer::block_linear_workspace(a) : 0;
}

}  // extern "C"
