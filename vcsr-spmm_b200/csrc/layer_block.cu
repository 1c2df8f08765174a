// layer_block.cu — 8-bit (e4m3) operands with an FP32 scale for each block of 128 values:
// made from rows (1 x 128) or from weights (128 x 128), turned back into values, and their
// product (the kernels are in layer_gemm_rows.cu).
//
// Making codes is bound by HBM and by instructions: a block's values stay in registers
// between its largest magnitude and their codes, so x is read once.  16384 x 4096 bf16 by rows
// 42 us (4.8 TB/s; 72% of issue slots), FP32 52 (6.5 TB/s), 16384 x 8192 by 128 x 128 FP32 107
// (6.3), bf16 112 (3.6); values of 16384 x 4096 codes as bf16 43 (4.7).  Rows off 16 bytes are
// moved by their elements: 16384 x 4097 bf16 180 us, its values 374.  Eight lanes take a block:
// with sixteen, whose exchanges and scales serve half as many values, rows took 63 us and values
// 60.  scale is the largest magnitude times 1/448 and a code x / scale, each rounded once to
// nearest (CodeScale gives correctly rounded quotients), so codes are those of the same formula
// in any IEEE arithmetic.
#include <algorithm>

#include "layer_gemm_rows.cuh"
#include "layer_linear.cuh"

namespace vcsr {
namespace layer {
namespace {

constexpr int kLanes = 8, kPer = kScaleBlock / kLanes;  // that hold 128 values, and how many each

// kPer values at p, the first n of them (zeros beyond), moved `bytes` at a time: a power of
// two from the element's size to 16 that p is a multiple of.
template <int BYTES, class T>
__device__ __forceinline__ void load_by(const T *p, Vec<T, kPer> &v) {
  constexpr int W = BYTES / sizeof(T);
#pragma unroll
  for (int i = 0; i < kPer; i += W) *reinterpret_cast<Vec<T, W> *>(v.v + i) = load_vec<T, W>(p + i);
}
template <class T>
__device__ __forceinline__ Vec<T, kPer> load_some(const T *p, int n, int bytes) {
  Vec<T, kPer> v;
  if (n >= kPer && bytes == 16) {
    load_by<16>(p, v);
  } else if (n >= kPer && bytes == 8) {
    load_by<8>(p, v);
  } else if (n >= kPer && bytes == 4) {
    load_by<4>(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) v.v[j] = j < n ? p[j] : T{};
  }
  return v;
}
template <int BYTES, class T>
__device__ __forceinline__ void store_by(T *p, const Vec<T, kPer> &v) {
  constexpr int W = BYTES / sizeof(T);
#pragma unroll
  for (int i = 0; i < kPer; i += W) store_vec<T, W>(p + i, *reinterpret_cast<const Vec<T, W> *>(v.v + i));
}
template <class T>
__device__ __forceinline__ void store_some(T *p, int n, int bytes, const Vec<T, kPer> &v) {
  if (n >= kPer && bytes == 16) {
    store_by<16>(p, v);
  } else if (n >= kPer && bytes == 8) {
    store_by<8>(p, v);
  } else if (n >= kPer && bytes == 4) {
    store_by<4>(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (j < n) p[j] = v.v[j];
  }
}

// The largest magnitude, NaN where a value is one: 16-bit values two at a time.
template <class T>
__device__ __forceinline__ float top_of(const Vec<T, kPer> &v) {
  if constexpr (sizeof(T) == 2) {
    using P = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    const P *pairs = reinterpret_cast<const P *>(v.v);
    P top = __habs2(pairs[0]);
#pragma unroll
    for (int j = 1; j < kPer / 2; ++j) top = __hmax2_nan(top, __habs2(pairs[j]));
    return max_or_nan(widen(top.x), widen(top.y));
  } else {
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) top = max_or_nan(top, fabsf(widen(v.v[j])));
    return top;
  }
}
// Codes of a lane's values.
template <class T>
__device__ __forceinline__ Vec<uint8_t, kPer> codes_of(const CodeScale &c, const Vec<T, kPer> &v) {
  float2 q[kPer / 2];
  if (c.raise == 1.0f) {
#pragma unroll
    for (int j = 0; j < kPer / 2; ++j) q[j] = c.quotients<false>(make_float2(widen(v.v[2 * j]), widen(v.v[2 * j + 1])));
  } else {
#pragma unroll
    for (int j = 0; j < kPer / 2; ++j) q[j] = c.quotients<true>(make_float2(widen(v.v[2 * j]), widen(v.v[2 * j + 1])));
  }
  Vec<uint8_t, kPer> o;
#pragma unroll
  for (int j = 0; j < kPer / 2; ++j)
    reinterpret_cast<uint16_t *>(o.v)[j] = __nv_cvt_float2_to_fp8x2(q[j], __NV_SATFINITE, __NV_E4M3);
  return o;
}

constexpr int kBlocksPerSm = 6;

struct BlockArgs {
  const void *x;  // values, or codes to be turned back
  void *out;      // codes, or values
  float *scale;
  int64_t ldx, ldo, lds, rows;
  int dim, across;     // values and blocks of a row
  int x_bytes, o_bytes;  // that neighbouring values can be moved by
  int block_rows;
};

// A thread's place: groups of 8 lanes take neighbouring blocks of columns, and rows where
// the blocks are fewer than a thread block's 32 groups; no division.
struct Place {
  int block, lane, n;  // n: values of the lane's that are in the row
  int64_t row, step;
  __device__ __forceinline__ Place(const BlockArgs &a, int wide) {  // log2 of groups side by side
    const int group = threadIdx.x / kLanes;
    lane = threadIdx.x % kLanes;
    block = (blockIdx.x << wide) + (group & ((1 << wide) - 1));
    const int down = (blockDim.x / kLanes) >> wide;
    row = (int64_t)blockIdx.y * down + (group >> wide);
    step = (int64_t)gridDim.y * down;
    n = (int)max((int64_t)0, min((int64_t)kPer, a.dim - ((int64_t)block * kScaleBlock + lane * kPer)));
  }
};

// Blocks of 1 x 128, 8 lanes each.
template <class T>
__global__ void __launch_bounds__(256, kBlocksPerSm) quantize_rows_kernel(const __grid_constant__ BlockArgs a, int wide) {
  const Place at(a, wide);
  const int64_t column = (int64_t)at.block * kScaleBlock + at.lane * kPer;
  const T *x = static_cast<const T *>(a.x) + column;
  uint8_t *codes = static_cast<uint8_t *>(a.out) + column;
  // the rows of a warp's groups may differ: all take the turns of the first
  const int64_t warp_row = __shfl_sync(0xffffffffu, at.row, 0);
  for (int64_t r = at.row, w = warp_row; w < a.rows; r += at.step, w += at.step) {
    const Vec<T, kPer> v = load_some<T>(x + r * a.ldx, r < a.rows ? at.n : 0, a.x_bytes);
    float top = top_of(v);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o /= 2) top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (r >= a.rows || at.n == 0) continue;
    const CodeScale s = code_scale(top);
    store_some<uint8_t>(codes + r * a.ldo, at.n, a.o_bytes, codes_of(s, v));
    if (at.lane == 0) a.scale[r * a.lds + at.block] = s.scale;
  }
}

// Blocks of 128 x 128: 512 threads each, 64 rows at a time.
template <class T>
__global__ void __launch_bounds__(512, sizeof(T) == 2 ? 3 : 2) quantize_tiles_kernel(const __grid_constant__ BlockArgs a) {
  __shared__ float tops[16];
  const int lane = threadIdx.x % kLanes, sub = threadIdx.x / kLanes;
  constexpr int kAtOnce = 512 / kLanes, kTurns = kScaleBlock / kAtOnce;
  const int64_t down = blockIdx.x / a.across, block = blockIdx.x - down * a.across;
  const int64_t column = block * kScaleBlock + lane * kPer, r0 = down * kScaleBlock + sub;
  const int n = (int)max((int64_t)0, min((int64_t)kPer, a.dim - column));
  const T *x = static_cast<const T *>(a.x) + column;
  uint8_t *codes = static_cast<uint8_t *>(a.out) + column;
  Vec<T, kPer> v[kTurns];
#pragma unroll
  for (int k = 0; k < kTurns; ++k) {
    const int64_t r = r0 + k * kAtOnce;
    v[k] = load_some<T>(x + r * a.ldx, r < a.rows ? n : 0, a.x_bytes);
  }
  float top = 0.0f;
#pragma unroll
  for (int k = 0; k < kTurns; ++k) top = max_or_nan(top, top_of(v[k]));
#pragma unroll
  for (int o = 16; o > 0; o /= 2) top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
  top = tops[threadIdx.x & 15];
#pragma unroll
  for (int o = 8; o > 0; o /= 2) top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  const CodeScale s = code_scale(top);
#pragma unroll
  for (int k = 0; k < kTurns; ++k) {
    const int64_t r = r0 + k * kAtOnce;
    if (r < a.rows) store_some<uint8_t>(codes + r * a.ldo, n, a.o_bytes, codes_of(s, v[k]));
  }
  if (threadIdx.x == 0) a.scale[down * a.lds + block] = s.scale;
}

// Values of codes.
template <class T>
__global__ void __launch_bounds__(256, kBlocksPerSm)
    dequantize_blocks_kernel(const __grid_constant__ BlockArgs a, int wide) {
  const Place at(a, wide);
  const int64_t column = (int64_t)at.block * kScaleBlock + at.lane * kPer;
  const uint8_t *codes = static_cast<const uint8_t *>(a.x) + column;
  T *out = static_cast<T *>(a.out) + column;
  if (at.n == 0) return;
  for (int64_t r = at.row; r < a.rows; r += at.step) {
    const Vec<uint8_t, kPer> q = load_some<uint8_t>(codes + r * a.ldx, at.n, a.x_bytes);
    const float s = a.scale[(a.block_rows == 1 ? r : r / kScaleBlock) * a.lds + at.block];
    float o[kPer];
#pragma unroll
    for (int j = 0; j < kPer; j += 2) {
      const __nv_fp8x2_storage_t two = *reinterpret_cast<const __nv_fp8x2_storage_t *>(q.v + j);
      const float2 y = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3)));
      o[j] = y.x * s;
      o[j + 1] = y.y * s;
    }
    store_some<T>(out + r * a.ldo, at.n, a.o_bytes, narrow_vec<T, kPer>(o));
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

// The most bytes, up to 16, that neighbouring values of a matrix can be moved by.
int access_bytes(const void *p, int64_t ld, int type) {
  const uint64_t bits = reinterpret_cast<uintptr_t>(p) | (uint64_t)(ld * (int64_t)type_size(type)) | 16;
  return (int)(bits & (~bits + 1));
}

// kernel(a, log2 of groups side by side) on blocks of 256 threads, 32 groups of 8 lanes.
template <class K>
void launch_blocks(K kernel, const BlockArgs &a, cudaStream_t st) {
  int wide = 0;
  while (wide < 5 && (1 << wide) < a.across) ++wide;
  const int64_t down = 32 >> wide, columns = ceil_div(a.across, 1 << wide);
  // some rows each, where there are many
  const int64_t rows = std::min<int64_t>(ceil_div(a.rows, down), std::max<int64_t>(1, ceil_div(sm_count() * 4 * kBlocksPerSm, columns)));
  kernel<<<dim3((unsigned)columns, (unsigned)std::min<int64_t>(rows, 65535)), 256, 0, st>>>(a, wide);
}

vcsr_status quantize(const void *x, int64_t ldx, int64_t rows, int64_t dim, int x_dtype, int block_rows, void *codes,
                     int64_t ldc, float *scale, int64_t lds, cudaStream_t st) {
  VCSR_TRY(check_blocks(rows, dim, block_rows));
  if (!is_float16_or_32(x_dtype)) return fail(VCSR_ERR_UNSUPPORTED, "x type %d", x_dtype);
  if (rows == 0 || dim == 0) return VCSR_OK;
  VCSR_TRY(check_matrix("x", x, ldx, dim, x_dtype, false));
  VCSR_TRY(check_matrix("codes", codes, ldc, dim, VCSR_E4M3, false));
  VCSR_TRY(check_matrix("scale", scale, lds, ceil_div(dim, kScaleBlock), VCSR_F32, false));
  const BlockArgs a{x, codes, scale, ldx, ldc, lds, rows, (int)dim, (int)ceil_div(dim, kScaleBlock),
                    access_bytes(x, ldx, x_dtype), access_bytes(codes, ldc, VCSR_E4M3), block_rows};
  const int64_t tiles = a.across * ceil_div(rows, kScaleBlock);
  if (block_rows != 1 && tiles > 0x7fffffffll) return fail(VCSR_ERR_RANGE, "more than 2^31 - 1 blocks");
  for_type(x_dtype, [&](auto t) {
    using T = decltype(t);
    if (block_rows == 1)
      launch_blocks(quantize_rows_kernel<T>, a, st);
    else
      quantize_tiles_kernel<T><<<(unsigned)tiles, 512, 0, st>>>(a);
  });
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
  const BlockArgs a{codes, out, const_cast<float *>(scale), ldc, ldo, lds, rows, (int)dim, (int)ceil_div(dim, kScaleBlock),
                    access_bytes(codes, ldc, VCSR_E4M3), access_bytes(out, ldo, out_dtype), block_rows};
  for_type(out_dtype, [&](auto t) { launch_blocks(dequantize_blocks_kernel<decltype(t)>, a, st); });
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
