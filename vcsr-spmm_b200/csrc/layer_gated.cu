// layer_gated.cu — vcsr_gated_linear and its gradient: argument checks, and the parts that
// are no matrix product.
//
//   z = x w^T + bias (w: N rows for the gate g, then N for u),  y = act(g) u.
//
// 16- and 8-bit operands: one kernel (layer_gemm_rows.cu) holds both sums of an output.
// FP32 operands take the FP32 product of all 2N columns (layer_gemm_f32.cu, whose tiles hold
// 128 neighbouring columns) into pre, or scratch, and one pass over that.
//
// Gradient: dg = dy u act'(g) and du = dy act(g) are the two halves of dz's rows, rounded to
// the operands' type, made in one pass with dbias' partial sums of the unrounded ones; then
// dx = dz w and dw = dz^T x are single products over 2N values of k and for 2N rows.
// The rounding of dz is a choice: an MMA's operands have one type, and of 16 bits here as w
// and x are, so a second part that held what it drops would be as many products again (392 us
// each below).  It adds 0.0016 (bf16; float16 0.0002) of their norm to dx and dw, whose own
// rounding is 0.0017 (0.0002) of it.
// 4096 x 8192, k = 4096 bf16: dz 52 us (335 MB, 6.4 TB/s), the products 392 each (1,402 TFLOP/s);
// FP32 1024 x 2048, k = 1024 with pre 84 us with operands in L2 and 96 from memory, of which the
// pass over pre takes 15.
#include <algorithm>

#include "layer_gemm_rows.cuh"
#include "layer_linear.cuh"

namespace vcsr {
namespace layer {
namespace {

// V values of act(z) and of its slope.
template <int V, bool FAST>
__device__ __forceinline__ void activate_both(int act, const float *z, float *value, float *slope) {
  if (act == VCSR_ACT_GELU && FAST && V % 2 == 0) {
#pragma unroll
    for (int j = 0; j + 1 < V; j += 2) {
      const float2 at = make_float2(z[j], z[j + 1]);
      float2 g;
      const float2 q = lower_tails(at, &g);
      const float2 y = __ffma2_rn(make_float2(-fminf(fabsf(at.x), 64.0f), -fminf(fabsf(at.y), 64.0f)), q,
                                  make_float2(fmaxf(at.x, 0.0f), fmaxf(at.y, 0.0f)));
      const float2 phi = make_float2(at.x < 0.0f ? q.x : 1.0f - q.x, at.y < 0.0f ? q.y : 1.0f - q.y);
      const float2 s = __ffma2_rn(__fmul2_rn(at, make_float2(0.39894228f, 0.39894228f)), g, phi);
      value[j] = y.x;
      value[j + 1] = y.y;
      slope[j] = s.x;
      slope[j + 1] = s.y;
    }
  } else if (act == VCSR_ACT_SILU) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float s = FAST ? __fdividef(1.0f, 1.0f + __expf(-z[j])) : 1.0f / (1.0f + expf(-z[j]));
      value[j] = z[j] * s;
      slope[j] = s * (1.0f + z[j] * (1.0f - s));
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      value[j] = activate<FAST>(act, z[j]);
      slope[j] = activate_slope<FAST>(act, z[j]);
    }
  }
}

// y = act(g) u from z = [g | u].
template <class T, int V>
__global__ void __launch_bounds__(256)
    combine_kernel(const T *z, int64_t ldz, T *y, int64_t ldy, int64_t M, int64_t N, int act) {
  const int64_t per_row = N / V, total = M * per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per_row, c = (i - r * per_row) * V;
    const Vec<T, V> g = load_vec<T, V>(z + r * ldz + c), u = load_vec<T, V>(z + r * ldz + N + c);
    float o[V];
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = activate<sizeof(T) == 2>(act, widen(g.v[j])) * widen(u.v[j]);
    store_narrow<T, V>(y + r * ldy + c, o);
  }
}

template <class T>
void launch_combine(const void *z, int64_t ldz, void *y, int64_t ldy, int64_t M, int64_t N, int act, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const T *from = static_cast<const T *>(z);
  T *to = static_cast<T *>(y);
  const bool vec = N % V == 0 && ldz % V == 0 && ldy % V == 0 && aligned(z, 16) && aligned(y, 16);
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(M * (vec ? N / V : N), 256), (int64_t)sm_count() * 16);
  if (vec)
    combine_kernel<T, V><<<grid, 256, 0, st>>>(from, ldz, to, ldy, M, N, act);
  else
    combine_kernel<T, 1><<<grid, 256, 0, st>>>(from, ldz, to, ldy, M, N, act);
}

// Block (c, r): columns [c * 32 V, ...) of both halves, a chunk of rows; a lane holds V
// columns of each, the warps take every 8th row of the chunk.  partial: one row of 2N sums
// per chunk.
// Three blocks an SM in one round: with two 79 us (4096 x 8192 bf16, dbias alone), three 66, and
// 50 with chunks for just that many.
template <class T, int V, bool SUMS>
__global__ void __launch_bounds__(kDzWarps * 32, 3)
    gated_dz_kernel(const T *dy, int64_t lddy, const T *pre, int64_t ldp, T *dz, int64_t lddz, int64_t M, int64_t N,
                    int64_t chunk, int act, float *partial) {
  __shared__ float joined[kDzWarps][32 * V + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t first = (int64_t)blockIdx.x * 32 * V, col = first + lane * V;
  const int64_t r0 = (int64_t)blockIdx.y * chunk, r1 = min(M, r0 + chunk);
  float sum[2][V];
#pragma unroll
  for (int j = 0; j < V; ++j) sum[0][j] = sum[1][j] = 0.0f;
  if (col < N) {
#pragma unroll 2
    for (int64_t r = r0 + warp; r < r1; r += kDzWarps) {
      const Vec<T, V> d = load_vec<T, V>(dy + r * lddy + col), g = load_vec<T, V>(pre + r * ldp + col),
                      u = load_vec<T, V>(pre + r * ldp + N + col);
      float z[V], value[V], slope[V], dg[V], du[V];
#pragma unroll
      for (int j = 0; j < V; ++j) z[j] = widen(g.v[j]);
      activate_both<V, sizeof(T) == 2>(act, z, value, slope);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        // rounded products, stored or not: dbias is then the same with and without dz
        dg[j] = __fmul_rn(__fmul_rn(widen(d.v[j]), widen(u.v[j])), slope[j]);
        du[j] = __fmul_rn(widen(d.v[j]), value[j]);
        if (SUMS) {
          sum[0][j] += dg[j];
          sum[1][j] += du[j];
        }
      }
      if (dz) {
        store_narrow<T, V>(dz + r * lddz + col, dg);
        store_narrow<T, V>(dz + r * lddz + N + col, du);
      }
    }
  }
  if (!SUMS) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; ++j) joined[warp][lane * V + j] = sum[which][j];
    __syncthreads();
    for (int c = threadIdx.x; c < 32 * V; c += kDzWarps * 32) {
      if (first + c < N) {
        float t = 0.0f;
#pragma unroll
        for (int w = 0; w < kDzWarps; ++w) t += joined[w][c];
        partial[((int64_t)blockIdx.y * 2 + which) * N + first + c] = t;
      }
    }
  }
}

// How the gradient's pass covers its matrices: columns of a block, and chunks of rows (the
// partial rows of dbias), which fill three blocks an SM once.
struct DzShape {
  bool vec;
  int64_t across, chunks;
};
DzShape dz_shape(const vcsr_gated_linear_grad_args *a) {
  const int64_t v = 16 / (int64_t)type_size(a->dtype);
  DzShape s;
  s.vec = a->N % v == 0 && a->lddy % v == 0 && a->ldp % v == 0 && aligned(a->dy, 16) && aligned(a->pre, 16);
  s.across = ceil_div(a->N, s.vec ? 32 * v : 32);
  s.chunks = std::max<int64_t>(1, std::min(ceil_div(a->M, 32), sm_count() * 3 / s.across));
  return s;
}

template <class T>
void launch_dz(const vcsr_gated_linear_grad_args *a, void *to, int64_t lddz, float *partial, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const T *dy = static_cast<const T *>(a->dy), *pre = static_cast<const T *>(a->pre);
  T *dz = static_cast<T *>(to);
  const DzShape s = dz_shape(a);
  const int64_t chunk = ceil_div(a->M, s.chunks);
  const dim3 grid((unsigned)s.across, (unsigned)s.chunks);
  auto run = [&](auto kernel) {
    kernel<<<grid, kDzWarps * 32, 0, st>>>(dy, a->lddy, pre, a->ldp, dz, lddz, a->M, a->N, chunk, a->act, partial);
  };
  if (s.vec)
    run(partial ? gated_dz_kernel<T, V, true> : gated_dz_kernel<T, V, false>);
  else
    run(partial ? gated_dz_kernel<T, 1, true> : gated_dz_kernel<T, 1, false>);
}

vcsr_status check_gated_sizes(int64_t M, int64_t N, int64_t K) {
  VCSR_TRY(check_sizes(M, N, K));
  if (N > 0x3fffffffll) return fail(VCSR_ERR_RANGE, "2 N above 2^31 - 1");
  return VCSR_OK;
}

// Whether the sums go through memory: all 2N of them in FP32, and those over no k.
bool in_two_steps(const vcsr_gated_linear_args *a) { return a->dtype == VCSR_F32 || a->K == 0; }

struct ForwardPlan {
  Packed x, w;
  size_t pre = 0, total = 0;
};
ForwardPlan forward_plan(const vcsr_gated_linear_args *a) {
  ForwardPlan p;
  if (a->M <= 0 || a->N <= 0 || a->K < 0) return p;
  if (a->K > 0) {
    p.x = packed(a->x, a->ldx, a->M, a->K, a->dtype);
    p.w = packed(a->w, a->ldw, 2 * a->N, a->K, a->dtype);
  }
  if (in_two_steps(a) && !a->pre) p.pre = round_up((size_t)a->M * 2 * a->N * type_size(a->out_dtype));
  p.total = p.x.bytes + p.w.bytes + p.pre;
  return p;
}

vcsr_status gated_linear(const vcsr_gated_linear_args *a, cudaStream_t st) {
  if (!a) return fail(VCSR_ERR_INVALID, "no arguments");
  VCSR_TRY(check_gated_sizes(a->M, a->N, a->K));
  const bool codes = a->dtype == VCSR_E4M3;
  if (!codes && !is_float16_or_32(a->dtype)) return fail(VCSR_ERR_UNSUPPORTED, "type %d", a->dtype);
  if (codes ? !is_float16_or_32(a->out_dtype) : a->out_dtype != a->dtype)
    return fail(VCSR_ERR_UNSUPPORTED, "output type %d for operands of type %d", a->out_dtype, a->dtype);
  if (a->act < VCSR_ACT_NONE || a->act > VCSR_ACT_SILU)
    return fail(VCSR_ERR_UNSUPPORTED, "activation %d", a->act);
  if (a->M == 0 || a->N == 0) return VCSR_OK;
  if (a->K > 0) {
    VCSR_TRY(check_matrix("x", a->x, a->ldx, a->K, a->dtype, false));
    VCSR_TRY(check_matrix("w", a->w, a->ldw, a->K, a->dtype, false));
  }
  if (codes && (!a->x_scale || !a->w_scale))
    return fail(VCSR_ERR_INVALID, "8-bit operands need x_scale and w_scale");
  if (!codes && (a->x_scale || a->w_scale))
    return fail(VCSR_ERR_INVALID, "scales are for 8-bit operands");
  VCSR_TRY(check_matrix("x_scale", a->x_scale, 1, 1, VCSR_F32, true));
  VCSR_TRY(check_matrix("w_scale", a->w_scale, 1, 1, VCSR_F32, true));
  VCSR_TRY(check_matrix("bias", a->bias, 2 * a->N, 2 * a->N, a->out_dtype, true));
  VCSR_TRY(check_matrix("y", a->y, a->ldy, a->N, a->out_dtype, false));
  VCSR_TRY(check_matrix("pre", a->pre, a->ldp, 2 * a->N, a->out_dtype, true));
  const ForwardPlan p = forward_plan(a);
  VCSR_TRY(check_workspace(a->workspace, a->workspace_bytes, p.total));
  const void *x = a->x, *w = a->w;
  if (a->K > 0) {
    Prepare before(a->workspace);
    x = before.matrix(p.x, x, a->ldx, a->M, a->K, a->dtype);
    w = before.matrix(p.w, w, a->ldw, 2 * a->N, a->K, a->dtype);
    VCSR_TRY(before.run(a->dtype, st));
  }
  if (!in_two_steps(a)) {
    RowsGemm g{};
    g.M = a->M;
    g.N = a->N;
    g.K = a->K;
    g.x = x;
    g.w = w;
    g.ldx = p.x.ld;
    g.ldw = p.w.ld;
    g.dtype = a->dtype;
    g.e = {a->x_scale, a->w_scale, a->bias, nullptr, a->y, a->pre, 0, a->ldy, a->ldp, a->act, a->out_dtype};
    return launch_gated_tc(g, st);
  }
  void *z = a->pre ? a->pre : static_cast<char *>(a->workspace) + p.x.bytes + p.w.bytes;
  const int64_t ldz = a->pre ? a->ldp : 2 * a->N;
  VCSR_TRY(launch_gemm({a->M, 2 * a->N, a->K, {x, p.x.ld, false}, {w, p.w.ld, false}, a->dtype,
                        {a->x_scale, a->w_scale, a->bias, nullptr, z, nullptr, 0, ldz, 0, VCSR_ACT_NONE, a->out_dtype}},
                       st));
  for_type(a->out_dtype, [&](auto t) { launch_combine<decltype(t)>(z, ldz, a->y, a->ldy, a->M, a->N, a->act, st); });
  VCSR_CUDA(cudaGetLastError());
  return VCSR_OK;
}

// The parts of the gradient's workspace: dz, partial sums of dbias, aligned x and w.
struct GradPlan {
  int64_t lddz = 0;
  size_t dz = 0, partial = 0, total = 0;
  Packed x, w;
};
GradPlan grad_plan(const vcsr_gated_linear_grad_args *a) {
  GradPlan p;
  p.lddz = packed_pitch(2 * a->N, a->dtype);
  if (a->dx || a->dw) p.dz = round_up((size_t)a->M * p.lddz * type_size(a->dtype));
  if (a->dbias) p.partial = round_up((size_t)dz_shape(a).chunks * 2 * a->N * sizeof(float));
  if (a->K > 0) {
    if (a->dw) p.x = packed(a->x, a->ldx, a->M, a->K, a->dtype);
    if (a->dx) p.w = packed(a->w, a->ldw, 2 * a->N, a->K, a->dtype);
  }
  p.total = p.dz + p.partial + p.x.bytes + p.w.bytes;
  return p;
}

vcsr_status gated_linear_grad(const vcsr_gated_linear_grad_args *a, cudaStream_t st) {
  if (!a) return fail(VCSR_ERR_INVALID, "no arguments");
  VCSR_TRY(check_gated_sizes(a->M, a->N, a->K));
  if (!is_float16_or_32(a->dtype)) return fail(VCSR_ERR_UNSUPPORTED, "type %d", a->dtype);
  if (a->act < VCSR_ACT_NONE || a->act > VCSR_ACT_SILU)
    return fail(VCSR_ERR_UNSUPPORTED, "activation %d", a->act);
  const int64_t N2 = 2 * a->N;
  VCSR_TRY(check_matrix("dx", a->dx, a->lddx, a->K, a->dtype, true));
  VCSR_TRY(check_matrix("dw", a->dw, a->lddw, a->K, a->dtype, true));
  VCSR_TRY(check_matrix("dbias", a->dbias, N2, N2, a->dtype, true));
  if (a->M == 0 || a->N == 0) {
    if (a->dx) VCSR_TRY(zero_matrix(a->dx, a->lddx, a->M, a->K, a->dtype, st));
    if (a->dw) VCSR_TRY(zero_matrix(a->dw, a->lddw, N2, a->K, a->dtype, st));
    if (a->dbias) VCSR_TRY(zero_matrix(a->dbias, N2, 1, N2, a->dtype, st));
    return VCSR_OK;
  }
  VCSR_TRY(check_matrix("dy", a->dy, a->lddy, a->N, a->dtype, false));
  VCSR_TRY(check_matrix("pre", a->pre, a->ldp, N2, a->dtype, false));
  if (a->K > 0 && a->dx) VCSR_TRY(check_matrix("w", a->w, a->ldw, a->K, a->dtype, false));
  if (a->K > 0 && a->dw) VCSR_TRY(check_matrix("x", a->x, a->ldx, a->K, a->dtype, false));
  if (!a->dx && !a->dw && !a->dbias) return VCSR_OK;
  const GradPlan p = grad_plan(a);
  VCSR_TRY(check_workspace(a->workspace, a->workspace_bytes, p.total));
  char *ws = static_cast<char *>(a->workspace);
  void *dz = p.dz ? ws : nullptr;
  float *partial = p.partial ? reinterpret_cast<float *>(ws + p.dz) : nullptr;
  for_type(a->dtype, [&](auto t) { launch_dz<decltype(t)>(a, dz, p.lddz, partial, st); });
  VCSR_CUDA(cudaGetLastError());
  Prepare before(ws + p.dz + p.partial);
  if (a->dbias) before.column_sums(partial, (int)dz_shape(a).chunks, N2, a->dbias);
  const void *x = before.matrix(p.x, a->x, a->ldx, a->M, a->K, a->dtype);
  const void *w = before.matrix(p.w, a->w, a->ldw, N2, a->K, a->dtype);
  VCSR_TRY(before.run(a->dtype, st));
  if (a->K == 0 || (!a->dx && !a->dw)) return VCSR_OK;
  Epilogue e{};
  e.type = a->dtype;
  e.out = a->dx;
  e.ldo = a->lddx;
  const Gemm dx{a->M, a->K, N2, {dz, p.lddz, false}, {w, p.w.ld, true}, a->dtype, e};
  e.out = a->dw;
  e.ldo = a->lddw;
  const Gemm dw{N2, a->K, a->M, {dz, p.lddz, true}, {x, p.x.ld, true}, a->dtype, e};
  if (a->dtype != VCSR_F32) return launch_gemms_tc(dx, dw, st);
  if (a->dx) VCSR_TRY(launch_gemm(dx, st));
  if (a->dw) VCSR_TRY(launch_gemm(dw, st));
  return VCSR_OK;
}

}  // namespace
}  // namespace layer
}  // namespace vcsr

extern "C" {

vcsr_status vcsr_gated_linear(const vcsr_gated_linear_args *a, vcsr_stream_t stream) {
  vcsr::clear_error();
  return vcsr::no_throw([&] { return vcsr::layer::gated_linear(a, (cudaStream_t)stream); });
}

size_t vcsr_gated_linear_workspace(const vcsr_gated_linear_args *a) {
  return a ? vcsr::layer::forward_plan(a).total : 0;
}

vcsr_status vcsr_gated_linear_grad(const vcsr_gated_linear_grad_args *a, vcsr_stream_t stream) {
  vcsr::clear_error();
  return vcsr::no_throw([&] { return vcsr::layer::gated_linear_grad(a, (cudaStream_t)stream); });
}

size_t vcsr_gated_linear_grad_workspace(const vcsr_gated_linear_grad_args *a) {
  if (!a || a->M <= 0 || a->N <= 0 || a->K < 0) return 0;
  return vcsr::layer::grad_plan(a).total;
}

}  // extern "C"
