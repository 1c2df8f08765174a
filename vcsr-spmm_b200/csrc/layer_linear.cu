// layer_linear.cu — vcsr_linear and its gradient: argument checks, the
// activation's gradient, and which product kernel runs.
//
// The gradient takes up to four launches: dz = dy act'(pre), rounded to the operands'
// type, with dbias' partial column sums of the unrounded dz in the same pass (one pass
// over dy and pre; without an activation dz is dy itself and only the sums are made);
// dbias from the partial sums, with aligned copies of operands that TMA cannot read;
// dx = dz w and dw = dz^T x, in one launch where both are small.
//
// The rounding of dz is the price of 16-bit operands: a tensor core takes no wider one
// beside them, and dz in two parts would double both products.  It is one rounding more
// than the results' own (error against exact sums 0.0023 instead of 0.0017 in bfloat16).
//
// 8192 x 4096, k = 4096 bf16 with gelu: dz 44 us (4.6 TB/s), the products 195 us each
// (1,410 TFLOP/s); 512 x 1024, k = 1024: 22 us in three launches.
#include <algorithm>

#include "layer_gemm.cuh"

namespace vcsr {
namespace layer {
namespace {

constexpr int kDzWarps = 8;

// Block (c, r): columns [c * 32 V, ...) of a chunk of rows; a lane holds V
// columns, the warps take every 8th row of the chunk.  partial: one row of N
// sums per chunk.
template <class T, int V>
__global__ void __launch_bounds__(kDzWarps * 32, 4)  // dz_chunks counts on four an SM
    dz_kernel(const T *dy, int64_t lddy, const T *pre, int64_t ldp, T *dz, int64_t lddz, int64_t M,
              int64_t N, int64_t chunk, int act, float *partial) {
  __shared__ float joined[kDzWarps][32 * V + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t col = ((int64_t)blockIdx.x * 32 + lane) * V;
  const int64_t r0 = (int64_t)blockIdx.y * chunk, r1 = min(M, r0 + chunk);
  float sum[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] = 0.0f;
  if (col < N) {
#pragma unroll 4
    for (int64_t r = r0 + warp; r < r1; r += kDzWarps) {
      const Vec<T, V> d = load_vec<T, V>(dy + r * lddy + col);
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = widen(d.v[j]);
      if (act != VCSR_ACT_NONE) {
        const Vec<T, V> z = load_vec<T, V>(pre + r * ldp + col);
        float at[V];
#pragma unroll
        for (int j = 0; j < V; ++j) at[j] = widen(z.v[j]);
        times_slopes<V, sizeof(T) == 2>(act, at, o);
        if (dz) store_narrow<T, V>(dz + r * lddz + col, o);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += o[j];
    }
  }
  if (!partial) return;
#pragma unroll
  for (int j = 0; j < V; ++j) joined[warp][lane * V + j] = sum[j];
  __syncthreads();
  for (int c = threadIdx.x; c < 32 * V; c += kDzWarps * 32) {
    const int64_t at = (int64_t)blockIdx.x * 32 * V + c;
    if (at < N) {
      float t = 0.0f;
#pragma unroll
      for (int w = 0; w < kDzWarps; ++w) t += joined[w][c];
      partial[(int64_t)blockIdx.y * N + at] = t;
    }
  }
}

int64_t dz_chunks(int64_t M, int64_t N) {
  // enough chunks of at least 32 rows for four blocks an SM
  const int64_t across = ceil_div(N, 256);
  return std::max<int64_t>(1, std::min(ceil_div(M, 32), ceil_div((int64_t)sm_count() * 4, across)));
}

template <class T>
void launch_dz(const vcsr_linear_grad_args *a, T *dz, int64_t lddz, float *partial, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const T *dy = static_cast<const T *>(a->dy), *pre = static_cast<const T *>(a->pre);
  const bool vec = a->N % V == 0 && a->lddy % V == 0 && aligned(dy, 16) &&
                   (a->act == VCSR_ACT_NONE || (a->ldp % V == 0 && aligned(pre, 16)));
  const int64_t chunks = dz_chunks(a->M, a->N), chunk = ceil_div(a->M, chunks);
  const dim3 grid((unsigned)ceil_div(a->N, vec ? 32 * V : 32), (unsigned)chunks);
  if (vec)
    dz_kernel<T, V><<<grid, kDzWarps * 32, 0, st>>>(dy, a->lddy, pre, a->ldp, dz, lddz, a->M, a->N,
                                                    chunk, a->act, partial);
  else
    dz_kernel<T, 1><<<grid, kDzWarps * 32, 0, st>>>(dy, a->lddy, pre, a->ldp, dz, lddz, a->M, a->N,
                                                    chunk, a->act, partial);
}

constexpr size_t kAlign = 256;
size_t round_up(size_t n) { return (n + kAlign - 1) / kAlign * kAlign; }

// Matrices whose base or pitch is no multiple of 16 bytes, which TMA cannot read,
// copied to ones whose pitch is.
struct PackJob {
  const void *src;
  void *dst;
  int64_t ld, ldd, rows, cols;
};
// The copies, and the column sums of dbias' partial rows, that go before the products.
struct PrepareJobs {
  PackJob job[3];
  int packs;
  const float *partial;
  int partials, dtype;
  int64_t N;
  void *dbias;
};

// Block row y copies job y, a thread 16 bytes at a time; the row after the last sums
// columns.
template <class T>
__global__ void __launch_bounds__(256) prepare_kernel(const __grid_constant__ PrepareJobs jobs) {
  if (blockIdx.y == jobs.packs) {
    __shared__ float part[8][33];
    for (int64_t group = blockIdx.x; group * 32 < jobs.N; group += gridDim.x) {
      column_sum_block(jobs.partial, jobs.partials, jobs.N, jobs.dbias, jobs.dtype, group, part);
      __syncthreads();
    }
    return;
  }
  constexpr int V = 16 / sizeof(T);
  const PackJob &p = jobs.job[blockIdx.y];
  const T *src = static_cast<const T *>(p.src);
  T *dst = static_cast<T *>(p.dst);
  const int64_t per_row = p.ldd / V, total = p.rows * per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per_row, c = (i - r * per_row) * V;
    const T *from = src + r * p.ld + c;
    Vec<T, V> v;
    if (c + V <= p.cols) {
#pragma unroll
      for (int j = 0; j < V; ++j) v.v[j] = from[j];
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v.v[j] = c + j < p.cols ? from[j] : T{};
    }
    store_vec<T, V>(dst + r * p.ldd + c, v);
  }
}

int64_t packed_pitch(int64_t cols, int dtype) {
  const int64_t v = 16 / (int64_t)type_size(dtype);
  return ceil_div(cols, v) * v;
}

// What the tensor cores read of a matrix: itself, or a copy in the workspace.
struct Packed {
  bool copy = false;
  int64_t ld = 0;
  size_t bytes = 0;
};
Packed packed(const void *p, int64_t ld, int64_t rows, int64_t cols, int dtype) {
  Packed k;
  k.ld = rows == 1 ? packed_pitch(cols, dtype) : ld;  // the pitch of one row is free
  if (!tc_aligned(p, k.ld, dtype)) {
    k.copy = true;
    k.ld = packed_pitch(cols, dtype);
    k.bytes = round_up((size_t)rows * k.ld * type_size(dtype));
  }
  return k;
}
// What goes before a call's products, made by one launch.
struct Prepare {
  PrepareJobs jobs{};
  int64_t most = 0;  // blocks of the largest job
  char *ws;
  explicit Prepare(void *workspace) : ws(static_cast<char *>(workspace)) {}
  // Where the tensor cores read matrix p: the matrix, or its copy to be.
  const void *matrix(const Packed &k, const void *p, int64_t ld, int64_t rows, int64_t cols, int dtype) {
    if (!k.copy) return p;
    jobs.job[jobs.packs++] = {p, ws, ld, k.ld, rows, cols};
    most = std::max(most, ceil_div(rows * k.ld * (int64_t)type_size(dtype) / 16, 256));
    p = ws;
    ws += k.bytes;
    return p;
  }
  void column_sums(const float *partial, int count, int64_t N, void *out) {
    jobs.partial = partial;
    jobs.partials = count;
    jobs.N = N;
    jobs.dbias = out;
    most = std::max(most, ceil_div(N, 32));
  }
  vcsr_status run(int dtype, cudaStream_t st) {
    const int rows = jobs.packs + (jobs.dbias ? 1 : 0);
    if (rows == 0) return VCSR_OK;
    jobs.dtype = dtype;
    const dim3 grid((unsigned)std::min<int64_t>(most, (int64_t)sm_count() * 8), (unsigned)rows);
    if (dtype == VCSR_E4M3)
      prepare_kernel<uint8_t><<<grid, 256, 0, st>>>(jobs);
    else if (dtype == VCSR_F32)
      prepare_kernel<float><<<grid, 256, 0, st>>>(jobs);
    else
      prepare_kernel<uint16_t><<<grid, 256, 0, st>>>(jobs);
    VCSR_CUDA(cudaGetLastError());
    return VCSR_OK;
  }
};

// A product over no k: act(bias) + residual.
__global__ void __launch_bounds__(256) empty_sum_kernel(const __grid_constant__ Gemm g) {
  const Epilogue &e = g.e;
  for (int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x; n < g.M * g.N; n += (int64_t)gridDim.x * 256) {
    const int64_t i = n / g.N, j = n - i * g.N;
    float z = 0.0f, t = 0.0f;
    if (e.bias) load_as_float<1>(e.bias, e.type, j, &z);
    if (e.pre) store_as<1>(e.pre, e.type, i * e.ldp + j, &z);
    z = activate<false>(e.act, z);
    if (e.residual) load_as_float<1>(e.residual, e.type, i * e.ldr + j, &t);
    z += t;
    store_as<1>(e.out, e.type, i * e.ldo + j, &z);
  }
}

vcsr_status launch_gemm(const Gemm &g, cudaStream_t st) {
  if (g.K == 0) {
    const int64_t blocks = std::min<int64_t>(ceil_div(g.M * g.N, 256), (int64_t)sm_count() * 16);
    empty_sum_kernel<<<(unsigned)blocks, 256, 0, st>>>(g);
    VCSR_CUDA(cudaGetLastError());
    return VCSR_OK;
  }
  return g.dtype == VCSR_F32 ? launch_gemm_f32(g, st) : launch_gemm_tc(g, st);
}

vcsr_status check_workspace(const void *ws, size_t bytes, size_t need) {
  if (need > 0 && (!ws || bytes < need || !aligned(ws, kAlign)))
    return fail(VCSR_ERR_INVALID, "the call needs %zu bytes of 256-byte aligned workspace", need);
  return VCSR_OK;
}

vcsr_status check_sizes(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 0) return fail(VCSR_ERR_INVALID, "negative size");
  if (M > 0x7fffffffll || N > 0x7fffffffll || K > 0x7fffffffll)
    return fail(VCSR_ERR_RANGE, "a size above 2^31 - 1");
  return VCSR_OK;
}

size_t linear_workspace(const vcsr_linear_args *a) {
  if (a->M <= 0 || a->N <= 0 || a->K <= 0) return 0;
  return packed(a->x, a->ldx, a->M, a->K, a->dtype).bytes + packed(a->w, a->ldw, a->N, a->K, a->dtype).bytes;
}

vcsr_status linear(const vcsr_linear_args *a, cudaStream_t st) {
  if (!a) return fail(VCSR_ERR_INVALID, "no arguments");
  VCSR_TRY(check_sizes(a->M, a->N, a->K));
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
  VCSR_TRY(check_matrix("bias", a->bias, a->N, a->N, a->out_dtype, true));
  VCSR_TRY(check_matrix("residual", a->residual, a->ldr, a->N, a->out_dtype, true));
  VCSR_TRY(check_matrix("y", a->y, a->ldy, a->N, a->out_dtype, false));
  VCSR_TRY(check_matrix("pre", a->pre, a->ldp, a->N, a->out_dtype, true));
  const Packed px = packed(a->x, a->ldx, a->M, a->K, a->dtype), pw = packed(a->w, a->ldw, a->N, a->K, a->dtype);
  VCSR_TRY(check_workspace(a->workspace, a->workspace_bytes, linear_workspace(a)));
  const void *x = a->x, *w = a->w;
  if (a->K > 0) {
    Prepare before(a->workspace);
    x = before.matrix(px, x, a->ldx, a->M, a->K, a->dtype);
    w = before.matrix(pw, w, a->ldw, a->N, a->K, a->dtype);
    VCSR_TRY(before.run(a->dtype, st));
  }
  return launch_gemm({a->M, a->N, a->K, {x, px.ld, false}, {w, pw.ld, false}, a->dtype,
                      {a->x_scale, a->w_scale, a->bias, a->residual, a->y, a->pre, a->ldr, a->ldy,
                       a->ldp, a->act, a->out_dtype}}, st);
}

// The parts of the gradient's workspace: dz (or an aligned dy), partial sums
// of dbias, aligned x and w.
struct GradPlan {
  int64_t lddz = 0;
  size_t dz = 0, partial = 0, total = 0;
  Packed dy, x, w;
};

GradPlan grad_plan(const vcsr_linear_grad_args *a) {
  GradPlan p;
  p.lddz = packed_pitch(a->N, a->dtype);
  if (a->act != VCSR_ACT_NONE && (a->dx || a->dw))
    p.dz = round_up((size_t)a->M * p.lddz * type_size(a->dtype));
  if (a->dbias) p.partial = round_up((size_t)dz_chunks(a->M, a->N) * a->N * sizeof(float));
  if (a->K > 0) {
    if (!p.dz && (a->dx || a->dw)) p.dy = packed(a->dy, a->lddy, a->M, a->N, a->dtype);
    if (a->dw) p.x = packed(a->x, a->ldx, a->M, a->K, a->dtype);
    if (a->dx) p.w = packed(a->w, a->ldw, a->N, a->K, a->dtype);
  }
  p.total = p.dz + p.partial + p.dy.bytes + p.x.bytes + p.w.bytes;
  return p;
}

vcsr_status zero_matrix(void *p, int64_t ld, int64_t rows, int64_t cols, int type, cudaStream_t st) {
  const size_t s = type_size(type);
  if (rows > 0 && cols > 0)
    VCSR_CUDA(cudaMemset2DAsync(p, (size_t)ld * s, 0, (size_t)cols * s, (size_t)rows, st));
  return VCSR_OK;
}

vcsr_status linear_grad(const vcsr_linear_grad_args *a, cudaStream_t st) {
  if (!a) return fail(VCSR_ERR_INVALID, "no arguments");
  VCSR_TRY(check_sizes(a->M, a->N, a->K));
  if (!is_float16_or_32(a->dtype)) return fail(VCSR_ERR_UNSUPPORTED, "type %d", a->dtype);
  if (a->act < VCSR_ACT_NONE || a->act > VCSR_ACT_SILU)
    return fail(VCSR_ERR_UNSUPPORTED, "activation %d", a->act);
  VCSR_TRY(check_matrix("dx", a->dx, a->lddx, a->K, a->dtype, true));
  VCSR_TRY(check_matrix("dw", a->dw, a->lddw, a->K, a->dtype, true));
  VCSR_TRY(check_matrix("dbias", a->dbias, a->N, a->N, a->dtype, true));
  if (a->M == 0 || a->N == 0) {
    if (a->dx) VCSR_TRY(zero_matrix(a->dx, a->lddx, a->M, a->K, a->dtype, st));
    if (a->dw) VCSR_TRY(zero_matrix(a->dw, a->lddw, a->N, a->K, a->dtype, st));
    if (a->dbias) VCSR_TRY(zero_matrix(a->dbias, a->N, 1, a->N, a->dtype, st));
    return VCSR_OK;
  }
  VCSR_TRY(check_matrix("dy", a->dy, a->lddy, a->N, a->dtype, false));
  VCSR_TRY(check_matrix("pre", a->pre, a->ldp, a->N, a->dtype, a->act == VCSR_ACT_NONE));
  if (a->K > 0 && a->dx) VCSR_TRY(check_matrix("w", a->w, a->ldw, a->K, a->dtype, false));
  if (a->K > 0 && a->dw) VCSR_TRY(check_matrix("x", a->x, a->ldx, a->K, a->dtype, false));
  const GradPlan p = grad_plan(a);
  VCSR_TRY(check_workspace(a->workspace, a->workspace_bytes, p.total));
  char *ws = static_cast<char *>(a->workspace);
  void *dz = p.dz ? ws : nullptr;
  float *partial = p.partial ? reinterpret_cast<float *>(ws + p.dz) : nullptr;
  if (dz || partial) {
    if (a->dtype == VCSR_F32)
      launch_dz<float>(a, static_cast<float *>(dz), p.lddz, partial, st);
    else if (a->dtype == VCSR_BF16)
      launch_dz<__nv_bfloat16>(a, static_cast<__nv_bfloat16 *>(dz), p.lddz, partial, st);
    else
      launch_dz<__half>(a, static_cast<__half *>(dz), p.lddz, partial, st);
    VCSR_CUDA(cudaGetLastError());
  }
  Prepare before(ws + p.dz + p.partial);
  if (a->dbias) before.column_sums(partial, (int)dz_chunks(a->M, a->N), a->N, a->dbias);
  const void *d = dz ? dz : before.matrix(p.dy, a->dy, a->lddy, a->M, a->N, a->dtype);
  const void *x = before.matrix(p.x, a->x, a->ldx, a->M, a->K, a->dtype);
  const void *w = before.matrix(p.w, a->w, a->ldw, a->N, a->K, a->dtype);
  VCSR_TRY(before.run(a->dtype, st));
  if (a->K == 0 || (!a->dx && !a->dw)) return VCSR_OK;
  const int64_t ldd = dz ? p.lddz : p.dy.ld;
  Epilogue e{};
  e.type = a->dtype;
  e.out = a->dx;
  e.ldo = a->lddx;
  const Gemm dx{a->M, a->K, a->N, {d, ldd, false}, {w, p.w.ld, true}, a->dtype, e};
  e.out = a->dw;
  e.ldo = a->lddw;
  const Gemm dw{a->N, a->K, a->M, {d, ldd, true}, {x, p.x.ld, true}, a->dtype, e};
  if (a->dtype != VCSR_F32) return launch_gemms_tc(dx, dw, st);
  if (a->dx) VCSR_TRY(launch_gemm(dx, st));
  if (a->dw) VCSR_TRY(launch_gemm(dw, st));
  return VCSR_OK;
}

}  // namespace
}  // namespace layer
}  // namespace vcsr

extern "C" {

vcsr_status vcsr_linear(const vcsr_linear_args *a, vcsr_stream_t stream) {
  vcsr::clear_error();
  return vcsr::no_throw([&] { return vcsr::layer::linear(a, (cudaStream_t)stream); });
}

size_t vcsr_linear_workspace(const vcsr_linear_args *a) {
  return a ? vcsr::layer::linear_workspace(a) : 0;
}

vcsr_status vcsr_linear_grad(const vcsr_linear_grad_args *a, vcsr_stream_t stream) {
  vcsr::clear_error();
  return vcsr::no_throw([&] { return vcsr::layer::linear_grad(a, (cudaStream_t)stream); });
}

size_t vcsr_linear_grad_workspace(const vcsr_linear_grad_args *a) {
  if (!a || a->M <= 0 || a->N <= 0 || a->K < 0) return 0;
  return vcsr::layer::grad_plan(a).total;
}

}  // extern "C"
