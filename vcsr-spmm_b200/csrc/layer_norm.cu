// layer_norm.cu — root-mean-square norm with the residual's addition, 32-,
// 16- or 8-bit output, its gradient, and the values of 8-bit codes.
//
// Forward, per row: s = x + residual, rstd = 1/sqrt(mean(s^2) + eps),
// y = s rstd weight.  Bound by HBM (x, residual in; s, y out; about 6 FLOP per
// value), so a row is read once: a team of threads holds it in registers, 8 to
// 32 values each, between the sum of squares and the store.  Teams of up to
// 32 threads share warps (shuffles only); larger teams are one block each and
// join their warps' sums through shared memory.  Rows past 32,768 values
// do not fit a block's registers and are walked by one block in passes.
//
// Gradient, per row: with h = s rstd, g = dy weight,
// dx = rstd (g - h mean(g h)) + dsum, dweight = sum over rows of dy h.  Bound
// by HBM as well.  Teams take every (team count)-th row and keep their
// columns' dweight sums in registers over all of them; teams of a block join
// theirs in shared memory, blocks write one partial row each, and a second
// kernel adds the partial rows in block order (no atomics: the same result on
// every run).
#include <algorithm>
#include <type_traits>

#include "layer_common.cuh"

namespace vcsr {
namespace layer {

vcsr_status check_matrix(const char *name, const void *p, int64_t ld, int64_t dim, int type,
                         bool optional) {
  if (!p) return optional ? VCSR_OK : fail(VCSR_ERR_INVALID, "%s is NULL", name);
  if (ld < dim) return fail(VCSR_ERR_INVALID, "pitch of %s (%lld) below its row length %lld", name,
                            (long long)ld, (long long)dim);
  if (!aligned(p, type_size(type))) return fail(VCSR_ERR_INVALID, "%s is not aligned to its type", name);
  return VCSR_OK;
}

namespace {

// out[c] = sum of `count` partial rows, in order within each of 8 slices of
// them, the slices then added in order.  A block takes 32 columns.
__global__ void __launch_bounds__(256)
    column_sum_kernel(const float *partial, int count, int64_t dim, void *out, int dtype) {
  __shared__ float part[8][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
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

}  // namespace

vcsr_status column_sum(const float *partial, int count, int64_t dim, void *out, int dtype,
                       cudaStream_t st) {
  column_sum_kernel<<<(unsigned)ceil_div(dim, 32), 256, 0, st>>>(partial, count, dim, out, dtype);
  VCSR_CUDA(cudaGetLastError());
  return VCSR_OK;
}

namespace {

constexpr int kMaxThreads = 1024;
// The most values a thread holds, in V-value vectors, and the largest block
// that leaves it registers for them without spills (the gradient holds three
// arrays of them).  Single values need an address each and stop at 16.
template <int V>
constexpr int kMostHeld = V == 1 ? 16 : 32;
template <int V, int E>
constexpr int kNormBlock = E == kMostHeld<V> ? 1024 : 512;
constexpr int kGradBlock = 512;

struct NormArgs {
  int64_t rows, dim;
  const void *x, *residual, *weight;
  void *y, *sum;
  float *rstd, *scale;
  int64_t ldx, ldr, ldy, lds;
  float eps;
  int w_dtype, y_dtype;
};

// Sum or maximum over a team's threads; every thread gets it.  Teams of up to
// 32 threads are a power of two of neighbouring lanes.
template <bool MAX>
__device__ __forceinline__ float team_reduce(float v, int team, float *shared) {
  for (int o = min(team, 32) >> 1; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? fmaxf(v, w) : v + w;
  }
  if (team > 32) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = team >> 5;
    if (lane == 0) shared[warp] = v;
    __syncthreads();
    float t = lane < warps ? shared[lane] : 0.0f;
    for (int o = 16; o > 0; o >>= 1) {
      const float w = __shfl_xor_sync(0xffffffffu, t, o);
      t = MAX ? fmaxf(t, w) : t + w;
    }
    v = t;
  }
  return v;
}

// One row per team; E values per thread, V at a time (V values from one
// 16-byte access of x, or single values where a pitch, a base or dim is not
// aligned).
template <class T, int V, int E>
__global__ void __launch_bounds__(kNormBlock<V, E>) rmsnorm_kernel(const NormArgs a, int team) {
  const int dim = (int)a.dim;
  __shared__ float shared[2][32];
  const int t = threadIdx.x % team;
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / team) + threadIdx.x / team;
  const bool live = row < a.rows;
  constexpr int kN = E / V;
  float s[E];
  float ss = 0.0f;
  const T *x = static_cast<const T *>(a.x) + row * a.ldx;
  const T *r = static_cast<const T *>(a.residual) + row * a.ldr;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const int at = (t + i * team) * V;
    if (live && at < dim) {
      const Vec<T, V> xv = load_vec<T, V>(x + at);
#pragma unroll
      for (int j = 0; j < V; ++j) s[i * V + j] = widen(xv.v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) s[i * V + j] = 0.0f;
    }
  }
  if (a.residual) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int at = (t + i * team) * V;
      if (live && at < dim) {
        const Vec<T, V> rv = load_vec<T, V>(r + at);
#pragma unroll
        for (int j = 0; j < V; ++j) s[i * V + j] += widen(rv.v[j]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) ss = fmaf(s[e], s[e], ss);
  if (a.sum) {
    T *so = static_cast<T *>(a.sum) + row * a.lds;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int at = (t + i * team) * V;
      if (live && at < dim) store_narrow<T, V>(so + at, s + i * V);
    }
  }
  ss = team_reduce<false>(ss, team, shared[0]);
  const float rstd = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
  if (a.rstd && live && t == 0) a.rstd[row] = rstd;
  float top = 0.0f;
  auto weigh = [&](auto type) {
    using W = decltype(type);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int at = (t + i * team) * V;
      if (at < dim) {
        const Vec<W, V> w = load_vec<W, V>(static_cast<const W *>(a.weight) + at);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          s[i * V + j] *= rstd * widen(w.v[j]);
          top = fmaxf(top, fabsf(s[i * V + j]));
        }
      }
    }
  };
  if (a.w_dtype == VCSR_F32)
    weigh(float{});
  else
    weigh(T{});
  if (a.y_dtype == VCSR_E4M3) {
    const CodeScale c = code_scale(team_reduce<true>(top, team, shared[1]));
    if (live && t == 0) a.scale[row] = c.scale;
    uint8_t *y = static_cast<uint8_t *>(a.y) + row * a.ldy;
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] = c.quotient(s[e]);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int at = (t + i * team) * V;
      if (live && at < dim) store_codes<V>(y + at, s + i * V);
    }
  } else {
    with_type(a.y_dtype, [&](auto type) {
      using Y = decltype(type);
      Y *y = static_cast<Y *>(a.y) + row * a.ldy;
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int at = (t + i * team) * V;
        if (live && at < dim) store_narrow<Y, V>(y + at, s + i * V);
      }
    });
  }
}

// Rows of any length, one block each, in passes over the row: the sum of
// squares; the largest |y| (8-bit output); the stores.  s is stored in the
// last pass, so that it may replace x or residual.
template <class T>
__global__ void __launch_bounds__(kMaxThreads) rmsnorm_long_kernel(const NormArgs a) {
  __shared__ float shared[2][32];
  const int64_t row = blockIdx.x;
  const T *x = static_cast<const T *>(a.x) + row * a.ldx;
  const T *r = static_cast<const T *>(a.residual) + row * a.ldr;
  auto value = [&](int64_t i) {
    const float v = widen(x[i]);
    return a.residual ? v + widen(r[i]) : v;
  };
  float ss = 0.0f;
  for (int64_t i = threadIdx.x; i < a.dim; i += blockDim.x) {
    const float s = value(i);
    ss = fmaf(s, s, ss);
  }
  ss = team_reduce<false>(ss, blockDim.x, shared[0]);
  const float rstd = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
  if (a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
  CodeScale c = code_scale(448.0f);
  if (a.y_dtype == VCSR_E4M3) {
    float top = 0.0f;
    for (int64_t i = threadIdx.x; i < a.dim; i += blockDim.x) {
      float w;
      load_as_float<1>(a.weight, a.w_dtype, i, &w);
      top = fmaxf(top, fabsf(value(i) * (rstd * w)));
    }
    c = code_scale(team_reduce<true>(top, blockDim.x, shared[1]));
    if (threadIdx.x == 0) a.scale[row] = c.scale;
  }
  for (int64_t i = threadIdx.x; i < a.dim; i += blockDim.x) {
    const float s = value(i);
    float w;
    load_as_float<1>(a.weight, a.w_dtype, i, &w);
    const float y = a.y_dtype == VCSR_E4M3 ? c.quotient(s * (rstd * w)) : s * (rstd * w);
    if (a.sum) static_cast<T *>(a.sum)[row * a.lds + i] = narrow<T>(s);
    store_as<1>(a.y, a.y_dtype, row * a.ldy + i, &y);
  }
}

struct GradArgs {
  int64_t rows, dim;
  const void *dy, *s, *weight, *dsum;
  const float *rstd;
  void *dx;
  float *partial;  // blocks x dim; NULL = no dweight
  int64_t lddy, lds, ldds, lddx;
  int w_dtype, dy_dtype;
};

template <class T, int V, int E>
__global__ void __launch_bounds__(kGradBlock) rmsnorm_grad_kernel(const GradArgs a, int team) {
  __shared__ float shared[2][32];
  extern __shared__ float joined[];  // (teams of the block) x dim
  constexpr int kN = E / V;
  const int dim = (int)a.dim;
  const int t = threadIdx.x % team, teams = blockDim.x / team, mine = threadIdx.x / team;
  float dw[E];
#pragma unroll
  for (int e = 0; e < E; ++e) dw[e] = 0.0f;
  int flip = 0;  // two sets of shared words: one barrier per row is enough
  for (int64_t first = (int64_t)blockIdx.x * teams; first < a.rows;
       first += (int64_t)gridDim.x * teams, flip ^= 1) {
    const int64_t row = first + mine;
    const bool live = row < a.rows;
    const float rstd = live ? a.rstd[row] : 0.0f;
    const T *s = static_cast<const T *>(a.s) + row * a.lds;
    float h[E], g[E];
    float dot = 0.0f;
    with_type(a.dy_dtype, [&](auto type) {
      using D = decltype(type);
      const D *dy = static_cast<const D *>(a.dy) + row * a.lddy;
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int at = (t + i * team) * V;
        if (live && at < dim) {
          const Vec<T, V> sv = load_vec<T, V>(s + at);
          const Vec<D, V> dv = load_vec<D, V>(dy + at);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            h[i * V + j] = widen(sv.v[j]);
            g[i * V + j] = widen(dv.v[j]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) h[i * V + j] = g[i * V + j] = 0.0f;
        }
      }
    });
    auto weigh = [&](auto type) {
      using W = decltype(type);
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int at = (t + i * team) * V;
        if (at < dim) {
          const Vec<W, V> w = load_vec<W, V>(static_cast<const W *>(a.weight) + at);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int e = i * V + j;
            h[e] *= rstd;
            dw[e] = fmaf(g[e], h[e], dw[e]);
            g[e] *= widen(w.v[j]);
            dot = fmaf(g[e], h[e], dot);
          }
        }
      }
    };
    if (a.w_dtype == VCSR_F32)
      weigh(float{});
    else
      weigh(T{});
    const float mean = team_reduce<false>(dot, team, shared[flip]) / (float)a.dim;
    const T *ds = static_cast<const T *>(a.dsum) + row * a.ldds;
    T *dx = static_cast<T *>(a.dx) + row * a.lddx;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int at = (t + i * team) * V;
      if (live && at < dim) {
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = rstd * (g[i * V + j] - h[i * V + j] * mean);
        if (a.dsum) {
          const Vec<T, V> dv = load_vec<T, V>(ds + at);
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] += widen(dv.v[j]);
        }
        store_narrow<T, V>(dx + at, o);
      }
    }
  }
  if (!a.partial) return;
  float *out = a.partial + (int64_t)blockIdx.x * a.dim;
  if (teams == 1) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int at = (t + i * team) * V;
      if (at < dim) {
#pragma unroll
        for (int j = 0; j < V; ++j) out[at + j] = dw[i * V + j];
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const int at = (t + i * team) * V;
    if (at < dim) {
#pragma unroll
      for (int j = 0; j < V; ++j) joined[mine * a.dim + at + j] = dw[i * V + j];
    }
  }
  __syncthreads();
  for (int64_t c = threadIdx.x; c < a.dim; c += blockDim.x) {
    float sum = 0.0f;
    for (int k = 0; k < teams; ++k) sum += joined[k * a.dim + c];
    out[c] = sum;
  }
}

// dx of rows of any length, one block each; their dweight comes from
// rmsnorm_long_dweight_kernel.
template <class T>
__global__ void __launch_bounds__(kMaxThreads) rmsnorm_long_grad_kernel(const GradArgs a) {
  __shared__ float shared[32];
  const int64_t row = blockIdx.x;
  const float rstd = a.rstd[row];
  const T *s = static_cast<const T *>(a.s) + row * a.lds;
  float dot = 0.0f;
  for (int64_t i = threadIdx.x; i < a.dim; i += blockDim.x) {
    float g, w;
    load_as_float<1>(a.dy, a.dy_dtype, row * a.lddy + i, &g);
    load_as_float<1>(a.weight, a.w_dtype, i, &w);
    dot = fmaf(g * w, widen(s[i]) * rstd, dot);
  }
  const float mean = team_reduce<false>(dot, blockDim.x, shared) / (float)a.dim;
  for (int64_t i = threadIdx.x; i < a.dim; i += blockDim.x) {
    float g, w;
    load_as_float<1>(a.dy, a.dy_dtype, row * a.lddy + i, &g);
    load_as_float<1>(a.weight, a.w_dtype, i, &w);
    float o = rstd * (g * w - widen(s[i]) * rstd * mean);
    if (a.dsum) o += widen(static_cast<const T *>(a.dsum)[row * a.ldds + i]);
    static_cast<T *>(a.dx)[row * a.lddx + i] = narrow<T>(o);
  }
}

// Partial dweight rows for rows of any length: block (c, p) sums every
// gridDim.y-th row of 256 columns.
template <class T>
__global__ void __launch_bounds__(256) rmsnorm_long_dweight_kernel(const GradArgs a) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= a.dim) return;
  float sum = 0.0f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    float g;
    load_as_float<1>(a.dy, a.dy_dtype, row * a.lddy + c, &g);
    sum = fmaf(g, widen(static_cast<const T *>(a.s)[row * a.lds + c]) * a.rstd[row], sum);
  }
  a.partial[(int64_t)blockIdx.y * a.dim + c] = sum;
}

template <int V>
__global__ void __launch_bounds__(256)
    dequantize_kernel(const uint8_t *codes, int64_t ldc, const float *scale, int64_t rows,
                      int64_t dim, void *out, int64_t ldo, int dtype, int squared) {
  const int64_t per_row = (dim + V - 1) / V, total = rows * per_row;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / per_row, at = (i - row * per_row) * V;
    const Vec<uint8_t, V> c = load_vec<uint8_t, V>(codes + row * ldc + at);
    const float k = scale[row];
    float o[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      o[j] = e4m3_value(c.v[j]) * k;
      if (squared) o[j] *= o[j];
    }
    store_as<V>(out, dtype, row * ldo + at, o);
  }
}

// ------------------------------------------------------------------ host

// Values per access for rows of `dim` values: 16 bytes of the widest type
// where every pitch and base allows it, else one value.
bool vector_rows(int64_t dim, int v, const void *p, int64_t ld, int type) {
  return !p || (dim % v == 0 && ld % v == 0 && aligned(p, std::min<size_t>(16, v * type_size(type))));
}

struct Shape {
  int held, team, threads;  // values per thread, threads per row, threads per block
  bool fits;
};

// Teams: enough threads to hold the row at 16 values each (32 to 64 bytes of
// loads in flight a thread and tensor), 8 where there are too few rows to
// fill the GPU otherwise, 32 where the row is too long.
template <int V>
Shape shape_for(int64_t rows, int64_t dim, bool grad) {
  Shape s;
  auto most = [&](int held) {
    return (int64_t)held * (grad ? kGradBlock : held == kMostHeld<V> ? 1024 : 512);
  };
  s.held = rows * dim < (int64_t)sm_count() * 2048 * 8 ? 8 : 16;
  while (s.held < kMostHeld<V> && dim > most(s.held)) s.held *= 2;
  s.fits = dim <= most(s.held);
  int64_t team = ceil_div(ceil_div(dim, V), s.held / V);
  if (team <= 32) {
    int p = 1;
    while (p < team) p *= 2;
    team = p;
  } else {
    team = ceil_div(team, 32) * 32;
  }
  s.team = (int)std::min<int64_t>(team, kMaxThreads);
  s.threads = s.team > 32 ? s.team : 128;
  return s;
}

template <class T, int V>
void launch_norm(const NormArgs &a, cudaStream_t st) {
  const Shape s = shape_for<V>(a.rows, a.dim, false);
  if (!s.fits) {
    rmsnorm_long_kernel<T><<<(unsigned)a.rows, kMaxThreads, 0, st>>>(a);
    return;
  }
  const unsigned grid = (unsigned)ceil_div(a.rows, s.threads / s.team);
  if (s.held == 8)
    rmsnorm_kernel<T, V, 8><<<grid, s.threads, 0, st>>>(a, s.team);
  else if (s.held == 16)
    rmsnorm_kernel<T, V, 16><<<grid, s.threads, 0, st>>>(a, s.team);
  else
    rmsnorm_kernel<T, V, kMostHeld<V>><<<grid, s.threads, 0, st>>>(a, s.team);
}

// Blocks of the gradient kernel, which are also the partial rows of dweight.
int grad_blocks(int64_t rows) { return (int)std::min<int64_t>(rows, (int64_t)sm_count() * 4); }

template <class T, int V>
void launch_grad(const GradArgs &a, int blocks, cudaStream_t st) {
  const Shape s = shape_for<V>(a.rows, a.dim, true);
  if (!s.fits) {
    rmsnorm_long_grad_kernel<T><<<(unsigned)a.rows, kMaxThreads, 0, st>>>(a);
    if (a.partial)
      rmsnorm_long_dweight_kernel<T>
          <<<dim3((unsigned)ceil_div(a.dim, 256), (unsigned)blocks), 256, 0, st>>>(a);
    return;
  }
  const int teams = s.threads / s.team;
  const size_t smem = teams > 1 && a.partial ? (size_t)teams * a.dim * sizeof(float) : 0;
  if (s.held == 8)
    rmsnorm_grad_kernel<T, V, 8><<<blocks, s.threads, smem, st>>>(a, s.team);
  else if (s.held == 16)
    rmsnorm_grad_kernel<T, V, 16><<<blocks, s.threads, smem, st>>>(a, s.team);
  else
    rmsnorm_grad_kernel<T, V, kMostHeld<V>><<<blocks, s.threads, smem, st>>>(a, s.team);
}

template <class F>
void by_type(int type, bool vec, F &&f) {
  if (type == VCSR_F32)
    vec ? f(float{}, std::integral_constant<int, 4>{}) : f(float{}, std::integral_constant<int, 1>{});
  else if (type == VCSR_BF16)
    vec ? f(__nv_bfloat16{}, std::integral_constant<int, 8>{})
        : f(__nv_bfloat16{}, std::integral_constant<int, 1>{});
  else
    vec ? f(__half{}, std::integral_constant<int, 8>{}) : f(__half{}, std::integral_constant<int, 1>{});
}

vcsr_status rmsnorm(const vcsr_rmsnorm_args *a, cudaStream_t st) {
  if (!a) return fail(VCSR_ERR_INVALID, "no arguments");
  if (a->rows < 0 || a->dim < 0) return fail(VCSR_ERR_INVALID, "negative size");
  if (!is_float16_or_32(a->x_dtype)) return fail(VCSR_ERR_UNSUPPORTED, "x type %d", a->x_dtype);
  if (a->w_dtype != a->x_dtype && a->w_dtype != VCSR_F32)
    return fail(VCSR_ERR_UNSUPPORTED, "weight type %d for x type %d", a->w_dtype, a->x_dtype);
  if (!is_float16_or_32(a->y_dtype) && a->y_dtype != VCSR_E4M3)
    return fail(VCSR_ERR_UNSUPPORTED, "y type %d", a->y_dtype);
  if (!(a->eps >= 0.0f)) return fail(VCSR_ERR_INVALID, "eps must be >= 0");
  if (a->rows == 0 || a->dim == 0) return VCSR_OK;
  if (a->rows > 0x7fffffffll) return fail(VCSR_ERR_RANGE, "more than 2^31 - 1 rows");
  VCSR_TRY(check_matrix("x", a->x, a->ldx, a->dim, a->x_dtype, false));
  VCSR_TRY(check_matrix("residual", a->residual, a->ldr, a->dim, a->x_dtype, true));
  VCSR_TRY(check_matrix("weight", a->weight, a->dim, a->dim, a->w_dtype, false));
  VCSR_TRY(check_matrix("y", a->y, a->ldy, a->dim, a->y_dtype, false));
  VCSR_TRY(check_matrix("sum", a->sum, a->lds, a->dim, a->x_dtype, true));
  if (a->y_dtype == VCSR_E4M3 && !a->scale)
    return fail(VCSR_ERR_INVALID, "an 8-bit y needs scale");
  NormArgs k{a->rows, a->dim, a->x,   a->residual, a->weight, a->y,       a->sum,
             a->rstd, a->scale, a->ldx, a->ldr,      a->ldy,    a->lds,     a->eps,
             a->w_dtype, a->y_dtype};
  const int v = a->x_dtype == VCSR_F32 ? 4 : 8;
  const bool vec = vector_rows(a->dim, v, a->x, a->ldx, a->x_dtype) &&
                   vector_rows(a->dim, v, a->residual, a->ldr, a->x_dtype) &&
                   vector_rows(a->dim, v, a->weight, v, a->w_dtype) &&
                   vector_rows(a->dim, v, a->y, a->ldy, a->y_dtype) &&
                   vector_rows(a->dim, v, a->sum, a->lds, a->x_dtype);
  by_type(a->x_dtype, vec, [&](auto t, auto n) { launch_norm<decltype(t), decltype(n)::value>(k, st); });
  VCSR_CUDA(cudaGetLastError());
  return VCSR_OK;
}

vcsr_status rmsnorm_grad(const vcsr_rmsnorm_grad_args *a, cudaStream_t st) {
  if (!a) return fail(VCSR_ERR_INVALID, "no arguments");
  if (a->rows < 0 || a->dim < 0) return fail(VCSR_ERR_INVALID, "negative size");
  if (!is_float16_or_32(a->x_dtype)) return fail(VCSR_ERR_UNSUPPORTED, "x type %d", a->x_dtype);
  if (a->w_dtype != a->x_dtype && a->w_dtype != VCSR_F32)
    return fail(VCSR_ERR_UNSUPPORTED, "weight type %d for x type %d", a->w_dtype, a->x_dtype);
  if (!is_float16_or_32(a->dy_dtype)) return fail(VCSR_ERR_UNSUPPORTED, "dy type %d", a->dy_dtype);
  if (a->dim == 0) return VCSR_OK;
  if (a->rows > 0x7fffffffll) return fail(VCSR_ERR_RANGE, "more than 2^31 - 1 rows");
  if (a->dweight && !aligned(a->dweight, type_size(a->w_dtype)))
    return fail(VCSR_ERR_INVALID, "dweight is not aligned to its type");
  if (a->rows == 0) {
    if (a->dweight)
      VCSR_CUDA(cudaMemsetAsync(a->dweight, 0, (size_t)a->dim * type_size(a->w_dtype), st));
    return VCSR_OK;
  }
  VCSR_TRY(check_matrix("dy", a->dy, a->lddy, a->dim, a->dy_dtype, false));
  VCSR_TRY(check_matrix("s", a->s, a->lds, a->dim, a->x_dtype, false));
  VCSR_TRY(check_matrix("weight", a->weight, a->dim, a->dim, a->w_dtype, false));
  VCSR_TRY(check_matrix("dsum", a->dsum, a->ldds, a->dim, a->x_dtype, true));
  VCSR_TRY(check_matrix("dx", a->dx, a->lddx, a->dim, a->x_dtype, false));
  VCSR_TRY(check_matrix("rstd", a->rstd, 1, 1, VCSR_F32, false));
  const int blocks = grad_blocks(a->rows);
  if (a->dweight) {
    const size_t need = vcsr_rmsnorm_grad_workspace(a->rows, a->dim);
    if (!a->workspace || a->workspace_bytes < need || !aligned(a->workspace, 16))
      return fail(VCSR_ERR_INVALID, "dweight needs %zu bytes of 16-byte aligned workspace", need);
  }
  GradArgs k{a->rows, a->dim, a->dy, a->s, a->weight, a->dsum, a->rstd, a->dx,
             a->dweight ? static_cast<float *>(a->workspace) : nullptr,
             a->lddy, a->lds, a->ldds, a->lddx, a->w_dtype, a->dy_dtype};
  const int v = a->x_dtype == VCSR_F32 ? 4 : 8;
  const bool vec = vector_rows(a->dim, v, a->dy, a->lddy, a->dy_dtype) &&
                   vector_rows(a->dim, v, a->s, a->lds, a->x_dtype) &&
                   vector_rows(a->dim, v, a->weight, v, a->w_dtype) &&
                   vector_rows(a->dim, v, a->dsum, a->ldds, a->x_dtype) &&
                   vector_rows(a->dim, v, a->dx, a->lddx, a->x_dtype);
  by_type(a->x_dtype, vec,
          [&](auto t, auto n) { launch_grad<decltype(t), decltype(n)::value>(k, blocks, st); });
  VCSR_CUDA(cudaGetLastError());
  return a->dweight ? column_sum(k.partial, blocks, a->dim, a->dweight, a->w_dtype, st) : VCSR_OK;
}

vcsr_status dequantize(const void *codes, int64_t ldc, const float *scale, int64_t rows, int64_t dim,
                       void *out, int64_t ldo, int out_dtype, int squared, cudaStream_t st) {
  if (rows < 0 || dim < 0) return fail(VCSR_ERR_INVALID, "negative size");
  if (!is_float16_or_32(out_dtype)) return fail(VCSR_ERR_UNSUPPORTED, "out type %d", out_dtype);
  if (rows == 0 || dim == 0) return VCSR_OK;
  VCSR_TRY(check_matrix("codes", codes, ldc, dim, VCSR_E4M3, false));
  VCSR_TRY(check_matrix("scale", scale, 1, 1, VCSR_F32, false));
  VCSR_TRY(check_matrix("out", out, ldo, dim, out_dtype, false));
  const bool vec = dim % 16 == 0 && ldc % 16 == 0 && ldo % 16 == 0 && aligned(codes, 16) &&
                   aligned(out, 16);
  const int64_t total = rows * ceil_div(dim, vec ? 16 : 1);
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(total, 256), (int64_t)sm_count() * 16);
  const uint8_t *c = static_cast<const uint8_t *>(codes);
  if (vec)
    dequantize_kernel<16><<<grid, 256, 0, st>>>(c, ldc, scale, rows, dim, out, ldo, out_dtype, squared);
  else
    dequantize_kernel<1><<<grid, 256, 0, st>>>(c, ldc, scale, rows, dim, out, ldo, out_dtype, squared);
  VCSR_CUDA(cudaGetLastError());
  return VCSR_OK;
}

}  // namespace
}  // namespace layer
}  // namespace vcsr

extern "C" {

vcsr_status vcsr_rmsnorm(const vcsr_rmsnorm_args *a, vcsr_stream_t stream) {
  vcsr::clear_error();
  return vcsr::no_throw([&] { return vcsr::layer::rmsnorm(a, (cudaStream_t)stream); });
}

size_t vcsr_rmsnorm_grad_workspace(int64_t rows, int64_t dim) {
  if (rows <= 0 || dim <= 0) return 0;
  return (size_t)vcsr::layer::grad_blocks(rows) * (size_t)dim * sizeof(float);
}

vcsr_status vcsr_rmsnorm_grad(const vcsr_rmsnorm_grad_args *a, vcsr_stream_t stream) {
  vcsr::clear_error();
  return vcsr::no_throw([&] { return vcsr::layer::rmsnorm_grad(a, (cudaStream_t)stream); });
}

vcsr_status vcsr_dequantize(const void *codes, int64_t ldc, const float *scale, int64_t rows,
                            int64_t dim, void *out, int64_t ldo, int out_dtype, int squared,
                            vcsr_stream_t stream) {
  vcsr::clear_error();
  return vcsr::no_throw([&] {
    return vcsr::layer::dequantize(codes, ldc, scale, rows, dim, out, ldo, out_dtype, squared,
                                   (cudaStream_t)stream);
  });
}

}  // extern "C"
