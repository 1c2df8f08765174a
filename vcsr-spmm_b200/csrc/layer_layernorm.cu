// layer_layernorm.cu — layer norm with the residual's addition, 32-, 16- or 8-bit
// output, and its gradient.
//
// Forward, per row: s = x + residual, mean = sum(s) / dim,
// rstd = 1/sqrt(sum((s - mean)^2) / dim + eps), y = (s - mean) rstd weight + bias.
// Bound by HBM (x, residual in; s, y out), so a row is read once: a team of threads holds
// it in registers through two sums, of the values and then of the squared distances from
// their mean (one sum of squares less the mean's square would cancel where the mean is
// large against the spread).  Teams, vector access and ragged rows are those of
// layer_norm.cu; rows past a block's registers are walked by one block in passes.
//
// Gradient, per row: with h = (s - mean) rstd, g = dy weight,
//   dx = rstd (g - mean(g) - h mean(g h)) + dsum,
//   dweight = sum over rows of dy h,  dbias = sum over rows of dy.
// Teams take every (team count)-th row, copy rows into shared memory ahead of their use
// and keep their columns' two sums in registers over all of them.  Both means of a row
// need a barrier; R rows are taken between two barriers.  Teams of a block join their
// sums in shared memory, blocks write one partial row of each, and a second kernel adds
// the partial rows in block order (no atomics: the same result on every run).
#include <algorithm>

#include "layer_rows.cuh"

namespace vcsr {
namespace layer {
namespace {

// The most values a thread holds, in V-value vectors; single values need an address each.
template <int V>
constexpr int kMostHeld = V == 1 ? 16 : 32;
template <int V, int E>
constexpr int kNormBlock = E == kMostHeld<V> ? 1024 : 512;

struct NormArgs {
  int64_t rows, dim;
  const void *x, *residual, *weight, *bias;
  void *y, *sum;
  float *mean, *rstd, *scale;
  int64_t ldx, ldr, ldy, lds;
  float eps;
  int x_dtype, w_dtype, y_dtype;
};

// f(W{}) for the type of weight and bias, T or float.
template <class T, class F>
__device__ __forceinline__ void with_weight_type(int w_dtype, F &&f) {
  if (w_dtype == VCSR_F32)
    f(float{});
  else
    f(T{});
}

// One row per team; E values per thread, V at a time.
template <class T, int V, int E, bool RAGGED>
__global__ void __launch_bounds__(kNormBlock<V, E>)
    layernorm_kernel(const __grid_constant__ NormArgs a, int team) {
  __shared__ float2 shared[3][32];
  const int dim = (int)a.dim;
  const int t = threadIdx.x;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = row < a.rows;
  const int shift = RAGGED ? (int)(row * a.ldx & (V - 1)) : 0;
  constexpr int kN = E / V;
  float s[E];
  const T *x = static_cast<const T *>(a.x) + row * a.ldx;
  const T *r = static_cast<const T *>(a.residual) + row * a.ldr;
  // what lies past a row is the next rows', as far as there are some
  auto whole = [&](int at) { return live && at < dim && (!RAGGED || at + V <= (a.rows - row) * a.dim); };
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const int at = (t + i * team) * V - shift;
    row_load<T, V, RAGGED>(x, at, live ? dim : 0, whole(at), s + i * V);
  }
  if (a.residual) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int at = (t + i * team) * V - shift;
      float v[V];
      row_load<T, V, RAGGED>(r, at, live ? dim : 0, whole(at), v);
#pragma unroll
      for (int j = 0; j < V; ++j) s[i * V + j] += v[j];
    }
  }
  float total = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) total += s[e];
  if (a.sum) {
    T *so = static_cast<T *>(a.sum) + row * a.lds;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int at = (t + i * team) * V - shift;
      if (live && at < dim) row_store<T, V, RAGGED>(so, at, dim, s + i * V);
    }
  }
  const float mean = team_sum(total, team, shared[0], 1) / (float)a.dim;
  // s becomes the distance from the mean, zero outside the row
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const int at = (t + i * team) * V - shift;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float &v = s[i * V + j];
      v = (RAGGED ? (unsigned)(at + j) < (unsigned)dim : at < dim) ? v - mean : 0.0f;
      ss = fmaf(v, v, ss);
    }
  }
  ss = team_sum(ss, team, shared[1], 1);
  const float rstd = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
  if (live && t == 0) {
    if (a.mean) a.mean[row] = mean;
    if (a.rstd) a.rstd[row] = rstd;
  }
  // s becomes y
  with_weight_type<T>(a.w_dtype, [&](auto type) {
    using W = decltype(type);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int at = (t + i * team) * V - shift;
      if (at >= dim) continue;
      float w[V], b[V];
      if (a.weight) weight_load<W, V, RAGGED>(static_cast<const W *>(a.weight), at, dim, w);
      if (a.bias) weight_load<W, V, RAGGED>(static_cast<const W *>(a.bias), at, dim, b);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float &v = s[i * V + j];
        v *= rstd;
        if (a.weight) v *= w[j];
        if (a.bias) v += b[j];
      }
    }
  });
  if (a.y_dtype == VCSR_E4M3) {
    // outside the row s is zero still, or zero times an rstd that is not finite
    float top = 0.0f, none = 0.0f;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int at = (t + i * team) * V - shift;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (RAGGED ? (unsigned)(at + j) < (unsigned)dim : at < dim) top = max_or_nan(top, fabsf(s[i * V + j]));
    }
    team_reduce<true>(none, top, team, shared[2], 1);
    const CodeScale c = code_scale(top);
    if (live && t == 0) a.scale[row] = c.scale;
    uint8_t *y = static_cast<uint8_t *>(a.y) + row * a.ldy;
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] = c.quotient(s[e]);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int at = (t + i * team) * V - shift;
      if (live && at < dim) {
        if (!RAGGED || (at >= 0 && at + V <= dim)) {
          store_codes<V>(y + at, s + i * V);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if ((unsigned)(at + j) < (unsigned)dim) y[at + j] = e4m3_code(s[i * V + j]);
        }
      }
    }
  } else {
    with_type(a.y_dtype, [&](auto type) {
      using Y = decltype(type);
      Y *y = static_cast<Y *>(a.y) + row * a.ldy;
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int at = (t + i * team) * V - shift;
        if (live && at < dim) row_store<Y, V, RAGGED>(y, at, dim, s + i * V);
      }
    });
  }
}

// Rows of any length, one block each, in passes over the row: the mean; the distances
// from it; the largest |y| (8-bit output); the stores.  s is stored in the last pass, so
// that it may replace x or residual.
template <class T>
__global__ void __launch_bounds__(kMaxThreads) layernorm_long_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float2 shared[3][32];
  const int64_t row = blockIdx.x;
  const T *x = static_cast<const T *>(a.x) + row * a.ldx;
  const T *r = static_cast<const T *>(a.residual) + row * a.ldr;
  auto value = [&](int64_t i) {
    const float v = widen(x[i]);
    return a.residual ? v + widen(r[i]) : v;
  };
  float total = 0.0f, ss = 0.0f;
  for (int64_t i = threadIdx.x; i < a.dim; i += blockDim.x) total += value(i);
  const float mean = team_sum(total, blockDim.x, shared[0], 1) / (float)a.dim;
  for (int64_t i = threadIdx.x; i < a.dim; i += blockDim.x) {
    const float v = value(i) - mean;
    ss = fmaf(v, v, ss);
  }
  ss = team_sum(ss, blockDim.x, shared[1], 1);
  const float rstd = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
  if (threadIdx.x == 0) {
    if (a.mean) a.mean[row] = mean;
    if (a.rstd) a.rstd[row] = rstd;
  }
  auto normed = [&](int64_t i, float s) {
    float y = (s - mean) * rstd, w;
    if (a.weight) {
      load_as_float<1>(a.weight, a.w_dtype, i, &w);
      y *= w;
    }
    if (a.bias) {
      load_as_float<1>(a.bias, a.w_dtype, i, &w);
      y += w;
    }
    return y;
  };
  CodeScale c = code_scale(448.0f);
  if (a.y_dtype == VCSR_E4M3) {
    float top = 0.0f, none = 0.0f;
    for (int64_t i = threadIdx.x; i < a.dim; i += blockDim.x) top = max_or_nan(top, fabsf(normed(i, value(i))));
    team_reduce<true>(none, top, blockDim.x, shared[2], 1);
    c = code_scale(top);
    if (threadIdx.x == 0) a.scale[row] = c.scale;
  }
  for (int64_t i = threadIdx.x; i < a.dim; i += blockDim.x) {
    const float s = value(i);
    float y = normed(i, s);
    if (a.y_dtype == VCSR_E4M3) y = c.quotient(y);
    if (a.sum) static_cast<T *>(a.sum)[row * a.lds + i] = narrow<T>(s);
    store_as<1>(a.y, a.y_dtype, row * a.ldy + i, &y);
  }
}

// --------------------------------------------------------------- gradient

struct GradArgs {
  int64_t rows, dim;
  const void *dy, *s, *weight, *dsum;
  const float *mean, *rstd;
  void *dx;
  float *partial;  // blocks x 2 x dim: dweight, dbias; NULL = neither
  int64_t lddy, lds, ldds, lddx;
  int w_dtype, dy_dtype;
  int depth;  // groups of R rows in flight per team (16-byte access)
};

// N sums over a team's threads (N = 2, 4 or 8); every thread gets them.  In a warp each
// step but the last few halves what a lane still adds up: 9 shuffles for 8 values.
// words: N x 32.
template <int N>
__device__ __forceinline__ void team_sums(float (&v)[N], int team, float *words, int id) {
  constexpr unsigned kAll = 0xffffffffu;
  if (team <= 32) {
    for (int o = team >> 1; o > 0; o >>= 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(kAll, v[i], o);
    }
    return;
  }
  constexpr int kLanes = 32 / N;  // that end with the same value
  const int lane = threadIdx.x & 31, which = lane / kLanes, part = lane % kLanes, warps = team >> 5;
  int o = 16;
#pragma unroll
  for (int half = N / 2; half >= 1; half /= 2, o /= 2) {
    const bool upper = lane & o;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      if (i >= half) break;
      const float send = upper ? v[i] : v[i + half], keep = upper ? v[i + half] : v[i];
      v[i] = keep + __shfl_xor_sync(kAll, send, o);
    }
  }
  float sum = v[0];
#pragma unroll
  for (o = kLanes / 2; o > 0; o /= 2) sum += __shfl_xor_sync(kAll, sum, o);
  if (part == 0) words[which * 32 + (threadIdx.x >> 5)] = sum;
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(team) : "memory");
  sum = 0.0f;
  for (int w = part; w < warps; w += kLanes) sum += words[which * 32 + w];
#pragma unroll
  for (o = kLanes / 2; o > 0; o /= 2) sum += __shfl_xor_sync(kAll, sum, o);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = __shfl_sync(kAll, sum, i * kLanes);
}

constexpr int kGradThreads = 640;  // the most of a block
// Rows a team takes between two barriers.
template <int V, int E>
constexpr int kGradRows = E == 8 ? 2 : 1;
// What the registers are sized for.
template <int V, int E>
constexpr int kGradBound = E == 8 ? 640 : 512;

// With 16-byte access a thread copies its own vectors of R rows, and of the next
// depth - 1 times R, into shared memory ahead of their use (nobody else reads them: no
// barrier); single values are loaded as they come.
template <class T, int V, int E, bool RAGGED>
__global__ void __launch_bounds__(kGradBound<V, E>, 1)
    layernorm_grad_kernel(const __grid_constant__ GradArgs a, int team) {
  constexpr int kN = E / V, R = kGradRows<V, E>;
  __shared__ float words[2][kGradThreads / 64][2 * R * 32];
  extern __shared__ __align__(16) unsigned char dynamic[];
  const int dim = (int)a.dim;
  const int t = threadIdx.x, teams = blockDim.y, mine = threadIdx.y, linear = mine * team + t;
  const int64_t stride = (int64_t)gridDim.x * teams, first = (int64_t)blockIdx.x * teams + mine;
  // the same for all rows of a team: their distance is a multiple of V
  const int shift = RAGGED ? (int)(first * a.lds & (V - 1)) : 0;
  auto whole = [&](int64_t row, int at) {
    return row < a.rows && at < dim && (!RAGGED || at + V <= (a.rows - row) * a.dim);
  };
  // what one row takes of shared memory, and of it s, dy, dsum
  const int dy_size = a.dy_dtype == VCSR_F32 ? 4 : 2, slot = team * E;
  const int dy_at = slot * (int)sizeof(T), ds_at = dy_at + slot * dy_size,
            row_bytes = ds_at + (a.dsum ? slot * (int)sizeof(T) : 0);
  unsigned char *ring = dynamic + (size_t)mine * a.depth * R * row_bytes;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  float dw[E], db[E];
#pragma unroll
  for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.0f;

  // the row to be copied next, this thread's first vector of it
  int64_t ahead = first;
  const int64_t begin = t * V - shift;
  const char *s_next = static_cast<const char *>(a.s) + (first * a.lds + begin) * (int64_t)sizeof(T),
             *dy_next = static_cast<const char *>(a.dy) + (first * a.lddy + begin) * dy_size,
             *ds_next = static_cast<const char *>(a.dsum) + (first * a.ldds + begin) * (int64_t)sizeof(T);
  const int64_t s_hop = stride * a.lds * (int64_t)sizeof(T), dy_hop = stride * a.lddy * dy_size,
                ds_hop = stride * a.ldds * (int64_t)sizeof(T);
  auto fetch = [&](int stage) {
#pragma unroll
    for (int q = 0; q < R; ++q) {
      if (ahead < a.rows) {
        const uint32_t to = ring_at + (uint32_t)((stage * R + q) * row_bytes);
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          const int place = (t + i * team) * V, further = i * team * V;
          if (whole(ahead, place - shift)) {
            copy_async(to + place * (int)sizeof(T), s_next + further * (int)sizeof(T), V * sizeof(T));
            copy_async(to + dy_at + place * dy_size, dy_next + further * dy_size, V * dy_size);
            if (a.dsum)
              copy_async(to + ds_at + place * (int)sizeof(T), ds_next + further * (int)sizeof(T), V * sizeof(T));
          }
        }
      }
      ahead += stride;
      s_next += s_hop;
      dy_next += dy_hop;
      ds_next += ds_hop;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if constexpr (V > 1) {
    for (int k = 0; k + 1 < a.depth; ++k) fetch(k);
  }

  // the rows' means and roots, read a turn ahead of their use
  float mean_next[R], rstd_next[R];
  auto stats = [&](int64_t row) {
#pragma unroll
    for (int q = 0; q < R; ++q, row += stride) {
      mean_next[q] = row < a.rows ? a.mean[row] : 0.0f;
      rstd_next[q] = row < a.rows ? a.rstd[row] : 0.0f;
    }
  };
  stats(first);

  int stage = 0, flip = 0;  // two sets of words: one barrier per turn is enough
  // every thread of a warp takes the same number of turns (a warp may hold teams)
  const int64_t warp_first = (int64_t)blockIdx.x * teams + (linear & ~31) / team;
  for (int64_t turn = team > 32 ? first : warp_first, row = first; turn < a.rows;
       turn += R * stride, row += R * stride, flip ^= 1) {
    float mean[R], rstd[R], h[R][E], g[R][E], sums[2 * R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      mean[q] = mean_next[q];
      rstd[q] = rstd_next[q];
    }
    stats(row + R * stride);
    const unsigned char *from = ring + (size_t)stage * R * row_bytes;
    if constexpr (V > 1) {
      int next = stage + a.depth - 1;
      if (next >= a.depth) next -= a.depth;
      // the places of the turn before this one, read by this thread then
      fetch(next);
      copies_wait_oldest(a.depth);
      if (++stage == a.depth) stage = 0;
    }
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const int64_t now = row + q * stride;
      const bool live = now < a.rows;
      const T *s = static_cast<const T *>(a.s) + now * a.lds;
      with_type(a.dy_dtype, [&](auto type) {
        using D = decltype(type);
        const D *dy = static_cast<const D *>(a.dy) + now * a.lddy;
        if constexpr (V > 1) {
          const unsigned char *at_row = from + q * row_bytes;
#pragma unroll
          for (int i = 0; i < kN; ++i) {
            const int place = (t + i * team) * V, at = place - shift;
            if (whole(now, at)) {  // from shared memory, the thread's own place
              row_load<T, V, RAGGED>(reinterpret_cast<const T *>(at_row) + shift, at, dim, true, h[q] + i * V);
              row_load<D, V, RAGGED>(reinterpret_cast<const D *>(at_row + dy_at) + shift, at, dim, true, g[q] + i * V);
            } else {  // the last row's end, or nothing
              row_load<T, V, RAGGED>(s, at, live ? dim : 0, false, h[q] + i * V);
              row_load<D, V, RAGGED>(dy, at, live ? dim : 0, false, g[q] + i * V);
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const int at = t + e * team;
            const bool in = live && at < dim;
            h[q][e] = in ? widen(s[at]) : 0.0f;
            g[q][e] = in ? widen(dy[at]) : 0.0f;
          }
        }
      });
    }
#pragma unroll
    for (int q = 0; q < 2 * R; ++q) sums[q] = 0.0f;
    // outside the row g is zero and nothing is stored, whatever h is
    with_weight_type<T>(a.w_dtype, [&](auto type) {
      using W = decltype(type);
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int at = (t + i * team) * V - shift;
        if (at >= dim) continue;
        float w[V];
        if (a.weight) weight_load<W, V, RAGGED>(static_cast<const W *>(a.weight), at, dim, w);
#pragma unroll
        for (int q = 0; q < R; ++q)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int e = i * V + j;
            float &hv = h[q][e], &gv = g[q][e];
            hv = (hv - mean[q]) * rstd[q];
            dw[e] = fmaf(gv, hv, dw[e]);
            db[e] += gv;
            if (a.weight) gv *= w[j];
            sums[2 * q] += gv;
            sums[2 * q + 1] = fmaf(gv, hv, sums[2 * q + 1]);
          }
      }
    });
    team_sums<2 * R>(sums, team, words[flip][team > 32 ? mine : 0], 1 + mine);
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const int64_t now = row + q * stride;
      if (now >= a.rows) continue;
      const float shift_mean = sums[2 * q] / (float)a.dim, dot_mean = sums[2 * q + 1] / (float)a.dim;
      T *dx = static_cast<T *>(a.dx) + now * a.lddx;
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int at = (t + i * team) * V - shift;
        if (at >= dim) continue;
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j)
          o[j] = rstd[q] * fmaf(-h[q][i * V + j], dot_mean, g[q][i * V + j] - shift_mean);
        if (a.dsum) {
          float d[V];
          if (V > 1 && whole(now, at))
            row_load<T, V, RAGGED>(reinterpret_cast<const T *>(from + q * row_bytes + ds_at) + shift, at, dim, true, d);
          else
            row_load<T, V, true>(static_cast<const T *>(a.dsum) + now * a.ldds, at, dim, false, d);
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] += d[j];
        }
        row_store<T, V, RAGGED>(dx, at, dim, o);
      }
    }
  }
  if constexpr (V > 1) asm volatile("cp.async.wait_all;" ::: "memory");
  if (!a.partial) return;
  float *out = a.partial + (int64_t)blockIdx.x * 2 * a.dim;
  float *joined = reinterpret_cast<float *>(dynamic);  // teams x 2 x dim
  if (teams > 1) __syncthreads();  // every team is done with its rows in shared memory
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const int at = (t + i * team) * V - shift;
    float *to = teams == 1 ? out + at : joined + mine * 2 * dim + at;
#pragma unroll
    for (int j = 0; j < V; ++j)
      if ((unsigned)(at + j) < (unsigned)dim) {
        to[j] = dw[i * V + j];
        to[dim + j] = db[i * V + j];
      }
  }
  if (teams == 1) return;
  __syncthreads();
  for (int c = linear; c < 2 * dim; c += teams * team) {
    float sum = 0.0f;
    for (int k = 0; k < teams; ++k) sum += joined[k * 2 * dim + c];
    out[c] = sum;
  }
}

// dx of rows of any length, one block each; their sums over rows come from
// layernorm_long_sums_kernel.
template <class T>
__global__ void __launch_bounds__(kMaxThreads) layernorm_long_grad_kernel(const __grid_constant__ GradArgs a) {
  __shared__ float2 shared[2][32];
  const int64_t row = blockIdx.x;
  const float mean = a.mean[row], rstd = a.rstd[row];
  const T *s = static_cast<const T *>(a.s) + row * a.lds;
  auto weighed = [&](int64_t i) {
    float g, w;
    load_as_float<1>(a.dy, a.dy_dtype, row * a.lddy + i, &g);
    if (!a.weight) return g;
    load_as_float<1>(a.weight, a.w_dtype, i, &w);
    return g * w;
  };
  float total = 0.0f, dot = 0.0f;
  for (int64_t i = threadIdx.x; i < a.dim; i += blockDim.x) {
    const float g = weighed(i);
    total += g;
    dot = fmaf(g, (widen(s[i]) - mean) * rstd, dot);
  }
  total = team_sum(total, blockDim.x, shared[0], 1) / (float)a.dim;
  dot = team_sum(dot, blockDim.x, shared[1], 1) / (float)a.dim;
  for (int64_t i = threadIdx.x; i < a.dim; i += blockDim.x) {
    float o = rstd * fmaf(-(widen(s[i]) - mean) * rstd, dot, weighed(i) - total);
    if (a.dsum) o += widen(static_cast<const T *>(a.dsum)[row * a.ldds + i]);
    static_cast<T *>(a.dx)[row * a.lddx + i] = narrow<T>(o);
  }
}

// Partial sums for rows of any length: block (c, p) sums every gridDim.y-th row of 256
// columns.
template <class T>
__global__ void __launch_bounds__(256) layernorm_long_sums_kernel(const __grid_constant__ GradArgs a) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= a.dim) return;
  float dw = 0.0f, db = 0.0f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    float g;
    load_as_float<1>(a.dy, a.dy_dtype, row * a.lddy + c, &g);
    dw = fmaf(g, (widen(static_cast<const T *>(a.s)[row * a.lds + c]) - a.mean[row]) * a.rstd[row], dw);
    db += g;
  }
  float *out = a.partial + (int64_t)blockIdx.y * 2 * a.dim + c;
  out[0] = dw;
  out[a.dim] = db;
}

// Partial rows to their sums; a block takes 32 columns of one of the two.
__global__ void __launch_bounds__(256)
    layernorm_sums_kernel(const float *partial, int count, int64_t dim, void *dweight, void *dbias, int dtype) {
  __shared__ float part[8][33];
  void *out = blockIdx.y ? dbias : dweight;
  if (!out) return;
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  // in order within each of 8 slices of the rows, the slices then added in order
  float sum = 0.0f;
  if (c < dim) {
    const int per = (count + 7) / 8, lo = slice * per, hi = min(count, lo + per);
    const float *from = partial + blockIdx.y * dim + c;
#pragma unroll 8
    for (int p = lo; p < hi; ++p) sum += from[(int64_t)p * 2 * dim];
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

// ------------------------------------------------------------------ host

struct Shape {
  int held, team, threads;  // values per thread, threads per row, threads per block
  bool fits;
};

int team_of(int64_t vectors, int per_thread) {
  int64_t team = ceil_div(vectors, per_thread);
  if (team > 32) return (int)std::min<int64_t>(ceil_div(team, 32) * 32, kMaxThreads);
  int p = 1;
  while (p < team) p *= 2;
  return p;
}

// Enough threads to hold the row at 16 values each, 8 where there are too few rows to
// fill the GPU otherwise, 32 where the row is too long.
template <int V>
Shape norm_shape(int64_t rows, int64_t dim, bool ragged) {
  if (ragged) dim += V - 1;  // a row may start inside its first vector
  Shape s;
  auto most = [&](int held) { return (int64_t)held * (held == kMostHeld<V> ? 1024 : 512); };
  s.held = rows * dim < (int64_t)sm_count() * 2048 * 8 ? 8 : 16;
  while (s.held < kMostHeld<V> && dim > most(s.held)) s.held *= 2;
  s.fits = dim <= most(s.held);
  s.team = team_of(ceil_div(dim, V), s.held / V);
  s.threads = s.team > 32 ? s.team : 128;
  return s;
}

template <class T, int V, bool RAGGED>
void launch_norm(const NormArgs &a, cudaStream_t st) {
  const Shape s = norm_shape<V>(a.rows, a.dim, RAGGED);
  if (!s.fits) {
    layernorm_long_kernel<T><<<(unsigned)a.rows, kMaxThreads, 0, st>>>(a);
    return;
  }
  const unsigned grid = (unsigned)ceil_div(a.rows, s.threads / s.team);
  const dim3 block((unsigned)s.team, (unsigned)(s.threads / s.team));
  if (s.held == 8)
    layernorm_kernel<T, V, 8, RAGGED><<<grid, block, 0, st>>>(a, s.team);
  else if (s.held == 16)
    layernorm_kernel<T, V, 16, RAGGED><<<grid, block, 0, st>>>(a, s.team);
  else
    layernorm_kernel<T, V, kMostHeld<V>, RAGGED><<<grid, block, 0, st>>>(a, s.team);
}

// The most blocks of the gradient kernel, which are also partial rows: one an SM, and a
// multiple of 8, so that the rows of a team have one misalignment.
int grad_blocks(int64_t rows) { return (int)std::min<int64_t>(rows, std::max(8, sm_count() / 8 * 8)); }

// Shared memory of a block's rows in flight.
constexpr size_t kGradRing = 200 * 1024;

template <class T, int V, bool RAGGED>
vcsr_status launch_grad(GradArgs a, int blocks, cudaStream_t st) {
  const int64_t dim = a.dim + (RAGGED ? V - 1 : 0);
  auto run = [&](auto kernel, int held, int rows, int bound) -> vcsr_status {
    const int team = team_of(ceil_div(dim, V), held / V);
    // teams that share a block join their sums
    const int teams = std::max(1, std::min<int>(512 / team, (int)ceil_div(a.rows, blocks)));
    const int threads = (int)ceil_div(teams * team, 32) * 32, in_block = threads / team;
    if (threads > bound) return fail(VCSR_ERR_RANGE, "block of %d threads", threads);
    size_t smem = in_block > 1 && a.partial ? (size_t)in_block * 2 * a.dim * sizeof(float) : 0;
    if (V > 1) {
      const size_t group = (size_t)team * held * ((a.dsum ? 2 : 1) * sizeof(T) + type_size(a.dy_dtype)) *
                           in_block * rows;
      a.depth = (int)std::max<size_t>(1, std::min<size_t>(4, kGradRing / group));
      smem = std::max(smem, group * a.depth);
    }
    VCSR_TRY(allow_shared(reinterpret_cast<const void *>(kernel), smem));
    kernel<<<blocks, dim3((unsigned)team, (unsigned)in_block), smem, st>>>(a, team);
    return VCSR_OK;
  };
  if (dim <= 8 * kGradBound<V, 8>) return run(layernorm_grad_kernel<T, V, 8, RAGGED>, 8, kGradRows<V, 8>, kGradBound<V, 8>);
  if (dim <= 16 * 512) return run(layernorm_grad_kernel<T, V, 16, RAGGED>, 16, kGradRows<V, 16>, 512);
  if (V > 1 && dim <= 32 * 512) {
    constexpr int kHeld = kMostHeld<V>;
    return run(layernorm_grad_kernel<T, V, kHeld, RAGGED>, kHeld, kGradRows<V, kHeld>, 512);
  }
  layernorm_long_grad_kernel<T><<<(unsigned)a.rows, kMaxThreads, 0, st>>>(a);
  if (a.partial)
    layernorm_long_sums_kernel<T><<<dim3((unsigned)ceil_div(a.dim, 256), (unsigned)blocks), 256, 0, st>>>(a);
  return VCSR_OK;
}

// Weight and bias are read by vectors where the rows are, which needs them aligned.
Access with_vectors(Access how, const void *bias) { return how == kVector && !aligned(bias, 16) ? kRagged : how; }

vcsr_status layernorm(const vcsr_layernorm_args *a, cudaStream_t st) {
  if (!a) return fail(VCSR_ERR_INVALID, "no arguments");
  if (a->rows < 0 || a->dim < 0) return fail(VCSR_ERR_INVALID, "negative size");
  if (!is_float16_or_32(a->x_dtype)) return fail(VCSR_ERR_UNSUPPORTED, "x type %d", a->x_dtype);
  if (a->w_dtype != a->x_dtype && a->w_dtype != VCSR_F32)
    return fail(VCSR_ERR_UNSUPPORTED, "weight type %d for x type %d", a->w_dtype, a->x_dtype);
  if (!is_float16_or_32(a->y_dtype) && a->y_dtype != VCSR_E4M3)
    return fail(VCSR_ERR_UNSUPPORTED, "y type %d", a->y_dtype);
  if (!(a->eps >= 0.0f)) return fail(VCSR_ERR_INVALID, "eps must be >= 0");
  if (a->rows == 0) return VCSR_OK;
  if (a->dim == 0) {  // means of nothing: NaN (all bits set); a largest value of nothing: 0
    const size_t bytes = (size_t)a->rows * sizeof(float);
    if (a->mean) VCSR_CUDA(cudaMemsetAsync(a->mean, 0xff, bytes, st));
    if (a->rstd) VCSR_CUDA(cudaMemsetAsync(a->rstd, 0xff, bytes, st));
    if (a->y_dtype == VCSR_E4M3 && a->scale) VCSR_CUDA(cudaMemsetAsync(a->scale, 0, bytes, st));
    return VCSR_OK;
  }
  if (a->rows > 0x7fffffffll) return fail(VCSR_ERR_RANGE, "more than 2^31 - 1 rows");
  VCSR_TRY(check_matrix("x", a->x, a->ldx, a->dim, a->x_dtype, false));
  VCSR_TRY(check_matrix("residual", a->residual, a->ldr, a->dim, a->x_dtype, true));
  VCSR_TRY(check_matrix("weight", a->weight, a->dim, a->dim, a->w_dtype, true));
  VCSR_TRY(check_matrix("bias", a->bias, a->dim, a->dim, a->w_dtype, true));
  VCSR_TRY(check_matrix("y", a->y, a->ldy, a->dim, a->y_dtype, false));
  VCSR_TRY(check_matrix("sum", a->sum, a->lds, a->dim, a->x_dtype, true));
  if (a->y_dtype == VCSR_E4M3 && !a->scale) return fail(VCSR_ERR_INVALID, "an 8-bit y needs scale");
  VCSR_TRY(check_matrix("mean", a->mean, 1, 1, VCSR_F32, true));
  VCSR_TRY(check_matrix("rstd", a->rstd, 1, 1, VCSR_F32, true));
  VCSR_TRY(check_matrix("scale", a->scale, 1, 1, VCSR_F32, true));
  const NormArgs k{a->rows, a->dim,  a->x,     a->residual, a->weight, a->bias, a->y,   a->sum,     a->mean,    a->rstd,
                   a->scale, a->ldx, a->ldr,   a->ldy,      a->lds,    a->eps,  a->x_dtype, a->w_dtype, a->y_dtype};
  const int v = a->x_dtype == VCSR_F32 ? 4 : 8;
  const Access how = with_vectors(
      access_of(a->rows, a->dim, v, a->weight, {{a->x, a->ldx, a->x_dtype}, {a->residual, a->ldr, a->x_dtype},
                                                {a->y, a->ldy, a->y_dtype}, {a->sum, a->lds, a->x_dtype}}),
      a->bias);
  by_type(a->x_dtype, how, [&](auto t, auto n, auto ragged) {
    launch_norm<decltype(t), decltype(n)::value, decltype(ragged)::value>(k, st);
  });
  VCSR_CUDA(cudaGetLastError());
  return VCSR_OK;
}

size_t grad_workspace(int64_t rows, int64_t dim) {
  if (rows <= 0 || dim <= 0) return 0;
  return (size_t)grad_blocks(rows) * 2 * (size_t)dim * sizeof(float);
}

vcsr_status layernorm_grad(const vcsr_layernorm_grad_args *a, cudaStream_t st) {
  if (!a) return fail(VCSR_ERR_INVALID, "no arguments");
  if (a->rows < 0 || a->dim < 0) return fail(VCSR_ERR_INVALID, "negative size");
  if (!is_float16_or_32(a->x_dtype)) return fail(VCSR_ERR_UNSUPPORTED, "x type %d", a->x_dtype);
  if (a->w_dtype != a->x_dtype && a->w_dtype != VCSR_F32)
    return fail(VCSR_ERR_UNSUPPORTED, "weight type %d for x type %d", a->w_dtype, a->x_dtype);
  if (!is_float16_or_32(a->dy_dtype)) return fail(VCSR_ERR_UNSUPPORTED, "dy type %d", a->dy_dtype);
  if (a->dim == 0) return VCSR_OK;
  if (a->rows > 0x7fffffffll) return fail(VCSR_ERR_RANGE, "more than 2^31 - 1 rows");
  const size_t w_size = type_size(a->w_dtype);
  VCSR_TRY(check_matrix("dweight", a->dweight, a->dim, a->dim, a->w_dtype, true));
  VCSR_TRY(check_matrix("dbias", a->dbias, a->dim, a->dim, a->w_dtype, true));
  if (a->rows == 0) {
    if (a->dweight) VCSR_CUDA(cudaMemsetAsync(a->dweight, 0, (size_t)a->dim * w_size, st));
    if (a->dbias) VCSR_CUDA(cudaMemsetAsync(a->dbias, 0, (size_t)a->dim * w_size, st));
    return VCSR_OK;
  }
  VCSR_TRY(check_matrix("dy", a->dy, a->lddy, a->dim, a->dy_dtype, false));
  VCSR_TRY(check_matrix("s", a->s, a->lds, a->dim, a->x_dtype, false));
  VCSR_TRY(check_matrix("weight", a->weight, a->dim, a->dim, a->w_dtype, true));
  VCSR_TRY(check_matrix("dsum", a->dsum, a->ldds, a->dim, a->x_dtype, true));
  VCSR_TRY(check_matrix("dx", a->dx, a->lddx, a->dim, a->x_dtype, false));
  VCSR_TRY(check_matrix("mean", a->mean, 1, 1, VCSR_F32, false));
  VCSR_TRY(check_matrix("rstd", a->rstd, 1, 1, VCSR_F32, false));
  const bool sums = a->dweight || a->dbias;
  if (sums) {
    const size_t need = grad_workspace(a->rows, a->dim);
    if (!a->workspace || a->workspace_bytes < need || !aligned(a->workspace, 16))
      return fail(VCSR_ERR_INVALID, "dweight and dbias need %zu bytes of 16-byte aligned workspace", need);
  }
  const int blocks = grad_blocks(a->rows);
  const GradArgs k{a->rows, a->dim,  a->dy,  a->s,    a->weight, a->dsum, a->mean, a->rstd, a->dx,
                   sums ? static_cast<float *>(a->workspace) : nullptr,
                   a->lddy, a->lds,  a->ldds, a->lddx, a->w_dtype, a->dy_dtype, 0};
  const int v = a->x_dtype == VCSR_F32 ? 4 : 8;
  const Access how = access_of(a->rows, a->dim, v, a->weight, {{a->dy, a->lddy, a->dy_dtype}, {a->s, a->lds, a->x_dtype},
                                                    {a->dsum, a->ldds, a->x_dtype}, {a->dx, a->lddx, a->x_dtype}});
  vcsr_status done = VCSR_OK;
  by_type(a->x_dtype, how, [&](auto t, auto n, auto ragged) {
    done = launch_grad<decltype(t), decltype(n)::value, decltype(ragged)::value>(k, blocks, st);
  });
  VCSR_TRY(done);
  VCSR_CUDA(cudaGetLastError());
  if (sums) {
    layernorm_sums_kernel<<<dim3((unsigned)ceil_div(a->dim, 32), 2), 256, 0, st>>>(k.partial, blocks, a->dim, a->dweight,
                                                                                 a->dbias, a->w_dtype);
    VCSR_CUDA(cudaGetLastError());
  }
  return VCSR_OK;
}

}  // namespace
}  // namespace layer
}  // namespace vcsr

extern "C" {

vcsr_status vcsr_layernorm(const vcsr_layernorm_args *a, vcsr_stream_t stream) {
  vcsr::clear_error();
  return vcsr::no_throw([&] { return vcsr::layer::layernorm(a, (cudaStream_t)stream); });
}

size_t vcsr_layernorm_grad_workspace(int64_t rows, int64_t dim) { return vcsr::layer::grad_workspace(rows, dim); }

vcsr_status vcsr_layernorm_grad(const vcsr_layernorm_grad_args *a, vcsr_stream_t stream) {
  vcsr::clear_error();
  return vcsr::no_throw([&] { return vcsr::layer::layernorm_grad(a, (cudaStream_t)stream); });
}

}  // extern "C"
