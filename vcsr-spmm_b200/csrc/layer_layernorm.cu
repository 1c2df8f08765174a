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
// 16384 x 4096 bf16 with residual 92 us (5.9 TB/s), to 8 bits 100 (4.7), 62451 x 128 FP32 to
// bf16 19.7 (5.7 TB/s); for 16-bit rows the instructions come close to the bandwidth (60% of
// issue slots), so two values are worked on at a time.
//
// Gradient, per row: with h = (s - mean) rstd, g = dy weight,
//   dx = rstd (g - mean(g) - h mean(g h)) + dsum,
//   dweight = sum over rows of dy h,  dbias = sum over rows of dy.
// Teams take every (team count)-th row, copy rows into shared memory ahead of their use
// and keep their columns' two sums in registers over all of them.  Teams of a block join
// their sums in shared memory, blocks write one partial row of each, and a second kernel
// adds the partial rows in block order (no atomics: the same result on every run).
// 8191 x 5120 bf16 with dsum 77 us (4.4 TB/s), 16384 x 4096 109 (4.9), 60000 x 1000 FP32 157
// (6.1): bound by instructions (60% of issue slots) at few warps an SM, whose registers
// hold the sums: 20 at 5,120 16-bit values, 16 at 4,096 and at 8,192, 11 just past 5,120 and 9
// just past 8,192.
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
template <int V, int E, bool RAGGED>
constexpr int kNormBlocksPerSm = V == 8 && E == 16 && !RAGGED ? 3 : E <= 16 && (V == 8 || (V > 1 && RAGGED)) ? 2 : 1;

struct NormArgs {
  int64_t rows, dim;
  const void *x, *residual, *weight, *bias;
  void *y, *sum;
  float *mean, *rstd, *scale;
  int64_t ldx, ldr, ldy, lds;
  float eps;
  int w_dtype, y_dtype;
};

// f(W{}) for the type of weight and bias, T or float.
template <class T, class F>
__device__ __forceinline__ void with_weight_type(int w_dtype, F &&f) {
  if (w_dtype == VCSR_F32)
    f(float{});
  else
    f(T{});
}

// row_load that looks at single values only in a row's first and last vector.
template <class X, int V, bool RAGGED>
__device__ __forceinline__ void row_load_ends(const X *row, int at, int dim, bool whole, float *out) {
  if (RAGGED && whole && at >= 0 && at + V <= dim)
    row_load<X, V, false>(row, at, dim, true, out);
  else
    row_load<X, V, RAGGED>(row, at, dim, whole, out);
}

// One row per team; E values per thread, V at a time.
template <class T, int V, int E, bool RAGGED>
__global__ void __launch_bounds__(kNormBlock<V, E>, (kNormBlocksPerSm<V, E, RAGGED>))
    layernorm_kernel(const __grid_constant__ NormArgs a, int team) {
  __shared__ float2 shared[3][32];
  const int dim = (int)a.dim;
  const int t = threadIdx.x;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = row < a.rows;
  const int shift = RAGGED ? (int)(row * a.ldx & (V - 1)) : 0;
  constexpr int kN = E / V;
  float s[E];
  // s[e] = f(s[e], u), two values at a time where there are two
  auto pairs = [](float *x, int n, auto &&f) {
    if constexpr (V > 1) {
#pragma unroll
      for (int j = 0; j < n; j += 2) {
        const float2 y = f(make_float2(x[j], x[j + 1]), j);
        x[j] = y.x;
        x[j + 1] = y.y;
      }
    } else {
      x[0] = f(make_float2(x[0], 0.0f), 0).x;
    }
  };
  auto both = [](float v) { return make_float2(v, v); };
  const T *x = static_cast<const T *>(a.x) + row * a.ldx;
  const T *r = static_cast<const T *>(a.residual) + row * a.ldr;
  // what lies past a row is the next rows', as far as there are some
  auto whole = [&](int at) { return live && at < dim && (!RAGGED || at + V <= (a.rows - row) * a.dim); };
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const int at = (t + i * team) * V - shift;
    row_load_ends<T, V, RAGGED>(x, at, live ? dim : 0, whole(at), s + i * V);
  }
  if (a.residual) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int at = (t + i * team) * V - shift;
      float v[V + 1];
      row_load_ends<T, V, RAGGED>(r, at, live ? dim : 0, whole(at), v);
      pairs(s + i * V, V, [&](float2 u, int j) { return __fadd2_rn(u, make_float2(v[j], v[j + 1])); });
    }
  }
  float2 total = both(0.0f);
#pragma unroll
  for (int i = 0; i < kN; ++i)
    pairs(s + i * V, V, [&](float2 u, int) {
      total = __fadd2_rn(total, u);
      return u;
    });
  if (a.sum) {
    T *so = static_cast<T *>(a.sum) + row * a.lds;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int at = (t + i * team) * V - shift;
      if (live && at < dim) row_store<T, V, RAGGED>(so, at, dim, s + i * V);
    }
  }
  const float mean = team_sum(total.x + total.y, team, shared[0], 1) / (float)a.dim;
  // s becomes the distance from the mean, zero outside the row
  float2 squares = both(0.0f);
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const int at = (t + i * team) * V - shift;
    if (at < dim) {
      pairs(s + i * V, V, [&](float2 u, int) { return __fadd2_rn(u, both(-mean)); });
      if (RAGGED && (at < 0 || at + V > dim)) {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if ((unsigned)(at + j) >= (unsigned)dim) s[i * V + j] = 0.0f;
      }
      pairs(s + i * V, V, [&](float2 u, int) {
        if (V == 1) u.y = 0.0f;
        squares = __ffma2_rn(u, u, squares);
        return u;
      });
    }
  }
  const float rstd = 1.0f / sqrtf(team_sum(squares.x + squares.y, team, shared[1], 1) / (float)a.dim + a.eps);
  if (live && t == 0) {
    if (a.mean) a.mean[row] = mean;
    if (a.rstd) a.rstd[row] = rstd;
  }
  // s becomes y, a vector's weights loaded at a time
  with_weight_type<T>(a.w_dtype, [&](auto type) {
    using W = decltype(type);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int at = (t + i * team) * V - shift;
      if (at >= dim) continue;
      float w[V + 1];
      float *y = s + i * V;
      pairs(y, V, [&](float2 u, int) { return __fmul2_rn(u, both(rstd)); });
      if (a.weight) {
        weight_load<W, V, RAGGED>(static_cast<const W *>(a.weight), at, dim, w);
        pairs(y, V, [&](float2 u, int j) { return __fmul2_rn(u, make_float2(w[j], w[j + 1])); });
      }
      if (a.bias) {
        weight_load<W, V, RAGGED>(static_cast<const W *>(a.bias), at, dim, w);
        pairs(y, V, [&](float2 u, int j) { return __fadd2_rn(u, make_float2(w[j], w[j + 1])); });
      }
      if (kNormBlocksPerSm<V, E, RAGGED> > 1) asm volatile("" ::: "memory");  // the next vector's loads stay behind
    }
  });
  if (a.y_dtype == VCSR_E4M3) {
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
  int x_dtype, w_dtype, dy_dtype;
  // 16-byte access: rows in flight per team; bytes that a row takes of shared memory, and
  // where dy and dsum start in it; bytes from a row of a team to its next
  int depth, row_bytes, dy_at, ds_at;
  int64_t s_hop, dy_hop, ds_hop, dx_hop;
};

// The two sums of a row over a team's threads, in two steps with the team's barrier (for
// teams of more than a warp) between them, so that other work can stand there too.
// After the first a smaller team has its sums in v; words: 2 x 32.
__device__ __forceinline__ void team_sums_begin(float2 &v, int team, float *words) {
  constexpr unsigned kAll = 0xffffffffu;
  if (team <= 32) {
    for (int o = team >> 1; o > 0; o >>= 1) {
      v.x += __shfl_xor_sync(kAll, v.x, o);
      v.y += __shfl_xor_sync(kAll, v.y, o);
    }
    return;
  }
  const int lane = threadIdx.x & 31;
  const bool upper = lane & 16;  // the upper lanes go on with v.y
  float sum = (upper ? v.y : v.x) + __shfl_xor_sync(kAll, upper ? v.x : v.y, 16);
#pragma unroll
  for (int o = 8; o > 0; o /= 2) sum += __shfl_xor_sync(kAll, sum, o);
  if ((lane & 15) == 0) words[(lane >> 4) * 32 + (threadIdx.x >> 5)] = sum;
}
__device__ __forceinline__ void team_barrier(int team, int id) {
  if (team > 32) asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(team) : "memory");
}
__device__ __forceinline__ void team_sums_end(float2 &v, int team, const float *words) {
  if (team <= 32) return;
  constexpr unsigned kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31, part = lane & 15, warps = team >> 5;
  const float *mine = words + (lane >> 4) * 32;
  float sum = part < warps ? mine[part] : 0.0f;
  if (part + 16 < warps) sum += mine[part + 16];
#pragma unroll
  for (int o = 8; o > 0; o /= 2) sum += __shfl_xor_sync(kAll, sum, o);
  v = make_float2(__shfl_sync(kAll, sum, 0), __shfl_sync(kAll, sum, 16));
}

constexpr int kGradTeams = 512 / 64;  // of more than a warp, in a block

// This block's sums over rows to its partial row: each thread's columns of its team's
// row (first(i): of vector i), teams added in order through shared memory.
template <int V, int E, class AT>
__device__ __forceinline__ void store_partial(const GradArgs &a, const float *dw, const float *db, int team,
                                              unsigned char *dynamic, AT &&first) {
  const int dim = (int)a.dim, teams = blockDim.y, linear = threadIdx.y * team + threadIdx.x;
  float *out = a.partial + (int64_t)blockIdx.x * 2 * a.dim;
  float *joined = reinterpret_cast<float *>(dynamic);  // teams x 2 x dim
  if (teams > 1) __syncthreads();  // every team is done with its rows in shared memory
#pragma unroll
  for (int i = 0; i < E / V; ++i) {
    const int at = first(i);
    float *to = teams == 1 ? out + at : joined + threadIdx.y * 2 * dim + at;
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

// Waits until all but the latest n groups of copies have landed, n < 8.
__device__ __forceinline__ void copies_wait_but(int n) {
  switch (n) {
    case 0: return copies_wait<0>();
    case 1: return copies_wait<1>();
    case 2: return copies_wait<2>();
    case 3: return copies_wait<3>();
    case 4: return copies_wait<4>();
    case 5: return copies_wait<5>();
    case 6: return copies_wait<6>();
    default: return copies_wait<7>();
  }
}

// Vector access.  A thread copies its own vectors of the next rows into shared memory
// ahead of their use (nobody else reads them: no barrier).  A row is worked on twice, for
// its two sums and for dx, and the first half of the next row comes before the second
// half of this one: the barrier and the shuffles that join a row's sums then have a row's
// work to stand behind.  RAGGED: vectors are cut at the memory's boundaries, so a row's
// first and last may hold values of its neighbours.
template <class T, class W, int V, int E, int BOUND, bool RAGGED>
__global__ void __launch_bounds__(BOUND, 1) layernorm_grad_kernel(const __grid_constant__ GradArgs a, int team) {
  constexpr int kN = E / V;
  // kept in registers where they are enough; BOUND 640 leaves no two vectors' values either
  constexpr bool kKeepWeight = E <= 16, kOneByOne = BOUND > 512;
  __shared__ float words[3][kGradTeams][64];
  extern __shared__ __align__(16) unsigned char dynamic[];
  const int dim = (int)a.dim, t = threadIdx.x, teams = blockDim.y, mine = threadIdx.y;
  const unsigned rows = (unsigned)a.rows, block_first = blockIdx.x * teams, stride = gridDim.x * teams;
  const int64_t first = block_first + mine;
  const int turns = block_first < rows ? (int)((rows - block_first - 1) / stride) + 1 : 0;
  const float inverse_dim = 1.0f / (float)dim;
  const int dy_size = a.dy_dtype == VCSR_F32 ? 4 : 2;
  // the same for all rows of a team: their distance is a multiple of V
  const int shift = RAGGED ? (int)(first * a.lds & (V - 1)) : 0;
  // this thread's place in the first of its team's rows
  unsigned char *ring = dynamic + mine * a.depth * a.row_bytes;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  const int dy_place = a.dy_at + t * V * dy_size, ds_place = a.ds_at + t * V * (int)sizeof(T);
  auto at_of = [&](int i) { return (t + i * team) * V - shift; };
  // whether vector i may be read whole: what lies past a row is the next rows', as far as
  // there are some
  auto whole = [&](int i, unsigned row) {
    const int at = at_of(i);
    return !RAGGED || at + V <= dim || at + V <= (int64_t)(rows - row) * a.dim;
  };
  bool in[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) in[i] = at_of(i) < dim;

  // the weights of vector i, as they are stored
  auto weight_at = [&](int i) {
    const W *from = static_cast<const W *>(a.weight) + at_of(i);
    Vec<W, V> w;
#pragma unroll
    for (int j = 0; j < V; ++j) w.v[j] = narrow<W>(1.0f);
    if (a.weight && in[i]) {
      if constexpr (RAGGED) {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if ((unsigned)(at_of(i) + j) < (unsigned)dim) w.v[j] = from[j];
      } else {
        w = load_vec<W, V>(from);
      }
    }
    return w;
  };
  float2 dw[E / 2], db[E / 2];
  Vec<W, V> weight[kKeepWeight ? kN : 1];
#pragma unroll
  for (int e = 0; e < E / 2; ++e) dw[e] = db[e] = make_float2(0.0f, 0.0f);
  if constexpr (kKeepWeight) {
#pragma unroll
    for (int i = 0; i < kN; ++i) weight[i] = weight_at(i);
  }

  // the row to be copied next, and its place in the ring
  unsigned ahead = (unsigned)first;
  int ahead_stage = 0;
  const int begin = t * V - shift;
  const char *s_next = static_cast<const char *>(a.s) + (first * a.lds + begin) * (int64_t)sizeof(T),
             *dy_next = static_cast<const char *>(a.dy) + (first * a.lddy + begin) * dy_size,
             *ds_next = static_cast<const char *>(a.dsum) + (first * a.ldds + begin) * (int64_t)sizeof(T);
  auto fetch = [&] {
    if (ahead < rows) {
      const uint32_t to = ring_at + (uint32_t)(ahead_stage * a.row_bytes);
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        if (!in[i] || !whole(i, ahead)) continue;
        const int further = i * team * V;
        copy_async(to + (t * V + further) * (int)sizeof(T), s_next + further * (int)sizeof(T), V * sizeof(T));
        copy_async(to + dy_place + further * dy_size, dy_next + further * dy_size, V * dy_size);
        if (a.dsum)
          copy_async(to + ds_place + further * (int)sizeof(T), ds_next + further * (int)sizeof(T), V * sizeof(T));
      }
      ahead += stride;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    s_next += a.s_hop;
    dy_next += a.dy_hop;
    ds_next += a.ds_hop;
    if (++ahead_stage == a.depth) ahead_stage = 0;
  };
  for (int k = 0; k < a.depth; ++k) fetch();

  // what a row keeps between its halves
  struct Row {
    float2 sums;
    float mean, rstd;
    bool live;
  };
  unsigned row_now = (unsigned)first;  // whose first half is next
  float mean_next = row_now < rows ? a.mean[row_now] : 0.0f, rstd_next = row_now < rows ? a.rstd[row_now] : 0.0f;
  unsigned row_done = (unsigned)first;  // whose second half is next
  char *dx_next = static_cast<char *>(a.dx) + (first * a.lddx + begin) * (int64_t)sizeof(T);

  with_type(a.dy_dtype, [&](auto type) {
    using D = decltype(type);
    // vector i of the row in a slot as h and g, both zero outside the row
    auto read = [&](const unsigned char *from, int i, unsigned row, const Row &r, float2 *h, float2 *g) {
      const int further = i * team * V;
      Vec<T, V> s;
      Vec<D, V> dy;
      if (whole(i, row)) {
        s = load_vec<T, V>(reinterpret_cast<const T *>(from) + t * V + further);
        dy = load_vec<D, V>(reinterpret_cast<const D *>(from + dy_place) + further);
      } else {  // the end of the last rows
        const T *s_row = static_cast<const T *>(a.s) + row * a.lds + at_of(i);
        const D *dy_row = static_cast<const D *>(a.dy) + row * a.lddy + at_of(i);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const bool is = (unsigned)(at_of(i) + j) < (unsigned)dim;
          s.v[j] = is ? s_row[j] : T{};
          dy.v[j] = is ? dy_row[j] : D{};
        }
      }
      const float2 away = make_float2(-r.mean, -r.mean), by = make_float2(r.rstd, r.rstd);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        h[j] = __fmul2_rn(__fadd2_rn(make_float2(widen(s.v[2 * j]), widen(s.v[2 * j + 1])), away), by);
        g[j] = make_float2(widen(dy.v[2 * j]), widen(dy.v[2 * j + 1]));
      }
      if (RAGGED && (at_of(i) < 0 || at_of(i) + V > dim)) {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if ((unsigned)(at_of(i) + j) >= (unsigned)dim) (&h[j / 2].x)[j % 2] = (&g[j / 2].x)[j % 2] = 0.0f;
      }
    };
    auto weigh = [&](int i, float2 *g) {
      const Vec<W, V> w = kKeepWeight ? weight[kKeepWeight ? i : 0] : weight_at(i);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) g[j] = __fmul2_rn(g[j], make_float2(widen(w.v[2 * j]), widen(w.v[2 * j + 1])));
    };
    int stage = 0;  // of the row whose first half is next
    auto first_half = [&](Row &r, int k) {
      r.mean = mean_next;
      r.rstd = rstd_next;
      const unsigned row = row_now;
      r.live = row < rows;
      if (r.live) row_now += stride;
      if (row_now < rows) {
        mean_next = a.mean[row_now];
        rstd_next = a.rstd[row_now];
      }
      float2 sg = make_float2(0.0f, 0.0f), sgh = sg;
      const unsigned char *from = ring + stage * a.row_bytes;
      if (++stage == a.depth) stage = 0;
      if (r.live) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          if (kOneByOne && i > 0) asm volatile("" ::: "memory");
          if (!in[i]) continue;
          float2 h[V / 2], g[V / 2];
          read(from, i, row, r, h, g);
#pragma unroll
          for (int j = 0; j < V / 2; ++j) {
            const int e = i * (V / 2) + j;
            dw[e] = __ffma2_rn(g[j], h[j], dw[e]);
            db[e] = __fadd2_rn(db[e], g[j]);
          }
          weigh(i, g);
#pragma unroll
          for (int j = 0; j < V / 2; ++j) {
            sg = __fadd2_rn(sg, g[j]);
            sgh = __ffma2_rn(g[j], h[j], sgh);
          }
        }
      }
      __syncwarp();
      r.sums = make_float2(sg.x + sg.y, sgh.x + sgh.y);
      team_sums_begin(r.sums, team, words[k % 3][team > 32 ? mine : 0]);
    };
    int done_stage = 0;
    auto second_half = [&](Row &r, int k) {
      team_sums_end(r.sums, team, words[k % 3][team > 32 ? mine : 0]);
      const unsigned char *from = ring + done_stage * a.row_bytes;
      if (++done_stage == a.depth) done_stage = 0;
      const float m1 = -r.sums.x * inverse_dim, m2 = -r.sums.y * inverse_dim;
      const float2 away = make_float2(m1, m1), dot = make_float2(m2, m2), by = make_float2(r.rstd, r.rstd);
      if (r.live) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          if (!in[i]) continue;
          if (kOneByOne && i > 0) asm volatile("" ::: "memory");
          float2 h[V / 2], g[V / 2];
          read(from, i, row_done, r, h, g);
          weigh(i, g);
          float o[V];
#pragma unroll
          for (int j = 0; j < V / 2; ++j) {
            const float2 v = __fmul2_rn(by, __ffma2_rn(h[j], dot, __fadd2_rn(g[j], away)));
            o[2 * j] = v.x;
            o[2 * j + 1] = v.y;
          }
          if (a.dsum) {
            float d[V];
            if (whole(i, row_done))
              row_load<T, V, false>(reinterpret_cast<const T *>(from + ds_place) + i * team * V, 0, V, true, d);
            else
              row_load<T, V, RAGGED>(static_cast<const T *>(a.dsum) + row_done * a.ldds, at_of(i), dim, false, d);
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] += d[j];
          }
          row_store<T, V, RAGGED>(reinterpret_cast<T *>(dx_next) - begin, at_of(i), dim, o);
        }
        row_done += stride;
      }
      dx_next += a.dx_hop;
      fetch();  // into this row's place
    };
    // one row ahead in the first half; the rows' sums have three sets of words, since a
    // warp may be a barrier ahead of one that still reads
    Row held[2];
    auto turn = [&](Row &now, Row &next, int k) {
      if (k + 1 < turns) {
        copies_wait_but(a.depth - 2);
        first_half(next, k + 1);
      }
      team_barrier(team, 1 + mine);
      second_half(now, k);
    };
    if (turns > 0) {
      copies_wait_but(a.depth - 1);
      first_half(held[0], 0);
    }
    for (int k = 0; k < turns; k += 2) {
      turn(held[0], held[1], k);
      if (k + 1 < turns) turn(held[1], held[0], k + 1);
    }
  });
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (!a.partial) return;
  float dw_out[E], db_out[E];
#pragma unroll
  for (int e = 0; e < E / 2; ++e) {
    dw_out[2 * e] = dw[e].x;
    dw_out[2 * e + 1] = dw[e].y;
    db_out[2 * e] = db[e].x;
    db_out[2 * e + 1] = db[e].y;
  }
  store_partial<V, E>(a, dw_out, db_out, team, dynamic, at_of);
}

// Single values, loaded as they come: for matrices whose rows are off 16 bytes unlike.
template <class T, int E>
__global__ void __launch_bounds__(512, 1) layernorm_grad_odd_kernel(const __grid_constant__ GradArgs a, int team) {
  __shared__ float words[2][kGradTeams][64];
  extern __shared__ __align__(16) unsigned char dynamic[];
  const int dim = (int)a.dim;
  const int t = threadIdx.x, teams = blockDim.y, mine = threadIdx.y, linear = mine * team + t;
  const int64_t stride = (int64_t)gridDim.x * teams, first = (int64_t)blockIdx.x * teams + mine;
  float dw[E], db[E];
#pragma unroll
  for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.0f;
  int flip = 0;  // two sets of words: one barrier per turn is enough
  // every thread of a warp takes the same number of turns (a warp may hold teams)
  const int64_t warp_first = (int64_t)blockIdx.x * teams + (linear & ~31) / team;
  for (int64_t turn = team > 32 ? first : warp_first, row = first; turn < a.rows;
       turn += stride, row += stride, flip ^= 1) {
    const bool live = row < a.rows;
    const float mean = live ? a.mean[row] : 0.0f, rstd = live ? a.rstd[row] : 0.0f;
    float h[E], g[E];
    const T *s = static_cast<const T *>(a.s) + row * a.lds;
    with_type(a.dy_dtype, [&](auto type) {
      using D = decltype(type);
      const D *dy = static_cast<const D *>(a.dy) + row * a.lddy;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int at = t + e * team;
        const bool in = live && at < dim;
        h[e] = in ? widen(s[at]) : 0.0f;
        g[e] = in ? widen(dy[at]) : 0.0f;
      }
    });
    // outside the row g is zero and nothing is stored, whatever h is
    float2 sums = make_float2(0.0f, 0.0f);
    with_weight_type<T>(a.w_dtype, [&](auto type) {
      using W = decltype(type);
      const W *weight = static_cast<const W *>(a.weight);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int at = t + e * team;
        if (at >= dim) continue;
        h[e] = (h[e] - mean) * rstd;
        dw[e] = fmaf(g[e], h[e], dw[e]);
        db[e] += g[e];
        if (weight) g[e] *= widen(weight[at]);
        sums.x += g[e];
        sums.y = fmaf(g[e], h[e], sums.y);
      }
    });
    float *const team_words = words[flip][team > 32 ? mine : 0];
    team_sums_begin(sums, team, team_words);
    team_barrier(team, 1 + mine);
    team_sums_end(sums, team, team_words);
    if (live) {
      const float away = sums.x / (float)a.dim, dot = sums.y / (float)a.dim;
      T *dx = static_cast<T *>(a.dx) + row * a.lddx;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int at = t + e * team;
        if (at >= dim) continue;
        float o = rstd * fmaf(-h[e], dot, g[e] - away);
        if (a.dsum) o += widen(static_cast<const T *>(a.dsum)[row * a.ldds + at]);
        dx[at] = narrow<T>(o);
      }
    }
    __syncwarp();
  }
  if (a.partial) store_partial<1, E>(a, dw, db, team, dynamic, [&](int e) { return t + e * team; });
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
// fill the GPU otherwise, 32 where the row is too long, and for 16-bit rows from 4,096
// values on, where what a thread does once a row counts (8191 x 5120 66.6 -> 61.4 us, 16384 x
// 4096 94.1 -> 89.9, 8191 x 5121 157 -> 129; 20000 x 1024 30.1 against 30.4, FP32 8192 x 4096 77.4
// against 80.6).  Single values stay at 8 while 512 threads hold the row so: 16 addresses and
// values spill (20000 x 200 bf16 with residual 22 us against 31, 9000 x 4000 186 against 208; FP32
// 22 against 34, 176 against 219).
template <int V>
Shape norm_shape(int64_t rows, int64_t dim, bool ragged) {
  if (ragged) dim += V - 1;  // a row may start inside its first vector
  Shape s;
  auto most = [&](int held) { return (int64_t)held * (held == kMostHeld<V> ? 1024 : 512); };
  s.held = rows * dim < (int64_t)sm_count() * 2048 * 8 ? 8 : 16;
  if (V == 8 && dim >= 4096 && s.held == 16) s.held = 32;
  if (V == 1) s.held = 8;
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

// The most blocks of the gradient kernels, which are also partial rows: one an SM.
int grad_blocks(int64_t rows) { return (int)std::min<int64_t>(rows, sm_count()); }

// Shared memory of a block's rows in flight, and the most of them per team.
constexpr size_t kGradRing = 200 * 1024;
constexpr int kGradDepth = 8;

// Launches kernel(a, team) with teams that hold `held` values a thread, as many as fit
// into `bound` threads a block; `ring`: with rows in flight.
template <int V, class K>
vcsr_status launch_teams(K kernel, GradArgs a, int64_t dim, int held, int bound, int blocks, bool ring,
                         cudaStream_t st) {
  const int team = team_of(ceil_div(dim, V), held / V);
  if (ring) {
    const int x_size = (int)type_size(a.x_dtype), dy_size = (int)type_size(a.dy_dtype);
    a.dy_at = team * held * x_size;
    a.ds_at = a.dy_at + team * held * dy_size;
    a.row_bytes = a.ds_at + (a.dsum ? team * held * x_size : 0);
    bound = (int)std::min<size_t>(bound, kGradRing / (2 * a.row_bytes) * team);  // two rows each
  }
  // teams that share a block join their sums
  const int teams = std::max(1, std::min<int>(bound / team, (int)ceil_div(a.rows, blocks)));
  const int in_block = (int)ceil_div(teams * team, 32) * 32 / team;
  size_t smem = in_block > 1 && a.partial ? (size_t)in_block * 2 * a.dim * sizeof(float) : 0;
  if (ring) {
    const int64_t x_size = (int64_t)type_size(a.x_dtype), dy_size = (int64_t)type_size(a.dy_dtype),
                  stride = (int64_t)blocks * in_block;
    a.depth = std::min<int>(kGradDepth, (int)kGradRing / (a.row_bytes * in_block));
    a.s_hop = stride * a.lds * x_size;
    a.dy_hop = stride * a.lddy * dy_size;
    a.ds_hop = stride * a.ldds * x_size;
    a.dx_hop = stride * a.lddx * x_size;
    smem = std::max(smem, (size_t)a.row_bytes * in_block * a.depth);
  }
  VCSR_TRY(allow_shared(reinterpret_cast<const void *>(kernel), smem));
  kernel<<<blocks, dim3((unsigned)team, (unsigned)in_block), smem, st>>>(a, team);
  return VCSR_OK;
}

template <class T, int V, bool RAGGED>
vcsr_status launch_grad(const GradArgs &a, int &blocks, cudaStream_t st) {
  const int64_t dim = a.dim + (RAGGED ? V - 1 : 0);  // a row may start inside its first vector
  if constexpr (V > 1) {
    // a multiple of 8 blocks, so that the rows of a team have one misalignment (or each
    // team has one row)
    if (RAGGED && blocks < a.rows) blocks = blocks / 8 * 8;
    auto run = [&](auto held, auto bound) {
      constexpr int E = decltype(held)::value, B = decltype(bound)::value;
      if (a.w_dtype == VCSR_F32)
        return launch_teams<V>(layernorm_grad_kernel<T, float, V, E, B, RAGGED>, a, dim, E, B, blocks, true, st);
      return launch_teams<V>(layernorm_grad_kernel<T, T, V, E, B, RAGGED>, a, dim, E, B, blocks, true, st);
    };
    using std::integral_constant;
    const size_t value = (a.dsum ? 2 : 1) * sizeof(T) + type_size(a.dy_dtype);  // bytes in the ring
    auto two_rows_fit = [&](int held) {
      return 2 * value * held * team_of(ceil_div(dim, V), held / V) <= kGradRing;
    };
    if (dim <= 16 * 512 && two_rows_fit(16)) {
      // 16-bit rows: 640 threads a block where they hold two teams and 512 only one (8191 x
      // 4608 bf16 with dsum 74 us against 99, 8191 x 5120 77 against 100, with FP32 dy 93 against 99
      // and 96 against 102).  Not FP32 rows, whose one team keeps HBM busier with its 128 registers
      // a thread (8191 x 4608 107 us against 123 in two teams, 8191 x 5120 111 against 125).
      if constexpr (V == 8 && !RAGGED)
        if (const int team = team_of(ceil_div(dim, V), 16 / V); 2 * team > 512 && 2 * team <= 640)
          return run(integral_constant<int, 16>{}, integral_constant<int, 640>{});
      return run(integral_constant<int, 16>{}, integral_constant<int, 512>{});
    }
    if (dim <= 32 * 512 && two_rows_fit(32)) return run(integral_constant<int, 32>{}, integral_constant<int, 512>{});
  } else {
    if (dim <= 8 * 512) return launch_teams<1>(layernorm_grad_odd_kernel<T, 8>, a, dim, 8, 512, blocks, false, st);
    if (dim <= 16 * 512) return launch_teams<1>(layernorm_grad_odd_kernel<T, 16>, a, dim, 16, 512, blocks, false, st);
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
                   a->scale, a->ldx, a->ldr,   a->ldy,      a->lds,    a->eps,  a->w_dtype, a->y_dtype};
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
  int blocks = grad_blocks(a->rows);
  const GradArgs k{a->rows, a->dim,  a->dy,  a->s,    a->weight, a->dsum, a->mean, a->rstd, a->dx,
                   sums ? static_cast<float *>(a->workspace) : nullptr,
                   a->lddy, a->lds,  a->ldds, a->lddx, a->x_dtype, a->w_dtype, a->dy_dtype};
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
