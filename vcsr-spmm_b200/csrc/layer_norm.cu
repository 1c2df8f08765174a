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
// Rows that do not start on 16 bytes (odd lengths) are still moved 16 bytes at a
// time where all matrices share their rows' misalignment, as contiguous ones do:
// vectors are cut at the memory's boundaries, so the first starts up to V - 1 values
// before the row.  Loads take it whole (it is the end of the row before; values
// outside the row are then set to zero), stores write its values one by one: FP32
// 20000 x 2001 to bf16 140 us, where the bytes take 87.  Other layouts are moved by single
// values (216 us).
//
// Gradient, per row: with h = s rstd, g = dy weight,
// dx = rstd (g - h mean(g h)) + dsum, dweight = sum over rows of dy h.  Its
// floor is HBM as well.  Teams take every (team count)-th row, with the next rows on
// their way while one is worked on, and keep their columns' dweight sums in
// registers over all of them; teams of a block join theirs in shared memory, blocks
// write one partial row each, and a second kernel adds the partial rows in block
// order (no atomics: the same result on every run).  8192 x 5120 bf16 with dsum:
// 72 us and 5 for the second kernel, 4.4 TB/s, bound by a barrier a row at 20 warps an SM.
#include <algorithm>
#include <atomic>
#include <initializer_list>
#include <mutex>
#include <type_traits>
#include <vector>

#include "layer_common.cuh"

namespace vcsr {
namespace layer {

namespace {
constexpr int kDevices = 64;
}

int sm_count() {
  static std::atomic<int> known[kDevices];
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kDevices) return sms;
  const int have = known[dev].load(std::memory_order_relaxed);
  if (have) return have;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess)
    known[dev].store(sms, std::memory_order_relaxed);
  return sms;
}

vcsr_status allow_shared(const void *kernel, size_t bytes) {
  struct Known {
    const void *kernel;
    int dev;
    size_t bytes;
  };
  static std::mutex mu;
  static std::vector<Known> known;
  int dev = 0;
  VCSR_CUDA(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lk(mu);
  for (Known &k : known)
    if (k.kernel == kernel && k.dev == dev) {
      if (bytes <= k.bytes) return VCSR_OK;
      VCSR_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
      k.bytes = bytes;
      return VCSR_OK;
    }
  VCSR_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  known.push_back({kernel, dev, bytes});
  return VCSR_OK;
}

vcsr_status check_matrix(const char *name, const void *p, int64_t ld, int64_t dim, int type,
                         bool optional) {
  if (!p) return optional ? VCSR_OK : fail(VCSR_ERR_INVALID, "%s is NULL", name);
  if (ld < dim) return fail(VCSR_ERR_INVALID, "pitch of %s (%lld) below its row length %lld", name,
                            (long long)ld, (long long)dim);
  if (!aligned(p, type_size(type))) return fail(VCSR_ERR_INVALID, "%s is not aligned to its type", name);
  return VCSR_OK;
}

namespace {

// Partial rows to their sums; a block takes 32 columns.
__global__ void __launch_bounds__(256)
    column_sum_kernel(const float *partial, int count, int64_t dim, void *out, int dtype) {
  __shared__ float part[8][33];
  column_sum_block(partial, count, dim, out, dtype, blockIdx.x, part);
}

constexpr int kMaxThreads = 1024;
// The most values a thread holds, in V-value vectors, and the largest block that
// leaves it registers for them (the gradient holds three arrays of them).  Single values
// need an address each and stop at 16.  Up to 16 values there are next to no spills; the
// forms of 32, for rows past 8,192 values, spill where rows are ragged (220 to 280 bytes
// stored a thread) and in the gradient (24 to 388).
template <int V>
constexpr int kMostHeld = V == 1 ? 16 : 32;
template <int V, int E>
constexpr int kNormBlock = E == kMostHeld<V> ? 1024 : 512;
constexpr int kGradBlock = 512;
// What the gradient's registers are sized for: 640 threads an SM, which is two blocks of
// teams of up to 320 (16-bit rows of 4,097 to 5,120 values, 8192 x 5120: 72 us; bounds of
// 512 and 1024 threads took 88 and 100) or one block of 512 made of smaller teams (8192 x
// 4096: 69 us with the second kernel, against a floor of 42); or two blocks of 512 with 8 single values.
template <int V, int E>
constexpr int kGradBound = E == 32 ? 512 : V == 1 ? 512 : 640;
template <int V, int E>
constexpr int kGradBlocksPerSm = V == 1 && E == 8 ? 2 : 1;

// V values of a row at `at`, a multiple of V less the row's misalignment when
// RAGGED: `whole` if they may all be read, then those outside the row become zero.
template <class X, int V, bool RAGGED>
__device__ __forceinline__ void row_load(const X *row, int at, int dim, bool whole, float *out) {
  if (whole) {
    const Vec<X, V> v = load_vec<X, V>(row + at);
#pragma unroll
    for (int j = 0; j < V; ++j)
      out[j] = !RAGGED || (unsigned)(at + j) < (unsigned)dim ? widen(v.v[j]) : 0.0f;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      out[j] = RAGGED && (unsigned)(at + j) < (unsigned)dim ? widen(row[at + j]) : 0.0f;
  }
}
// V values into a row, those in range.
template <class X, int V, bool RAGGED>
__device__ __forceinline__ void row_store(X *row, int at, int dim, const float *x) {
  if (!RAGGED || (at >= 0 && at + V <= dim)) {
    store_narrow<X, V>(row + at, x);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if ((unsigned)(at + j) < (unsigned)dim) row[at + j] = narrow<X>(x[j]);
  }
}
// Weights lie from value 0 on, whatever the rows do.
template <class X, int V, bool RAGGED>
__device__ __forceinline__ void weight_load(const X *w, int at, int dim, float *out) {
  if (!RAGGED) {
    const Vec<X, V> v = load_vec<X, V>(w + at);
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = widen(v.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = (unsigned)(at + j) < (unsigned)dim ? widen(w[at + j]) : 0.0f;
  }
}

struct NormArgs {
  int64_t rows, dim;
  const void *x, *residual, *weight;
  void *y, *sum;
  float *rstd, *scale;
  int64_t ldx, ldr, ldy, lds;
  float eps;
  int w_dtype, y_dtype;
};

// A sum, and with MAX a maximum of magnitudes, over a team's threads; every thread
// gets them.  Teams of up to 32 threads are a power of two of neighbouring lanes; a
// larger team has whole warps, `words` of its own (two per warp) and the block's
// barrier `id`.  Blocks are (threads of a team, teams): threadIdx.x is the thread's place
// in its team without a division.
template <bool MAX>
__device__ __forceinline__ void team_reduce(float &sum, float &top, int team, float2 *words, int id) {
  if (team >= 32) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (MAX) top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
  } else {
    for (int o = team >> 1; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (MAX) top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
  }
  if (team > 32) {
    const int lane = threadIdx.x & 31, warps = team >> 5;
    if (lane == 0) words[threadIdx.x >> 5] = make_float2(sum, top);
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(team) : "memory");
    const float2 w = lane < warps ? words[lane] : make_float2(0.0f, 0.0f);
    sum = w.x;
    top = w.y;
    for (int o = 16; o > 0; o >>= 1) {
      if (o >= warps) continue;  // the lanes from `warps` on hold zeros
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (MAX) top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    // the sums now stand in the lanes below the power of two at `warps`
    sum = __shfl_sync(0xffffffffu, sum, 0);
    if (MAX) top = __shfl_sync(0xffffffffu, top, 0);
  }
}
__device__ __forceinline__ float team_sum(float v, int team, float2 *words, int id) {
  float none = 0.0f;
  team_reduce<false>(v, none, team, words, id);
  return v;
}

// An asynchronous copy of `bytes` (8, 16 or 32, 8- or 16-byte aligned) of a
// row into this thread's own place in shared memory.
__device__ __forceinline__ void copy_async(uint32_t d, const void *src, int bytes) {
  if (bytes == 8) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(d), "l"(src) : "memory");
  } else {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
    if (bytes == 32)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d + 16),
                   "l"(static_cast<const char *>(src) + 16)
                   : "memory");
  }
}

template <int PENDING>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}
// Waits until all but the latest depth - 1 groups of copies have landed.
__device__ __forceinline__ void copies_wait_oldest(int depth) {
  if (depth == 4)
    copies_wait<3>();
  else if (depth == 3)
    copies_wait<2>();
  else if (depth == 2)
    copies_wait<1>();
  else
    copies_wait<0>();
}

// One row per team; E values per thread, V at a time (V values from one 16-byte
// access of x, or single values).  16384 x 4096 bf16 with residual to bf16 or to 8 bits:
// 83 us, 6.4 TB/s and 5.6 TB/s.  Blocks that stay and copy rows into shared memory ahead,
// as the gradient's do, gave no more there and 162 instead of 125 for 60000 x 1000 FP32:
// there are enough
// blocks to keep loads in flight.
template <class T, int V, int E, bool RAGGED>
__global__ void __launch_bounds__(kNormBlock<V, E>)
    rmsnorm_kernel(const __grid_constant__ NormArgs a, int team) {
  __shared__ float2 shared[32];
  const int dim = (int)a.dim;
  const int t = threadIdx.x;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = row < a.rows;
  const int shift = RAGGED ? (int)(row * a.ldx & (V - 1)) : 0;
  constexpr int kN = E / V;
  float s[E];
  float ss = 0.0f;
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
#pragma unroll
  for (int e = 0; e < E; ++e) ss = fmaf(s[e], s[e], ss);
  if (a.sum) {
    T *so = static_cast<T *>(a.sum) + row * a.lds;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int at = (t + i * team) * V - shift;
      if (live && at < dim) row_store<T, V, RAGGED>(so, at, dim, s + i * V);
    }
  }
  // s becomes s * weight, which rstd then makes y
  float top = 0.0f;
  auto weigh = [&](auto type) {
    using W = decltype(type);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int at = (t + i * team) * V - shift;
      if (at < dim) {
        float w[V];
        weight_load<W, V, RAGGED>(static_cast<const W *>(a.weight), at, dim, w);
#pragma unroll
        for (int j = 0; j < V; ++j) s[i * V + j] *= w[j];
      }
    }
  };
  if (a.w_dtype == VCSR_F32)
    weigh(float{});
  else
    weigh(T{});
  if (a.y_dtype == VCSR_E4M3) {
#pragma unroll
    for (int e = 0; e < E; ++e) top = max_or_nan(top, fabsf(s[e]));
    team_reduce<true>(ss, top, team, shared, 1);
  } else {
    ss = team_sum(ss, team, shared, 1);
  }
  const float rstd = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
  if (a.rstd && live && t == 0) a.rstd[row] = rstd;
  if (a.y_dtype == VCSR_E4M3) {
    // y / scale = s weight * 448 / max|s weight|: rstd, which is alike for the row,
    // falls out of the codes.  The factor and the product are rounded, so beside a tie
    // (within 2^-23 of it) a code may be the neighbouring one; so it may by rstd's own
    // rounding in the kernel for long rows, which divides.
    if (live && t == 0) a.scale[row] = top * rstd * (1.0f / 448.0f);
    const float raise = top < 1e-30f ? 0x1p64f : 1.0f;  // 448 / top would overflow
    const float k = rstd != rstd ? rstd : top > 0.0f ? 448.0f / (top * raise) : 0.0f;
    uint8_t *y = static_cast<uint8_t *>(a.y) + row * a.ldy;
    if (raise != 1.0f) {
#pragma unroll
      for (int e = 0; e < E; ++e) s[e] *= raise;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] *= k;
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
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] *= rstd;
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

// Rows of any length, one block each, in passes over the row: the sum of
// squares; the largest |y| (8-bit output); the stores.  s is stored in the
// last pass, so that it may replace x or residual.
template <class T>
__global__ void __launch_bounds__(kMaxThreads) rmsnorm_long_kernel(const NormArgs a) {
  __shared__ float2 shared[2][32];
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
  ss = team_sum(ss, blockDim.x, shared[0], 1);
  const float rstd = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
  if (a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
  CodeScale c = code_scale(448.0f);
  if (a.y_dtype == VCSR_E4M3) {
    float top = 0.0f;
    for (int64_t i = threadIdx.x; i < a.dim; i += blockDim.x) {
      float w;
      load_as_float<1>(a.weight, a.w_dtype, i, &w);
      top = max_or_nan(top, fabsf(value(i) * (rstd * w)));
    }
    float none = 0.0f;
    team_reduce<true>(none, top, blockDim.x, shared[1], 1);
    c = code_scale(top);
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
  int depth;  // rows in flight per team (16-byte access)
};

// Teams take every (team count)-th row.  With 16-byte access a thread copies its
// own vectors of this row and the next depth - 1 into shared memory ahead of their use
// (nobody else reads them: no barrier); single values are loaded as they come, by
// more teams at a time.
template <class T, int V, int E, bool RAGGED>
__global__ void __launch_bounds__(kGradBound<V, E>, kGradBlocksPerSm<V, E>)
    rmsnorm_grad_kernel(const __grid_constant__ GradArgs a, int team) {
  __shared__ float2 words[2][kGradBlock / 32];
  extern __shared__ __align__(16) unsigned char dynamic[];
  constexpr int kN = E / V;
  const int dim = (int)a.dim;
  const int t = threadIdx.x, teams = blockDim.y, mine = threadIdx.y, linear = mine * team + t;
  const int64_t stride = (int64_t)gridDim.x * teams, first = (int64_t)blockIdx.x * teams + mine;
  const int id = 1 + mine;
  // the same for all rows of a team: their distance is a multiple of 8
  const int shift = RAGGED ? (int)(first * a.lds & (V - 1)) : 0;
  // what lies past a row is the next rows', as far as there are some
  auto whole = [&](int64_t row, int at) {
    return row < a.rows && at < dim && (!RAGGED || at + V <= (a.rows - row) * a.dim);
  };
  // what one row takes of shared memory, and of it s, dy, dsum
  const int dy_size = a.dy_dtype == VCSR_F32 ? 4 : 2, slot = team * E;
  const int dy_at = slot * (int)sizeof(T), ds_at = dy_at + slot * dy_size,
            row_bytes = ds_at + (a.dsum ? slot * (int)sizeof(T) : 0);
  unsigned char *ring = dynamic + (size_t)mine * a.depth * row_bytes;
  float dw[E];
#pragma unroll
  for (int e = 0; e < E; ++e) dw[e] = 0.0f;

  // the row to be copied next, this thread's first vector of it
  int64_t ahead = first;
  const int64_t begin = t * V - shift;
  const char *s_next = static_cast<const char *>(a.s) + (first * a.lds + begin) * (int64_t)sizeof(T),
             *dy_next = static_cast<const char *>(a.dy) + (first * a.lddy + begin) * dy_size,
             *ds_next = static_cast<const char *>(a.dsum) + (first * a.ldds + begin) * (int64_t)sizeof(T);
  const int64_t s_hop = stride * a.lds * (int64_t)sizeof(T), dy_hop = stride * a.lddy * dy_size,
                ds_hop = stride * a.ldds * (int64_t)sizeof(T);
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  auto fetch = [&](int stage) {
    if (ahead < a.rows) {
      const uint32_t to = ring_at + (uint32_t)(stage * row_bytes);
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
    asm volatile("cp.async.commit_group;" ::: "memory");
    ahead += stride;
    s_next += s_hop;
    dy_next += dy_hop;
    ds_next += ds_hop;
  };
  if constexpr (V > 1) {
    for (int k = 0; k + 1 < a.depth; ++k) fetch(k);
  }

  int stage = 0, flip = 0;  // two sets of shared words: one barrier per row is enough
  // every thread of a warp takes the same number of turns (a warp may hold teams)
  const int64_t warp_first = (int64_t)blockIdx.x * teams + (linear & ~31) / team;
  for (int64_t turn = team > 32 ? first : warp_first, row = first; turn < a.rows;
       turn += stride, row += stride, flip ^= 1) {
    const bool live = row < a.rows;
    const float rstd = live ? a.rstd[row] : 0.0f;
    float h[E], g[E];
    const unsigned char *from = ring + (size_t)stage * row_bytes;
    if constexpr (V > 1) {
      int next = stage + a.depth - 1;
      if (next >= a.depth) next -= a.depth;
      // the place of the row before this one, read by this thread a turn ago
      fetch(next);
      copies_wait_oldest(a.depth);
      if (++stage == a.depth) stage = 0;
      const T *s = static_cast<const T *>(a.s) + row * a.lds;
      with_type(a.dy_dtype, [&](auto type) {
        using D = decltype(type);
        const D *dy = static_cast<const D *>(a.dy) + row * a.lddy;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          const int place = (t + i * team) * V, at = place - shift;
          if (whole(row, at)) {  // from shared memory, the thread's own place
            row_load<T, V, RAGGED>(reinterpret_cast<const T *>(from) + shift, at, dim, true, h + i * V);
            row_load<D, V, RAGGED>(reinterpret_cast<const D *>(from + dy_at) + shift, at, dim, true, g + i * V);
          } else {  // the last row's end, or nothing
            row_load<T, V, RAGGED>(s, at, live ? dim : 0, false, h + i * V);
            row_load<D, V, RAGGED>(dy, at, live ? dim : 0, false, g + i * V);
          }
        }
      });
    } else {
      with_type(a.dy_dtype, [&](auto type) {
        using D = decltype(type);
        const T *s = static_cast<const T *>(a.s) + row * a.lds;
        const D *dy = static_cast<const D *>(a.dy) + row * a.lddy;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int at = t + e * team;
          const bool in = live && at < dim;
          h[e] = in ? widen(s[at]) : 0.0f;
          g[e] = in ? widen(dy[at]) : 0.0f;
        }
      });
    }
    float dot = 0.0f;
    auto weigh = [&](auto type) {
      using W = decltype(type);
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int at = (t + i * team) * V - shift;
        if (at < dim) {
          float w[V];
          weight_load<W, V, RAGGED>(static_cast<const W *>(a.weight), at, dim, w);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int e = i * V + j;
            h[e] *= rstd;
            dw[e] = fmaf(g[e], h[e], dw[e]);
            g[e] *= w[j];
            dot = fmaf(g[e], h[e], dot);
          }
        }
      }
    };
    if (a.w_dtype == VCSR_F32)
      weigh(float{});
    else
      weigh(T{});
    const float mean = team_sum(dot, team, words[flip] + mine * (team >> 5), id) / (float)a.dim;
    T *dx = static_cast<T *>(a.dx) + row * a.lddx;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int at = (t + i * team) * V - shift;
      if (live && at < dim) {
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = rstd * (g[i * V + j] - h[i * V + j] * mean);
        if (a.dsum) {
          float d[V];
          if (V > 1 && whole(row, at))
            row_load<T, V, RAGGED>(reinterpret_cast<const T *>(from + ds_at) + shift, at, dim, true, d);
          else
            row_load<T, V, true>(static_cast<const T *>(a.dsum) + row * a.ldds, at, dim, false, d);
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] += d[j];
        }
        row_store<T, V, RAGGED>(dx, at, dim, o);
      }
    }
  }
  if constexpr (V > 1) asm volatile("cp.async.wait_all;" ::: "memory");
  if (!a.partial) return;
  float *out = a.partial + (int64_t)blockIdx.x * a.dim;
  float *joined = reinterpret_cast<float *>(dynamic);  // teams x dim
  if (teams > 1) __syncthreads();  // every team is done with its rows in shared memory
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const int at = (t + i * team) * V - shift;
    float *to = teams == 1 ? out + at : joined + mine * dim + at;
#pragma unroll
    for (int j = 0; j < V; ++j)
      if ((unsigned)(at + j) < (unsigned)dim) to[j] = dw[i * V + j];
  }
  if (teams == 1) return;
  __syncthreads();
  for (int c = linear; c < dim; c += teams * team) {
    float sum = 0.0f;
    for (int k = 0; k < teams; ++k) sum += joined[k * dim + c];
    out[c] = sum;
  }
}

// dx of rows of any length, one block each; their dweight comes from
// rmsnorm_long_dweight_kernel.
template <class T>
__global__ void __launch_bounds__(kMaxThreads) rmsnorm_long_grad_kernel(const GradArgs a) {
  __shared__ float2 shared[32];
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
  const float mean = team_sum(dot, blockDim.x, shared, 1) / (float)a.dim;
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

// How rows of `dim` values are moved: v values of every matrix at once where all
// rows start on v values, or all are off them alike (weights are then read one by
// one), else by single values.
enum Access { kSingle, kRagged, kVector };
struct Rows {
  const void *p;
  int64_t ld;
  int type;
};
Access access_of(int64_t rows, int64_t dim, int v, const void *weight, std::initializer_list<Rows> all) {
  bool even = dim % v == 0 && aligned(weight, 16), same = true;
  int64_t first = -1;
  for (const Rows &r : all) {
    if (!r.p) continue;
    if (!aligned(r.p, std::min<size_t>(16, v * type_size(r.type)))) return kSingle;
    const int64_t off = rows > 1 ? r.ld % v : 0;
    even = even && off == 0;
    same = same && (first < 0 || off == first);
    first = off;
  }
  return even ? kVector : same ? kRagged : kSingle;
}

struct Shape {
  int held, team, threads;  // values per thread, threads per row, threads per block
  bool fits;
};

// Teams: enough threads to hold the row at 16 values each (32 to 64 bytes of
// loads in flight a thread and tensor), 8 where there are too few rows to
// fill the GPU otherwise, 32 where the row is too long.
template <int V>
Shape shape_for(int64_t rows, int64_t dim, bool grad, bool ragged) {
  if (ragged) dim += V - 1;  // a row may start inside its first vector
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

template <class T, int V, bool RAGGED>
void launch_norm(const NormArgs &a, cudaStream_t st) {
  const Shape s = shape_for<V>(a.rows, a.dim, false, RAGGED);
  if (!s.fits) {
    rmsnorm_long_kernel<T><<<(unsigned)a.rows, kMaxThreads, 0, st>>>(a);
    return;
  }
  const unsigned grid = (unsigned)ceil_div(a.rows, s.threads / s.team);
  const dim3 block((unsigned)s.team, (unsigned)(s.threads / s.team));
  if (s.held == 8)
    rmsnorm_kernel<T, V, 8, RAGGED><<<grid, block, 0, st>>>(a, s.team);
  else if (s.held == 16)
    rmsnorm_kernel<T, V, 16, RAGGED><<<grid, block, 0, st>>>(a, s.team);
  else
    rmsnorm_kernel<T, V, kMostHeld<V>, RAGGED><<<grid, block, 0, st>>>(a, s.team);
}

// Blocks of the gradient kernel, which are also the partial rows of dweight.
// A multiple of 8 unless every row has a team of its own (see rmsnorm_grad_kernel).
int grad_blocks(int64_t rows) { return (int)std::min<int64_t>(rows, (int64_t)sm_count() * 2 / 8 * 8); }

// Shared memory of a block's rows in flight: two blocks an SM.
constexpr size_t kGradRing = 104 * 1024;

template <class T, int V, bool RAGGED>
vcsr_status launch_grad(GradArgs a, int blocks, cudaStream_t st) {
  const Shape s = shape_for<V>(a.rows, a.dim, true, RAGGED);
  if (!s.fits) {
    rmsnorm_long_grad_kernel<T><<<(unsigned)a.rows, kMaxThreads, 0, st>>>(a);
    if (a.partial)
      rmsnorm_long_dweight_kernel<T>
          <<<dim3((unsigned)ceil_div(a.dim, 256), (unsigned)blocks), 256, 0, st>>>(a);
    return VCSR_OK;
  }
  // blocks of about 512 threads, two an SM: teams that share one join their dweight
  const int teams = std::max(1, std::min<int>(kGradBlock / s.team, (int)ceil_div(a.rows, blocks)));
  const int threads = (int)ceil_div(teams * s.team, 32) * 32, in_block = threads / s.team;
  size_t smem = in_block > 1 && a.partial ? (size_t)in_block * a.dim * sizeof(float) : 0;
  if (V > 1) {
    const size_t row = (size_t)s.team * s.held *
                       ((a.dsum ? 2 : 1) * sizeof(T) + type_size(a.dy_dtype)) * in_block;
    a.depth = row * 4 <= kGradRing ? 4 : row * 3 <= kGradRing ? 3 : row * 2 <= 2 * kGradRing ? 2 : 1;
    smem = std::max(smem, row * a.depth);
  }
  auto run = [&](auto kernel) -> vcsr_status {
    VCSR_TRY(allow_shared(reinterpret_cast<const void *>(kernel), smem));
    kernel<<<blocks, dim3((unsigned)s.team, (unsigned)in_block), smem, st>>>(a, s.team);
    return VCSR_OK;
  };
  if (s.held == 8) return run(rmsnorm_grad_kernel<T, V, 8, RAGGED>);
  if (s.held == 16) return run(rmsnorm_grad_kernel<T, V, 16, RAGGED>);
  return run(rmsnorm_grad_kernel<T, V, kMostHeld<V>, RAGGED>);
}

template <class F>
void by_type(int type, Access how, F &&f) {
  auto go = [&](auto t, auto v) {
    if (how == kVector)
      f(t, v, std::false_type{});
    else if (how == kRagged)
      f(t, v, std::true_type{});
    else
      f(t, std::integral_constant<int, 1>{}, std::false_type{});
  };
  if (type == VCSR_F32)
    go(float{}, std::integral_constant<int, 4>{});
  else if (type == VCSR_BF16)
    go(__nv_bfloat16{}, std::integral_constant<int, 8>{});
  else
    go(__half{}, std::integral_constant<int, 8>{});
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
  if (a->rows == 0) return VCSR_OK;
  if (a->dim == 0) {  // a mean of nothing: NaN (all bits set); a largest value of nothing: 0
    if (a->rstd) VCSR_CUDA(cudaMemsetAsync(a->rstd, 0xff, (size_t)a->rows * sizeof(float), st));
    if (a->y_dtype == VCSR_E4M3 && a->scale)
      VCSR_CUDA(cudaMemsetAsync(a->scale, 0, (size_t)a->rows * sizeof(float), st));
    return VCSR_OK;
  }
  if (a->rows > 0x7fffffffll) return fail(VCSR_ERR_RANGE, "more than 2^31 - 1 rows");
  VCSR_TRY(check_matrix("x", a->x, a->ldx, a->dim, a->x_dtype, false));
  VCSR_TRY(check_matrix("residual", a->residual, a->ldr, a->dim, a->x_dtype, true));
  VCSR_TRY(check_matrix("weight", a->weight, a->dim, a->dim, a->w_dtype, false));
  VCSR_TRY(check_matrix("y", a->y, a->ldy, a->dim, a->y_dtype, false));
  VCSR_TRY(check_matrix("sum", a->sum, a->lds, a->dim, a->x_dtype, true));
  if (a->y_dtype == VCSR_E4M3 && !a->scale)
    return fail(VCSR_ERR_INVALID, "an 8-bit y needs scale");
  VCSR_TRY(check_matrix("rstd", a->rstd, 1, 1, VCSR_F32, true));
  VCSR_TRY(check_matrix("scale", a->scale, 1, 1, VCSR_F32, true));
  NormArgs k{a->rows, a->dim, a->x,   a->residual, a->weight, a->y,       a->sum,
             a->rstd, a->scale, a->ldx, a->ldr,      a->ldy,    a->lds,     a->eps,
             a->w_dtype, a->y_dtype};
  const int v = a->x_dtype == VCSR_F32 ? 4 : 8;
  const Access how = access_of(a->rows, a->dim, v, a->weight, {{a->x, a->ldx, a->x_dtype}, {a->residual, a->ldr, a->x_dtype},
                                                    {a->y, a->ldy, a->y_dtype}, {a->sum, a->lds, a->x_dtype}});
  by_type(a->x_dtype, how, [&](auto t, auto n, auto ragged) {
    launch_norm<decltype(t), decltype(n)::value, decltype(ragged)::value>(k, st);
  });
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
             a->lddy, a->lds, a->ldds, a->lddx, a->w_dtype, a->dy_dtype, 0};
  const int v = a->x_dtype == VCSR_F32 ? 4 : 8;
  const Access how = access_of(a->rows, a->dim, v, a->weight, {{a->dy, a->lddy, a->dy_dtype}, {a->s, a->lds, a->x_dtype},
                                                    {a->dsum, a->ldds, a->x_dtype}, {a->dx, a->lddx, a->x_dtype}});
  vcsr_status done = VCSR_OK;
  by_type(a->x_dtype, how, [&](auto t, auto n, auto ragged) {
    done = launch_grad<decltype(t), decltype(n)::value, decltype(ragged)::value>(k, blocks, st);
  });
  VCSR_TRY(done);
  VCSR_CUDA(cudaGetLastError());
  if (a->dweight) {
    column_sum_kernel<<<(unsigned)ceil_div(a->dim, 32), 256, 0, st>>>(k.partial, blocks, a->dim, a->dweight,
                                                                    a->w_dtype);
    VCSR_CUDA(cudaGetLastError());
  }
  return VCSR_OK;
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
