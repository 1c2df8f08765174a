// layer_rows.cuh — what the kernels that work row by row share (layer_norm.cu,
// layer_layernorm.cu): values of a row held in a team's registers, sums over a team, copies
// into shared memory ahead of their use, and how rows are moved.
#pragma once
#include <initializer_list>
#include <type_traits>

#include "layer_common.cuh"

namespace vcsr {
namespace layer {

constexpr int kMaxThreads = 1024;

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
inline Access access_of(int64_t rows, int64_t dim, int v, const void *weight, std::initializer_list<Rows> all) {
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

// f(T{}, V, RAGGED) for rows of `type` moved as `how` says.
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

}  // namespace layer
}  // namespace vcsr
