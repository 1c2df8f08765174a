// layer_gemm_tc.cuh — what the tensor-core products (layer_gemm_tc.cu for 16- and
// 8-bit operands, layer_gemm_f32.cu for FP32) share: the epilogue on accumulator
// rows, operand descriptors, the order of tiles and the launch.
#pragma once
#include <cuda.h>

#include "layer_gemm.cuh"
#include "tcgen05.cuh"

namespace vcsr {
namespace layer {

// Activation of N values, the branch outside the loop.
template <int N, bool FAST>
__device__ __forceinline__ void activate_all(int act, float *z) {
  if (act == VCSR_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = activate<FAST>(VCSR_ACT_RELU, z[j]);
  } else if (act == VCSR_ACT_GELU && FAST) {
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const float2 y = gelu_pair(make_float2(z[j], z[j + 1]));
      z[j] = y.x;
      z[j + 1] = y.y;
    }
  } else if (act == VCSR_ACT_GELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = activate<FAST>(VCSR_ACT_GELU, z[j]);
  } else if (act == VCSR_ACT_SILU) {
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = activate<FAST>(VCSR_ACT_SILU, z[j]);
  }
}

// The epilogue of output column f, rows r0 .. r0 + N - 1 (the first n of them).  The
// warp calls it together; lanes without an output pass n <= 0.  get(z) fills in the
// sums, or returns false: it is called after the residual's loads are issued, which
// so overlap with the wait for the sums.  F32: e.type is known to be FP32.
template <int N, bool F32, class GET>
__device__ __forceinline__ bool finish(const Epilogue &e, int f, int r0, int n, GET &&get) {
  bool ok = true;
  auto all = [&](auto type) {
    using T = decltype(type);
    T res[N];
    if (e.residual) {
      const T *p = static_cast<const T *>(e.residual) + (int64_t)r0 * e.ldr + f;
      const int64_t ld = e.ldr;
      if (n >= N) {
#pragma unroll
        for (int j = 0; j < N; ++j) res[j] = p[j * ld];
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (j < n) res[j] = p[j * ld];
      }
      __syncwarp();
    }
    float z[N];
    ok = get(z);
    if (n <= 0 || !ok) return;
    if (e.row_scale) {
      const float cs = e.col_scale[f];
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < n) z[j] *= e.row_scale[r0 + j] * cs;
    }
    if (e.bias) {
      const float b = widen(static_cast<const T *>(e.bias)[f]);
#pragma unroll
      for (int j = 0; j < N; ++j) z[j] += b;
    }
    auto store = [&](void *to, int64_t pitch) {
      T *p = static_cast<T *>(to) + (int64_t)r0 * pitch + f;
      const int64_t ld = pitch;
      if (n >= N) {
#pragma unroll
        for (int j = 0; j < N; ++j) p[j * ld] = narrow<T>(z[j]);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (j < n) p[j * ld] = narrow<T>(z[j]);
      }
    };
    if (e.pre) store(e.pre, e.ldp);
    activate_all<N, sizeof(T) == 2>(e.act, z);
    if (e.residual) {
#pragma unroll
      for (int j = 0; j < N; ++j) z[j] += widen(res[j]);
    }
    store(e.out, e.ldo);
  };
  if constexpr (F32)
    all(float{});
  else
    with_type(e.type, all);
  return ok;
}

// Asks L2 for the residual of a tile, `features` by `rows` from (f0, r0): thread t of
// `threads`, a 128-byte line at a time.
__device__ __forceinline__ void prefetch_residual(const Epilogue &e, int f0, int P, int features, int r0, int Q,
                                                  int rows, int t, int threads) {
  if (!e.residual) return;
  const int size = e.type == VCSR_F32 ? 4 : 2, lines = features * size / 128;
  for (int i = t; i < rows * lines; i += threads) {
    const int r = r0 + i / lines, f = f0 + i % lines * (128 / size);
    if (r < Q && f < P)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const char *>(e.residual) +
                                                     ((int64_t)r * e.ldr + f) * size));
  }
}

// 4 neighbouring values, or the first n of them.
template <class T, bool WHOLE>
__device__ __forceinline__ void load_four(const T *p, int n, float *out) {
  if constexpr (WHOLE) {
    const Vec<T, 4> v = load_vec<T, 4>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = widen(v.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) out[j] = widen(p[j]);
  }
}
template <class T, bool WHOLE>
__device__ __forceinline__ void store_four(T *p, int n, const float *x) {
  if constexpr (WHOLE) {
    store_narrow<T, 4>(p, x);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) p[j] = narrow<T>(x[j]);
  }
}

// Whether all of an epilogue's matrices take 4 values at a time from features that
// are multiples of 4.
__device__ __forceinline__ bool fours(const Epilogue &e) {
  const unsigned mask = e.type == VCSR_F32 ? 15 : 7;
  auto bits = [&](const void *p, int64_t ld) {
    return p ? ((unsigned)reinterpret_cast<uintptr_t>(p) & mask) | ((unsigned)ld & 3) : 0u;
  };
  return (bits(e.out, e.ldo) | bits(e.pre, e.ldp) | bits(e.residual, e.ldr) | bits(e.bias, 0)) == 0;
}

// The epilogue from sums in shared memory, `sums` [row][128 features] of this CTA
// and its peers (splits of them, added in rank order): rows first, first + step, ...
// below n of the tile at (f0, r0).  A warp takes whole rows, a lane 4 features, two
// rows at a time; a block needs many warps here, since one alone issues an
// instruction every 7 cycles or so.  FIX(f, r, z) may mend a lane's 4 sums.
template <bool F32, class FIX>
__device__ __forceinline__ void finish_rows(const Epilogue &e, uint32_t sums, int splits, int f0, int P, int r0,
                                            int first, int step, int n, FIX &&fix) {
  const int lane = threadIdx.x & 31, f = f0 + lane * 4, left = P - f;
  auto rows = [&](auto type, auto whole) {
    using T = decltype(type);
    constexpr bool WHOLE = decltype(whole)::value;
    constexpr int kAt = 2;
    float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f}, cs[4] = {1.0f, 1.0f, 1.0f, 1.0f};
    if (e.bias) load_four<T, WHOLE>(static_cast<const T *>(e.bias) + f, left, bias);
    if (e.col_scale) load_four<float, false>(e.col_scale + f, left, cs);
    const int64_t at = (int64_t)(r0 + first);
    const T *residual = static_cast<const T *>(e.residual) + at * e.ldr + f;
    T *pre = static_cast<T *>(e.pre) + at * e.ldp + f, *out = static_cast<T *>(e.out) + at * e.ldo + f;
    const int64_t dr = step * e.ldr, dp = step * e.ldp, dout = step * e.ldo;
    for (int row = first; row < n; row += step * kAt) {
      float z[kAt][4], res[kAt][4];
#pragma unroll
      for (int q = 0; q < kAt; ++q)
        if (e.residual && row + q * step < n) load_four<T, WHOLE>(residual + q * dr, left, res[q]);
#pragma unroll
      for (int q = 0; q < kAt; ++q) {
        const uint32_t from = sums + lane * 16 + (row + q * step) * 512;
        if (row + q * step >= n) break;
        if (splits == 1) {
          asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(z[q][0]), "=f"(z[q][1]), "=f"(z[q][2]), "=f"(z[q][3])
                       : "r"(from));
        } else {
          float part[8][4];  // every peer's asked for before the first is used
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < splits)
              asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                           : "=f"(part[k][0]), "=f"(part[k][1]), "=f"(part[k][2]), "=f"(part[k][3])
                           : "r"(tc::cluster_map(from, k)));
#pragma unroll
          for (int j = 0; j < 4; ++j) z[q][j] = part[0][j];
#pragma unroll
          for (int k = 1; k < 8; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (k < splits) z[q][j] += part[k][j];
        }
      }
#pragma unroll
      for (int q = 0; q < kAt; ++q) {
        if (row + q * step >= n) break;
        const int r = r0 + row + q * step;
        fix(f, r, z[q]);
        if (e.row_scale) {
          const float rs = e.row_scale[r];
#pragma unroll
          for (int j = 0; j < 4; ++j) z[q][j] *= rs * cs[j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) z[q][j] += bias[j];
        if (e.pre) store_four<T, WHOLE>(pre + q * dp, left, z[q]);
        activate_all<4, sizeof(T) == 2>(e.act, z[q]);
        if (e.residual) {
#pragma unroll
          for (int j = 0; j < 4; ++j) z[q][j] += res[q][j];
        }
        store_four<T, WHOLE>(out + q * dout, left, z[q]);
      }
      residual += kAt * dr;
      pre += kAt * dp;
      out += kAt * dout;
    }
  };
  if (left <= 0) return;
  auto all = [&](auto type) {
    if (left >= 4 && fours(e))
      rows(type, std::true_type{});
    else
      rows(type, std::false_type{});
  };
  if constexpr (F32)
    all(float{});
  else
    with_type(e.type, all);
}

// A place in a ring of N stages and the parity of its round.  full() is the parity
// that a consumer waits for; a producer waits for the other one on the stage's
// "empty" barrier, which passes at once in the first round.
template <int N>
struct RingPlace {
  int stage = 0;
  uint32_t round = 0;
  __device__ __forceinline__ void next() {
    if (++stage == N) {
      stage = 0;
      round ^= 1;
    }
  }
  __device__ __forceinline__ uint32_t full() const { return round; }
  __device__ __forceinline__ uint32_t empty() const { return round ^ 1; }
};

// Descriptor of a staged operand's first MMA slice (32 bytes of k, or 16 rows of
// k).  Along k: 8-row groups of 128-byte rows 1024 bytes apart.  Along the operand's
// own index: chunks of 64 values 8192 bytes apart (a box each), groups of 8 k 1024
// bytes apart.  Later slices and stages are further by their distance in 16-byte
// units: the issuing thread adds that, a few instructions per MMA (building each
// descriptor anew took it longer than the tensor core takes for the MMA).
__device__ __forceinline__ uint64_t stage_desc(uint32_t addr, int mn) {
  return mn ? tc::smem_desc(addr, 8192, 1024, 2) : tc::smem_desc(addr, 16, 1024, 2);
}
__device__ __forceinline__ uint32_t slice_step(int mn) { return (mn ? 2048 : 32) / 16; }

// Tile t in an order that keeps the tiles in flight in a block of 8 P tiles by
// as many Q tiles as it takes: each staged row is then read from L2 by the
// whole block at about the same time.
__device__ __forceinline__ void tile_of(int t, int tiles_p, int tiles_q, int *p, int *q) {
  constexpr int kGroup = 8;
  const int per = kGroup * tiles_q, g = t / per, first = g * kGroup,
            width = min(kGroup, tiles_p - first), in = t - g * per;
  *p = first + in % width;
  *q = in / width;
}

// Clusters of `size` blocks of a kernel that the current device runs at once (asked of
// the runtime once): with 128 KB of shared memory and more a block has an SM to itself,
// and an eight-block cluster eight SMs of one of the GPU's unequal parts, so that 16 of
// them, 128 blocks, are more than fit on 148 SMs.
int cluster_slots(const void *kernel, int threads, size_t smem, int size);

// How many CTAs share each tile's sum over k: as many as still run at once, up to 8,
// with at least two stages each.
inline int choose_splits(const void *kernel, int threads, size_t smem, int64_t tiles, int64_t stages) {
  int splits = 1;
  while (splits < 8 && stages >= 4 * splits && tiles * splits * 2 <= sm_count() &&
         tiles <= cluster_slots(kernel, threads, smem, splits * 2))
    splits *= 2;
  return splits;
}

// Whether this launch is the one that vcsr_layers_test_withhold_signal spoils (asks once).
bool take_withhold();

template <class K, class... A>
inline vcsr_status launch(K kernel, int grid, int threads, size_t smem, int cluster, cudaStream_t st, A... args) {
  VCSR_TRY(allow_shared(reinterpret_cast<const void *>(kernel), smem));
  cudaLaunchConfig_t c{};
  c.gridDim = dim3((unsigned)grid);
  c.blockDim = dim3((unsigned)threads);
  c.dynamicSmemBytes = smem;
  c.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  c.attrs = at;
  c.numAttrs = 1;
  VCSR_CUDA(cudaLaunchKernelEx(&c, kernel, args...));
  return VCSR_OK;
}

}  // namespace layer
}  // namespace vcsr
