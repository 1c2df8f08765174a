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
  } else if (act == VCSR_ACT_GELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = activate<FAST>(VCSR_ACT_GELU, z[j]);
  } else if (act == VCSR_ACT_SILU) {
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = activate<FAST>(VCSR_ACT_SILU, z[j]);
  }
}

// The epilogue of output column f, rows r0 + j * step (j < n of N).  The warp
// calls it together; lanes without an output pass n <= 0.  get(z) fills in the
// sums: it is called after the residual's loads are issued, which so overlap
// with it and with the activation.  F32: e.type is known to be FP32.
template <int N, bool F32, class GET>
__device__ __forceinline__ void finish(const Epilogue &e, int f, int r0, int step, int n, GET &&get) {
  auto all = [&](auto type) {
    using T = decltype(type);
    T res[N];
    if (e.residual) {
      const T *p = static_cast<const T *>(e.residual) + (int64_t)r0 * e.ldr + f;
      const int64_t ld = e.ldr * step;
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
    get(z);
    if (n <= 0) return;
    if (e.row_scale) {
      const float cs = e.col_scale[f];
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < n) z[j] *= e.row_scale[r0 + j * step] * cs;
    }
    if (e.bias) {
      const float b = widen(static_cast<const T *>(e.bias)[f]);
#pragma unroll
      for (int j = 0; j < N; ++j) z[j] += b;
    }
    auto store = [&](void *to, int64_t pitch) {
      T *p = static_cast<T *>(to) + (int64_t)r0 * pitch + f;
      const int64_t ld = pitch * step;
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
}

// Descriptor of one MMA's slice (32 bytes of k, or 16 rows of k) of a staged
// operand, and how far it moves from slice to slice.  Along k: 8-row groups of
// 128-byte rows 1024 bytes apart.  Along the operand's own index: chunks of 64
// values 8192 bytes apart (a box each), groups of 8 k 1024 bytes apart.
__device__ __forceinline__ uint64_t slice_desc(uint32_t addr, int mn, int slice) {
  return mn ? tc::smem_desc(addr + slice * 2048, 8192, 1024, 2)
            : tc::smem_desc(addr + slice * 32, 16, 1024, 2);
}

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

template <class K, class... A>
inline vcsr_status launch(K kernel, int grid, int threads, size_t smem, int cluster, cudaStream_t st, A... args) {
  VCSR_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
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
