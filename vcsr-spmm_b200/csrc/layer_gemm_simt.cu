// layer_gemm_simt.cu — the product on the FP32 units: 64 x 64 tiles of the
// output, 16 values of k at a time through shared memory, 4 x 4 sums per
// thread.  Any type, order, pitch and alignment.
#include "layer_gemm.cuh"

namespace vcsr {
namespace layer {
namespace {

constexpr int kTile = 64, kStep = 16;

__device__ __forceinline__ float element(const void *p, int type, int64_t at) {
  if (type == VCSR_E4M3) return e4m3_value(static_cast<const uint8_t *>(p)[at]);
  float v;
  load_as_float<1>(p, type, at, &v);
  return v;
}

__device__ __forceinline__ void fill(float (*tile)[kTile + 1], const Operand &o, int type,
                                     int64_t row0, int64_t rows, int64_t k0, int64_t K) {
  for (int i = threadIdx.x; i < kTile * kStep; i += 256) {
    const int r = o.transposed ? i % kTile : i / kStep, k = o.transposed ? i / kTile : i % kStep;
    const int64_t row = row0 + r, kk = k0 + k;
    float v = 0.0f;
    if (row < rows && kk < K)
      v = element(o.p, type, o.transposed ? kk * o.ld + row : row * o.ld + kk);
    tile[k][r] = v;
  }
}

__global__ void __launch_bounds__(256) gemm_simt_kernel(const __grid_constant__ Gemm g) {
  __shared__ float ta[kStep][kTile + 1], tb[kStep][kTile + 1];
  const int64_t tiles_n = (g.N + kTile - 1) / kTile;
  const int64_t i0 = blockIdx.x / tiles_n * kTile, j0 = blockIdx.x % tiles_n * kTile;
  const int ti = threadIdx.x / 16, tj = threadIdx.x % 16;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < g.K; k0 += kStep) {
    fill(ta, g.a, g.dtype, i0, g.M, k0, g.K);
    fill(tb, g.b, g.dtype, j0, g.N, k0, g.K);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kStep; ++k) {
      float a[4], b[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        a[u] = ta[k][ti + 16 * u];
        b[u] = tb[k][tj + 16 * u];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[u][v] = fmaf(a[u], b[v], acc[u][v]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int64_t i = i0 + ti + 16 * u, j = j0 + tj + 16 * v;
      if (i < g.M && j < g.N) {
        const Epilogue &e = g.e;
        float z = acc[u][v], t;
        if (e.row_scale) z *= e.row_scale[i] * e.col_scale[j];
        if (e.bias) {
          load_as_float<1>(e.bias, e.type, j, &t);
          z += t;
        }
        if (e.pre) store_as<1>(e.pre, e.type, i * e.ldp + j, &z);
        z = activate(e.act, z);
        if (e.residual) {
          load_as_float<1>(e.residual, e.type, i * e.ldr + j, &t);
          z += t;
        }
        store_as<1>(e.out, e.type, i * e.ldo + j, &z);
      }
    }
}

}  // namespace

vcsr_status launch_gemm_simt(const Gemm &g, cudaStream_t st) {
  const int64_t tiles = ceil_div(g.M, kTile) * ceil_div(g.N, kTile);
  if (tiles > 0x7fffffffll) return fail(VCSR_ERR_RANGE, "more than 2^31 - 1 output tiles");
  gemm_simt_kernel<<<(unsigned)tiles, 256, 0, st>>>(g);
  VCSR_CUDA(cudaGetLastError());
  return VCSR_OK;
}

}  // namespace layer
}  // namespace vcsr
