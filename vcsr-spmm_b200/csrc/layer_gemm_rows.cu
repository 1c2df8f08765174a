// layer_gemm_rows.cu — products on the tensor cores (tcgen05, FP32 accumulators in tensor
// memory) whose epilogue works along an output row:
//
//   gated:  h[i, j] = act(g) u, g and u the sums with rows j and N + j of w;
//   blocks: 8-bit operands with a scale for each 128 values of k, so the sums of 128 values
//           are multiplied by their two scales and added up in registers.
//
// x is the MMA's M side here, so a tensor-memory lane is an output row and its columns are
// the output's (layer_gemm_tc.cu has it the other way round): a thread then holds g and u
// of the same output without an exchange between lanes, and the sums of a block of k take
// one scale per thread, x_scale[row] * w_scale, since 128 neighbouring rows of w share
// theirs.  Operands come by TMA in 128-byte rows (128-byte swizzle), 64 16-bit or 128 8-bit
// values of k per row and stage; reads past an edge are zeros.
//
// rows_pair_kernel — many rows: persistent pairs of CTAs (cta_group::2), 256 rows by 256
// columns per pair and tile: 128 columns of g and the same 128 of u, each staged by one
// CTA of the pair, or 256 columns.  Two accumulators alternate: from tile to tile (gated),
// or from one block of k to the next, while eight warps add up the one before in 128
// registers a thread (the loading and issuing warps give theirs up for that).
// Gated bf16 8192 x 8192, k = 4096: 665 to 690 us (1,593 TFLOP/s and more, by the power cap), 707
// to 734 with both factors kept; the tensor pipe is 88% busy.  Block-scaled 8192 x 8192, k = 4096:
// 292 us (1,885 TFLOP/s), 335 to 385 with a residual from memory.  There a block of k takes 0.51 us: two accumulators' way from the
// MMAs to the adding warps and back alone takes 0.39, reading them 0.07, adding 0.06 (in scratch
// copies without these parts); a tile's epilogue, which no other tile's sums can run under for
// want of registers, 3.4 us of 21.  Not kept, all the same or slower: 32 columns at a time,
// sixteen adding warps, outputs and residual through shared memory (a stage less for the ring).
//
// rows_split_kernel — few rows or few tiles: one tile of 128 rows by 128 columns (64 of g
// and 64 of u, or 128) per cluster of 1 to 8 CTAs, which split k between them and join
// their sums through distributed shared memory in rank order.  Few rows of x are staged
// as they are; lanes of the MMA past them read what lies there and are not used.  1 x 8192,
// k = 4096: gated bf16 27 us, of which reading 134 MB takes 21; block-scaled 11 (34 MB, 5).
//
// Every wait is bounded: a role that gives up records where, the CTA drains its own copies
// and MMAs, frees its tensor memory and returns, and vcsr_layers_check reports it.
#include <algorithm>

#include "layer_gemm_rows.cuh"
#include "layer_gemm_tc.cuh"
#include "spmm_tc.h"

namespace vcsr {
namespace layer {
namespace {

using namespace tc;

constexpr int kRows = 128;                // rows of x per CTA and tile
constexpr int kTileBytes = kRows * 128;   // of a staged operand of 128 rows
constexpr int kRing = 192 * 1024;         // stage ring of a CTA, bytes

__device__ int g_wait_error = 0;  // wait site | block << 4 of the first wait that ran out

struct RowsArgs {
  int M, N;
  int blocks;      // 128-byte blocks of k
  int block_k;     // values of k in one
  uint32_t idesc;
  int tiles_n, tiles_m;
  int box_rows;    // rows of x per copy (split kernel)
  const float *x_scale, *w_scale;
  int64_t ldxs, ldws;
  Epilogue e;
};

// What the epilogue of four columns f .. f + 3 (n of them) needs of vectors along the row.
struct Columns {
  float scale[2][4], bias[2][4];  // of g and u; a product without pairs has the first only
};
template <class T, bool PAIRS>
__device__ __forceinline__ Columns columns_at(const Epilogue &e, int64_t N, int f, int n) {
  Columns c;
#pragma unroll
  for (int h = 0; h < (PAIRS ? 2 : 1); ++h)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c.scale[h][j] = PAIRS && e.col_scale && j < n ? e.col_scale[h * N + f + j] : 1.0f;
      c.bias[h][j] = e.bias && j < n ? widen(static_cast<const T *>(e.bias)[h * N + f + j]) : 0.0f;
    }
  return c;
}

// The outputs of four columns of row r from the sums of g and u.  WHOLE, here and below: all
// four are there, and their matrices are moved four values at a time.
template <class T, bool CODES, bool WHOLE>
__device__ __forceinline__ void finish_pairs(const Epilogue &e, int64_t N, int64_t r, int f, int n, float row_scale,
                                             const Columns &c, float *g, float *u) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (CODES) {
      g[j] *= row_scale * c.scale[0][j];
      u[j] *= row_scale * c.scale[1][j];
    }
    g[j] += c.bias[0][j];
    u[j] += c.bias[1][j];
  }
  if (e.pre) {
    T *pre = static_cast<T *>(e.pre) + r * e.ldp + f;
    store_four<T, WHOLE>(pre, n, g);
    store_four<T, WHOLE>(pre + N, n, u);
  }
  activate_all<4, sizeof(T) == 2>(e.act, g);
#pragma unroll
  for (int j = 0; j < 4; ++j) g[j] *= u[j];
  store_four<T, WHOLE>(static_cast<T *>(e.out) + r * e.ldo + f, n, g);
}

// The outputs of four columns of row r of a product of block-scaled operands.
template <class T, bool WHOLE>
__device__ __forceinline__ void finish_four(const Epilogue &e, int64_t r, int f, int n, const Columns &c,
                                            const float *residual, float *z) {
#pragma unroll
  for (int j = 0; j < 4; ++j) z[j] += c.bias[0][j];
  activate_all<4, sizeof(T) == 2>(e.act, z);
  if (e.residual) {
#pragma unroll
    for (int j = 0; j < 4; ++j) z[j] += residual[j];
  }
  store_four<T, WHOLE>(static_cast<T *>(e.out) + r * e.ldo + f, n, z);
}

// f(T{}, WHOLE) for the type of the outputs and whether `n` columns and their matrices
// (pairs: u's part of pre too) take four values at a time.
template <bool PAIRS, class F>
__device__ __forceinline__ void with_outputs(const Epilogue &e, int64_t N, int n, F &&f) {
  const bool whole = n >= 4 && fours(e) && (!PAIRS || !e.pre || N % 4 == 0);
  with_type(e.type, [&](auto type) {
    if (whole)
      f(type, std::true_type{});
    else
      f(type, std::false_type{});
  });
}

// 32 bytes of a lane in one access (16-byte ones take twice the time where each lane has
// a row of its own).
struct alignas(32) Wide {
  uint32_t w[8];
};
__device__ __forceinline__ Wide load_wide(const void *p) {
  Wide v;
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7])
               : "l"(p)
               : "memory");
  return v;
}
__device__ __forceinline__ void store_wide(void *p, const Wide &v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v.w[0]), "r"(v.w[1]), "r"(v.w[2]),
               "r"(v.w[3]), "r"(v.w[4]), "r"(v.w[5]), "r"(v.w[6]), "r"(v.w[7])
               : "memory");
}
__device__ __forceinline__ bool wide(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0; }

// 16 neighbouring values, or the first n of them; VEC: 32 or 16 bytes at a time.
template <class T, bool VEC>
__device__ __forceinline__ void load_sixteen(const T *p, int n, float *out) {
  if constexpr (VEC) {
    if (wide(p)) {
      constexpr int V = 32 / sizeof(T);
#pragma unroll
      for (int i = 0; i < 16; i += V) {
        const Wide v = load_wide(p + i);
#pragma unroll
        for (int j = 0; j < V; ++j) out[i + j] = widen(reinterpret_cast<const T *>(v.w)[j]);
      }
      return;
    }
    constexpr int V = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 16; i += V) {
      const Vec<T, V> v = load_vec<T, V>(p + i);
#pragma unroll
      for (int j = 0; j < V; ++j) out[i + j] = widen(v.v[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) out[j] = j < n ? widen(p[j]) : 0.0f;
  }
}
template <class T, bool VEC>
__device__ __forceinline__ void store_sixteen(T *p, int n, const float *x) {
  if constexpr (VEC) {
    if (wide(p)) {
      constexpr int V = 32 / sizeof(T);
#pragma unroll
      for (int i = 0; i < 16; i += V) {
        Wide v;
        *reinterpret_cast<Vec<T, V> *>(v.w) = narrow_vec<T, V>(x + i);
        store_wide(p + i, v);
      }
      return;
    }
    constexpr int V = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 16; i += V) store_narrow<T, V>(p + i, x + i);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < n) p[j] = narrow<T>(x[j]);
  }
}
// Whether all of an epilogue's matrices take 16 bytes at a time from columns that are
// multiples of 16 (pairs: u's part of pre and of the vectors too).
template <bool PAIRS>
__device__ __forceinline__ bool sixteens(const Epilogue &e, int64_t N) {
  const int size = e.type == VCSR_F32 ? 4 : 2;
  auto bits = [&](const void *p, int64_t ld) { return p ? reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * size) : 0; };
  const uintptr_t all = bits(e.out, e.ldo) | bits(e.pre, e.ldp) | bits(e.residual, e.ldr) | bits(e.bias, 0) |
                        bits(e.col_scale, 0) | (PAIRS ? (uintptr_t)N * size : 0);
  return (all & 15) == 0;
}
// f(T{}, VEC) for 16 columns, n of them there.
template <bool PAIRS, class F>
__device__ __forceinline__ void with_sixteen(const Epilogue &e, int64_t N, int n, F &&f) {
  const bool vec = n >= 16 && sixteens<PAIRS>(e, N);
  with_type(e.type, [&](auto type) {
    if (vec)
      f(type, std::true_type{});
    else
      f(type, std::false_type{});
  });
}

// The outputs of columns f .. f + 15 (n of them) of row r from the sums of g and u.
template <class T, bool CODES, bool VEC>
__device__ __forceinline__ void finish_row_pairs(const Epilogue &e, int64_t N, int64_t r, int f, int n, float row_scale,
                                                 float *g, float *u) {
  auto scaled = [&](float *z, int64_t column) {
    float c[16];
    if (CODES) {
      load_sixteen<float, VEC>(e.col_scale + column, n, c);
#pragma unroll
      for (int j = 0; j < 16; ++j) z[j] *= row_scale * c[j];
    }
    if (e.bias) {
      load_sixteen<T, VEC>(static_cast<const T *>(e.bias) + column, n, c);
#pragma unroll
      for (int j = 0; j < 16; ++j) z[j] += c[j];
    }
    if (e.pre) store_sixteen<T, VEC>(static_cast<T *>(e.pre) + r * e.ldp + column, n, z);
  };
  scaled(u, N + f);
  scaled(g, f);
  activate_all<16, sizeof(T) == 2>(e.act, g);
#pragma unroll
  for (int j = 0; j < 16; ++j) g[j] *= u[j];
  store_sixteen<T, VEC>(static_cast<T *>(e.out) + r * e.ldo + f, n, g);
}

// The outputs of 16 columns of row r of a product of block-scaled operands.
template <class T, bool VEC>
__device__ __forceinline__ void finish_row(const Epilogue &e, int64_t r, int f, int n, const float *residual, float *z) {
  if (e.bias) {
    float c[16];
    load_sixteen<T, VEC>(static_cast<const T *>(e.bias) + f, n, c);
#pragma unroll
    for (int j = 0; j < 16; ++j) z[j] += c[j];
  }
  activate_all<16, sizeof(T) == 2>(e.act, z);
  if (e.residual) {
#pragma unroll
    for (int j = 0; j < 16; ++j) z[j] += residual[j];
  }
  store_sixteen<T, VEC>(static_cast<T *>(e.out) + r * e.ldo + f, n, z);
}

// Waits for this warp's loads from tensor memory, among them the 16 values at z: naming
// them keeps their uses behind the wait.
__device__ __forceinline__ void loaded16(float *z) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(z[0]), "+f"(z[1]), "+f"(z[2]), "+f"(z[3]), "+f"(z[4]), "+f"(z[5]), "+f"(z[6]), "+f"(z[7]),
                 "+f"(z[8]), "+f"(z[9]), "+f"(z[10]), "+f"(z[11]), "+f"(z[12]), "+f"(z[13]), "+f"(z[14]), "+f"(z[15])
               :
               : "memory");
}

// sums += scale * the next N columns of this warp's lanes of an accumulator, 16 at a time,
// the next 16 on their way meanwhile.  loaded() is called when the last have been read.
template <int N, class F>
__device__ __forceinline__ void add_scaled(uint32_t from, float scale, float2 *sums, F &&loaded) {
  float z[2][16];
  tmem_load16(from, z[0]);
#pragma unroll
  for (int c = 0; c < N; c += 16) {
    float *now = z[c / 16 % 2];
    loaded16(now);
    if (c + 16 < N)
      tmem_load16(from + c + 16, z[(c / 16 + 1) % 2]);
    else
      loaded();
#pragma unroll
    for (int j = 0; j < 16; j += 2)
      sums[(c + j) / 2] = __ffma2_rn(make_float2(now[j], now[j + 1]), make_float2(scale, scale), sums[(c + j) / 2]);
  }
}

// Four neighbouring scales of a row from block b on, those below `blocks`.  (A row per lane
// is a line of L1 per lane: by fours they take a quarter of its time.)
__device__ __forceinline__ float4 four_scales(const float *p, int b, int blocks, bool aligned) {
  if (aligned && b + 4 <= blocks) return *reinterpret_cast<const float4 *>(p + b);
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (b < blocks) v.x = p[b];
  if (b + 1 < blocks) v.y = p[b + 1];
  if (b + 2 < blocks) v.z = p[b + 2];
  if (b + 3 < blocks) v.w = p[b + 3];
  return v;
}

// ------------------------------------------------------------- pair kernel

constexpr int kPairWarps = 8;  // of the epilogue
// Two of the four that follow do nothing, but a register split is by fours.
template <bool BLOCKS>
constexpr int kPairThreads = 32 * (kPairWarps + (BLOCKS ? 4 : 2));
// Registers of a thread after the split (block-scaled sums take 128 of them): the
// launch's 168 x 384 in all.
constexpr int kPairFew = 40, kPairMany = 232;
static_assert(kPairFew * 128 + kPairMany * 256 <= 168 * 384, "");
constexpr int kPairStage = 2 * kTileBytes, kPairStages = kRing / kPairStage;
constexpr size_t kPairSmem = (size_t)kRing + 1024 + 512;
constexpr int kColumns = 256;  // of an accumulator

// WITHHOLD (a test), here and below: the first block (or pair) waits for a signal that is
// not sent.
template <bool BLOCKS, bool CODES, bool WITHHOLD>
__global__ void __launch_bounds__(kPairThreads<BLOCKS>, 1)
    rows_pair_kernel(const __grid_constant__ RowsArgs a, const __grid_constant__ CUtensorMap mx,
                     const __grid_constant__ CUtensorMap mw) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  unsigned char *ring = reinterpret_cast<unsigned char *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t *full = reinterpret_cast<uint64_t *>(ring + kRing), *empty = full + kPairStages;
  uint64_t *dfull = empty + kPairStages, *dfree = dfull + 2, *drain = dfree + 2;
  uint32_t *holder = reinterpret_cast<uint32_t *>(drain + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(holder + 1);
  volatile int *consumed = abort_flag + 1;

  // the same in all lanes, and known to be: what the MMA warp computes then stays in
  // uniform registers
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int tiles = a.tiles_n * a.tiles_m, first = blockIdx.x / 2, stride = gridDim.x / 2;
  constexpr int kOut = BLOCKS ? 256 : 128;  // output columns of a tile
  const bool withheld = WITHHOLD && first == 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(dfull + b, 1);
      mbar_init(dfree + b, 2 * kPairWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    *consumed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kPairWarps) tmem_alloc<2>(holder, 2 * kColumns);
  fence_before_sync();
  __syncthreads();
  cluster_sync();  // the peer's barriers are ready
  fence_after_sync();
  const uint32_t tmem = *holder;

  // (each part with its own register count, which a common one would limit both to)
  if (warp >= kPairWarps) {
    if (BLOCKS) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPairFew));
  }
  if (warp == kPairWarps) {
    if (lane == 0) {
      // copies of this CTA's halves, complete on the leader's barrier
      RingPlace<kPairStages> at;
      bool go = true;
      for (int t = first; t < tiles && go; t += stride) {
        int tn, tm;
        tile_of(t, a.tiles_n, a.tiles_m, &tn, &tm);
        const int r0 = tm * 2 * kRows + (int)rank * kRows;
        // the first CTA stages rows of w for g, the second those for u
        const int w0 = BLOCKS ? tn * kOut + (int)rank * kRows : tn * kOut + (int)rank * a.N;
        for (int b = 0; b < a.blocks; ++b, at.next()) {
          const int s = at.stage;
          if (!mbar_wait(empty + s, at.empty(), abort_flag, kWaitEmpty)) {
            go = false;
            break;
          }
          unsigned char *st = ring + s * kPairStage;
          const uint32_t bar = cluster_map(smem_u32(full + s), 0);
          if (rank == 0) mbar_arrive_tx(full + s, 2 * kPairStage);
          tma_load_2d_pair(st, &mx, b * a.block_k, r0, bar);
          tma_load_2d_pair(st + kTileBytes, &mw, b * a.block_k, w0, bar);
        }
      }
    }
  } else if (warp == kPairWarps + 1) {
    if (rank == 0) {
      const uint64_t x_first = stage_desc(smem_u32(ring), 0), w_first = stage_desc(smem_u32(ring) + kTileBytes, 0);
      RingPlace<kPairStages> at;
      RingPlace<2> acc;  // of the accumulators
      int g = 0;
      bool go = true;
      for (int t = first; t < tiles && go; t += stride) {
        for (int b = 0; b < a.blocks; ++b, ++g, at.next()) {
          const int s = at.stage, buf = acc.stage;
          bool ready = true;
          if (BLOCKS || b == 0) ready = mbar_wait(dfree + buf, acc.empty(), abort_flag, kWaitAccFree);
          if (!__all_sync(0xffffffffu, ready && mbar_wait(full + s, at.full(), abort_flag, kWaitFull))) {
            go = false;
            break;
          }
          fence_after_sync();
          const uint64_t xd = x_first + s * (kPairStage / 16), wd = w_first + s * (kPairStage / 16);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma<2, CODES>(tmem + buf * kColumns, xd + k * 2, wd + k * 2, a.idesc,
                            ((!BLOCKS && b > 0) || k > 0) ? 1u : 0u);
            mma_commit_pair(empty + s);
            if ((BLOCKS || b == a.blocks - 1) && !withheld) mma_commit_pair(dfull + buf);
          }
          __syncwarp();
          if (BLOCKS) acc.next();
        }
        if (!BLOCKS) acc.next();
      }
      if (elect_one()) {
        *consumed = g;
        // every MMA issued here has finished before the pair leaves
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                smem_u32(drain))
            : "memory");
        volatile int keep = 0;
        if (!mbar_wait(drain, 0, &keep, kWaitDrain)) *abort_flag = kWaitDrain;
      }
    }
  } else if (warp < kPairWarps) {
    if (BLOCKS) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPairMany));
    RingPlace<2> acc;
    const int quarter = warp & 3, half = warp >> 2;  // of the lanes, and of the columns
    bool go = true;
    if (withheld) go = __all_sync(0xffffffffu, mbar_wait(dfull, 0, abort_flag, kWaitAccFull, kTestPollLimit));
    auto ready = [&] {
      const bool now = mbar_wait(dfull + acc.stage, acc.full(), abort_flag, kWaitAccFull);
      if (!__all_sync(0xffffffffu, now)) return false;
      fence_after_sync();
      return true;
    };
    // the accumulator is read: free it
    auto release = [&] {
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_relaxed_at(cluster_map(smem_u32(dfree + acc.stage), 0));
    };
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    for (int t = first; t < tiles && go; t += stride) {
      int tn, tm;
      tile_of(t, a.tiles_n, a.tiles_m, &tn, &tm);
      const int r0 = tm * 2 * kRows + (int)rank * kRows + quarter * 32, r = r0 + lane;
      const bool live = r < a.M;
      if constexpr (!BLOCKS) {
        if (!(go = ready())) break;
        const float row_scale = CODES && live ? a.e.row_scale[r] : 1.0f;
        const uint32_t from = lanes + acc.stage * kColumns + half * 64;
#pragma unroll 1
        for (int c = 0; c < 64; c += 16) {
          float g[16], u[16];
          tmem_load16(from + c, g);
          tmem_load16(from + 128 + c, u);
          loaded16(g);
          loaded16(u);
          if (c + 16 == 64) release();
          const int f = tn * kOut + half * 64 + c, n = a.N - f;
          if (live && n > 0)
            with_sixteen<true>(a.e, a.N, n, [&](auto type, auto vec) {
              finish_row_pairs<decltype(type), CODES, decltype(vec)::value>(a.e, a.N, r, f, n, row_scale, g, u);
            });
          __syncwarp();
        }
        acc.next();
      } else {
        float2 sums[64];
#pragma unroll
        for (int j = 0; j < 64; ++j) sums[j] = make_float2(0.0f, 0.0f);
        // four blocks' scales are read while the four before are added up
        const float *xs = a.x_scale + (live ? r : 0) * a.ldxs;
        const float *ws = a.w_scale + (int64_t)min(tn * 2 + half, (a.N - 1) / kScaleBlock) * a.ldws;
        const bool by_four = ((reinterpret_cast<uintptr_t>(a.x_scale) | reinterpret_cast<uintptr_t>(a.w_scale)) & 15) == 0 &&
                             ((a.ldxs | a.ldws) & 3) == 0;
        float4 xs_next = four_scales(xs, 0, a.blocks, by_four), ws_next = four_scales(ws, 0, a.blocks, by_four);
        // the tile's sums are under way: its residual comes to L2 meanwhile
        prefetch_residual(a.e, tn * kOut + half * 128, a.N, 128, r0, a.M, 32, lane, 32);
#pragma unroll 1
        for (int b0 = 0; b0 < a.blocks && go; b0 += 4) {
          float scale[4] = {xs_next.x * ws_next.x, xs_next.y * ws_next.y, xs_next.z * ws_next.z, xs_next.w * ws_next.w};
          xs_next = four_scales(xs, b0 + 4, a.blocks, by_four);
          ws_next = four_scales(ws, b0 + 4, a.blocks, by_four);
#pragma unroll 1
          for (int b = b0; b < min(b0 + 4, a.blocks); ++b) {
            if (!(go = ready())) break;
            add_scaled<128>(lanes + acc.stage * kColumns + half * 128, scale[0], sums, release);
            acc.next();
            scale[0] = scale[1];
            scale[1] = scale[2];
            scale[2] = scale[3];
          }
        }
        if (!go) break;
        with_type(a.e.type, [&](auto type) {
          using T = decltype(type);
          const bool vec = sixteens<false>(a.e, a.N);
#pragma unroll
          for (int c = 0; c < 128; c += 16) {
            const int f = tn * kOut + half * 128 + c, n = a.N - f;
            float z[16], residual[16];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              z[2 * j] = sums[c / 2 + j].x;
              z[2 * j + 1] = sums[c / 2 + j].y;
            }
            if (!live || n <= 0) continue;
            const T *from = static_cast<const T *>(a.e.residual) + (int64_t)r * a.e.ldr + f;
            if (vec && n >= 16) {
              if (a.e.residual) load_sixteen<T, true>(from, n, residual);
              finish_row<T, true>(a.e, r, f, n, residual, z);
            } else {
              if (a.e.residual) load_sixteen<T, false>(from, n, residual);
              finish_row<T, false>(a.e, r, f, n, residual, z);
            }
          }
        });
        __syncwarp();
      }
    }
  }
  __syncwarp();
  fence_before_sync();
  __syncthreads();
  cluster_sync();  // no copy, commit or arrival of the peer is still to come
  fence_after_sync();
  if (*abort_flag && threadIdx.x == 0) {
    if (rank == 0) {  // copies that no MMA waited for
      volatile int keep = 0;
      for (int g = *consumed, n = 0; n < kPairStages; ++g, ++n)
        if (!mbar_wait(full + g % kPairStages, (uint32_t)((g / kPairStages) & 1), &keep, kWaitFull, 1 << 16)) break;
    }
    atomicCAS(&g_wait_error, 0, *abort_flag | (int)(blockIdx.x << 4));
  }
  __syncthreads();
  cluster_sync();
  if (warp == kPairWarps) tmem_free<2>(tmem, 2 * kColumns);
}

// ------------------------------------------------------------ split kernel

constexpr int kSplitWarps = 16;  // that add up and finish rows
constexpr int kSplitThreads = 32 * (kSplitWarps + 2);
constexpr int kMaxStages = 10;
constexpr size_t kSplitSmem = (size_t)kRing + 1024 + 512;
constexpr int kSplitColumns = 128;  // of an accumulator
constexpr int kFew = 16;
constexpr int kSplitSums = 4;       // accumulators of blocks of k
// Floats from a row of sums to the next: 16-byte accesses of 8 neighbouring rows then
// touch all banks once.
constexpr int kSumPitch = kSplitColumns + 4;
static_assert(kRows * kSumPitch * 4 <= kRing, "");

// Four sums of this CTA and its peers, added in rank order.
__device__ __forceinline__ void gather_four(uint32_t from, int splits, float *z) {
  if (splits == 1) {
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(z[0]), "=f"(z[1]), "=f"(z[2]), "=f"(z[3])
                 : "r"(from));
    return;
  }
  float part[8][4];  // every peer's asked for before the first is used
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < splits)
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(part[k][0]), "=f"(part[k][1]), "=f"(part[k][2]), "=f"(part[k][3])
                   : "r"(cluster_map(from, k)));
#pragma unroll
  for (int j = 0; j < 4; ++j) z[j] = part[0][j];
#pragma unroll
  for (int k = 1; k < 8; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (k < splits) z[j] += part[k][j];
}

// FEW: up to 16 rows of x, which are the MMA's N side here: a lane is a column of the
// output, and the MMA costs as much as 16 rows do, not 128 (1 x 8192, k = 4096: 11.0 us in
// 8 bits with block scales, against 12.2).
template <bool BLOCKS, bool CODES, bool FEW, bool WITHHOLD>
__global__ void __launch_bounds__(kSplitThreads, 1)
    rows_split_kernel(const __grid_constant__ RowsArgs a, const __grid_constant__ CUtensorMap mx,
                      const __grid_constant__ CUtensorMap mw, int splits) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  unsigned char *ring = reinterpret_cast<unsigned char *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t *full = reinterpret_cast<uint64_t *>(ring + kRing), *empty = full + kMaxStages;
  uint64_t *dfull = empty + kMaxStages, *dfree = dfull + kSplitSums, *drain = dfree + kSplitSums;
  uint32_t *holder = reinterpret_cast<uint32_t *>(drain + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(holder + 1);
  constexpr int kOut = BLOCKS ? 128 : 64;  // output columns of a tile
  constexpr int kTile = FEW ? kFew : kRows;                // rows of x
  constexpr int kWidth = FEW ? kFew : kSplitColumns;       // tensor-memory columns of an accumulator
  constexpr int kColumn = FEW ? kFew : 32;                 // of them, an adding warp's
  constexpr uint32_t kTmem = BLOCKS ? kSplitSums * kWidth : FEW ? 32 : kWidth;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = splits > 1 ? (int)cluster_rank() : 0, tile = blockIdx.x / splits;
  const int f0 = tile % a.tiles_n * kOut, r0 = tile / a.tiles_n * kTile;
  const int b0 = (int)((int64_t)a.blocks * rank / splits), b1 = (int)((int64_t)a.blocks * (rank + 1) / splits);
  // x's staged rows, then w's: the MMA's 128 lanes read on from the former into the latter
  const int x_bytes = a.box_rows * 128, stage_bytes = x_bytes + kTileBytes, stages = min(kMaxStages, kRing / stage_bytes);
  const bool withheld = WITHHOLD && blockIdx.x == 0;
  const int quarter = warp & 3, column = (warp >> 2) * kColumn;  // of an adding warp
  const int nr = min(kTile, a.M - r0);                           // output rows of the tile
  const bool mine = FEW ? column == 0 : quarter * 32 < nr;       // any of them in this warp
  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int b = 0; b < kSplitSums; ++b) {
      mbar_init(dfull + b, 1);
      mbar_init(dfree + b, FEW ? 4 : 4 * ((nr + 31) / 32));  // the warps with rows
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kSplitWarps) tmem_alloc<1>(holder, kTmem);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = *holder;
  float2 sums[kColumn / 2];
#pragma unroll
  for (int j = 0; j < kColumn / 2; ++j) sums[j] = make_float2(0.0f, 0.0f);

  if (warp == kSplitWarps) {
    if (lane == 0) {
      int s = 0, b = b0;
      uint32_t round = 1;
      for (; b < b1; ++b) {
        if (!mbar_wait(empty + s, round, abort_flag, kWaitEmpty)) break;
        unsigned char *st = ring + s * stage_bytes;
        mbar_arrive_tx(full + s, (uint32_t)stage_bytes);
        tma_load_2d(st, &mx, b * a.block_k, r0, full + s);
        if (BLOCKS) {
          tma_load_2d(st + x_bytes, &mw, b * a.block_k, f0, full + s);
        } else {  // 64 rows of w for g, 64 for u
          tma_load_2d(st + x_bytes, &mw, b * a.block_k, f0, full + s);
          tma_load_2d(st + x_bytes + kTileBytes / 2, &mw, b * a.block_k, a.N + f0, full + s);
        }
        if (++s == stages) {
          s = 0;
          round ^= 1;
        }
      }
      // every copy lands before the CTA leaves, whoever gave up
      volatile int keep = 0;
      for (int n = max(0, b - b0 - stages); n < b - b0; ++n)
        mbar_wait(full + n % stages, (uint32_t)(n / stages & 1), &keep, kWaitFull);
    }
  } else if (warp == kSplitWarps + 1) {
    const uint64_t x_first = stage_desc(smem_u32(ring), 0), w_first = stage_desc(smem_u32(ring) + x_bytes, 0);
    RingPlace<kSplitSums> acc;
    int s = 0;
    uint32_t round = 0;
    for (int b = b0; b < b1; ++b) {
      bool ready = true;
      if (BLOCKS) ready = mbar_wait(dfree + acc.stage, acc.empty(), abort_flag, kWaitAccFree);
      if (!__all_sync(0xffffffffu, ready && mbar_wait(full + s, round, abort_flag, kWaitFull))) break;
      fence_after_sync();
      const uint64_t xd = x_first + s * (stage_bytes / 16), wd = w_first + s * (stage_bytes / 16);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma<1, CODES>(tmem + acc.stage * kWidth, (FEW ? wd : xd) + k * 2, (FEW ? xd : wd) + k * 2, a.idesc,
                        ((!BLOCKS && b > b0) || k > 0) ? 1u : 0u);
        mma_commit(empty + s);
        if (BLOCKS && !withheld) mma_commit(dfull + acc.stage);
      }
      __syncwarp();
      if (BLOCKS) acc.next();
      if (++s == stages) {
        s = 0;
        round ^= 1;
      }
    }
    if (elect_one()) {
      if (!BLOCKS && withheld) mbar_wait(drain, 0, abort_flag, kWaitAccFull, kTestPollLimit);
      mma_commit(drain);
      volatile int keep = 0;  // wait for the issued MMAs even when another role gave up
      if (!mbar_wait(drain, 0, &keep, kWaitDrain)) *abort_flag = kWaitDrain;
    }
  } else if (BLOCKS && mine) {
    RingPlace<kSplitSums> acc;
    // the scales of this lane's row; FEW: of row `lane % 16`, for the lanes to share out
    const int r = r0 + (FEW ? lane % kFew : quarter * 32 + lane);
    const float *xs = a.x_scale + (r < a.M ? r : 0) * a.ldxs;
    const float *ws = a.w_scale + (int64_t)(f0 / kScaleBlock) * a.ldws;
    const bool by_four = ((reinterpret_cast<uintptr_t>(a.x_scale) | reinterpret_cast<uintptr_t>(a.w_scale)) & 15) == 0 &&
                         ((a.ldxs | a.ldws | b0) & 3) == 0;
    float4 xs_next = four_scales(xs, b0, b1, by_four), ws_next = four_scales(ws, b0, b1, by_four);
    bool go = true;
#pragma unroll 1
    for (int g = b0; g < b1 && go; g += 4) {
      float scale[4] = {xs_next.x * ws_next.x, xs_next.y * ws_next.y, xs_next.z * ws_next.z, xs_next.w * ws_next.w};
      xs_next = four_scales(xs, g + 4, b1, by_four);
      ws_next = four_scales(ws, g + 4, b1, by_four);
#pragma unroll 1
      for (int b = g; b < min(g + 4, b1); ++b, acc.next()) {
        const bool now = mbar_wait(dfull + acc.stage, acc.full(), abort_flag, kWaitAccFull,
                                   withheld ? kTestPollLimit : kPollLimit);
        if (!(go = __all_sync(0xffffffffu, now))) break;
        fence_after_sync();
        auto release = [&] {
          fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(dfree + acc.stage);
        };
        const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + acc.stage * kWidth + column;
        if constexpr (FEW) {
          float z[kFew];
          tmem_load16(from, z);
          loaded16(z);
          release();
#pragma unroll
          for (int j = 0; j < kFew; j += 2) {
            const float2 s = make_float2(__shfl_sync(0xffffffffu, scale[0], j), __shfl_sync(0xffffffffu, scale[0], j + 1));
            sums[j / 2] = __ffma2_rn(make_float2(z[j], z[j + 1]), s, sums[j / 2]);
          }
        } else {
          add_scaled<32>(from, scale[0], sums, release);
        }
        scale[0] = scale[1];
        scale[1] = scale[2];
        scale[2] = scale[3];
      }
    }
  }
  __syncwarp();
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const bool ok = *abort_flag == 0;
  // sums over the ring: its copies have landed and its MMAs have read it
  const uint32_t to = smem_u32(ring);
  if (warp < kSplitWarps && mine) {
    float z[kColumn];
    if constexpr (BLOCKS) {
#pragma unroll
      for (int j = 0; j < kColumn / 2; ++j) {
        z[2 * j] = sums[j].x;
        z[2 * j + 1] = sums[j].y;
      }
    } else {
      const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + column;
      if constexpr (FEW)
        tmem_load16(from, z);
      else
        tmem_load32(from, z);
      loaded16(z);
      if (!FEW) loaded16(z + kColumn - 16);
    }
    if constexpr (FEW) {
      const uint32_t at = to + (quarter * 32 + lane) * 4;
#pragma unroll
      for (int j = 0; j < kColumn; ++j)
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + j * kSumPitch * 4), "f"(z[j]) : "memory");
    } else {
      const uint32_t at = to + ((quarter * 32 + lane) * kSumPitch + column) * 4;
#pragma unroll
      for (int j = 0; j < kColumn; j += 4)
        asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at + j * 4), "f"(z[j]), "f"(z[j + 1]),
                     "f"(z[j + 2]), "f"(z[j + 3])
                     : "memory");
    }
  }
  __syncwarp();
  if (splits > 1)
    cluster_sync();
  else
    __syncthreads();
  // CTA k of a cluster finishes rows k, k + splits, ..., shared out among its warps: a
  // lane takes four columns, of one row per warp, or of two where outputs are pairs
  constexpr int kLanes = kOut / 4, kAtOnce = 32 / kLanes;
  if (ok && warp < kSplitWarps) {
    const int c = lane % kLanes * 4, f = f0 + c, n = a.N - f;
    for (int i = warp * kAtOnce + lane / kLanes; rank + i * splits < nr; i += kSplitWarps * kAtOnce) {
      if (n <= 0) break;
      const int local = rank + i * splits;
      const int64_t r = r0 + local;
      const uint32_t from = to + (local * kSumPitch + c) * 4;
      float z[4], u[4];
      gather_four(from, splits, z);
      if (!BLOCKS) gather_four(from + kOut * 4, splits, u);
      with_outputs<!BLOCKS>(a.e, a.N, n, [&](auto type, auto whole) {
        using T = decltype(type);
        constexpr bool WHOLE = decltype(whole)::value;
        const Columns columns = columns_at<T, !BLOCKS>(a.e, a.N, f, n);
        if constexpr (!BLOCKS) {
          finish_pairs<T, CODES, WHOLE>(a.e, a.N, r, f, n, CODES ? a.e.row_scale[r] : 1.0f, columns, z, u);
        } else {
          float residual[4];
          if (a.e.residual) load_four<T, WHOLE>(static_cast<const T *>(a.e.residual) + r * a.e.ldr + f, n, residual);
          finish_four<T, WHOLE>(a.e, r, f, n, columns, residual, z);
        }
      });
    }
  }
  __syncwarp();
  if (splits > 1) cluster_sync();  // until every peer has read this CTA's sums
  if (!ok && threadIdx.x == 0) atomicCAS(&g_wait_error, 0, *abort_flag | (int)(blockIdx.x << 4));
  fence_before_sync();
  __syncthreads();
  if (warp == kSplitWarps) {
    fence_after_sync();
    tmem_free<1>(tmem, kTmem);
  }
}

// ------------------------------------------------------------------- host

// A tensor map of rows x K values stored along k: boxes of 128 bytes of k by box_rows rows.
vcsr_status make_map(CUtensorMap *m, const void *p, int64_t ld, int64_t rows, int64_t K, int dtype, int box_rows) {
  EncodeTiledFn enc;
  VCSR_TRY(tensor_map_encoder(&enc));
  const size_t size = type_size(dtype);
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * size};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / size), (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType type = dtype == VCSR_BF16  ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                   : dtype == VCSR_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                       : CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const CUresult r = enc(m, type, 2, const_cast<void *>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(VCSR_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return VCSR_OK;
}

RowsArgs args_of(const RowsGemm &g) {
  RowsArgs a{};
  a.M = (int)g.M;
  a.N = (int)g.N;
  a.block_k = 128 / (int)type_size(g.dtype);
  a.blocks = (int)ceil_div(g.K, a.block_k);
  a.x_scale = g.x_scale;
  a.w_scale = g.w_scale;
  a.ldxs = g.ldxs;
  a.ldws = g.ldws;
  a.e = g.e;
  return a;
}

template <bool BLOCKS>
int64_t w_rows(const RowsGemm &g) {
  return BLOCKS ? g.N : 2 * g.N;
}

template <bool BLOCKS, bool CODES>
vcsr_status launch_pair(const RowsGemm &g, cudaStream_t st) {
  RowsArgs a = args_of(g);
  CUtensorMap mx, mw;
  VCSR_TRY(make_map(&mx, g.x, g.ldx, g.M, g.K, g.dtype, kRows));
  VCSR_TRY(make_map(&mw, g.w, g.ldw, w_rows<BLOCKS>(g), g.K, g.dtype, kRows));
  a.tiles_n = (int)ceil_div(a.N, BLOCKS ? 256 : 128);
  a.tiles_m = (int)ceil_div(a.M, 2 * kRows);
  const int64_t tiles = (int64_t)a.tiles_n * a.tiles_m;
  if (tiles > (1 << 30)) return fail(VCSR_ERR_RANGE, "more than 2^30 output tiles");
  a.idesc = instr_desc(g.dtype == VCSR_BF16 ? 1 : 0, 0, 0, 256, kColumns);
  const int grid = 2 * (int)std::min<int64_t>(tiles, sm_count() / 2);
  const auto kernel = take_withhold() ? rows_pair_kernel<BLOCKS, CODES, true> : rows_pair_kernel<BLOCKS, CODES, false>;
  return launch(kernel, grid, kPairThreads<BLOCKS>, kPairSmem, 2, st, a, mx, mw);
}

template <bool BLOCKS, bool FEW>
int64_t split_tiles(const RowsGemm &g) {
  return ceil_div(g.N, BLOCKS ? 128 : 64) * ceil_div(g.M, FEW ? kFew : kRows);
}
template <bool BLOCKS, bool CODES, bool FEW>
int splits_of(const RowsGemm &g) {
  return choose_splits(reinterpret_cast<const void *>(rows_split_kernel<BLOCKS, CODES, FEW, false>), kSplitThreads,
                       kSplitSmem, split_tiles<BLOCKS, FEW>(g), args_of(g).blocks);
}

template <bool BLOCKS, bool CODES, bool FEW>
vcsr_status launch_split(const RowsGemm &g, cudaStream_t st) {
  RowsArgs a = args_of(g);
  CUtensorMap mx, mw;
  a.box_rows = FEW ? kFew : kRows;
  while (!FEW && a.box_rows / 2 >= g.M) a.box_rows /= 2;
  VCSR_TRY(make_map(&mx, g.x, g.ldx, g.M, g.K, g.dtype, a.box_rows));
  VCSR_TRY(make_map(&mw, g.w, g.ldw, w_rows<BLOCKS>(g), g.K, g.dtype, BLOCKS ? 128 : 64));
  a.tiles_n = (int)ceil_div(a.N, BLOCKS ? 128 : 64);
  a.tiles_m = (int)ceil_div(a.M, FEW ? kFew : kRows);
  a.idesc = instr_desc(g.dtype == VCSR_BF16 ? 1 : 0, 0, 0, 128, FEW ? kFew : kSplitColumns);
  const int splits = splits_of<BLOCKS, CODES, FEW>(g);
  const int64_t grid = split_tiles<BLOCKS, FEW>(g) * splits;
  if (grid > 0x7fffffffll) return fail(VCSR_ERR_RANGE, "more than 2^31 - 1 thread blocks");
  const auto kernel = take_withhold() ? rows_split_kernel<BLOCKS, CODES, FEW, true> : rows_split_kernel<BLOCKS, CODES, FEW, false>;
  return launch(kernel, (int)grid, kSplitThreads, kSplitSmem, splits, st, a, mx, mw, splits);
}

// Expected microseconds, as in layer_gemm_tc.cu: a launch, then for every round of tiles a
// fixed part and a part per stage of k.  The best of the three kernels, or within 8% of it,
// for 132 products of 1 to 2048 rows, 256 to 8192 columns and k of 256 to 4096, gated bf16
// and block-scaled.  Some of them, up to 16 rows a tile / up to 128 / pairs: gated 17 x 8192,
// k = 4096 47.8 / 26.6 / 29.8; 128 x 256, k = 1024 7.4 / 9.3 / 11.4; 512 x 8192, k = 1024 - / 41.1 /
// 17.9; block-scaled 64 x 1024, k = 1024 6.1 / 7.3 / 12.0; 1024 x 4096, k = 4096 - / 37.3 / 25.4.
template <bool BLOCKS, bool CODES, bool FEW>
double split_cost(const RowsGemm &g) {
  const int splits = splits_of<BLOCKS, CODES, FEW>(g);
  const double fixed = FEW ? 4.6 : 5.0 + (double)std::min<int64_t>(g.M, kRows) / 64;
  return 1.2 + (splits > 1 ? 0.7 : 0.0) +
         (double)ceil_div(split_tiles<BLOCKS, FEW>(g) * splits, sm_count()) *
             (fixed + 0.36 * (double)ceil_div(args_of(g).blocks, splits));
}
template <bool BLOCKS>
double pair_cost(const RowsGemm &g) {
  const int blocks = args_of(g).blocks;
  const int64_t tiles = ceil_div(g.N, BLOCKS ? 256 : 128) * ceil_div(g.M, 256);
  return 11.5 + 0.33 * blocks + (double)(ceil_div(tiles, sm_count() / 2) - 1) * std::max(8.0, 0.42 * blocks);
}

template <bool BLOCKS, bool CODES>
vcsr_status launch_rows(const RowsGemm &g, cudaStream_t st) {
  // the kernels' 32-bit rows and columns run to the end of a tile
  if (std::max(g.M, g.N) > 0x7fffffffll - 512) return fail(VCSR_ERR_RANGE, "M or N above 2^31 - 513");
  const double few = split_cost<BLOCKS, CODES, true>(g), split = split_cost<BLOCKS, CODES, false>(g),
               pair = pair_cost<BLOCKS>(g);
  if (g.M <= kFew || (few <= split && few <= pair)) return launch_split<BLOCKS, CODES, true>(g, st);
  return split <= pair ? launch_split<BLOCKS, CODES, false>(g, st) : launch_pair<BLOCKS, CODES>(g, st);
}

}  // namespace

vcsr_status launch_gated_tc(const RowsGemm &g, cudaStream_t st) {
  return g.dtype == VCSR_E4M3 ? launch_rows<false, true>(g, st) : launch_rows<false, false>(g, st);
}
vcsr_status launch_blocks_tc(const RowsGemm &g, cudaStream_t st) { return launch_rows<true, true>(g, st); }

vcsr_status take_wait_error_rows(int *word) {
  const int zero = 0;
  VCSR_CUDA(cudaMemcpyFromSymbol(word, g_wait_error, sizeof(int)));
  if (*word) VCSR_CUDA(cudaMemcpyToSymbol(g_wait_error, &zero, sizeof(int)));
  return VCSR_OK;
}

}  // namespace layer
}  // namespace vcsr
