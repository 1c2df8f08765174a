// layer_gemm_tc.cu — the product of 16- and 8-bit operands on the tensor cores
// (tcgen05, kind::f16 and kind::f8f6f4, FP32 accumulators in tensor memory).
//
// out[r, f] = epilogue(sum_k Q(r, k) P(f, k)).  P, the operand of the output's
// contiguous index f, is the MMA's M side, so a tensor-memory lane is an
// output column: the epilogue's warps read 32 lanes of one accumulator column
// at a time and store (and load the residual) 32 neighbouring values of one
// output row, without a transposition through shared memory.  Operands come by
// TMA in 128-byte rows (128-byte swizzle): stored along k, 64 16-bit (128 8-bit)
// values of k per row and stage; stored along f or r, 64 of them per row and a
// row per k.  Reads past an operand's edge are zeros.
//
// Two kernels, by the size of the output:
//
// gemm_pair_kernel — many rows: persistent pairs of CTAs (cta_group::2), 256
// features x 256 rows per pair and tile.  Each CTA stages 128 rows of each
// operand (32 KB per 64 values of k, half of what a CTA alone with a 128 x 256
// tile would read from L2 per MMA), two accumulators alternate, so that the
// epilogue of a tile runs under the next tile's MMAs.  Bound by the tensor cores and, in
// a long run, by power: bf16 16384 x 8192, k = 4096 708 to 732 us (1,503 to 1,554 TFLOP/s),
// 805 with every part of the epilogue; e4m3 4096 x 8192, k = 4096 with gelu 105 us (2,630 TFLOP/s).
//
// gemm_split_kernel — few rows or few tiles: one tile of 128 features x 16 to
// 128 rows per cluster of 1 to 8 CTAs, which split k between them and join their
// partial sums through distributed shared memory in rank order (no workspace, no
// atomics: the same result on every run).  For few rows it is bound by reading
// the weights once; the split is what puts every SM on that: 1 x 4096, k = 4096 bf16
// 9.5 us, of which reading 34 MB takes 5.
//
// Every wait is bounded: a role that gives up records where, the CTA drains its
// own copies and MMAs, frees its tensor memory and returns, and vcsr_layers_check
// reports it.
#include <algorithm>
#include <atomic>
#include <mutex>
#include <vector>

#include "layer_gemm_tc.cuh"
#include "spmm_tc.h"

namespace vcsr {
namespace layer {
namespace {

using namespace tc;

constexpr int kPRows = 128;         // rows of P per CTA
constexpr int kPBytes = kPRows * 128;
constexpr int kRing = 192 * 1024;   // stage ring of a CTA, bytes

__device__ int g_wait_error = 0;  // wait site | block << 4 of the first wait that ran out

struct TcArgs {
  int P, Q;        // extents of f and r
  int blocks;      // 128-byte blocks of k
  int block_k;     // values of k in one
  int p_mn, q_mn;  // operand stored along its own index
  uint32_t idesc;
  int tiles_p, tiles_q;
  Epilogue e;
};

// Copies of `rows` rows (a multiple of 64 where mn) of an operand, block b of
// k, to `dst`; LOAD(dst, x, y) issues one.
template <class LOAD>
__device__ __forceinline__ void load_operand(unsigned char *dst, int mn, int row0, int rows, int b,
                                             int block_k, LOAD &&load) {
  if (mn) {
    for (int c = 0; c < rows; c += 64) load(dst + c * 128, row0 + c, b * block_k);
  } else {
    load(dst, b * block_k, row0);
  }
}

// ------------------------------------------------------------ split kernel

constexpr int kSplitThreads = 512;  // for the epilogue: two warps do the rest

template <int BN>
constexpr int kSplitStages = kRing / (kPBytes + BN * 128);
template <int BN>
constexpr size_t kSplitSmem = (size_t)kSplitStages<BN> * (kPBytes + BN * 128) + 1024 + 512;

// One product, or two that share a launch: the clusters from `second` on are the other's.
struct SplitJobs {
  TcArgs a[2];
  CUtensorMap p[2], q[2];
  int splits, second;
};

// WITHHOLD (a test), here and below: the first block (or pair) waits for a signal that is
// not sent.  Kernels of their own: the branches alone took registers and time from these.
template <int BN, bool CODES, bool WITHHOLD>
__global__ void __launch_bounds__(kSplitThreads, 1) gemm_split_kernel(const __grid_constant__ SplitJobs jobs) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  unsigned char *ring = reinterpret_cast<unsigned char *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  constexpr int kStages = kSplitStages<BN>, kStage = kPBytes + BN * 128;
  constexpr uint32_t kColumns = BN < 32 ? 32 : BN;
  uint64_t *full = reinterpret_cast<uint64_t *>(ring + kStages * kStage), *empty = full + kStages;
  uint64_t *done = empty + kStages;
  uint32_t *holder = reinterpret_cast<uint32_t *>(done + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(holder + 1);

  // the same in all lanes, and known to be: what the MMA warp computes then stays in
  // uniform registers, where its instructions want their operands
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int splits = jobs.splits, rank = splits > 1 ? (int)cluster_rank() : 0;
  const int cluster = blockIdx.x / splits, which = cluster >= jobs.second ? 1 : 0;
  const int tile = cluster - which * jobs.second;
  const TcArgs &a = jobs.a[which];
  const CUtensorMap *mp = &jobs.p[which], *mq = &jobs.q[which];
  const int f0 = tile % a.tiles_p * kPRows, r0 = tile / a.tiles_p * BN;
  const int b0 = (int)((int64_t)a.blocks * rank / splits),
            b1 = (int)((int64_t)a.blocks * (rank + 1) / splits);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4) tmem_alloc<1>(holder, kColumns);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = *holder;

  if (warp == 4) {
    if (lane == 0) {
      RingPlace<kStages> at;
      for (int b = b0; b < b1; ++b, at.next()) {
        const int s = at.stage;
        if (!mbar_wait(empty + s, at.empty(), abort_flag, kWaitEmpty)) break;
        unsigned char *st = ring + s * kStage;
        mbar_arrive_tx(full + s, kStage);
        load_operand(st, a.p_mn, f0, kPRows, b, a.block_k,
                     [&](void *d, int x, int y) { tma_load_2d(d, mp, x, y, full + s); });
        load_operand(st + kPBytes, a.q_mn, r0, BN, b, a.block_k,
                     [&](void *d, int x, int y) { tma_load_2d(d, mq, x, y, full + s); });
      }
    }
  } else if (warp == 5) {
    const uint64_t p_first = stage_desc(smem_u32(ring), a.p_mn),
                   q_first = stage_desc(smem_u32(ring) + kPBytes, a.q_mn);
    const uint32_t p_step = slice_step(a.p_mn), q_step = slice_step(a.q_mn);
    RingPlace<kStages> at;
    int b = b0;
    for (; b < b1; ++b, at.next()) {
      const int s = at.stage;
      if (!__all_sync(0xffffffffu, mbar_wait(full + s, at.full(), abort_flag, kWaitFull))) break;
      fence_after_sync();
      const uint64_t pd = p_first + s * (kStage / 16), qd = q_first + s * (kStage / 16);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma<1, CODES>(tmem, pd + k * p_step, qd + k * q_step, a.idesc, (b > b0 || k > 0) ? 1u : 0u);
        mma_commit(empty + s);
      }
      __syncwarp();
    }
    if (elect_one()) {
      if (WITHHOLD && blockIdx.x == 0) mbar_wait(done, 0, abort_flag, kWaitAccFull, kTestPollLimit);
      mma_commit(done);
      volatile int keep = 0;  // wait for the issued MMAs even when another role gave up
      if (!mbar_wait(done, 0, &keep, kWaitDrain)) *abort_flag = kWaitDrain;
      // copies that nobody waited for land before the CTA leaves
      for (; b < b1; ++b, at.next())
        if (!mbar_wait(full + at.stage, at.full(), &keep, kWaitFull)) break;
    }
  }
  __syncwarp();
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const bool ok = *abort_flag == 0;
  const int nr = min(BN, a.Q - r0);  // output rows of the tile
  // sums, [row][feature], over the ring: its copies have landed and its MMAs have
  // read it
  float *sums = reinterpret_cast<float *>(ring);
  constexpr int kN = BN < 32 ? BN : 32;
  for (int c = (warp >> 2) * kN; c < nr; c += kSplitThreads / 128 * kN) {
    const int lanes = (warp & 3) * 32;
    float z[kN];
    if constexpr (kN == 16)
      tmem_load16(tmem + ((uint32_t)lanes << 16) + c, z);
    else
      tmem_load32(tmem + ((uint32_t)lanes << 16) + c, z);
    tmem_load_wait();
#pragma unroll
    for (int j = 0; j < kN; ++j) sums[(c + j) * kPRows + lanes + lane] = z[j];
  }
  __syncwarp();
  if (splits > 1)
    cluster_sync();
  else
    __syncthreads();
  // CTA k of a cluster finishes rows k, k + splits, ..., shared out among its warps
  if (ok)
    finish_rows<false>(a.e, smem_u32(sums), splits, f0, a.P, r0, rank + splits * warp,
                       splits * (kSplitThreads / 32), nr, [](int, int, float *) {});
  __syncwarp();
  if (splits > 1) cluster_sync();  // until every peer has read this CTA's sums
  if (!ok && threadIdx.x == 0) atomicCAS(&g_wait_error, 0, *abort_flag | (int)(blockIdx.x << 4));
  fence_before_sync();
  __syncthreads();
  if (warp == 4) {
    fence_after_sync();
    tmem_free<1>(tmem, kColumns);
  }
}

// ------------------------------------------------------------- pair kernel

constexpr int kPairEpilogueWarps = 8;
constexpr int kPairThreads = 32 * (kPairEpilogueWarps + 2);

template <int BN>
constexpr int kPairStages = kRing / (kPBytes + BN / 2 * 128);
template <int BN>
constexpr size_t kPairSmem = (size_t)kPairStages<BN> * (kPBytes + BN / 2 * 128) + 1024 + 512;

template <int BN, bool CODES, bool WITHHOLD>
__global__ void __launch_bounds__(kPairThreads, 1)
    gemm_pair_kernel(const __grid_constant__ TcArgs a, const __grid_constant__ CUtensorMap mp,
                     const __grid_constant__ CUtensorMap mq) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  unsigned char *ring = reinterpret_cast<unsigned char *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  constexpr int kStages = kPairStages<BN>, kQRows = BN / 2, kStage = kPBytes + kQRows * 128;
  constexpr uint32_t kColumns = 2 * BN;
  uint64_t *full = reinterpret_cast<uint64_t *>(ring + kStages * kStage), *empty = full + kStages;
  uint64_t *dfull = empty + kStages, *dfree = dfull + 2, *drain = dfree + 2;
  uint32_t *holder = reinterpret_cast<uint32_t *>(drain + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(holder + 1);
  volatile int *consumed = abort_flag + 1;

  // the same in all lanes, and known to be: what the MMA warp computes then stays in
  // uniform registers, where its instructions want their operands
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int tiles = a.tiles_p * a.tiles_q, first = blockIdx.x / 2, stride = gridDim.x / 2;
  const bool withheld = WITHHOLD && first == 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(dfull + b, 1);
      mbar_init(dfree + b, 2 * kPairEpilogueWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    *consumed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kPairEpilogueWarps) tmem_alloc<2>(holder, kColumns);
  fence_before_sync();
  __syncthreads();
  cluster_sync();  // the peer's barriers are ready
  fence_after_sync();
  const uint32_t tmem = *holder;

  if (warp == kPairEpilogueWarps) {
    if (lane == 0) {
      // copies of this CTA's half, complete on the leader's barrier
      RingPlace<kStages> at;
      bool go = true;
      for (int t = first; t < tiles && go; t += stride) {
        int tp, tq;
        tile_of(t, a.tiles_p, a.tiles_q, &tp, &tq);
        const int f0 = tp * 2 * kPRows + (int)rank * kPRows, r0 = tq * BN + (int)rank * kQRows;
        for (int b = 0; b < a.blocks; ++b, at.next()) {
          const int s = at.stage;
          if (!mbar_wait(empty + s, at.empty(), abort_flag, kWaitEmpty)) {
            go = false;
            break;
          }
          unsigned char *st = ring + s * kStage;
          const uint32_t bar = cluster_map(smem_u32(full + s), 0);
          if (rank == 0) mbar_arrive_tx(full + s, 2 * kStage);
          load_operand(st, a.p_mn, f0, kPRows, b, a.block_k,
                       [&](void *d, int x, int y) { tma_load_2d_pair(d, &mp, x, y, bar); });
          load_operand(st + kPBytes, a.q_mn, r0, kQRows, b, a.block_k,
                       [&](void *d, int x, int y) { tma_load_2d_pair(d, &mq, x, y, bar); });
        }
      }
    }
  } else if (warp == kPairEpilogueWarps + 1) {
    if (rank == 0) {
      const uint64_t p_first = stage_desc(smem_u32(ring), a.p_mn),
                     q_first = stage_desc(smem_u32(ring) + kPBytes, a.q_mn);
      const uint32_t p_step = slice_step(a.p_mn), q_step = slice_step(a.q_mn);
      RingPlace<kStages> at;
      RingPlace<2> acc;  // of the accumulators
      int g = 0;
      bool go = true;
      for (int t = first; t < tiles && go; t += stride, acc.next()) {
        const int buf = acc.stage;
        if (!__all_sync(0xffffffffu, mbar_wait(dfree + buf, acc.empty(), abort_flag, kWaitAccFree))) break;
        fence_after_sync();
        for (int b = 0; b < a.blocks; ++b, ++g, at.next()) {
          const int s = at.stage;
          if (!__all_sync(0xffffffffu, mbar_wait(full + s, at.full(), abort_flag, kWaitFull))) {
            go = false;
            break;
          }
          fence_after_sync();
          const uint64_t pd = p_first + s * (kStage / 16), qd = q_first + s * (kStage / 16);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma<2, CODES>(tmem + buf * BN, pd + k * p_step, qd + k * q_step, a.idesc,
                            (b > 0 || k > 0) ? 1u : 0u);
            mma_commit_pair(empty + s);
          }
          __syncwarp();
        }
        if (go && !withheld && elect_one()) mma_commit_pair(dfull + buf);
        __syncwarp();
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
  } else {
    RingPlace<2> acc;
    bool go = true;
    if (withheld) go = __all_sync(0xffffffffu, mbar_wait(dfull, 0, abort_flag, kWaitAccFull, kTestPollLimit));
    for (int t = first; t < tiles && go; t += stride, acc.next()) {
      int tp, tq;
      tile_of(t, a.tiles_p, a.tiles_q, &tp, &tq);
      const int buf = acc.stage, quarter = warp & 3, half = warp >> 2;
      const int f0 = tp * 2 * kPRows + (int)rank * kPRows, f = f0 + quarter * 32 + lane;
      const int r0 = tq * BN + half * (BN / 2);
      const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + buf * BN + half * (BN / 2);
      // the tile's MMAs are still under way: its residual comes to L2 meanwhile
      prefetch_residual(a.e, f0, a.P, kPRows, r0, a.Q, BN / 2, threadIdx.x & 127, 128);
      // 16 rows at a time: of 8192 x 4096 outputs with gelu and residual, 107 us
      // against 121 with 32, which leave the compiler short of registers
#pragma unroll 1
      for (int c = 0; c < BN / 2 && go; c += 16) {
        go = finish<16, false>(a.e, f, r0 + c, f < a.P ? a.Q - r0 - c : 0, [&](float *z) {
          if (c == 0) {
            const bool full_now = mbar_wait(dfull + buf, acc.full(), abort_flag, kWaitAccFull);
            if (!__all_sync(0xffffffffu, full_now)) return false;
            fence_after_sync();
          }
          tmem_load16(from + c, z);
          tmem_load_wait();
          if (c + 16 == BN / 2) {  // the accumulator is read: free it for the tile after next
            fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_relaxed_at(cluster_map(smem_u32(dfree + buf), 0));
          }
          return true;
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
      for (int g = *consumed, n = 0; n < kStages; ++g, ++n)
        if (!mbar_wait(full + g % kStages, (uint32_t)((g / kStages) & 1), &keep, kWaitFull, 1 << 16)) break;
    }
    atomicCAS(&g_wait_error, 0, *abort_flag | (int)(blockIdx.x << 4));
  }
  __syncthreads();
  cluster_sync();
  if (warp == kPairEpilogueWarps) tmem_free<2>(tmem, kColumns);
}

// ------------------------------------------------------------------- host

// A tensor map of an operand (rows x K values): boxes of 128 bytes of k by
// box_rows rows, or of 64 rows by 64 values of k where it lies along its rows.
vcsr_status make_map(CUtensorMap *m, const Operand &o, int64_t rows, int64_t K, int dtype, int box_rows) {
  EncodeTiledFn enc;
  VCSR_TRY(tensor_map_encoder(&enc));
  const size_t size = type_size(dtype);
  const cuuint64_t dims[2] = {(cuuint64_t)(o.transposed ? rows : K), (cuuint64_t)(o.transposed ? K : rows)};
  const cuuint64_t strides[1] = {(cuuint64_t)o.ld * size};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / size), (cuuint32_t)(o.transposed ? 64 : box_rows)};
  const cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType type = dtype == VCSR_BF16  ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                   : dtype == VCSR_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                       : CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const CUresult r = enc(m, type, 2, const_cast<void *>(o.p), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(VCSR_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return VCSR_OK;
}

template <int BN>
const void *split_kernel(int dtype) {
  return dtype == VCSR_E4M3 ? reinterpret_cast<const void *>(gemm_split_kernel<BN, true, false>)
                            : reinterpret_cast<const void *>(gemm_split_kernel<BN, false, false>);
}

TcArgs args_of(const Gemm &g) {
  TcArgs a{};
  a.P = (int)g.N;
  a.Q = (int)g.M;
  a.block_k = 128 / (int)type_size(g.dtype);
  a.blocks = (int)ceil_div(g.K, a.block_k);
  a.p_mn = g.b.transposed;
  a.q_mn = g.a.transposed;
  a.e = g.e;
  return a;
}

template <int BN>
int64_t split_tiles(const Gemm &g) {
  return ceil_div(g.N, kPRows) * ceil_div(g.M, BN);
}

// How many CTAs share a tile's k: of one product, or of two of one type in one launch.
template <int BN>
int splits_of(const Gemm &g, const Gemm *g1) {
  const int64_t tiles = split_tiles<BN>(g) + (g1 ? split_tiles<BN>(*g1) : 0);
  const int b0 = args_of(g).blocks;
  return choose_splits(split_kernel<BN>(g.dtype), kSplitThreads, kSplitSmem<BN>, tiles,
                       g1 ? std::min(b0, args_of(*g1).blocks) : b0);
}

// One product, or two of one type (g1).
template <int BN>
vcsr_status launch_split(const Gemm &g, const Gemm *g1, int splits, cudaStream_t st) {
  SplitJobs jobs{};
  int64_t tiles = 0;
  for (int i = 0; i < (g1 ? 2 : 1); ++i) {
    const Gemm &gi = i ? *g1 : g;
    TcArgs &a = jobs.a[i];
    a = args_of(gi);
    VCSR_TRY(make_map(&jobs.p[i], gi.b, gi.N, gi.K, gi.dtype, kPRows));
    VCSR_TRY(make_map(&jobs.q[i], gi.a, gi.M, gi.K, gi.dtype, BN));
    a.tiles_p = (int)ceil_div(a.P, kPRows);
    a.tiles_q = (int)ceil_div(a.Q, BN);
    a.idesc = instr_desc(gi.dtype == VCSR_BF16 ? 1 : 0, a.p_mn, a.q_mn, 128, BN);
    tiles += split_tiles<BN>(gi);
    if (i == 0) jobs.second = tiles > 0x7fffffffll ? 0x7fffffff : (int)tiles;
  }
  jobs.splits = splits;
  if (tiles * jobs.splits > 0x7fffffffll) return fail(VCSR_ERR_RANGE, "more than 2^31 - 1 thread blocks");
  const int grid = (int)(tiles * jobs.splits);
  const bool withhold = take_withhold(), codes = g.dtype == VCSR_E4M3;
  const auto kernel = withhold ? (codes ? gemm_split_kernel<BN, true, true> : gemm_split_kernel<BN, false, true>)
                               : (codes ? gemm_split_kernel<BN, true, false> : gemm_split_kernel<BN, false, false>);
  return launch(kernel, grid, kSplitThreads, kSplitSmem<BN>, jobs.splits, st, jobs);
}

// Expected microseconds, to choose between the kernels: a launch, then for every round
// of tiles on the GPU a fixed part (filling the pipeline, the epilogue) and a part per
// stage of k.  Fitted to 200 products of 1 to 4096 rows, 128 to 4096 features and k of
// 128 to 4096 (bf16, bias, silu and residual) in each kernel; within about 10% of them.
// Some of them, split kernel with 16 / 32 / 64 / 128 rows and pair kernel: 16 x 4096,
// k = 4096: 10.9 / 10.9 / 11.1 / 11.3 / 27.5; 64 x 2048, k = 512: 7.1 / 6.7 / 6.9 / 7.3 /
// 11.0; 512 x 1024, k = 1024: - / - / 9.4 / 10.0 / 16.5; 1024 x 4096, k = 1024: - / - /
// 41.3 / 25.5 / 17.2.
template <int BN>
double split_cost(const Gemm &g, const Gemm *g1 = nullptr) {
  constexpr double kFixed = BN == 16 ? 3.8 : BN == 32 ? 4.2 : BN == 64 ? 5.0 : 7.0;
  constexpr double kStage = BN == 16 ? 0.29 : BN == 128 ? 0.36 : 0.32;
  // boxes along the operand's own index are 64 rows
  if (BN < 64 && (g.a.transposed || (g1 && g1->a.transposed))) return 1e30;
  const int64_t tiles = split_tiles<BN>(g) + (g1 ? split_tiles<BN>(*g1) : 0);
  const int64_t b0 = args_of(g).blocks, b1 = g1 ? args_of(*g1).blocks : b0;
  const int splits = splits_of<BN>(g, g1);
  if (g1 && tiles * splits > sm_count()) return 1e30;  // two products share one round or none
  return 1.2 + (splits > 1 ? 0.7 : 0.0) +
         (double)ceil_div(tiles * splits, sm_count()) * (kFixed + kStage * (double)ceil_div(std::max(b0, b1), splits));
}
double pair_cost(const Gemm &g) {
  const int blocks = args_of(g).blocks;
  const int64_t rounds = ceil_div(ceil_div(g.N, 256) * ceil_div(g.M, 256), sm_count() / 2);
  return 11.5 + 0.33 * blocks + (double)(rounds - 1) * std::max(8.0, 0.42 * blocks);
}

template <int BN>
vcsr_status launch_pair(const Gemm &g, cudaStream_t st) {
  TcArgs a = args_of(g);
  CUtensorMap mp, mq;
  VCSR_TRY(make_map(&mp, g.b, g.N, g.K, g.dtype, kPRows));
  VCSR_TRY(make_map(&mq, g.a, g.M, g.K, g.dtype, BN / 2));
  a.tiles_p = (int)ceil_div(a.P, 2 * kPRows);
  a.tiles_q = (int)ceil_div(a.Q, BN);
  const int64_t tiles = (int64_t)a.tiles_p * a.tiles_q;
  if (tiles > (1 << 30)) return fail(VCSR_ERR_RANGE, "more than 2^30 output tiles");
  const int grid = 2 * (int)std::min<int64_t>(tiles, sm_count() / 2);
  const int format = g.dtype == VCSR_BF16 ? 1 : 0;
  a.idesc = instr_desc(format, a.p_mn, a.q_mn, 256, BN);
  const bool withhold = take_withhold(), codes = g.dtype == VCSR_E4M3;
  const auto kernel = withhold ? (codes ? gemm_pair_kernel<BN, true, true> : gemm_pair_kernel<BN, false, true>)
                               : (codes ? gemm_pair_kernel<BN, true, false> : gemm_pair_kernel<BN, false, false>);
  return launch(kernel, grid, kPairThreads, kPairSmem<BN>, 2, st, a, mp, mq);
}

std::atomic<bool> g_withhold{false};

}  // namespace

bool take_withhold() { return g_withhold.load(std::memory_order_relaxed) && g_withhold.exchange(false); }
void set_withhold() { g_withhold.store(true); }

bool tc_aligned(const void *p, int64_t ld, int dtype) {
  return aligned(p, 16) && (ld * (int64_t)type_size(dtype)) % 16 == 0;
}

namespace {

struct Choice {
  int kernel;  // 0 to 3: split, 16 to 128 rows; 4: pair
  double cost;
};
Choice choose(const Gemm &g) {
  const double costs[5] = {split_cost<16>(g), split_cost<32>(g), split_cost<64>(g), split_cost<128>(g), pair_cost(g)};
  const int best = (int)(std::min_element(costs, costs + 5) - costs);
  return {best, costs[best]};
}
vcsr_status launch_chosen(const Choice &c, const Gemm &g, cudaStream_t st) {
  switch (c.kernel) {
    case 0: return launch_split<16>(g, nullptr, splits_of<16>(g, nullptr), st);
    case 1: return launch_split<32>(g, nullptr, splits_of<32>(g, nullptr), st);
    case 2: return launch_split<64>(g, nullptr, splits_of<64>(g, nullptr), st);
    case 3: return launch_split<128>(g, nullptr, splits_of<128>(g, nullptr), st);
    default: return launch_pair<256>(g, st);
  }
}

}  // namespace

vcsr_status launch_gemm_tc(const Gemm &g, cudaStream_t st) { return launch_chosen(choose(g), g, st); }

vcsr_status launch_gemms_tc(const Gemm &g0, const Gemm &g1, cudaStream_t st) {
  if (!g0.e.out && !g1.e.out) return VCSR_OK;
  const Choice c0 = choose(g0), c1 = choose(g1);
  const double both64 = split_cost<64>(g0, &g1), both128 = split_cost<128>(g0, &g1);
  const bool narrow = both64 <= both128;
  // two microseconds for the launch that one call saves on the host
  if (std::min(both64, both128) < c0.cost + c1.cost + 2.0) {
    const int splits = narrow ? splits_of<64>(g0, &g1) : splits_of<128>(g0, &g1);
    // one of them alone is summed as it is beside the other: the same result
    const Gemm &first = g0.e.out ? g0 : g1;
    const Gemm *second = g0.e.out && g1.e.out ? &g1 : nullptr;
    return narrow ? launch_split<64>(first, second, splits, st) : launch_split<128>(first, second, splits, st);
  }
  if (g0.e.out) VCSR_TRY(launch_chosen(c0, g0, st));
  if (g1.e.out) VCSR_TRY(launch_chosen(c1, g1, st));
  return VCSR_OK;
}

int cluster_slots(const void *kernel, int threads, size_t smem, int size) {
  struct Known {
    const void *kernel;
    int dev, size, slots;
  };
  static std::mutex mu;
  static std::vector<Known> known;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  std::lock_guard<std::mutex> lk(mu);
  for (const Known &k : known)
    if (k.kernel == kernel && k.dev == dev && k.size == size) return k.slots;
  if (allow_shared(kernel, smem) != VCSR_OK) return 0;
  cudaLaunchConfig_t c{};
  c.gridDim = dim3((unsigned)size);
  c.blockDim = dim3((unsigned)threads);
  c.dynamicSmemBytes = smem;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)size;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  c.attrs = at;
  c.numAttrs = 1;
  int slots = 0;
  if (cudaOccupancyMaxActiveClusters(&slots, kernel, &c) != cudaSuccess) {
    cudaGetLastError();
    slots = 0;
  }
  known.push_back({kernel, dev, size, slots});
  return slots;
}

vcsr_status check_waits(cudaStream_t st) {
  VCSR_CUDA(cudaStreamSynchronize(st));
  int word = 0, zero = 0;
  VCSR_CUDA(cudaMemcpyFromSymbol(&word, g_wait_error, sizeof(int)));
  if (word) VCSR_CUDA(cudaMemcpyToSymbol(g_wait_error, &zero, sizeof(int)));
  if (!word) VCSR_TRY(take_wait_error_f32(&word));
  if (!word) return VCSR_OK;
  char text[128];
  describe_tc_error(word, text, sizeof(text));
  return fail(VCSR_ERR_TIMEOUT, "%s", text);
}

}  // namespace layer
}  // namespace vcsr

extern "C" vcsr_status vcsr_layers_test_withhold_signal(void) {
  vcsr::clear_error();
  vcsr::layer::set_withhold();
  return VCSR_OK;
}

extern "C" vcsr_status vcsr_layers_check(vcsr_stream_t stream) {
  vcsr::clear_error();
  return vcsr::no_throw([&] { return vcsr::layer::check_waits((cudaStream_t)stream); });
}
