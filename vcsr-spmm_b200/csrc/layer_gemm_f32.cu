// layer_gemm_f32.cu — the product of FP32 operands on the tensor cores at FP32
// accuracy (tcgen05 kind::f16 on bfloat16 parts).
//
// An FP32 value is the exact sum of three bfloat16 values, its leading, middle and last
// 8 significant bits (cut off, not rounded, so that the leading part never overflows).
// Of the nine products of two values' parts the six down to 2^-16 of the largest are
// summed; the three left out are below 2^-24 of it.  A tensor core may cut its sums off,
// not round them, so no sum is long: each 32 values of k start a new accumulator in
// tensor memory, smallest products first, and the epilogue's warps add the accumulators
// in registers, rounded to nearest.  An output that comes out NaN or infinite (a product
// of an infinity's zero parts is NaN) is summed again in FP32 from the operands
// themselves, by the warps that drain: where k is long that outlasts the other roles'
// bounded waits, which therefore start anew while a count of such sums goes on rising.
// Values below 2^-110 lose bits under 2^-133, the least bfloat16.
//
// Tile: 128 features x 32, 64 or 128 rows per CTA (layer_gemm_tc.cu says why
// features are the MMA's M side), 32 values of k per stage.  One thread brings the
// FP32 tiles in by TMA (128-byte rows, 128-byte swizzle); eight warps split them into
// three parts, the features' into tensor memory, where the MMAs take their M side from
// (a third of the shared-memory traffic gone), the rows' into planes of shared memory
// in the order the MMAs read (stored along k: 64-byte rows, 64-byte swizzle; along the
// operand's own index: 128-byte rows of 64 values); one thread issues 12 MMAs per stage;
// four to sixteen warps drain the accumulators, three or four of which take turns.  All
// roles run at once.  Bound by the splitting warps' instructions: 0.5 to 0.9 us a stage,
// of which the MMAs take 0.4 (128 x 128).  Two groups of splitting warps that take
// stages in turn were no faster (255 against 239 us, 4096 x 4096, k = 1024).
// Persistent over tiles; where tiles are too few for the SMs, clusters of 2 to 8 CTAs
// split k and join their sums in rank order through distributed shared memory.
// 4096 x 4096, k = 1024: 214 to 219 us, 157 to 160 TFLOP/s; 16 x 4096, k = 4096: 28 us, 2.4 TB/s
// (22 with w in L2); 62451 x 128, k = 128 with every part of the epilogue: 33 us, 3.9 TB/s.
// Registers are short at 832 threads a CTA (72 each, 726 bytes spilled a thread; tiles of 64
// rows 96 and 186, of 32 none).
#include <algorithm>

#include "layer_gemm_tc.cuh"
#include "spmm_tc.h"

namespace vcsr {
namespace layer {
namespace {

using namespace tc;

constexpr int kRows = 128;  // features per tile
constexpr int kK = 32;      // values of k per stage
// Warps: eight split, BN / 8 drain (32 lanes by 32 columns each), one loads, one
// issues MMAs.
constexpr int kSplitters = 8;
template <int BN>
constexpr int kDraining = BN / 8;
template <int BN>
constexpr int kThreads = 32 * (kSplitters + kDraining<BN> + 2);
constexpr int kPart = kK / 2;   // tensor-memory columns of one part of P's tile

// Bytes and counts of the FP32 stages and of the split ones.
template <int BN>
constexpr int kRaw = (kRows + BN) * kK * 4;
template <int BN>
constexpr int kSplit = 3 * BN * kK * 2;
template <int BN>
constexpr int kRaws = BN == 128 ? 5 : BN == 64 ? 6 : 8;
template <int BN>
constexpr int kSplits = BN == 128 ? 2 : 4;
// Accumulators, as many as tensor memory holds beside P's parts: the next tile's first
// stages are multiplied while the draining warps are in this one's epilogue.
template <int BN>
constexpr int kSums = BN == 128 ? 3 : 4;
constexpr int kColumns = 512;  // of tensor memory; one CTA an SM
static_assert(kSums<128> * 128 + kSplits<128> * 3 * kPart <= kColumns, "");
static_assert(kSums<64> * 64 + kSplits<64> * 3 * kPart <= kColumns, "");
template <int BN>
constexpr size_t kSmem = (size_t)kRaws<BN> * kRaw<BN> + kSplits<BN> * kSplit<BN> + 1024 + 512;

__device__ int g_wait_error = 0;

struct F32Args {
  const float *p, *q;
  int64_t ldp, ldq;
  int P, Q, K;
  int stages;      // of 32 values of k
  int p_mn, q_mn;  // operand stored along its own index
  int tiles_p, tiles_q, splits;
  Epilogue e;
};

// Copies of one FP32 tile (`rows` by 32 k) to `dst`: a box of 128-byte rows of k,
// or boxes of 32 rows by 32 k, a 128-byte row per k, 4 KB each.
__device__ __forceinline__ void load_raw(unsigned char *dst, const CUtensorMap *m, int mn, int row0, int rows,
                                         int k0, uint64_t *bar) {
  if (mn) {
    for (int c = 0; c < rows; c += 32) tma_load_2d(dst + c * 128, m, row0 + c, k0, bar);
  } else {
    tma_load_2d(dst, m, k0, row0, bar);
  }
}

// Two values' leading 16 bits as one word.
__device__ __forceinline__ uint32_t pair(float lo, float hi) {
  return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
}
// Takes both from the values, exactly.
__device__ __forceinline__ void take_leading(uint32_t p, float &lo, float &hi) {
  constexpr unsigned short kMinusOne = 0xbf80;
  asm("{ .reg .b16 l, h; mov.b32 {l, h}, %2; fma.rn.f32.bf16 %0, l, %3, %0; fma.rn.f32.bf16 %1, h, %3, %1; }"
      : "+f"(lo), "+f"(hi)
      : "r"(p), "h"(kMinusOne));
}
// The leading parts of 2 N values, which are left with the rest.  The 16-bit operands
// save the masks that would widen them: the split bounds a stage (1.01 us with masks,
// 0.83 without, tiles of 128 rows).
template <int N>
__device__ __forceinline__ void cut(float *v, uint32_t *p) {
#pragma unroll
  for (int j = 0; j < N; ++j) p[j] = pair(v[2 * j], v[2 * j + 1]);
#pragma unroll
  for (int j = 0; j < N; ++j) take_leading(p[j], v[2 * j], v[2 * j + 1]);
}

// The 16 values of v in three parts to `column` (of this warp's 32 lanes) and kPart,
// 2 kPart further.
__device__ __forceinline__ void parts_to_tmem(uint32_t column, float *v) {
#pragma unroll
  for (int part = 0; part < 3; ++part) {
    uint32_t p[8];
    cut<8>(v, p);
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(
                     column + part * kPart),
                 "r"(p[0]), "r"(p[1]), "r"(p[2]), "r"(p[3]), "r"(p[4]), "r"(p[5]), "r"(p[6]), "r"(p[7])
                 : "memory");
  }
}

// Splits P's tile of 128 rows by 32 values of k from `raw` to tensor memory, a row per
// lane.  Warps w and w + 4 take the rows whose lanes they reach, 16 values of k each.
__device__ __forceinline__ void split_p(uint32_t raw, uint32_t column, int mn, int warp, int lane) {
  const int quarter = warp & 3, half = warp >> 2;
  float v[16];
  if (mn) {  // boxes of 32 rows: a 128-byte row per k
    const uint32_t box = raw + quarter * 4096 + (lane & 3) * 4;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int k = half * 16 + j;
      asm volatile("ld.shared.f32 %0, [%1];"
                   : "=f"(v[j])
                   : "r"(box + k * 128 + (((lane >> 2) ^ (k & 7)) << 4)));
    }
  } else {
    const int row = quarter * 32 + lane;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(v[4 * c]), "=f"(v[4 * c + 1]), "=f"(v[4 * c + 2]), "=f"(v[4 * c + 3])
                   : "r"(raw + row * 128 + (((half * 4 + c) ^ (row & 7)) << 4)));
  }
  parts_to_tmem(column + ((uint32_t)(quarter * 32) << 16) + half * 8, v);
}

// Splits Q's tile, ROWS (a multiple of 64, or 32) by 32 values of k, from `raw`
// to three planes, `plane` bytes apart, from `out` on.  A thread takes 8 values
// that are neighbours in memory: two 16-byte pieces in, one per plane out.  In both
// orders 8 neighbouring lanes touch all banks once.
template <int ROWS>
__device__ __forceinline__ void split_tile(uint32_t raw, uint32_t out, int mn, int t) {
  constexpr int kPlaneBytes = ROWS * kK * 2;
#pragma unroll
  for (int u = 0; u < (ROWS + 63) / 64; ++u) {
    uint32_t in0, in1, at;
    int swap = 0;
    if (mn) {  // row k of 128 bytes: boxes of 32 values in, chunks of 64 out
      const int k = t >> 3, c = t & 7;
      const uint32_t box = raw + (u * 2 + (c >> 2)) * 4096 + k * 128;
      swap = c >> 2;  // the two boxes of a chunk take their pieces in turn
      in0 = box + (((2 * (c & 3) + swap) ^ (k & 7)) << 4);
      in1 = box + (((2 * (c & 3) + 1 - swap) ^ (k & 7)) << 4);
      at = out + u * 4096 + k * 128 + ((c ^ (k & 7)) << 4);
    } else {  // rows of 128 bytes in, of 64 bytes out
      const int r = u * 64 + (t >> 2), c = t & 3;
      if (ROWS < 64 && r >= ROWS) break;
      in0 = raw + r * 128 + (((2 * c) ^ (r & 7)) << 4);
      in1 = raw + r * 128 + (((2 * c + 1) ^ (r & 7)) << 4);
      at = out + r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
    }
    float v[8];
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
                 : "r"(in0));
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "r"(in1));
    if (mn) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float first = v[j];
        v[j] = swap ? v[4 + j] : first;
        v[4 + j] = swap ? first : v[4 + j];
      }
    }
#pragma unroll
    for (int part = 0; part < 3; ++part) {
      uint32_t p[4];
      cut<4>(v, p);
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + part * kPlaneBytes), "r"(p[0]),
                   "r"(p[1]), "r"(p[2]), "r"(p[3])
                   : "memory");
    }
  }
}

// Descriptor of the first 16 values of k of a plane; the second 16 and the other
// planes are further by their distance in 16-byte units.
__device__ __forceinline__ uint64_t plane_desc(uint32_t addr, int mn) {
  return mn ? smem_desc(addr, 4096, 1024, 2) : smem_desc(addr, 16, 512, 4);
}

// The sum of an output, in order.  `alive` tells the waits of the other roles that it is
// under way, often enough for loads that all come from memory.
__device__ __noinline__ float sum_again(const F32Args &a, int f, int r, int *alive) {
  float s = 0.0f;
  for (int64_t k = 0; k < a.K && s == s; ++k) {
    if (k % 4096 == 0) atomicAdd(alive, 1);
    s = fmaf(a.q_mn ? a.q[k * a.ldq + r] : a.q[r * a.ldq + k],
             a.p_mn ? a.p[k * a.ldp + f] : a.p[f * a.ldp + k], s);
  }
  return s;
}

// Sums that are not finite made anew, those that IN(j) names.
template <int N, class IN, class AGAIN>
__device__ __forceinline__ void mend(float *z, IN &&in, AGAIN &&again) {
  float total = 0.0f;  // not finite where a sum is not (or where finite ones add up to that)
#pragma unroll
  for (int j = 0; j < N; ++j) total += fabsf(z[j]);
  if (total <= 3.402823466e38f) return;
  float copy[N];
#pragma unroll
  for (int j = 0; j < N; ++j) copy[j] = z[j];
#pragma unroll 1
  for (int j = 0; j < N; ++j)
    if (in(j) && !(fabsf(copy[j]) <= 3.402823466e38f)) copy[j] = again(j);
#pragma unroll
  for (int j = 0; j < N; ++j) z[j] = copy[j];
}

// The epilogue of N rows of column f.
template <int N, class GET>
__device__ __forceinline__ void finish_f32(const F32Args &a, int f, int r0, int n, int *alive, GET &&get) {
  if (f >= a.P) n = 0;
  finish<N, true>(a.e, f, r0, n, [&](float *z) {
    get(z);
    if (n > 0) mend<N>(z, [&](int j) { return j < n; }, [&](int j) { return sum_again(a, f, r0 + j, alive); });
    return true;
  });
}

// WITHHOLD (a test): the first block waits for a signal that is not sent.  A kernel of its
// own, since the branches alone cost this one registers (62451 x 128, k = 128 30 -> 34 us).
template <int BN, bool WITHHOLD>
__global__ void __launch_bounds__(kThreads<BN>, 1) gemm_f32_kernel(const __grid_constant__ F32Args a,
                                                             const __grid_constant__ CUtensorMap mp,
                                                             const __grid_constant__ CUtensorMap mq) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  unsigned char *ring = reinterpret_cast<unsigned char *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  constexpr int R = kRaws<BN>, S = kSplits<BN>;
  constexpr int kLoadWarp = kSplitters + kDraining<BN>, kMmaWarp = kLoadWarp + 1;
  unsigned char *raw = ring + S * kSplit<BN>;
  uint64_t *full = reinterpret_cast<uint64_t *>(raw + R * kRaw<BN>), *empty = full + S;
  uint64_t *rfull = empty + S, *rempty = rfull + R;
  uint64_t *dfull = rempty + R, *dfree = dfull + kSums<BN>, *drain = dfree + kSums<BN>;
  uint32_t *holder = reinterpret_cast<uint32_t *>(drain + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(holder + 1);
  int *alive = reinterpret_cast<int *>(holder + 2);  // rises while sums are made again

  // the same in all lanes, and known to be: what the MMA warp computes then stays in
  // uniform registers, where its instructions want their operands
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = a.splits > 1 ? (int)cluster_rank() : 0;
  const int tiles = a.tiles_p * a.tiles_q, first = blockIdx.x / a.splits, stride = gridDim.x / a.splits;
  const int b0 = (int)((int64_t)a.stages * rank / a.splits), b1 = (int)((int64_t)a.stages * (rank + 1) / a.splits);
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full + s, kSplitters);
      mbar_init(empty + s, 1);
    }
    for (int s = 0; s < R; ++s) {
      mbar_init(rfull + s, 1);
      mbar_init(rempty + s, kSplitters);
    }
    for (int b = 0; b < kSums<BN>; ++b) {
      mbar_init(dfull + b, 1);
      mbar_init(dfree + b, kDraining<BN>);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    *alive = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) tmem_alloc<1>(holder, kColumns);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = *holder, p_parts = tmem + kSums<BN> * BN;

  float acc[32];  // draining warps
#pragma unroll
  for (int j = 0; j < 32; ++j) acc[j] = 0.0f;
  const int drainer = warp - kSplitters, quarter = drainer & 3, col0 = (drainer >> 2) * 32;

  if (warp < kSplitters) {
    RingPlace<R> in;
    RingPlace<S> out;
    bool go = true;
    for (int t = first; t < tiles && go; t += stride) {
      for (int b = b0; b < b1; ++b, in.next(), out.next()) {
        const int r = in.stage, s = out.stage;
        const bool ready = mbar_wait<true>(rfull + r, in.full(), abort_flag, kWaitFull) &&
                           mbar_wait<true>(empty + s, out.empty(), abort_flag, kWaitEmpty);
        if (!__all_sync(0xffffffffu, ready)) {
          go = false;
          break;
        }
        fence_after_sync();
        const uint32_t from = smem_u32(raw + r * kRaw<BN>), to = smem_u32(ring + s * kSplit<BN>);
        split_p(from, p_parts + s * 3 * kPart, a.p_mn, warp, lane);
        split_tile<BN>(from + kRows * kK * 4, to, a.q_mn, threadIdx.x);
        // the MMAs read what was written by plain stores, and to tensor memory
        fence_async();
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(full + s);
          mbar_arrive(rempty + r);
        }
      }
    }
  } else if (warp == kLoadWarp) {
    if (lane == 0) {
      int g = 0;
      bool go = true;
      for (int t = first; t < tiles && go; t += stride) {
        int tp, tq;
        tile_of(t, a.tiles_p, a.tiles_q, &tp, &tq);
        for (int b = b0; b < b1; ++b, ++g) {
          const int r = g % R;
          if (g >= R && !mbar_wait<true>(rempty + r, (uint32_t)((g / R - 1) & 1), abort_flag, kWaitEmpty)) {
            go = false;
            break;
          }
          unsigned char *to = raw + r * kRaw<BN>;
          mbar_arrive_tx(rfull + r, kRaw<BN>);
          load_raw(to, &mp, a.p_mn, tp * kRows, kRows, b * kK, rfull + r);
          load_raw(to + kRows * kK * 4, &mq, a.q_mn, tq * BN, BN, b * kK, rfull + r);
        }
      }
      // every copy lands before the CTA leaves, whoever gave up
      volatile int keep = 0;
      for (int n = max(0, g - R); n < g; ++n)
        mbar_wait(rfull + n % R, (uint32_t)((n / R) & 1), &keep, kWaitFull);
    }
  } else if (warp == kMmaWarp) {
    const uint32_t idesc = instr_desc(1, 0, a.q_mn, kRows, BN);
    const uint32_t q_step = a.q_mn ? 2048 / 16 : 32 / 16;
    const bool withheld = WITHHOLD && blockIdx.x == 0;
    RingPlace<S> at;
    RingPlace<kSums<BN>> sums;
    bool go = true;
    for (int t = first; t < tiles && go; t += stride) {
      for (int b = b0; b < b1; ++b, at.next(), sums.next()) {
        const int s = at.stage, buf = sums.stage;
        const bool ready = mbar_wait<true>(full + s, at.full(), abort_flag, kWaitFull) &&
                           mbar_wait<true>(dfree + buf, sums.empty(), abort_flag, kWaitAccFree);
        if (!__all_sync(0xffffffffu, ready)) {
          go = false;
          break;
        }
        fence_after_sync();
        const uint32_t pa = p_parts + s * 3 * kPart;
        const uint64_t qd = plane_desc(smem_u32(ring + s * kSplit<BN>), a.q_mn);
        if (elect_one()) {
          // parts of P and Q, smallest products first
          constexpr int kParts[6][2] = {{0, 2}, {2, 0}, {1, 1}, {0, 1}, {1, 0}, {0, 0}};
#pragma unroll
          for (int m = 0; m < 6; ++m)
#pragma unroll
            for (int k = 0; k < 2; ++k)
              mma_tmem(tmem + buf * BN, pa + kParts[m][0] * kPart + k * 8,
                       qd + kParts[m][1] * (BN * kK * 2 / 16) + k * q_step, idesc,
                       (m > 0 || k > 0) ? 1u : 0u);
          mma_commit(empty + s);
          if (!withheld || b > b0) mma_commit(dfull + buf);
        }
        __syncwarp();
      }
    }
    if (elect_one()) {
      mma_commit(drain);
      volatile int keep = 0;  // wait for the issued MMAs even when another role gave up
      if (!mbar_wait(drain, 0, &keep, kWaitDrain)) *abort_flag = kWaitDrain;
    }
  } else if (drainer >= 0 && drainer < kDraining<BN>) {
    RingPlace<kSums<BN>> sums;
    bool go = true;
    if (WITHHOLD && blockIdx.x == 0)
      go = __all_sync(0xffffffffu, mbar_wait(dfull, 0, abort_flag, kWaitAccFull, kTestPollLimit));
    for (int t = first; t < tiles && go; t += stride) {
      int tp, tq;
      tile_of(t, a.tiles_p, a.tiles_q, &tp, &tq);
      if (a.splits == 1)  // the residual comes to L2 while the sums are made
        prefetch_residual(a.e, tp * kRows, a.P, kRows, tq * BN, a.Q, BN, drainer * 32 + lane, 32 * kDraining<BN>);
#pragma unroll
      for (int j = 0; j < 32; ++j) acc[j] = 0.0f;
      for (int b = b0; b < b1; ++b, sums.next()) {
        const int buf = sums.stage;
        const bool ready = mbar_wait<true>(dfull + buf, sums.full(), abort_flag, kWaitAccFull);
        if (!__all_sync(0xffffffffu, ready)) {
          go = false;
          break;
        }
        fence_after_sync();
#pragma unroll
        for (int c = 0; c < 32; c += 16) {
          float z[16];
          tmem_load16(tmem + ((uint32_t)(quarter * 32) << 16) + buf * BN + col0 + c, z);
          tmem_load_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[c + j] += z[j];
        }
        fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(dfree + buf);
      }
      if (go && a.splits == 1) {
#pragma unroll
        for (int c = 0; c < 32; c += 16)
          finish_f32<16>(a, tp * kRows + quarter * 32 + lane, tq * BN + col0 + c,
                         a.Q - (tq * BN + col0 + c), alive, [&](float *z) {
#pragma unroll
                           for (int j = 0; j < 16; ++j) z[j] = acc[c + j];
                         });
      }
    }
  }
  __syncwarp();
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const bool ok = *abort_flag == 0;
  if (a.splits > 1) {  // one tile per cluster
    int tp, tq;
    tile_of(first, a.tiles_p, a.tiles_q, &tp, &tq);
    const int f0 = tp * kRows, r0 = tq * BN, nr = min(BN, a.Q - r0);
    // sums of this CTA's k, [row][feature], over the ring, which the MMAs have read
    float *sums = reinterpret_cast<float *>(ring);
    if (drainer >= 0 && drainer < kDraining<BN>) {
#pragma unroll
      for (int j = 0; j < 32; ++j) sums[(col0 + j) * kRows + quarter * 32 + lane] = acc[j];
    }
    __syncwarp();
    cluster_sync();
    // CTA k finishes rows k, k + splits, ..., shared out among its warps
    if (ok)
      finish_rows<true>(a.e, smem_u32(sums), a.splits, f0, a.P, r0, rank + a.splits * warp,
                        a.splits * (kThreads<BN> / 32), nr, [&](int f, int r, float *z) {
                          mend<4>(z, [&](int j) { return f + j < a.P; },
                                  [&](int j) { return sum_again(a, f + j, r, alive); });
                        });
    __syncwarp();
    cluster_sync();  // until every peer has read this CTA's sums
  }
  if (!ok && threadIdx.x == 0) atomicCAS(&g_wait_error, 0, *abort_flag | (int)(blockIdx.x << 4));
  fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    fence_after_sync();
    tmem_free<1>(tmem, kColumns);
  }
}

vcsr_status make_map(CUtensorMap *m, const Operand &o, int64_t rows, int64_t K, int box_rows) {
  EncodeTiledFn enc;
  VCSR_TRY(tensor_map_encoder(&enc));
  const cuuint64_t dims[2] = {(cuuint64_t)(o.transposed ? rows : K), (cuuint64_t)(o.transposed ? K : rows)};
  const cuuint64_t strides[1] = {(cuuint64_t)o.ld * 4};
  const cuuint32_t box[2] = {32, (cuuint32_t)(o.transposed ? kK : box_rows)};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<void *>(o.p), dims, strides, box,
                         estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(VCSR_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return VCSR_OK;
}

template <int BN>
vcsr_status launch_tiles(F32Args &a, const Gemm &g, cudaStream_t st) {
  CUtensorMap mp, mq;
  VCSR_TRY(make_map(&mp, g.b, g.N, g.K, kRows));
  VCSR_TRY(make_map(&mq, g.a, g.M, g.K, BN));
  a.tiles_p = (int)ceil_div(a.P, kRows);
  a.tiles_q = (int)ceil_div(a.Q, BN);
  const int64_t tiles = (int64_t)a.tiles_p * a.tiles_q;
  if (tiles > (1 << 30)) return fail(VCSR_ERR_RANGE, "more than 2^30 output tiles");
  a.splits = choose_splits(reinterpret_cast<const void *>(gemm_f32_kernel<BN, false>), kThreads<BN>, kSmem<BN>, tiles,
                           a.stages);
  const int grid = a.splits > 1 ? (int)tiles * a.splits : (int)std::min<int64_t>(tiles, sm_count());
  const auto kernel = take_withhold() ? gemm_f32_kernel<BN, true> : gemm_f32_kernel<BN, false>;
  return launch(kernel, grid, kThreads<BN>, kSmem<BN>, a.splits, st, a, mp, mq);
}

// Expected microseconds, to choose the rows of a tile: a launch, then for every round
// of tiles on the GPU a fixed part (the epilogue) and a part per stage of k.  Fitted to
// 216 products of 1 to 62451 rows, 128 to 4096 features and k of 128 to 4096 in each
// tile, with bias, silu and residual (1% over the best tile of each on average).
// Tiles of 32 / 64 / 128 rows took, for 512 x 512, k = 512: 11.2 / 12.3 / 20.5 us;
// 62451 x 128, k = 128: 70.5 / 47.9 / 55.3; 4096 x 4096, k = 1024: 504 / 323 / 261.
template <int BN>
double tiles_cost(const F32Args &a) {
  constexpr double kFixed = BN == 32 ? 2.1 : BN == 64 ? 3.3 : 7.8, kStageUs = BN == 32 ? 0.52 : BN == 64 ? 0.64 : 0.95;
  const int64_t tiles = ceil_div(a.P, kRows) * ceil_div(a.Q, BN), stages = a.stages;
  const int splits = choose_splits(reinterpret_cast<const void *>(gemm_f32_kernel<BN, false>), kThreads<BN>, kSmem<BN>,
                                   tiles, stages);
  return 4.8 + (double)ceil_div(tiles * splits, sm_count()) * (kFixed + kStageUs * (double)ceil_div(stages, splits));
}

}  // namespace

vcsr_status launch_gemm_f32(const Gemm &g, cudaStream_t st) {
  F32Args a{};
  a.p = static_cast<const float *>(g.b.p);
  a.q = static_cast<const float *>(g.a.p);
  a.ldp = g.b.ld;
  a.ldq = g.a.ld;
  a.P = (int)g.N;
  a.Q = (int)g.M;
  a.K = (int)g.K;
  a.stages = (int)ceil_div(g.K, kK);
  a.p_mn = g.b.transposed;
  a.q_mn = g.a.transposed;
  a.e = g.e;
  // 32 rows per tile are for operands stored along k (the planes of one stored along its
  // own index come in chunks of 64)
  const double c32 = a.q_mn ? 1e30 : tiles_cost<32>(a), c64 = tiles_cost<64>(a), c128 = tiles_cost<128>(a);
  if (c32 <= c64 && c32 <= c128) return launch_tiles<32>(a, g, st);
  return c64 <= c128 ? launch_tiles<64>(a, g, st) : launch_tiles<128>(a, g, st);
}

vcsr_status take_wait_error_f32(int *word) {
  const int zero = 0;
  VCSR_CUDA(cudaMemcpyFromSymbol(word, g_wait_error, sizeof(int)));
  if (*word) VCSR_CUDA(cudaMemcpyToSymbol(g_wait_error, &zero, sizeof(int)));
  return VCSR_OK;
}

}  // namespace layer
}  // namespace vcsr
