// layer_linear.cuh — host parts that the dense products share (layer_linear.cu,
// layer_gated.cu, layer_block.cu): aligned copies of operands, the sums behind dbias, argument
// checks, and which product kernel runs.
#pragma once
#include <algorithm>

#include "layer_gemm.cuh"

namespace vcsr {
namespace layer {

constexpr size_t kAlign = 256;
inline size_t round_up(size_t n) { return (n + kAlign - 1) / kAlign * kAlign; }

// Matrices whose base or pitch is no multiple of 16 bytes, which TMA cannot read,
// copied to ones whose pitch is.
struct PackJob {
  const void *src;
  void *dst;
  int64_t ld, ldd, rows, cols;
};
// The copies, and the column sums of dbias' partial rows, that go before the products.
struct PrepareJobs {
  PackJob job[3];
  int packs;
  const float *partial;
  int partials, dtype;
  int64_t N;
  void *dbias;
};

inline int64_t packed_pitch(int64_t cols, int dtype) {
  const int64_t v = 16 / (int64_t)type_size(dtype);
  return ceil_div(cols, v) * v;
}

// What the tensor cores read of a matrix: itself, or a copy in the workspace.
struct Packed {
  bool copy = false;
  int64_t ld = 0;
  size_t bytes = 0;
};
inline Packed packed(const void *p, int64_t ld, int64_t rows, int64_t cols, int dtype) {
  Packed k;
  k.ld = rows == 1 ? packed_pitch(cols, dtype) : ld;  // the pitch of one row is free
  if (!tc_aligned(p, k.ld, dtype)) {
    k.copy = true;
    k.ld = packed_pitch(cols, dtype);
    k.bytes = round_up((size_t)rows * k.ld * type_size(dtype));
  }
  return k;
}
// What goes before a call's products, made by one launch.
struct Prepare {
  PrepareJobs jobs{};
  int64_t most = 0;  // blocks of the largest job
  char *ws;
  explicit Prepare(void *workspace) : ws(static_cast<char *>(workspace)) {}
  // Where the tensor cores read matrix p: the matrix, or its copy to be.
  const void *matrix(const Packed &k, const void *p, int64_t ld, int64_t rows, int64_t cols, int dtype) {
    if (!k.copy) return p;
    jobs.job[jobs.packs++] = {p, ws, ld, k.ld, rows, cols};
    most = std::max(most, ceil_div(rows * k.ld * (int64_t)type_size(dtype) / 16, 256));
    p = ws;
    ws += k.bytes;
    return p;
  }
  void column_sums(const float *partial, int count, int64_t N, void *out) {
    jobs.partial = partial;
    jobs.partials = count;
    jobs.N = N;
    jobs.dbias = out;
    most = std::max(most, ceil_div(N, 32));
  }
  vcsr_status run(int dtype, cudaStream_t st);
};

constexpr int kDzWarps = 8;  // of the blocks that make dz

// f(T{}) for the element type named by `type`, which is F32, BF16 or F16.
template <class F>
inline void for_type(int type, F &&f) {
  if (type == VCSR_F32)
    f(float{});
  else if (type == VCSR_BF16)
    f(__nv_bfloat16{});
  else
    f(__half{});
}

// The product by the kernel for its type; over no k, the epilogue of zeros.
vcsr_status launch_gemm(const Gemm &g, cudaStream_t st);

vcsr_status check_workspace(const void *ws, size_t bytes, size_t need);
vcsr_status check_sizes(int64_t M, int64_t N, int64_t K);
vcsr_status zero_matrix(void *p, int64_t ld, int64_t rows, int64_t cols, int type, cudaStream_t st);

}  // namespace layer
}  // namespace vcsr
