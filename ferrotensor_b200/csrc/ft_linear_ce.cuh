// What the files of the linear cross entropy share: the problem, the row bookkeeping in the
// workspace and the way the workspace is cut up.
#pragma once

#include <algorithm>

#include "ft_common.cuh"

namespace ft_ce {

// |g| is at most max |s w|; the power of two that brings that bound into [2^13, 2^14) keeps a
// probability down to 2^-27 in f16's normal range with a factor of four to spare at the top.
constexpr int G_EXP = 14;
// an f32 operand is brought to the same range before it is split into f16 planes
constexpr int OPERAND_EXP = 14;

// The power of two that brings this magnitude into [2^(exp-1), 2^exp).
__device__ __forceinline__ float power_for(float amax, int exp) {
  if (!(amax > 0.f) || !(amax < INFINITY)) return 1.f;
  int e;
  frexpf(amax, &e);
  return ldexpf(1.f, min(exp - e, 100));
}

// Written by k_ce_gather, read by every kernel after it.
struct Head {
  int count;          // supervised rows
  float g_scale;      // power of two that g carries while it is held in f16
  float g_unscale;
  float h_scale, h_unscale, w_unscale;   // of the f16 planes of f32 operands, else 1
  float z_scale;      // h_unscale * w_unscale (w_unscale alone where rows have scales of their own)
};

// Blocks of k_ce_amax for each operand, and the values that it leaves.
constexpr int AMAX_BLOCKS = 512;

// The largest of n values, in every thread of a block of 256; `red` holds 8.
__device__ __forceinline__ float block_max_of(const float* __restrict__ v, int n, float* red) {
  float m = 0.f;
  for (int i = threadIdx.x; i < n; i += 256) m = fmaxf(m, v[i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) m = fmaxf(m, red[w]);
  return m;
}

// Per packed row, except where noted.
struct Rows {
  Head* head;
  float *h_max, *w_max;   // [AMAX_BLOCKS] largest finite magnitudes of parts of the f32 operands
  int* place;         // [source row] its packed row, -1 for a skipped one
  int* source;        // its row in the caller's tensors
  uint32_t* target;
  float* weight;      // grad_scale * weights[row]
  float* unscale;     // of the row's f16 planes, or null: all rows have the head's
  float2* stat;       // running {maximum, sum of exponentials against it}; E, at the end: factors of dh's two terms
  float* picked;      // logit of the target
  float* exact;       // the same from f32 products, beside the tensor cores' sum
  float* lse;
  float* base;        // E: the point R that the row's sums are scaled against, in log2 units
  float2* kept;       // E: {value, reference point} of the target
};

struct Problem {
  FtLinearCeParams p;
  int T, H, V;
  bool grad_hidden, grad_weight;
};

struct Tensors {
  const void *hidden, *weight;
  const uint32_t* targets;
  const float* weights;
  float* row_loss;
  void *grad_hidden, *grad_weight;
};

// Cuts 256-byte aligned pieces off a block; with a null base it only adds up their sizes.
class Carver {
 public:
  explicit Carver(void* base) : base_((uintptr_t)base), at_(ft_align_up((uintptr_t)base, 256)) {}
  template <typename T>
  T* take(size_t count) {
    T* p = (T*)at_;
    at_ += ft_align_up(count * sizeof(T), 256);
    return p;
  }
  // 256 bytes more than the sum: the base may begin anywhere
  size_t bytes() const { return (size_t)(at_ - base_) + 256; }

 private:
  uintptr_t base_, at_;
};

inline Rows carve_rows(Carver& c, int T) {
  Rows r;
  r.head = c.take<Head>(1);
  r.h_max = c.take<float>(AMAX_BLOCKS);
  r.w_max = c.take<float>(AMAX_BLOCKS);
  r.place = c.take<int>(T);
  r.source = c.take<int>(T);
  r.target = c.take<uint32_t>(T);
  r.weight = c.take<float>(T);
  r.unscale = c.take<float>(T);
  r.stat = c.take<float2>(T);
  r.picked = c.take<float>(T);
  r.exact = c.take<float>(T);
  r.lse = c.take<float>(T);
  r.base = c.take<float>(T);
  r.kept = c.take<float2>(T);
  return r;
}

// Rows that a block of k_ce_gather packs.  Each block reads all targets, so the number of blocks is
// bounded: 1024 of them read at most 1024 x 4 x rows bytes, a small share of any product's time.
inline int gather_rows(int T) { return std::max(8, ft_cdiv(T, 1024)); }

// ft_linear_ce_tc.cu
size_t tc_workspace(const FtContext* ctx, const Problem& q, const void* weight);
int tc_path(FtContext* ctx, const Problem& q, const Tensors& t, void* ws);
// ft_linear_ce_few.cu: calls of a few rows
bool few_serves(const FtContext* ctx, const Problem& q);
size_t few_workspace(const FtContext* ctx, const Problem& q, const void* weight);
int few_path(FtContext* ctx, const Problem& q, const Tensors& t, void* ws);
// ft_linear_ce.cu: packs the supervised rows as f16 planes [planes][plane_rows][ld]
int launch_gather_f16(FtContext* ctx, const Problem& q, const Tensors& t, const Rows& rw, __half* out, int ld,
                      int plane_rows, int planes);

// Reference point for exponentials of a row whose maximum is m: a row that is -inf throughout
// would otherwise meet (-inf) - (-inf).
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.f : m; }

}  // namespace ft_ce
