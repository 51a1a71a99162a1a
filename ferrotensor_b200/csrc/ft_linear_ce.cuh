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

// Written with the packed rows, read by every kernel after that.
struct Head {
  int count;          // supervised rows
  float g_scale;      // power of two that g carries while it is held in f16
  float g_unscale;
  float h_scale, h_unscale, w_unscale;   // of the f16 planes of f32 operands, else 1
  float z_scale;      // h_unscale * w_unscale (w_unscale alone where rows have scales of their own)
};

// Most blocks of k_ce_amax for an operand, each of which leaves a value: eight a multiprocessor (512 x 576 x
// 49152 f32, the whole call: 363 us with 512 blocks, 351 with 888, 347 with these).
constexpr int AMAX_BLOCKS = 1184;

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
  float *h_max, *w_max;   // [up to AMAX_BLOCKS] largest finite magnitudes of parts of the f32 operands
  int* place;         // [source row] its packed row, -1 for a skipped one
  int* source;        // its row in the caller's tensors
  uint32_t* target;
  float* weight;      // grad_scale * weights[row]
  float* unscale;     // of the row's f16 planes, or null: all rows have the head's
  float2* stat;       // running {maximum, sum of exponentials against it}; E, at the end: factors of dh's two terms
  float* picked;      // logit of the target
  float* exact;       // the same from f32 products, beside the tensor cores' sum
  float* lse;
  float* at_target;   // p - 1 at the target, from the loss: -(1 - e^-loss) is exact where 1 - p is small
  float* base;        // E: the point R that the row's sums are scaled against, in log2 units
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
  r.at_target = c.take<float>(T);
  r.base = c.take<float>(T);
  return r;
}

// Rows that a block packs.  Each block reads all targets, so the number of blocks is
// bounded: 1024 of them read at most 1024 x 4 x rows bytes, a small share of any product's time.
inline int gather_rows(int T) { return std::max(8, ft_cdiv(T, 1024)); }

// ------------------------------------------------------------------------------ row bookkeeping
constexpr int GATHER_THREADS = 256;

// One row -> f16 (and its rounding remainder, when `lo` is given), eight values a lane.
template <typename TH>
__device__ __forceinline__ void pack_row(const TH* __restrict__ from, int H, float S, __half* __restrict__ hi, int ld,
                                         __half* __restrict__ lo, int lane) {
  const bool vec = (((uintptr_t)from) & 15) == 0;
  for (int c = lane * 8; c < ld; c += 256) {
    if constexpr (sizeof(TH) == 2) {
      if (vec && c + 8 <= H) {
        *(uint4*)(hi + c) = *(const uint4*)(from + c);
        continue;
      }
    }
    float v[8];
    if (vec && c + 8 <= H && sizeof(TH) == 4) {
      const float4 a = *(const float4*)(from + c), b = *(const float4*)(from + c + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = c + k < H ? (float)from[c + k] : 0.f;
    }
    __half2 h[4], l[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float a = v[2 * k] * S, b = v[2 * k + 1] * S;
      h[k] = __floats2half2_rn(a, b);
      const float2 f = __half22float2(h[k]);
      l[k] = __floats2half2_rn(a - f.x, b - f.y);
    }
    *(uint4*)(hi + c) = *(const uint4*)h;
    if (lo) *(uint4*)(lo + c) = *(const uint4*)l;
  }
}

// largest finite magnitude of a row, in every lane
template <typename TH>
__device__ __forceinline__ float row_amax(const TH* __restrict__ from, int H, int lane) {
  float m = 0.f;
#pragma unroll 8
  for (int c = lane; c < H; c += 32) {
    const float x = fabsf((float)from[c]);
    if (x < INFINITY) m = fmaxf(m, x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

// Block `block` of `blocks` packs rows [block * per, ...).  Every block counts the supervised rows of the
// whole batch itself (targets are 4 bytes a row and come from L2), which gives it the place of its
// first row and the total without a launch of its own or a wait on its neighbours.
// TO = __half: as `planes` f16 planes of `plane_rows` rows, times the power of two of the largest
// value (of each row's, with rw.unscale) where they are f32, and with zero rows up to the next multiple of 64 (a K block of dW).
template <typename TH, typename TO>
__device__ __forceinline__ void gather_block(int block, int blocks, const TH* __restrict__ hidden,
                                             const uint32_t* __restrict__ targets, const float* __restrict__ weights,
                                             float grad_scale, int rows, int H, int per, Rows rw, TO* __restrict__ out, int ld,
                                             int plane_rows, int planes, int h_parts, int w_parts, float* __restrict__ row_loss) {
  constexpr int WARPS = GATHER_THREADS / 32;
  __shared__ int red[WARPS], counts[2][WARPS];
  __shared__ float tops[3][WARPS];
  __shared__ int src_row[GATHER_THREADS];
  const int r0 = block * per, r1 = min(rows, r0 + per);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // What has to be known of the whole batch, every thread's share first: all loads are under way
  // before the one join.
  int before = 0, all = 0;
  float big = 0.f, h_top = 0.f, w_top = 0.f;   // of |s w_t|, of the operands
  {
    if (sizeof(TO) == 2 && sizeof(TH) == 4 && !rw.unscale)
      for (int i = tid; i < h_parts; i += GATHER_THREADS) h_top = fmaxf(h_top, rw.h_max[i]);
    if (sizeof(TO) == 2 && block == 0)
      for (int i = tid; i < w_parts; i += GATHER_THREADS) w_top = fmaxf(w_top, rw.w_max[i]);
    auto count = [&](int i, uint32_t y) {
      const int one = y != FT_MASKED_CE_SKIP;
      all += one;
      before += i < r0 ? one : 0;
    };
    const int vec = (((uintptr_t)targets) & 15) == 0 ? rows / 4 : 0;
    for (int i = tid; i < vec; i += GATHER_THREADS) {
      const uint4 y = ((const uint4*)targets)[i];
      count(4 * i, y.x); count(4 * i + 1, y.y); count(4 * i + 2, y.z); count(4 * i + 3, y.w);
    }
    for (int i = 4 * vec + tid; i < rows; i += GATHER_THREADS) count(i, targets[i]);
    if (block == 0 && weights)
      for (int i = tid; i < rows; i += GATHER_THREADS) {
        const float w = fabsf(weights[i] * grad_scale);
        if (targets[i] != FT_MASKED_CE_SKIP) big = fmaxf(big, w);
      }
    before = __reduce_add_sync(0xffffffffu, before);
    all = __reduce_add_sync(0xffffffffu, all);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
      h_top = fmaxf(h_top, __shfl_xor_sync(0xffffffffu, h_top, o));
      w_top = fmaxf(w_top, __shfl_xor_sync(0xffffffffu, w_top, o));
    }
    if (lane == 0) {
      counts[0][warp] = before; counts[1][warp] = all;
      tops[0][warp] = big; tops[1][warp] = h_top; tops[2][warp] = w_top;
    }
    __syncthreads();
    before = all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      before += counts[0][w]; all += counts[1][w];
      big = fmaxf(big, tops[0][w]); h_top = fmaxf(h_top, tops[1][w]); w_top = fmaxf(w_top, tops[2][w]);
    }
  }
  const float h_scale = sizeof(TO) == 2 && sizeof(TH) == 4 ? power_for(h_top, OPERAND_EXP) : 1.f;
  if (block == 0 && tid == 0) {
    const float S = power_for(big, G_EXP);
    rw.head->count = all;
    rw.head->g_scale = S;
    rw.head->g_unscale = 1.0f / S;
    if constexpr (sizeof(TO) == 2) {
      const float wu = w_parts ? 1.0f / power_for(w_top, OPERAND_EXP) : 1.0f;
      rw.head->h_unscale = 1.0f / h_scale;
      rw.head->w_unscale = wu;
      rw.head->z_scale = wu / h_scale;
    }
  }
  int at = before;
  for (int base = r0; base < r1; base += GATHER_THREADS) {
    const int r = base + tid;
    const uint32_t y = r < r1 ? targets[r] : FT_MASKED_CE_SKIP;
    const bool live = y != FT_MASKED_CE_SKIP;
    const uint32_t mask = __ballot_sync(0xffffffffu, live);
    __syncthreads();
    if (lane == 0) red[warp] = __popc(mask);
    __syncthreads();
    int mine = __popc(mask & ((1u << lane) - 1u)), total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) mine += red[w];
      total += red[w];
    }
    if (live) {
      src_row[mine] = r;
      rw.source[at + mine] = r;
      rw.target[at + mine] = y;
      rw.weight[at + mine] = weights ? weights[r] * grad_scale : 0.f;
    } else if (r < r1) {
      row_loss[r] = 0.f;
    }
    if (r < r1) rw.place[r] = live ? at + mine : -1;
    __syncthreads();
    for (int k = warp; k < total; k += GATHER_THREADS / 32) {
      const TH* from = hidden + (size_t)src_row[k] * H;
      TO* to = out + (size_t)(at + k) * ld;
      if constexpr (sizeof(TO) == 4) {
        for (int c = lane; c < H; c += 32) to[c] = (float)from[c];
      } else {
        float S = h_scale;
        if (sizeof(TH) == 4 && rw.unscale) {
          S = power_for(row_amax(from, H, lane), OPERAND_EXP);
          if (lane == 0) rw.unscale[at + k] = 1.0f / S;
        }
        pack_row(from, H, S, to, ld, planes == 2 ? to + (size_t)plane_rows * ld : nullptr, lane);
      }
    }
    at += total;
    __syncthreads();
  }
  if constexpr (sizeof(TO) == 2) {
    const int end = max(64, (all + 63) / 64 * 64);
    for (int p = 0; p < planes; ++p)
      for (int r = all + block * (GATHER_THREADS / 32) + warp; r < end; r += blocks * (GATHER_THREADS / 32))
        for (int c = lane * 8; c < ld; c += 256)
          *(uint4*)(out + ((size_t)p * plane_rows + r) * ld + c) = make_uint4(0u, 0u, 0u, 0u);
  }
}

// ft_linear_ce_tc.cu
size_t tc_workspace(const FtContext* ctx, const Problem& q, const void* weight);
int tc_path(FtContext* ctx, const Problem& q, const Tensors& t, void* ws);
// ft_linear_ce_few.cu: calls of a few rows
bool few_serves(const FtContext* ctx, const Problem& q);
size_t few_workspace(const FtContext* ctx, const Problem& q, const void* weight);
int few_path(FtContext* ctx, const Problem& q, const Tensors& t, void* ws);
// Reference point for exponentials of a row whose maximum is m: a row that is -inf throughout
// would otherwise meet (-inf) - (-inf).
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.f : m; }

}  // namespace ft_ce
