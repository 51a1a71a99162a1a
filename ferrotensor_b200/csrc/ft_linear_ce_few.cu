// The linear cross entropy of at most 16 rows, on f32 multiply-adds.
//
// So few rows leave a matrix tile nearly empty, and what a call takes is the reading of W (and the
// writing of dW).  So W is read once for the logits and once for dh, as it lies, in its own type:
// no conversion, no packing, no scales, and two launches for the losses, three or four with
// gradients.  The rows are taken as they lie too; a skipped one counts as a row of zeros.
//
//   logits     z[t, v] = sum_k h[t, k] W(k, v), kept for the gradients (16 values a column of W), with
//              each block's running {maximum, sum} of every row
//   loss       joins the blocks' statistics.  With gradients each block of theirs does that for itself.
//   gradients  g = s w (exp(z - lse) - onehot), in shared memory, a slice of the vocabulary at a time;
//              dW written from h and g, dh summed from W and g in one walk over the slice
//   dh         the sum of the slices' parts
//
// All sums are f32, in an order that the sizes fix.  TR is the number of rows that a kernel is built for.
//
// At most four rows the reading bounds (1 row x 576 x 49152 f32: 113 MB in 29 us with both launches, 4.0 TB/s);
// from there on shared memory and multiply-adds do: a row costs a 16-byte load of h for 16 multiply-adds (16
// rows of the same: 66 us).  One block of 16 warps a multiprocessor: the sums of 16 rows fill the registers.
// Columns of W are loaded one step ahead and converted where they are used: with the conversion behind the
// load, 4 rows x 2048 x 49152 f16 took 255 us for dh, now 144.
#include <math.h>

#include "ft_linear_ce.cuh"
#include "ft_tc.cuh"

namespace {

using namespace ft_ce;
using ft_tc::ffma2;

constexpr int MAX_ROWS = 16;
constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr size_t MAX_SMEM = 200 << 10;

struct FewArgs {
  const void *hidden, *weight;
  const uint32_t* targets;
  const float* weights;
  float grad_scale;
  int h16, T, H, V;
  float* z;                                 // [T, V]; null: no gradient follows
  float2* part;                             // [parts, MAX_ROWS]: {maximum, sum of exponentials against it}
  float* picked;                            // [MAX_ROWS]
  int parts;
  float* row_loss;
  void* grad_weight;
  int dw16;
  float* slabs;                             // dh of each slice, [slices, T, H]
  int slice;                                // columns
};

__device__ __forceinline__ float value_at(const void* p, int is16, size_t i) {
  return is16 ? __half2float(((const __half*)p)[i]) : ((const float*)p)[i];
}
// a value of the rows as the products see it
__device__ __forceinline__ float hidden_at(const FewArgs& a, int t, int k) {
  return t < a.T && k < a.H && a.targets[t] != FT_MASKED_CE_SKIP ? value_at(a.hidden, a.h16, (size_t)t * a.H + k) : 0.f;
}
// N neighbouring values of W as they lie in memory: turned into f32 where they are used, so that a value
// loaded ahead is not waited for where it is loaded.  (W is not written here: __ldg may go ahead of dW's stores.)
// VEC: one load; else one a value, whatever the alignment.
template <typename TW, int N, bool VEC = true>
struct Raw {
  static constexpr int WORDS = VEC ? (N * (int)sizeof(TW) + 3) / 4 : N;
  uint32_t w[WORDS];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0u;
  }
  // the first n of them; VEC: all or none
  __device__ __forceinline__ void load(const TW* p, int n = N) {
    zero();
    if constexpr (!VEC || N == 1) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < n) {
          if constexpr (sizeof(TW) == 2) w[j] = __ldg((const unsigned short*)p + j);
          else w[j] = __ldg((const uint32_t*)p + j);
        }
    } else if (n > 0) {
      if constexpr (WORDS == 1) {
        w[0] = __ldg((const uint32_t*)p);
      } else if constexpr (WORDS == 2) {
        const uint2 v = __ldg((const uint2*)p);
        w[0] = v.x; w[1] = v.y;
      } else {
        const uint4 v = __ldg((const uint4*)p);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
      }
    }
  }
  __device__ __forceinline__ float at(int j) const {
    if constexpr (sizeof(TW) == 4) return __uint_as_float(w[j]);
    const __half2 h = *(const __half2*)&w[VEC ? j / 2 : j];
    return VEC && (j & 1) ? __high2float(h) : __low2float(h);
  }
};
__device__ __forceinline__ void online(float x, float& m, float& s) {
  const float mn = fmaxf(m, x), ref = finite_max(mn);
  s = s * expf(m - ref) + expf(x - ref);
  m = mn;
}
__device__ __forceinline__ void merge(float m2, float s2, float& m, float& s) {
  const float mn = fmaxf(m, m2), ref = finite_max(mn);
  s = s * expf(m - ref) + s2 * expf(m2 - ref);
  m = mn;
}
// The sums over a warp of N values a lane: value lane * N / 32 + i is left in a[i].
template <int N>
__device__ __forceinline__ void sum_and_spread(float (&a)[N], int lane) {
  int n = N;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (n == 1) {
      a[0] += __shfl_xor_sync(0xffffffffu, a[0], o);
      continue;
    }
    n >>= 1;
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      if (i >= n) break;
      const float give = up ? a[i] : a[i + n], keep = up ? a[i + n] : a[i];
      a[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
}

// ------------------------------------------------------------------------------ logits, [vocab, hidden]
// A warp takes VR rows of W at a time, a lane 4 of every 128 values of K.
template <typename TW, int TR, bool VEC>
__global__ void __launch_bounds__(THREADS, 1)
k_ce_few_logits_vh(const FewArgs a) {
  constexpr int VR = TR == 4 ? 8 : 4, N = TR * VR, NV = N / 32;
  // A pair of rows side by side, for packed pairs of multiply-adds: value (t, k) at [t / 2][k / 2 % 2][k / 4][k % 2][t % 2].
  extern __shared__ __align__(16) float hs[];                        // [TR][ld]
  __shared__ float2 red[WARPS][TR];
  ft_pdl_wait();
  ft_pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, H = a.H, V = a.V;
  const int ld = (H + 127) / 128 * 128;
#pragma unroll 2
  for (int t = 0; t < TR; ++t) {
    const bool live = t < a.T && a.targets[t] != FT_MASKED_CE_SKIP;
#pragma unroll 4
    for (int k = threadIdx.x; k < ld; k += THREADS) hs[(t / 2 * 2 + k / 2 % 2) * ld + k / 4 * 4 + k % 2 * 2 + t % 2] = live && k < H ? value_at(a.hidden, a.h16, (size_t)t * H + k) : 0.f;
  }
  __syncthreads();
  const int t = lane * NV / VR, r0 = lane * NV % VR;                 // what a lane has of a warp's sums
  const uint32_t y = t < a.T ? a.targets[t] : FT_MASKED_CE_SKIP;
  float m = -INFINITY, s = 0.f;
  const int step = gridDim.x * WARPS * VR;
  for (long long v0 = (long long)(blockIdx.x * WARPS + warp) * VR; v0 < V; v0 += step) {
    const TW* w = (const TW*)a.weight + (size_t)v0 * H;
    const int rows = min(VR, (int)(V - v0));
    int row_at[VR];
#pragma unroll
    for (int r = 0; r < VR; ++r) row_at[r] = min(r, rows - 1) * H;
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
#pragma unroll 2
    for (int k = lane * 4; k < ld; k += 128) {
      Raw<TW, 4, VEC> x[VR];
#pragma unroll
      for (int r = 0; r < VR; ++r) {
        x[r].load(w + row_at[r] + k, H - k);
      }
#pragma unroll
      for (int i = 0; i < TR; i += 2) {
        const float4 h0 = *(const float4*)(hs + i * ld + k), h1 = *(const float4*)(hs + (i + 1) * ld + k);
#pragma unroll
        for (int r = 0; r < VR; ++r) {
          float &c = acc[i * VR + r], &d = acc[(i + 1) * VR + r];
          ffma2(c, d, h0.x, h0.y, x[r].at(0), x[r].at(0), c, d);
          ffma2(c, d, h0.z, h0.w, x[r].at(1), x[r].at(1), c, d);
          ffma2(c, d, h1.x, h1.y, x[r].at(2), x[r].at(2), c, d);
          ffma2(c, d, h1.z, h1.w, x[r].at(3), x[r].at(3), c, d);
        }
      }
    }
    sum_and_spread(acc, lane);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (t >= a.T || r0 + i >= rows) continue;
      const int v = (int)v0 + r0 + i;
      if (a.z) a.z[(size_t)t * V + v] = acc[i];
      if (y == (uint32_t)v) a.picked[t] = acc[i];
      online(acc[i], m, s);
    }
  }
#pragma unroll
  for (int o = 1; o < VR / NV; o <<= 1) merge(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o), m, s);
  if (r0 == 0) red[warp][t] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x < TR) {
    float M = -INFINITY, S = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) merge(red[w][threadIdx.x].x, red[w][threadIdx.x].y, M, S);
    a.part[blockIdx.x * MAX_ROWS + threadIdx.x] = make_float2(M, S);
  }
}

// Sums over the warps what they hold of 4 rows and 32 COLS columns; `use(row of the four, column, sum)`.
template <int COLS, typename F>
__device__ __forceinline__ void over_warps(float* red, const float (&mine)[4][COLS], int warp, int lane, F use) {
  constexpr int C = 32 * COLS;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int c = 0; c < COLS; ++c) red[(warp * 4 + j) * C + lane * COLS + c] = mine[j][c];
  __syncthreads();
  for (int i = threadIdx.x; i < 4 * C; i += THREADS) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) x += red[w * 4 * C + i];
    use(i / C, i % C, x);
  }
}

// ------------------------------------------------------------------------------ logits, [hidden, vocab]
// A block takes 32 COLS columns at a time, a lane COLS of them, a warp its sixteenth of K.
template <typename TW, int TR, int COLS>
__global__ void __launch_bounds__(THREADS, 1)
k_ce_few_logits_hv(const FewArgs a) {
  constexpr int C = 32 * COLS, Q = TR / 4;
  extern __shared__ __align__(16) float hs[];                        // [H][TR], then [WARPS][4][C]
  __shared__ float2 top[Q][WARPS];
  ft_pdl_wait();
  ft_pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, H = a.H, V = a.V;
  float* red = hs + (size_t)H * TR;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    bool live[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) live[j] = 4 * q + j < a.T && a.targets[4 * q + j] != FT_MASKED_CE_SKIP;
#pragma unroll 2
    for (int k = threadIdx.x; k < H; k += THREADS) {
      float e[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) e[j] = live[j] ? value_at(a.hidden, a.h16, (size_t)(4 * q + j) * H + k) : 0.f;
      *(float4*)(hs + k * TR + 4 * q) = make_float4(e[0], e[1], e[2], e[3]);
    }
  }
  __syncthreads();
  const int k0 = H * warp / WARPS, k1 = H * (warp + 1) / WARPS;
  float m[Q], s[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) { m[q] = -INFINITY; s[q] = 0.f; }
  for (int tile = blockIdx.x; tile * (long long)C < V; tile += gridDim.x) {
    const int c = tile * C + lane * COLS;
    float acc[TR][COLS];
#pragma unroll
    for (int t = 0; t < TR; ++t)
#pragma unroll
      for (int j = 0; j < COLS; ++j) acc[t][j] = 0.f;
    if (c < V) {
      const TW* w = (const TW*)a.weight + (size_t)k0 * V + c;
#pragma unroll (COLS == 1 ? 16 : TR * COLS == 64 ? 4 : 8)
      for (int k = k0; k < k1; ++k, w += V) {
        Raw<TW, COLS> raw;
        raw.load(w);
        float x[COLS];
#pragma unroll
        for (int j = 0; j < COLS; ++j) x[j] = raw.at(j);
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          const float4 h = *(const float4*)(hs + k * TR + 4 * q);
#pragma unroll
          for (int j = 0; j < COLS; ++j) {
            // (packed pairs cost 8% here: four columns of 16 rows leave them no registers)
            acc[4 * q][j] = fmaf(h.x, x[j], acc[4 * q][j]);
            acc[4 * q + 1][j] = fmaf(h.y, x[j], acc[4 * q + 1][j]);
            acc[4 * q + 2][j] = fmaf(h.z, x[j], acc[4 * q + 2][j]);
            acc[4 * q + 3][j] = fmaf(h.w, x[j], acc[4 * q + 3][j]);
          }
        }
      }
    }
#pragma unroll
    for (int q = 0; q < Q; ++q)
      over_warps<COLS>(red, *(const float(*)[4][COLS]) & acc[4 * q], warp, lane, [&](int j, int col, float x) {
        const int t = 4 * q + j, v = tile * C + col;
        if (t >= a.T || v >= V) return;
        if (a.z) a.z[(size_t)t * V + v] = x;
        if (a.targets[t] == (uint32_t)v) a.picked[t] = x;
        online(x, m[q], s[q]);
      });
  }
  // (a warp's threads hold columns of one row; the first C / 32 x 4 warps hold something)
#pragma unroll
  for (int q = 0; q < Q; ++q) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) merge(__shfl_xor_sync(0xffffffffu, m[q], o), __shfl_xor_sync(0xffffffffu, s[q], o), m[q], s[q]);
    if (lane == 0) top[q][warp] = make_float2(m[q], s[q]);
  }
  __syncthreads();
  if (threadIdx.x < TR) {
    float M = -INFINITY, S = 0.f;
#pragma unroll
    for (int w = 0; w < COLS; ++w) {
      const float2 x = top[threadIdx.x / 4][(threadIdx.x % 4) * COLS + w];
      merge(x.x, x.y, M, S);
    }
    a.part[blockIdx.x * MAX_ROWS + threadIdx.x] = make_float2(M, S);
  }
}

// ------------------------------------------------------------------------------ losses
struct FewRow { float lse, weight, at_target; uint32_t target; };
// Warp t joins row t, of at most 16; the block has to meet before others read it.
__device__ __forceinline__ void join_row(const FewArgs& a, int t, int lane, FewRow* rows, bool write_loss) {
  float m = -INFINITY, s = 0.f;
  for (int p = lane; p < a.parts; p += 32) {
    const float2 x = a.part[p * MAX_ROWS + t];
    merge(x.x, x.y, m, s);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) merge(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o), m, s);
  if (lane == 0) {
    const uint32_t y = a.targets[t];
    const float ref = finite_max(m), l = logf(s);
    // (ref - z) first: a row that is sure of its target loses nothing to the size of its logits
    const float loss = y < (uint32_t)a.V ? (ref - a.picked[t]) + l : 0.f;
    if (write_loss) a.row_loss[t] = loss;
    const float w = a.weights && y != FT_MASKED_CE_SKIP ? a.weights[t] * a.grad_scale : 0.f;
    rows[t] = FewRow{ref + l, w, w * expm1f(-loss), y};
  }
}
__global__ void __launch_bounds__(THREADS)
k_ce_few_loss(const FewArgs a) {
  __shared__ FewRow rows[MAX_ROWS];
  ft_pdl_wait();
  ft_pdl_launch();
  if ((int)threadIdx.x / 32 < a.T) join_row(a, threadIdx.x / 32, threadIdx.x & 31, rows, true);
}
__device__ __forceinline__ float g_of(const FewRow& r, float z, int v) {
  if (r.target == FT_MASKED_CE_SKIP) return 0.f;
  return r.target == (uint32_t)v ? r.at_target : r.weight * expf(z - r.lse);
}
// how the gradients' kernels are cut, by the rows they are built for
__host__ __device__ constexpr int rows_at_once(int tr) { return tr == 8 ? 4 : 8; }      // [vocab, hidden]: of W, a warp
__host__ __device__ constexpr int hidden_at_once(int tr) { return tr == 16 ? 2 : 4; }   // [hidden, vocab]: rows of W, a warp

__device__ __forceinline__ void put(const FewArgs& a, size_t i, float x) {
  if (a.dw16) ((__half*)a.grad_weight)[i] = __float2half_rn(x);
  else ((float*)a.grad_weight)[i] = x;
}

// ------------------------------------------------------------------------------ gradients, [vocab, hidden]
// A block has 32 COLS of the hidden columns (blockIdx.x) and a slice of the vocabulary, a lane COLS columns,
// a warp every sixteenth row of W and dW.
template <typename TW, int TR, bool VEC>
__global__ void __launch_bounds__(THREADS, 1)
k_ce_few_grad_vh(const FewArgs a) {
  constexpr int COLS = TR == 16 ? 2 : 4, C = 32 * COLS, LD = TR + 4;
  constexpr int U = rows_at_once(TR), SUB = U * WARPS;               // a warp's rows of W at a time, the block's
  constexpr int EACH = SUB * TR / THREADS;                           // values of g a thread makes of those
  __shared__ __align__(16) float g[2][SUB][LD];
  __shared__ FewRow rows[MAX_ROWS];
  __shared__ float red[WARPS * 4 * C];
  ft_pdl_wait();
  ft_pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, H = a.H;
  const int c = blockIdx.x * C + lane * COLS;
  const int v_begin = blockIdx.y * a.slice, v_end = min(a.V, v_begin + a.slice);
  const bool dw = a.grad_weight != nullptr, dh = a.slabs != nullptr;
  Raw<TW, COLS, VEC> x[U];
  float z[EACH];
  auto load_w = [&](int v0, int u) {
    const int v = v0 + warp + WARPS * u;
    x[u].load((const TW*)a.weight + (size_t)v * H + c, dh && v < v_end ? H - c : 0);
  };
  auto load_z = [&](int v0) {
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int v = v0 + (i * THREADS + threadIdx.x) % SUB, t = (i * THREADS + threadIdx.x) / SUB;
      z[i] = t < a.T && v < v_end ? a.z[(size_t)t * a.V + v] : 0.f;
    }
  };
#pragma unroll
  for (int u = 0; u < U; ++u) load_w(v_begin, u);
  load_z(v_begin);
  if (warp < a.T) join_row(a, warp, lane, rows, blockIdx.x == 0 && blockIdx.y == 0);
  float h[TR][COLS], acc[TR][COLS];
#pragma unroll
  for (int t = 0; t < TR; ++t)
#pragma unroll
    for (int j = 0; j < COLS; ++j) {
      h[t][j] = dw ? hidden_at(a, t, c + j) : 0.f;
      acc[t][j] = 0.f;
    }
  __syncthreads();
  int buf = 0;
  for (int v0 = v_begin; v0 < v_end; v0 += SUB, buf ^= 1) {
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int v = (i * THREADS + threadIdx.x) % SUB, t = (i * THREADS + threadIdx.x) / SUB;
      g[buf][v][t] = t < a.T ? g_of(rows[t], z[i], v0 + v) : 0.f;
    }
    __syncthreads();
    // the next rows of W and logits are on their way while these are worked on
    load_z(v0 + SUB);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = warp + WARPS * u;
      const bool on = v0 + v < v_end && c < H;
      const size_t at = (size_t)(v0 + v) * H + c;
      float o[COLS], o2[COLS];                                       // of even and odd rows
#pragma unroll
      for (int j = 0; j < COLS; ++j) o[j] = o2[j] = 0.f;
#pragma unroll
      for (int q = 0; q < TR; q += 4) {
        const float4 e = *(const float4*)&g[buf][v][q];
        if (dw) {
#pragma unroll
          for (int j = 0; j < COLS; ++j) {
            ffma2(o[j], o2[j], e.x, e.y, h[q][j], h[q + 1][j], o[j], o2[j]);
            ffma2(o[j], o2[j], e.z, e.w, h[q + 2][j], h[q + 3][j], o[j], o2[j]);
          }
        }
        if (dh && on) {
#pragma unroll
          for (int j = 0; j < COLS; ++j) {
            const float w = x[u].at(j);
            ffma2(acc[q][j], acc[q + 1][j], e.x, e.y, w, w, acc[q][j], acc[q + 1][j]);
            ffma2(acc[q + 2][j], acc[q + 3][j], e.z, e.w, w, w, acc[q + 2][j], acc[q + 3][j]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < COLS; ++j) o[j] += o2[j];
      load_w(v0 + SUB, u);
      if (dw && on) {
        if (VEC && !a.dw16) {
          float* p = (float*)a.grad_weight + at;
          if constexpr (COLS == 4) *(float4*)p = make_float4(o[0], o[1], o[2], o[3]);
          else *(float2*)p = make_float2(o[0], o[1]);
        } else {
#pragma unroll
          for (int j = 0; j < COLS; ++j)
            if (c + j < H) put(a, at + j, o[j]);
        }
      }
    }
  }
  if (dh)
#pragma unroll
    for (int q = 0; q < TR / 4; ++q)
      over_warps<COLS>(red, *(const float(*)[4][COLS]) & acc[4 * q], warp, lane, [&](int j, int col, float x) {
        const int t = 4 * q + j, k = blockIdx.x * C + col;
        if (t < a.T && k < H) a.slabs[((size_t)blockIdx.y * a.T + t) * H + k] = x;
      });
}

// ------------------------------------------------------------------------------ gradients, [hidden, vocab]
// A block has a slice of the vocabulary (blockIdx.x) and a share of the hidden rows, a warp HP of them at
// a time, its lanes neighbouring columns.
template <typename TW, int TR>
__global__ void __launch_bounds__(THREADS, 1)
k_ce_few_grad_hv(const FewArgs a) {
  constexpr int HP = hidden_at_once(TR), U = HP == 2 ? 4 : 2, N = HP * TR;   // U: 32 columns each, loaded ahead
  extern __shared__ __align__(16) float g[];                         // [TR][slice]
  __shared__ FewRow rows[MAX_ROWS];
  ft_pdl_wait();
  ft_pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, H = a.H, V = a.V;
  const int v0 = blockIdx.x * a.slice, n = min(a.slice, V - v0);
  const bool dw = a.grad_weight != nullptr, dh = a.slabs != nullptr;
  const int k_step = gridDim.y * WARPS * HP;
  Raw<TW, 1> x[U][HP];
  auto load_w = [&](int k, int v, int u) {
#pragma unroll
    for (int p = 0; p < HP; ++p) x[u][p].load((const TW*)a.weight + (size_t)min(k + p, H - 1) * V + v0 + v, dh && k < H && v < n ? 1 : 0);
  };
  int k = (blockIdx.y * WARPS + warp) * HP;
#pragma unroll
  for (int u = 0; u < U; ++u) load_w(k, lane + 32 * u, u);
  if (warp < a.T) join_row(a, warp, lane, rows, blockIdx.x == 0 && blockIdx.y == 0);
  __syncthreads();
#pragma unroll 4
  for (int t = 0; t < TR; ++t)
#pragma unroll 2
    for (int v = threadIdx.x; v < n; v += THREADS) g[t * a.slice + v] = t < a.T ? g_of(rows[t], a.z[(size_t)t * V + v0 + v], v0 + v) : 0.f;
  __syncthreads();
  for (; k < H; k += k_step) {
    float h[TR][HP], acc[N];
#pragma unroll
    for (int t = 0; t < TR; ++t)
#pragma unroll
      for (int p = 0; p < HP; ++p) h[t][p] = dw ? hidden_at(a, t, k + p) : 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    const size_t first = (size_t)k * V + v0;
    for (int vb = lane; vb < n + lane; vb += 32 * U) {
      // what is loaded next: the columns behind these, or the next rows' first
      const bool more = vb - lane + 32 * U < n;
      const int k_next = more ? k : k + k_step, v_next = more ? vb + 32 * U : lane;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int v = vb + 32 * u;
        if (v < n) {
          float e[TR];
#pragma unroll
          for (int t = 0; t < TR; ++t) e[t] = g[t * a.slice + v];
          if (dh) {
#pragma unroll
            for (int p = 0; p < HP; ++p) {
              const float w = x[u][p].at(0);
#pragma unroll
              for (int t = 0; t < TR; t += 2) {
                float &c = acc[p * TR + t], &d = acc[p * TR + t + 1];
                ffma2(c, d, e[t], e[t + 1], w, w, c, d);
              }
            }
          }
          if (dw) {
#pragma unroll
            for (int p = 0; p < HP; ++p) {
              if (k + p >= H) break;
              float o = 0.f, o2 = 0.f;                               // of even and odd rows
#pragma unroll
              for (int t = 0; t < TR; t += 2) ffma2(o, o2, e[t], e[t + 1], h[t][p], h[t + 1][p], o, o2);
              put(a, first + (size_t)p * V + v, o + o2);
            }
          }
        }
        load_w(k_next, v_next + 32 * u, u);
      }
    }
    if (dh) {
      sum_and_spread(acc, lane);
      const int i = lane * N / 32, p = i / TR, t = i % TR;
      if (lane % (32 / N) == 0 && t < a.T && k + p < H) a.slabs[((size_t)blockIdx.x * a.T + t) * H + k + p] = acc[0];
    }
  }
}

// grad_hidden: the sum of the slices' parts, eight warps a share each, 32 columns a block
template <typename T>
__global__ void __launch_bounds__(256)
k_ce_few_join(const FewArgs a, int slices, T* __restrict__ out) {
  __shared__ float red[8][32];
  ft_pdl_wait();
  ft_pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = blockIdx.y, k = blockIdx.x * 32 + lane;
  float x = 0.f;
  if (k < a.H) {
    constexpr int AT_ONCE = 8;
    for (int s0 = warp; s0 < slices; s0 += 8 * AT_ONCE) {
      float v[AT_ONCE];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) v[j] = s0 + 8 * j < slices ? a.slabs[((size_t)(s0 + 8 * j) * a.T + t) * a.H + k] : 0.f;
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) x += v[j];
    }
  }
  red[warp][lane] = x;
  __syncthreads();
  if (warp == 0 && k < a.H) {
#pragma unroll
    for (int w = 1; w < 8; ++w) x += red[w][lane];
    if (a.targets[t] == FT_MASKED_CE_SKIP) x = 0.f;                  // (0 times an infinite weight)
    out[(size_t)t * a.H + k] = (T)x;
  }
}

// ------------------------------------------------------------------------------ host side
struct FewPlan {
  FewArgs a;
  int tr, blocks, slices;
  size_t logit_smem;
  int cols;                                 // [hidden, vocab]: columns a lane of the logits' kernel
  int share;                                // [hidden, vocab]: blocks that share the hidden rows of a slice
  size_t bytes;
};

int template_rows(int T) { return T <= 4 ? 4 : T <= 8 ? 8 : 16; }
size_t logits_smem(const Problem& q, int tr) {
  return q.p.weight_vocab_major ? (size_t)tr * ft_align_up((size_t)q.H, 128) * 4 : ((size_t)tr * q.H + WARPS * 4 * 128) * 4;
}

FewPlan few_plan(const FtContext* ctx, const Problem& q, const void* weight, void* base) {
  FewPlan pl = {};
  const int sms = std::max(1, ctx->sm_count);
  pl.tr = template_rows(q.T);
  pl.logit_smem = logits_smem(q, pl.tr);
  const bool vm = q.p.weight_vocab_major != 0;
  const size_t we = q.p.weight_type == FT_TYPE_F16 ? 2 : 4;
  // as many columns a lane as still give most multiprocessors a tile (and as the rows are aligned for)
  pl.cols = 1;
  for (int n = 2; n <= 4; n *= 2)
    if (q.V % n == 0 && ((uintptr_t)weight % (n * we)) == 0 && ft_cdiv(q.V, 32 * n) >= sms * 3 / 4) pl.cols = n;
  pl.blocks = std::min(sms, ft_cdiv(q.V, vm ? WARPS * (pl.tr == 4 ? 8 : 4) : 32 * pl.cols));
  // How the vocabulary (and for [hidden, vocab] weights the hidden rows) is shared out for the gradients: of
  // the ways that fill the multiprocessors a whole number of times, the one that should take the fewest
  // cycles, a block's start (its join of the statistics) and its steps counted.
  pl.slices = 0;
  double least = 1e30;
  if (!q.grad_hidden && !q.grad_weight) {
  } else if (vm) {
    const int across = ft_cdiv(q.H, pl.tr == 16 ? 64 : 128), sub = rows_at_once(pl.tr) * WARPS;
    for (int rounds = 1; rounds <= 8; ++rounds) {
      const int slice = (int)ft_align_up((size_t)ft_cdiv(q.V, std::max(1, rounds * sms / across)), WARPS);
      const long long blocks = (long long)across * ft_cdiv(q.V, slice);
      const double cost = (double)((blocks + sms - 1) / sms) * (6000.0 + 2500.0 * ft_cdiv(slice, sub));
      if (cost < least * 0.99) { least = cost; pl.a.slice = slice; }
    }
    pl.slices = ft_cdiv(q.V, pl.a.slice);
  } else {
    // g of a slice lies in shared memory, 64 KiB of it at most
    const int groups = ft_cdiv(q.H, WARPS * hidden_at_once(pl.tr));
    for (int slice : {128, 192, 256, 384, 512, 768, 1024})
      for (int rounds = 1; rounds <= 8; ++rounds) {
        const int slices = ft_cdiv(q.V, slice), share = std::max(1, std::min(rounds * sms / slices, groups));
        const double cost = (double)(((long long)slices * share + sms - 1) / sms) * (6000.0 + 4.0 * slice + ft_cdiv(groups, share) * (1000.0 + 13.0 * slice));
        if (cost < least * 0.99) { least = cost; pl.a.slice = slice; pl.share = share; }
      }
    pl.slices = ft_cdiv(q.V, pl.a.slice);
  }
  Carver c(base);
  pl.a.part = c.take<float2>((size_t)pl.blocks * MAX_ROWS);
  pl.a.picked = c.take<float>(MAX_ROWS);
  if (q.grad_hidden || q.grad_weight) pl.a.z = c.take<float>((size_t)q.T * q.V);
  if (q.grad_hidden) pl.a.slabs = c.take<float>((size_t)pl.slices * q.T * q.H);
  pl.bytes = c.bytes();
  return pl;
}

// once a device: a block may have all the shared memory that any call asks for
template <auto KERNEL>
int launch_few(FtContext* ctx, const char* name, dim3 grid, size_t smem, const FewArgs& a) {
  static bool ready[FT_MAX_DEVICES] = {};
  if (!ready[ctx->device]) {
    FT_CUDA(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)MAX_SMEM));
    ready[ctx->device] = true;
  }
  if (ctx->profile_all) ft_prof_begin(ctx, name);
  cudaError_t e = ft_launch_ex(ctx, KERNEL, grid, THREADS, smem, a);
  if (ctx->profile_all) ft_prof_end(ctx);
  ctx->launches++;
  if (e == cudaSuccess) e = cudaPeekAtLastError();
  if (e != cudaSuccess) return ft_cuda_fail(e, name, __FILE__, __LINE__);
  return FT_OK;
}

template <typename TW, int TR>
int few_run(FtContext* ctx, const Problem& q, const Tensors& t, FewPlan& pl) {
  FewArgs& a = pl.a;
  const bool vm = q.p.weight_vocab_major != 0;
  constexpr int COLS = TR == 16 ? 2 : 4;
  const bool vec = q.H % 4 == 0 && ((uintptr_t)t.weight % (4 * sizeof(TW))) == 0;
  const char* name = "k_ce_few_logits";
  if (vm && vec) FT_TRY((launch_few<k_ce_few_logits_vh<TW, TR, true>>(ctx, name, pl.blocks, pl.logit_smem, a)));
  else if (vm) FT_TRY((launch_few<k_ce_few_logits_vh<TW, TR, false>>(ctx, name, pl.blocks, pl.logit_smem, a)));
  else if (pl.cols == 4) FT_TRY((launch_few<k_ce_few_logits_hv<TW, TR, 4>>(ctx, name, pl.blocks, pl.logit_smem, a)));
  else if (pl.cols == 2) FT_TRY((launch_few<k_ce_few_logits_hv<TW, TR, 2>>(ctx, name, pl.blocks, pl.logit_smem, a)));
  else FT_TRY((launch_few<k_ce_few_logits_hv<TW, TR, 1>>(ctx, name, pl.blocks, pl.logit_smem, a)));
  if (!t.grad_hidden && !t.grad_weight) {
    FT_LAUNCH_PDL(ctx, k_ce_few_loss, 1, THREADS, 0, a);
    return FT_OK;
  }
  if (vm) {
    const bool vec_out = vec && (!t.grad_weight || ((uintptr_t)t.grad_weight & 15) == 0);
    const dim3 grid(ft_cdiv(q.H, 32 * COLS), pl.slices);
    if (vec_out) FT_LAUNCH_PDL(ctx, (k_ce_few_grad_vh<TW, TR, true>), grid, THREADS, 0, a);
    else FT_LAUNCH_PDL(ctx, (k_ce_few_grad_vh<TW, TR, false>), grid, THREADS, 0, a);
  } else {
    const size_t smem = (size_t)TR * a.slice * 4;
    FT_TRY((launch_few<k_ce_few_grad_hv<TW, TR>>(ctx, "k_ce_few_grad", dim3(pl.slices, pl.share), smem, a)));
  }
  if (t.grad_hidden) {
    const dim3 grid(ft_cdiv(q.H, 32), q.T);
    if (q.p.grad_hidden_type == FT_TYPE_F16) FT_LAUNCH_PDL(ctx, k_ce_few_join<__half>, grid, 256, 0, a, pl.slices, (__half*)t.grad_hidden);
    else FT_LAUNCH_PDL(ctx, k_ce_few_join<float>, grid, 256, 0, a, pl.slices, (float*)t.grad_hidden);
  }
  return FT_OK;
}

}  // namespace

namespace ft_ce {

// Where these kernels take a call from the others.  FT_GEMM_F32's other kernel has tiles of 128 rows, so there
// always (1 row x 576 x 49152 f16: 271 -> 30 us; 16 x 896 x 151936 f32 with both gradients: 2429 -> 628).
// The tensor cores' path reads W no more often, but starts with launches that find scales, pack rows and
// write f32 weights (and f16 ones whose pitch TMA does not take) as f16 planes; what these kernels take on
// top grows with rows x weights.  Weights up to which they are the faster ones, in millions, by the rows that
// the kernel is built for (4, 8, 16); microseconds there -> here beside the limits:
//   all f16              losses: 1 x 576 x 49152 27 -> 29; dh: 4 x 512 x 8192 30 -> 24, 4 x 1280 x 15744 40 -> 47; both
//                        gradients: 4 x 576 x 49152 95 -> 82, 4 x 2048 x 49152 225 -> 222, 8 x 1280 x 15744 85 -> 85
//   f32 rows             losses: 1 x 896 x 151936 93 -> 80, 8 x 1280 x 15744 38 -> 34, 8 x 2048 x 49152 85 -> 90; dh: 4 x
//                        576 x 49152 69 -> 65, 4 x 896 x 151936 174 -> 230; both: 4 x 896 x 151936 340 -> 315, 8 x 576
//                        x 49152 130 -> 109, 16 x 1280 x 15744 107 -> 132
//   f32 weights          losses: 1 x 576 x 49152 114 -> 40, 16 x 896 x 151936 408 -> 200; dh: 8 x 896 x 151936 538 -> 355,
//                        16 x 1280 x 15744 121 -> 117, 16 x 896 x 151936 536 -> 580; both: 16 x 896 x 151936 735 -> 720
bool few_serves(const FtContext* ctx, const Problem& q) {
  if (q.T < 1 || q.T > MAX_ROWS || q.p.vocab_piece != 0 || logits_smem(q, template_rows(q.T)) > MAX_SMEM) return false;
  if (ctx->gemm_mode == FT_GEMM_F32) return true;
  constexpr float ALL = 1e9f;
  constexpr float LIMIT[3][3][3] = {{{0, 0, 0}, {8, 4, 0}, {32, 16, 4}},
                                    {{ALL, 16, 0}, {32, 20, 4}, {ALL, 32, 4}},
                                    {{ALL, ALL, ALL}, {ALL, ALL, 24}, {ALL, ALL, ALL}}};
  const bool staged = (q.p.weight_vocab_major ? q.H : q.V) % 8 != 0;
  const int kind = q.p.weight_type == FT_TYPE_F32 ? 2 : q.p.hidden_type == FT_TYPE_F32 || staged ? 1 : 0;
  const int wanted = q.grad_weight ? 2 : q.grad_hidden ? 1 : 0;
  return (double)q.H * q.V <= 1e6 * LIMIT[kind][wanted][q.T <= 4 ? 0 : q.T <= 8 ? 1 : 2];
}

size_t few_workspace(const FtContext* ctx, const Problem& q, const void* weight) { return few_plan(ctx, q, weight, nullptr).bytes; }

int few_path(FtContext* ctx, const Problem& q, const Tensors& t, void* ws) {
  FewPlan pl = few_plan(ctx, q, t.weight, ws);
  FewArgs& a = pl.a;
  a.hidden = t.hidden; a.weight = t.weight; a.targets = t.targets; a.weights = t.weights;
  a.grad_scale = q.p.grad_scale;
  a.h16 = q.p.hidden_type == FT_TYPE_F16;
  a.T = q.T; a.H = q.H; a.V = q.V;
  a.parts = pl.blocks;
  a.row_loss = t.row_loss;
  a.grad_weight = t.grad_weight;
  a.dw16 = q.p.grad_weight_type == FT_TYPE_F16;
  const bool w16 = q.p.weight_type == FT_TYPE_F16;
  if (pl.tr == 4) return w16 ? few_run<__half, 4>(ctx, q, t, pl) : few_run<float, 4>(ctx, q, t, pl);
  if (pl.tr == 8) return w16 ? few_run<__half, 8>(ctx, q, t, pl) : few_run<float, 8>(ctx, q, t, pl);
  return w16 ? few_run<__half, 16>(ctx, q, t, pl) : few_run<float, 16>(ctx, q, t, pl);
}

}  // namespace ft_ce
