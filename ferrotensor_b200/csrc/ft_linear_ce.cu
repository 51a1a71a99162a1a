// Linear cross entropy: output projection, masked softmax loss and both gradients without the
// [rows, vocab] logits (ferrotensor-graph/src/lfm.rs:597-623 and engine/training.rs:207-258 in one).
//
//   z = h W,  lse_t = log sum_v exp z_tv,  loss_t = lse_t - z[t, y_t]
//   g_tv = s w_t (exp(z_tv - lse_t) - [v == y_t]),  dh = g W^T,  dW = h^T g
//
// A softmax gradient needs the whole row's lse before its first element, so here, with gradients wanted,
// the logits are computed twice: one pass over the vocabulary that keeps the running maximum and
// sum of each row, then piece by piece the logits again, g of that piece, and g's two products.  (Not where the
// vocabulary is one piece, nor on the tensor cores for dh alone: see there.)
//
// Only supervised rows take part.  gather_block packs them (in order) into the workspace, so a batch
// whose prompt is masked costs its supervised tokens only, and what a skipped row holds (NaN
// included) reaches nothing.  How many there are is known on the device alone: launches are sized
// for all rows, and the kernels read the count.
//
// This file holds the entry points and the exact f32 products (FT_GEMM_F32); ft_linear_ce_tc.cu those on the
// tensor cores, ft_linear_ce_few.cu the calls of a few rows, ft_linear_ce.cuh the row bookkeeping.
//
// Times beside the code of these files compare forms of it over tens of calls from an idle GPU, at its full clock.
// Over hundreds in a row the power cap lowers that, and calls that keep the tensor cores busy take longer
// (512 rows x 576 x 49152, all f32, both gradients: 348 us over 60 calls, 373 over 400, 392 over 2000; 4096 rows,
// a quarter skipped, x 960 x 49152: 404, 443, 458), whether operands repeat or change.
#include <math.h>
#include <string.h>

#include <algorithm>

#include "ft_linear_ce.cuh"
#include "ft_tc.cuh"

namespace {

using namespace ft_ce;

template <typename TH>
__global__ void __launch_bounds__(GATHER_THREADS)
k_ce_gather(const TH* __restrict__ hidden, const uint32_t* __restrict__ targets, const float* __restrict__ weights,
            float grad_scale, int rows, int H, int per, Rows rw, float* __restrict__ out, float* __restrict__ row_loss) {
  ft_pdl_wait();
  ft_pdl_launch();
  gather_block<TH, float>(blockIdx.x, gridDim.x, hidden, targets, weights, grad_scale, rows, H, per, rw, out, H, rows, 1, 0, 0,
                          row_loss);
}

// ------------------------------------------------------------------------------ exact products
// C(m, n) (+)= alpha sum_k A(m, k) B(k, n) on f32 FMA, A f32, B f32 or f16, any element strides; 128 x
// 128 tiles, 8 x 8 values a thread.  The M or the K extent may be the device's row count.  Bound by what
// issues: 64 multiply-adds a thread and step of K as 32 packed pairs, beside 4 loads from shared memory and
// the pairing (8192 x 2048 x 49152 with dh: 110 ms, 45 TFLOP/s over three products; 133 without pairs).
constexpr int ET = 128, EK = 16;

struct ExactProduct {
  const float* a; long long sam, sak;
  const void* b; long long sbk, sbn;
  void* c; long long scm, scn;
  int M, N, K;
  int live_m, live_k;        // 1: M (K) is the number of supervised rows
  int accumulate;
  int splits;                // parts of K, each into its own slab of C (few tiles would leave most of the
  long long slab;            // multiprocessors idle through a long K)
};

template <typename TB, typename TC>
__global__ void __launch_bounds__(256, 2)
k_ce_exact(ExactProduct p, const Head* __restrict__ head) {
  // two buffers: while a step is multiplied the next one's values travel into registers
  __shared__ __align__(16) float As[2][EK][ET + 4], Bs[2][EK][ET + 4];
  ft_pdl_wait();
  ft_pdl_launch();
  const int M = p.live_m ? head->count : p.M, K = p.live_k ? head->count : p.K;
  const int m0 = blockIdx.x * ET, n0 = blockIdx.y * ET;
  if (m0 >= M) return;
  const int steps = (K + EK - 1) / EK;
  const int k_begin = (int)((long long)steps * blockIdx.z / p.splits) * EK;
  const int k_end = min(K, (int)((long long)steps * (blockIdx.z + 1) / p.splits) * EK);
  const TB* bp = (const TB*)p.b;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  // A warp reads along whichever index is contiguous: value i of a thread lies at (mn, k) or, i steps
  // further, 16 of M/N (K contiguous) or 2 of K.
  constexpr int PER = ET * EK / 256;
  const bool a_kfast = p.sak == 1, b_kfast = p.sbk == 1;
  const int am = a_kfast ? tid / EK : tid % ET, ak = a_kfast ? tid % EK : tid / ET;
  const int bn = b_kfast ? tid / EK : tid % ET, bk = b_kfast ? tid % EK : tid / ET;
  const long long a_step = a_kfast ? 16 * p.sam : 2 * p.sak, b_step = b_kfast ? 16 * p.sbn : 2 * p.sbk;
  const float* ap = p.a + (m0 + am) * p.sam + (k_begin + ak) * p.sak;
  const TB* bq = bp + (n0 + bn) * p.sbn + (k_begin + bk) * p.sbk;
  const int a_left = M - m0 - am, b_left = p.N - n0 - bn;          // of M/N, for this thread's first value
  float ar[PER], br[PER];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool oka = a_kfast ? 16 * i < a_left && k0 + ak < k_end : a_left > 0 && k0 + ak + 2 * i < k_end;
      const bool okb = b_kfast ? 16 * i < b_left && k0 + bk < k_end : b_left > 0 && k0 + bk + 2 * i < k_end;
      ar[i] = oka ? ap[i * a_step] : 0.f;
      br[i] = okb ? (float)bq[i * b_step] : 0.f;
    }
    ap += EK * p.sak;
    bq += EK * p.sbk;
  };
  auto settle = [&](int buf) {
    float* as = &As[buf][ak][am];
    float* bs = &Bs[buf][bk][bn];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      as[a_kfast ? 16 * i : 2 * i * (ET + 4)] = ar[i];
      bs[b_kfast ? 16 * i : 2 * i * (ET + 4)] = br[i];
    }
  };
  float acc[8][8] = {};
  if (k_begin < k_end) {
    fetch(k_begin);
    settle(0);
  }
  __syncthreads();
  int buf = 0;
  for (int k0 = k_begin; k0 < k_end; k0 += EK, buf ^= 1) {
    if (k0 + EK < k_end) fetch(k0 + EK);
#pragma unroll
    for (int k = 0; k < EK; ++k) {
      float av[8], bv[8];
      *(float4*)av = *(const float4*)&As[buf][k][ty * 4];
      *(float4*)(av + 4) = *(const float4*)&As[buf][k][64 + ty * 4];
      *(float4*)bv = *(const float4*)&Bs[buf][k][tx * 4];
      *(float4*)(bv + 4) = *(const float4*)&Bs[buf][k][64 + tx * 4];
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; j += 2)
          ft_tc::ffma2(acc[i][j], acc[i][j + 1], av[i], av[i], bv[j], bv[j + 1], acc[i][j], acc[i][j + 1]);
    }
    if (k0 + EK < k_end) settle(buf ^ 1);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int m = m0 + (i & 4) * 16 + ty * 4 + (i & 3);
    if (m >= M) continue;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int n = n0 + (j & 4) * 16 + tx * 4 + (j & 3);
      if (n >= p.N) continue;
      TC* c = (TC*)p.c + blockIdx.z * p.slab + m * p.scm + n * p.scn;
      *c = (TC)(p.accumulate ? (float)*c + acc[i][j] : acc[i][j]);
    }
  }
}

// Running maximum, sum and target logit of every supervised row over one piece of logits.
__global__ void __launch_bounds__(256)
k_ce_exact_stats(const float* __restrict__ z, int v0, int cols, Rows rw, int first) {
  __shared__ float red[8];
  ft_pdl_wait();
  ft_pdl_launch();
  const int r = blockIdx.x;
  if (r >= rw.head->count) return;
  const float* row = z + (size_t)r * cols;
  float m = -INFINITY;
  for (int i = threadIdx.x; i < cols; i += 256) m = fmaxf(m, row[i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  for (int w = 0; w < 8; ++w) m = fmaxf(m, red[w]);
  const float before = first ? -INFINITY : rw.stat[r].x;
  m = fmaxf(m, before);
  const float ref = finite_max(m);
  float s = 0.f;
  for (int i = threadIdx.x; i < cols; i += 256) s += expf(row[i] - ref);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.f;
    for (int w = 0; w < 8; ++w) s += red[w];
    if (!first) s += rw.stat[r].y * expf(before - ref);
    rw.stat[r] = make_float2(m, s);
    const uint32_t y = rw.target[r] - (uint32_t)v0;
    if (y < (uint32_t)cols) rw.picked[r] = row[y];
  }
}

__global__ void __launch_bounds__(256)
k_ce_exact_loss(Rows rw, int vocab, float* __restrict__ row_loss) {
  ft_pdl_wait();
  ft_pdl_launch();
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r >= rw.head->count) return;
  const float2 st = rw.stat[r];
  const float ref = finite_max(st.x), l = logf(st.y);
  rw.lse[r] = ref + l;
  // (ref - z) first: a row that is sure of its target loses nothing to the size of its logits
  const float loss = rw.target[r] < (uint32_t)vocab ? (ref - rw.picked[r]) + l : 0.f;
  row_loss[rw.source[r]] = loss;
  rw.at_target[r] = expm1f(-loss);
}

// logits -> g, in place
__global__ void __launch_bounds__(256)
k_ce_exact_grad(float* __restrict__ z, int v0, int cols, Rows rw) {
  ft_pdl_wait();
  ft_pdl_launch();
  const int r = blockIdx.x;
  if (r >= rw.head->count) return;
  float* row = z + (size_t)r * cols;
  const float lse = rw.lse[r], w = rw.weight[r], at_target = w * rw.at_target[r];
  const uint32_t y = rw.target[r] - (uint32_t)v0;
  for (int i = threadIdx.x; i < cols; i += 256) {
    row[i] = (uint32_t)i == y ? at_target : w * expf(row[i] - lse);
  }
}

// packed f32 rows -> grad_hidden, zeros for the rows that were skipped
template <typename T>
__global__ void __launch_bounds__(256)
k_ce_exact_scatter(const float* __restrict__ acc, size_t slab, int splits, Rows rw, int H, T* __restrict__ out) {
  ft_pdl_wait();
  ft_pdl_launch();
  const int r = blockIdx.x;
  const int at = rw.place[r];
  for (int c = threadIdx.x; c < H; c += 256) {
    float v = 0.f;
    if (at >= 0)
      for (int s = 0; s < splits; ++s) v += acc[s * slab + (size_t)at * H + c];
    out[(size_t)r * H + c] = (T)v;
  }
}

// ------------------------------------------------------------------------------ the exact path
constexpr size_t EXACT_PIECE_BYTES = (size_t)256 << 20;
constexpr size_t EXACT_PIECE_COLUMNS = (size_t)1 << 22;   // of 65535 x 128 that a grid reaches

struct ExactPlan {
  Rows rows;
  float *hidden, *z, *acc;
  int piece, splits;
  size_t bytes;
};

int launch_gather(FtContext* ctx, const Problem& q, const Tensors& t, const Rows& rw, float* out) {
  const int per = gather_rows(q.T), blocks = ft_cdiv(q.T, per);
  if (q.p.hidden_type == FT_TYPE_F16)
    FT_LAUNCH_PDL(ctx, k_ce_gather<__half>, blocks, GATHER_THREADS, 0, (const __half*)t.hidden, t.targets, t.weights,
                  q.p.grad_scale, q.T, q.H, per, rw, out, t.row_loss);
  else
    FT_LAUNCH_PDL(ctx, k_ce_gather<float>, blocks, GATHER_THREADS, 0, (const float*)t.hidden, t.targets, t.weights,
                  q.p.grad_scale, q.T, q.H, per, rw, out, t.row_loss);
  return FT_OK;
}

ExactPlan exact_plan(const FtContext* ctx, const Problem& q, void* base) {
  ExactPlan pl;
  Carver c(base);
  pl.rows = carve_rows(c, q.T);
  size_t cols = q.p.vocab_piece ? q.p.vocab_piece : std::max<size_t>(64, EXACT_PIECE_BYTES / 4 / std::max(q.T, 1) / 64 * 64);
  pl.piece = (int)std::min({cols, (size_t)q.V, EXACT_PIECE_COLUMNS});
  pl.hidden = c.take<float>((size_t)q.T * q.H);
  pl.z = c.take<float>((size_t)q.T * pl.piece);
  // parts of the vocabulary for dh: two blocks for every multiprocessor, 512 columns each at least, 256 MB of slabs
  const size_t slab = (size_t)std::max(q.T, 1) * q.H * 4;
  const long long tiles = (long long)ft_cdiv(std::max(q.T, 1), ET) * ft_cdiv(q.H, ET);
  pl.splits = (int)std::max<long long>(1, std::min({2ll * ctx->sm_count / tiles, (long long)pl.piece / 512,
                                                    (long long)(((size_t)256 << 20) / slab), 32ll}));
  pl.acc = q.grad_hidden ? c.take<float>((size_t)pl.splits * q.T * q.H) : nullptr;
  pl.bytes = c.bytes();
  return pl;
}

int launch_exact(FtContext* ctx, const ExactProduct& p, bool b_f16, bool c_f16, const Head* head) {
  if (p.M <= 0 || p.N <= 0) return FT_OK;
  const dim3 grid(ft_cdiv(p.M, ET), ft_cdiv(p.N, ET), p.splits);
  if (b_f16) {
    if (c_f16) FT_LAUNCH_PDL(ctx, (k_ce_exact<__half, __half>), grid, 256, 0, p, head);
    else FT_LAUNCH_PDL(ctx, (k_ce_exact<__half, float>), grid, 256, 0, p, head);
  } else {
    if (c_f16) FT_LAUNCH_PDL(ctx, (k_ce_exact<float, __half>), grid, 256, 0, p, head);
    else FT_LAUNCH_PDL(ctx, (k_ce_exact<float, float>), grid, 256, 0, p, head);
  }
  return FT_OK;
}

int exact_path(FtContext* ctx, const Problem& q, const Tensors& t, void* ws) {
  const ExactPlan pl = exact_plan(ctx, q, ws);
  const int T = q.T, H = q.H, V = q.V;
  FT_TRY(launch_gather(ctx, q, t, pl.rows, pl.hidden));
  const bool w16 = q.p.weight_type == FT_TYPE_F16;
  const long long swk = q.p.weight_vocab_major ? 1 : V, swv = q.p.weight_vocab_major ? H : 1;   // strides of W(k, v)
  const size_t we = w16 ? 2 : 4;
  auto logits = [&](int v0, int cols) {
    ExactProduct p = {};
    p.a = pl.hidden; p.sam = H; p.sak = 1;
    p.b = (const char*)t.weight + (size_t)v0 * swv * we; p.sbk = swk; p.sbn = swv;
    p.c = pl.z; p.scm = cols; p.scn = 1;
    p.M = T; p.N = cols; p.K = H; p.live_m = 1; p.splits = 1;
    return launch_exact(ctx, p, w16, false, pl.rows.head);
  };
  for (int v0 = 0; v0 < V; v0 += pl.piece) {
    const int cols = std::min(pl.piece, V - v0);
    FT_TRY(logits(v0, cols));
    FT_LAUNCH_PDL(ctx, k_ce_exact_stats, T, 256, 0, pl.z, v0, cols, pl.rows, v0 == 0 ? 1 : 0);
  }
  FT_LAUNCH_PDL(ctx, k_ce_exact_loss, ft_cdiv(T, 256), 256, 0, pl.rows, V, t.row_loss);
  if (!t.grad_hidden && !t.grad_weight) return FT_OK;
  for (int v0 = 0; v0 < V; v0 += pl.piece) {
    const int cols = std::min(pl.piece, V - v0);
    if (pl.piece < V) FT_TRY(logits(v0, cols));   // one piece: the logits of the first pass still lie there
    FT_LAUNCH_PDL(ctx, k_ce_exact_grad, T, 256, 0, pl.z, v0, cols, pl.rows);
    if (t.grad_hidden) {
      ExactProduct p = {};
      p.a = pl.z; p.sam = cols; p.sak = 1;
      p.b = (const char*)t.weight + (size_t)v0 * swv * we; p.sbk = swv; p.sbn = swk;
      p.c = pl.acc; p.scm = H; p.scn = 1;
      p.M = T; p.N = H; p.K = cols; p.live_m = 1; p.accumulate = v0 > 0;
      p.splits = pl.splits; p.slab = (long long)T * H;
      FT_TRY(launch_exact(ctx, p, w16, false, pl.rows.head));
    }
    if (t.grad_weight) {
      const size_t ge = q.p.grad_weight_type == FT_TYPE_F16 ? 2 : 4;
      ExactProduct p = {};
      p.a = pl.z; p.sam = 1; p.sak = cols;
      p.b = pl.hidden; p.sbk = H; p.sbn = 1;
      p.c = (char*)t.grad_weight + (size_t)v0 * swv * ge; p.scm = swv; p.scn = swk;
      p.M = cols; p.N = H; p.K = T; p.live_k = 1; p.splits = 1;
      FT_TRY(launch_exact(ctx, p, false, ge == 2, pl.rows.head));
    }
  }
  if (t.grad_hidden) {
    if (q.p.grad_hidden_type == FT_TYPE_F16)
      FT_LAUNCH_PDL(ctx, k_ce_exact_scatter<__half>, T, 256, 0, pl.acc, (size_t)T * H, pl.splits, pl.rows, H, (__half*)t.grad_hidden);
    else
      FT_LAUNCH_PDL(ctx, k_ce_exact_scatter<float>, T, 256, 0, pl.acc, (size_t)T * H, pl.splits, pl.rows, H, (float*)t.grad_hidden);
  }
  return FT_OK;
}

int check_params(const char* who, FtContext* ctx, const FtLinearCeParams* p) {
  FT_REQUIRE(ctx && p, "%s: NULL argument", who);
  FT_REQUIRE(p->rows <= (1u << 24) && p->hidden >= 1 && p->hidden <= (1u << 16) && p->vocab >= 1 && p->vocab <= (1u << 24),
             "%s: %u rows, hidden %u, vocab %u are outside 0..2^24, 1..2^16, 1..2^24", who, p->rows, p->hidden, p->vocab);
  const uint32_t types[4] = {p->hidden_type, p->weight_type, p->grad_hidden_type, p->grad_weight_type};
  for (uint32_t t : types) FT_REQUIRE(t == FT_TYPE_F32 || t == FT_TYPE_F16, "%s: unknown type %u", who, t);
  FT_REQUIRE(isfinite(p->grad_scale), "%s: grad_scale %g is not finite", who, (double)p->grad_scale);
  return FT_OK;
}

Problem make_problem(const FtLinearCeParams& p, bool gh, bool gw) {
  Problem q;
  q.p = p;
  q.T = (int)p.rows; q.H = (int)p.hidden; q.V = (int)p.vocab;
  q.grad_hidden = gh; q.grad_weight = gw;
  return q;
}

size_t type_size(uint32_t t) { return t == FT_TYPE_F16 ? 2 : 4; }

}  // namespace

extern "C" int ft_linear_cross_entropy_workspace(FtContext* ctx, const void* weight, const FtLinearCeParams* p,
                                                 int want_grad_hidden, int want_grad_weight, size_t* bytes) {
  FT_TRY(check_params("ft_linear_cross_entropy_workspace", ctx, p));
  FT_REQUIRE(bytes, "ft_linear_cross_entropy_workspace: NULL argument");
  const Problem q = make_problem(*p, want_grad_hidden != 0, want_grad_weight != 0);
  *bytes = few_serves(ctx, q)              ? few_workspace(ctx, q, weight)
           : ctx->gemm_mode == FT_GEMM_F32 ? exact_plan(ctx, q, nullptr).bytes : tc_workspace(ctx, q, weight);
  return FT_OK;
}

extern "C" int ft_linear_cross_entropy(FtContext* ctx, const void* hidden, const void* weight, const uint32_t* targets,
                                       const float* weights, float* row_loss, void* grad_hidden, void* grad_weight,
                                       void* workspace, size_t workspace_bytes, const FtLinearCeParams* p) {
  const char* who = "ft_linear_cross_entropy";
  FT_TRY(check_params(who, ctx, p));
  const size_t T = p->rows, H = p->hidden, V = p->vocab;
  FT_REQUIRE(weight && (!T || (hidden && targets && row_loss)), "%s: NULL argument", who);
  FT_REQUIRE(weights || !T || (!grad_hidden && !grad_weight), "%s: a gradient needs the rows' weights", who);
  size_t need = 0;
  FT_TRY(ft_linear_cross_entropy_workspace(ctx, weight, p, grad_hidden != nullptr, grad_weight != nullptr, &need));
  FT_REQUIRE(workspace && workspace_bytes >= need, "%s: the workspace has %zu bytes, %zu are needed", who,
             workspace ? workspace_bytes : (size_t)0, need);
  struct Range { const char* name; const void* p; size_t bytes; size_t align; };
  const Range in[4] = {{"hidden", hidden, T * H * type_size(p->hidden_type), type_size(p->hidden_type)},
                       {"weight", weight, H * V * type_size(p->weight_type), type_size(p->weight_type)},
                       {"targets", targets, T * 4, 4}, {"weights", weights, weights ? T * 4 : 0, 4}};
  const Range out[4] = {{"row_loss", row_loss, T * 4, 4},
                        {"grad_hidden", grad_hidden, grad_hidden ? T * H * type_size(p->grad_hidden_type) : 0, type_size(p->grad_hidden_type)},
                        {"grad_weight", grad_weight, grad_weight ? H * V * type_size(p->grad_weight_type) : 0, type_size(p->grad_weight_type)},
                        {"workspace", workspace, need, 1}};
  auto meet = [](const Range& a, const Range& b) {
    const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
    return a.bytes && b.bytes && x < y + b.bytes && y < x + a.bytes;
  };
  for (int i = 0; i < 4; ++i) {
    FT_REQUIRE(((uintptr_t)in[i].p % in[i].align) == 0, "%s: %s is not aligned to its elements", who, in[i].name);
    FT_REQUIRE(((uintptr_t)out[i].p % out[i].align) == 0, "%s: %s is not aligned to its elements", who, out[i].name);
    for (int j = 0; j < 4; ++j) {
      FT_REQUIRE(!meet(out[i], in[j]), "%s: %s overlaps %s", who, out[i].name, in[j].name);
      FT_REQUIRE(j <= i || !meet(out[i], out[j]), "%s: %s overlaps %s", who, out[i].name, out[j].name);
    }
  }
  FtDeviceScope on(ctx);
  if (!T) {
    if (grad_weight) FT_CUDA(cudaMemsetAsync(grad_weight, 0, out[2].bytes, ctx->stream));
    return FT_OK;
  }
  const Problem q = make_problem(*p, grad_hidden != nullptr, grad_weight != nullptr);
  const Tensors t = {hidden, weight, targets, weights, row_loss, grad_hidden, grad_weight};
  if (few_serves(ctx, q)) return few_path(ctx, q, t, workspace);
  return ctx->gemm_mode == FT_GEMM_F32 ? exact_path(ctx, q, t, workspace) : tc_path(ctx, q, t, workspace);
}
