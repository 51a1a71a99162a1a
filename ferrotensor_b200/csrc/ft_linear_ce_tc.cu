// The products of the linear cross entropy on the tensor cores (FT_GEMM_F16 and FT_GEMM_F16X2).
//
// One kernel serves all of them: C[256 x tile_n tile] = sum over (plane pairs, K) of A . B^T on a CTA
// pair (tcgen05 cta_group::2), with either operand K-contiguous or M/N-contiguous in memory, so no
// operand is ever transposed:
//   logits   A = packed rows,    B = W            K = hidden    epilogue: row statistics, E, or g
//   dh       A = E or g,         B = W            K = a vocabulary piece (in `splits` parts)
//   dW       A = g,              B = packed rows  K = rows (turned over for [hidden, vocab] weights)
//
// dW's K runs over rows, so its operand g must be normalised, which needs every row's log-sum-exp
// first: the logits are computed twice (or, in the split mode when the vocabulary is one piece and that is
// cheaper, g is made of E in place).  dh alone does not need that.  The pass that finds the
// statistics writes E = 2^(z2 - ref + 14) for each column tile (z2 in log2 units, ref the row's maximum in
// that tile: E has f16's full precision whatever the row's normaliser turns out to be, down to 2^-28 of
// that maximum), and the product E W is drained from tensor memory once a tile of K and scaled there,
// in f32, by the row's 2^(ref - R).  R is the row's maximum when its first piece was done; the rest of
// the normaliser and the target's term, w (p - 1) W(:, y), which E leaves out, are applied by the pass
// that unpacks the rows.  That saves a third of the multiplications of a frozen head's gradient.
//
// Planes: an f16 operand, and an f32 one in FT_GEMM_F16, is one f16 plane.  FT_GEMM_F16X2 carries an
// f32 operand and g (or E) as two planes, hi = f16(x) and lo = f16(x - hi), of which the products
// hi.hi, hi.lo and lo.hi are summed: 22 bits, and 2^-38 of the largest for values so small that lo meets
// f16's smallest step (all are scaled to end near 2^14).  The tensor core adds each group of 16 products into
// its f32 accumulator with the low bits cut off, a loss of up to K/16 x 2^-24 of the sum, so that mode
// also sums at most 512 of K in tensor memory and adds the slices up in registers.
//
// Roles and barriers as in ft_gemm_tc.cu's pair kernel: warp 0 loads (TMA), warp 1 of the even CTA
// issues the products, the eight or sixteen after them drain, and two more compute the targets' logits.
// Every wait is bounded; a wait that runs out sets the status word, and all roles fall through.
#include <math.h>
#include <string.h>

#include "ft_linear_ce.cuh"
#include "ft_tc.cuh"

namespace {

using namespace ft_tc;
using namespace ft_ce;

constexpr int TILE = 256;                 // rows (and most columns) of a pair's tile
constexpr int OPERAND_BYTES = 128 * BK * 2;
constexpr int STAGE_BYTES = 2 * OPERAND_BYTES;
constexpr int MAX_BUFFERS = 4;            // accumulators: two of 256 columns, four of 128

// STATS: row statistics.  EXP: statistics and E.  GRAD: g.  STORE: the sum.  FACTOR: the sum with every
// TILE of K scaled by its row's factor.
enum Epi { EPI_STATS, EPI_EXP, EPI_GRAD, EPI_STORE, EPI_FACTOR };
// Warps that drain.  FACTOR's empty an accumulator for every 2048 cycles of the tensor cores, which eight
// warps do not manage (4096 x 2048 x 24576: 345 us, 317 with sixteen, of 286 with no drain at all).
// The statistics bound small K (a tile takes eight warps 6100 cycles, sixteen 4400, the products 512
// for each 64 of K).  Where results are staged or slices summed, sixteen cost a stage or spills:
// eight there (8 x 4 KiB beside six stages; g at K = 2048 takes 412 thousand cycles, with sixteen and
// five stages 419).  With at most 128 rows (single CTAs) nothing is bound by the products: sixteen.
constexpr int drain_warps(int epi, bool two, bool pair) { return !pair || epi == EPI_FACTOR || (epi == EPI_STATS && !two) ? 16 : 8; }
// Statistics of a row that a tile leaves: one a warp of its quadrant.
constexpr int parts_of(int epi, bool two, bool pair) { return drain_warps(epi, two, pair) / 4; }
// The statistics' launches have two warps more, for the targets' logits.
constexpr int threads_of(int epi, bool two, bool pair) { return 64 + 32 * drain_warps(epi, two, pair) + (epi <= EPI_EXP ? 64 : 0); }
// Shared memory: the stages (six, or five, of 32 KiB; more where few rows or narrow tiles make them
// smaller), 4 KiB for each draining warp that stages results, the barriers (full, empty, tfull, tempty,
// one a quadrant), and room to align all that.
constexpr int MAX_STAGES = 16;
constexpr int epi_offset(int epi, bool pair) { return (epi == EPI_STATS || (pair && epi != EPI_FACTOR) ? 6 : 5) * STAGE_BYTES; }
constexpr int bar_offset(int epi, bool two, bool pair) {
  return epi_offset(epi, pair) + (epi == EPI_STATS ? 16384 : drain_warps(epi, two, pair) * 4096);
}
constexpr int BARRIERS = 2 * MAX_STAGES + 2 * MAX_BUFFERS + 4;
constexpr int smem_bytes(int epi, bool two, bool pair) { return bar_offset(epi, two, pair) + BARRIERS * 8 + 16 + 1024; }
// what E is held times: unscaled, a token below 2^-14 of its tile's maximum would fall under f16's normal range
constexpr float E_SCALE = 16384.f;
// k-blocks of 64 that are summed in tensor memory; 0: all.  TWO for STORE means slices, of TcProduct::slice blocks: 512
// of K with two planes.  With one plane its sums, which run over rows or the vocabulary and have no limit to
// their length, are taken over 2048 at most (128 groups of 16: 2^-16 of the sum is cut off; a million rows
// in one sum lose 0.4%): where there are more, by the instance in slices (2048 of 4096 rows x 896 x 151936,
// whole call: 2.01 -> 2.03 ms).
constexpr int slice_of(int epi, bool two) { return epi == EPI_FACTOR ? TILE / BK : two ? 8 : 0; }
constexpr int ONE_PLANE_SLICE = 32;

struct TcProduct {
  int M, N, K;
  int live_m, live_k;               // 1: that extent is the number of supervised rows
  int unpacked;                     // STATS, EXP, FACTOR: the rows are the caller's own, all M of them (no head, no scales)
  int carry;                        // STATS: one tile of rows; a pair joins its column tiles before it writes them
  int splits;                       // parts of K, each with a slab of its own
  int slice;                        // STORE in slices: k-blocks of one
  int tile_n;                       // columns of a tile: a multiple of 32 up to TILE
  int n_fast, band;                 // order of the tiles
  int a_bytes, stage_bytes;         // of A in a stage, of a stage (multiples of 1024)
  int stage_tx;                     // what the tile's CTAs load into one
  int terms;                        // plane pairs, the small ones first
  int a_plane[3], b_plane[3];
  int b_mn0, b_k0;                  // where N and K begin in B's tensor
  // EPI_STATS, EPI_GRAD
  Rows rw;
  float2* part;                     // [parts of a tile * column tiles][part_ld]: {maximum in log2 units, sum}
  int part_ld;
  int w_early;                      // STATS: W is the caller's, not made by a launch of this call
  int piece, pieces;                // STATS, EXP: which launch this is, of how many
  float* base_out;                  // FACTOR: a part of K chooses its own point of reference, [splits][part_ld]
  __half* wy;                       // EXP: the targets' columns of W, [planes][part_ld][wy_ld]
  int wy_ld;
  int v0, vocab;                    // first vocabulary column of the launch, columns in all
  // EPI_STATS, EPI_EXP: the operands again, for the targets' logits
  const __half *h, *w;              // value (k, plane) of a row at h + row * h_ld + plane * h_plane + k,
  long long h_ld, h_plane;          // W(k, v) at w + k * w_sk + v * w_sv + plane * w_plane
  long long w_sk, w_sv, w_plane;
  int h_planes, w_planes;
  // EPI_STORE
  int out_type;                     // FT_TYPE_*
  int accumulate;
  int unscale;                      // multiply by the scales of g and of the rows
  int transposed;                   // the output is [N, M]
  int out_x0, out_y0;
  void* direct;                     // when the output breaks a TMA rule: plain stores
  long long direct_ld;
};

template <bool PAIR>
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, uint32_t leader_bar, int c0, int c1, int c2) {
  if constexpr (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, "
        "{%3, %4, %5}], [%2];" ::"r"(dst), "l"((uint64_t)map), "r"(leader_bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"((uint64_t)map), "r"(leader_bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
__device__ __forceinline__ void l2_prefetch_3d(const CUtensorMap* map, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global [%0, {%1, %2, %3}];" ::"l"((uint64_t)map), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"((uint64_t)map),
               "r"(src), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ void tma_add_3d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2) {
  asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   (uint64_t)map),
               "r"(src), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
// Hands an accumulator back to the leader.  What has to be done before it are the warp's reads of tensor
// memory, which tcgen05.wait::ld and the fence before have seen to; no memory is published.
__device__ __forceinline__ void mbar_arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// the staging tile may be written again: the copies have read it
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
// ... all copies but the last have
__device__ __forceinline__ void bulk_wait_read_but_one() { asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Accumulator -> logit in log2 units: the operands' scales undone.  Their product may leave f32 at either end where
// every logit of the row that is neither 0 nor infinite does so too; 0 times a masked -inf, or
// infinity times 0, would be NaN.
__device__ __forceinline__ float logit_factor(float scales) {
  return fminf(fmaxf(scales * 1.4426950408889634f, 1.17549435e-38f), 3.40282347e38f);
}

// 2^((v - ref) c2) of a chunk in place, its sum.  (The difference first: 2^(v c2 - ref c2) with a rounded second
// product is not 1 at the maximum but off by half a step of the logits, 4e-5 at 1000, which a row that is
// sure of its target has as the error of its loss.)
__device__ __forceinline__ float exponentials(float (&v)[32], float ref, float c2) {
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < 32; k += 2) {
    fadd2(v[k], v[k + 1], v[k], v[k + 1], -ref, -ref);
    fmul2(v[k], v[k + 1], v[k], v[k + 1], c2, c2);
    v[k] = ex2(v[k]);
    v[k + 1] = ex2(v[k + 1]);
    s[k & 2] += v[k];
    s[(k & 2) + 1] += v[k + 1];
  }
  return (s[0] + s[1]) + (s[2] + s[3]);
}

// an arrival in every CTA of the tile once the products issued so far are complete
template <bool PAIR>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (PAIR) tc_commit_pair(bar, 3);
  else tc_commit(bar);
}

struct Unit { int mt, nt, sp; };
__device__ __forceinline__ Unit decode_unit(int u, int tiles_m, int tiles_n, const TcProduct& g) {
  Unit r;
  if (g.n_fast) {
    // parts of K slowest: the tiles that run together read the same slice of B
    r.nt = u % tiles_n;
    const int v = u / tiles_n;
    r.mt = v % tiles_m;
    r.sp = v / tiles_m;
  } else {
    const int per_band = g.band * tiles_n * g.splits;
    const int b = u / per_band, in = u - b * per_band;
    const int rows = min(g.band, tiles_m - b * g.band);
    r.mt = b * g.band + in % rows;
    const int v = in / rows;
    r.nt = v % tiles_n;
    r.sp = v / tiles_n;
  }
  return r;
}

// The 32 x 32 block of a warp (a row a lane, 32 consecutive f32 columns) -> its staging tile, in the
// 128-byte swizzle of the output map: 16-byte unit j of row r at unit j ^ (r & 7).
__device__ __forceinline__ void stage_f32(uint8_t* st, int lane, const float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    *(float4*)(st + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
}
// half `part` (32 columns, 64 bytes) of a 64-column f16 row
__device__ __forceinline__ void stage_f16(uint8_t* st, int lane, int part, const uint32_t (&h)[16]) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    *(uint4*)(st + lane * 128 + (((part * 4 + j) ^ (lane & 7)) << 4)) = make_uint4(h[4 * j], h[4 * j + 1], h[4 * j + 2], h[4 * j + 3]);
}

// h_row . W(:, target) of the packed rows [r0, r1) on f32 FMA.  The tensor core's sums are cut off, not
// rounded (see above): 4e-6 of a logit at K = 256, 4e-5 at 2048.  For most logits that is noise under
// the softmax, but the loss of a row that is sure of its target is as exact, relative to itself, as
// that one logit is exact in absolute terms.
// A warp takes R rows with 32 / R lanes each, a lane 16 values of K at a time.  [hidden, vocab] weights
// cost a 32-byte sector for every 2 bytes; with many rows (R = 32) all warps walk down K together,
// so that DRAM reads a row of W once for all targets in it (with a row a warp, 4096 rows x 2048
// read 540 MB for 100 MB of W and the products waited for them: 390 against 277 us).
// With g.wy the columns are kept, for the target's term of dh.
__device__ __forceinline__ void target_dots(const TcProduct& g, int r0, int r1, int worker, int workers, float scale, int lane) {
  const int rows = r1 - r0;
  int R = 1;
  if (g.w_sk != 1)
    while (R < 32 && rows > R * workers) R *= 2;
  const int share = 32 / R, sub = lane % share;
  for (int base = r0 + worker * R; base < r1; base += workers * R) {
    const int r = base + lane / share;
    const uint32_t y = r < r1 ? g.rw.target[r] : FT_MASKED_CE_SKIP;
    const bool on = y < (uint32_t)g.vocab;
    float acc = 0.f;
    for (int pw = 0; pw < g.w_planes && on; ++pw) {
      const __half* h = g.h + (long long)r * g.h_ld;
      const __half* w = g.w + pw * g.w_plane + (long long)y * g.w_sv;
      __half* keep = g.wy ? g.wy + ((long long)pw * g.part_ld + r) * g.wy_ld : nullptr;
      // (pitches of h and wy are multiples of 8, and so is W's where K is the contiguous index)
      for (int k0 = sub * 16; k0 < g.h_ld; k0 += share * 16) {
        uint4 hv[2], lv[2], wv[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int k = k0 + 8 * j;
          hv[j] = lv[j] = wv[j] = make_uint4(0u, 0u, 0u, 0u);
          if (k >= g.h_ld) continue;
          hv[j] = *(const uint4*)(h + k);
          if (g.h_planes == 2) lv[j] = *(const uint4*)(h + g.h_plane + k);
          if (g.w_sk == 1) {
            wv[j] = *(const uint4*)(w + k);
          } else {
            __half e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = k + i < g.K ? w[(k + i) * g.w_sk] : __float2half(0.f);
            wv[j] = *(const uint4*)e;
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const __half2 *a = (const __half2*)&hv[j], *l = (const __half2*)&lv[j], *b = (const __half2*)&wv[j];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 x = __half22float2(a[i]), z = __half22float2(l[i]), f = __half22float2(b[i]);
            acc = fmaf(x.x + z.x, f.x, acc);
            acc = fmaf(x.y + z.y, f.y, acc);
          }
          if (keep && k0 + 8 * j < g.h_ld) *(uint4*)(keep + k0 + 8 * j) = wv[j];
        }
      }
    }
    for (int o = share / 2; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (sub == 0 && on) g.rw.exact[r] = acc * logit_factor(g.rw.unscale ? scale * g.rw.unscale[r] : scale);
  }
}

template <bool PAIR, int EPI, bool A_MN, bool B_MN, bool TWO>
__global__ void __cluster_dims__(PAIR ? 2 : 1, 1, 1) __launch_bounds__(threads_of(EPI, TWO, PAIR), 1)
k_ce_gemm(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
          const __grid_constant__ CUtensorMap map_o, const __grid_constant__ TcProduct g, int* status) {
  constexpr int WARPS = drain_warps(EPI, TWO, PAIR), PARTS = parts_of(EPI, TWO, PAIR);
  constexpr int EPI_OFFSET = epi_offset(EPI, PAIR), BAR_OFFSET = bar_offset(EPI, TWO, PAIR);
  constexpr int CHUNKS = 32 / WARPS;        // of 32 columns, at most, a draining warp
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const uint32_t bar_full = base + BAR_OFFSET;
  const uint32_t bar_empty = bar_full + MAX_STAGES * 8;
  const uint32_t bar_tfull = bar_empty + MAX_STAGES * 8;
  const uint32_t bar_tempty = bar_tfull + MAX_BUFFERS * 8;
  const uint32_t bar_quad = bar_tempty + MAX_BUFFERS * 8;
  uint32_t* tmem_slot = (uint32_t*)(gbase + BAR_OFFSET + BARRIERS * 8);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int TM = PAIR ? 256 : 128;       // rows of a tile
  const uint32_t rank = PAIR ? cluster_ctarank() : 0;
  const int pair = PAIR ? blockIdx.x >> 1 : blockIdx.x, npairs = PAIR ? gridDim.x >> 1 : gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < MAX_STAGES; ++s) {
      mbar_init(bar_full + s * 8, 1);
      mbar_init(bar_empty + s * 8, 1);
    }
    for (int b = 0; b < MAX_BUFFERS; ++b) {
      mbar_init(bar_tfull + b * 8, 1);
      mbar_init(bar_tempty + b * 8, (PAIR ? 2 : 1) * WARPS);
    }
    for (int b = 0; b < 4; ++b) mbar_init(bar_quad + b * 8, WARPS / 4);   // the warps of a quadrant
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t stages = (uint32_t)min(MAX_STAGES, EPI_OFFSET / g.stage_bytes);
  if (EPI == EPI_STATS && g.w_early && warp == 0 && elect_one()) {
    // the first tile of W, where it is the caller's: on its way into L2 while the launch before this
    // one ends (nothing is read here, and L2 is where later writes to it would go too)
    const int first = pair / ((g.M + TM - 1) / TM);
    const int bn = first * g.tile_n + (PAIR ? (int)rank * (g.tile_n / 2) : 0);
    for (int k = 0; k < g.K && bn < g.N; k += BK) {
      if (B_MN) l2_prefetch_3d(&map_b, bn, k, 0);
      else l2_prefetch_3d(&map_b, k, bn, 0);
    }
  }
  ft_pdl_wait();
  ft_pdl_launch();

  const uint32_t lead_full = PAIR ? mapa_shared(bar_full, 0) : bar_full;
  const uint32_t lead_tempty = PAIR ? mapa_shared(bar_tempty, 0) : bar_tempty;
  const bool unpacked = (EPI <= EPI_EXP || EPI == EPI_FACTOR) && g.unpacked;
  const int live = unpacked ? g.M : g.rw.head->count;
  // no supervised row at all still makes one tile (of zeros): gradients are overwritten, not left
  const int tiles_m = g.live_m ? max(1, (live + TM - 1) / TM) : (g.M + TM - 1) / TM;
  const int tile_n = EPI == EPI_EXP || EPI == EPI_GRAD ? TILE : g.tile_n;
  const int tiles_n = (g.N + tile_n - 1) / tile_n;
  // accumulators in tensor memory, in turn
  const uint32_t buffers = tile_n <= 128 ? 4 : 2, buffer_cols = 512 / buffers;
  const int units = tiles_m * tiles_n * g.splits;
  const int kb_all = g.live_k ? max(1, (live + BK - 1) / BK) : (g.K + BK - 1) / BK;
  constexpr int SLICE = slice_of(EPI, TWO);
  const int slice = SLICE == 0 ? kb_all : EPI == EPI_STORE ? g.slice : SLICE;
  // FACTOR: parts of K begin with a tile of E
  constexpr int GRAIN = EPI == EPI_FACTOR ? SLICE : 1;
  const int grains = (kb_all + GRAIN - 1) / GRAIN;
  auto k_begin = [&](int sp) { return min(kb_all, GRAIN * (int)((long long)grains * sp / g.splits)); };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer (both CTAs)
    if (elect_one()) {
      uint32_t stage = 0, phase = 0;
      for (int u = pair; u < units && !*abort_flag; u += npairs) {
        const Unit un = decode_unit(u, tiles_m, tiles_n, g);
        const int kb0 = k_begin(un.sp), kb1 = k_begin(un.sp + 1);
        const int am = un.mt * TM + (int)rank * 128;
        const int bn = g.b_mn0 + un.nt * tile_n + (PAIR ? (int)rank * (tile_n / 2) : 0);
        const int b_cols = PAIR ? tile_n / 2 : tile_n;
        for (int s0 = kb0; s0 < kb1 && !*abort_flag; s0 += slice) {
          const int s1 = min(kb1, s0 + slice);
          for (int t = 0; t < g.terms; ++t) {
            const int pa = g.a_plane[t], pb = g.b_plane[t];
            for (int kb = s0; kb < s1; ++kb) {
              if (!mbar_wait(bar_empty + stage * 8, phase ^ 1, abort_flag, status, 21)) break;
              const uint32_t sa = base + stage * g.stage_bytes, sb = sa + g.a_bytes;
              const uint32_t bar = lead_full + stage * 8;
              if (rank == 0) mbar_expect_tx(bar_full + stage * 8, (uint32_t)g.stage_tx);
              if constexpr (A_MN) {
                load_3d<PAIR>(sa, &map_a, bar, am, kb * BK, pa);
                load_3d<PAIR>(sa + 8192, &map_a, bar, am + 64, kb * BK, pa);
              } else {
                load_3d<PAIR>(sa, &map_a, bar, kb * BK, am, pa);
              }
              if constexpr (B_MN) {
                for (int c = 0; c < b_cols; c += 64) load_3d<PAIR>(sb + c * 128, &map_b, bar, bn + c, g.b_k0 + kb * BK, pb);
              } else {
                load_3d<PAIR>(sb, &map_b, bar, g.b_k0 + kb * BK, bn, pb);
              }
              if (++stage == stages) { stage = 0; phase ^= 1; }
            }
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (leader only)
    if (rank == 0 && elect_one()) {
      const uint32_t idesc = make_idesc(TM, tile_n, 0, 0) | ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16);
      uint32_t stage = 0, phase = 0;
      int local = 0;
      for (int u = pair; u < units && !*abort_flag; u += npairs) {
        const Unit un = decode_unit(u, tiles_m, tiles_n, g);
        const int kb0 = k_begin(un.sp), kb1 = k_begin(un.sp + 1);
        for (int s0 = kb0; s0 < kb1 && !*abort_flag; s0 += slice, ++local) {
          const int todo = (min(kb1, s0 + slice) - s0) * g.terms;
          const uint32_t buf = (uint32_t)local & (buffers - 1), acc_phase = ((uint32_t)local / buffers) & 1;
          if (!mbar_wait(bar_tempty + buf * 8, acc_phase ^ 1, abort_flag, status, 22)) break;
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + buf * buffer_cols;
          for (int i = 0; i < todo; ++i) {
            if (!mbar_wait(bar_full + stage * 8, phase, abort_flag, status, 23)) break;
            tc_fence_after();
            const uint32_t sa = base + stage * g.stage_bytes, sb = sa + g.a_bytes;
            const uint64_t da = A_MN ? make_desc_mn_sw128(sa, 8192) : make_desc_sw128(sa);
            const uint64_t db = B_MN ? make_desc_mn_sw128(sb, 8192) : make_desc_sw128(sb);
#pragma unroll
            for (int k = 0; k < BK / UMMA_K; ++k) {
              const uint64_t ka = da + (uint64_t)(k * (A_MN ? 128 : 2)), kb = db + (uint64_t)(k * (B_MN ? 128 : 2));
              if constexpr (PAIR) tc_mma_f16_pair(d_tmem, ka, kb, idesc, (i > 0 || k > 0) ? 1u : 0u);
              else tc_mma_f16(d_tmem, ka, kb, idesc, (i > 0 || k > 0) ? 1u : 0u);
            }
            commit<PAIR>(bar_empty + stage * 8);
            if (++stage == stages) { stage = 0; phase ^= 1; }
          }
          if (*abort_flag) break;
          commit<PAIR>(bar_tfull + buf * 8);
        }
      }
    }
    __syncwarp();
  } else if (EPI <= EPI_EXP && warp >= 2 + WARPS) {
    // ------------------------------------------------------------------ the targets' logits
    const float scale = unpacked ? 1.f : g.rw.head->z_scale;
    // each launch of a vocabulary in pieces takes its share of the rows
    const int r0 = (int)((long long)live * g.piece / g.pieces), r1 = (int)((long long)live * (g.piece + 1) / g.pieces);
    target_dots(g, r0, r1, (int)blockIdx.x * 2 + warp - 2 - WARPS, (int)gridDim.x * 2, scale, lane);
  } else {
    // ------------------------------------------------------------------ epilogue (both CTAs)
    // A warp reaches the 32 TMEM lanes (rows) of its quadrant; the warps of a quadrant share the
    // columns, in chunks of 32.
    const int quad = warp & 3, grp = (warp - 2) >> 2;
    const int share = (tile_n / 32 + WARPS / 4 - 1) / (WARPS / 4), mine = max(0, min(share, tile_n / 32 - grp * share));
    uint8_t* st = gbase + EPI_OFFSET + (warp - 2) * 4096;
    const uint32_t st_addr = smem_u32(st);
    const uint32_t t_lane = tmem_base + ((uint32_t)(quad * 32) << 16) + grp * share * 32;
    const float z_scale = unpacked ? 1.f : g.rw.head->z_scale, c2_all = logit_factor(z_scale);
    // rows that a store may reach (packed ones: whole warps of them, their buffers end with a tile)
    const int rows_end = g.live_m ? live : g.M;
    int local = 0;
    uint32_t quad_phase = 0;
    uint32_t stored = 0;                                           // STORE: blocks handed to TMA, over all tiles
    float run_m = -INFINITY, run_s = 0.f, run_c2 = 0.f;              // the maximum as the accumulators have it
    for (int u = pair; u < units && !*abort_flag; u += npairs) {
      const Unit un = decode_unit(u, tiles_m, tiles_n, g);
      const int kb0 = k_begin(un.sp), kb1 = k_begin(un.sp + 1);
      const int y0 = un.mt * TM + (int)rank * 128 + quad * 32;   // first row of this warp
      const int row = y0 + lane;
      const int col = un.nt * tile_n + grp * share * 32;            // its first column, from the launch's first
      uint32_t target = FT_MASKED_CE_SKIP;
      float lse2 = 0.f, wg = 0.f, g_target = 0.f, alpha = 1.f, base2 = 0.f, c2 = c2_all;
      if constexpr (EPI <= EPI_GRAD) {
        if (row < live) {
          if (EPI <= EPI_EXP && g.rw.unscale) c2 = logit_factor(z_scale * g.rw.unscale[row]);
          target = g.rw.target[row] - (uint32_t)(g.v0 + col);      // relative to this warp's columns
          if constexpr (EPI == EPI_GRAD) {
            lse2 = g.rw.lse[row];
            wg = g.rw.weight[row] * g.rw.head->g_scale;
            g_target = wg * g.rw.at_target[row];
          }
        }
      } else if constexpr (EPI == EPI_STORE) {
        if (g.unscale) alpha = g.rw.head->g_unscale * g.rw.head->h_unscale;
      } else if (g.base_out) {
        float m = -INFINITY;
        if (row < live) {
#pragma unroll 8
          for (int s0 = kb0; s0 < kb1; s0 += SLICE)
            m = fmaxf(m, g.part[(size_t)(parts_of(EPI_EXP, false, PAIR) * (s0 / SLICE)) * g.part_ld + row].x);
          base2 = finite_max(m);
          if (un.nt == 0 && grp == 0) g.base_out[(size_t)un.sp * g.part_ld + row] = base2;
        }
      } else {
        if (row < live) base2 = g.rw.base[row];
      }
      // a warp without a supervised row hands the accumulators back as they come (g's rows behind the
      // last one are zeros that dW reads)
      const bool idle = (EPI <= EPI_EXP || EPI == EPI_FACTOR) && y0 >= live;
      if (EPI != EPI_STATS || !g.carry || u == pair) { run_m = -INFINITY; run_s = 0.f; }
      run_c2 = c2;                                                  // (a carried row keeps its scale)
      uint32_t low[TWO && (EPI == EPI_EXP || EPI == EPI_GRAD) ? 2 : 1][16];   // the second plane, until its store

      auto mask_columns = [&](int c0, float (&v)[32]) {
        const int left = g.vocab - (g.v0 + c0);                    // columns of the chunk inside the vocabulary
        if (left < 32) {
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (k >= left) v[k] = -INFINITY;
        }
      };
      auto max_of = [&](const float (&v)[32]) {
        float m[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int k = 4; k < 32; ++k) m[k & 3] = fmaxf(m[k & 3], v[k]);
        return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
      };
      auto store_f16_pair = [&](int x, int y, int plane) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          tma_store_3d(&map_o, st_addr, x, y, plane);
          bulk_commit();
        }
      };
      // chunk i of an f16 result (v: its values): two chunks make the 64 columns of a store
      auto put_f16 = [&](int i, int c0, const float (&v)[32]) {
        uint32_t hi[16];
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          hi[k >> 1] = pack_h2(v[k], v[k + 1]);
          if constexpr (TWO) {
            const float2 f = __half22float2(*(const __half2*)&hi[k >> 1]);
            low[i & 1][k >> 1] = pack_h2(v[k] - f.x, v[k + 1] - f.y);
          }
        }
        if ((i & 1) == 0) {
          if (lane == 0) bulk_wait_read();
          __syncwarp();
        }
        stage_f16(st, lane, i & 1, hi);
        if (i & 1) {
          store_f16_pair(c0 - 32, y0, 0);
          if constexpr (TWO) {
            if (lane == 0) bulk_wait_read();
            __syncwarp();
            stage_f16(st, lane, 0, low[0]);
            stage_f16(st, lane, 1, low[1]);
            store_f16_pair(c0 - 32, y0, 1);
          }
        }
      };

      // what happens to chunk i (columns col + 32 i .. + 31) of the finished sum
      auto finish = [&](int i, float (&v)[32]) {
        const int c0 = col + 32 * i;
        const uint32_t y = target - 32u * (uint32_t)i;
        if constexpr (EPI == EPI_STATS) {
          mask_columns(c0, v);
          const float m = fmaxf(run_m, max_of(v));
          if (y < 32u) {
            float z = 0.f;
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (y == (uint32_t)k) z = v[k];
            g.rw.picked[row] = z * c2;
          }
          const float ref = finite_max(m);
          run_s = run_s * ex2((run_m - ref) * c2) + exponentials(v, ref, c2);
          run_m = m;
        } else if constexpr (EPI == EPI_EXP) {
          // (run_m is the whole tile's maximum by now)
          mask_columns(c0, v);
          const float ref = finite_max(run_m);
          if (y < 32u) {
            // The target has no part in E: its whole gradient, p - 1, is applied from the loss.  (Both parts, p by
            // E W and -1 later, would leave a sure row's gradient to the last bits of their sums.)
            float z = 0.f;
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (y == (uint32_t)k) {
                z = v[k];
                v[k] = -INFINITY;
              }
            g.rw.picked[row] = z * c2;
            run_s += ex2((z - ref) * c2);
          }
          run_s += exponentials(v, ref, c2);
#pragma unroll
          for (int k = 0; k < 32; k += 2) fmul2(v[k], v[k + 1], v[k], v[k + 1], E_SCALE, E_SCALE);
          put_f16(i, c0, v);
        } else if constexpr (EPI == EPI_GRAD) {
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            v[k] = wg * ex2(fmaf(v[k], c2, -lse2));
            // (p - 1 would be as wrong as the tensor cores' sum: a row that is sure of its target loses it all)
            if (y == (uint32_t)k) v[k] = g_target;
            // rows behind the last supervised one hold zeros: they are part of dW's K
            if (row >= live) v[k] = 0.f;
          }
          put_f16(i, c0, v);
        } else {
          if (c0 >= g.N || y0 >= rows_end) return;                 // the whole block lies outside
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] *= alpha;
          if (g.direct != nullptr) {
            // a pitch or a base that TMA cannot address
            if (g.transposed) {
              // a lane is a column of the output: 32 consecutive ones a store
              if (row < rows_end) {
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                  const long long at = (long long)(c0 + k) * g.direct_ld + g.out_x0 + row;
                  if (c0 + k >= g.N) break;
                  if (g.out_type == FT_TYPE_F16) ((__half*)g.direct)[at] = __float2half_rn(v[k]);
                  else ((float*)g.direct)[at] = v[k];
                }
              }
              return;
            }
            // a row at a time, a column a lane
            __syncwarp();
            stage_f32(st, lane, v);
            __syncwarp();
            if (c0 + lane < g.N) {
#pragma unroll 8
              for (int r = 0; r < 32; ++r) {
                if (y0 + r >= rows_end) break;
                const float x = *(const float*)(st + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
                const long long at = (long long)(g.out_y0 + y0 + r) * g.direct_ld + g.out_x0 + c0 + lane;
                if (g.out_type == FT_TYPE_F16) ((__half*)g.direct)[at] = __float2half_rn(x);
                else ((float*)g.direct)[at] = x;
              }
            }
            return;
          }
          // An f16 block fills half of the staging tile: the halves take turns, over all tiles and the blocks
          // left out (with the chunk's number an odd count of them would put two blocks in a row in one
          // half, and the wait below lets the last copy go on reading).
          uint8_t* to = st + (g.out_type == FT_TYPE_F16 ? (stored++ & 1) * 2048 : 0);
          if (lane == 0) {
            if (g.out_type == FT_TYPE_F16) bulk_wait_read_but_one();
            else bulk_wait_read();
          }
          __syncwarp();
          if (g.transposed) {
            // the block turned over: output row k in staging row k, this lane's value in column `lane`
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              if (g.out_type == FT_TYPE_F16) *(__half*)(to + k * 64 + (((lane >> 3) ^ ((k >> 1) & 3)) << 4) + (lane & 7) * 2) = __float2half_rn(v[k]);
              else *(float*)(to + k * 128 + (((lane >> 2) ^ (k & 7)) << 4) + (lane & 3) * 4) = v[k];
            }
          } else if (g.out_type == FT_TYPE_F16) {
            uint32_t h[16];
#pragma unroll
            for (int k = 0; k < 32; k += 2) h[k >> 1] = pack_h2(v[k], v[k + 1]);
            // 32 columns are 64 bytes: a tile of its own swizzle (64-byte rows)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *(uint4*)(to + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = make_uint4(h[4 * j], h[4 * j + 1], h[4 * j + 2], h[4 * j + 3]);
          } else {
            stage_f32(to, lane, v);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            const int x = g.out_x0 + (g.transposed ? y0 : c0), y = g.out_y0 + (g.transposed ? c0 : y0);
            if (g.accumulate) tma_add_3d(&map_o, smem_u32(to), x, y, un.sp);
            else tma_store_3d(&map_o, smem_u32(to), x, y, un.sp);
            bulk_commit();
          }
        }
      };
      // EXP: the maximum over the tile's 256 columns, half of which the quadrant's other warp holds
      auto meet = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_quad + quad * 8);
        const bool ok = mbar_wait(bar_quad + quad * 8, quad_phase, abort_flag, status, 25);
        quad_phase ^= 1;
        return ok;
      };
      auto join_max = [&](float m) {
        float* slot = (float*)(gbase + EPI_OFFSET) + (warp - 2) * 1024;       // the staging tiles, free at this point
        if (lane == 0) bulk_wait_read();
        __syncwarp();
        slot[lane] = m;
        if (!meet()) return m;
#pragma unroll
        for (int j = 1; j < WARPS / 4; ++j)
          m = fmaxf(m, ((const float*)(gbase + EPI_OFFSET))[((warp - 2 + 4 * j) % WARPS) * 1024 + lane]);
        meet();
        return m;
      };
      auto release = [&](uint32_t buf) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIR) mbar_arrive_remote(lead_tempty + buf * 8);
          else mbar_arrive(lead_tempty + buf * 8);
        }
      };

      if constexpr (SLICE > 0) {
        float acc[CHUNKS][32];
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
          for (int k = 0; k < 32; ++k) acc[i][k] = 0.f;
        float* factors = (float*)st;                                  // FACTOR: of the next 32 slices, [slice][row]
        if constexpr (EPI == EPI_FACTOR) {
          if (lane == 0) bulk_wait_read();
          __syncwarp();
        }
        for (int s0 = kb0; s0 < kb1; s0 += slice, ++local) {
          const uint32_t buf = (uint32_t)local & (buffers - 1), acc_phase = ((uint32_t)local / buffers) & 1;
          float f = 1.f;
          if constexpr (EPI == EPI_FACTOR) {
            const int at = ((s0 - kb0) / SLICE) & 31;
            if (at == 0 && !idle) {
              // 32 slices' at once: a load from memory in every slice, even one asked for a slice
              // ahead, kept each at 3900 cycles (390 us for the product above)
#pragma unroll 4
              for (int j = 0; j < 32 && s0 + SLICE * j < kb1; ++j) {
                const float m = row < live ? g.part[(size_t)(parts_of(EPI_EXP, false, PAIR) * (s0 / SLICE + j)) * g.part_ld + row].x : 0.f;
                // (a difference of two infinities belongs to a row of NaN anyway)
                factors[j * 32 + lane] = ex2(finite_max(m) - base2) * (1.f / E_SCALE);
              }
            }
            f = factors[at * 32 + lane];
          }
          if (!mbar_wait(bar_tfull + buf * 8, acc_phase, abort_flag, status, 24)) break;
          tc_fence_after();
          if (idle) {
            release(buf);
            continue;
          }
          // 16 columns at a time
#pragma unroll
          for (int i = 0; i < 2 * CHUNKS; ++i) {
            if (i >= 2 * mine) continue;
            uint32_t r[16];
            tc_ld16(t_lane + buf * buffer_cols + i * 16, r);
            tc_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; k += 2) {
              float& a0 = acc[i >> 1][(i & 1) * 16 + k];
              float& a1 = acc[i >> 1][(i & 1) * 16 + k + 1];
              const float x0 = __uint_as_float(r[k]), x1 = __uint_as_float(r[k + 1]);
              if constexpr (EPI == EPI_FACTOR) ffma2(a0, a1, f, f, x0, x1, a0, a1);
              else fadd2(a0, a1, a0, a1, x0, x1);
            }
          }
          release(buf);
        }
        if (*abort_flag) break;
        if (idle) continue;
        if constexpr (EPI == EPI_EXP) {
          float m = -INFINITY;
#pragma unroll
          for (int i = 0; i < CHUNKS; ++i) {
            mask_columns(col + 32 * i, acc[i]);
            m = fmaxf(m, max_of(acc[i]));
          }
          run_m = join_max(m);
        }
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i)
          if (i < mine) finish(i, acc[i]);
      } else {
        const uint32_t buf = (uint32_t)local & (buffers - 1), acc_phase = ((uint32_t)local / buffers) & 1;
        ++local;
        if (!mbar_wait(bar_tfull + buf * 8, acc_phase, abort_flag, status, 24)) break;
        tc_fence_after();
        if (idle) {
          release(buf);
          continue;
        }
        if constexpr (EPI == EPI_EXP) {
          float m = -INFINITY;
#pragma unroll
          for (int i = 0; i < CHUNKS; ++i) {
            float v[32];
            tc_ld32(t_lane + buf * buffer_cols + i * 32, *(uint32_t(*)[32])v);
            tc_wait_ld();
            mask_columns(col + 32 * i, v);
            m = fmaxf(m, max_of(v));
          }
          run_m = join_max(m);
        }
        if (mine == 0) release(buf);
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
          if (i >= mine) continue;
          float v[32];
          tc_ld32(t_lane + buf * buffer_cols + i * 32, *(uint32_t(*)[32])v);
          tc_wait_ld();
          if (i == mine - 1) release(buf);                         // all chunks have been read
          finish(i, v);
        }
      }
      if constexpr (EPI <= EPI_EXP) {
        if (EPI != EPI_STATS || !g.carry) g.part[(size_t)(un.nt * PARTS + grp) * g.part_ld + row] = make_float2(run_m * c2, run_s);
      }
    }
    if (EPI == EPI_STATS && g.carry && pair < units) {
      const int row = (int)rank * 128 + quad * 32 + lane;
      g.part[(size_t)(pair * PARTS + grp) * g.part_ld + row] = make_float2(run_m * run_c2, run_s);
    }
    // what was stored is complete before the launch ends
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
    __syncthreads();
  }
  if constexpr (PAIR) cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
  }
}

// ------------------------------------------------------------------------------ around the products
// The loss of a row from its log-sum-exp ref + l2 and its target's logit, as the tensor cores summed it (z)
// and exactly (z + d), all in log2 units: the sum with that logit replaced,
//   log(e^(lse - z) + e^d - 1) - d = (lse - z) - d + log(1 + p (e^d - 1)),  p = e^(z - lse)
// (ref - z) first: a row that is sure of its target loses nothing to the size of its logits.
__device__ __forceinline__ float loss_of(float ref, float l2, float z, float exact) {
  const float above = ((ref - z) + l2) * 0.6931471805599453f;
  const float d = exact == z ? 0.f : (exact - z) * 0.6931471805599453f;   // (both may be -inf: the loss is +inf)
  return above - d + log1pf(expf(-above) * expm1f(d));
}

// Joins the column tiles' {maximum, sum} of 32 rows, tiles over the warps in a fixed order, with what
// the pieces before (not `first`) have left; after the last piece writes the row's log-sum-exp (in
// log2 units, as the gradient's epilogue wants it) and its loss.
// With `acc` (E is in use): sets the point R that the row's E W is scaled against.  It stays the maximum
// of the first piece, and f32 carries what later pieces are above it, unless that is 2^64 or
// more: then it moves, and the row's sums so far are scaled down.
constexpr int JOIN_WARPS = 32;            // at most; few parts of many rows take eight
__global__ void __launch_bounds__(32 * JOIN_WARPS)
k_ce_join(const float2* __restrict__ part, int part_ld, int parts, Rows rw, int unpacked_rows, int first, int last,
          int vocab, float* __restrict__ row_loss, float* __restrict__ acc, size_t slab, int splits, int ld, int H) {
  __shared__ float2 red[JOIN_WARPS][32];
  __shared__ float shrink[32];
  ft_pdl_wait();
  ft_pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int row = blockIdx.x * 32 + lane;
  const int live = unpacked_rows ? unpacked_rows : rw.head->count;
  if ((int)blockIdx.x * 32 >= live) return;
  float m = -INFINITY, s = 0.f;
  constexpr int AT_ONCE = 16;
  for (int p0 = warp; p0 < parts; p0 += AT_ONCE * warps) {
    float2 v[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const int p = p0 + j * warps;
      v[j] = p < parts ? part[(size_t)p * part_ld + row] : make_float2(-INFINITY, 0.f);
    }
    float mn = m;
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) mn = fmaxf(mn, v[j].x);
    const float ref = finite_max(mn);
    s *= ex2(m - ref);
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) s += v[j].y * ex2(v[j].x - ref);
    m = mn;
  }
  red[warp][lane] = make_float2(m, s);
  __syncthreads();
  if (warp == 0) {
    shrink[lane] = 1.f;
    if (row < live) {
      const float2 old = first ? make_float2(-INFINITY, 0.f) : rw.stat[row];
      float M = old.x;
      for (int w = 0; w < warps; ++w) M = fmaxf(M, red[w][lane].x);
      const float ref = finite_max(M);
      float S = old.y * ex2(old.x - ref);
      for (int w = 0; w < warps; ++w) S += red[w][lane].y * ex2(red[w][lane].x - ref);
      if (!last) rw.stat[row] = make_float2(M, S);
      if (acc) {
        if (first) {
          rw.base[row] = ref;
        } else if (ref > rw.base[row] + 64.f) {
          shrink[lane] = ex2(rw.base[row] - ref);
          rw.base[row] = ref;
        }
      }
      if (last) {
        const float l2 = log2f(S);
        if (!unpacked_rows) rw.lse[row] = ref + l2;
        float loss = 0.f;
        if (rw.target[row] < (uint32_t)vocab) {
          loss = loss_of(ref, l2, rw.picked[row], rw.exact[row]);
        }
        row_loss[unpacked_rows ? row : rw.source[row]] = loss;
        if (!unpacked_rows) rw.at_target[row] = expm1f(-loss);
        if (acc) {
          // the gradient at the target, p - 1, is -(1 - e^-loss), exact for a row that is sure of it
          const float w = rw.weight[row] * rw.head->w_unscale;
          rw.stat[row] = make_float2(w * ex2(rw.base[row] - rw.lse[row]), w * rw.at_target[row]);
        }
      }
    }
  }
  if (!acc || first) return;
  __syncthreads();
  for (int r = 0; r < 32; ++r) {
    const float f = shrink[r];
    if (f == 1.f) continue;
    for (int sp = 0; sp < splits; ++sp)
      for (int c = threadIdx.x; c < H; c += blockDim.x) acc[sp * slab + (size_t)(blockIdx.x * 32 + r) * ld + c] *= f;
  }
}

// E -> g in place, both planes, for a vocabulary that is one piece: g = w 2^(ref - lse) 2^-14 E, with the
// gradient at the target, where E is zero, as k_ce_join has it, and zero rows up to a K block of dW.
// One read and one write of E against a second product for the logits (makes_g_in_place).  With one plane it would round g's values twice, so FT_GEMM_F16 has no use for it.
__global__ void __launch_bounds__(256)
k_ce_normalise(__half* __restrict__ e, size_t plane, int ld, const float2* __restrict__ part, int part_ld, Rows rw, int cols,
               int tile_parts) {
  ft_pdl_wait();
  ft_pdl_launch();
  const int live = rw.head->count, end = max(64, (live + 63) / 64 * 64);
  for (int r = blockIdx.y; r < end; r += gridDim.y) {
    float lse2 = 0.f, w = 0.f, at_target = 0.f;
    uint32_t y = FT_MASKED_CE_SKIP;
    if (r < live) {
      lse2 = rw.lse[r];
      w = rw.weight[r] * rw.head->g_scale;
      y = rw.target[r];
      at_target = w * rw.at_target[r];
    }
    for (int c = (blockIdx.x * 256 + threadIdx.x) * 8; c < cols; c += gridDim.x * 2048) {
      __half* p = e + (size_t)r * ld + c;
      uint4 hi = make_uint4(0u, 0u, 0u, 0u), lo = hi;
      if (r < live) {
        const float f = w * (1.f / E_SCALE) * ex2(finite_max(part[(size_t)(tile_parts * (c / TILE)) * part_ld + r].x) - lse2);
        hi = *(const uint4*)p;
        lo = *(const uint4*)(p + plane);
        uint32_t* a = (uint32_t*)&hi;
        uint32_t* b = (uint32_t*)&lo;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 x = __half22float2(*(const __half2*)&a[k]), z = __half22float2(*(const __half2*)&b[k]);
          float g0 = f * (x.x + z.x), g1 = f * (x.y + z.y);
          if (y == (uint32_t)(c + 2 * k)) g0 = at_target;
          if (y == (uint32_t)(c + 2 * k + 1)) g1 = at_target;
          a[k] = pack_h2(g0, g1);
          const float2 q = __half22float2(*(const __half2*)&a[k]);
          b[k] = pack_h2(g0 - q.x, g1 - q.y);
        }
      }
      *(uint4*)p = hi;
      *(uint4*)(p + plane) = lo;
    }
  }
}

// Largest finite magnitudes of W (first `w_blocks` blocks) and of the supervised rows
// (the others), one value a block.
__global__ void __launch_bounds__(256)
k_ce_amax(const float* __restrict__ w, long long n, int w_blocks, const float* __restrict__ hidden,
          const uint32_t* __restrict__ targets, int rows, int H, Rows rw) {
  __shared__ float red[8];
  ft_pdl_wait();
  ft_pdl_launch();
  float m = 0.f;
  if ((int)blockIdx.x < w_blocks) {
    const long long step = (long long)w_blocks * 256;
    long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    auto see = [&](float x) {
      const float a = fabsf(x);
      if (a < INFINITY) m = fmaxf(m, a);
    };
    if (((uintptr_t)w & 15) == 0) {
      constexpr int AT_ONCE = 4;
      const float4* w4 = (const float4*)w;
      for (; i < n / 4; i += AT_ONCE * step) {
        float4 v[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) v[j] = i + j * step < n / 4 ? w4[i + j * step] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) { see(v[j].x); see(v[j].y); see(v[j].z); see(v[j].w); }
      }
      i = n / 4 * 4 + (long long)blockIdx.x * 256 + threadIdx.x;
    }
    for (; i < n; i += step) see(w[i]);
  } else {
    for (int r = blockIdx.x - w_blocks; r < rows; r += gridDim.x - w_blocks) {
      if (targets[r] == FT_MASKED_CE_SKIP) continue;
      for (int c = threadIdx.x; c < H; c += 256) {
        const float x = fabsf(hidden[(size_t)r * H + c]);
        if (x < INFINITY) m = fmaxf(m, x);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < 8; ++k) m = fmaxf(m, red[k]);
    if ((int)blockIdx.x < w_blocks) rw.w_max[blockIdx.x] = m;
    else rw.h_max[blockIdx.x - w_blocks] = m;
  }
}

// Eight values from any place of a tensor that begins at `first`, of which the first n are there; the rest are zeros.
__device__ __forceinline__ void load_eight(const float* p, const float*, int n, float (&v)[8]) {
  if (n >= 8 && ((uintptr_t)p & 15) == 0) {
    const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = k < n ? p[k] : 0.f;
}
// f16 rows of an odd length begin between two words: whole words, shifted (the neighbours that come along
// are values of the same tensor)
__device__ __forceinline__ void load_eight(const __half* p, const __half* first, int n, float (&v)[8]) {
  if (n > 8 && p > first) {
    const bool odd = (uintptr_t)p & 2;
    const uint32_t* q = (const uint32_t*)((uintptr_t)p & ~(uintptr_t)3);
    uint32_t w[5];
#pragma unroll
    for (int k = 0; k < 5; ++k) w[k] = k < 4 || odd ? q[k] : 0u;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t x = odd ? __funnelshift_r(w[k], w[k + 1], 16) : w[k];
      const float2 f = __half22float2(*(const __half2*)&x);
      v[2 * k] = f.x;
      v[2 * k + 1] = f.y;
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = k < n ? (float)p[k] : 0.f;
}

// W [rows, cols] -> f16 planes [planes][rows][ld], times the power of two of its largest value; block
// (bx, by) of (gx, ...): a warp takes 1024 columns of a row
template <typename T>
__device__ __forceinline__ void weight_block(int bx, int by, int gx, const T* __restrict__ w, int rows, int cols,
                                             __half* __restrict__ out, int ld, int planes, const float* __restrict__ w_max,
                                             int w_parts) {
  __shared__ float red[8];
  const float S = sizeof(T) == 4 ? power_for(block_max_of(w_max, w_parts, red), OPERAND_EXP) : 1.f;
  const size_t plane = (size_t)rows * ld;
  const int c_end = min(ld, (by + 1) * 1024);
  for (int r = bx * 8 + threadIdx.x / 32; r < rows; r += gx * 8)
  for (int c = by * 1024 + (threadIdx.x % 32) * 8; c < c_end; c += 256) {
    float v[8];
    load_eight(w + (size_t)r * cols + c, w, cols - c, v);
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      const float a = v[k] * S, b = v[k + 1] * S;
      hi[k >> 1] = pack_h2(a, b);
      const float2 f = __half22float2(*(const __half2*)&hi[k >> 1]);
      lo[k >> 1] = pack_h2(a - f.x, b - f.y);
    }
    *(uint4*)(out + (size_t)r * ld + c) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    if (planes == 2) *(uint4*)(out + plane + (size_t)r * ld + c) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
}

// The operands as the products want them: the first `gather_blocks` blocks pack rows, the others (a grid of
// gx x ...; none where W is taken as it lies) write W's planes.
struct PackArgs {
  const void *hidden, *weight;
  const uint32_t* targets;
  const float* weights;
  float grad_scale;
  int rows, H, per, gather_blocks, gx;
  Rows rw;
  __half* h;
  int h_ld, plane_rows, h_planes, h_parts, w_parts;
  float* row_loss;
  __half* w;
  int w_rows, w_cols, w_ld, w_planes;
};
template <typename TH, typename TW>
__global__ void __launch_bounds__(GATHER_THREADS)
k_ce_pack(const __grid_constant__ PackArgs a) {
  ft_pdl_wait();
  ft_pdl_launch();
  const int block = blockIdx.x;
  if (block < a.gather_blocks) {
    gather_block<TH, __half>(block, a.gather_blocks, (const TH*)a.hidden, a.targets, a.weights, a.grad_scale, a.rows, a.H, a.per,
                             a.rw, a.h, a.h_ld, a.plane_rows, a.h_planes, a.h_parts, a.w_parts, a.row_loss);
  } else {
    const int b = block - a.gather_blocks;
    weight_block<TW>(b % a.gx, b / a.gx, a.gx, (const TW*)a.weight, a.w_rows, a.w_cols, a.w, a.w_ld, a.w_planes, a.rw.w_max,
                     a.w_parts);
  }
}

// Four columns of a row over the slabs, in their order, each times its factor (none: 1); eight loads at
// once, since small calls have many slabs and little else to wait for.
__device__ __forceinline__ float4 sum_slabs(const float* __restrict__ p, size_t slab, int splits, const float* factor) {
  constexpr int AT_ONCE = 8;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < splits; s0 += AT_ONCE) {
    float4 x[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j)
      if (s0 + j < splits) x[j] = *(const float4*)(p + (s0 + j) * slab);
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j)
      if (s0 + j < splits) {
        const float f = factor ? factor[s0 + j] : 1.f;
        v.x = fmaf(f, x[j].x, v.x); v.y = fmaf(f, x[j].y, v.y); v.z = fmaf(f, x[j].z, v.z); v.w = fmaf(f, x[j].w, v.w);
      }
  }
  return v;
}

// grad_hidden[r] = unscale * (sum of the splits' slabs) at the row's packed place, zero where skipped
template <typename T>
__global__ void __launch_bounds__(256)
k_ce_scatter(const float* __restrict__ acc, size_t slab, int splits, int ld, Rows rw, int H, int rows, T* __restrict__ out) {
  ft_pdl_wait();
  ft_pdl_launch();
  const float alpha = rw.head->g_unscale * rw.head->w_unscale;
  // a warp takes 128 columns of a row
  const int c = blockIdx.y * 128 + (threadIdx.x % 32) * 4;
  if (c >= ld) return;
  for (int r = blockIdx.x * 8 + threadIdx.x / 32; r < rows; r += gridDim.x * 8) {
    const int at = rw.place[r];
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (at >= 0) {
      const float* p = acc + (size_t)at * ld + c;
      v = sum_slabs(p, slab, splits, nullptr);
    }
    T* o = out + (size_t)r * H + c;
    const float e[4] = {v.x * alpha, v.y * alpha, v.z * alpha, v.w * alpha};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (c + k < H) {
        if constexpr (sizeof(T) == 2) o[k] = __float2half_rn(e[k]);
        else o[k] = e[k];
      }
  }
}

// The same for E: stat holds the factors of the row's sums and of its target's column of W.
template <typename T>
__global__ void __launch_bounds__(256)
k_ce_scatter_exp(const float* __restrict__ acc, size_t slab, int splits, int ld, Rows rw, const __half* __restrict__ wy,
                 size_t wy_plane, int wy_ld, int w_planes, int H, int rows, T* __restrict__ out) {
  ft_pdl_wait();
  ft_pdl_launch();
  // a warp takes 128 columns of a row
  const int c = blockIdx.y * 128 + (threadIdx.x % 32) * 4;
  if (c >= ld) return;
  for (int r = blockIdx.x * 8 + threadIdx.x / 32; r < rows; r += gridDim.x * 8) {
    const int at = rw.place[r];
    float e[4] = {0.f, 0.f, 0.f, 0.f};
    if (at >= 0) {
      const float2 f = rw.stat[at];
      const float* p = acc + (size_t)at * ld + c;
      const float4 v = sum_slabs(p, slab, splits, nullptr);
      uint2 y[2] = {make_uint2(0u, 0u), make_uint2(0u, 0u)};
      // a target outside the vocabulary has no column (wy's pitch is a multiple of 8)
      if (f.y != 0.f) {
        y[0] = *(const uint2*)(wy + (size_t)at * wy_ld + c);
        if (w_planes == 2) y[1] = *(const uint2*)(wy + wy_plane + (size_t)at * wy_ld + c);
      }
      const float2 y0 = __half22float2(*(const __half2*)&y[0].x), y1 = __half22float2(*(const __half2*)&y[0].y);
      const float2 z0 = __half22float2(*(const __half2*)&y[1].x), z1 = __half22float2(*(const __half2*)&y[1].y);
      e[0] = fmaf(f.x, v.x, f.y * (y0.x + z0.x));
      e[1] = fmaf(f.x, v.y, f.y * (y0.y + z0.y));
      e[2] = fmaf(f.x, v.z, f.y * (y1.x + z1.x));
      e[3] = fmaf(f.x, v.w, f.y * (y1.y + z1.y));
    }
    T* o = out + (size_t)r * H + c;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (c + k < H) {
        if constexpr (sizeof(T) == 2) o[k] = __float2half_rn(e[k]);
        else o[k] = e[k];
      }
  }
}

// All that is left after E W when the vocabulary was one piece: the join of the statistics, the loss and
// grad_hidden, for four rows a block.  Every part of K has its own point of reference (base, [splits]
// [part_ld]).  `unpacked` rows are the caller's own, with their targets and weights.
template <typename T>
__global__ void __launch_bounds__(256)
k_ce_finish(const float2* __restrict__ part, int part_ld, int parts, Rows rw, int unpacked, const float* __restrict__ weights,
            float grad_scale, int vocab, float* __restrict__ row_loss, const float* __restrict__ base,
            const float* __restrict__ acc, size_t slab, int splits, int ld, const __half* __restrict__ wy, size_t wy_plane,
            int wy_ld, int w_planes, int H, int rows, T* __restrict__ out) {
  constexpr int ROWS = 4, MAX_SPLITS = 64;
  __shared__ float2 red[8][ROWS];
  __shared__ float factor[ROWS][MAX_SPLITS], onehot[ROWS], lse_of[ROWS], weight_of[ROWS];
  ft_pdl_wait();
  ft_pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int mine = blockIdx.x * ROWS + (threadIdx.x & 3);            // (source row)
  int at = -1;
  if (mine < rows) at = unpacked ? (rw.target[mine] == FT_MASKED_CE_SKIP ? -1 : mine) : rw.place[mine];
  float m = -INFINITY, s = 0.f;
  if (at >= 0) {
    constexpr int AT_ONCE = 8;
    for (int p0 = threadIdx.x >> 2; p0 < parts; p0 += AT_ONCE * 64) {
      float2 v[AT_ONCE];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) v[j] = p0 + 64 * j < parts ? part[(size_t)(p0 + 64 * j) * part_ld + at] : make_float2(-INFINITY, 0.f);
      float mn = m;
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) mn = fmaxf(mn, v[j].x);
      const float ref = finite_max(mn);
      s *= ex2(m - ref);
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) s += v[j].y * ex2(v[j].x - ref);
      m = mn;
    }
  }
#pragma unroll
  for (int o = 16; o >= 4; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    const float mn = fmaxf(m, m2), ref = finite_max(mn);
    s = s * ex2(m - ref) + s2 * ex2(m2 - ref);
    m = mn;
  }
  if (lane < ROWS) red[warp][lane] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x < ROWS && mine < rows) {
    const int i = threadIdx.x;
    float loss = 0.f;
    if (at >= 0) {
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < 8; ++w) M = fmaxf(M, red[w][i].x);
      const float ref = finite_max(M);
      float S = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) S += red[w][i].y * ex2(red[w][i].x - ref);
      const float l2 = log2f(S), lse2 = ref + l2;
      const float w = unpacked ? weights[at] * grad_scale : rw.weight[at] * rw.head->w_unscale;
      float b = 0.f;
      if (rw.target[at] < (uint32_t)vocab) {
        loss = loss_of(ref, l2, rw.picked[at], rw.exact[at]);
        b = expm1f(-loss);
      }
      onehot[i] = w * b;
      lse_of[i] = lse2;
      weight_of[i] = w;
    }
    if (blockIdx.y == 0) row_loss[mine] = loss;
  }
  __syncthreads();
  if (at >= 0)
    for (int sp = threadIdx.x >> 2; sp < splits; sp += 64)
      factor[threadIdx.x & 3][sp] = weight_of[threadIdx.x & 3] * ex2(base[(size_t)sp * part_ld + at] - lse_of[threadIdx.x & 3]);
  __syncthreads();
  // two warps a row, 256 columns a block of grid.y (which has the rows' numbers from its own join)
  const int i = warp >> 1, r = blockIdx.x * ROWS + i;
  if (r >= rows) return;
  const int place = __shfl_sync(0xffffffffu, at, i);                 // lane i holds row i
  const float b = place >= 0 ? onehot[i] : 0.f;
  for (int c = (blockIdx.y * 2 + (warp & 1)) * 128 + lane * 4; c < ld; c += gridDim.y * 256) {
    float e[4] = {0.f, 0.f, 0.f, 0.f};
    if (place >= 0) {
      uint2 y[2] = {make_uint2(0u, 0u), make_uint2(0u, 0u)};
      // a target outside the vocabulary has no column (wy's pitch is a multiple of 8)
      if (b != 0.f) {
        y[0] = *(const uint2*)(wy + (size_t)place * wy_ld + c);
        if (w_planes == 2) y[1] = *(const uint2*)(wy + wy_plane + (size_t)place * wy_ld + c);
      }
      const float4 v = sum_slabs(acc + (size_t)place * ld + c, slab, splits, factor[i]);
      const float2 y0 = __half22float2(*(const __half2*)&y[0].x), y1 = __half22float2(*(const __half2*)&y[0].y);
      const float2 z0 = __half22float2(*(const __half2*)&y[1].x), z1 = __half22float2(*(const __half2*)&y[1].y);
      e[0] = fmaf(b, y0.x + z0.x, v.x); e[1] = fmaf(b, y0.y + z0.y, v.y);
      e[2] = fmaf(b, y1.x + z1.x, v.z); e[3] = fmaf(b, y1.y + z1.y, v.w);
    }
    T* o = out + (size_t)r * H + c;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (c + k < H) {
        if constexpr (sizeof(T) == 2) o[k] = __float2half_rn(e[k]);
        else o[k] = e[k];
      }
  }
}

// ------------------------------------------------------------------------------ host side
int make_map3(FtContext* ctx, CUtensorMap* map, const void* ptr, bool f32, uint64_t inner, uint64_t rows, uint64_t planes,
              uint64_t ld, uint32_t box_inner, uint32_t box_rows, CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
  auto encode = (PFN_cuTensorMapEncodeTiled_v12000)ctx->encode_tiled;
  if (!encode) {
    ft_set_error("linear_cross_entropy: cuTensorMapEncodeTiled is not available from this driver");
    return FT_ERR_UNSUPPORTED;
  }
  const uint64_t size = f32 ? 4 : 2;
  cuuint64_t dims[3] = {inner, rows, planes};
  cuuint64_t strides[2] = {ld * size, rows * ld * size};
  cuuint32_t box[3] = {box_inner, box_rows, 1}, step[3] = {1, 1, 1};
  const CUresult r = encode(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                            const_cast<void*>(ptr), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    ft_set_error("linear_cross_entropy: cuTensorMapEncodeTiled failed with %d (%llu x %llu, pitch %llu)", (int)r,
                 (unsigned long long)inner, (unsigned long long)rows, (unsigned long long)ld);
    return FT_ERR_UNSUPPORTED;
  }
  return FT_OK;
}

template <bool PAIR, int EPI, bool A_MN, bool B_MN, bool TWO>
int launch_gemm(FtContext* ctx, const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& o, const TcProduct& g,
                int* workers_used) {
  auto kernel = k_ce_gemm<PAIR, EPI, A_MN, B_MN, TWO>;
  constexpr int CTAS = PAIR ? 2 : 1;
  static bool ready[FT_MAX_DEVICES] = {};
  static int most[FT_MAX_DEVICES] = {};
  if (!ready[ctx->device]) {
    FT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(EPI, TWO, PAIR)));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(ctx->sm_count / CTAS * CTAS));
    cfg.blockDim = dim3(threads_of(EPI, TWO, PAIR));
    cfg.dynamicSmemBytes = smem_bytes(EPI, TWO, PAIR);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = CTAS; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int n = 0;
    FT_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
    most[ctx->device] = std::max(1, std::min(n, ctx->sm_count / CTAS));
    ready[ctx->device] = true;
  }
  const long long units = (long long)ft_cdiv(g.M, CTAS * 128) * ft_cdiv(g.N, g.tile_n) * g.splits;
  // the targets' logits want a warp a row, of two a CTA, however few tiles there are
  const long long wanted = EPI <= EPI_EXP ? std::max(units, (long long)ft_cdiv(g.M, 2 * CTAS * g.pieces)) : units;
  const int workers = (int)std::max<long long>(1, std::min<long long>(wanted, most[ctx->device]));
  if (workers_used) *workers_used = (int)std::min<long long>(units, workers);   // that have a tile
  const char* const names[5] = {"k_ce_gemm<statistics>", "k_ce_gemm<E>", "k_ce_gemm<g>",
                                A_MN ? "k_ce_gemm<dW>" : "k_ce_gemm<dh>", "k_ce_gemm<dh of E>"};
  if (ctx->profile_all) ft_prof_begin(ctx, names[EPI]);
  cudaError_t e = ft_launch_ex(ctx, kernel, CTAS * workers, threads_of(EPI, TWO, PAIR), smem_bytes(EPI, TWO, PAIR), a, b, o, g, ctx->status_dev);
  if (ctx->profile_all) ft_prof_end(ctx);
  ctx->launches++;
  if (e == cudaSuccess) e = cudaPeekAtLastError();
  if (e != cudaSuccess) return ft_cuda_fail(e, "k_ce_gemm", __FILE__, __LINE__);
  return FT_OK;
}

// One CTA a tile (128 rows) where there are no more rows than that, else pairs (256).  `b_mn`: W's layout
// makes B M/N-contiguous.
template <int EPI>
int launch_rows(FtContext* ctx, bool pair, bool b_mn, bool two, const CUtensorMap& a, const CUtensorMap& b,
                const CUtensorMap& o, const TcProduct& g, int* workers_used = nullptr) {
  constexpr bool F = EPI == EPI_FACTOR;   // planes make no difference there
  if (pair) {
    if (b_mn) return two && !F ? launch_gemm<true, EPI, false, true, !F>(ctx, a, b, o, g, workers_used)
                               : launch_gemm<true, EPI, false, true, false>(ctx, a, b, o, g, workers_used);
    return two && !F ? launch_gemm<true, EPI, false, false, !F>(ctx, a, b, o, g, workers_used)
                     : launch_gemm<true, EPI, false, false, false>(ctx, a, b, o, g, workers_used);
  }
  if (b_mn) return two && !F ? launch_gemm<false, EPI, false, true, !F>(ctx, a, b, o, g, workers_used)
                             : launch_gemm<false, EPI, false, true, false>(ctx, a, b, o, g, workers_used);
  return two && !F ? launch_gemm<false, EPI, false, false, !F>(ctx, a, b, o, g, workers_used)
                   : launch_gemm<false, EPI, false, false, false>(ctx, a, b, o, g, workers_used);
}

// plane pairs of a product, the smallest first: sums grow as late as they can
void set_terms(TcProduct& g, int pa, int pb) {
  g.terms = 0;
  auto add = [&](int a, int b) { g.a_plane[g.terms] = a; g.b_plane[g.terms] = b; ++g.terms; };
  if (pa == 2) add(1, 0);
  if (pb == 2) add(0, 1);
  add(0, 0);
}

// Bytes of E or g at a time, when the caller leaves the choice.  A piece costs launches whose last wave is
// not full: 8192 x 2048 x 49152 takes 3.27 ms in pieces of 128 MB, 3.09 of 256, 3.03 of 512, 2.95 in one
// piece (805 MB: half of the logits in f32), 2048 x 896 x 151936 2.34, 2.17, 2.10 and 2.05.
constexpr size_t G_PIECE_BYTES = (size_t)512 << 20;

// Where g is made of E in place and not of a second product for the logits, in the split mode: from hidden =
// 320 or so on (512 rows x 128 x 49152, both gradients: 176 us in place, 160 by the product; hidden 256: 212 and
// 207, 384: 271 and 290; 7002 x 128 x 15104: 508 and 416), and always for few rows, where E stays in L2 (200 x 256 x
// 15104: 64 and 71).
bool makes_g_in_place(int rows, int hidden) { return hidden > 256 || rows <= 256; }
// Up to here one launch after E W costs less than one before it and one after (150 rows x 832 x 2048: 34 against
// 36 us; 1000 x 832 x 15104: 80 both ways; 7002 x 128 x 15104: 180 against 163).
constexpr int FINISH_ROWS = 1024;

struct TcPlan {
  Rows rows;
  __half *h, *w, *grad, *wy;
  float2* part;
  float *acc, *base;
  int Tp, h_ld, h_planes, w_ld, w_planes, w_rows, w_cols, g_planes, piece, splits, acc_ld;
  int stat_n, out_n;         // columns of a tile: of the statistics alone, of dh and (vocab-major) dW
  int tile_m;                // rows of a tile of the products whose rows are the packed ones
  bool pair, w_staged, by_exp, one_piece;
  bool in_place;             // g is made of E, see k_ce_normalise
  bool finish;               // of E W alone: k_ce_finish does what is left
  size_t bytes;
};

// Columns of a tile, a multiple of 32, for n columns and `rows` tiles of rows (times parts): whole
// waves of tiles as full as they get.  A tile costs its columns and about 24 more.
int pick_tile_n(long long n, long long row_tiles, int workers) {
  int best = TILE;
  double least = 1e30;
  for (int t = TILE; t >= 64; t -= 32) {
    const long long tiles = row_tiles * ft_cdiv(n, t);
    const double cost = (double)((tiles + workers - 1) / workers) * (t + 24);
    if (cost < least * 0.995) { least = cost; best = t; }
  }
  return best;
}

TcPlan tc_plan(const FtContext* ctx, const Problem& q, const void* weight, void* base) {
  TcPlan pl = {};
  Carver c(base);
  const bool two = ctx->gemm_mode == FT_GEMM_F16X2;
  pl.pair = q.T > 128;
  pl.tile_m = pl.pair ? 256 : 128;
  const int workers = std::max(1, pl.pair ? ctx->sm_count / 2 : ctx->sm_count);
  pl.rows = carve_rows(c, q.T);
  pl.Tp = (int)ft_align_up((size_t)std::max(q.T, 1), TILE);
  pl.h_ld = (int)ft_align_up((size_t)q.H, 8);
  pl.h_planes = two && q.p.hidden_type == FT_TYPE_F32 ? 2 : 1;
  pl.w_planes = two && q.p.weight_type == FT_TYPE_F32 ? 2 : 1;
  pl.g_planes = two ? 2 : 1;
  pl.w_rows = q.p.weight_vocab_major ? q.V : q.H;
  pl.w_cols = q.p.weight_vocab_major ? q.H : q.V;
  pl.w_staged = q.p.weight_type == FT_TYPE_F32 || pl.w_cols % 8 != 0 || ((uintptr_t)weight & 15) != 0;
  pl.w_ld = (int)ft_align_up((size_t)pl.w_cols, 8);
  pl.by_exp = q.grad_hidden && !q.grad_weight;
  pl.h = c.take<__half>((size_t)pl.h_planes * pl.Tp * pl.h_ld);
  pl.w = pl.w_staged ? c.take<__half>((size_t)pl.w_planes * pl.w_rows * pl.w_ld) : nullptr;
  // few row tiles: the columns of a tile follow the number of waves (the last one may be nearly empty)
  pl.stat_n = q.T <= 2 * TILE && !pl.by_exp ? pick_tile_n(q.V, ft_cdiv(q.T, pl.tile_m), workers) : TILE;
  pl.out_n = pick_tile_n(q.H, 1 << 20, workers);
  size_t part_bytes = (size_t)parts_of(EPI_STATS, two, pl.pair) * ft_cdiv(q.V, pl.stat_n) * pl.Tp * sizeof(float2), grad_bytes = 0;
  if (q.grad_hidden || q.grad_weight) {
    const size_t column = (size_t)pl.Tp * 2 * pl.g_planes;
    size_t cols = q.p.vocab_piece ? q.p.vocab_piece : std::max<size_t>(TILE, G_PIECE_BYTES / column);
    const int pieces = ft_cdiv(q.V, (long long)std::min<size_t>(cols, (size_t)q.V));
    // equal pieces of whole tiles
    pl.piece = (int)ft_align_up((size_t)ft_cdiv(q.V, pieces), TILE);
    grad_bytes = column * pl.piece;
    pl.one_piece = pieces == 1;
    pl.in_place = two && q.grad_weight && pl.one_piece && makes_g_in_place(q.T, q.H);
    pl.finish = pl.one_piece && q.T <= FINISH_ROWS;
    if (pl.by_exp || pl.in_place) part_bytes = (size_t)parts_of(EPI_EXP, two, pl.pair) * (pl.piece / TILE) * pl.Tp * sizeof(float2);
  }
  if (pl.by_exp || pl.in_place) {
    pl.part = (float2*)c.take<char>(part_bytes);
    pl.grad = (__half*)c.take<char>(grad_bytes);
    if (pl.by_exp) pl.wy = c.take<__half>((size_t)pl.w_planes * pl.Tp * pl.h_ld);
  } else {
    // the statistics of the column tiles are done with before the first piece of g is written
    char* shared = c.take<char>(std::max(part_bytes, grad_bytes));
    pl.part = (float2*)shared;
    pl.grad = (__half*)shared;
  }
  pl.splits = 1;
  if (q.grad_hidden) {
    // Parts of K, by what they should take: rounds of tiles at the workers' rate and 2 us each to fill and
    // drain, and the slabs written and read once more (1225 x 575 x 50021: as many as fit 256 MB were
    // 57, and 97 us for dh and its unpacking where 9 take 82).  How many rows are supervised is not
    // known here: the sum of the times for all of them and for half (4096 rows, 2048 of them
    // supervised: 4% of the whole call between the best number for 4096 and this one).
    pl.acc_ld = (int)ft_align_up((size_t)q.H, 4);
    const double rate = 1.2e9 / (pl.pair ? 74 : 148);              // flops of a worker in a microsecond
    const double tile_us = 2.0 * pl.tile_m * pl.out_n * std::min(pl.piece, q.V) * (pl.g_planes + pl.w_planes - 1) / rate;
    const int grains = ft_cdiv(std::min(pl.piece, q.V), pl.by_exp ? TILE : BK);   // of the first piece: it fills every slab
    auto cost = [&](int rows, int s) {
      const int row_tiles = ft_cdiv(std::max(rows, 1), pl.tile_m);
      const long long units = (long long)row_tiles * ft_cdiv(q.H, pl.out_n) * s;
      return (double)((units + workers - 1) / workers) * (tile_us / s + 2.0) + 2.0 * s * row_tiles * pl.tile_m * pl.acc_ld * 4.0 / 4e6;
    };
    double best = 1e30;
    for (int s = 1; s <= std::min(64, grains); ++s) {
      const double us = cost(q.T, s) + cost(q.T / 2, s);
      if (us < best) { best = us; pl.splits = s; }
    }
    pl.acc = c.take<float>((size_t)pl.splits * pl.Tp * pl.acc_ld);
    pl.base = c.take<float>((size_t)pl.splits * pl.Tp);
  }
  pl.bytes = c.bytes();
  return pl;
}

}  // namespace

namespace ft_ce {

size_t tc_workspace(const FtContext* ctx, const Problem& q, const void* weight) { return tc_plan(ctx, q, weight, nullptr).bytes; }

int tc_path(FtContext* ctx, const Problem& q, const Tensors& t, void* ws) {
  TcPlan pl = tc_plan(ctx, q, t.weight, ws);
  const int T = q.T, H = q.H, V = q.V;
  const bool vm = q.p.weight_vocab_major != 0, two = pl.g_planes == 2;
  const bool h32 = q.p.hidden_type == FT_TYPE_F32, w32 = q.p.weight_type == FT_TYPE_F32;
  // dW sums over the rows, which then need one scale, found by a pass of its own; else a row has its own
  // (4096 f32 rows, a quarter of them skipped, x 960 x 49152: 419 -> 407 us)
  if (!h32 || t.grad_weight) pl.rows.unscale = nullptr;
  const bool h_scan = h32 && t.grad_weight;
  const long long w_values = (long long)pl.w_rows * pl.w_cols;
  const int wb = w32 ? (int)std::min<long long>(AMAX_BLOCKS, ft_cdiv(w_values, 4096)) : 0, hb = h_scan ? std::min(T, AMAX_BLOCKS) : 0;
  if (wb + hb) {
    FT_LAUNCH_PDL(ctx, k_ce_amax, wb + hb, 256, 0, (const float*)t.weight, w_values, wb,
                  (const float*)t.hidden, t.targets, T, H, pl.rows);
  }
  // One tile of rows and no dW: packing would save nothing, and what a row gets is its own whatever the
  // others hold.
  const bool unpacked = T <= 128 && !t.grad_weight && (!t.grad_hidden || pl.finish) && !h32 && !w32 && H % 8 == 0 &&
                        ((uintptr_t)t.hidden & 15) == 0;
  const void* w = pl.w_staged ? pl.w : t.weight;
  if (!unpacked || pl.w_staged) {
    PackArgs a = {};
    a.hidden = t.hidden; a.weight = t.weight; a.targets = t.targets; a.weights = t.weights;
    a.grad_scale = q.p.grad_scale;
    a.rows = T; a.H = H; a.per = gather_rows(T);
    a.rw = pl.rows;
    a.h = pl.h; a.h_ld = pl.h_ld; a.plane_rows = pl.Tp; a.h_planes = pl.h_planes; a.h_parts = hb; a.w_parts = wb;
    a.row_loss = t.row_loss;
    a.w = pl.w; a.w_rows = pl.w_rows; a.w_cols = pl.w_cols; a.w_ld = pl.w_ld; a.w_planes = pl.w_planes;
    a.gather_blocks = unpacked ? 0 : ft_cdiv(T, a.per);
    a.gx = std::min(ft_cdiv(pl.w_rows, 8), ctx->sm_count * 16);
    const int blocks = a.gather_blocks + (pl.w_staged ? a.gx * ft_cdiv(pl.w_ld, 1024) : 0);
    if (h32 && w32) FT_LAUNCH_PDL(ctx, (k_ce_pack<float, float>), blocks, GATHER_THREADS, 0, a);
    else if (h32) FT_LAUNCH_PDL(ctx, (k_ce_pack<float, __half>), blocks, GATHER_THREADS, 0, a);
    else if (w32) FT_LAUNCH_PDL(ctx, (k_ce_pack<__half, float>), blocks, GATHER_THREADS, 0, a);
    else FT_LAUNCH_PDL(ctx, (k_ce_pack<__half, __half>), blocks, GATHER_THREADS, 0, a);
  }
  // K-contiguous operands come in boxes of 64 x 128 rows (B: half a tile's columns), M/N-contiguous ones
  // in two of 64 x 64
  auto k_map = [&](CUtensorMap* m, const void* p, int inner, int rows, int planes, int ld, int box) {
    return make_map3(ctx, m, p, false, inner, rows, planes, ld, 64, box);
  };
  auto mn_map = [&](CUtensorMap* m, const void* p, int inner, int rows, int planes, int ld) {
    return make_map3(ctx, m, p, false, inner, rows, planes, ld, 64, 64);
  };
  auto tile = [&](TcProduct& p, bool pair, int tile_n, int a_rows, bool b_mn) {
    p.tile_n = tile_n;
    p.a_bytes = a_rows * 128;
    const int b_cols = pair ? tile_n / 2 : tile_n, b_bytes = (b_mn ? (int)ft_align_up((size_t)b_cols, 64) : b_cols) * 128;
    p.stage_bytes = (int)ft_align_up((size_t)(p.a_bytes + b_bytes), 1024);
    p.stage_tx = (pair ? 2 : 1) * (p.a_bytes + b_bytes);
  };
  // columns of a K-contiguous B that a CTA loads
  auto b_box = [&](int tile_n) { return pl.pair ? tile_n / 2 : tile_n; };
  // at most 128 rows: only as many are loaded
  const int a_rows = pl.pair ? 128 : (int)ft_align_up((size_t)T, 8);
  CUtensorMap h_k, w_k, w_mn;
  FT_TRY(k_map(&h_k, unpacked ? t.hidden : pl.h, H, unpacked ? T : pl.Tp, pl.h_planes, pl.h_ld, a_rows));
  if (!vm || t.grad_hidden) FT_TRY(mn_map(&w_mn, w, pl.w_cols, pl.w_rows, pl.w_planes, pl.w_ld));

  TcProduct z = {};
  z.M = T; z.N = V; z.K = H; z.live_m = 1; z.splits = 1;
  z.band = 32;
  set_terms(z, pl.h_planes, pl.w_planes);
  z.rw = pl.rows; z.part = pl.part; z.part_ld = pl.Tp; z.vocab = V;
  if (unpacked) z.rw.target = const_cast<uint32_t*>(t.targets);
  z.unpacked = unpacked ? 1 : 0;
  z.h = unpacked ? (const __half*)t.hidden : pl.h; z.h_ld = pl.h_ld; z.h_plane = (long long)pl.Tp * pl.h_ld; z.h_planes = pl.h_planes;
  z.w = (const __half*)w; z.w_plane = (long long)pl.w_rows * pl.w_ld; z.w_planes = pl.w_planes;
  z.w_sk = vm ? 1 : pl.w_ld; z.w_sv = vm ? pl.w_ld : 1;
  z.wy = pl.wy; z.wy_ld = pl.h_ld;
  z.pieces = pl.by_exp ? ft_cdiv(V, pl.piece) : 1;
  const size_t slab = (size_t)pl.Tp * pl.acc_ld;
  const int join_grid = ft_cdiv(T, 32);
  auto join_threads = [](int parts) { return parts > 256 ? 32 * JOIN_WARPS : 256; };
  CUtensorMap acc_out;
  if (t.grad_hidden) FT_TRY(make_map3(ctx, &acc_out, pl.acc, true, pl.acc_ld, pl.Tp, pl.splits, pl.acc_ld, 32, 32));
  const dim3 unpack_grid((unsigned)std::min(ft_cdiv(T, 8), ctx->sm_count * 16), (unsigned)ft_cdiv(std::max(pl.acc_ld, 1), 128));
  CUtensorMap g_out, g_k;
  if (t.grad_hidden || t.grad_weight)
    FT_TRY(make_map3(ctx, &g_out, pl.grad, false, pl.piece, pl.Tp, pl.g_planes, pl.piece, 64, 32));

  // the product with W of one piece of E or g, into the slabs
  auto dh_product = [&](int v0, int cols) {
    TcProduct p = {};
    p.rw = pl.rows;
    p.M = T; p.N = H; p.K = cols; p.live_m = 1;
    p.splits = std::min(pl.splits, ft_cdiv(cols, pl.by_exp ? TILE : BK));
    p.n_fast = 1; p.band = 1;
    set_terms(p, pl.g_planes, pl.w_planes);
    p.b_k0 = v0;
    p.out_type = FT_TYPE_F32; p.accumulate = v0 > 0;
    p.part = pl.part; p.part_ld = pl.Tp;
    p.unpacked = unpacked ? 1 : 0;
    p.base_out = pl.by_exp && pl.finish ? pl.base : nullptr;
    tile(p, pl.pair, pl.out_n, a_rows, vm);
    p.slice = two ? slice_of(EPI_STORE, true) : ONE_PLANE_SLICE;
    return p;
  };

  if (pl.by_exp) {
    FT_TRY(k_map(&w_k, w, pl.w_cols, pl.w_rows, pl.w_planes, pl.w_ld, b_box(vm ? TILE : pl.out_n)));
    tile(z, pl.pair, TILE, a_rows, !vm);
    for (int v0 = 0; v0 < V; v0 += pl.piece) {
      const int cols = std::min(pl.piece, V - v0);
      const bool first = v0 == 0, last = v0 + cols == V;
      z.N = cols; z.v0 = v0; z.b_mn0 = v0; z.piece = v0 / pl.piece;
      FT_TRY(launch_rows<EPI_EXP>(ctx, pl.pair, !vm, two, h_k, vm ? w_k : w_mn, g_out, z));
      const int parts = parts_of(EPI_EXP, two, pl.pair) * ft_cdiv(cols, TILE);
      if (!pl.finish)
        FT_LAUNCH_PDL(ctx, k_ce_join, join_grid, join_threads(parts), 0, pl.part, pl.Tp, parts,
                      pl.rows, 0, first ? 1 : 0, last ? 1 : 0, V, t.row_loss, pl.acc, slab, pl.splits, pl.acc_ld, H);
      if (first || cols != pl.piece) FT_TRY(k_map(&g_k, pl.grad, cols, pl.Tp, pl.g_planes, pl.piece, a_rows));
      const TcProduct p = dh_product(v0, cols);
      FT_TRY(launch_rows<EPI_FACTOR>(ctx, pl.pair, vm, two, g_k, vm ? w_mn : w_k, acc_out, p));
    }
    if (pl.finish) {
      const int parts = parts_of(EPI_EXP, two, pl.pair) * ft_cdiv(V, TILE), across = T <= 32 ? ft_cdiv(pl.acc_ld, 256) : 1;
      const dim3 grid((unsigned)ft_cdiv(T, 4), (unsigned)across);
      const size_t plane = (size_t)pl.Tp * pl.h_ld;
      if (q.p.grad_hidden_type == FT_TYPE_F16)
        FT_LAUNCH_PDL(ctx, k_ce_finish<__half>, grid, 256, 0, pl.part, pl.Tp, parts, z.rw, unpacked ? 1 : 0, t.weights,
                      q.p.grad_scale, V, t.row_loss, pl.base, pl.acc, slab, pl.splits, pl.acc_ld, pl.wy, plane, pl.h_ld,
                      pl.w_planes, H, T, (__half*)t.grad_hidden);
      else
        FT_LAUNCH_PDL(ctx, k_ce_finish<float>, grid, 256, 0, pl.part, pl.Tp, parts, z.rw, unpacked ? 1 : 0, t.weights,
                      q.p.grad_scale, V, t.row_loss, pl.base, pl.acc, slab, pl.splits, pl.acc_ld, pl.wy, plane, pl.h_ld,
                      pl.w_planes, H, T, (float*)t.grad_hidden);
      return FT_OK;
    }
    if (q.p.grad_hidden_type == FT_TYPE_F16)
      FT_LAUNCH_PDL(ctx, k_ce_scatter_exp<__half>, unpack_grid, 256, 0, pl.acc, slab, pl.splits, pl.acc_ld, pl.rows, pl.wy,
                    (size_t)pl.Tp * pl.h_ld, pl.h_ld, pl.w_planes, H, T, (__half*)t.grad_hidden);
    else
      FT_LAUNCH_PDL(ctx, k_ce_scatter_exp<float>, unpack_grid, 256, 0, pl.acc, slab, pl.splits, pl.acc_ld, pl.rows, pl.wy,
                    (size_t)pl.Tp * pl.h_ld, pl.h_ld, pl.w_planes, H, T, (float*)t.grad_hidden);
    return FT_OK;
  }

  if (pl.in_place) {
    tile(z, pl.pair, TILE, a_rows, !vm);
    if (vm) FT_TRY(k_map(&w_k, w, pl.w_cols, pl.w_rows, pl.w_planes, pl.w_ld, b_box(TILE)));
    FT_TRY(launch_rows<EPI_EXP>(ctx, pl.pair, !vm, two, h_k, vm ? w_k : w_mn, g_out, z));
    const int parts = parts_of(EPI_EXP, two, pl.pair) * ft_cdiv(V, TILE);
    FT_LAUNCH_PDL(ctx, k_ce_join, join_grid, join_threads(parts), 0, pl.part, pl.Tp, parts, pl.rows,
                  0, 1, 1, V, t.row_loss, (float*)nullptr, (size_t)0, 0, 0, 0);
    const dim3 grid(ft_cdiv(V, 2048), std::max(1, std::min(pl.Tp, ctx->sm_count * 32 / ft_cdiv(V, 2048))));
    FT_LAUNCH_PDL(ctx, k_ce_normalise, grid, 256, 0, pl.grad, (size_t)pl.Tp * pl.piece, pl.piece, pl.part, pl.Tp, pl.rows, pl.piece,
                  parts_of(EPI_EXP, two, pl.pair));
  } else {
    tile(z, pl.pair, pl.stat_n, a_rows, !vm);
    z.w_early = !pl.w_staged;
    z.carry = T <= pl.tile_m ? 1 : 0;
    int workers = 0;
    if (vm) FT_TRY(k_map(&w_k, w, pl.w_cols, pl.w_rows, pl.w_planes, pl.w_ld, b_box(pl.stat_n)));
    FT_TRY(launch_rows<EPI_STATS>(ctx, pl.pair, !vm, two, h_k, vm ? w_k : w_mn, h_k, z, &workers));
    const int parts = parts_of(EPI_STATS, two, pl.pair) * (z.carry ? workers : ft_cdiv(V, pl.stat_n));
    FT_LAUNCH_PDL(ctx, k_ce_join, join_grid, join_threads(parts), 0, pl.part, pl.Tp, parts, z.rw, unpacked ? T : 0, 1, 1, V, t.row_loss,
                  (float*)nullptr, (size_t)0, 0, 0, 0);
  }
  if (!t.grad_hidden && !t.grad_weight) return FT_OK;

  CUtensorMap g_mn, h_mn, dw_out;
  FT_TRY(k_map(&w_k, w, pl.w_cols, pl.w_rows, pl.w_planes, pl.w_ld, b_box(vm ? TILE : pl.out_n)));
  FT_TRY(mn_map(&h_mn, pl.h, H, pl.Tp, pl.h_planes, pl.h_ld));
  const bool dw16 = q.p.grad_weight_type == FT_TYPE_F16;
  const bool dw_tma = t.grad_weight && ((uintptr_t)t.grad_weight & 15) == 0 && pl.w_cols % (dw16 ? 8 : 4) == 0;
  if (dw_tma)
    FT_TRY(make_map3(ctx, &dw_out, t.grad_weight, !dw16, pl.w_cols, pl.w_rows, 1, pl.w_cols, 32, 32,
                     dw16 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B));
  tile(z, pl.pair, TILE, a_rows, !vm);
  for (int v0 = 0; v0 < V; v0 += pl.piece) {
    const int cols = std::min(pl.piece, V - v0);
    z.N = cols; z.v0 = v0; z.b_mn0 = v0;
    if (!pl.in_place) FT_TRY(launch_rows<EPI_GRAD>(ctx, pl.pair, !vm, two, h_k, vm ? w_k : w_mn, g_out, z));
    // as operands, the piece ends with the vocabulary: what lies behind reads as zero
    if (v0 == 0 || cols != pl.piece) {
      FT_TRY(k_map(&g_k, pl.grad, cols, pl.Tp, pl.g_planes, pl.piece, a_rows));
      FT_TRY(mn_map(&g_mn, pl.grad, cols, pl.Tp, pl.g_planes, pl.piece));
    }
    if (t.grad_hidden) {
      const TcProduct p = dh_product(v0, cols);
      const bool slices = two || ft_cdiv(ft_cdiv(cols, BK), p.splits) > ONE_PLANE_SLICE;
      FT_TRY(launch_rows<EPI_STORE>(ctx, pl.pair, vm, slices, g_k, vm ? w_mn : w_k, acc_out, p));
    }
    if (t.grad_weight) {
      TcProduct p = {};
      p.rw = pl.rows;
      p.K = T; p.live_k = 1; p.splits = 1;
      p.unscale = 1;
      p.out_type = (int)q.p.grad_weight_type;
      if (!dw_tma) { p.direct = t.grad_weight; p.direct_ld = pl.w_cols; }
      // rows of a tile are vocabulary either way: their number is a multiple of the tile, hidden's is not
      p.M = cols; p.N = H;
      p.transposed = vm ? 0 : 1;
      if (vm) p.out_y0 = v0;
      else p.out_x0 = v0;
      set_terms(p, pl.g_planes, pl.h_planes);
      tile(p, true, pl.out_n, 128, true);
      p.n_fast = p.M >= p.N; p.band = ft_cdiv(p.M, TILE);
      const CUtensorMap& po = dw_tma ? dw_out : g_mn;
      p.slice = two ? slice_of(EPI_STORE, true) : ONE_PLANE_SLICE;
      if (two || ft_cdiv(T, BK) > ONE_PLANE_SLICE) FT_TRY((launch_gemm<true, EPI_STORE, true, true, true>(ctx, g_mn, h_mn, po, p, nullptr)));
      else FT_TRY((launch_gemm<true, EPI_STORE, true, true, false>(ctx, g_mn, h_mn, po, p, nullptr)));
    }
  }
  if (t.grad_hidden) {
    if (q.p.grad_hidden_type == FT_TYPE_F16)
      FT_LAUNCH_PDL(ctx, k_ce_scatter<__half>, unpack_grid, 256, 0, pl.acc, slab, pl.splits, pl.acc_ld, pl.rows, H, T, (__half*)t.grad_hidden);
    else
      FT_LAUNCH_PDL(ctx, k_ce_scatter<float>, unpack_grid, 256, 0, pl.acc, slab, pl.splits, pl.acc_ld, pl.rows, H, T, (float*)t.grad_hidden);
  }
  return FT_OK;
}

}  // namespace ft_ce
