// Global gradient norm and clipping over a list of tensors (ferrotensor-trainer/src/lib.rs:328-343,
// where the host loops over the tensors, reads their chunk sums back and launches a scaling for
// each).
//
//   n = |s| sqrt(sum_i sum_j g_ij^2),   f = s (n > max ? max / (n + 1e-6) : 1),   out_ij = f g_ij
//
// Two launches, whatever the number of tensors: k_list_squares sums the squares, k_list_scale joins
// the sums and writes the scaled values.  Both walk a table of chunks (at most CHUNK elements of
// one tensor each) that lies on the device since the list was made.  HBM-bound: a value is read
// once for the norm and once for the scaling, which walks the chunks in the reverse order so that
// its first reads find in L2 what the norm read last.  A list of a few thousand values is bound by
// its launches: k_list_small does both in one.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <exception>
#include <type_traits>
#include <vector>

#include "ft_common.cuh"

namespace {

constexpr int LIST_THREADS = 256;
constexpr int CHUNK = 8192;            // elements; a thread's share of one is eight 16-byte loads of f32
constexpr int LIST_BLOCKS_PER_SM = 4;  // of k_list_squares: 128 KB of loads in flight a multiprocessor
constexpr int SCALE_BLOCKS_PER_SM = 4;

// A list that makes at most SMALL_CHUNKS chunks of SMALL_CHUNK values: one block, a warp a chunk,
// two chunks a warp at most, whose values stay in registers between the two steps.
constexpr int SMALL_CHUNK = 256, SMALL_CHUNKS = 64, SMALL_THREADS = 1024;

struct Chunk {
  void* p;
  uint32_t n;
  uint32_t type;
};

// Eight values at a 16-byte boundary.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const __half* p, float (&v)[8]) {
  const uint4 a = *(const uint4*)p;
  const __half2* h = (const __half2*)&a;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
// Four values at a boundary of four.
__device__ __forceinline__ float4 load4(const float* p) { return *(const float4*)p; }
__device__ __forceinline__ float4 load4(const __half* p) {
  const uint2 a = *(const uint2*)p;
  const float2 x = __half22float2(*(const __half2*)&a.x), y = __half22float2(*(const __half2*)&a.y);
  return make_float4(x.x, x.y, y.x, y.y);
}
__device__ __forceinline__ void store4(float* p, float4 v) { *(float4*)p = v; }
__device__ __forceinline__ void store4(__half* p, float4 v) {
  const __half2 x = __floats2half2_rn(v.x, v.y), y = __floats2half2_rn(v.z, v.w);
  *(uint2*)p = make_uint2(*(const uint32_t*)&x, *(const uint32_t*)&y);
}
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__half* p, float v) { *p = __float2half_rn(v); }

// Elements before the first 16-byte boundary.
template <typename T>
__device__ __forceinline__ uint32_t ahead_of_boundary(const T* p, uint32_t n) {
  return min(n, (uint32_t)((16 - ((uintptr_t)p & 15)) & 15) / (uint32_t)sizeof(T));
}

// Squares are taken and summed in f64: an f32 square leaves the f32 range for |g| above 1.8e19 or
// below 1e-19.  Squares of f16 values are exact in f32 and far from its ends, so eight of them are
// added there first (conversions to f64 would bound the f16 rate otherwise).
__device__ __forceinline__ double squares8(const float (&v)[8], float) {
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) s = fma((double)v[i], (double)v[i], s);
  return s;
}
__device__ __forceinline__ double squares8(const float (&v)[8], __half) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s = fmaf(v[i], v[i], s);
  return (double)s;
}

template <typename T>
__device__ __forceinline__ double sum_squares(const T* __restrict__ x, uint32_t n) {
  double acc = 0.0;
  const uint32_t head = ahead_of_boundary(x, n);
  if (threadIdx.x < head) {
    const double v = (double)(float)x[threadIdx.x];
    acc = v * v;
  }
  const T* body = x + head;
  const uint32_t groups = (n - head) / 8;
  // all loads of a thread's share first
  float v[CHUNK / 8 / LIST_THREADS][8];
#pragma unroll
  for (int k = 0; k < CHUNK / 8 / LIST_THREADS; ++k) {
    const uint32_t g = threadIdx.x + k * LIST_THREADS;
    if (g < groups) load8(body + 8 * g, v[k]);
    else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[k][i] = 0.f;
    }
  }
#pragma unroll
  for (int k = 0; k < CHUNK / 8 / LIST_THREADS; ++k) acc += squares8(v[k], T());
  const uint32_t tail = head + 8 * groups + threadIdx.x;
  if (tail < n) {
    const double t = (double)(float)x[tail];
    acc = fma(t, t, acc);
  }
  return acc;
}

__device__ __forceinline__ double sum_squares_chunk(const Chunk& c) {
  return c.type == FT_TYPE_F32 ? sum_squares((const float*)c.p, c.n) : sum_squares((const __half*)c.p, c.n);
}

__device__ __forceinline__ double block_sum_f64(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < LIST_THREADS / 32; ++w) s += red[w];
  __syncthreads();
  return s;
}

__global__ void __launch_bounds__(LIST_THREADS, LIST_BLOCKS_PER_SM)
k_list_squares(const Chunk* __restrict__ chunks, int count, double* __restrict__ partials) {
  __shared__ double red[LIST_THREADS / 32];
  ft_pdl_wait();
  ft_pdl_launch();
  double acc = 0.0;
  Chunk now = {};
  if ((int)blockIdx.x < count) now = chunks[blockIdx.x];
  for (int c = blockIdx.x; c < count; c += gridDim.x) {
    // the next chunk's place is on its way while this one's values are
    Chunk next = {};
    if (c + (int)gridDim.x < count) next = chunks[c + gridDim.x];
    acc += sum_squares_chunk(now);
    now = next;
  }
  acc = block_sum_f64(acc, red);
  if (threadIdx.x == 0) partials[blockIdx.x] = acc;
}

// out = f x over one chunk: four values a lane, so that a warp's loads and stores are whole lines in
// either type, where both sides reach a boundary of four values at the same element, else one.
template <typename TI, typename TO>
__device__ __forceinline__ void scale_chunk(const TI* x, TO* out, uint32_t n, float f) {
  constexpr int BATCH = 4;
  const uint32_t head = min(n, (uint32_t)((4 * sizeof(TI) - ((uintptr_t)x & (4 * sizeof(TI) - 1))) & (4 * sizeof(TI) - 1)) / (uint32_t)sizeof(TI));
  if (((uintptr_t)(out + head) & (4 * sizeof(TO) - 1)) == 0) {
    if (threadIdx.x < head) store1(out + threadIdx.x, f * (float)x[threadIdx.x]);
    const uint32_t groups = (n - head) / 4;
#pragma unroll 1
    for (uint32_t g = threadIdx.x; g < groups; g += BATCH * LIST_THREADS) {
      // (one base and constant offsets: indices of their own cost two registers each)
      const TI* xb = x + head + 4 * (size_t)g;
      TO* ob = out + head + 4 * (size_t)g;
      const int left = (int)((groups - g + LIST_THREADS - 1) / LIST_THREADS);
      float4 v[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k)
        if (k < left) v[k] = load4(xb + 4 * k * LIST_THREADS);
#pragma unroll
      for (int k = 0; k < BATCH; ++k)
        if (k < left) store4(ob + 4 * k * LIST_THREADS, make_float4(f * v[k].x, f * v[k].y, f * v[k].z, f * v[k].w));
    }
    const uint32_t tail = head + 4 * groups + threadIdx.x;
    if (tail < n) store1(out + tail, f * (float)x[tail]);
  } else {
#pragma unroll 1
    for (uint32_t i = threadIdx.x; i < n; i += BATCH * LIST_THREADS) {
      const TI* xb = x + i;
      TO* ob = out + i;
      const int left = (int)((n - i + LIST_THREADS - 1) / LIST_THREADS);
      float v[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k)
        if (k < left) v[k] = (float)xb[k * LIST_THREADS];
#pragma unroll
      for (int k = 0; k < BATCH; ++k)
        if (k < left) store1(ob + k * LIST_THREADS, f * v[k]);
    }
  }
}

// What follows from the sum of squares.
struct Outcome {
  float norm, factor;
  bool finite;
  __device__ __forceinline__ void publish(float* o) const {
    o[0] = norm;
    o[1] = finite ? 1.f : 0.f;
    o[2] = factor;
  }
};
__device__ __forceinline__ Outcome decide(double squares, float grad_scale, float max_norm) {
  const double norm = sqrt(squares) * fabs((double)grad_scale);
  Outcome d;
  d.norm = (float)norm;
  d.finite = isfinite(d.norm);
  d.factor = grad_scale;
  if (d.finite && max_norm > 0.f && norm > (double)max_norm)
    d.factor = (float)((double)grad_scale * (double)max_norm / (norm + 1e-6));
  return d;
}

// Every block joins the partial sums itself (the same order everywhere), block 0 publishes.
// out == NULL: measure only.  TI, TO: the types of all chunks; void: each chunk's own.  (The four pairs
// of types in one body spill 180 bytes a thread, so only lists of both types take it.)
template <typename TI, typename TO>
__global__ void __launch_bounds__(LIST_THREADS, SCALE_BLOCKS_PER_SM)
k_list_scale(const Chunk* __restrict__ chunks, const Chunk* __restrict__ out, int count,
             const double* __restrict__ partials, int parts, float grad_scale, float max_norm,
             float* __restrict__ norm_out, int in_place) {
  __shared__ double red[LIST_THREADS / 32];
  ft_pdl_wait();
  ft_pdl_launch();
  double acc = 0.0;
  for (int i = threadIdx.x; i < parts; i += LIST_THREADS) acc += partials[i];
  const Outcome d = decide(block_sum_f64(acc, red), grad_scale, max_norm);
  if (blockIdx.x == 0 && threadIdx.x == 0 && norm_out) d.publish(norm_out);
  if (!out || !d.finite || (in_place && d.factor == 1.0f)) return;
  const float factor = d.factor;
  Chunk src = {}, dst = {};
  int c = count - 1 - (int)blockIdx.x;
  if (c >= 0) { src = chunks[c]; dst = out[c]; }
  while (c >= 0) {
    // the next chunk's place is on its way while this one's values are
    c -= (int)gridDim.x;
    Chunk next_src = {}, next_dst = {};
    if (c >= 0) { next_src = chunks[c]; next_dst = out[c]; }
    if constexpr (!std::is_void<TI>::value) {
      scale_chunk((const TI*)src.p, (TO*)dst.p, src.n, factor);
    } else if (src.type == FT_TYPE_F32) {
      if (dst.type == FT_TYPE_F32) scale_chunk((const float*)src.p, (float*)dst.p, src.n, factor);
      else scale_chunk((const float*)src.p, (__half*)dst.p, src.n, factor);
    } else {
      if (dst.type == FT_TYPE_F32) scale_chunk((const __half*)src.p, (float*)dst.p, src.n, factor);
      else scale_chunk((const __half*)src.p, (__half*)dst.p, src.n, factor);
    }
    src = next_src;
    dst = next_dst;
  }
}

__device__ __forceinline__ float load_any(const Chunk& c, int i) {
  return c.type == FT_TYPE_F32 ? ((const float*)c.p)[i] : __half2float(((const __half*)c.p)[i]);
}

__global__ void __launch_bounds__(SMALL_THREADS)
k_list_small(const Chunk* __restrict__ chunks, const Chunk* __restrict__ out, int count, float grad_scale,
             float max_norm, float* __restrict__ norm_out, int in_place) {
  __shared__ double red[SMALL_THREADS / 32];
  constexpr int WARPS = SMALL_THREADS / 32, PER = SMALL_CHUNKS / WARPS, VALUES = SMALL_CHUNK / 32;
  ft_pdl_wait();
  ft_pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float v[PER][VALUES];
  Chunk dst[PER];
  double acc = 0.0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int c = warp + j * WARPS;
    Chunk src = {};
    dst[j] = Chunk{};
    if (c < count) {
      src = chunks[c];
      if (out) dst[j] = out[c];
    }
#pragma unroll
    for (int k = 0; k < VALUES; ++k) v[j][k] = lane + 32 * k < (int)src.n ? load_any(src, lane + 32 * k) : 0.f;
  }
#pragma unroll
  for (int j = 0; j < PER; ++j)
#pragma unroll
    for (int k = 0; k < VALUES; ++k) acc = fma((double)v[j][k], (double)v[j][k], acc);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (lane == 0) red[warp] = acc;
  __syncthreads();
  double sum = red[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const Outcome d = decide(sum, grad_scale, max_norm);
  if (threadIdx.x == 0 && norm_out) d.publish(norm_out);
  if (!out || !d.finite || (in_place && d.factor == 1.0f)) return;
#pragma unroll
  for (int j = 0; j < PER; ++j)
#pragma unroll
    for (int k = 0; k < VALUES; ++k) {
      const int i = lane + 32 * k;
      if (i >= (int)dst[j].n) continue;
      if (dst[j].type == FT_TYPE_F32) ((float*)dst[j].p)[i] = d.factor * v[j][k];
      else ((__half*)dst[j].p)[i] = __float2half_rn(d.factor * v[j][k]);
    }
}

struct Span {
  uintptr_t begin, end;
  size_t index;
};

}  // namespace

struct FtGradList {
  FtContext* ctx = nullptr;
  size_t count = 0;
  std::vector<void*> ptrs;
  std::vector<size_t> elements;
  std::vector<int> types;
  std::vector<Span> spans;      // of the tensors that are not empty, by address
  bool disjoint = true;
  int type = -1;                // FT_TYPE_* of every tensor, -1 for a list of both
  int chunks = 0;
  bool small = false;           // chunks of SMALL_CHUNK for k_list_small, else of CHUNK
  Chunk* table = nullptr;       // [chunks] on the device
  double* partials = nullptr;   // one sum for each block of k_list_squares
  FtGradList* next = nullptr;   // in the context's list of destroyed ones
};

namespace {

int list_grid(const FtGradList* l) {
  return std::max(1, std::min(l->chunks, l->ctx->sm_count * LIST_BLOCKS_PER_SM));
}

int check_list(const char* who, FtContext* ctx, const FtGradList* l) {
  FT_REQUIRE(ctx && l, "%s: NULL argument", who);
  FT_REQUIRE(l->ctx == ctx, "%s: the list belongs to another context", who);
  return FT_OK;
}

bool overlaps_any(const std::vector<Span>& spans, bool disjoint, uintptr_t b, uintptr_t e) {
  if (!disjoint) {
    for (const Span& s : spans)
      if (s.begin < e && b < s.end) return true;
    return false;
  }
  auto it = std::lower_bound(spans.begin(), spans.end(), b, [](const Span& s, uintptr_t v) { return s.end <= v; });
  return it != spans.end() && it->begin < e;
}

int create_list(FtContext* ctx, size_t count, void* const* ptrs, const size_t* elements, const int* types,
                FtGradList* l) {
  l->ctx = ctx;
  l->count = count;
  l->ptrs.assign(ptrs, ptrs + count);
  l->elements.assign(elements, elements + count);
  l->types.assign(types, types + count);
  std::vector<Chunk> host;
  size_t pieces = 0;
  for (size_t i = 0; i < count; ++i) pieces += (elements[i] + SMALL_CHUNK - 1) / SMALL_CHUNK;
  l->small = pieces <= SMALL_CHUNKS;
  const size_t chunk = l->small ? SMALL_CHUNK : CHUNK;
  for (size_t i = 0; i < count; ++i) {
    const size_t size = types[i] == FT_TYPE_F32 ? 4 : 2;
    for (size_t at = 0; at < elements[i]; at += chunk)
      host.push_back({(char*)ptrs[i] + at * size, (uint32_t)std::min<size_t>(chunk, elements[i] - at), (uint32_t)types[i]});
    if (elements[i])
      l->spans.push_back({(uintptr_t)ptrs[i], (uintptr_t)ptrs[i] + elements[i] * size, i});
    FT_REQUIRE(host.size() < 0x7fffffffull, "ft_grad_list_create: too many elements");
  }
  std::sort(l->spans.begin(), l->spans.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
  uintptr_t reach = 0;
  for (const Span& s : l->spans) {
    if (s.begin < reach) l->disjoint = false;
    reach = std::max(reach, s.end);
  }
  l->chunks = (int)host.size();
  if (count && std::count(l->types.begin(), l->types.end(), types[0]) == (long)count) l->type = types[0];
  FT_CUDA(cudaMalloc((void**)&l->table, std::max<size_t>(1, host.size()) * sizeof(Chunk)));
  FT_CUDA(cudaMalloc((void**)&l->partials, (size_t)list_grid(l) * sizeof(double)));
  if (!host.empty()) {
    FT_CUDA(cudaMemcpyAsync(l->table, host.data(), host.size() * sizeof(Chunk), cudaMemcpyHostToDevice, ctx->stream));
    FT_CUDA(cudaStreamSynchronize(ctx->stream));   // `host` goes away
  }
  return FT_OK;
}

void free_list(FtGradList* l) {
  if (l->table) cudaFree(l->table);
  if (l->partials) cudaFree(l->partials);
  delete l;
}

template <typename TI, typename TO>
int launch_scale(FtContext* ctx, FtGradList* l, const FtGradList* out, float grad_scale, float max_norm, float* norm_out) {
  const int grid = out ? std::max(1, std::min(l->chunks, ctx->sm_count * SCALE_BLOCKS_PER_SM)) : 1;
  FT_LAUNCH_PDL(ctx, (k_list_scale<TI, TO>), grid, LIST_THREADS, 0, l->table, out ? out->table : nullptr, l->chunks,
                l->partials, list_grid(l), grad_scale, max_norm, norm_out, out == l ? 1 : 0);
  return FT_OK;
}

int launch_list(FtContext* ctx, FtGradList* l, const FtGradList* out, float grad_scale, float max_norm, float* norm_out) {
  if (l->small) {   // so is `out`: that follows from the counts alone
    FT_LAUNCH_PDL(ctx, k_list_small, 1, SMALL_THREADS, 0, l->table, out ? out->table : nullptr, l->chunks, grad_scale,
                  max_norm, norm_out, out == l ? 1 : 0);
    return FT_OK;
  }
  FT_LAUNCH_PDL(ctx, k_list_squares, list_grid(l), LIST_THREADS, 0, l->table, l->chunks, l->partials);
  const int from = l->type, to = out ? out->type : -1;
  if (from < 0 || to < 0) return launch_scale<void, void>(ctx, l, out, grad_scale, max_norm, norm_out);
  if (from == FT_TYPE_F32)
    return to == FT_TYPE_F32 ? launch_scale<float, float>(ctx, l, out, grad_scale, max_norm, norm_out)
                             : launch_scale<float, __half>(ctx, l, out, grad_scale, max_norm, norm_out);
  return to == FT_TYPE_F32 ? launch_scale<__half, float>(ctx, l, out, grad_scale, max_norm, norm_out)
                           : launch_scale<__half, __half>(ctx, l, out, grad_scale, max_norm, norm_out);
}

}  // namespace

extern "C" int ft_grad_list_create(FtContext* ctx, size_t count, void* const* ptrs, const size_t* elements,
                                   const int* types, FtGradList** out) {
  FT_REQUIRE(ctx && out && (!count || (ptrs && elements && types)), "ft_grad_list_create: NULL argument");
  *out = nullptr;
  for (size_t i = 0; i < count; ++i) {
    FT_REQUIRE(types[i] == FT_TYPE_F32 || types[i] == FT_TYPE_F16, "ft_grad_list_create: tensor %zu has type %d", i,
               types[i]);
    FT_REQUIRE(ptrs[i] || !elements[i], "ft_grad_list_create: tensor %zu is NULL", i);
    FT_REQUIRE(((uintptr_t)ptrs[i] & (types[i] == FT_TYPE_F32 ? 3 : 1)) == 0,
               "ft_grad_list_create: tensor %zu is not aligned to its elements", i);
    FT_REQUIRE(elements[i] <= ((size_t)1 << 44), "ft_grad_list_create: tensor %zu is too large", i);
  }
  FtDeviceScope on(ctx);
  FtGradList* l = nullptr;
  try {
    l = new FtGradList();
    const int r = create_list(ctx, count, ptrs, elements, types, l);
    if (r != FT_OK) {
      free_list(l);
      return r;
    }
  } catch (const std::exception& e) {   // out of host memory, or a count beyond it
    if (l) free_list(l);
    ft_set_error("ft_grad_list_create: %zu tensors: %s", count, e.what());
    return FT_ERR_INVALID;
  }
  ft_free_retired_lists(ctx);
  *out = l;
  return FT_OK;
}

// Makes no CUDA call: a garbage collector may come here in the middle of a stream capture, which a
// wait or a cudaFree would end.  The next list or the context's end releases the memory.
extern "C" int ft_grad_list_destroy(FtGradList* l) {
  if (!l) return FT_OK;
  l->next = l->ctx->retired_lists;
  l->ctx->retired_lists = l;
  return FT_OK;
}

void ft_free_retired_lists(FtContext* ctx) {
  if (!ctx->retired_lists) return;
  cudaStreamSynchronize(ctx->stream);
  while (FtGradList* l = ctx->retired_lists) {
    ctx->retired_lists = l->next;
    free_list(l);
  }
}

extern "C" int ft_global_grad_norm(FtContext* ctx, FtGradList* grads, float grad_scale, float* norm_out) {
  FT_TRY(check_list("ft_global_grad_norm", ctx, grads));
  FT_REQUIRE(norm_out, "ft_global_grad_norm: norm_out is NULL");
  FT_REQUIRE(((uintptr_t)norm_out & 3) == 0, "ft_global_grad_norm: norm_out is not aligned");
  FT_REQUIRE(isfinite(grad_scale), "ft_global_grad_norm: grad_scale %g is not finite", (double)grad_scale);
  FT_REQUIRE(!overlaps_any(grads->spans, grads->disjoint, (uintptr_t)norm_out, (uintptr_t)(norm_out + 4)),
             "ft_global_grad_norm: norm_out overlaps a gradient");
  FtDeviceScope on(ctx);
  return launch_list(ctx, grads, nullptr, grad_scale, 0.f, norm_out);
}

extern "C" int ft_clip_grad_global_norm(FtContext* ctx, FtGradList* grads, FtGradList* out, float grad_scale,
                                        float max_norm, float* norm_out) {
  const char* who = "ft_clip_grad_global_norm";
  FT_TRY(check_list(who, ctx, grads));
  if (!out) out = grads;
  FT_TRY(check_list(who, ctx, out));
  FT_REQUIRE(isfinite(grad_scale) && !isnan(max_norm), "%s: grad_scale %g or max_norm %g is not a number to scale by", who,
             (double)grad_scale, (double)max_norm);
  FT_REQUIRE(out->disjoint, "%s: tensors that are written overlap one another", who);
  if (out != grads) {
    FT_REQUIRE(out->count == grads->count && out->elements == grads->elements,
               "%s: the two lists hold different numbers of tensors or elements", who);
    // by address, every tensor that is written against those read from where it lies
    size_t j = 0;
    const std::vector<Span>& rd = grads->spans;
    for (const Span& w : out->spans) {
      if (grads->disjoint)
        while (j < rd.size() && rd[j].end <= w.begin) ++j;
      for (size_t k = grads->disjoint ? j : 0; k < rd.size() && rd[k].begin < w.end; ++k)
        FT_REQUIRE(rd[k].end <= w.begin || (rd[k].index == w.index && rd[k].begin == w.begin &&
                                            grads->types[w.index] == out->types[w.index]),
                   "%s: tensor %zu of the output overlaps gradient %zu", who, w.index, rd[k].index);
    }
  }
  if (norm_out) {
    const uintptr_t b = (uintptr_t)norm_out, e = (uintptr_t)(norm_out + 4);
    FT_REQUIRE((b & 3) == 0, "%s: norm_out is not aligned", who);
    FT_REQUIRE(!overlaps_any(grads->spans, grads->disjoint, b, e) && !overlaps_any(out->spans, true, b, e),
               "%s: norm_out overlaps a tensor", who);
  }
  FtDeviceScope on(ctx);
  return launch_list(ctx, grads, out, grad_scale, max_norm, norm_out);
}
