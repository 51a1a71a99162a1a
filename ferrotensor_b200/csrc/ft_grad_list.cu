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
// its first reads find in L2 what the norm read last.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <new>
#include <vector>

#include "ft_common.cuh"

namespace {

constexpr int LIST_THREADS = 256;
constexpr int CHUNK = 8192;            // elements; a thread's share of one is eight 16-byte loads of f32
constexpr int LIST_BLOCKS_PER_SM = 8;

struct Chunk {
  void* p;
  uint32_t n;
  uint32_t type;
};

// Squares are taken and summed in f64: an f32 square leaves the f32 range for |g| above 1.8e19 or
// below 1e-19.
__device__ __forceinline__ double sum_squares_chunk(const Chunk& c) {
  double acc = 0.0;
  if (c.type == FT_TYPE_F32) {
    const float* x = (const float*)c.p;
    for (uint32_t i = threadIdx.x; i < c.n; i += LIST_THREADS) acc = fma((double)x[i], (double)x[i], acc);
  } else {
    const __half* x = (const __half*)c.p;
    for (uint32_t i = threadIdx.x; i < c.n; i += LIST_THREADS) {
      const double v = (double)__half2float(x[i]);
      acc = fma(v, v, acc);
    }
  }
  return acc;
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

__global__ void __launch_bounds__(LIST_THREADS)
k_list_squares(const Chunk* __restrict__ chunks, int count, double* __restrict__ partials) {
  __shared__ double red[LIST_THREADS / 32];
  ft_pdl_wait();
  ft_pdl_launch();
  double acc = 0.0;
  for (int c = blockIdx.x; c < count; c += gridDim.x) acc += sum_squares_chunk(chunks[c]);
  acc = block_sum_f64(acc, red);
  if (threadIdx.x == 0) partials[blockIdx.x] = acc;
}

__device__ __forceinline__ float load_one(const Chunk& c, uint32_t i) {
  return c.type == FT_TYPE_F32 ? ((const float*)c.p)[i] : __half2float(((const __half*)c.p)[i]);
}

// Every block joins the partial sums itself (the same order everywhere), block 0 publishes.
// out == NULL: measure only.
__global__ void __launch_bounds__(LIST_THREADS)
k_list_scale(const Chunk* __restrict__ chunks, const Chunk* __restrict__ out, int count,
             const double* __restrict__ partials, int parts, float grad_scale, float max_norm,
             float* __restrict__ norm_out, int in_place) {
  __shared__ double red[LIST_THREADS / 32];
  ft_pdl_wait();
  ft_pdl_launch();
  double acc = 0.0;
  for (int i = threadIdx.x; i < parts; i += LIST_THREADS) acc += partials[i];
  const double norm = sqrt(block_sum_f64(acc, red)) * fabs((double)grad_scale);
  const bool finite = isfinite((float)norm);
  float factor = grad_scale;
  if (finite && max_norm > 0.f && norm > (double)max_norm)
    factor = (float)((double)grad_scale * (double)max_norm / (norm + 1e-6));
  if (blockIdx.x == 0 && threadIdx.x == 0 && norm_out) {
    norm_out[0] = (float)norm;
    norm_out[1] = finite ? 1.f : 0.f;
    norm_out[2] = factor;
  }
  if (!out || !finite || (in_place && factor == 1.0f)) return;
  for (int k = blockIdx.x; k < count; k += gridDim.x) {
    const int c = count - 1 - k;
    const Chunk src = chunks[c], dst = out[c];
    if (dst.type == FT_TYPE_F32) {
      for (uint32_t i = threadIdx.x; i < src.n; i += LIST_THREADS) ((float*)dst.p)[i] = factor * load_one(src, i);
    } else {
      for (uint32_t i = threadIdx.x; i < src.n; i += LIST_THREADS)
        ((__half*)dst.p)[i] = __float2half_rn(factor * load_one(src, i));
    }
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
  int chunks = 0;
  Chunk* table = nullptr;       // [chunks] on the device
  double* partials = nullptr;   // one sum for each block of k_list_squares
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
  for (size_t i = 0; i < count; ++i) {
    const size_t size = types[i] == FT_TYPE_F32 ? 4 : 2;
    for (size_t at = 0; at < elements[i]; at += CHUNK)
      host.push_back({(char*)ptrs[i] + at * size, (uint32_t)std::min<size_t>(CHUNK, elements[i] - at), (uint32_t)types[i]});
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

int launch_list(FtContext* ctx, FtGradList* l, const Chunk* out, float grad_scale, float max_norm, float* norm_out,
                bool in_place) {
  const int grid = list_grid(l);
  FT_LAUNCH_PDL(ctx, k_list_squares, grid, LIST_THREADS, 0, l->table, l->chunks, l->partials);
  FT_LAUNCH_PDL(ctx, k_list_scale, out ? grid : 1, LIST_THREADS, 0, l->table, out, l->chunks, l->partials, grid,
                grad_scale, max_norm, norm_out, in_place ? 1 : 0);
  return FT_OK;
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
  } catch (const std::bad_alloc&) {
    if (l) free_list(l);
    ft_set_error("ft_grad_list_create: out of host memory");
    return FT_ERR_INVALID;
  }
  *out = l;
  return FT_OK;
}

extern "C" int ft_grad_list_destroy(FtGradList* l) {
  if (!l) return FT_OK;
  FtDeviceScope on(l->ctx);
  cudaStreamSynchronize(l->ctx->stream);
  free_list(l);
  return FT_OK;
}

extern "C" int ft_global_grad_norm(FtContext* ctx, FtGradList* grads, float grad_scale, float* norm_out) {
  FT_TRY(check_list("ft_global_grad_norm", ctx, grads));
  FT_REQUIRE(norm_out, "ft_global_grad_norm: norm_out is NULL");
  FT_REQUIRE(((uintptr_t)norm_out & 3) == 0, "ft_global_grad_norm: norm_out is not aligned");
  FT_REQUIRE(isfinite(grad_scale), "ft_global_grad_norm: grad_scale %g is not finite", (double)grad_scale);
  FT_REQUIRE(!overlaps_any(grads->spans, grads->disjoint, (uintptr_t)norm_out, (uintptr_t)(norm_out + 4)),
             "ft_global_grad_norm: norm_out overlaps a gradient");
  FtDeviceScope on(ctx);
  return launch_list(ctx, grads, nullptr, grad_scale, 0.f, norm_out, false);
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
  return launch_list(ctx, grads, out->table, grad_scale, max_norm, norm_out, out == grads);
}
