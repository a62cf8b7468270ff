// Global gradient norm over many tensors, and clipping them in place (ldm_grad_norm).
//
//   norm   = sqrt(sum g^2), max |g| or sum |g| over every element of every tensor
//   factor = min(1, max_norm / (norm + 1e-6));  g *= factor   (torch.nn.utils.clip_grad_norm_)
// The spans' addresses travel as kernel arguments, up to TABLE of them to a launch: nothing is
// copied to the device, nothing is kept between calls, and a captured graph holds its own table.
// Squares are summed in fp64 (a square of any fp32 value is finite there), per thread, block and
// partial in a fixed order: the same gradients give the same bits.
#include "common.h"

#include <math.h>

#include <algorithm>
#include <vector>

namespace {

constexpr int TABLE = 224;               // spans to a launch: 16 B each, below the 4 KB of kernel arguments
constexpr int PACKS = 8;                 // 16-byte packs of a chunk to a thread, all in flight: 32 KB to a block
constexpr int MAX_BLOCKS = 2048;

template <typename T> struct Pack { T v[16 / sizeof(T)]; };
template <typename T> constexpr int chunk_of() { return 256 * PACKS * 16 / (int)sizeof(T); }

struct Entry {
  uint64_t ptr;                          // bit 63: bf16
  uint32_t n, chunk0;                    // elements, first chunk
};
struct Table {
  Entry e[TABLE];
  int count, chunks;
};

__device__ __forceinline__ int entry_of(const Table& t, int chunk) {   // the last entry with chunk0 <= chunk
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((int)t.e[mid].chunk0 <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <int NORM> __device__ __forceinline__ double norm_add(double acc, float g) {
  if (NORM == LDM_NORM_2) return fma((double)g, (double)g, acc);
  if (NORM == LDM_NORM_1) return acc + fabs((double)g);
  const double a = fabs((double)g);
  return (a > acc || a != a) ? a : acc;          // a NaN stays
}
template <int NORM> __device__ __forceinline__ double norm_join(double a, double b) {
  if (NORM != LDM_NORM_INF) return a + b;
  return (b > a || b != b) ? b : a;
}
template <int NORM> __device__ __forceinline__ double block_join(double v) {
  __shared__ double part[4];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = norm_join<NORM>(v, __shfl_xor(v, o, 64));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return norm_join<NORM>(norm_join<NORM>(part[0], part[1]), norm_join<NORM>(part[2], part[3]));
}

// A thread's packs of a chunk's elements [0, n), at any address aligned to one element: all loads in flight.
// pack(index, pack) for each whole one, rest(element) for the elements behind the last.
template <typename T, typename P, typename R>
__device__ __forceinline__ void each_pack(const T* g, int n, P pack, R rest) {
  constexpr int V = 16 / (int)sizeof(T);
  Pack<T> p[PACKS];
  if (n == chunk_of<T>()) {
#pragma unroll
    for (int i = 0; i < PACKS; ++i) __builtin_memcpy(&p[i], g + (i * 256 + threadIdx.x) * V, 16);
#pragma unroll
    for (int i = 0; i < PACKS; ++i) pack(i * 256 + (int)threadIdx.x, p[i]);
    return;
  }
  const int whole = n / V, last = whole * V + (int)threadIdx.x;
#pragma unroll
  for (int i = 0; i < PACKS; ++i)
    if (i * 256 + (int)threadIdx.x < whole) __builtin_memcpy(&p[i], g + (i * 256 + threadIdx.x) * V, 16);
  if (last < n) rest(last);
#pragma unroll
  for (int i = 0; i < PACKS; ++i)
    if (i * 256 + (int)threadIdx.x < whole) pack(i * 256 + (int)threadIdx.x, p[i]);
}

template <int NORM, typename T>
__device__ __forceinline__ double chunk_norm(const T* g, int n, double acc) {
  each_pack(g, n, [&](int, const Pack<T>& p) {
#pragma unroll
    for (int j = 0; j < 16 / (int)sizeof(T); ++j) acc = norm_add<NORM>(acc, to_f(p.v[j]));
  }, [&](int i) { acc = norm_add<NORM>(acc, to_f(g[i])); });
  return acc;
}

// chunk c of a table: calls f(pointer, elements) with the span's type
template <typename F> __device__ __forceinline__ void with_chunk(const Table& t, int c, F f) {
  const Entry e = t.e[entry_of(t, c)];
  const int64_t k = c - (int)e.chunk0;
  if (e.ptr >> 63) {
    const int64_t at = k * chunk_of<bf16_t>();
    f((bf16_t*)(e.ptr & ~(1ull << 63)) + at, (int)min((int64_t)chunk_of<bf16_t>(), (int64_t)e.n - at));
  } else {
    const int64_t at = k * chunk_of<float>();
    f((float*)e.ptr + at, (int)min((int64_t)chunk_of<float>(), (int64_t)e.n - at));
  }
}

template <int NORM>
__global__ __launch_bounds__(256) void norm_parts(const Table t, double* __restrict__ part) {
  double acc = 0.0;
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x)
    with_chunk(t, c, [&](const auto* g, int n) { acc = chunk_norm<NORM>(g, n, acc); });
  acc = block_join<NORM>(acc);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

// min(1, max / (norm + 1e-6)) with a NaN kept, in fp32 from the rounded norm
__device__ __forceinline__ float factor_of(float norm, float max_norm) {
  const float f = max_norm / (norm + 1e-6f);
  return f > 1.f ? 1.f : f;
}

// the partials joined: the norm and the factor, in every thread of the block
template <int NORM>
__device__ __forceinline__ float2 norm_of(const double* __restrict__ part, int parts, float max_norm) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < parts; i += 256) acc = norm_join<NORM>(acc, part[i]);
  acc = block_join<NORM>(acc);
  const float norm = (float)(NORM == LDM_NORM_2 ? sqrt(acc) : acc);
  return make_float2(norm, factor_of(norm, max_norm));
}

template <int NORM>
__global__ __launch_bounds__(256) void norm_final(const double* __restrict__ part, int parts, float max_norm,
                                                  float* __restrict__ out) {
  const float2 r = norm_of<NORM>(part, parts, max_norm);
  if (threadIdx.x == 0) { out[0] = r.x; out[1] = r.y; }
}

// a gradient is multiplied by the factor as its own type holds it and rounded once, as torch's in-place product
// of a tensor with a device scalar is: a bf16 gradient's factor has 8 bits
template <typename T>
__device__ __forceinline__ void chunk_scale(T* g, int n, float factor) {
  constexpr int V = 16 / (int)sizeof(T);
  const float f = to_f(from_f<T>(factor));
  if (f == 1.f) return;
  each_pack(g, n, [&](int i, Pack<T> p) {
#pragma unroll
    for (int j = 0; j < V; ++j) p.v[j] = from_f<T>(to_f(p.v[j]) * f);
    __builtin_memcpy(g + i * V, &p, 16);
  }, [&](int i) { g[i] = from_f<T>(to_f(g[i]) * f); });
}

// the last chunks first: the norm's pass has left them in the memory-side cache
__device__ __forceinline__ void scale_chunks(const Table& t, float f) {
  if (f == 1.f) return;
  for (int c = t.chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x)
    with_chunk(t, c, [&](auto* g, int n) { chunk_scale(g, n, f); });
}
__global__ __launch_bounds__(256) void scale_all(const Table t, const float* __restrict__ out) {
  scale_chunks(t, out[1]);
}
// the same for one table with few partials: every block joins them itself, which takes a launch less
template <int NORM>
__global__ __launch_bounds__(256) void scale_joined(const Table t, const double* __restrict__ part, int parts,
                                                    float max_norm, float* __restrict__ out) {
  const float2 r = norm_of<NORM>(part, parts, max_norm);
  if (blockIdx.x == 0 && threadIdx.x == 0) { out[0] = r.x; out[1] = r.y; }
  scale_chunks(t, r.y);
}

// a span above 2^30 elements is listed in pieces (of whole chunks)
constexpr int64_t PIECE = 1LL << 30;
int64_t entries_of(const int64_t* numel, int n) {
  int64_t c = 0;
  for (int i = 0; i < n; ++i) c += (numel[i] + PIECE - 1) / PIECE;
  return c;
}

constexpr int JOIN_PARTS = 512;          // two partials a thread

template <int NORM>
int launch(const std::vector<Table>& tables, float max_norm, int clip, float* out, double* part, hipStream_t s) {
  int parts = 0;
  if (clip != 2) {
    for (const Table& t : tables) {
      const int blocks = std::min(t.chunks, MAX_BLOCKS);
      hipLaunchKernelGGL((norm_parts<NORM>), dim3(blocks), dim3(256), 0, s, t, part + parts);
      LDM_CHECK_LAUNCH();
      parts += blocks;
    }
    if (clip == 1 && tables.size() == 1 && parts <= JOIN_PARTS) {
      hipLaunchKernelGGL((scale_joined<NORM>), dim3(parts), dim3(256), 0, s, tables[0], part, parts, max_norm, out);
      LDM_CHECK_LAUNCH();
      return LDM_OK;
    }
    hipLaunchKernelGGL((norm_final<NORM>), dim3(1), dim3(256), 0, s, part, parts, max_norm, out);
    LDM_CHECK_LAUNCH();
  }
  if (clip)
    for (size_t i = tables.size(); i-- > 0;) {
      const Table& t = tables[i];
      hipLaunchKernelGGL(scale_all, dim3(std::min(t.chunks, MAX_BLOCKS)), dim3(256), 0, s, t, out);
      LDM_CHECK_LAUNCH();
    }
  return LDM_OK;
}

}  // namespace

extern "C" size_t ldm_grad_norm_workspace_bytes(const int64_t* numel, int ntensors) {
  if (!numel || ntensors <= 0) return 0;
  return (size_t)((entries_of(numel, ntensors) + TABLE - 1) / TABLE) * MAX_BLOCKS * sizeof(double);
}

extern "C" int ldm_grad_norm(const void* const* ptrs, const int64_t* numel, const uint8_t* dtypes, int ntensors,
                             int norm_type, double max_norm, int clip, float* out, void* workspace,
                             int64_t workspace_bytes, ldm_stream_t stream) {
  if (!ptrs || !numel || !dtypes || !out || ntensors <= 0 || clip < 0 || clip > 2) return LDM_ERR_ARG;
  if (norm_type < LDM_NORM_2 || norm_type > LDM_NORM_1 || !(max_norm >= 0.0)) return LDM_ERR_ARG;
  const int64_t need = clip == 2 ? 0 : (int64_t)ldm_grad_norm_workspace_bytes(numel, ntensors);
  if (need && (!workspace || workspace_bytes < need)) return LDM_ERR_ARG;
  // Tensors in the order of their addresses; those that lie back to back (views of a bucket) are one span.
  struct Span { uint64_t lo, hi, size; };
  std::vector<Span> spans;
  std::vector<Table> tables;
  try {
    spans.reserve(ntensors);
    for (int i = 0; i < ntensors; ++i) {
      if (numel[i] < 0 || dtypes[i] > LDM_BF16) return LDM_ERR_ARG;
      if (numel[i] == 0) continue;
      const uint64_t a = reinterpret_cast<uint64_t>(ptrs[i]);
      const uint64_t size = dtypes[i] == LDM_BF16 ? 2 : 4;
      if (!a || (a >> 63)) return LDM_ERR_ARG;
      if (a % size) return LDM_ERR_ALIGN;
      spans.push_back({a, a + size * (uint64_t)numel[i], size});
    }
    std::sort(spans.begin(), spans.end(), [](const Span& p, const Span& q) { return p.lo < q.lo; });
    size_t last = 0;
    for (size_t i = 1; i < spans.size(); ++i) {
      if (spans[i].lo < spans[last].hi) return LDM_ERR_OVERLAP;
      if (spans[i].lo == spans[last].hi && spans[i].size == spans[last].size) spans[last].hi = spans[i].hi;
      else spans[++last] = spans[i];
    }
    if (!spans.empty()) spans.resize(last + 1);
    for (const Span& p : spans) {
      const int64_t total = (int64_t)((p.hi - p.lo) / p.size);
      const int64_t chunk = p.size == 2 ? chunk_of<bf16_t>() : chunk_of<float>();
      for (int64_t at = 0; at < total; at += PIECE) {
        if (tables.empty() || tables.back().count == TABLE) {
          tables.emplace_back();
          tables.back().count = tables.back().chunks = 0;
        }
        Table& t = tables.back();
        const int64_t n = std::min(PIECE, total - at);
        t.e[t.count++] = {(p.lo + p.size * (uint64_t)at) | ((uint64_t)(p.size == 2) << 63), (uint32_t)n,
                          (uint32_t)t.chunks};
        t.chunks += (int)((n + chunk - 1) / chunk);
      }
    }
  } catch (...) {
    return LDM_ERR_ARG;
  }
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  double* part = static_cast<double*>(workspace);
  if (norm_type == LDM_NORM_2) return launch<LDM_NORM_2>(tables, (float)max_norm, clip, out, part, s);
  if (norm_type == LDM_NORM_INF) return launch<LDM_NORM_INF>(tables, (float)max_norm, clip, out, part, s);
  return launch<LDM_NORM_1>(tables, (float)max_norm, clip, out, part, s);
}
