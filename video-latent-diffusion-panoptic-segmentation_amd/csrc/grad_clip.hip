// Global gradient norm over many tensors, and clipping them in place (ldm_grad_norm).
//
//   norm   = sqrt(sum g^2), max |g| or sum |g| over every element of every tensor
//   factor = min(1, max_norm / (norm + 1e-6));  g *= factor   (torch.nn.utils.clip_grad_norm_)
// The spans' addresses travel as kernel arguments, up to TABLE of them to a launch; more are listed
// in the workspace by a launch for each table.  Nothing is copied from the host, nothing is kept
// between calls, and a captured graph holds its own tables.
// Squares are summed in fp64 (a square of any fp32 value is finite there), per thread, block and
// partial in an order that the addresses fix: the same call gives the same bits.
// Memory bounds it: a norm reads every gradient, a clip reads them twice and writes them once.  815 M fp32 values:
// 1.83 ms of clip (5.3 TB/s, a copy's rate), the norm alone of as many in bf16 0.26 to 0.29 ms (5.6 to 6.3 TB/s).
#include "common.h"

#include <math.h>

#include <algorithm>
#include <vector>

namespace {

constexpr int TABLE = 224;               // spans to a launch: 16 B each, below the 4 KB of kernel arguments
// A chunk is a block's: PACKS packs of 16 bytes to a thread, all in flight.  8 of them (32 KB) carry the most bytes a
// second; a call of less than SMALL_BYTES takes 2, for more blocks (1.2 MB: 8.5 us, 10.2 us with 8).
constexpr int LARGE_PACKS = 8, SMALL_PACKS = 2;
constexpr int64_t SMALL_BYTES = 8 << 20;
constexpr int MAX_BLOCKS = 2048;
constexpr int JOIN_CHUNKS = 1024;        // up to here a launch costs more than every block's own join of the partials
                                         // (1.8 M values: 9.4 us joined, 11.1 us with a launch between)

template <typename T> struct Pack { T v[16 / sizeof(T)]; };
constexpr int chunk_bytes(int packs) { return 256 * 16 * packs; }
template <typename T, int PACKS> constexpr int chunk_of() { return chunk_bytes(PACKS) / (int)sizeof(T); }

struct Entry {
  uint64_t ptr;                          // bit 63: bf16
  uint32_t n, chunk0;                    // elements, first chunk
};
template <int P> struct Table {
  static constexpr int packs = P;
  Entry e[TABLE];
  int count, chunks;
};

template <int P> __device__ __forceinline__ int entry_of(const Table<P>& t, int chunk) {   // the last entry with chunk0 <= chunk
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
template <int NORM, int WAVES = 4> __device__ __forceinline__ double block_join(double v) {
  __shared__ double part[WAVES];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = norm_join<NORM>(v, __shfl_xor(v, o, 64));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) v = norm_join<NORM>(v, part[w]);
  return v;
}

// A thread's packs of a chunk's elements [0, n), at any address aligned to one element: all loads in flight, then
// ready() (false: nothing more), pack(index, pack) for each whole one and rest(element, value) for an element behind
// the last.
template <int PACKS, typename T, typename Q, typename P, typename R>
__device__ __forceinline__ void each_pack(const T* g, int n, Q ready, P pack, R rest) {
  constexpr int V = 16 / (int)sizeof(T);
  Pack<T> p[PACKS];
  if (n == chunk_of<T, PACKS>()) {
#pragma unroll
    for (int i = 0; i < PACKS; ++i) __builtin_memcpy(&p[i], g + (i * 256 + threadIdx.x) * V, 16);
    if (!ready()) return;
#pragma unroll
    for (int i = 0; i < PACKS; ++i) pack(i * 256 + (int)threadIdx.x, p[i]);
    return;
  }
  const int whole = n / V, last = whole * V + (int)threadIdx.x;
  T tail = T(0);
  if (last < n) tail = g[last];
#pragma unroll
  for (int i = 0; i < PACKS; ++i)
    if (i * 256 + (int)threadIdx.x < whole) __builtin_memcpy(&p[i], g + (i * 256 + threadIdx.x) * V, 16);
  if (!ready()) return;
  if (last < n) rest(last, tail);
#pragma unroll
  for (int i = 0; i < PACKS; ++i)
    if (i * 256 + (int)threadIdx.x < whole) pack(i * 256 + (int)threadIdx.x, p[i]);
}

template <int NORM, int PACKS, typename T>
__device__ __forceinline__ double chunk_norm(const T* g, int n, double acc) {
  each_pack<PACKS>(g, n, [] { return true; }, [&](int, const Pack<T>& p) {
#pragma unroll
    for (int j = 0; j < 16 / (int)sizeof(T); ++j) acc = norm_add<NORM>(acc, to_f(p.v[j]));
  }, [&](int, T v) { acc = norm_add<NORM>(acc, to_f(v)); });
  return acc;
}

// Where a kernel's chunks come from: a table in its arguments, or (more spans than a table holds) a list in the
// workspace that list_chunks wrote.  with_chunk calls f(pointer, elements) with chunk c's type.
struct Chunk {
  uint64_t ptr;                          // bit 63: bf16
  int n;
};
template <int P> struct ChunkList {
  static constexpr int packs = P;
  const Chunk* at;
  int chunks;
};
template <int P> __device__ __forceinline__ Chunk chunk_at(const ChunkList<P>& l, int c) { return l.at[c]; }
template <int P> __device__ __forceinline__ Chunk chunk_of_entry(const Entry& e, int k) {
  const int64_t len = e.ptr >> 63 ? chunk_of<bf16_t, P>() : chunk_of<float, P>(), at = k * len;
  return {e.ptr + (uint64_t)k * chunk_bytes(P), (int)min(len, (int64_t)e.n - at)};
}
template <int P> __device__ __forceinline__ Chunk chunk_at(const Table<P>& t, int c) {
  const Entry e = t.e[entry_of(t, c)];
  return chunk_of_entry<P>(e, c - (int)e.chunk0);
}
template <typename S, typename F> __device__ __forceinline__ void with_chunk(const S& s, int c, F f) {
  const Chunk k = chunk_at(s, c);
  if (k.ptr >> 63) f((bf16_t*)(k.ptr & ~(1ull << 63)), k.n);
  else f((float*)k.ptr, k.n);
}

// a table's chunks, a block for each span
template <int P>
__global__ __launch_bounds__(64) void list_chunks(const Table<P> t, Chunk* __restrict__ to) {
  const Entry e = t.e[blockIdx.x];
  const int n = (blockIdx.x + 1 < (unsigned)t.count ? (int)t.e[blockIdx.x + 1].chunk0 : t.chunks) - (int)e.chunk0;
  for (int k = threadIdx.x; k < n; k += 64) to[(int)e.chunk0 + k] = chunk_of_entry<P>(e, k);
}

template <int NORM, typename S>
__global__ __launch_bounds__(256) void norm_parts(const S t, double* __restrict__ part) {
  double acc = 0.0;
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x)
    with_chunk(t, c, [&](const auto* g, int n) { acc = chunk_norm<NORM, S::packs>(g, n, acc); });
  acc = block_join<NORM>(acc);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

// min(1, max / (norm + 1e-6)) with a NaN kept, in fp32 from the rounded norm
__device__ __forceinline__ float factor_of(float norm, float max_norm) {
  const float f = max_norm / (norm + 1e-6f);
  return f > 1.f ? 1.f : f;
}

// the threads' sums joined: the norm and the factor, in every thread of the block
template <int NORM>
__device__ __forceinline__ float2 norm_of(double acc, float max_norm) {
  acc = block_join<NORM>(acc);
  const float norm = (float)(NORM == LDM_NORM_2 ? sqrt(acc) : acc);
  return make_float2(norm, factor_of(norm, max_norm));
}

template <int NORM>
__global__ __launch_bounds__(256) void norm_final(const double* __restrict__ part, int parts, float max_norm,
                                                  float* __restrict__ out) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < parts; i += 256) acc = norm_join<NORM>(acc, part[i]);
  const float2 r = norm_of<NORM>(acc, max_norm);
  if (threadIdx.x == 0) { out[0] = r.x; out[1] = r.y; }
}

// a gradient is multiplied by the factor as its own type holds it and rounded once, as torch's in-place product
// of a tensor with a device scalar is: a bf16 gradient's factor has 8 bits
template <int PACKS, typename T, typename F>
__device__ __forceinline__ void chunk_scale(T* g, int n, F factor) {
  constexpr int V = 16 / (int)sizeof(T);
  float f;
  each_pack<PACKS>(g, n, [&] { f = to_f(from_f<T>(factor())); return f != 1.f; }, [&](int i, Pack<T> p) {
#pragma unroll
    for (int j = 0; j < V; ++j) p.v[j] = from_f<T>(to_f(p.v[j]) * f);
    __builtin_memcpy(g + i * V, &p, 16);
  }, [&](int i, T v) { g[i] = from_f<T>(to_f(v) * f); });
}

// the last chunks first: the norm's pass has left them in the memory-side cache (400 MB: 213 us, 244 us from the
// front; 3.3 GB: no difference).  A block to each 4 KB would scale 3.3 GB in 1.10 ms for 1.29, but its 3 million waves
// cost 0.17 ms where the factor is 1 and there is nothing to do; 2048 blocks leave that at 5 us.
template <typename S>
__global__ __launch_bounds__(256) void scale_all(const S t, const float* __restrict__ out) {
  const float f = out[1];
  if (f == 1.f) return;
  for (int c = t.chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x)
    with_chunk(t, c, [&](auto* g, int n) { chunk_scale<S::packs>(g, n, [&] { return f; }); });
}
// the same where partials are few: every block joins them itself, beside its first chunk's loads, which takes a
// launch less
template <int NORM, typename S>
__global__ __launch_bounds__(256) void scale_joined(const S t, const double* __restrict__ part, int parts,
                                                    float max_norm, float* __restrict__ out) {
  double p[JOIN_CHUNKS / 256];
#pragma unroll
  for (int j = 0; j < JOIN_CHUNKS / 256; ++j) {
    const int i = j * 256 + (int)threadIdx.x;
    p[j] = i < parts ? part[i] : 0.0;              // 0 adds nothing to any of the norms
  }
  float f = -1.f;
  for (int c = t.chunks - 1 - (int)blockIdx.x; c >= 0 && f != 1.f; c -= gridDim.x)
    with_chunk(t, c, [&](auto* g, int n) {
      chunk_scale<S::packs>(g, n, [&] {
        if (f == -1.f) {
          double acc = p[0];
#pragma unroll
          for (int j = 1; j < JOIN_CHUNKS / 256; ++j) acc = norm_join<NORM>(acc, p[j]);
          const float2 r = norm_of<NORM>(acc, max_norm);
          if (blockIdx.x == 0 && threadIdx.x == 0) { out[0] = r.x; out[1] = r.y; }
          f = r.y;
        }
        return f;
      });
    });
}

// Few gradients in one launch of one block: every thread holds up to UNITS packs between the norm and the product,
// so nothing is read twice.  A unit is a wave's 64 packs of one span; `span` names each unit's.  16 KB: 5.4 us, 8 us
// in two launches; above 80 KB one compute unit's share of the bandwidth costs more than the launch.
constexpr int UNITS = 5, SMALL_WAVES = 16, SMALL_SPANS = 64;
struct SmallTable {
  Entry e[SMALL_SPANS];                    // chunk0: the span's first unit
  uint8_t span[UNITS * SMALL_WAVES];
  int units;
};
template <typename T> __device__ __forceinline__ uint4 load_part(const T* g, int n) {   // n elements, then zeros
  constexpr int V = 16 / (int)sizeof(T);
  Pack<T> p;
  if (n >= V) {
    __builtin_memcpy(&p, g, 16);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) p.v[j] = j < n ? g[j] : T(0);
  }
  return __builtin_bit_cast(uint4, p);
}
template <int NORM, typename T> __device__ __forceinline__ double part_norm(const uint4& r, double acc) {
  const Pack<T> p = __builtin_bit_cast(Pack<T>, r);
#pragma unroll
  for (int j = 0; j < 16 / (int)sizeof(T); ++j) acc = norm_add<NORM>(acc, to_f(p.v[j]));
  return acc;
}
template <typename T> __device__ __forceinline__ void store_part(T* g, int n, const uint4& r, float f) {
  constexpr int V = 16 / (int)sizeof(T);
  Pack<T> p = __builtin_bit_cast(Pack<T>, r);
#pragma unroll
  for (int j = 0; j < V; ++j) p.v[j] = from_f<T>(to_f(p.v[j]) * f);
  if (n >= V) {
    __builtin_memcpy(g, &p, 16);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < n) g[j] = p.v[j];
  }
}
template <int NORM>
__global__ __launch_bounds__(64 * SMALL_WAVES) void clip_small(const SmallTable t, float max_norm, int clip,
                                                               float* __restrict__ out) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  uint4 r[UNITS];
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    const int u = i * SMALL_WAVES + wave;
    if (u < t.units) {
      const Entry e = t.e[t.span[u]];
      const int pack = (u - (int)e.chunk0) * 64 + lane, n = (int)e.n;
      r[i] = e.ptr >> 63 ? load_part((const bf16_t*)(e.ptr & ~(1ull << 63)) + min(pack * 8, n), n - pack * 8)
                         : load_part((const float*)e.ptr + min(pack * 4, n), n - pack * 4);
    }
  }
  double acc = 0.0;
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    const int u = i * SMALL_WAVES + wave;
    if (u < t.units) acc = t.e[t.span[u]].ptr >> 63 ? part_norm<NORM, bf16_t>(r[i], acc) : part_norm<NORM, float>(r[i], acc);
  }
  acc = block_join<NORM, SMALL_WAVES>(acc);
  const float norm = (float)(NORM == LDM_NORM_2 ? sqrt(acc) : acc), f = factor_of(norm, max_norm);
  if (threadIdx.x == 0) { out[0] = norm; out[1] = f; }
  if (!clip || f == 1.f) return;
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    const int u = i * SMALL_WAVES + wave;
    if (u < t.units) {
      const Entry e = t.e[t.span[u]];
      const int pack = (u - (int)e.chunk0) * 64 + lane, n = (int)e.n;
      if (e.ptr >> 63) store_part((bf16_t*)(e.ptr & ~(1ull << 63)) + min(pack * 8, n), n - pack * 8, r[i], to_f(from_f<bf16_t>(f)));
      else store_part((float*)e.ptr + min(pack * 4, n), n - pack * 4, r[i], f);
    }
  }
}

// a span above 2^30 elements is listed in pieces (of whole chunks)
constexpr int64_t PIECE = 1LL << 30;
// Values of a call at most: no sum of sizes or addresses below leaves 64 bits
constexpr int64_t MOST_VALUES = 1LL << 46;
int64_t entries_of(const int64_t* numel, int n) {
  int64_t c = 0;
  for (int i = 0; i < n; ++i) c += (numel[i] + PIECE - 1) / PIECE;
  return c;
}

template <int NORM, typename S>
int launch(const S& t, float max_norm, int clip, float* out, double* part, hipStream_t s) {
  const dim3 grid(std::max(1, std::min(t.chunks, MAX_BLOCKS))), block(256);
  if (clip != 2) {
    hipLaunchKernelGGL((norm_parts<NORM, S>), grid, block, 0, s, t, part);
    LDM_CHECK_LAUNCH();
    if (clip == 1 && t.chunks > 0 && t.chunks <= JOIN_CHUNKS) {
      hipLaunchKernelGGL((scale_joined<NORM, S>), grid, block, 0, s, t, part, (int)grid.x, max_norm, out);
      LDM_CHECK_LAUNCH();
      return LDM_OK;
    }
    hipLaunchKernelGGL((norm_final<NORM>), dim3(1), block, 0, s, part, (int)grid.x, max_norm, out);
    LDM_CHECK_LAUNCH();
  }
  if (clip) {
    hipLaunchKernelGGL((scale_all<S>), grid, block, 0, s, t, out);
    LDM_CHECK_LAUNCH();
  }
  return LDM_OK;
}
template <typename S>
int launch(const S& t, int norm_type, float max_norm, int clip, float* out, double* part, hipStream_t s) {
  if (norm_type == LDM_NORM_2) return launch<LDM_NORM_2>(t, max_norm, clip, out, part, s);
  if (norm_type == LDM_NORM_INF) return launch<LDM_NORM_INF>(t, max_norm, clip, out, part, s);
  return launch<LDM_NORM_1>(t, max_norm, clip, out, part, s);
}

int launch_small(const SmallTable& t, int norm_type, float max_norm, int clip, float* out, hipStream_t s) {
  const dim3 one(1), block(64 * SMALL_WAVES);
  if (norm_type == LDM_NORM_2) hipLaunchKernelGGL((clip_small<LDM_NORM_2>), one, block, 0, s, t, max_norm, clip, out);
  else if (norm_type == LDM_NORM_INF) hipLaunchKernelGGL((clip_small<LDM_NORM_INF>), one, block, 0, s, t, max_norm, clip, out);
  else hipLaunchKernelGGL((clip_small<LDM_NORM_1>), one, block, 0, s, t, max_norm, clip, out);
  LDM_CHECK_LAUNCH();
  return LDM_OK;
}

}  // namespace

// partials, and behind them the chunk list where there may be more spans than a table holds: no more chunks than
// fp32 ones of the size that the call may take
extern "C" size_t ldm_grad_norm_workspace_bytes(const int64_t* numel, int ntensors) {
  if (!numel || ntensors <= 0) return 0;
  int64_t total = 0, small = 0, large = 0, units = 0;
  for (int i = 0; i < ntensors; ++i)
    if (numel[i] > 0) {
      if (numel[i] > MOST_VALUES - total) return 0;                           // ldm_grad_norm refuses it
      total += numel[i];
      units += (numel[i] * 4 + 1023) / 1024;
      small += (numel[i] + chunk_of<float, SMALL_PACKS>() - 1) / chunk_of<float, SMALL_PACKS>();
      large += (numel[i] + chunk_of<float, LARGE_PACKS>() - 1) / chunk_of<float, LARGE_PACKS>();
    }
  if (units <= UNITS * SMALL_WAVES && ntensors <= SMALL_SPANS) return 0;      // one block, whatever the types
  const int64_t chunks = total * 2 < SMALL_BYTES ? small : large;       // 2 bytes an element at least
  return MAX_BLOCKS * sizeof(double) + (entries_of(numel, ntensors) > TABLE ? (size_t)chunks * sizeof(Chunk) : 0);
}

namespace {
struct Span { uint64_t lo, hi, size; };

// spans laid out in tables, and the launches
template <int P>
int run(const std::vector<Span>& spans, int norm_type, float max_norm, int clip, float* out, double* part, hipStream_t s) {
  std::vector<Table<P>> tables(1);
  tables[0].count = tables[0].chunks = 0;
  int64_t chunks = 0;
  for (const Span& p : spans) {
    const int64_t total = (int64_t)((p.hi - p.lo) / p.size);
    for (int64_t at = 0; at < total; at += PIECE) {
      if (tables.back().count == TABLE) {
        tables.emplace_back();
        tables.back().count = tables.back().chunks = 0;
      }
      Table<P>& t = tables.back();
      const int64_t n = std::min(PIECE, total - at);
      t.e[t.count++] = {(p.lo + p.size * (uint64_t)at) | ((uint64_t)(p.size == 2) << 63), (uint32_t)n, (uint32_t)t.chunks};
      const int more = (int)((n * (int64_t)p.size + chunk_bytes(P) - 1) / chunk_bytes(P));
      t.chunks += more;
      chunks += more;
    }
  }
  if (tables.size() == 1) return launch(tables[0], norm_type, max_norm, clip, out, part, s);
  if (chunks > 0x7fffffff) return LDM_ERR_ARG;
  Chunk* list = reinterpret_cast<Chunk*>(part + MAX_BLOCKS);
  chunks = 0;
  for (const Table<P>& t : tables) {
    hipLaunchKernelGGL((list_chunks<P>), dim3(t.count), dim3(64), 0, s, t, list + chunks);
    LDM_CHECK_LAUNCH();
    chunks += t.chunks;
  }
  return launch(ChunkList<P>{list, (int)chunks}, norm_type, max_norm, clip, out, part, s);
}
}  // namespace

extern "C" int ldm_grad_norm(const void* const* ptrs, const int64_t* numel, const uint8_t* dtypes, int ntensors,
                             int norm_type, double max_norm, int clip, float* out, void* workspace,
                             int64_t workspace_bytes, ldm_stream_t stream) {
  if (!ptrs || !numel || !dtypes || !out || ntensors <= 0 || clip < 0 || clip > 2) return LDM_ERR_ARG;
  if (norm_type < LDM_NORM_2 || norm_type > LDM_NORM_1 || !(max_norm >= 0.0)) return LDM_ERR_ARG;
  const int64_t need = (int64_t)ldm_grad_norm_workspace_bytes(numel, ntensors);
  if (need && (!workspace || workspace_bytes < need)) return LDM_ERR_ARG;
  // Tensors in the order of their addresses; those that lie back to back (views of a bucket) are one span.
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  double* part = static_cast<double*>(workspace);
  try {
    std::vector<Span> spans;
    spans.reserve(ntensors);
    int64_t total = 0;
    for (int i = 0; i < ntensors; ++i) {
      if (numel[i] < 0 || dtypes[i] > LDM_BF16) return LDM_ERR_ARG;
      if (numel[i] == 0) continue;
      const uint64_t a = reinterpret_cast<uint64_t>(ptrs[i]);
      const uint64_t size = dtypes[i] == LDM_BF16 ? 2 : 4;
      if (numel[i] > MOST_VALUES - total) return LDM_ERR_ARG;
      total += numel[i];
      if (!a || (a >> 63) || ((a + size * (uint64_t)numel[i]) >> 63)) return LDM_ERR_ARG;
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
    int64_t units = 0, bytes = 0;
    for (const Span& p : spans) {
      bytes += (int64_t)(p.hi - p.lo);
      units += (int64_t)(p.hi - p.lo + 1023) / 1024;
    }
    if (clip != 2 && units <= UNITS * SMALL_WAVES && spans.size() <= SMALL_SPANS) {
      SmallTable t;
      t.units = 0;
      for (size_t i = 0; i < spans.size(); ++i) {
        const Span& p = spans[i];
        t.e[i] = {p.lo | ((uint64_t)(p.size == 2) << 63), (uint32_t)((p.hi - p.lo) / p.size), (uint32_t)t.units};
        for (int64_t k = (int64_t)(p.hi - p.lo + 1023) / 1024; k > 0; --k) t.span[t.units++] = (uint8_t)i;
      }
      return launch_small(t, norm_type, (float)max_norm, clip, out, s);
    }
    return bytes < SMALL_BYTES ? run<SMALL_PACKS>(spans, norm_type, (float)max_norm, clip, out, part, s)
                               : run<LARGE_PACKS>(spans, norm_type, (float)max_norm, clip, out, part, s);
  } catch (...) {                  // no exception leaves a C entry; std::bad_alloc is the only one
    return LDM_ERR_ARG;
  }
}
