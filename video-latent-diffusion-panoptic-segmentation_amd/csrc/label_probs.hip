// Log probability of a given label, entropy and the most likely classes of every position, and the
// gradient of the first two (ldm_label_log_probs / ldm_label_log_probs_bwd).
//
// One pass over the logits x_j of a position with the running maximum and sums of its softmax,
// z_j = x_j / T, m = max x_j:
//   r = sum_{j != argmax} exp((x_j - m) / T)             (the maximum's own 1 stays out)
//   t = sum_{j != argmax} (x_j - m) exp((x_j - m) / T)
//   log_prob(y) = (x_y - m) / T - log1p(r)               entropy = log1p(r) - (t / T) / (1 + r)
// Both terms of the entropy have one sign and log1p keeps a confident row's digits: nothing
// cancels where 1 - p is small.  Backward, from the saved m, log1p(r) and entropy:
//   p_j = exp((x_j - m) / T - log1p(r))
//   d x_j = (g_l (1[j == y] - p_j) - g_H p_j (log p_j + H)) / T
// Sums are fp32 over at most 512 logits of a thread and fp64 beyond; the logits are exact in fp32 and d x_j is rounded
// once to their type.
// The logits are read once each way and the gradient written once: memory bounds the fp32 kernels (copies reach 5.3
// TB/s here), the vector pipe the bf16 ones, whose 13 instructions and one exp a class take about as long as 2 bytes.
// exp is the hardware's exp2 of a product: x - m, log2(e) / T, their product and exp2 round, so a term e^z carries a
// relative error of at most (4 |z| + 5) 2^-24, which is no more than 5 x 2^-24 of the largest term.
#include "common.h"

#include <algorithm>
#include <math.h>
#include <type_traits>

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float LOWEST = -3e38f;   // finite stand-in for x_j - m = -inf: 0 * LOWEST is 0, 0 * inf is NaN

struct Args {
  const void* x;
  int64_t n1, n2, s0, s1, s2, sc, positions;       // n1 = 0: all positions are in the last dim
  int classes;
  const int64_t* labels;
  int64_t ignore;
  int has_ignore;
  const uint8_t* mask;
  int64_t mask_stride, mask_div, inner;
  float c2, inv_t, slack;          // log2(e) / T, 1 / T, T ln 2
  float *lp, *ent, *top_lp, *stats;
  int32_t* top_id;
  int k;
};

// a / b, a < all: in 32 bits where all and b fit, which every thread of a launch decides alike
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b, int64_t all) {
  if ((uint64_t)(all | b) >> 32 == 0) return (int64_t)((uint32_t)a / (uint32_t)b);
  return a / b;
}
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// order-preserving float -> int32 with NaN above everything and -0 equal to +0
__device__ __forceinline__ int order_key(float x) {
  const int b = __float_as_int(x + 0.f);
  return x != x ? 0x7fffffff : b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float key_value(int k) {
  return k == 0x7fffffff ? __int_as_float(0x7fc00000) : __int_as_float(k ^ ((k >> 31) & 0x7fffffff));
}
constexpr int KEY_NONE = (int)0x807fffff;   // order_key(-inf): a class without probability is no candidate

// v_max / v_min as they are: fmaxf of a loaded value costs one more to quieten signalling NaNs, and a row with any
// NaN is known by other means
__device__ __forceinline__ float raw_max(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ float raw_min(float a, float b) {
  float r;
  asm("v_min_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}

// maximum and sums of one set of logits; the maximum's own term is in neither sum
struct Soft {
  float m, r, t;
  __device__ __forceinline__ void clear() { m = -INFINITY; r = t = 0.f; }
  __device__ __forceinline__ void rescale(float to, float c2) {   // sums relative to `to` > -inf
    const float d = fmaxf(m - to, LOWEST), s = exp2_fast(d * c2);
    t = s * t + (s * d) * r;
    r *= s;
  }
  __device__ __forceinline__ void join(const Soft& o, float c2) { // o's classes and these
    const float hi = fmaxf(m, o.m), lo = fminf(m, o.m), to = hi == -INFINITY ? 0.f : hi;
    Soft b = o;
    rescale(to, c2);
    b.rescale(to, c2);
    const float d = fmaxf(lo - to, LOWEST), e = exp2_fast(d * c2);
    r += b.r + e;
    t += b.t + d * e;
    m = hi;
  }
};

// The same of a thread's logits while it walks them.  Their number does not show in the sums' rounding: a chunk's
// terms are added up by themselves, FOLD chunks in fp32 and those in fp64 (131072 strided logits of one value but the
// maximum in one accumulator: 5e-4 off).  R and T are relative to `ref`, a former maximum that is replaced where the
// maximum has passed it by a factor of two: what came before then loses half its weight, and with it the rounding of
// its product with e^(ref - m), however often a slowly rising row does this.  Threads of no more than FOLD chunks have
// FOLDS false: 1 x 19 x 512 x 1024 fp32 12.9 us, 13.7 us with the folds' code and registers beside the loop.
constexpr int FOLD = 32;
template <bool FOLDS> struct Run {
  float m, r, t, ref;
  double R, T;
  int chunks;
  __device__ __forceinline__ void clear() { m = ref = -INFINITY; r = t = 0.f; R = T = 0.0; chunks = 0; }
  // N logits, no NaN heeded: one move of the maximum.  It is carried through them: what each passes on is the lesser
  // of the two, so the set {m, f} becomes {new m} and the f that are left to sum.
  template <int N> __device__ __forceinline__ void add_all(float (&f)[N], float c2, float slack) {
    float hi = m;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const float v = f[u];
      f[u] = raw_min(hi, v);
      hi = raw_max(hi, v);
    }
    const float to = hi == -INFINITY ? 0.f : hi, dm = fmaxf(m - to, LOWEST), s = exp2_fast(dm * c2);
    float rr, tt;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const float d = fmaxf(f[u] - to, LOWEST), e = exp2_fast(d * c2);
      rr = u ? rr + e : e;
      tt = u ? fmaf(d, e, tt) : d * e;
    }
    t = fmaf(s, t, fmaf(s * dm, r, tt));
    r = fmaf(s, r, rr);
    m = hi;
    if constexpr (FOLDS)
      if (++chunks % FOLD == 0) fold(c2, slack);
  }
  __device__ __forceinline__ void fold(float c2, float slack) {
    if (m == -INFINITY) return;                   // nothing so far
    if (ref == -INFINITY || m > ref + slack) {
      const float d = fmaxf(ref - m, LOWEST);
      const double s = exp2_fast(d * c2);
      T = s * (T + d * R);
      R *= s;
      ref = m;
    }
    const float d = m - ref;
    const double s = exp2_fast(d * c2);
    R += s * r;
    T += s * ((double)t + (double)d * r);
    r = t = 0.f;
  }
  __device__ __forceinline__ Soft sums(float c2, float slack) {
    if (!FOLDS || chunks < FOLD || m == -INFINITY) return {m, r, t};
    fold(c2, slack);
    Soft s = {ref, (float)R, (float)T};
    s.rescale(m, c2);
    s.m = m;
    return s;
  }
};

// the K largest (key, class), larger key first; a later class needs a larger key
template <int K>
struct Top {
  int key[K > 0 ? K : 1], id[K > 0 ? K : 1];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < K; ++i) { key[i] = KEY_NONE; id[i] = -1; }
  }
  __device__ __forceinline__ void add(int k, int c) {
    if constexpr (K > 0) {
      if (k > key[K - 1]) {
#pragma unroll
        for (int i = K - 1; i > 0; --i) {
          const bool up = k > key[i - 1], here = k > key[i];
          id[i] = up ? id[i - 1] : here ? c : id[i];
          key[i] = up ? key[i - 1] : here ? k : key[i];
        }
        if (k > key[0]) { key[0] = k; id[0] = c; }
      }
    }
  }
};

// log(1 + r), r >= 0, to a few roundings of itself: what 1 + r loses, r / ((1 + r) - 1) gives back (Goldberg 1991)
__device__ __forceinline__ float log1p_of(float r) {
  const float w = 1.f + r, l = LN2 * __builtin_amdgcn_logf(w);
  return w == 1.f ? r : l * (r * __builtin_amdgcn_rcpf(w - 1.f));
}

// In the saved label: its logit is the row's maximum.  Classes are numbered below it.
constexpr int MOST_CLASSES = 1 << 30, LABEL_LEADS = 1 << 30;

// what a position's sums come to
struct Result { float ls, ent, lp; int label; };
__device__ __forceinline__ Result result_of(const Args& a, const Soft& s, bool nan, int64_t y, float xy) {
  Result q;
  const float none = __int_as_float(0x7fc00000);
  const bool empty = s.m == -INFINITY, bad = nan || s.m == INFINITY;
  q.ls = bad ? none : log1p_of(s.r);
  q.ent = bad ? none : empty ? 0.f : q.ls - s.t * a.inv_t * __builtin_amdgcn_rcpf(1.f + s.r);
  const bool known = !(a.has_ignore && y == a.ignore), inside = y >= 0 && y < a.classes;
  if (!known) q.lp = 0.f;
  else if (!inside || bad) q.lp = none;
  else q.lp = xy == -INFINITY ? -INFINITY : (xy - s.m) * a.inv_t - q.ls;
  q.label = !(known && inside && q.lp > -INFINITY) ? -1          // NaN > -inf is false: the row is NaN anyway
            : xy == s.m ? (int)y | LABEL_LEADS : (int)y;
  return q;
}
__device__ __forceinline__ void store_top(const Args& a, int64_t pos, int j, int key, int id, const Soft& s, float ls) {
  const int64_t o = a.inner == 1 ? pos : quotient(pos, a.inner, a.positions), at = (o * a.k + j) * a.inner + (pos - o * a.inner);
  a.top_id[at] = id;
  a.top_lp[at] = id < 0 ? -INFINITY : (key_value(key) - s.m) * a.inv_t - ls;
}

// a position's three indices
struct Place {
  int64_t i0, i1, i2;
  __device__ __forceinline__ int64_t at(int64_t s0, int64_t s1, int64_t s2) const { return i0 * s0 + i1 * s1 + i2 * s2; }
};
__device__ __forceinline__ Place place_of(int64_t pos, int64_t all, int64_t n1, int64_t n2) {
  if (n1 == 0) return {0, 0, pos};                 // all positions in one dim
  const int64_t line = quotient(pos, n2, all), i0 = n1 == 1 ? line : quotient(line, n1, all);
  return {i0, line - i0 * n1, pos - line * n2};
}

// Reductions by DPP, in the vector pipe; a shuffle is a trip through LDS.
// Over G = 1 .. 64 neighbouring lanes, in each of them: quads, then mirrored halves of 8 and 16, then rows of 16.
template <int CTRL, typename V> __device__ __forceinline__ V dpp(V v) {
  return __builtin_bit_cast(V, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int G, typename V, typename F> __device__ __forceinline__ V lanes_join(V v, F f) {
  if constexpr (G >= 2) v = f(v, dpp<0xB1>(v));      // quad_perm 1 0 3 2
  if constexpr (G >= 4) v = f(v, dpp<0x4E>(v));      // quad_perm 2 3 0 1
  if constexpr (G >= 8) v = f(v, dpp<0x141>(v));     // row_half_mirror
  if constexpr (G >= 16) v = f(v, dpp<0x140>(v));    // row_mirror
  if constexpr (G >= 32) v = f(v, __shfl_xor(v, 16, 64));
  if constexpr (G >= 64) v = f(v, __shfl_xor(v, 32, 64));
  return v;
}
// Over the wave, as a scalar: rows of 16 as above, then the row totals to the last lane.  `none` changes nothing.
template <typename V, typename F> __device__ __forceinline__ V wave_all(V v, V none, F f) {
  v = lanes_join<16>(v, f);
  const int n = __builtin_bit_cast(int, none);
  v = f(v, __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(n, __builtin_bit_cast(int, v), 0x142, 0xa, 0xf, false)));
  v = f(v, __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(n, __builtin_bit_cast(int, v), 0x143, 0xc, 0xf, false)));
  return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
struct Add { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };
struct Max {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
  __device__ __forceinline__ int operator()(int a, int b) const { return max(a, b); }
};
struct Min { __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const { return min(a, b); } };

// the wave's Softs joined, in every lane
__device__ __forceinline__ Soft wave_join(const Soft& s, float c2) {
  const float m = wave_all(s.m, -INFINITY, Max()), to = m == -INFINITY ? 0.f : m;
  const bool holds = s.m == m;     // the first lane that holds the maximum keeps its term out of the sums
  const bool keeper = holds && (int)(threadIdx.x & 63) == __ffsll((unsigned long long)__ballot(holds)) - 1;
  Soft o = s;
  o.rescale(to, c2);
  const float d = fmaxf(s.m - to, LOWEST), e = keeper ? 0.f : exp2_fast(d * c2);
  o.m = m;
  o.r = wave_all(o.r + e, 0.f, Add());
  o.t = wave_all(fmaf(d, e, o.t), 0.f, Add());
  return o;
}

// N adjacent elements at any address aligned to one element: one wide load or store (the card takes unaligned ones)
template <typename T, int N> struct Pack { T v[N]; };
template <typename T, int N> __device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
  Pack<T, N> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
template <typename T, int N> __device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& r) {
  __builtin_memcpy(p, &r, sizeof(r));
}

template <int VEC, typename T> __device__ __forceinline__ void store_own(T* p, const Pack<T, VEC>& r, int skip) {
  if (VEC == 1 || skip == 0) {
    store_pack<T, VEC>(p, r);
  } else {
#pragma unroll
    for (int j = 1; j < VEC; ++j)
      if (j >= skip) p[j] = r.v[j];
  }
}

__device__ __forceinline__ void store_row(const Args& a, int64_t pos, const Soft& s, const Result& q) {
  a.ent[pos] = q.ent;
  if (a.labels) a.lp[pos] = q.lp;
  if (a.stats) {
    a.stats[pos] = s.m;
    a.stats[a.positions + pos] = q.ls;
    a.stats[2 * a.positions + pos] = q.ent;
    a.stats[3 * a.positions + pos] = __int_as_float(a.labels ? q.label : -1);
  }
}

// Short rows of adjacent classes: G lanes to a row, E packs of VEC classes to a lane (16 classes), all of it in
// registers.  A row's last pack reaches back over its neighbour; the classes it has in common with it count once.
// 32768 x 30 bf16 with 3 alternatives: 5.2 us, the latency of one launch, load, reduction and store.
template <typename T, int VEC, int G, int E, bool TOP>
__global__ __launch_bounds__(256) void probs_short_rows(const Args a) {
  constexpr int N = VEC * E;
  const int lane = threadIdx.x & 63, sub = lane & (G - 1);
  const int64_t want = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  const bool live = want < a.positions;
  const int64_t pos = live ? want : a.positions - 1;
  const T* x = (const T*)a.x + place_of(pos, a.positions, a.n1, a.n2).at(a.s0, a.s1, a.s2);
  const uint8_t* mask = a.mask ? a.mask + quotient(pos, a.mask_div, a.positions) * a.mask_stride : nullptr;
  Pack<T, VEC> v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = load_pack<T, VEC>(x + min((sub + e * G) * VEC, a.classes - VEC));
  const int64_t y = a.labels ? a.labels[pos] : -1;
  float xy = -INFINITY;
  if (y >= 0 && y < a.classes && !(mask && !mask[y])) xy = to_f(x[y]);
  float f[N];
  int key[TOP ? N : 1];
  bool nan = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int at = (sub + e * G) * VEC, c0 = min(at, a.classes - VEC);
    Pack<uint8_t, VEC> m;
    if (mask) m = load_pack<uint8_t, VEC>(mask + c0);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int i = e * VEC + j;
      const bool in = c0 + j >= at && (!mask || m.v[j]);
      f[i] = in ? to_f(v[e].v[j]) : -INFINITY;
      nan |= f[i] != f[i];
      if constexpr (TOP) key[i] = order_key(f[i]);
    }
  }
  // the lane's maximum is carried out of f; the row's first lane that holds the row's keeps it out of the sums
  float hi = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float w = f[i];
    f[i] = fminf(hi, w);
    hi = fmaxf(hi, w);
  }
  Soft s;
  s.m = lanes_join<G>(hi, Max());
  const float to = s.m == -INFINITY ? 0.f : s.m;
  const uint64_t mine = (G == 64 ? ~0ull : ((1ull << (G & 63)) - 1)) << (lane & ~(G - 1));
  const uint64_t holds = __ballot(hi == s.m) & mine;
  const bool keeper = lane == __ffsll((unsigned long long)holds) - 1;
  nan = (__ballot(nan) & mine) != 0;
  const float dh = fmaxf(hi - to, LOWEST), eh = keeper ? 0.f : exp2_fast(dh * a.c2);
  float r = eh, t = dh * eh;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = fmaxf(f[i] - to, LOWEST), e = exp2_fast(d * a.c2);
    r += e;
    t = fmaf(d, e, t);
  }
  s.r = lanes_join<G>(r, Add());
  s.t = lanes_join<G>(t, Add());
  const Result q = result_of(a, s, nan, y, xy);
  if (live && sub == 0) store_row(a, pos, s, q);
  if constexpr (TOP) {
    for (int n = 0; n < a.k; ++n) {
      int k = KEY_NONE, c = -1;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int ci = min((sub + i / VEC * G) * VEC, a.classes - VEC) + i % VEC;
        if (key[i] > k) { k = key[i]; c = ci; }
      }
      const int best = lanes_join<G>(k, Max());
      c = (int)lanes_join<G>(k == best ? (unsigned)c : ~0u, Min());
      k = best;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int ci = min((sub + i / VEC * G) * VEC, a.classes - VEC) + i % VEC;
        if (ci == c) key[i] = KEY_NONE;
      }
      if (live && sub == (n & (G - 1))) store_top(a, pos, n, k, c, s, q.ls);
    }
  }
}

// Long rows of adjacent classes: a block has one segment of one row, its threads packs of VEC classes, UNR of them
// in flight.  One segment to a row: the block finishes it.  More: what the segments come to goes to the workspace
// and probs_join finishes the row.  4096 x 16384 fp32: 57 us (4.7 TB/s), bf16 31 us back to back (4.3 TB/s, the vector pipe), 38
// one at a time; four packs in flight: 55 and 31, but rows of 4096 took 68 us for 44.  One row of 65537 fp32: 6 us in 65 segments, with 8
// alternatives 12 us, 7 in the first launch and 5 in the second.
struct Part { float m, r, t; int nan; };
// (key, class) as one number: larger is earlier in the answer (larger key, then lower class), 0 is none
__device__ __forceinline__ uint64_t candidate(int key, int id) {
  return id < 0 ? 0 : (uint64_t)(uint32_t)(key ^ (int)0x80000000) << 32 | (uint32_t)~id;
}
__device__ __forceinline__ void wave_lds_fence() {   // a wave's LDS accesses stay in order: only the compiler is held
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
// The first n <= 16 of the values that the wave's leading `lanes` lanes hold (0: none), in their order, in every lane
// j < n: each value finds its place by counting those before it.
__device__ __forceinline__ uint64_t first_of(uint64_t mine, int lanes, int n, uint64_t* sorted) {
  const int lane = threadIdx.x & 63;
  int place = 0;
  for (int j = 0; j < lanes; ++j) {
    const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), j) << 32 |
                           (uint32_t)__builtin_amdgcn_readlane((int)mine, j);
    place += other > mine;
  }
  if (lane < 16) sorted[lane] = 0;
  wave_lds_fence();
  if (mine && place < n) sorted[place] = mine;
  wave_lds_fence();
  const uint64_t r = lane < n ? sorted[lane] : 0;
  wave_lds_fence();
  return r;
}
// What a wave keeps for the answer of its row: candidates in any order, among them the first n of all it was given.
struct Best {
  uint64_t some[64], sorted[16];
};
__device__ __forceinline__ void absorb(Best& b, int& count, uint64_t mine, int n) {   // a candidate (or 0) a lane
  const int lane = threadIdx.x & 63;
  uint64_t who = __ballot(mine != 0);
  if (count + __popcll(who) > 64) {
    const uint64_t r = first_of(lane < count ? b.some[lane] : 0, count, n, b.sorted);
    if (lane < n) b.some[lane] = r;
    count = __popcll(__ballot(r != 0));
    if (count + __popcll(who) > 64) {
      mine = first_of(mine, 64, n, b.sorted);
      who = __ballot(mine != 0);
    }
  }
  if (mine) b.some[count + __popcll(who & ((1ull << lane) - 1))] = mine;
  count += __popcll(who);
  wave_lds_fence();
}
// the n-th largest of the wave's lane values, or one that is not above `floor`
__device__ __forceinline__ int nth_largest(int mine, int n, int floor) {
  int nth = KEY_NONE;
  for (int j = 0; j < n; ++j) {
    nth = wave_all(mine, KEY_NONE, Max());
    if (nth <= floor) break;
    if ((int)(threadIdx.x & 63) == __ffsll((unsigned long long)__ballot(mine == nth)) - 1) mine = KEY_NONE;
  }
  return nth;
}

template <bool TOP, int WAVES>
struct RowParts {
  Soft part[WAVES];
  int nan[WAVES], count[WAVES];
  Best best[TOP ? WAVES : 1];
};
// the block's threads' sums and candidates joined, in wave 0 (lane j < n: the j-th of the answer); other waves get
// nothing
template <bool TOP>
__device__ __forceinline__ bool block_join_row(RowParts<TOP, 4>& sh, Soft& s, int count, bool& nan, int n, float c2,
                                               uint64_t& answer) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  s = wave_join(s, c2);
  if constexpr (TOP) {
    Best& b = sh.best[wave];
    if (count > 16) {
      const uint64_t r = first_of(lane < count ? b.some[lane] : 0, count, n, b.sorted);
      if (lane < n) b.some[lane] = r;
      count = n;
    }
    if (lane == 0) sh.count[wave] = count;
  }
  const bool any = __ballot(nan) != 0;
  if (lane == 0) { sh.part[wave] = s; sh.nan[wave] = any; }
  __syncthreads();
  if (wave) return false;
  s = sh.part[0];
  for (int w = 1; w < 4; ++w) s.join(sh.part[w], c2);
  nan = sh.nan[0] | sh.nan[1] | sh.nan[2] | sh.nan[3];
  if constexpr (TOP) {
    // the waves' candidates side by side: at most 16 of each
    const int n0 = sh.count[0], n1 = n0 + sh.count[1], n2 = n1 + sh.count[2], all = n2 + sh.count[3];
    const int w = lane < n0 ? 0 : lane < n1 ? 1 : lane < n2 ? 2 : 3, at = lane - (w == 0 ? 0 : w == 1 ? n0 : w == 2 ? n1 : n2);
    answer = first_of(lane < all ? sh.best[w].some[at] : 0, __builtin_amdgcn_readfirstlane(all), n, sh.best[0].sorted);
  }
  return true;
}
// a row's label and its logit (-inf where it is no class or is masked): fetched first, needed last
struct LabelAt { int64_t y; float xy; };
template <typename T>
__device__ __forceinline__ LabelAt label_at(const Args& a, int64_t pos) {
  LabelAt r = {-1, -INFINITY};
  if (!a.labels) return r;
  r.y = a.labels[pos];
  if (r.y >= 0 && r.y < a.classes && !(a.mask && !a.mask[quotient(pos, a.mask_div, a.positions) * a.mask_stride + r.y]))
    r.xy = to_f(((const T*)a.x + place_of(pos, a.positions, a.n1, a.n2).at(a.s0, a.s1, a.s2))[r.y]);
  return r;
}
__device__ __forceinline__ void finish_row(const Args& a, int64_t pos, const LabelAt& l, const Soft& s, bool nan,
                                           uint64_t answer) {
  const int lane = threadIdx.x & 63;
  const Result q = result_of(a, s, nan, l.y, l.xy);
  if (lane == 0) store_row(a, pos, s, q);
  if (lane < a.k)
    store_top(a, pos, lane, (int)(answer >> 32) ^ (int)0x80000000, answer ? (int)~(uint32_t)answer : -1, s, q.ls);
}

// A turn's classes become candidates only above a bar: the n-th largest of the wave's lane maxima, or what an earlier
// turn had; n classes at least are no less, and later ones lose ties.  So little but the answer is looked at twice.
template <int N, typename C>
__device__ __forceinline__ void enter_above_bar(Best& b, int& count, int& bar, int n, const float (&f)[N], bool odd,
                                                C class_of) {
  if (bar == 0x7fffffff) return;
  float most = f[0];
#pragma unroll
  for (int i = 1; i < N; ++i) most = fmaxf(most, f[i]);
  const int mine = odd ? 0x7fffffff : order_key(most);
  const uint64_t over = __ballot(mine > bar);
  if (!over) return;
  const int nth = __popcll(over) < n ? bar : nth_largest(mine, n, bar);
  const float least = key_value(max(nth, bar + 1));
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const bool in = !(f[i] < least);               // a NaN is
    if (__any(in)) absorb(b, count, in ? candidate(order_key(f[i]), class_of(i)) : 0, n);
  }
  bar = max(bar, nth);
}

// WAVES = 1: a wave to a row, four rows to a block, for rows that a block's start and end would outweigh (30000 x
// 2000 bf16: 35 us, 77 us with a block to a row; 16384 x 4096: 32 and 40; 3000 x 8000: 15.1 and 17.1).
template <typename T, int VEC, bool TOP, int WAVES>
__global__ __launch_bounds__(256) void probs_rows(const Args a, int segments, int seg_len, Part* __restrict__ parts,
                                                  uint64_t* __restrict__ part_top) {
  constexpr int UNR = 2, N = VEC * UNR, W = 64 * WAVES;
  __shared__ RowParts<TOP, WAVES> sh[4 / WAVES];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);     // a scalar, and so is the row's address
  const int64_t pos = WAVES == 1 ? (int64_t)blockIdx.x * 4 + wave
                                 : segments == 1 ? blockIdx.x : blockIdx.x / segments;
  if (WAVES == 1 && pos >= a.positions) return;
  const int seg = segments == 1 ? 0 : (int)(blockIdx.x - pos * segments);
  const int tid = threadIdx.x & (W - 1), lane = tid & 63;
  const T* x = (const T*)a.x + place_of(pos, a.positions, a.n1, a.n2).at(a.s0, a.s1, a.s2);
  const uint8_t* mask = a.mask ? a.mask + quotient(pos, a.mask_div, a.positions) * a.mask_stride : nullptr;
  const int end = min(a.classes, (seg + 1) * seg_len), last = a.classes - VEC;
  RowParts<TOP, WAVES>& mine = sh[WAVES == 1 ? wave : 0];
  Best& best = mine.best[TOP && WAVES == 4 ? wave : 0];
  int count = 0;                   // the wave's candidates
  Run<(WAVES > 1)> run;             // a wave's row has 16 chunks at most (WAVE_CLASSES)
  run.clear();
  uint64_t nans = 0;               // lanes that saw one
  LabelAt l;
  if (segments == 1) l = label_at<T>(a, pos);
  int bar = KEY_NONE;              // a.k of them are no less
  auto turn = [&](int at0, float (&f)[N]) {
    uint64_t odd = 0;
#pragma unroll
    for (int i = 0; i < N; i += 2) odd |= __ballot(__builtin_isunordered(f[i], f[i + 1]));
    nans |= odd;
    if constexpr (TOP)
      enter_above_bar<N>(best, count, bar, a.k, f, odd >> lane & 1,
                         [&](int i) { return min(at0 + i / VEC * W * VEC, last) + i % VEC; });
    run.template add_all<N>(f, a.c2, a.slack);
  };
  int base = seg * seg_len;        // the same turns in every lane: they exchange values
  if (!mask)
    for (; base + W * N <= end; base += W * N) {
      Pack<T, VEC> v[UNR];
      float f[N];
#pragma unroll
      for (int u = 0; u < UNR; ++u) v[u] = load_pack<T, VEC>(x + base + (u * W + tid) * VEC);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = to_f(v[i / VEC].v[i % VEC]);
      turn(base + tid * VEC, f);
    }
  for (; base < end; base += W * N) {
    const int at0 = base + tid * VEC;
    Pack<T, VEC> v[UNR];
    float f[N];
#pragma unroll
    for (int u = 0; u < UNR; ++u) v[u] = load_pack<T, VEC>(x + min(at0 + u * W * VEC, last));
#pragma unroll
    for (int u = 0; u < UNR; ++u) {
      const int at = at0 + u * W * VEC, c0 = min(at, last);
      Pack<uint8_t, VEC> m;
      if (mask) m = load_pack<uint8_t, VEC>(mask + c0);
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        // only the row's last segment ends inside a block's reach, and its last pack reaches back over its neighbour
        f[u * VEC + j] = at < end && c0 + j >= at && (!mask || m.v[j]) ? to_f(v[u].v[j]) : -INFINITY;
    }
    turn(at0, f);
  }
  uint64_t answer = 0;
  bool nan = nans != 0;
  Soft s = run.sums(a.c2, a.slack);
  if constexpr (WAVES == 1) {
    s = wave_join(s, a.c2);
    if constexpr (TOP) answer = first_of(lane < count ? best.some[lane] : 0, count, a.k, best.sorted);
    finish_row(a, pos, l, s, nan, answer);
  } else {
    if (!block_join_row<TOP>(mine, s, count, nan, a.k, a.c2, answer)) return;
    if (segments == 1) {
      finish_row(a, pos, l, s, nan, answer);
      return;
    }
    if (lane == 0) parts[blockIdx.x] = {s.m, s.r, s.t, nan};
    if (lane < a.k) part_top[(int64_t)blockIdx.x * a.k + lane] = answer;
  }
}

// One block per row: its segments' sums and answers joined.
template <typename T, bool TOP>
__global__ __launch_bounds__(256) void probs_join(const Args a, int segments, const Part* __restrict__ parts,
                                                  const uint64_t* __restrict__ part_top) {
  __shared__ RowParts<TOP, 4> sh;
  const int64_t pos = blockIdx.x;
  const int lane = threadIdx.x & 63;
  Best& best = sh.best[TOP ? threadIdx.x >> 6 : 0];
  Soft s;
  s.clear();
  bool nan = false;
  int count = 0, bar = KEY_NONE;
  const LabelAt l = label_at<T>(a, pos);
  for (int base = threadIdx.x & ~63; base < segments; base += 256) {   // the same turns in every lane of a wave
    const int i = base + lane;
    Part p = {-INFINITY, 0.f, 0.f, 0};
    uint64_t c[TOP ? 16 : 1];
    if (i < segments) p = parts[pos * segments + i];
    if constexpr (TOP)
#pragma unroll
      for (int j = 0; j < 16; ++j) c[j] = j < a.k && i < segments ? part_top[(pos * segments + i) * a.k + j] : 0;
    Soft o;
    o.m = p.m; o.r = p.r; o.t = p.t;
    s.join(o, a.c2);
    nan |= p.nan != 0;
    if constexpr (TOP) {
      const int first = c[0] ? (int)(c[0] >> 32) ^ (int)0x80000000 : KEY_NONE;
      bar = max(bar, nth_largest(first, a.k, bar));
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const bool in = c[j] && ((int)(c[j] >> 32) ^ (int)0x80000000) >= bar;
        if (!__any(in)) break;                     // each segment's are in falling order
        absorb(best, count, in ? c[j] : 0, a.k);
      }
    }
  }
  uint64_t answer = 0;
  if (block_join_row<TOP>(sh, s, count, nan, a.k, a.c2, answer)) finish_row(a, pos, l, s, nan, answer);
}

// What a thread of probs_planes keeps of the most likely classes of one position: values in falling order.  A new
// value's place is the median of its neighbours (v_med3); a later class needs a larger value.  NaNs are sorted out
// afterwards, from the position's logits: here they compare false.
template <int K>
struct TopValues {
  float v[K > 0 ? K : 1];
  int id[K > 0 ? K : 1];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < K; ++i) { v[i] = -INFINITY; id[i] = -1; }
  }
  __device__ __forceinline__ void add(float f, int c) {
    if constexpr (K > 0) {
      bool over[K];
#pragma unroll
      for (int i = 0; i < K; ++i) over[i] = f > v[i];
#pragma unroll
      for (int i = K - 1; i > 0; --i) {
        v[i] = __builtin_amdgcn_fmed3f(v[i - 1], f, v[i]);
        id[i] = over[i - 1] ? id[i - 1] : over[i] ? c : id[i];
      }
      id[0] = over[0] ? c : id[0];
      v[0] = over[0] ? f : v[0];
    }
  }
};
// The classes that a mask row leaves in, in order, listed by the whole block (8 KB of LDS at most): their number.
constexpr int LIST = 4096;
__device__ __forceinline__ int list_classes(const uint8_t* mask, int classes, uint16_t* list) {
  __shared__ int before_wave[4];
  const int per = (classes + 255) >> 8, c0 = threadIdx.x * per, c1 = min(classes, c0 + per);
  int n = 0;
  for (int c = c0; c < c1; ++c) n += mask[c] != 0;
  int upto = n;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(upto, o, 64);
    if ((int)(threadIdx.x & 63) >= o) upto += v;
  }
  if ((threadIdx.x & 63) == 63) before_wave[threadIdx.x >> 6] = upto;
  __syncthreads();
  int at = upto - n, all = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    at += w < (int)(threadIdx.x >> 6) ? before_wave[w] : 0;
    all += before_wave[w];
  }
  for (int c = c0; c < c1; ++c)
    if (mask[c]) list[at++] = (uint16_t)c;
  __syncthreads();
  return all;
}

// How the positions lie over the blocks: `run` of them to each row of the class mask, in `blocks` blocks of their
// own, so that a block's classes are one list (or one run of all)
struct Tiling { int64_t run; unsigned blocks; };

// Block b of a launch runs on XCD b mod 8, each with an L2 of its own.  The tile it takes instead of the b-th: `near`
// neighbours in a row go to one XCD, so that a line which two of them share, their planes being at any address, is
// fetched once.  1 x 128 x 187 x 613 fp32 split: 17 us with an eighth of the launch in a row, 20 us in launch order;
// not split, 16 in a row: 1 x 64 x 375 x 1242 fp32 29.7 us for 31.2, 1 x 19 x 512 x 1024 15.9 for 17.7, and 1 % more
// for 8 x 128 x 256 x 256, which has no shared lines (10 % more with an eighth of the launch in a row).
__device__ __forceinline__ unsigned tile_of(unsigned b, unsigned all, unsigned near) {
  const unsigned group = 8 * near, first = b / group * group, r = b - first;
  return first + group > all ? b : first + (r & 7) * near + (r >> 3);
}

constexpr int PLANES_UNR = 8;
// Forward over strided classes: a thread has one position and UNR classes of it in registers at a time (their loads
// are in flight together and the maximum's move costs one rescale); a wave reads 64 neighbours of each class plane.
// With SPLIT the block's four waves have the same 64 positions and a quarter of the classes each, joined through
// LDS: few positions still fill the card.  LISTED: only the planes of classes that the mask leaves in are read.
// 8 x 128 x 256 x 256 fp32 frames with 4 alternatives: 55 us (5.2 TB/s); four positions a thread took 70 us, fewer
// waves of which each waits for 256 positions' lists.  Of unrelated neighbours the lists cost 81 us, none 58.
// 16 x 128 x 128 x 128 bf16 with 70 % of the classes left: 17.5 us listed, 35 us with every plane read and tested.
// Unsplit bf16 takes 16 classes at a time: as many bytes in flight as 8 of fp32, and half the rescales (8 x 128 x 256 x
// 256: 36.4 us for 39.4); fp32 gains nothing by it and split calls lose 3 %.  Two positions a
// thread: 42 us.
// 1 x 400 x 40 x 50 fp32: 8.0 us split, 19.1 us not.
template <typename T, int K, bool SPLIT, bool LISTED, bool FOLDS>
__global__ __launch_bounds__(256) void probs_planes(const Args a, const Tiling tile) {
  constexpr int UNR = PLANES_UNR;
  __shared__ uint16_t list[LISTED ? LIST : 1];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const unsigned id = tile_of(blockIdx.x, gridDim.x, SPLIT ? max(1u, gridDim.x / 8) : 16);
  const unsigned row = LISTED ? id / tile.blocks : 0;
  const int64_t block = LISTED ? id - row * tile.blocks : id;
  const int64_t want = SPLIT ? block * 64 + lane : block * 256 + threadIdx.x;
  const bool live = want < tile.run && row * tile.run + want < a.positions;
  int n = a.classes;
  if (LISTED) n = list_classes(a.mask + row * a.mask_stride, a.classes, list);
  if (!SPLIT && !live) return;
  const int64_t pos = live ? row * tile.run + want : a.positions - 1;
  const T* x = (const T*)a.x + place_of(pos, a.positions, a.n1, a.n2).at(a.s0, a.s1, a.s2);
  const uint8_t* mask = a.mask ? a.mask + (LISTED ? row : quotient(pos, a.mask_div, a.positions)) * a.mask_stride : nullptr;
  const int c0 = SPLIT ? (int)((int64_t)n * wave >> 2) : 0;
  const int c1 = SPLIT ? (int)((int64_t)n * (wave + 1) >> 2) : n;
  int64_t y = -1;
  float xy = -INFINITY;
  if (a.labels && (!SPLIT || wave == 0)) {
    y = a.labels[pos];             // its logit is fetched beside the loop, which reads that line as well
    if (y >= 0 && y < a.classes && !(mask && !mask[y])) xy = to_f(x[y * a.sc]);
  }
  Run<FOLDS> run;
  run.clear();
  TopValues<K> top;
  top.clear();
  bool nan = false;
  auto chunk = [&](auto& cls, auto& f) {
    constexpr int N = sizeof(f) / sizeof(float);
#pragma unroll
    for (int u = 0; u < N; ++u) {
      if constexpr (K > 0)
        if (__any(f[u] > top.v[K - 1])) top.add(f[u], cls[u]);
      nan |= f[u] != f[u];
    }
    run.template add_all<N>(f, a.c2, a.slack);
  };
  auto class_at = [&](int i) { return LISTED ? __builtin_amdgcn_readfirstlane((int)list[i]) : i; };
  int c = c0;
  auto whole = [&](auto width) {
    constexpr int N = decltype(width)::value;
    for (; c + N <= c1; c += N) {
      T v[N];
      float f[N];
      int cls[N];
#pragma unroll
      for (int u = 0; u < N; ++u) cls[u] = class_at(c + u);
#pragma unroll
      for (int u = 0; u < N; ++u) v[u] = x[cls[u] * a.sc];
#pragma unroll
      for (int u = 0; u < N; ++u) f[u] = to_f(v[u]);
      chunk(cls, f);
    }
  };
  if (LISTED || !mask) {
    if constexpr (sizeof(T) == 2 && !SPLIT) whole(std::integral_constant<int, 16>());
    whole(std::integral_constant<int, UNR>());
  }
  for (; c < c1; c += UNR) {
    T v[UNR];
    float f[UNR];
    int cls[UNR];
    bool in[UNR];
#pragma unroll
    for (int u = 0; u < UNR; ++u) {
      cls[u] = class_at(min(c + u, c1 - 1));
      v[u] = x[cls[u] * a.sc];
      in[u] = c + u < c1 && (LISTED || !mask || mask[cls[u]]);
    }
#pragma unroll
    for (int u = 0; u < UNR; ++u) f[u] = in[u] ? to_f(v[u]) : -INFINITY;
    chunk(cls, f);
  }
  Soft s = run.sums(a.c2, a.slack);
  if constexpr (SPLIT) {
    __shared__ Soft part[4][64];
    __shared__ bool part_nan[4][64];
    __shared__ TopValues<K> part_top[K > 0 ? 4 : 1][K > 0 ? 64 : 1];
    if (wave) {
      part[wave][lane] = s;
      part_nan[wave][lane] = nan;
      if constexpr (K > 0) part_top[wave][lane] = top;
    }
    __syncthreads();
    if (wave || !live) return;
#pragma unroll 1
    for (int w = 1; w < 4; ++w) {
      s.join(part[w][lane], a.c2);
      nan |= part_nan[w][lane];
      if constexpr (K > 0)
#pragma unroll
        for (int i = 0; i < K; ++i) top.add(part_top[w][lane].v[i], part_top[w][lane].id[i]);
    }
  }
  const Result q = result_of(a, s, nan, y, xy);
  store_row(a, pos, s, q);
  if constexpr (K > 0) {
    const int64_t o = a.inner == 1 ? pos : quotient(pos, a.inner, a.positions), at = o * a.k * a.inner + pos - o * a.inner;
    if (nan) {
      // every value is NaN: the classes that are come first, lower class first, then the others by value
      Top<K> keys;
      keys.clear();
      for (int k = 0; k < a.classes; ++k)
        if (!mask || mask[k]) keys.add(order_key(to_f(x[k * a.sc])), k);
#pragma unroll
      for (int i = 0; i < K; ++i) top.id[i] = keys.id[i];
    }
#pragma unroll
    for (int i = 0; i < K; ++i)
      if (i < a.k) {
        a.top_lp[at + i * a.inner] = top.id[i] < 0 ? -INFINITY : (top.v[i] - s.m) * a.inv_t - q.ls;
        a.top_id[at + i * a.inner] = top.id[i];
      }
  }
}

template <typename T>
struct BwdArgs {
  const T* x;
  T* dx;
  int64_t n1, n2, s0, s1, s2, sc, o0, o1, o2, oc, positions;
  int classes;
  const uint8_t* mask;
  int64_t mask_stride, mask_div;
  float c2, inv_t;
  const float *stats, *gl, *ge;
};

// 1 - e^-x, x >= 0, to a few roundings of itself: the exponential's series where the difference would cancel
// (the first term left out is below 2^-30 of the sum)
__device__ __forceinline__ float one_minus_exp(float x) {
  constexpr float C[] = {1.f / 2, 1.f / 6, 1.f / 24, 1.f / 120, 1.f / 720, 1.f / 5040, 1.f / 40320, 1.f / 362880, 1.f / 3628800};
  float f = C[8];
#pragma unroll
  for (int k = 7; k >= 0; --k) f = fmaf(-x, f, C[k]);
  return x < LN2 ? fmaf(-x * x, f, x) : 1.f - exp2_fast(-x * LOG2E);
}

// d x_j = (1[j == y] g_y - p_j w_j) / T, w_j = g_l + g_H (log p_j + H) = w0 + w1 z2_j.  Of a label at the row's maximum,
// 1 - p_y and log p_y + H follow from the row's own sums, 1 - p_y = 1 - e^-ls without a difference of neighbours: g_y is
// its whole gradient, and its p_y w_y is kept out by an infinite `ls2_y`.  p of any other label is at most 1/2.
struct RowGrad { float m, ls2, ls2_y, w0, w1, g_y; int label; };
template <typename T>
__device__ __forceinline__ RowGrad row_grad(const BwdArgs<T>& a, int64_t pos) {
  RowGrad g;
  g.m = a.stats[pos];
  const float ls = a.stats[a.positions + pos], off = a.stats[2 * a.positions + pos] - ls;    // H - ls
  const int label = __float_as_int(a.stats[3 * a.positions + pos]);
  const bool leads = label >= 0 && (label & LABEL_LEADS);
  float gl = a.gl && label >= 0 ? a.gl[pos] * a.inv_t : 0.f, ge = a.ge ? a.ge[pos] * a.inv_t : 0.f;
  if (g.m == -INFINITY) g.m = gl = ge = 0.f;
  g.label = label < 0 ? -1 : label & ~LABEL_LEADS;
  g.ls2 = ls * LOG2E;
  g.ls2_y = leads ? INFINITY : g.ls2;
  g.w0 = fmaf(ge, off, gl);
  g.w1 = ge * LN2;
  g.g_y = leads ? gl * one_minus_exp(ls) - ge * exp2_fast(-g.ls2) * off : gl;
  return g;
}
template <typename T>
__device__ __forceinline__ float grad_of(const BwdArgs<T>& a, const RowGrad& g, float x, int c) {
  // below 2^-1000 p is 0 and its log stays finite; a row with a NaN or +inf has ls = NaN, and so has every p of it
  const float z2 = fmaxf((x - g.m) * a.c2, -1000.f);
  const bool own = c == g.label;
  const float p = exp2_fast(z2 - (own ? g.ls2_y : g.ls2));
  return (own ? g.g_y : 0.f) - p * fmaf(z2, g.w1, g.w0);
}

// Backward over strided classes: a thread has PV positions (bf16 two side by side, fp32 one) and `span` <= 64 classes, a
// wave reads and writes 64 PV neighbours of each class plane.  UNIFORM: a block's positions share a row of the class mask, whose bits for the
// span every wave gathers once; planes that it leaves out are not read.  8 x 128 x 256 x 256: fp32 100 us (5.4 TB/s),
// bf16 60 us (4.5 TB/s); spans of 8, 113 and 84 us: a position's 16 bytes of sums are read once a span.  Four
// positions a thread: 119 and 74 us; bf16 with one: 64 us, and 16 x 128 x 128 x 128 with 70 % of the classes 37 us for
// 30, but 16 x 4 x 512 x 512 38 us for 42.  Planes that do not begin on a line of 128 bytes are walked by tile_of (1 x 64 x
// 375 x 1242: fp32 55 us for 60, bf16 34 for 37; the aligned calls above would take 2 % more).
template <typename T, bool UNIFORM, int PV>
__global__ __launch_bounds__(256) void probs_bwd_planes(const BwdArgs<T> a, const Tiling tile, int span) {
  constexpr int UNR = 8;
  const bool apart = ((uint64_t)a.x | (uint64_t)a.sc * sizeof(T)) % 128 == 0;
  const unsigned id = apart ? blockIdx.x : tile_of(blockIdx.x, gridDim.x, 16);
  const unsigned row = UNIFORM ? id / tile.blocks : 0;
  const int64_t want = ((int64_t)(UNIFORM ? id - row * tile.blocks : id) * 256 + threadIdx.x) * PV;
  const int c0 = blockIdx.y * span, c1 = min(a.classes, c0 + span);
  uint64_t bits = ~0ull;
  if (UNIFORM) {
    const int c = c0 + (int)(threadIdx.x & 63);
    bits = __ballot(c < c1 && a.mask[row * a.mask_stride + c]);
  }
  const int64_t pos = row * tile.run + want;
  if (want >= tile.run || pos >= a.positions) return;
  const Place place = place_of(pos, a.positions, a.n1, a.n2);
  const T* x = a.x + place.at(a.s0, a.s1, a.s2);
  T* dx = a.dx + place.at(a.o0, a.o1, a.o2);
  const uint8_t* mask = !UNIFORM && a.mask ? a.mask + quotient(pos, a.mask_div, a.positions) * a.mask_stride : nullptr;
  Pack<T, PV> v[UNR];
  auto load = [&](int c) {
#pragma unroll
    for (int u = 0; u < UNR; ++u) {
      const int cu = min(c + u, c1 - 1);
      if (!UNIFORM || bits >> (cu - c0) & 1) v[u] = load_pack<T, PV>(x + cu * a.sc);
    }
  };
  load(c0);                        // under way before what the position's sums need
  RowGrad g[PV];
#pragma unroll
  for (int i = 0; i < PV; ++i) g[i] = row_grad(a, pos + i);
  for (int c = c0; c < c1; c += UNR) {
    if (c > c0) load(c);
#pragma unroll
    for (int u = 0; u < UNR; ++u) {
      const int cu = c + u;
      if (cu >= c1) break;
      const bool in = UNIFORM ? bits >> (cu - c0) & 1 : !mask || mask[cu];
      Pack<T, PV> d;
#pragma unroll
      for (int i = 0; i < PV; ++i) d.v[i] = from_f<T>(in ? grad_of(a, g[i], to_f(v[u].v[i]), cu) : 0.f);
      store_pack<T, PV>(dx + cu * a.oc, d);
    }
  }
}

// Backward over adjacent classes: a thread has UN packs of VEC classes of one row; a row's last pack reaches back
// over its neighbour and only its own classes are written.  FLAT: packs of short rows side by side in a block.
// 4096 x 16384 bf16: 44 us (6.1 TB/s: the forward has left part of the logits in the memory-side cache).
template <typename T, int VEC, int UN, bool FLAT>
__global__ __launch_bounds__(256) void probs_bwd_rows(const BwdArgs<T> a, unsigned per_row, unsigned blocks_per_row) {
  int64_t pos;
  unsigned first;
  if (FLAT) {
    const uint64_t q = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    pos = q >> 32 ? (int64_t)(q / per_row) : (int64_t)((uint32_t)q / per_row);
    first = (unsigned)(q - (uint64_t)pos * per_row);
    if (pos >= a.positions) return;
  } else {
    pos = blockIdx.x / blocks_per_row;
    first = (blockIdx.x - (unsigned)pos * blocks_per_row) * (256 * UN) + threadIdx.x;
  }
  const Place place = place_of(pos, a.positions, a.n1, a.n2);
  const T* x = a.x + place.at(a.s0, a.s1, a.s2);
  T* dx = a.dx + place.at(a.o0, a.o1, a.o2);
  const uint8_t* mask = a.mask ? a.mask + quotient(pos, a.mask_div, a.positions) * a.mask_stride : nullptr;
  Pack<T, VEC> v[UN];
#pragma unroll
  for (int u = 0; u < UN; ++u) {
    const unsigned q = min(first + u * 256, per_row - 1);
    v[u] = load_pack<T, VEC>(x + min((int)q * VEC, a.classes - VEC));
  }
  const RowGrad g = row_grad(a, pos);
#pragma unroll
  for (int u = 0; u < UN; ++u) {
    const unsigned q = first + u * 256;
    if (!FLAT && q >= per_row) break;
    const int at = (int)q * VEC, c0 = min(at, a.classes - VEC);
    Pack<T, VEC> d;
#pragma unroll
    for (int j = 0; j < VEC; ++j) d.v[j] = from_f<T>(grad_of(a, g, to_f(v[u].v[j]), c0 + j));
    if (mask) {
      const Pack<uint8_t, VEC> m = load_pack<uint8_t, VEC>(mask + c0);
#pragma unroll
      for (int j = 0; j < VEC; ++j) d.v[j] = m.v[j] ? d.v[j] : from_f<T>(0.f);
    }
    store_own<VEC>(dx + c0, d, at - c0);
  }
}

bool bad_positions(int64_t n0, int64_t n1, int64_t n2, int64_t classes, int64_t* n) {
  if (n0 < 0 || n1 < 0 || n2 < 0 || classes <= 0 || classes > MOST_CLASSES) return true;
  return __builtin_mul_overflow(n0, n1, n) || __builtin_mul_overflow(*n, n2, n) || *n > (1LL << 38);
}

// A launch has less than 2^32 threads, blocks of 256 here; a call that would need more is refused.
constexpr int64_t MOST_BLOCKS = (1LL << 24) - 1;
constexpr int MOST_SPANS = 65535, MOST_BWD_CLASSES = 1 << 21;

// whether whole blocks of positions can share a row of the class mask, and the runs then
bool mask_runs(const void* mask, int64_t mask_div, int64_t positions, int per_block, Tiling* t, int64_t* rows) {
  t->run = positions;
  *rows = 1;
  if (mask && mask_div < positions) {
    if (mask_div < 64) return false;
    t->run = mask_div;
    *rows = (positions + mask_div - 1) / mask_div;
  }
  t->blocks = (unsigned)((t->run + per_block - 1) / per_block);
  return mask && *rows * t->blocks <= MOST_BLOCKS;
}

template <typename T, int K, bool SPLIT, bool FOLDS>
void launch_planes_as(const Args& a, hipStream_t s) {
  constexpr int PER = SPLIT ? 64 : 256;
  Tiling t;
  int64_t rows;
  if (a.classes <= LIST && mask_runs(a.mask, a.mask_div, a.positions, PER, &t, &rows)) {
    hipLaunchKernelGGL((probs_planes<T, K, SPLIT, true, FOLDS>), dim3((unsigned)(rows * t.blocks)), dim3(256), 0, s, a, t);
  } else {
    t.run = a.positions;
    t.blocks = (unsigned)((t.run + PER - 1) / PER);
    hipLaunchKernelGGL((probs_planes<T, K, SPLIT, false, FOLDS>), dim3(t.blocks), dim3(256), 0, s, a, t);
  }
}
template <typename T, int K>
void launch_planes_split(const Args& a, hipStream_t s) {
  // four waves to 64 positions where whole ones would leave the card with less than 8 waves a CU
  if (a.positions < 64 * 2048 && a.classes >= 16) launch_planes_as<T, K, true, true>(a, s);
  else if (a.classes > FOLD * PLANES_UNR) launch_planes_as<T, K, false, true>(a, s);
  else launch_planes_as<T, K, false, false>(a, s);
}
template <typename T>
int launch_planes(const Args& a, hipStream_t s) {
  if ((a.positions + 255) / 256 > MOST_BLOCKS) return LDM_ERR_ARG;
  if (a.k == 0) launch_planes_split<T, 0>(a, s);
  else if (a.k == 1) launch_planes_split<T, 1>(a, s);
  else if (a.k == 2) launch_planes_split<T, 2>(a, s);
  else if (a.k <= 4) launch_planes_split<T, 4>(a, s);
  else if (a.k <= 8) launch_planes_split<T, 8>(a, s);
  else launch_planes_split<T, 16>(a, s);
  LDM_CHECK_LAUNCH();
  return LDM_OK;
}

constexpr int WAVE_CLASSES = 8192;       // a wave's row
constexpr int SHORT_CLASSES = 1024;      // at most 16 classes in a lane's registers
// segments of a long row: whole multiples of a block's reach, up to 512 blocks in all (8 x 131072 fp32: 4.9 us, 5.4 us
// with 256 blocks and 6.3 us with 1024; 256 x 32003 bf16 with 8 alternatives 20, 29 and 18 us, and a longer join)
int segments_of(int64_t positions, int64_t classes, int dtype) {
  const int64_t reach = 256 * 16 / (dtype == LDM_BF16 ? 2 : 4);
  const int64_t most = (classes + reach - 1) / reach;
  return (int)std::max<int64_t>(1, std::min(most, 512 / std::max<int64_t>(1, positions)));
}
bool long_rows(const ldm_label_probs_params* p) { return p->sc == 1 && p->classes > SHORT_CLASSES; }

template <typename T, int G>
void launch_short(const Args& a, hipStream_t s) {
  constexpr int VEC = 16 / (int)sizeof(T), E = 16 / VEC;
  const dim3 grid((unsigned)((a.positions + 256 / G - 1) / (256 / G)));
  if (a.k) hipLaunchKernelGGL((probs_short_rows<T, VEC, G, E, true>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((probs_short_rows<T, VEC, G, E, false>), grid, dim3(256), 0, s, a);
}
template <typename T, bool TOP>
void launch_long(const Args& a, int segments, void* ws, hipStream_t s) {
  constexpr int VEC = 16 / (int)sizeof(T);
  if (a.positions >= 2048 && a.classes <= WAVE_CLASSES) {
    hipLaunchKernelGGL((probs_rows<T, VEC, TOP, 1>), dim3((unsigned)((a.positions + 3) / 4)), dim3(256), 0, s, a, 1,
                       a.classes, (Part*)nullptr, (uint64_t*)nullptr);
    return;
  }
  const int reach = 256 * VEC, per = ((a.classes + reach - 1) / reach + segments - 1) / segments;
  Part* parts = (Part*)ws;
  uint64_t* tops = (uint64_t*)(parts + a.positions * segments);
  hipLaunchKernelGGL((probs_rows<T, VEC, TOP, 4>), dim3((unsigned)(a.positions * segments)), dim3(256), 0, s, a,
                     segments, per * reach, parts, tops);
  if (segments > 1)
    hipLaunchKernelGGL((probs_join<T, TOP>), dim3((unsigned)a.positions), dim3(256), 0, s, a, segments, parts, tops);
}

template <typename T>
int launch(const Args& a, void* ws, hipStream_t s) {
  constexpr int VEC = 16 / (int)sizeof(T);
  if (a.sc == 1 && a.classes > SHORT_CLASSES) {
    const int segments = segments_of(a.positions, a.classes, sizeof(T) == 2 ? LDM_BF16 : LDM_F32);
    if ((a.classes <= WAVE_CLASSES ? (a.positions + 3) / 4 : a.positions * segments) > MOST_BLOCKS) return LDM_ERR_ARG;
    if (a.k) launch_long<T, true>(a, segments, ws, s);
    else launch_long<T, false>(a, segments, ws, s);
  } else if (a.sc == 1 && a.classes >= VEC) {
    const int lanes = (a.classes + 15) / 16;
    if ((a.positions * lanes + 127) / 128 > MOST_BLOCKS) return LDM_ERR_ARG;      // lanes round up to a power of two
    if (lanes <= 1) launch_short<T, 1>(a, s);
    else if (lanes <= 2) launch_short<T, 2>(a, s);
    else if (lanes <= 4) launch_short<T, 4>(a, s);
    else if (lanes <= 8) launch_short<T, 8>(a, s);
    else if (lanes <= 16) launch_short<T, 16>(a, s);
    else if (lanes <= 32) launch_short<T, 32>(a, s);
    else launch_short<T, 64>(a, s);
  } else {
    return launch_planes<T>(a, s);
  }
  LDM_CHECK_LAUNCH();
  return LDM_OK;
}

template <typename T, int PV>
int launch_bwd_planes(const BwdArgs<T>& a, int64_t n, hipStream_t s) {
  if (a.classes > MOST_BWD_CLASSES || (n + 255) / 256 > MOST_BLOCKS) return LDM_ERR_ARG;
  // 32 classes to a thread, or down to 8 where the card would have less than 12 waves a CU; no more spans than a grid has
  // in y
  const int64_t waves = (n + 64 * PV - 1) / (64 * PV);
  auto spans_of = [&](int span) { return (a.classes + span - 1) / span; };
  int span = spans_of(32) > MOST_SPANS ? 64 : 32;
  while (span > 8 && waves * spans_of(span) < 12 * 256 && spans_of(span / 2) <= MOST_SPANS) span /= 2;
  const unsigned spans = (unsigned)spans_of(span);
  Tiling t;
  int64_t rows;
  if (mask_runs(a.mask, a.mask_div, n, 256 * PV, &t, &rows)) {
    hipLaunchKernelGGL((probs_bwd_planes<T, true, PV>), dim3((unsigned)(rows * t.blocks), spans), dim3(256), 0, s, a, t, span);
  } else {
    t.run = n;
    t.blocks = (unsigned)((n + 256 * PV - 1) / (256 * PV));
    hipLaunchKernelGGL((probs_bwd_planes<T, false, PV>), dim3(t.blocks, spans), dim3(256), 0, s, a, t, span);
  }
  LDM_CHECK_LAUNCH();
  return LDM_OK;
}

template <typename T>
int launch_bwd(const ldm_label_probs_bwd_params* p, int64_t n, hipStream_t s) {
  BwdArgs<T> a;
  a.x = (const T*)p->logits; a.dx = (T*)p->d_logits;
  a.n1 = n == p->n2 ? 0 : p->n1; a.n2 = p->n2;
  a.s0 = p->s0; a.s1 = p->s1; a.s2 = p->s2; a.sc = p->sc;
  a.o0 = p->o0; a.o1 = p->o1; a.o2 = p->o2; a.oc = p->oc;
  a.positions = n; a.classes = (int)p->classes;
  a.mask = (const uint8_t*)p->class_mask; a.mask_stride = p->mask_stride; a.mask_div = p->mask_div;
  a.inv_t = 1.f / p->temperature; a.c2 = (float)(1.4426950408889634 / p->temperature);
  a.stats = p->stats; a.gl = p->d_log_prob; a.ge = p->d_entropy;
  constexpr int RV = 16 / (int)sizeof(T);
  if (p->sc == 1 && p->oc == 1 && a.classes >= RV) {
    const unsigned per_row = (unsigned)((a.classes + RV - 1) / RV);
    if (per_row < 256) {
      const int64_t blocks = (n * per_row + 255) / 256;
      if (blocks > MOST_BLOCKS) return LDM_ERR_ARG;
      hipLaunchKernelGGL((probs_bwd_rows<T, RV, 1, true>), dim3((unsigned)blocks), dim3(256), 0, s, a, per_row, 1u);
    } else {
      // two packs to a thread where that leaves little of the row's last block without one (3000 x 5892 bf16, 737 packs:
      // 14.7 us with one, 18.6 us with two; 4096 x 16384, 2048 packs: 47 and 44 us)
      const unsigned two = (per_row + 511) / 512;
      const bool full = per_row * 10 >= two * 512 * 9;
      const unsigned bpr = full ? two : (per_row + 255) / 256;
      if (n * bpr > MOST_BLOCKS) return LDM_ERR_ARG;
      if (full) hipLaunchKernelGGL((probs_bwd_rows<T, RV, 2, false>), dim3((unsigned)(n * bpr)), dim3(256), 0, s, a, per_row, bpr);
      else hipLaunchKernelGGL((probs_bwd_rows<T, RV, 1, false>), dim3((unsigned)(n * bpr)), dim3(256), 0, s, a, per_row, bpr);
    }
    LDM_CHECK_LAUNCH();
    return LDM_OK;
  }
  if constexpr (sizeof(T) == 2) {
    // pairs of positions side by side, in one row of the mask; of few classes they would only halve the waves
    const bool whole = a.n2 % 2 == 0 && (!a.mask || a.mask_div >= n || a.mask_div % 2 == 0);
    if (a.s2 == 1 && a.o2 == 1 && whole && a.classes >= 16) return launch_bwd_planes<T, 2>(a, n, s);
  }
  return launch_bwd_planes<T, 1>(a, n, s);
}

bool bad_temperature(float t) { return !(t >= 1e-4f && t <= 1e4f); }

}  // namespace

extern "C" size_t ldm_label_log_probs_workspace_bytes(const ldm_label_probs_params* p) {
  int64_t n;
  if (!p || !long_rows(p) || bad_positions(p->n0, p->n1, p->n2, p->classes, &n) || n == 0) return 0;
  const int segments = segments_of(n, p->classes, p->dtype);
  return segments == 1 ? 0 : (size_t)(n * segments) * (sizeof(Part) + sizeof(uint64_t) * (size_t)std::max(0, p->topk));
}

extern "C" int ldm_label_log_probs(const ldm_label_probs_params* p, ldm_stream_t stream) {
  int64_t n;
  if (!p || bad_positions(p->n0, p->n1, p->n2, p->classes, &n) || bad_temperature(p->temperature)) return LDM_ERR_ARG;
  if (p->dtype != LDM_F32 && p->dtype != LDM_BF16) return LDM_ERR_ARG;
  if (p->topk < 0 || p->topk > LDM_LABEL_TOPK_MAX || p->topk > p->classes) return LDM_ERR_ARG;
  if (p->s0 < 0 || p->s1 < 0 || p->s2 < 0 || p->sc < 0) return LDM_ERR_ARG;
  if (n == 0) return LDM_OK;
  if (!p->logits || !p->entropy || (p->labels && !p->log_prob) || (p->topk && (!p->top_ids || !p->top_log_probs)))
    return LDM_ERR_ARG;
  if (p->inner <= 0 || n % p->inner || (p->class_mask && (p->mask_div <= 0 || p->mask_stride < 0))) return LDM_ERR_ARG;
  const int64_t need = (int64_t)ldm_label_log_probs_workspace_bytes(p);
  if (need && (!p->workspace || p->workspace_bytes < need)) return LDM_ERR_ARG;
  Args a;
  a.x = p->logits;
  a.n1 = n == p->n2 ? 0 : p->n1; a.n2 = p->n2; a.s0 = p->s0; a.s1 = p->s1; a.s2 = p->s2; a.sc = p->sc;
  a.positions = n; a.classes = (int)p->classes;
  a.labels = p->labels; a.ignore = p->ignore_label; a.has_ignore = p->has_ignore;
  a.mask = (const uint8_t*)p->class_mask; a.mask_stride = p->mask_stride; a.mask_div = p->mask_div;
  a.inner = p->inner;
  a.inv_t = 1.f / p->temperature; a.c2 = (float)(1.4426950408889634 / p->temperature); a.slack = p->temperature * LN2;
  a.lp = p->log_prob; a.ent = p->entropy; a.top_lp = p->top_log_probs; a.top_id = p->top_ids; a.stats = p->stats;
  a.k = p->topk;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return p->dtype == LDM_BF16 ? launch<bf16_t>(a, p->workspace, s) : launch<float>(a, p->workspace, s);
}

extern "C" int ldm_label_log_probs_bwd(const ldm_label_probs_bwd_params* p, ldm_stream_t stream) {
  int64_t n;
  if (!p || bad_positions(p->n0, p->n1, p->n2, p->classes, &n) || bad_temperature(p->temperature)) return LDM_ERR_ARG;
  if (p->dtype != LDM_F32 && p->dtype != LDM_BF16) return LDM_ERR_ARG;
  if (p->s0 < 0 || p->s1 < 0 || p->s2 < 0 || p->sc < 0 || p->o0 < 0 || p->o1 < 0 || p->o2 < 0 || p->oc < 0)
    return LDM_ERR_ARG;
  if (n == 0) return LDM_OK;
  if (!p->logits || !p->d_logits || !p->stats || (p->class_mask && (p->mask_div <= 0 || p->mask_stride < 0)))
    return LDM_ERR_ARG;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return p->dtype == LDM_BF16 ? launch_bwd<bf16_t>(p, n, s) : launch_bwd<float>(p, n, s);
}
