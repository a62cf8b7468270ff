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
// All sums are fp32; the logits are exact in fp32 and d x_j is rounded once to their type.
// exp is the hardware's exp2 of one rounded product, so a term e^z carries a relative error of
// about |z| 2^-24: at most 0.37 x 2^-24 of the largest term.
#include "common.h"

#include <algorithm>
#include <math.h>

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float LOWEST = -3e38f;   // finite stand-in for x_j - m = -inf: 0 * LOWEST is 0, 0 * inf is NaN

struct Args {
  const void* x;
  int64_t n1, n2, s0, s1, s2, sc, positions;
  int classes;
  const int64_t* labels;
  int64_t ignore;
  int has_ignore;
  const uint8_t* mask;
  int64_t mask_stride, mask_div, inner;
  float c2, inv_t;                 // log2(e) / T, 1 / T
  float *lp, *ent, *top_lp, *stats;
  int32_t* top_id;
  int k;
};

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

// running maximum and sums of one set of logits; the maximum's own term is in neither sum
struct Soft {
  float m, r, t;
  __device__ __forceinline__ void clear() { m = -INFINITY; r = t = 0.f; }
  __device__ __forceinline__ void rescale(float to, float c2) {   // sums relative to `to` >= m, to > -inf
    const float d = fmaxf(m - to, LOWEST), s = exp2_fast(d * c2);
    t = s * t + (s * d) * r;
    r *= s;
  }
  __device__ __forceinline__ void add(float x, float c2) {        // x is no NaN
    const float hi = fmaxf(m, x), lo = fminf(m, x), to = hi == -INFINITY ? 0.f : hi;
    rescale(to, c2);
    const float d = fmaxf(lo - to, LOWEST), e = exp2_fast(d * c2);
    r += e;
    t = fmaf(d, e, t);
    m = hi;
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

// what a position's sums come to
struct Result { float ls, ent, lp; int label; };
__device__ __forceinline__ Result result_of(const Args& a, const Soft& s, bool nan, int64_t y, float xy) {
  Result q;
  const float none = __int_as_float(0x7fc00000);
  const bool empty = s.m == -INFINITY, bad = nan || s.m == INFINITY;
  q.ls = bad ? none : log1pf(s.r);
  q.ent = bad ? none : empty ? 0.f : q.ls - s.t * a.inv_t / (1.f + s.r);
  const bool known = !(a.has_ignore && y == a.ignore), inside = y >= 0 && y < a.classes;
  if (!known) q.lp = 0.f;
  else if (!inside || bad) q.lp = none;
  else q.lp = xy == -INFINITY ? -INFINITY : (xy - s.m) * a.inv_t - q.ls;
  q.label = known && inside && q.lp > -INFINITY ? (int)y : -1;   // NaN > -inf is false: the row is NaN anyway
  return q;
}
__device__ __forceinline__ void store_result(const Args& a, int64_t pos, const Soft& s, const Result& q) {
  a.ent[pos] = q.ent;
  if (a.labels) a.lp[pos] = q.lp;
  if (a.stats) {
    a.stats[pos] = s.m;
    a.stats[a.positions + pos] = q.ls;
    a.stats[2 * a.positions + pos] = q.ent;
    a.stats[3 * a.positions + pos] = __int_as_float(a.labels ? q.label : -1);
  }
}
__device__ __forceinline__ void store_top(const Args& a, int64_t pos, int j, int key, int id, const Soft& s, float ls) {
  const int64_t o = pos / a.inner, at = (o * a.k + j) * a.inner + (pos - o * a.inner);
  a.top_id[at] = id;
  a.top_lp[at] = id < 0 ? -INFINITY : (key_value(key) - s.m) * a.inv_t - ls;
}

__device__ __forceinline__ int64_t offset_of(int64_t pos, int64_t n1, int64_t n2, int64_t s0, int64_t s1, int64_t s2) {
  const int64_t line = pos / n2;
  return (line / n1) * s0 + (line % n1) * s1 + (pos % n2) * s2;
}

// the wave's Softs joined, in every lane
__device__ __forceinline__ Soft wave_join(const Soft& s, float c2) {
  const float m = wave_max(s.m), to = m == -INFINITY ? 0.f : m;
  const bool holds = s.m == m;     // the first lane that holds the maximum keeps its term out of the sums
  const bool keeper = holds && (int)(threadIdx.x & 63) == __ffsll((unsigned long long)__ballot(holds)) - 1;
  Soft o = s;
  o.rescale(to, c2);
  const float d = fmaxf(s.m - to, LOWEST), e = keeper ? 0.f : exp2_fast(d * c2);
  o.m = m;
  o.r = wave_sum(o.r + e);
  o.t = wave_sum(fmaf(d, e, o.t));
  return o;
}

// (key, class) pairs in the order of the answer: larger key, then lower class; an empty one (-1) last
__device__ __forceinline__ bool before(int k, int c, int key, int id) {
  return k > key || (k == key && (unsigned)c < (unsigned)id);
}
// the n first of the wave's lists: lane j < n gets the j-th
template <int K>
__device__ __forceinline__ void wave_top(Top<K>& top, int n, int& key, int& id) {
  key = KEY_NONE;
  id = -1;
  for (int j = 0; j < n; ++j) {
    int k = top.key[0], c = top.id[0];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const int k2 = __shfl_xor(k, o, 64), c2 = __shfl_xor(c, o, 64);
      if (before(k2, c2, k, c)) { k = k2; c = c2; }
    }
    if ((int)(threadIdx.x & 63) == j) { key = k; id = c; }
    if (top.id[0] == c && c >= 0) {
#pragma unroll
      for (int i = 0; i + 1 < K; ++i) { top.key[i] = top.key[i + 1]; top.id[i] = top.id[i + 1]; }
      top.key[K - 1] = KEY_NONE;
      top.id[K - 1] = -1;
    }
  }
}

// one block per row of adjacent classes
template <typename T, int K>
__global__ __launch_bounds__(256) void probs_rows(const Args a) {
  __shared__ Soft part[4];
  __shared__ int part_key[64], part_id[64], part_nan[4];
  const int64_t pos = blockIdx.x;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const T* x = (const T*)a.x + offset_of(pos, a.n1, a.n2, a.s0, a.s1, a.s2);
  const uint8_t* mask = a.mask ? a.mask + (pos / a.mask_div) * a.mask_stride : nullptr;
  Soft s;
  s.clear();
  Top<K> top;
  top.clear();
  bool nan = false;
  for (int c = tid; c < a.classes; c += 256) {
    float v = to_f(x[c]);
    if (mask && !mask[c]) v = -INFINITY;
    top.add(order_key(v), c);
    nan |= v != v;
    s.add(v, a.c2);
  }
  s = wave_join(s, a.c2);
  if constexpr (K > 0) {
    int key, id;
    wave_top<K>(top, a.k, key, id);
    if (lane < a.k) { part_key[wave * a.k + lane] = key; part_id[wave * a.k + lane] = id; }
  }
  if (lane == 0) part[wave] = s;
  const bool any = __ballot(nan) != 0;
  if (lane == 0) part_nan[wave] = any;
  __syncthreads();
  if (wave) return;
  s = part[0];
  for (int w = 1; w < 4; ++w) s.join(part[w], a.c2);
  nan = part_nan[0] | part_nan[1] | part_nan[2] | part_nan[3];
  const int64_t y = a.labels ? a.labels[pos] : -1;
  float xy = -INFINITY;
  if (y >= 0 && y < a.classes && !(mask && !mask[y])) xy = to_f(x[y]);
  const Result q = result_of(a, s, nan, y, xy);
  if (lane == 0) store_result(a, pos, s, q);
  if constexpr (K > 0) {
    Top<1> one;
    one.key[0] = lane < 4 * a.k ? part_key[lane] : KEY_NONE;
    one.id[0] = lane < 4 * a.k ? part_id[lane] : -1;
    int key, id;
    wave_top<1>(one, a.k, key, id);
    if (lane < a.k) store_top(a, pos, lane, key, id, s, q.ls);
  }
}

// one thread per position
template <typename T, int K>
__global__ __launch_bounds__(256) void probs_positions(const Args a) {
  const int64_t pos = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (pos >= a.positions) return;
  const T* x = (const T*)a.x + offset_of(pos, a.n1, a.n2, a.s0, a.s1, a.s2);
  const uint8_t* mask = a.mask ? a.mask + (pos / a.mask_div) * a.mask_stride : nullptr;
  const int64_t y = a.labels ? a.labels[pos] : -1;
  Soft s;
  s.clear();
  Top<K> top;
  top.clear();
  bool nan = false;
  float xy = -INFINITY;
  for (int c = 0; c < a.classes; ++c) {
    float v = to_f(x[c * a.sc]);
    if (mask && !mask[c]) v = -INFINITY;
    top.add(order_key(v), c);
    nan |= v != v;
    xy = c == y ? v : xy;
    s.add(v, a.c2);
  }
  const Result q = result_of(a, s, nan, y, xy);
  store_result(a, pos, s, q);
#pragma unroll
  for (int j = 0; j < K; ++j)
    if (j < a.k) store_top(a, pos, j, top.key[j], top.id[j], s, q.ls);
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

struct RowGrad { float m, ls, ls2, h, gl, ge; int label; };
template <typename T>
__device__ __forceinline__ RowGrad row_grad(const BwdArgs<T>& a, int64_t pos) {
  RowGrad g;
  g.m = a.stats[pos];
  g.ls = a.stats[a.positions + pos];
  g.h = a.stats[2 * a.positions + pos];
  g.label = __float_as_int(a.stats[3 * a.positions + pos]);
  g.gl = a.gl && g.label >= 0 ? a.gl[pos] * a.inv_t : 0.f;
  g.ge = a.ge ? a.ge[pos] * a.inv_t : 0.f;
  g.ls2 = g.ls * LOG2E;
  if (g.m == -INFINITY) { g.m = 0.f; g.gl = g.ge = 0.f; }
  return g;
}
template <typename T>
__device__ __forceinline__ float grad_of(const BwdArgs<T>& a, const RowGrad& g, float x, int c) {
  // below 2^-1000 p is 0 and its log stays finite; a row with a NaN or +inf has ls = NaN, and so has every p of it
  const float z2 = fmaxf((x - g.m) * a.c2, -1000.f);
  const float p = exp2_fast(z2 - g.ls2);
  const float w = fmaf(g.ge, fmaf(z2, LN2, g.h - g.ls), g.gl);
  return (c == g.label ? g.gl : 0.f) - p * w;
}

template <typename T>
__global__ __launch_bounds__(256) void probs_bwd(const BwdArgs<T> a) {
  const int64_t pos = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (pos >= a.positions) return;
  const T* x = a.x + offset_of(pos, a.n1, a.n2, a.s0, a.s1, a.s2);
  T* dx = a.dx + offset_of(pos, a.n1, a.n2, a.o0, a.o1, a.o2);
  const uint8_t* mask = a.mask ? a.mask + (pos / a.mask_div) * a.mask_stride : nullptr;
  const RowGrad g = row_grad(a, pos);
  for (int c = 0; c < a.classes; ++c)
    dx[c * a.oc] = from_f<T>(mask && !mask[c] ? 0.f : grad_of(a, g, to_f(x[c * a.sc]), c));
}

bool bad_positions(int64_t n0, int64_t n1, int64_t n2, int64_t classes, int64_t* n) {
  if (n0 < 0 || n1 < 0 || n2 < 0 || classes <= 0 || classes > (1 << 30)) return true;
  *n = n0 * n1 * n2;
  return *n > (1LL << 38);                      // grids stay below 2^31 blocks of 256
}

template <typename T>
int launch(const Args& a, hipStream_t s) {
  const dim3 block(256);
  if (a.sc == 1 && a.classes >= 256) {
    if (a.positions > 0x7fffffff) return LDM_ERR_ARG;
    const dim3 grid((unsigned)a.positions);
    if (a.k == 0) hipLaunchKernelGGL((probs_rows<T, 0>), grid, block, 0, s, a);
    else if (a.k <= 4) hipLaunchKernelGGL((probs_rows<T, 4>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((probs_rows<T, 16>), grid, block, 0, s, a);
    LDM_CHECK_LAUNCH();
    return LDM_OK;
  }
  const dim3 grid((unsigned)((a.positions + 255) / 256));
  if (a.k == 0) hipLaunchKernelGGL((probs_positions<T, 0>), grid, block, 0, s, a);
  else if (a.k <= 4) hipLaunchKernelGGL((probs_positions<T, 4>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((probs_positions<T, 16>), grid, block, 0, s, a);
  LDM_CHECK_LAUNCH();
  return LDM_OK;
}

template <typename T>
int launch_bwd(const ldm_label_probs_bwd_params* p, int64_t n, hipStream_t s) {
  BwdArgs<T> a;
  a.x = (const T*)p->logits; a.dx = (T*)p->d_logits;
  a.n1 = p->n1; a.n2 = p->n2;
  a.s0 = p->s0; a.s1 = p->s1; a.s2 = p->s2; a.sc = p->sc;
  a.o0 = p->o0; a.o1 = p->o1; a.o2 = p->o2; a.oc = p->oc;
  a.positions = n; a.classes = (int)p->classes;
  a.mask = (const uint8_t*)p->class_mask; a.mask_stride = p->mask_stride; a.mask_div = p->mask_div;
  a.inv_t = 1.f / p->temperature; a.c2 = (float)(1.4426950408889634 / p->temperature);
  a.stats = p->stats; a.gl = p->d_log_prob; a.ge = p->d_entropy;
  hipLaunchKernelGGL((probs_bwd<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a);
  LDM_CHECK_LAUNCH();
  return LDM_OK;
}

bool bad_temperature(float t) { return !(t >= 1e-4f && t <= 1e4f); }

}  // namespace

extern "C" size_t ldm_label_log_probs_workspace_bytes(const ldm_label_probs_params* p) {
  (void)p;
  return 0;
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
  if (p->workspace_bytes < (int64_t)ldm_label_log_probs_workspace_bytes(p)) return LDM_ERR_ARG;
  Args a;
  a.x = p->logits;
  a.n1 = p->n1; a.n2 = p->n2; a.s0 = p->s0; a.s1 = p->s1; a.s2 = p->s2; a.sc = p->sc;
  a.positions = n; a.classes = (int)p->classes;
  a.labels = p->labels; a.ignore = p->ignore_label; a.has_ignore = p->has_ignore;
  a.mask = (const uint8_t*)p->class_mask; a.mask_stride = p->mask_stride; a.mask_div = p->mask_div;
  a.inner = p->inner;
  a.inv_t = 1.f / p->temperature; a.c2 = (float)(1.4426950408889634 / p->temperature);
  a.lp = p->log_prob; a.ent = p->entropy; a.top_lp = p->top_log_probs; a.top_id = p->top_ids; a.stats = p->stats;
  a.k = p->topk;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return p->dtype == LDM_BF16 ? launch<bf16_t>(a, s) : launch<float>(a, s);
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
