// k_scores.hip — scores of given tokens under a model's logits, and
// distillation of a student from such a score of its teacher.
//
// With z = x / T, m = max x, s = sum exp((x - m) / T) over a row's C classes:
//   log p_j = (x_j - m) / T - ln s
//   H       = ln s - (1 / s) sum exp((x_j - m) / T) (x_j - m) / T
//   d(g log p_t + h H) / dx_j = [g (delta_jt - p_j) - h p_j (log p_j + H)] / T
// and for a teacher's k classes of log probabilities v_i:
//   q_i = exp(v_i - Z), Z = ln sum exp v (renormalised) or 0 (with a tail)
//   q_t = max(0, 1 - sum q) (tail) or 0,  S = sum q + q_t
//   L   = sum q_i (ln q_i - log p_i) + q_t (ln q_t - ln p_t), p_t the sum of
//         the unlisted p
//   dL / dx_j = (S p_j - q_j) / T listed, p_j (S - q_t / p_t) / T unlisted
//
// A masked class is -inf and takes no part. A row with a NaN or +inf has no
// distribution: its outputs are NaN. A row with every class masked scores
// -inf and has zero gradients. No atomics on floats; every sum has a fixed
// order.
#include "device_common.h"
#include "kernels.h"

#include <cfloat>
#include <cmath>

namespace seeml_hip {

namespace {

constexpr int kBlock = 256;
constexpr float kLow = -1e30f;  // finite stand-in for (-inf) * 0 products
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));

// log2(e) / T as a sum of two floats, both positive: a difference of logits
// times the pair is right to half a unit in the last place, where one float
// would lean by its own rounding, the same way on every class.
struct TempScale {
  float hi, lo;
};
TempScale ScaleOf(double T) {
  const double c = M_LOG2E / T;
  TempScale s;
  s.hi = static_cast<float>(c);
  if (static_cast<double>(s.hi) > c) s.hi = std::nextafterf(s.hi, 0.0f);
  s.lo = fmaxf(static_cast<float>(c - s.hi), FLT_MIN);  // never 0: -inf * 0
  return s;
}
// (x - m) / T in base 2; -inf stays -inf.
__device__ __forceinline__ float scaled(float x, float m, TempScale c) {
  const float y = x - m;
  return fmaf(y, c.hi, y * c.lo);
}

// One logit as float, and a gradient rounded once to the logits' type.
typedef uint32_t uint32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t uint32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));
template <int DT> struct Elem;
template <> struct Elem<kF32> {
  using T = float;
  using rawu = uint32x4_at4;
  static __device__ float get(T v) { return v; }
  static __device__ T put(float v) { return v; }
};
template <> struct Elem<kBF16> {
  using T = __bf16;
  using rawu = uint32x4_at2;
  static __device__ float get(T v) { return static_cast<float>(v); }
  static __device__ T put(float v) { return static_cast<T>(v); }
};
template <> struct Elem<kF16> {
  using T = _Float16;
  using rawu = uint32x4_at2;
  static __device__ float get(T v) { return static_cast<float>(v); }
  static __device__ T put(float v) { return static_cast<T>(v); }
};

// Order of two logits as whole numbers: by value, -0 equal to +0.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// By value, then the lower class first; 0 is below every unmasked logit.
__device__ __forceinline__ uint64_t key_of(float v, uint32_t col) {
  return (static_cast<uint64_t>(ordered(v)) << 32) | (0xFFFFFFFFu - col);
}


// A row is read as whole 16-byte vectors from its first class on, at the
// alignment of its elements (a vector that straddles a line costs one more
// access, rows of any stride keep the wide loads), and the classes behind the
// last whole vector one by one.
template <int DT>
struct Row {
  using E = Elem<DT>;
  using T = typename E::T;
  static constexpr int V = 16 / sizeof(T);
  typedef uint32_t raw __attribute__((ext_vector_type(4)));
  using rawu = typename E::rawu;
  const T* x;

  __device__ __forceinline__ raw load(uint32_t j, bool nt) const {
    const rawu* p = reinterpret_cast<const rawu*>(x + static_cast<size_t>(j) * V);
    return nt ? __builtin_nontemporal_load(p) : *p;
  }
  static __device__ __forceinline__ void unpack(raw r, float* v) {
    if constexpr (DT == kF32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
    } else if constexpr (DT == kBF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(r[i] << 16);
        v[2 * i + 1] = __uint_as_float(r[i] & 0xFFFF0000u);
      }
    } else {
      typedef _Float16 h8 __attribute__((ext_vector_type(8)));
      const h8 h = __builtin_bit_cast(h8, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(h[i]);
    }
  }
  // Vector j of the row, whole or (the last) filled up with masked classes.
  __device__ __forceinline__ void any(uint32_t j, uint32_t C, float* v) const {
    if ((j + 1) * V <= C) {
      unpack(load(j, false), v);
      return;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = j * V + e < C ? E::get(x[j * V + e]) : -INFINITY;
  }
};

__device__ __forceinline__ float exp2_raw(float v) { return __builtin_amdgcn_exp2f(v); }

// A softmax's running sums: s = sum e, w = sum e d, with e = 2^d, d the scaled
// difference from m. m starts at the lowest finite value, so that masked
// classes add 0 and no difference of infinities arises; a NaN or +inf turns s
// into NaN.
struct Online {
  float m = -FLT_MAX, s = 0.0f, w = 0.0f;
  __device__ __forceinline__ void raise(float to, TempScale c) {
    if (to > m) {
      const float d = fmaxf(scaled(m, to, c), kLow), f = exp2_raw(d);
      w = fmaf(s, d, w) * f;
      s *= f;
      m = to;
    }
  }
  // n values of maximum `top`; their sums are formed apart, so that a
  // thread's chain of additions stays short.
  template <int n>
  __device__ __forceinline__ void add(const float* v, float top, TempScale c) {
    raise(top, c);
    float sb = 0.0f, wb = 0.0f;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float d = scaled(v[i], m, c), e = exp2_raw(d);
      sb += e;
      wb = fmaf(e, fmaxf(d, kLow), wb);
    }
    s += sb;
    w += wb;
  }
};

struct RowSums {
  float m;
  double s, w;
};
// The threads' sums joined: in a wavefront by a butterfly, the wavefronts in
// order. Every thread gets them.
template <int NT>
__device__ __forceinline__ RowSums join(const Online& o, TempScale c, RowSums* scratch) {
  RowSums t;
  t.m = wave_max(o.m);
  const float d = fmaxf(scaled(o.m, t.m, c), kLow), f = exp2_raw(d);
  t.s = wave_sum(static_cast<double>(o.s * f));
  t.w = wave_sum(static_cast<double>(fmaf(o.s, d, o.w) * f));
  if constexpr (NT == kWave) return t;
  if (threadIdx.x % kWave == 0) scratch[threadIdx.x / kWave] = t;
  __syncthreads();
  t = scratch[0];
#pragma unroll
  for (int i = 1; i < NT / kWave; ++i) t.m = fmaxf(t.m, scratch[i].m);
  double s = 0.0, w = 0.0;
#pragma unroll
  for (int i = 0; i < NT / kWave; ++i) {
    const float di = fmaxf(scaled(scratch[i].m, t.m, c), kLow);
    const double fi = exp2_raw(di);
    s += scratch[i].s * fi;
    w += (scratch[i].w + scratch[i].s * di) * fi;
  }
  t.s = s;
  t.w = w;
  return t;
}

// ---- the k likeliest classes -------------------------------------------------
//
// The sweep leaves the maximum of each thread's classes, and of up to kGroups
// groups of them. The k-th largest thread maximum (or a value a little below:
// any value that at least k threads reach) bounds the k-th largest class from
// below, so only groups that reach it are read again, and of those only the
// classes that do: about k, unless ties crowd them. They are ranked by
// counting, value first, then the lower class; keys are distinct, so neither
// the order in which they were collected nor the bound's slack shows.
constexpr int kGroups = 8;
constexpr int kBatch = 4;  // vectors in flight per thread

template <int NT>
struct Select {
  static constexpr uint32_t kCand = NT == kWave ? 256 : 1024;
  union {
    float group[kGroups * NT];  // maxima, until `list` is made from them
    uint64_t cand[kCand];       // keys of the classes that reach the bound
  };
  float best[NT];
  uint16_t list[kGroups * NT];
  int wave[NT / kWave];
  uint32_t n_list, n_cand;
};

// A whole-number value that at least k of the threads' maxima reach, near the
// k-th largest; the least finite one's if fewer than k are unmasked. The same
// for every wavefront.
constexpr uint32_t kLeast = 0x00800000u;  // ordered(-FLT_MAX)
template <int NT>
__device__ __forceinline__ uint32_t bound_of(const float* best, uint32_t k) {
  constexpr int n = NT / kWave;
  uint32_t key[n], hi = 0;
#pragma unroll
  for (int i = 0; i < n; ++i) {
    key[i] = ordered(best[i * kWave + threadIdx.x % kWave]);
    hi = key[i] > hi ? key[i] : hi;
  }
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) {
    const uint32_t o = __shfl_xor(hi, off, kWave);
    hi = o > hi ? o : hi;
  }
  const auto reach = [&](uint32_t th) {
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < n; ++i) c += static_cast<uint32_t>(__popcll(__ballot(key[i] >= th)));
    return c;
  };
  uint32_t lo = kLeast;
  if (reach(lo) < k) return lo;
  const uint32_t above = ++hi;
  // Maxima lie within a few octaves of each other: look near the top first.
  for (uint32_t step = 1u << 23; step != 0 && step < above - kLeast; step <<= 1) {
    if (reach(above - step) >= k) {
      lo = above - step;
      break;
    }
    hi = above - step;
  }
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2, c = reach(mid);
    if (c >= k) {
      lo = mid;
      if (c <= k + k / 4 + 2) break;
    } else {
      hi = mid;
    }
  }
  return lo;
}

// Classes of the row at or above `th`, counted by the whole workgroup.
template <int DT, int NT>
__device__ uint32_t count_reaching(const Row<DT>& row, uint32_t C, uint32_t th, int* scratch) {
  constexpr int V = Row<DT>::V;
  int n = 0;
  for (uint32_t j = threadIdx.x; j * V < C; j += NT) {
    float v[V];
    row.any(j, C, v);
#pragma unroll
    for (int e = 0; e < V; ++e) n += ordered(v[e]) >= th ? 1 : 0;
  }
  return static_cast<uint32_t>(block_sum<int, NT>(n, scratch));
}

// More classes reach the bound than `cand` holds: ties at one value (a row of
// equal logits, masks at the lowest value), or an order made for it. Finds the
// k-th largest value by halving between the bound and the row's maximum,
// counting over the row each time (once where the ties are at the bound), then
// takes the classes above it and the first of those equal to it.
template <int DT, int NT>
__device__ __noinline__ void select_crowded(const Row<DT>& row, uint32_t C, uint32_t k, uint32_t lo,
                                            uint32_t hi, Select<NT>& sel) {
  constexpr int V = Row<DT>::V;
  for (uint32_t mid = lo + 1; hi - lo > 1; mid = lo + (hi - lo) / 2) {
    if (count_reaching<DT, NT>(row, C, mid, sel.wave) >= k) lo = mid;
    else hi = mid;
  }
  __syncthreads();
  if (threadIdx.x == 0) sel.n_cand = 0;
  __syncthreads();
  for (uint32_t j = threadIdx.x; j * V < C; j += NT) {
    float v[V];
    row.any(j, C, v);
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (ordered(v[e]) > lo) sel.cand[atomicAdd(&sel.n_cand, 1u)] = key_of(v[e], j * V + e);
  }
  __syncthreads();
  uint32_t have = sel.n_cand;  // below k
  const int lane = threadIdx.x % kWave, wv = threadIdx.x / kWave;
  for (uint32_t j0 = 0; j0 * V < C && have < k; j0 += NT) {
    const uint32_t j = j0 + threadIdx.x;
    float v[V];
    int own = 0;
    if (j * V < C) {
      row.any(j, C, v);
#pragma unroll
      for (int e = 0; e < V; ++e) own += ordered(v[e]) == lo ? 1 : 0;
    }
    int before = own;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const int o = __shfl_up(before, off, kWave);
      if (lane >= off) before += o;
    }
    __syncthreads();
    if (lane == kWave - 1) sel.wave[wv] = before;
    __syncthreads();
    uint32_t at = have + static_cast<uint32_t>(before - own);
    for (int i = 0; i < NT / kWave; ++i) {
      if (i < wv) at += static_cast<uint32_t>(sel.wave[i]);
      have += static_cast<uint32_t>(sel.wave[i]);
    }
    if (own)
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (ordered(v[e]) == lo) {
          if (at < k) sel.cand[at] = key_of(v[e], j * V + e);
          ++at;
        }
  }
  __syncthreads();
  if (threadIdx.x == 0) sel.n_cand = have < k ? have : k;
  __syncthreads();
}

// Leaves at least the k largest unmasked classes' keys (or all of them) in
// sel.cand. `batches` and `per_group` are the sweep's.
template <int DT, int NT>
__device__ __forceinline__ void select_top(const Row<DT>& row, uint32_t C, uint32_t k, float top,
                                           uint32_t batches, uint32_t per_group, float best,
                                           Select<NT>& sel) {
  constexpr int V = Row<DT>::V;
  const uint32_t nv = C / V;
  sel.best[threadIdx.x] = best;
  if (threadIdx.x == 0) sel.n_list = sel.n_cand = 0;
  __syncthreads();
  const uint32_t th = bound_of<NT>(sel.best, k);
  if (ordered(best) >= th)
    for (uint32_t g = 0; g * per_group < batches; ++g)
      if (ordered(sel.group[g * NT + threadIdx.x]) >= th)
        sel.list[atomicAdd(&sel.n_list, 1u)] = static_cast<uint16_t>(g * NT + threadIdx.x);
  __syncthreads();
  const auto take = [&](float v, uint32_t col) {
    if (ordered(v) >= th) {
      const uint32_t at = atomicAdd(&sel.n_cand, 1u);
      if (at < Select<NT>::kCand) sel.cand[at] = key_of(v, col);
    }
  };
  const uint32_t each = per_group * kBatch, n = sel.n_list * each;
  for (uint32_t i = threadIdx.x; i < n; i += NT) {
    const uint32_t id = sel.list[i / each], at = i % each;
    const uint32_t j = ((id / NT) * per_group * kBatch + at) * NT + id % NT;
    if (j >= nv) continue;
    float v[V];
    row.any(j, C, v);
#pragma unroll
    for (int e = 0; e < V; ++e) take(v[e], j * V + e);
  }
  if (threadIdx.x < C - nv * V) {
    const uint32_t col = nv * V + threadIdx.x;
    take(Elem<DT>::get(row.x[col]), col);
  }
  __syncthreads();
  if (sel.n_cand > Select<NT>::kCand)
    select_crowded<DT, NT>(row, C, k, th, ordered(top) + 1, sel);
}

// ---- scores ---------------------------------------------------------------------

template <int DT, int NT>
__global__ __launch_bounds__(NT) void score_fwd_kernel(TokenScoreArgs a, TempScale c, int nt) {
  __shared__ Select<NT> sel;
  __shared__ RowSums sums[NT / kWave];
  using E = Elem<DT>;
  constexpr int V = Row<DT>::V;
  const size_t r = blockIdx.x;
  const Row<DT> row{static_cast<const typename E::T*>(a.logits) + r * a.stride};
  const uint32_t C = static_cast<uint32_t>(a.C), k = a.k, nv = C / V;
  const uint32_t batches = (nv + NT * kBatch - 1) / (NT * kBatch);
  const uint32_t per_group = (batches + kGroups - 1) / kGroups;
  int32_t t = -1;
  float xt = 0.0f;
  if (threadIdx.x == 0 && a.logp) {
    t = a.targets[r];
    if (t >= 0 && static_cast<uint32_t>(t) < C) xt = E::get(row.x[t]);
  }
  Online o;
  float best = -INFINITY, group = -INFINITY;
  for (uint32_t b = 0; b < batches; ++b) {
    typename Row<DT>::raw raw[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      raw[u] = row.load(min((b * kBatch + u) * NT + threadIdx.x, nv - 1), nt);
    float v[kBatch * V];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) Row<DT>::unpack(raw[u], v + u * V);
    if (b + 1 == batches)
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if ((b * kBatch + u) * NT + threadIdx.x >= nv)
#pragma unroll
          for (int e = 0; e < V; ++e) v[u * V + e] = -INFINITY;
    float top = v[0];
#pragma unroll
    for (int i = 1; i < kBatch * V; ++i) top = fmaxf(top, v[i]);
    o.add<kBatch * V>(v, top, c);
    if (k) {
      group = fmaxf(group, top);
      if ((b + 1) % per_group == 0 || b + 1 == batches) {
        sel.group[(b / per_group) * NT + threadIdx.x] = group;
        best = fmaxf(best, group);
        group = -INFINITY;
      }
    }
  }
  if (threadIdx.x < C - nv * V) {
    const float v = E::get(row.x[nv * V + threadIdx.x]);
    o.add<1>(&v, v, c);
  }
  const RowSums q = join<NT>(o, c, sums);
  const bool bad = q.s != q.s, empty = q.s == 0.0;
  const float nan = __builtin_nanf("");
  // In base 2 until the end: (x - m) / T = scaled ln 2.
  const double ls = log(q.s);
  if (threadIdx.x == 0) {
    const double inv_T = 1.0 / a.T, w = q.w * M_LN2;
    const float H = bad ? nan : empty ? 0.0f : static_cast<float>(ls - w / q.s);
    if (a.logp) {
      float lp = 0.0f;
      if (t >= 0)
        lp = static_cast<uint32_t>(t) >= C || bad ? nan
             : empty                              ? -INFINITY
                     : static_cast<float>((static_cast<double>(xt) - q.m) * inv_T - ls);
      a.logp[r] = lp;
    }
    if (a.entropy) a.entropy[r] = H;
    if (a.stats)
      *reinterpret_cast<float4u*>(a.stats + r * kScoreStats) =
          float4u{bad ? nan : empty ? 0.0f : q.m,
                  bad ? nan : empty ? INFINITY : static_cast<float>(ls), H,
                  bad ? nan : empty ? 0.0f : static_cast<float>(1.0 / q.s)};
  }
  if (!k) return;
  uint32_t n = 0;
  if (!bad && !empty) {
    select_top<DT, NT>(row, C, k, q.m, batches, per_group, best, sel);
    n = sel.n_cand;
  }
  int32_t* ids = a.top_ids + r * k;
  float* lps = a.top_logp + r * k;
  const double inv_T = 1.0 / a.T;
  for (uint32_t i = threadIdx.x; i < n; i += NT) {
    const uint64_t key = sel.cand[i];
    uint32_t rank = 0;
    for (uint32_t j = 0; j < n; ++j) rank += sel.cand[j] > key ? 1 : 0;
    if (rank >= k) continue;
    const uint32_t col = 0xFFFFFFFFu - static_cast<uint32_t>(key);
    const uint32_t o32 = static_cast<uint32_t>(key >> 32);
    const float v = __uint_as_float(o32 & 0x80000000u ? o32 & 0x7FFFFFFFu : ~o32);
    ids[rank] = static_cast<int32_t>(col);
    lps[rank] = static_cast<float>((static_cast<double>(v) - q.m) * inv_T - ls);
  }
  for (uint32_t i = n + threadIdx.x; i < k; i += NT) {
    ids[i] = -1;
    lps[i] = bad ? nan : -INFINITY;
  }
}

template <int DT>
__global__ __launch_bounds__(kBlock) void score_bwd_kernel(TokenScoreBwdArgs a, TempScale c2) {
  using E = Elem<DT>;
  const size_t r = blockIdx.x;
  const typename E::T* x = static_cast<const typename E::T*>(a.logits) + r * a.stride;
  typename E::T* dx = static_cast<typename E::T*>(a.dlogits) + r * a.dstride;
  const uint32_t C = static_cast<uint32_t>(a.C);
  const float* st = a.stats + r * kScoreStats;
  const float m = st[0], ls = st[1], H = st[2], inv_s = st[3];
  const float inv_T = static_cast<float>(1.0 / a.T);
  const int32_t t = a.targets ? a.targets[r] : -1;
  const bool empty = ls == INFINITY;
  float up = a.dlogp && t >= 0 ? a.dlogp[r] * inv_T : 0.0f;
  float bonus = a.dentropy ? a.dentropy[r] * inv_T : 0.0f;
  if (t >= 0 && static_cast<uint32_t>(t) >= C) up = __builtin_nanf("");
  if (empty) up = bonus = 0.0f;
  const float A = -fmaf(bonus, H, up), B = -bonus;
  const float ln2 = static_cast<float>(M_LN2);
  for (uint32_t j = threadIdx.x; j < C; j += kBlock) {
    const float d = scaled(E::get(x[j]), m, c2);
    const float p = exp2f(d) * inv_s;
    float g = empty ? 0.0f : p * fmaf(B, fmaxf(fmaf(d, ln2, -ls), kLow), A);
    if (static_cast<int32_t>(j) == t) g += up;
    dx[j] = E::put(g);
  }
}

// ---- distillation -----------------------------------------------------------

constexpr uint32_t kMarkCols = 65536;  // classes per bitmap sweep: 8 KiB of LDS

// What a row's teacher list says: q_i, S, q_t. Every thread gets them.
struct Teacher {
  double Z, S, left;
  bool bad;
};

// ids / v: the row's k entries in LDS. A negative id is an empty entry; an
// id of C or more, an id that stands twice, a NaN or +inf is a bad row.
__device__ Teacher read_teacher(const TopkDistillArgs& a, size_t r, int32_t* ids, float* v,
                                double* ds, int* is) {
  const uint32_t k = a.k;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < k; i += kBlock) {
    ids[i] = a.t_ids[r * k + i];
    v[i] = a.t_logp[r * k + i];
  }
  __syncthreads();
  int bad = 0;
  double mx = -INFINITY;
  for (uint32_t i = 0; i < k; ++i)
    if (ids[i] >= 0) mx = fmax(mx, static_cast<double>(v[i]));
  const double base = a.tail || mx == -INFINITY ? 0.0 : mx;
  double q = 0.0;
  for (uint32_t i = threadIdx.x; i < k; i += kBlock) {
    if (ids[i] < 0) continue;
    if (static_cast<uint64_t>(ids[i]) >= a.C || !(v[i] < INFINITY)) bad = 1;
    for (uint32_t j = 0; j < i; ++j)
      if (ids[j] == ids[i]) bad = 1;
    q += exp(static_cast<double>(v[i]) - base);
  }
  q = block_sum<double, kBlock>(q, ds);
  bad = block_sum<int, kBlock>(bad, is);
  Teacher t;
  t.bad = bad != 0;
  t.Z = a.tail ? 0.0 : q > 0.0 ? base + log(q) : INFINITY;
  t.left = a.tail ? fmax(0.0, 1.0 - q) : 0.0;
  t.S = a.tail ? q + t.left : q > 0.0 ? 1.0 : 0.0;
  bool none = true;
  for (uint32_t i = 0; i < k; ++i) none = none && ids[i] < 0;
  if (none) t.S = t.left = 0.0;  // no list, nothing to learn
  return t;
}

template <int DT>
__global__ __launch_bounds__(kBlock) void distill_fwd_kernel(TopkDistillArgs a, TempScale c2) {
  __shared__ float fs[kBlock / kWave];
  __shared__ double ds[kBlock / kWave];
  __shared__ int is[kBlock / kWave];
  __shared__ int32_t ids[kTopkMax];
  __shared__ float v[kTopkMax];
  __shared__ uint32_t marks[kMarkCols / 32];
  using E = Elem<DT>;
  const size_t r = blockIdx.x;
  const typename E::T* x = static_cast<const typename E::T*>(a.logits) + r * a.stride;
  const uint32_t C = static_cast<uint32_t>(a.C), k = a.k;
  const double inv_T = 1.0 / a.T;
  float* st = a.stats ? a.stats + r * kDistillStats : nullptr;
  if (a.weight && a.weight[r] == 0.0f) {  // a row that does not count
    if (threadIdx.x == 0) {
      a.row_loss[r] = 0.0f;
      if (st)
        for (int i = 0; i < kDistillStats; ++i) st[i] = 0.0f;
    }
    return;
  }
  const Teacher t = read_teacher(a, r, ids, v, ds, is);
  float m = -FLT_MAX;
  for (uint32_t j = threadIdx.x; j < C; j += kBlock) m = fmaxf(m, E::get(x[j]));
  m = block_max<kBlock>(m, fs);
  // The unlisted classes' own maximum, so that a tail far below the listed
  // classes keeps its digits.
  float mt = -FLT_MAX;
  double rest = 0.0;
  for (int pass = 0; pass < 2; ++pass) {
    for (uint32_t c0 = 0; c0 < C; c0 += kMarkCols) {
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < kMarkCols / 32; i += kBlock) marks[i] = 0;
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < k; i += kBlock) {
        const uint32_t at = static_cast<uint32_t>(ids[i]) - c0;
        if (ids[i] >= 0 && at < kMarkCols) atomicOr(&marks[at / 32], 1u << (at % 32));
      }
      __syncthreads();
      for (uint32_t j = c0 + threadIdx.x; j < C && j < c0 + kMarkCols; j += kBlock) {
        if (marks[(j - c0) / 32] >> ((j - c0) % 32) & 1) continue;
        const float xv = E::get(x[j]);
        if (pass == 0) mt = fmaxf(mt, xv);
        else rest += exp2f(scaled(xv, mt, c2));
      }
    }
    if (pass == 0) mt = block_max<kBlock>(mt, fs);
  }
  rest = block_sum<double, kBlock>(rest, ds);
  double in = 0.0;
  for (uint32_t i = threadIdx.x; i < k; i += kBlock)
    if (ids[i] >= 0 && static_cast<uint32_t>(ids[i]) < C)
      in += exp((static_cast<double>(E::get(x[ids[i]])) - m) * inv_T);
  in = block_sum<double, kBlock>(in, ds);
  const double log_rest = rest > 0.0 ? (static_cast<double>(mt) - m) * inv_T + log(rest) : rest != rest ? rest : -INFINITY;
  const double s = in + exp(log_rest);
  const double ls = log(s);
  const bool bad = t.bad || s != s, empty = s == 0.0;
  // No unmasked class outside the list: nothing is left for the teacher's rest.
  const double left = rest == 0.0 ? 0.0 : t.left;
  const double S = t.S - (t.left - left);
  double L = 0.0;
  for (uint32_t i = threadIdx.x; i < k; i += kBlock) {
    if (ids[i] < 0 || bad || empty) continue;
    const double lq = static_cast<double>(v[i]) - t.Z;
    if (lq == -INFINITY) continue;
    L += exp(lq) * (lq - ((static_cast<double>(E::get(x[ids[i]])) - m) * inv_T - ls));
  }
  L = block_sum<double, kBlock>(L, ds);
  if (left > 0.0) L += left * (log(left) - (log_rest - ls));
  if (empty) L = S > 0.0 ? INFINITY : 0.0;
  if (bad) L = __builtin_nan("");
  if (threadIdx.x != 0) return;
  a.row_loss[r] = static_cast<float>(L);
  if (!st) return;
  // Unlisted classes: p_j (S - q_t / p_t) as sign * exp((x_j - m) / T + lt).
  const double ct = S - (left > 0.0 ? left / exp(log_rest - ls) : 0.0);
  st[0] = bad ? __builtin_nanf("") : empty ? 0.0f : m;
  st[1] = static_cast<float>(empty ? 0.0 : 1.0 / s);
  st[2] = static_cast<float>(empty ? -INFINITY
                             : ct == -INFINITY || ct < -1e300 ? log(left) - log_rest
                                                             : log(fabs(ct)) - ls) *
          static_cast<float>(M_LOG2E);
  st[3] = ct < 0.0 ? -1.0f : 1.0f;
  st[4] = empty ? INFINITY : static_cast<float>(t.Z);
  st[5] = empty ? 0.0f : static_cast<float>(S);
  st[6] = st[7] = 0.0f;
}

template <int DT>
__global__ __launch_bounds__(kBlock) void distill_bwd_kernel(TopkDistillArgs a, TempScale c2) {
  __shared__ int32_t ids[kTopkMax];
  __shared__ uint32_t marks[kMarkCols / 32];
  using E = Elem<DT>;
  const size_t r = blockIdx.x;
  const typename E::T* x = static_cast<const typename E::T*>(a.logits) + r * a.stride;
  typename E::T* dx = static_cast<typename E::T*>(a.dlogits) + r * a.dstride;
  const uint32_t C = static_cast<uint32_t>(a.C), k = a.k;
  const float wr = a.weight ? a.weight[r] : static_cast<float>(1.0 / static_cast<double>(a.N));
  if (wr == 0.0f) {
    for (uint32_t j = threadIdx.x; j < C; j += kBlock) dx[j] = E::put(0.0f);
    return;
  }
  const float* st = a.stats + r * kDistillStats;
  const float m = st[0], inv_s = st[1], lt = st[2], Z = st[4], S = st[5];
  const float W = static_cast<float>(static_cast<double>(wr) * (a.seed ? a.seed[0] : 1.0f) / a.T);
  const float Wt = W * st[3];
  for (uint32_t i = threadIdx.x; i < k; i += kBlock) ids[i] = a.t_ids[r * k + i];
  for (uint32_t c0 = 0; c0 < C; c0 += kMarkCols) {
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kMarkCols / 32; i += kBlock) marks[i] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < k; i += kBlock) {
      const uint32_t at = static_cast<uint32_t>(ids[i]) - c0;
      if (ids[i] >= 0 && at < kMarkCols) atomicOr(&marks[at / 32], 1u << (at % 32));
    }
    __syncthreads();
    for (uint32_t j = c0 + threadIdx.x; j < C && j < c0 + kMarkCols; j += kBlock)
      if (!(marks[(j - c0) / 32] >> ((j - c0) % 32) & 1))
        dx[j] = E::put(Wt * exp2f(scaled(E::get(x[j]), m, c2) + lt));
  }
  for (uint32_t i = threadIdx.x; i < k; i += kBlock) {
    const int32_t j = ids[i];
    if (j < 0 || static_cast<uint32_t>(j) >= C) continue;
    const float p = exp2f(scaled(E::get(x[j]), m, c2)) * inv_s;
    dx[j] = E::put(W * (S * p - expf(a.t_logp[r * k + i] - Z)));
  }
}

// loss = sum of w_r L_r in row order, one workgroup.
__global__ __launch_bounds__(kBlock) void distill_loss_kernel(const float* __restrict__ row_loss,
                                                              const float* __restrict__ weight,
                                                              size_t N, float* __restrict__ loss) {
  __shared__ double ds[kBlock / kWave];
  double acc = 0.0;
  for (size_t r = threadIdx.x; r < N; r += kBlock) {
    const double w = weight ? static_cast<double>(weight[r]) : 1.0 / static_cast<double>(N);
    if (w != 0.0) acc += w * row_loss[r];
  }
  acc = block_sum<double, kBlock>(acc, ds);
  if (threadIdx.x == 0) *loss = static_cast<float>(acc);
}

#define DTYPE_LAUNCH(kernel, dtype, ...)                                          \
  do {                                                                            \
    if ((dtype) == kF32) hipLaunchKernelGGL(kernel<kF32>, __VA_ARGS__);           \
    else if ((dtype) == kBF16) hipLaunchKernelGGL(kernel<kBF16>, __VA_ARGS__);    \
    else hipLaunchKernelGGL(kernel<kF16>, __VA_ARGS__);                           \
  } while (0)

#define NT_LAUNCH(kernel, nt_, dtype, grid, ...)                                              \
  do {                                                                                        \
    if ((dtype) == kF32)                                                                      \
      hipLaunchKernelGGL((kernel<kF32, nt_>), grid, dim3(nt_), 0, c.stream, __VA_ARGS__);     \
    else if ((dtype) == kBF16)                                                                \
      hipLaunchKernelGGL((kernel<kBF16, nt_>), grid, dim3(nt_), 0, c.stream, __VA_ARGS__);    \
    else                                                                                      \
      hipLaunchKernelGGL((kernel<kF16, nt_>), grid, dim3(nt_), 0, c.stream, __VA_ARGS__);     \
  } while (0)

// Threads per row.
int ScoreThreads(const TokenScoreArgs& a) {
  if (a.C <= 1024 && a.k <= 32) return 64;
  return a.N >= 512 ? 256 : 1024;
}

}  // namespace

uint64_t TokenScoreScratch(uint64_t, uint64_t, int, uint64_t) { return 0; }
uint64_t TopkDistillScratch(uint64_t N, uint64_t, int, uint64_t) {
  return N * kDistillStats * sizeof(float);
}

Status TokenScoreFwd(const TokenScoreArgs& a, const Ctx& c) {
  const TempScale c2 = ScaleOf(a.T);
  const int nt = StreamPolicy(a.N * a.C * (a.dtype == kF32 ? 4 : 2)) ? 1 : 0;
  const int threads = ScoreThreads(a);
  const dim3 grid(static_cast<unsigned>(a.N));
  if (threads == 64) NT_LAUNCH(score_fwd_kernel, 64, a.dtype, grid, a, c2, nt);
  else if (threads == 256) NT_LAUNCH(score_fwd_kernel, 256, a.dtype, grid, a, c2, nt);
  else NT_LAUNCH(score_fwd_kernel, 1024, a.dtype, grid, a, c2, nt);
  return LaunchStatus("TokenLogprobs");
}

Status TokenScoreBwd(const TokenScoreBwdArgs& a, const Ctx& c) {
  const TempScale c2 = ScaleOf(a.T);
  DTYPE_LAUNCH(score_bwd_kernel, a.dtype, dim3(static_cast<unsigned>(a.N)), dim3(kBlock), 0,
               c.stream, a, c2);
  return LaunchStatus("TokenLogprobsBwd");
}

Status TopkDistillFwd(const TopkDistillArgs& a, const Ctx& c) {
  const TempScale c2 = ScaleOf(a.T);
  DTYPE_LAUNCH(distill_fwd_kernel, a.dtype, dim3(static_cast<unsigned>(a.N)), dim3(kBlock), 0,
               c.stream, a, c2);
  if (a.loss)
    hipLaunchKernelGGL(distill_loss_kernel, dim3(1), dim3(kBlock), 0, c.stream, a.row_loss,
                       a.weight, static_cast<size_t>(a.N), a.loss);
  return LaunchStatus("TopkDistill");
}

Status TopkDistillBwd(const TopkDistillArgs& a, const Ctx& c) {
  const TempScale c2 = ScaleOf(a.T);
  DTYPE_LAUNCH(distill_bwd_kernel, a.dtype, dim3(static_cast<unsigned>(a.N)), dim3(kBlock), 0,
               c.stream, a, c2);
  return LaunchStatus("TopkDistillBwd");
}

Status TopkDistillFwdBwd(const TopkDistillArgs& a, const Ctx& c) {
  TopkDistillArgs b = a;
  b.stats = static_cast<float*>(a.scratch);
  if (Status s = TopkDistillFwd(b, c); !s) return s;
  return TopkDistillBwd(b, c);
}

}  // namespace seeml_hip
