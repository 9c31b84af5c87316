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

#include <algorithm>
#include <cfloat>
#include <cmath>

namespace seeml_hip {

namespace {

constexpr float kLow = -1e30f;  // finite stand-in for (-inf) * 0 products
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));

// log2(e) / T as a sum of two floats, both positive: a difference of logits
// times the pair is right to half a unit in the last place, where one float
// would lean by its own rounding, the same way on every class.
struct TempScale {
  float hi, lo;
  double inv_T;
};
TempScale ScaleOf(double T) {
  const double c = M_LOG2E / T;
  TempScale s;
  s.hi = static_cast<float>(c);
  if (static_cast<double>(s.hi) > c) s.hi = std::nextafterf(s.hi, 0.0f);
  s.lo = fmaxf(static_cast<float>(c - s.hi), FLT_MIN);  // never 0: -inf * 0
  s.inv_T = 1.0 / T;
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
  // With the classes of `out` (a bit each) at -inf.
  static __device__ __forceinline__ raw masked(raw r, uint32_t out) {
    if constexpr (DT == kF32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = out >> i & 1 ? 0xFF800000u : r[i];
    } else {
      constexpr uint32_t inf = DT == kBF16 ? 0xFF80u : 0xFC00u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        r[i] = out >> (2 * i) & 1 ? (r[i] & 0xFFFF0000u) | inf : r[i];
        r[i] = out >> (2 * i + 1) & 1 ? (r[i] & 0xFFFFu) | inf << 16 : r[i];
      }
    }
    return r;
  }
  static __device__ __forceinline__ raw pack(const float* v) {
    raw r;
    if constexpr (DT == kF32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(v[i]);
    } else {
      typedef T t8 __attribute__((ext_vector_type(8)));
      t8 h;
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = E::put(v[i]);
      r = __builtin_bit_cast(raw, h);
    }
    return r;
  }
  static __device__ __forceinline__ void store(T* dx, uint32_t j, const float* v, bool nt) {
    const raw r = pack(v);
    rawu* p = reinterpret_cast<rawu*>(dx + static_cast<size_t>(j) * V);
    if (nt) __builtin_nontemporal_store(static_cast<rawu>(r), p);
    else *p = r;
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

template <int n>
__device__ __forceinline__ float max_of(const float* v) {
  float m = v[0];
#pragma unroll
  for (int i = 1; i < n; ++i) m = fmaxf(m, v[i]);
  return m;
}

// Keeps a packed vector packed: what was unpacked from it before is unpacked
// again instead of held in twice the registers.
template <typename R>
__device__ __forceinline__ void keep_packed(R& r) {
  asm volatile("" : "+v"(r));
}

__device__ __forceinline__ float exp2_raw(float v) { return __builtin_amdgcn_exp2f(v); }

// e^y for y <= 0 in 64 bits, to about 1e-11 of itself, and 0 far below: a row's
// few 64-bit terms are computed by one wavefront and were most of a short row's
// time with the library's last-bit functions. y = n ln 2 + r, the series in r.
__device__ __forceinline__ double exp_below(double y) {
  y = fmax(y, -800.0);
  const double n = rint(y * M_LOG2E);
  const double r = fma(n, -M_LN2, y);  // |r| < 0.35, off by 1e-13 at most
  double p = 1.0 / 3628800;
  p = fma(p, r, 1.0 / 362880);
  p = fma(p, r, 1.0 / 40320);
  p = fma(p, r, 1.0 / 5040);
  p = fma(p, r, 1.0 / 720);
  p = fma(p, r, 1.0 / 120);
  p = fma(p, r, 1.0 / 24);
  p = fma(p, r, 1.0 / 6);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return ldexp(p, static_cast<int>(n));
}
// ln v for v in float's range: the 32-bit logarithm, and one Newton step on
// e^-y v = 1, which squares its error.
__device__ __forceinline__ double log_near(double v) {
  const double y = __builtin_amdgcn_logf(static_cast<float>(v)) * M_LN2;
  const double e = y > 0.0 ? exp_below(-y) * v : v / exp_below(y);
  return y + (e - 1.0);
}

// A softmax's running sums: s = sum e, w = sum e d (where kW), with e = 2^d, d
// the scaled difference from m. m starts at the lowest finite value, so that masked
// classes add 0 and no difference of infinities arises; a NaN or +inf turns s
// into NaN.
struct Online {
  float m = -FLT_MAX;
  double s = 0.0, w = 0.0;
  __device__ __forceinline__ void raise(float to, TempScale c) {
    if (to > m) {
      const double d = fmaxf(scaled(m, to, c), kLow), f = exp2_raw(static_cast<float>(d));
      w = (w + s * d) * f;
      s *= f;
      m = to;
    }
  }
  // n values of maximum `top`: summed in 32 bits, and their sums in 64, so that
  // the error does not grow with the row.
  template <int n, bool kW = true>
  __device__ __forceinline__ void add(const float* v, float top, TempScale c) {
    raise(top, c);
    float sb = 0.0f, wb = 0.0f;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float d = scaled(v[i], m, c), e = exp2_raw(d);
      sb += e;
      if constexpr (kW) wb = fmaf(e, fmaxf(d, kLow), wb);
    }
    s += sb;
    w += wb;
  }
};

// Reductions over a wavefront by data-parallel moves within and across its rows
// of 16 lanes (a shuffle through LDS takes ten times as long), in a fixed order;
// every lane gets the result. `none` is what leaves the others as they are.
template <int ctrl, int rows>
__device__ __forceinline__ uint32_t moved(uint32_t none, uint32_t v) {
  return __builtin_amdgcn_update_dpp(none, v, ctrl, rows, 0xF, false);
}
template <int ctrl, int rows>
__device__ __forceinline__ float moved(float none, float v) {
  return __uint_as_float(moved<ctrl, rows>(__float_as_uint(none), __float_as_uint(v)));
}
template <int ctrl, int rows>
__device__ __forceinline__ double moved(double none, double v) {
  const uint64_t n = __double_as_longlong(none), b = __double_as_longlong(v);
  const uint64_t lo = moved<ctrl, rows>(static_cast<uint32_t>(n), static_cast<uint32_t>(b));
  const uint64_t hi =
      moved<ctrl, rows>(static_cast<uint32_t>(n >> 32), static_cast<uint32_t>(b >> 32));
  return __longlong_as_double(static_cast<long long>(hi << 32 | lo));
}
template <typename T>
__device__ __forceinline__ T last_lane(T v) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(
        T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), kWave - 1));
  } else {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(b), kWave - 1);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(b >> 32), kWave - 1);
    return __builtin_bit_cast(T, static_cast<uint64_t>(hi) << 32 | lo);
  }
}
template <typename T, typename F>
__device__ __forceinline__ T over_wave(T none, T v, F f) {
  v = f(v, moved<0x111, 0xF>(none, v));  // from 1 lane below, of the same row
  v = f(v, moved<0x112, 0xF>(none, v));  // 2
  v = f(v, moved<0x114, 0xF>(none, v));  // 4
  v = f(v, moved<0x118, 0xF>(none, v));  // 8
  v = f(v, moved<0x142, 0xA>(none, v));  // rows 1 and 3 from the last lane of 0 and 2
  v = f(v, moved<0x143, 0xC>(none, v));  // rows 2 and 3 from the last lane of 1
  return last_lane(v);
}
template <typename T>
__device__ __forceinline__ T lanes_sum(T v) {
  return over_wave(T(0), v, [](T x, T y) { return x + y; });
}
__device__ __forceinline__ float lanes_max(float v) {
  return over_wave(-INFINITY, v, [](float x, float y) { return fmaxf(x, y); });
}
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  return over_wave(0u, v, [](uint32_t x, uint32_t y) { return x > y ? x : y; });
}

struct RowSums {
  float m;
  double s, w;
};
// The lanes' sums joined.
__device__ __forceinline__ RowSums join_lanes(const RowSums& o, TempScale c) {
  RowSums t;
  t.m = lanes_max(o.m);
  const float d = fmaxf(scaled(o.m, t.m, c), kLow);
  const double f = exp2_raw(d);
  t.s = lanes_sum(o.s * f);
  t.w = lanes_sum((o.w + o.s * d) * f);
  return t;
}
// The threads' sums joined: each wavefront's, then the wavefronts'. Every
// thread gets them.
template <int NT>
__device__ __forceinline__ RowSums join(const Online& o, TempScale c, RowSums* scratch) {
  const RowSums t = join_lanes({o.m, o.s, o.w}, c);
  if constexpr (NT == kWave) return t;
  const int lane = threadIdx.x % kWave;
  if (lane == 0) scratch[threadIdx.x / kWave] = t;
  __syncthreads();
  return join_lanes(lane < NT / kWave ? scratch[lane] : RowSums{-FLT_MAX, 0.0, 0.0}, c);
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
  uint32_t best[NT];  // the threads' maxima, ordered
  uint16_t list[kGroups * NT];
  int wave[NT / kWave];
  uint32_t n_list, n_cand, bound;
};

// A value that at least k of `sets` maxima reach, near the k-th largest; the
// least finite one if fewer than k hold an unmasked class. For one wavefront,
// n maxima a lane.
constexpr uint32_t kLeast = 0x00800000u;  // ordered(-FLT_MAX)
template <int n>
__device__ __forceinline__ uint32_t bound_of(const uint32_t (&key)[n], uint32_t k, uint32_t slack) {
  uint32_t hi = key[0];
#pragma unroll
  for (int i = 1; i < n; ++i) hi = key[i] > hi ? key[i] : hi;
  hi = lanes_max(hi);
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
      if (c <= k + slack) break;
    } else {
      hi = mid;
    }
  }
  return lo;
}
// The same for a workgroup's threads, by its first wavefront. Beyond 256
// threads, threads share a set: the bound is a little lower, the search shorter.
template <int NT>
__device__ __forceinline__ void find_bound(Select<NT>& sel, uint32_t k) {
  constexpr int n = NT < 256 ? NT / kWave : 4, shared_by = NT / (n * kWave);
  if (threadIdx.x >= kWave) return;
  uint32_t key[n];
#pragma unroll
  for (int i = 0; i < n; ++i) {
    key[i] = 0;
#pragma unroll
    for (int j = 0; j < shared_by; ++j) {
      const uint32_t o = sel.best[(i * shared_by + j) * kWave + threadIdx.x];
      key[i] = o > key[i] ? o : key[i];
    }
  }
  const uint32_t th = bound_of(key, k, k / 4 + 2);
  if (threadIdx.x == 0) sel.bound = th;
}
// A closer bound from the maxima of the groups that reach the first one, which
// are finer sets, and the list without the groups below it. By the first
// wavefront; a long list (ties) stays as it is.
template <int NT>
__device__ __forceinline__ void refine_bound(Select<NT>& sel, uint32_t k) {
  constexpr int n = 4;
  const uint32_t have = sel.n_list, lane = threadIdx.x;
  if (have <= k + k / 8 || have > n * kWave) return;
  uint32_t key[n], kept = 0;
  uint16_t id[n];
#pragma unroll
  for (int i = 0; i < n; ++i) {
    const bool in = i * kWave + lane < have;
    id[i] = in ? sel.list[i * kWave + lane] : 0;
    key[i] = in ? ordered(sel.group[id[i]]) : 0;
  }
  const uint32_t th = bound_of(key, k, k / 16 + 1);
#pragma unroll
  for (int i = 0; i < n; ++i) {
    const uint64_t in = __ballot(key[i] >= th);
    if (key[i] >= th) sel.list[kept + __popcll(in & ((uint64_t{1} << lane) - 1))] = id[i];
    kept += static_cast<uint32_t>(__popcll(in));
  }
  if (lane == 0) {
    sel.n_list = kept;
    sel.bound = th;
  }
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
// counting over the row each time (once where the ties are at the bound, up to
// 32 times elsewhere), then takes the classes above it and the first of those
// equal to it. 2048 rows of 32000 float32, k 128, us: 64 with a vocabulary's
// logits, 122 with all of them equal, 1390 with 300 neighbouring classes over one
// floor value: they lie in fewer threads' sets than k, so that the bound is the
// least value and the whole row reaches it.
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
// sel.cand. `groups` groups of `each` vectors a thread are the sweep's.
// `meanwhile` runs beside the search for the bound.
template <int DT, int NT, typename F>
__device__ __forceinline__ void select_top(const Row<DT>& row, uint32_t C, uint32_t k, float top,
                                           uint32_t groups, uint32_t each, float best,
                                           Select<NT>& sel, F meanwhile) {
  constexpr int V = Row<DT>::V;
  const uint32_t nv = C / V;
  sel.best[threadIdx.x] = ordered(best);
  if (threadIdx.x == 0) sel.n_list = sel.n_cand = 0;
  __syncthreads();
  find_bound(sel, k);
  meanwhile();
  __syncthreads();
  uint32_t th = sel.bound;
  if (ordered(best) >= th)
    for (uint32_t g = 0; g < groups; ++g)
      if (ordered(sel.group[g * NT + threadIdx.x]) >= th)
        sel.list[atomicAdd(&sel.n_list, 1u)] = static_cast<uint16_t>(g * NT + threadIdx.x);
  __syncthreads();
  if (k > 64) {
    if (threadIdx.x < kWave) refine_bound(sel, k);
    __syncthreads();
    th = sel.bound;
  }
  const auto take = [&](float v, uint32_t col) {
    if (ordered(v) >= th) {
      const uint32_t at = atomicAdd(&sel.n_cand, 1u);
      if (at < Select<NT>::kCand) sel.cand[at] = key_of(v, col);
    }
  };
  const uint32_t n = sel.n_list * each;
  for (uint32_t i = threadIdx.x; i < n; i += NT) {
    const uint32_t id = sel.list[i / each], at = i % each;
    const uint32_t j = ((id / NT) * each + at) * NT + id % NT;
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

// A row's parts in scratch, where rows are too few to fill the chip: its sums,
// and its k likeliest classes' keys in order (0 behind the last).
struct ScorePart {
  RowSums sums;
};
__host__ __device__ inline ScorePart* score_parts(void* scratch) {
  return static_cast<ScorePart*>(scratch);
}
__host__ __device__ inline uint64_t* score_keys(void* scratch, size_t parts) {
  return reinterpret_cast<uint64_t*>(static_cast<ScorePart*>(scratch) + parts);
}

// What is known of a whole row: log s, and its short outputs. For one
// wavefront; t and xt are the target and its logit.
__device__ __forceinline__ double finish_score(const TokenScoreArgs& a, size_t r, const RowSums& q,
                                               int32_t t, float xt, double inv_T) {
  const float nan = __builtin_nanf("");
  const bool bad = q.s != q.s, empty = q.s == 0.0;
  const double ls = log_near(q.s);
  if (threadIdx.x % kWave != 0) return ls;
  const float H = bad ? nan : empty ? 0.0f : static_cast<float>(ls - q.w * M_LN2 / q.s);
  if (a.logp) {
    float lp = 0.0f;
    if (t >= 0)
      lp = static_cast<uint64_t>(t) >= a.C || bad ? nan
           : empty                                ? -INFINITY
                   : static_cast<float>((static_cast<double>(xt) - q.m) * inv_T - ls);
    a.logp[r] = lp;
  }
  if (a.entropy) a.entropy[r] = H;
  if (a.stats)
    *reinterpret_cast<float4u*>(a.stats + r * kScoreStats) =
        float4u{bad ? nan : empty ? 0.0f : q.m,
                bad ? nan : empty ? INFINITY : static_cast<float>(ls), H,
                bad ? nan : empty ? 0.0f : static_cast<float>(1.0 / q.s)};
  return ls;
}

// Ranks the n keys of `cand`, the k largest among them, and hands each of the
// first k with its rank to `put`.
template <int NT, typename F>
__device__ __forceinline__ void rank_keys(const uint64_t* cand, uint32_t n, uint32_t k, F put) {
  for (uint32_t i = threadIdx.x; i < n; i += NT) {
    const uint64_t key = cand[i];
    uint32_t rank = 0;
    for (uint32_t j = 0; j < n; ++j) rank += cand[j] > key ? 1 : 0;
    if (rank < k) put(rank, key);
  }
}

struct TopOut {
  int32_t* ids;
  float* lps;
  float m;
  double inv_T, ls;
  __device__ __forceinline__ void operator()(uint32_t rank, uint64_t key) const {
    const uint32_t o = static_cast<uint32_t>(key >> 32);
    const float v = __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
    ids[rank] = static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(key));
    lps[rank] = static_cast<float>((static_cast<double>(v) - m) * inv_T - ls);
  }
};

// A row, or one of its `parts` ranges of `each` vectors (the last with the
// classes behind the last whole vector). One read of the logits carries the
// maximum, both sums and the maxima of the selection; per logit 13 vector
// instructions, 15 with a list of 32, where HBM's rate leaves 28 for a float32
// and 14 for a 16-bit one. float32 is bound by HBM: 8192 rows of 32000 195 us
// without a list, 5.4 TB/s; 205 with 32 classes, whose search and second reads a
// row's workgroup does between its sweeps. 16 bits are bound by issue (the vector
// units are busy throughout): bf16 121 us, 4.3 TB/s, and 128. Few rows are bound by
// latency: 1 row of 32000, k 20, 8.9 us, of which an empty launch is 2, the sweep
// and its join 4, the selection 3.
template <int DT, int NT>
__global__ __launch_bounds__(NT) void score_fwd_kernel(TokenScoreArgs a, TempScale c,
                                                       uint32_t parts, uint32_t each, int nt) {
  __shared__ Select<NT> sel;
  __shared__ RowSums sums[NT / kWave];
  __shared__ double log_sum;
  using E = Elem<DT>;
  constexpr int V = Row<DT>::V;
  const size_t r = blockIdx.x / parts;
  const uint32_t part = blockIdx.x % parts, first = part * each * V;
  const uint32_t k = a.k;
  const uint32_t C = part + 1 < parts ? each * V : static_cast<uint32_t>(a.C) - first;
  const Row<DT> row{static_cast<const typename E::T*>(a.logits) + r * a.stride + first};
  const uint32_t nv = C / V;
  const uint32_t batches = (nv + NT * kBatch - 1) / (NT * kBatch);
  // Vectors a group: whole batches, or for a long list as few as kGroups allow,
  // since each group that is read again brings a line of memory a vector (777
  // rows of 10007 f16, us with k 64 and 128: 13.1 and 15.6 against 14.0 and
  // 21.8; with k 8 the finer groups' stores cost more, 11.6 against 10.9).
  const uint32_t unit = k > 32 && batches <= kGroups / 4   ? 1
                        : k > 32 && batches <= kGroups / 2 ? 2
                            : kBatch * max((batches + kGroups - 1) / kGroups, 1u);
  const uint32_t groups = (batches * kBatch + unit - 1) / unit;
  int32_t t = -1;
  float xt = 0.0f;
  // The last wavefront finishes the row while the first looks for the bound.
  const bool ends = threadIdx.x >= NT - kWave;
  if (ends && parts == 1 && a.logp) {
    t = a.targets[r];
    if (t >= 0 && static_cast<uint32_t>(t) < C) xt = E::get(row.x[t]);
  }
  Online o;
  float best = -INFINITY, group = -INFINITY;
  for (uint32_t b = 0; b < batches; ++b) {
    const uint32_t j0 = b * (kBatch * NT) + threadIdx.x;
    typename Row<DT>::raw raw[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) raw[u] = row.load(min(j0 + u * NT, nv - 1), nt);
    float tops[kBatch];
    if ((b + 1) * (kBatch * NT) <= nv) {
      float v[kBatch * V];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        Row<DT>::unpack(raw[u], v + u * V);
        tops[u] = max_of<V>(v + u * V);
      }
      o.add<kBatch * V>(v, max_of<kBatch>(tops), c);
    } else {  // the last one: whole wavefronts have nothing left
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        tops[u] = -INFINITY;
        if (j0 + u * NT >= nv) continue;
        float v[V];
        Row<DT>::unpack(raw[u], v);
        tops[u] = max_of<V>(v);
        o.add<V>(v, tops[u], c);
      }
    }
    if (!k) continue;
    best = fmaxf(best, max_of<kBatch>(tops));
    float* at = sel.group + threadIdx.x;
    if (unit == 1) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) at[(b * kBatch + u) * NT] = tops[u];
    } else if (unit == 2) {
#pragma unroll
      for (int u = 0; u < kBatch; u += 2)
        at[(b * kBatch + u) / 2 * NT] = fmaxf(tops[u], tops[u + 1]);
    } else {
      group = fmaxf(group, max_of<kBatch>(tops));
      if ((b + 1) * kBatch % unit == 0 || b + 1 == batches) {
        at[b * kBatch / unit * NT] = group;
        group = -INFINITY;
      }
    }
  }
  if (threadIdx.x < C - nv * V) {
    const float v = E::get(row.x[nv * V + threadIdx.x]);
    o.add<1>(&v, v, c);
  }
  const RowSums q = join<NT>(o, c, sums);
  const bool fit = q.s > 0.0;  // neither bad nor all masked
  if (parts > 1) {
    if (threadIdx.x == 0) score_parts(a.scratch)[blockIdx.x].sums = q;
  } else if (ends && !k) {
    finish_score(a, r, q, t, xt, c.inv_T);
  }
  if (!k) return;
  uint32_t n = 0;
  const auto finish = [&] {
    if (!ends || parts > 1) return;
    const double ls = finish_score(a, r, q, t, xt, c.inv_T);
    if (threadIdx.x == NT - 1) log_sum = ls;
  };
  if (!fit) finish();
  if (fit) {
    select_top<DT, NT>(row, C, k, q.m, groups, unit, best, sel, finish);
    n = sel.n_cand;
  }
  if (parts > 1) {
    uint64_t* keys = score_keys(a.scratch, gridDim.x) + static_cast<size_t>(blockIdx.x) * k;
    // The row's classes, not the part's.
    rank_keys<NT>(sel.cand, n, k, [&](uint32_t rank, uint64_t key) { keys[rank] = key - first; });
    for (uint32_t i = n + threadIdx.x; i < k; i += NT) keys[i] = 0;
    return;
  }
  const TopOut out{a.top_ids + r * k, a.top_logp + r * k, q.m, c.inv_T, log_sum};
  rank_keys<NT>(sel.cand, n, k, out);
  for (uint32_t i = n + threadIdx.x; i < k; i += NT) {
    out.ids[i] = -1;
    out.lps[i] = q.s != q.s ? __builtin_nanf("") : -INFINITY;
  }
}

// Joins a row's parts. At most kWave parts and kJoinKeys keys.
constexpr int kJoin = 256;
constexpr uint32_t kJoinKeys = 1024;
template <int DT>
__global__ __launch_bounds__(kJoin) void score_join_kernel(TokenScoreArgs a, TempScale c,
                                                           uint32_t parts) {
  __shared__ uint64_t keys[kJoinKeys], cand[kJoinKeys];
  __shared__ double log_sum;
  __shared__ uint32_t bound, n_cand;
  using E = Elem<DT>;
  const size_t r = blockIdx.x;
  const uint32_t k = a.k, n_keys = parts * k;
  const uint64_t* from = score_keys(a.scratch, parts * gridDim.x) + r * n_keys;
  for (uint32_t i = threadIdx.x; i < n_keys; i += kJoin) keys[i] = from[i];
  const uint32_t lane = threadIdx.x % kWave;
  RowSums part{-FLT_MAX, 0.0, 0.0};
  if (lane < parts) part = score_parts(a.scratch)[r * parts + lane].sums;
  const RowSums q = join_lanes(part, c);
  if (threadIdx.x == 0) n_cand = 0;
  __syncthreads();
  if (threadIdx.x < kWave) {
    int32_t t = -1;
    float xt = 0.0f;
    if (a.logp) {
      t = a.targets[r];
      if (t >= 0 && static_cast<uint64_t>(t) < a.C)
        xt = E::get(static_cast<const typename E::T*>(a.logits)[r * a.stride + t]);
    }
    const double ls = finish_score(a, r, q, t, xt, c.inv_T);
    if (threadIdx.x == 0) log_sum = ls;
  } else if (threadIdx.x < 2 * kWave && k) {
    uint32_t key[kJoinKeys / kWave];
#pragma unroll
    for (uint32_t i = 0; i < kJoinKeys / kWave; ++i)
      key[i] = i * kWave + lane < n_keys ? static_cast<uint32_t>(keys[i * kWave + lane] >> 32) : 0;
    const uint32_t th = bound_of(key, k, k / 4 + 2);
    if (lane == 0) bound = th;
  }
  if (!k) return;
  __syncthreads();
  const bool fit = q.s > 0.0;
  for (uint32_t i = threadIdx.x; fit && i < n_keys; i += kJoin)
    if (static_cast<uint32_t>(keys[i] >> 32) >= bound) cand[atomicAdd(&n_cand, 1u)] = keys[i];
  __syncthreads();
  const uint32_t n = n_cand;
  const TopOut out{a.top_ids + r * k, a.top_logp + r * k, q.m, c.inv_T, log_sum};
  rank_keys<kJoin>(cand, n, k, out);
  for (uint32_t i = n + threadIdx.x; i < k; i += kJoin) {
    out.ids[i] = -1;
    out.lps[i] = q.s != q.s ? __builtin_nanf("") : -INFINITY;
  }
}

// One workgroup per kBatch vectors of each of its threads; the last one of a
// row also takes the classes behind the last whole vector. Bound by HBM: 4096
// rows of 32000 float32 201 us, 5.2 TB/s, and 184 right behind the forward, which
// leaves logits in the memory-side cache; bf16 105, 5.0 TB/s.
template <int DT, int NT>
__global__ __launch_bounds__(NT) void score_bwd_kernel(TokenScoreBwdArgs a, TempScale c,
                                                       uint32_t parts, int nt) {
  using E = Elem<DT>;
  constexpr int V = Row<DT>::V;
  const size_t r = blockIdx.x / parts;
  const uint32_t part = blockIdx.x % parts;
  const Row<DT> row{static_cast<const typename E::T*>(a.logits) + r * a.stride};
  typename E::T* dx = static_cast<typename E::T*>(a.dlogits) + r * a.dstride;
  const uint32_t C = static_cast<uint32_t>(a.C), nv = C / V;
  const uint32_t j0 = part * (kBatch * NT) + threadIdx.x;
  typename Row<DT>::raw raw[kBatch];
  if (nv)
#pragma unroll
    for (int u = 0; u < kBatch; ++u) raw[u] = row.load(min(j0 + u * NT, nv - 1), nt);
  const float4u st = *reinterpret_cast<const float4u*>(a.stats + r * kScoreStats);
  const int32_t t = a.targets ? a.targets[r] : -1;
  const float ls = st[1], H = st[2], inv_s = st[3];
  const bool empty = ls == INFINITY;
  const bool out = t >= 0 && static_cast<uint32_t>(t) >= C && !empty;
  const float m = out ? __builtin_nanf("") : st[0];
  // A gradient over T may leave float32's range where p and a class's share in it
  // do not: then 1 / T is the last factor.
  float up = a.dlogp && t >= 0 ? a.dlogp[r] : 0.0f;
  float bonus = a.dentropy ? a.dentropy[r] : 0.0f;
  float last = static_cast<float>(c.inv_T);
  if (empty) up = bonus = 0.0f;
  if (fmaxf(fabsf(up), fabsf(bonus)) * last <= 1e36f) {
    up *= last;
    bonus *= last;
    last = 1.0f;
  }
  // -p up - bonus p (ln p + H). ln p is above -150 where p is not 0; p comes
  // first, so that a class without it has no gradient at any temperature.
  const float ln2 = static_cast<float>(M_LN2), shift = H - ls;
  const auto grad = [&](float x) {
    const float d = scaled(x, m, c), p = exp2_raw(d) * inv_s;
    return fmaf(-bonus, p * fmaxf(fmaf(d, ln2, shift), -1e4f), -up * p);
  };
#pragma unroll
  for (int u = 0; u < kBatch; ++u) {
    const uint32_t j = j0 + u * NT;
    if (j >= nv) continue;
    float v[V];
    Row<DT>::unpack(raw[u], v);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = grad(v[e]);
    if (static_cast<uint32_t>(t) / V == j)
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (static_cast<uint32_t>(t) % V == e) v[e] += up;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] *= last;
    Row<DT>::store(dx, j, v, nt);
  }
  if (part + 1 == parts && threadIdx.x < C - nv * V) {
    const uint32_t j = nv * V + threadIdx.x;
    float g = grad(E::get(row.x[j]));
    if (static_cast<int32_t>(j) == t) g += up;
    dx[j] = E::put(g * last);
  }
}

// ---- distillation -----------------------------------------------------------
//
// The listed classes are marked in a bitmap in LDS and left out of the sweep,
// whose maximum and sum are then the unlisted classes' own: a tail far below
// the listed classes keeps its digits, where the difference 1 - sum p would
// lose them all. One wavefront takes the list (at most two entries a lane) in
// 64 bits; its terms cancel, and are few.

// What a row's list gives, the same in every lane.
struct Listed {
  double S, left;          // sum q + left; the rest's mass
  float base, scale;       // q_i = exp(v_i - base) scale
  double q, q_log_q, q_x;  // sums of q, q ln q and q (x - m) / T
  double e;                // sum of exp((x - m) / T)
  float m;                 // the listed classes' own maximum
  bool bad;
};

// A lane's entries: an empty one has id -1 and v and x at -inf. sum_list puts q
// in v's place.
struct Entries {
  static constexpr int n = kTopkMax / kWave;
  int32_t id[n];
  float v[n], x[n];
};
template <int DT>
__device__ __forceinline__ Entries read_list(const TopkDistillArgs& a, const Row<DT>& row,
                                             size_t r) {
  Entries l;
#pragma unroll
  for (int i = 0; i < l.n; ++i) {
    const uint32_t at = threadIdx.x % kWave + i * kWave;
    l.id[i] = at < a.k ? max(a.t_ids[r * a.k + at], -1) : -1;
    l.v[i] = l.id[i] >= 0 ? a.t_logp[r * a.k + at] : -INFINITY;
    const bool in = l.id[i] >= 0 && static_cast<uint32_t>(l.id[i]) < static_cast<uint32_t>(a.C);
    l.x[i] = in ? Elem<DT>::get(row.x[l.id[i]]) : -INFINITY;
  }
  return l;
}

// A list may be off by a constant far above what tells its entries apart: only
// differences from its largest value count, which 32 bits hold.
__device__ __forceinline__ Listed sum_list(const TopkDistillArgs& a, Entries& t, double inv_T) {
  constexpr int n = Entries::n;
  float top = -INFINITY, m = -FLT_MAX;
  bool bad = false, any = false;
#pragma unroll
  for (int i = 0; i < n; ++i) {
    if (t.id[i] < 0) continue;
    any = true;
    bad = bad || static_cast<uint32_t>(t.id[i]) >= static_cast<uint32_t>(a.C) ||
          !(t.v[i] < INFINITY) || !(t.x[i] < INFINITY);
    top = fmaxf(top, t.v[i]);
    m = fmaxf(m, t.x[i]);
  }
  Listed l;
  l.m = lanes_max(m);
  const float base = a.tail ? 0.0f : fmaxf(lanes_max(top), -FLT_MAX);
  double q[n], mass = 0.0, e = 0.0;
#pragma unroll
  for (int i = 0; i < n; ++i) {
    q[i] = 0.0;
    if (i * kWave >= a.k) continue;
    // With a tail v is a logarithm of at most 1, or of a little more.
    const double y = static_cast<double>(t.v[i]) - base, up = fmax(y, 0.0);
    q[i] = up > 0.0 ? exp(y) : exp_below(y);
    mass += q[i];
    e += exp_below((static_cast<double>(t.x[i]) - l.m) * inv_T);
  }
  mass = lanes_sum(mass);
  l.e = lanes_sum(e);
  l.bad = __ballot(bad) != 0;
  const bool none = __ballot(any) == 0;
  const double scale = a.tail ? 1.0 : mass > 0.0 ? 1.0 / mass : 0.0;
  const double log_mass = a.tail || !(mass > 0.0) ? 0.0 : log_near(mass);
  l.base = base;
  l.scale = static_cast<float>(scale);
  l.left = a.tail && !none ? fmax(0.0, 1.0 - mass) : 0.0;
  double q_log_q = 0.0, q_x = 0.0;
#pragma unroll
  for (int i = 0; i < n; ++i) {
    q[i] *= scale;
    const double log_q = static_cast<double>(t.v[i]) - base - log_mass;
    t.v[i] = static_cast<float>(q[i]);
    if (!(q[i] > 0.0)) continue;
    q_log_q += q[i] * log_q;
    q_x += q[i] * ((static_cast<double>(t.x[i]) - l.m) * inv_T);
  }
  l.q_log_q = lanes_sum(q_log_q);
  l.q_x = lanes_sum(q_x);
  l.q = mass * scale;
  l.S = l.q + l.left;
  return l;
}

// A row's outcome from its list and the unlisted classes' maximum `mt` and sum
// `rest` of exp((x - mt) / T).
struct Outcome {
  double loss;
  float m, inv_s, mt, coef;  // p = exp((x - m) / T) inv_s;
  float base, scale, S;      // unlisted: gradient coef exp((x - mt) / T)
};
__device__ __forceinline__ Outcome row_outcome(const Listed& l, float mt, double rest, double inv_T,
                                               bool dup) {
  Outcome o;
  const bool bad = l.bad || dup || rest != rest;
  const bool empty = rest == 0.0 && l.e == 0.0;
  // Nothing unmasked outside the list: the rest of the teacher's mass is
  // rounding.
  const double left = rest > 0.0 ? l.left : 0.0, S = l.q + left;
  // (l.m - m) / T and (mt - m) / T: one of them is 0.
  const double gap = (static_cast<double>(l.m) - mt) * inv_T, low = exp_below(-fabs(gap));
  const double dl = fmin(gap, 0.0), dt = fmin(-gap, 0.0);
  const double ft = gap > 0.0 ? low : 1.0;
  const double s = l.e * (gap > 0.0 ? 1.0 : low) + rest * ft;
  const double ls = log_near(s), inv_s = 1.0 / s;
  double L = l.q_log_q - (l.q_x + l.q * dl) + l.q * ls, share = 0.0;
  if (left > 0.0) {
    share = left / rest;  // of the unlisted class at mt
    L += left * (log_near(share) - dt + ls);
  }
  if (empty) L = l.q > 0.0 ? INFINITY : 0.0;
  o.loss = bad ? __builtin_nan("") : L;
  o.m = fmaxf(l.m, mt);
  o.mt = mt;
  o.inv_s = empty ? 0.0f : static_cast<float>(inv_s);
  o.coef = empty || rest == 0.0 ? 0.0f : static_cast<float>(S * ft * inv_s - share);
  o.base = empty ? INFINITY : l.base;
  o.scale = empty ? 0.0f : l.scale;
  o.S = empty ? 0.0f : static_cast<float>(S);
  if (bad) o.m = o.mt = o.coef = o.S = __builtin_nanf("");
  return o;
}

// Marks class `id` in a bitmap of [first, first + 32 words), if it is there;
// whether it was marked already.
__device__ __forceinline__ bool mark(uint32_t* marks, uint32_t words, uint32_t first, int32_t id) {
  const uint32_t at = static_cast<uint32_t>(id) - first, bit = 1u << (at % 32);
  if (id < 0 || at >= words * 32) return false;
  return atomicOr(&marks[at / 32], bit) & bit;
}
// A row's listed classes, by the whole workgroup.
template <int NT>
__device__ __forceinline__ bool mark_listed(const TopkDistillArgs& a, size_t r, uint32_t* marks,
                                            uint32_t words, uint32_t first) {
  bool twice = false;
  for (uint32_t i = threadIdx.x; i < a.k; i += NT)
    twice = mark(marks, words, first, a.t_ids[r * a.k + i]) || twice;
  return twice;
}
// The marks of vector j's V classes, j counted from the bitmap's first.
template <int V>
__device__ __forceinline__ uint32_t marks_of(const uint32_t* marks, uint32_t j) {
  return (marks[j * V / 32] >> (j * V % 32)) & ((1u << V) - 1);
}

constexpr uint32_t kMarkCols = 65536;  // classes per sweep of the forward: 8 KiB

// A row's part in scratch.
struct DistillPart {
  float m;
  int dup;
  double s;
};
__host__ __device__ inline DistillPart* distill_parts(void* scratch, size_t N) {
  return reinterpret_cast<DistillPart*>(static_cast<float*>(scratch) + N * kDistillStats);
}

__device__ __forceinline__ void put_outcome(const TopkDistillArgs& a, size_t r, const Outcome& o) {
  a.row_loss[r] = static_cast<float>(o.loss);
  if (!a.stats) return;
  float* st = a.stats + r * kDistillStats;
  *reinterpret_cast<float4u*>(st) = float4u{o.m, o.inv_s, o.mt, o.coef};
  *reinterpret_cast<float4u*>(st + 4) = float4u{o.base, o.scale, o.S, 0.0f};
}
// A row that does not count.
__device__ __forceinline__ void put_nothing(const TopkDistillArgs& a, size_t r) {
  a.row_loss[r] = 0.0f;
  if (!a.stats) return;
  float* st = a.stats + r * kDistillStats;
  *reinterpret_cast<float4u*>(st) = float4u{0.0f, 0.0f, 0.0f, 0.0f};
  *reinterpret_cast<float4u*>(st + 4) = float4u{0.0f, 0.0f, 0.0f, 0.0f};
}

// A row, or one of its parts as in score_fwd_kernel. Bound by HBM where the
// list's 64-bit sums hide behind other rows' sweeps: 2048 rows of 32000 float32,
// an eighth of them of weight 0 and not read, 44 us with the loss's sum, 5.4 TB/s.
// 8192 rows of 1000: 18, bound by the lists.
template <int DT, int NT>
__global__ __launch_bounds__(NT) void distill_fwd_kernel(TopkDistillArgs a, TempScale c,
                                                         uint32_t parts, uint32_t each, int nt) {
  __shared__ uint32_t marks[kMarkCols / 32];
  __shared__ RowSums sums[NT / kWave];
  __shared__ Listed list;
  __shared__ int dup;
  using E = Elem<DT>;
  constexpr int V = Row<DT>::V;
  const size_t r = blockIdx.x / parts;
  const uint32_t part = blockIdx.x % parts, first = part * each * V;
  const uint32_t C = part + 1 < parts ? each * V : static_cast<uint32_t>(a.C) - first;
  const Row<DT> row{static_cast<const typename E::T*>(a.logits) + r * a.stride};
  if (a.weight && a.weight[r] == 0.0f) {
    if (threadIdx.x == 0 && parts == 1) put_nothing(a, r);
    return;
  }
  if (threadIdx.x == 0) dup = 0;
  if (parts == 1 && threadIdx.x < kWave) {
    Entries t = read_list<DT>(a, row, r);
    const Listed l = sum_list(a, t, c.inv_T);
    if (threadIdx.x == 0) list = l;
  }
  Online o;
  for (uint32_t c0 = 0; c0 < C; c0 += kMarkCols) {
    const uint32_t cols = min(C - c0, kMarkCols), words = (cols + 31) / 32;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < words; i += NT) marks[i] = 0;
    __syncthreads();
    if (mark_listed<NT>(a, r, marks, words, first + c0)) dup = 1;
    __syncthreads();
    const Row<DT> at{row.x + first + c0};
    const uint32_t nv = cols / V;
    for (uint32_t b = 0; b * (kBatch * NT) < nv; ++b) {
      const uint32_t j0 = b * (kBatch * NT) + threadIdx.x;
      typename Row<DT>::raw raw[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) raw[u] = at.load(min(j0 + u * NT, nv - 1), nt);
      if ((b + 1) * (kBatch * NT) <= nv) {
        float v[kBatch * V];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const uint32_t out = marks_of<V>(marks, j0 + u * NT);
          if (out) raw[u] = Row<DT>::masked(raw[u], out);
          Row<DT>::unpack(raw[u], v + u * V);
        }
        o.add<kBatch * V, false>(v, max_of<kBatch * V>(v), c);
      } else {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const uint32_t j = j0 + u * NT;
          if (j >= nv) break;
          const uint32_t out = marks_of<V>(marks, j);
          if (out) raw[u] = Row<DT>::masked(raw[u], out);
          float v[V];
          Row<DT>::unpack(raw[u], v);
          o.add<V, false>(v, max_of<V>(v), c);
        }
      }
    }
    if (threadIdx.x < cols - nv * V) {
      const uint32_t j = nv * V + threadIdx.x;
      const float v = marks[j / 32] >> (j % 32) & 1 ? -INFINITY : E::get(at.x[j]);
      o.add<1, false>(&v, v, c);
    }
  }
  const RowSums q = join<NT>(o, c, sums);
  if (threadIdx.x != 0) return;
  if (parts > 1) distill_parts(a.scratch, a.N)[blockIdx.x] = {q.m, dup, q.s};
  else put_outcome(a, r, row_outcome(list, q.m, q.s, c.inv_T, dup != 0));
}

// Joins a row's parts (at most kWave) with its list: one wavefront a row.
template <int DT>
__global__ __launch_bounds__(kWave) void distill_join_kernel(TopkDistillArgs a, TempScale c,
                                                             uint32_t parts) {
  const size_t r = blockIdx.x;
  if (a.weight && a.weight[r] == 0.0f) {
    if (threadIdx.x == 0) put_nothing(a, r);
    return;
  }
  const Row<DT> row{static_cast<const typename Elem<DT>::T*>(a.logits) + r * a.stride};
  DistillPart p{-FLT_MAX, 0, 0.0};
  if (threadIdx.x < parts) p = distill_parts(a.scratch, a.N)[r * parts + threadIdx.x];
  Entries t = read_list<DT>(a, row, r);
  const Listed l = sum_list(a, t, c.inv_T);
  const RowSums q = join_lanes({p.m, p.s, 0.0}, c);
  const Outcome o = row_outcome(l, q.m, q.s, c.inv_T, __ballot(p.dup != 0) != 0);
  if (threadIdx.x == 0) put_outcome(a, r, o);
}

__device__ __forceinline__ float row_weight(const TopkDistillArgs& a, size_t r) {
  return a.weight ? a.weight[r] : static_cast<float>(1.0 / static_cast<double>(a.N));
}

// loss = sum of w_r L_r in 64 bits and a fixed order, one workgroup. Eight rows
// a thread under way at once: 8192 rows in one round of loads of 1024 threads.
template <int NT>
__device__ __forceinline__ void sum_loss(const TopkDistillArgs& a) {
  __shared__ double sums[NT / kWave];
  constexpr int n = 8;
  double acc = 0.0;
  for (size_t r0 = threadIdx.x; r0 < a.N; r0 += n * NT) {
    float w[n], l[n];
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const size_t r = r0 + i * NT, at = r < a.N ? r : a.N - 1;
      w[i] = r < a.N ? row_weight(a, at) : 0.0f;
      l[i] = a.row_loss[at];
    }
#pragma unroll
    for (int i = 0; i < n; ++i)
      if (w[i] != 0.0f) acc += static_cast<double>(w[i]) * l[i];
  }
  acc = lanes_sum(acc);
  if (threadIdx.x % kWave == 0) sums[threadIdx.x / kWave] = acc;
  __syncthreads();
  if (threadIdx.x >= kWave) return;
  acc = lanes_sum(threadIdx.x < NT / kWave ? sums[threadIdx.x] : 0.0);
  if (threadIdx.x == 0) *a.loss = static_cast<float>(acc);
}

// w seed / T, which may leave float32's range where its product with a gradient
// does not.
__device__ __forceinline__ double grad_scale(const TopkDistillArgs& a, float wr, TempScale c) {
  return static_cast<double>(wr) * (a.seed ? a.seed[0] : 1.0f) * c.inv_T;
}
__device__ __forceinline__ float times(double W, float g) { return static_cast<float>(W * g); }

// The listed classes' gradients, one thread each, of those in
// [first, first + cols): W (S p - q).
template <int DT>
__device__ __forceinline__ void listed_grads(const TopkDistillArgs& a, size_t r, uint32_t first,
                                             uint32_t cols, const Row<DT>& row,
                                             typename Elem<DT>::T* dx, TempScale c, float m,
                                             float inv_s, const float* list, double W, int threads) {
  const float base = list[0], scale = list[1], S = list[2];
  for (uint32_t i = threadIdx.x; i < a.k; i += threads) {
    const int32_t id = a.t_ids[r * a.k + i];
    if (id < 0 || static_cast<uint32_t>(id) - first >= cols) continue;
    const float p = exp2_raw(scaled(Elem<DT>::get(row.x[id]), m, c)) * inv_s;
    dx[id] = Elem<DT>::put(times(W, S * p - expf(a.t_logp[r * a.k + i] - base) * scale));
  }
}

// As score_bwd_kernel (2048 rows of 8192 float32 23 us, 5.8 TB/s, part of it
// from the memory-side cache); a vector with listed classes is stored class by class,
// without them: each class is written by one thread, so the gradient may stand
// in the logits' place.
template <int DT, int NT>
__global__ __launch_bounds__(NT) void distill_bwd_kernel(TopkDistillArgs a, TempScale c,
                                                         uint32_t parts, int nt) {
  using E = Elem<DT>;
  constexpr int V = Row<DT>::V;
  constexpr uint32_t kCols = NT * kBatch * V, kWords = kCols / 32 + 1;
  __shared__ uint32_t marks[kWords];
  const size_t r = blockIdx.x / parts;
  if (r == a.N) {  // a workgroup behind the rows' (TopkDistillFwdBwd): the loss
    sum_loss<NT>(a);
    return;
  }
  const uint32_t part = blockIdx.x % parts, first = part * kCols;
  const uint32_t C = static_cast<uint32_t>(a.C);
  // The last part takes the classes behind the last whole vector, too.
  const uint32_t cols = min(C - first, kCols + (part + 1 == parts ? V : 0));
  const uint32_t nv = min(cols, kCols) / V;
  const Row<DT> all{static_cast<const typename E::T*>(a.logits) + r * a.stride};
  const Row<DT> row{all.x + first};
  typename E::T* dx = static_cast<typename E::T*>(a.dlogits) + r * a.dstride;
  const float wr = row_weight(a, r);
  typename Row<DT>::raw raw[kBatch];
  if (nv && wr != 0.0f)
#pragma unroll
    for (int u = 0; u < kBatch; ++u) raw[u] = row.load(min(threadIdx.x + u * NT, nv - 1), nt);
  const float* st = a.stats + r * kDistillStats;
  const float4u s0 = *reinterpret_cast<const float4u*>(st);
  const double W = grad_scale(a, wr, c);
  const float coef = times(W, s0[3]);
  for (uint32_t i = threadIdx.x; i < kWords; i += NT) marks[i] = 0;
  __syncthreads();
  if (wr != 0.0f) mark_listed<NT>(a, r, marks, kWords, first);
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kBatch; ++u) {
    const uint32_t j = threadIdx.x + u * NT;
    if (j >= nv) continue;
    float v[V];
    if (wr == 0.0f) {
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = 0.0f;
    } else {
      Row<DT>::unpack(raw[u], v);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = coef * exp2_raw(scaled(v[e], s0[2], c));
    }
    const uint32_t out = marks_of<V>(marks, j);
    if (!out) {
      Row<DT>::store(dx + first, j, v, nt);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (!(out >> e & 1)) dx[first + j * V + e] = E::put(v[e]);
    }
  }
  if (part + 1 == parts && threadIdx.x < cols - nv * V) {
    const uint32_t j = nv * V + threadIdx.x;
    const float g = wr == 0.0f ? 0.0f : coef * exp2_raw(scaled(E::get(row.x[j]), s0[2], c));
    if (!(marks[j / 32] >> (j % 32) & 1)) dx[first + j] = E::put(g);
  }
  if (wr != 0.0f)
    listed_grads<DT>(a, r, first, cols, all, dx, c, s0[0], s0[1], st + 4, W, NT);
}

// Loss and gradient in one pass: the row stays in the registers of NT threads
// (R vectors each) between its sums and its gradient, so the logits are read
// once. The row becomes its exponentials there; a 16-bit row, which they would
// take twice the registers of, only where two workgroups a CU still fit
// (kHold: 4096 rows of 32000 bf16 119 us against 128), else it stays packed and
// takes the exponentials twice. A wavefront of its own takes the list meanwhile:
// its 64-bit sums need as many registers as a row's vectors, and their latency
// hides behind the row's loads. Bound by HBM: 8192 rows of 32000 float32 394 us,
// 5.3 TB/s of logits read and gradients written (a copy of 1 GiB reaches 5.2), 373
// with an eighth of the rows of weight 0, whose logits are not read;
// 16-bit rows by the exponentials of the two workgroups, whose phases do not
// overlap enough: 4096 rows of 32000 bf16 119 us, 4.4 TB/s. The second launch
// bound keeps two workgroups of 960 threads a CU.
template <int DT, int NT, int R>
__global__ __launch_bounds__(NT + kWave, NT == 960 && R <= 9 ? 8 : 1) void distill_both_kernel(
    TopkDistillArgs a, TempScale c, int nt) {
  using E = Elem<DT>;
  constexpr int V = Row<DT>::V;
  constexpr uint32_t kWords = NT * R * V / 32 + 1;
  __shared__ uint32_t marks[kWords];
  __shared__ float tops[NT / kWave];
  __shared__ double rests[NT / kWave];
  __shared__ float coefs;
  __shared__ int dup;
  const size_t r = blockIdx.x;
  const uint32_t C = static_cast<uint32_t>(a.C), nv = C / V;
  const Row<DT> row{static_cast<const typename E::T*>(a.logits) + r * a.stride};
  typename E::T* dx = static_cast<typename E::T*>(a.dlogits) + r * a.dstride;
  const float wr = row_weight(a, r);
  const bool lists = threadIdx.x >= NT;
  const bool behind = threadIdx.x < C - nv * V;
  const uint32_t jb = nv * V + threadIdx.x;  // the thread's class behind the vectors
  if (wr == 0.0f) {
    if (lists) {
      if (threadIdx.x == NT) a.row_loss[r] = 0.0f;
      return;
    }
    const float zero[V] = {};
    for (uint32_t j = threadIdx.x; j < nv; j += NT) Row<DT>::store(dx, j, zero, nt);
    if (behind) dx[jb] = E::put(0.0f);
    return;
  }
  if (lists) {
    if (threadIdx.x == NT) dup = 0;
    Entries t = read_list<DT>(a, row, r);
    __syncthreads();  // marks are clear
#pragma unroll
    for (int i = 0; i < t.n; ++i)
      if (mark(marks, (C + 31) / 32, 0, t.id[i])) dup = 1;
    __syncthreads();  // marks are set
    const Listed l = sum_list(a, t, c.inv_T);
    __syncthreads();  // tops
    float top = -FLT_MAX;
#pragma unroll
    for (int i = 0; i < NT / kWave; ++i) top = fmaxf(top, tops[i]);
    __syncthreads();  // rests
    double rest = 0.0;
#pragma unroll
    for (int i = 0; i < NT / kWave; ++i) rest += rests[i];
    const Outcome o = row_outcome(l, top, rest, c.inv_T, dup != 0);
    const double W = grad_scale(a, wr, c);
    if (threadIdx.x == NT) coefs = times(W, o.coef);
    __syncthreads();  // coefs
    if (threadIdx.x == NT) a.row_loss[r] = static_cast<float>(o.loss);
#pragma unroll
    for (int i = 0; i < t.n; ++i) {
      if (t.id[i] < 0 || static_cast<uint32_t>(t.id[i]) >= C) continue;
      const float p = exp2_raw(scaled(t.x[i], o.m, c)) * o.inv_s;
      dx[t.id[i]] = E::put(times(W, o.S * p - (o.inv_s != 0.0f ? t.v[i] : 0.0f)));
    }
    return;
  }
  typename Row<DT>::raw raw[R];
  if (nv)
#pragma unroll
    for (int u = 0; u < R; ++u) raw[u] = row.load(min(threadIdx.x + u * NT, nv - 1), nt);
  float xb = behind ? E::get(row.x[jb]) : -INFINITY;
  for (uint32_t i = threadIdx.x; i < (C + 31) / 32; i += NT) marks[i] = 0;
  __syncthreads();  // marks are clear
  __syncthreads();  // marks are set
  // The unlisted classes' maximum. Every load of the row has been used by the
  // next barrier: the gradient may be stored in its place.
  float top = -FLT_MAX;
  uint32_t listed = 0;  // whether a vector holds listed classes, a bit each
#pragma unroll
  for (int u = 0; u < R; ++u) {
    const uint32_t j = threadIdx.x + u * NT;
    const uint32_t out = j < nv ? marks_of<V>(marks, j) : (1u << V) - 1;
    if (out) {
      listed |= 1u << u;
      raw[u] = Row<DT>::masked(raw[u], out);
    }
    float v[V];
    Row<DT>::unpack(raw[u], v);
#pragma unroll
    for (int e = 0; e < V; ++e) top = fmaxf(top, v[e]);
    if constexpr (DT != kF32) __builtin_amdgcn_sched_barrier(0);
  }
  if (behind && marks[jb / 32] >> (jb % 32) & 1) xb = -INFINITY;
  top = lanes_max(fmaxf(top, xb));
  if (threadIdx.x % kWave == 0) tops[threadIdx.x / kWave] = top;
  __syncthreads();  // tops
#pragma unroll
  for (int i = 0; i < NT / kWave; ++i) top = fmaxf(top, tops[i]);
  double rest = 0.0;
  constexpr bool kHold = DT != kF32 && (R <= 5 || NT == kWave);
  float held[kHold ? R * V : 1];
#pragma unroll
  for (int u = 0; u < R; ++u) {
    keep_packed(raw[u]);
    float v[V], s = 0.0f;
    Row<DT>::unpack(raw[u], v);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      v[e] = exp2_raw(scaled(v[e], top, c));
      s += v[e];
    }
    if constexpr (DT == kF32) raw[u] = Row<DT>::pack(v);
    if constexpr (kHold)
#pragma unroll
      for (int e = 0; e < V; ++e) held[u * V + e] = v[e];
    rest += threadIdx.x + u * NT < nv ? s : 0.0f;
    if constexpr (DT != kF32) __builtin_amdgcn_sched_barrier(0);
  }
  xb = exp2_raw(scaled(xb, top, c));
  rest = lanes_sum(rest + xb);
  if (threadIdx.x % kWave == 0) rests[threadIdx.x / kWave] = rest;
  __syncthreads();  // rests
  __syncthreads();  // coefs
  const float coef = coefs;
#pragma unroll
  for (int u = 0; u < R; ++u) {
    const uint32_t j = threadIdx.x + u * NT;
    if (j >= nv) continue;
    float v[V];
    if constexpr (kHold) {
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = held[u * V + e];
    } else {
      keep_packed(raw[u]);
      Row<DT>::unpack(raw[u], v);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if constexpr (DT != kF32 && !kHold) v[e] = exp2_raw(scaled(v[e], top, c));
      v[e] *= coef;
    }
    if (!(listed >> u & 1)) {
      Row<DT>::store(dx, j, v, nt);
    } else {
      const uint32_t out = marks_of<V>(marks, j);
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (!(out >> e & 1)) dx[j * V + e] = E::put(v[e]);
    }
  }
  if (behind && !(marks[jb / 32] >> (jb % 32) & 1)) dx[jb] = E::put(coef * xb);
}

constexpr int kLoss = 1024;
__global__ __launch_bounds__(kLoss) void distill_loss_kernel(TopkDistillArgs a) {
  sum_loss<kLoss>(a);
}

#define NT_LAUNCH(kernel, nt_, dtype, grid, ...)                                              \
  do {                                                                                        \
    if ((dtype) == kF32)                                                                      \
      hipLaunchKernelGGL((kernel<kF32, nt_>), grid, dim3(nt_), 0, c.stream, __VA_ARGS__);     \
    else if ((dtype) == kBF16)                                                                \
      hipLaunchKernelGGL((kernel<kBF16, nt_>), grid, dim3(nt_), 0, c.stream, __VA_ARGS__);    \
    else                                                                                      \
      hipLaunchKernelGGL((kernel<kF16, nt_>), grid, dim3(nt_), 0, c.stream, __VA_ARGS__);     \
  } while (0)

// One workgroup a row.
#define TYPE_LAUNCH(kernel, threads, ...)                                                     \
  do {                                                                                        \
    const dim3 rows(static_cast<unsigned>(a.N));                                              \
    if (a.dtype == kF32)                                                                      \
      hipLaunchKernelGGL(kernel<kF32>, rows, dim3(threads), 0, c.stream, __VA_ARGS__);        \
    else if (a.dtype == kBF16)                                                                \
      hipLaunchKernelGGL(kernel<kBF16>, rows, dim3(threads), 0, c.stream, __VA_ARGS__);       \
    else                                                                                      \
      hipLaunchKernelGGL(kernel<kF16>, rows, dim3(threads), 0, c.stream, __VA_ARGS__);        \
  } while (0)

// How the forward kernels cut the rows: `parts` ranges of `each` vectors for
// `threads` threads. `keys` is the score's k, 0 without one. Measured in graphs,
// us (scores k 20, float32, where not said):
//   64 threads where many short rows fill the chip: one wavefront has no
//   barriers to wait at. 8192 rows of 1000: 14.9 against 27.3 with 256 threads,
//   of 4000 36.1 against 34.6 (the limit of 1024 vectors is a little high for
//   that many rows); 2048 of 4000 11.9 against 12.1; 1024 of 1000 6.7 against
//   7.7, of 4000 10.1 against 8.8. With k past 32 its 64 maxima bound the k-th
//   class badly: 2000 rows of 2000, k 64, 87 against 13.
//   1024 threads where few rows leave a CU to each: 256 rows of 32000 11.1
//   against 13.5 with 256 threads; 300 rows of 50000 bf16 20.8 against 17.0.
//   Parts where that leaves most of the chip idle: 24 rows of 131072 bf16 12.2
//   in 8 parts against 16.7, 1 row of 131072 10.9 in 16 against 16.6, 64 rows of
//   131072 15.0 in 8 against 18.4; but 128 rows of 131072 21.1 in 4 against
//   19.3, 1 row of 32000 11.0 in 4 against 9.0.
struct Cut {
  int threads;
  uint32_t parts, each;
};
Cut CutRows(uint64_t N, uint64_t C, int dtype, uint64_t keys) {
  const uint64_t nv = C / (dtype == kF32 ? 4 : 8);
  Cut cut{256, 1, static_cast<uint32_t>(nv)};
  if (nv <= 1024 && N >= 1024 && N >= 2 * nv && keys <= 32) cut.threads = 64;
  else if (N <= 256 && nv >= 2048) cut.threads = 1024;
  uint64_t parts = std::min<uint64_t>(C / 8192, 512 / N);
  if (keys) parts = std::min<uint64_t>(parts, kJoinKeys / keys);
  parts = std::min<uint64_t>(parts, kWave);
  if (parts >= 8) {
    cut.each = static_cast<uint32_t>((nv + parts - 1) / parts);
    cut.parts = static_cast<uint32_t>((nv + cut.each - 1) / cut.each);
    cut.threads = 256;
  }
  return cut;
}

}  // namespace

uint64_t TokenScoreScratch(uint64_t N, uint64_t C, int dtype, uint64_t k) {
  const Cut cut = CutRows(N, C, dtype, k);
  return cut.parts > 1 ? N * cut.parts * (sizeof(ScorePart) + k * sizeof(uint64_t)) : 0;
}
uint64_t TopkDistillScratch(uint64_t N, uint64_t C, int dtype, uint64_t) {
  const Cut cut = CutRows(N, C, dtype, 0);
  const uint64_t parts = cut.parts > 1 ? cut.parts * sizeof(DistillPart) : 0;
  return N * (kDistillStats * sizeof(float) + parts);
}

Status TokenScoreFwd(const TokenScoreArgs& a, const Ctx& c) {
  const TempScale c2 = ScaleOf(a.T);
  const int nt = StreamPolicy(a.N * a.C * (a.dtype == kF32 ? 4 : 2)) ? 1 : 0;
  const Cut cut = CutRows(a.N, a.C, a.dtype, a.k);
  const dim3 grid(static_cast<unsigned>(a.N * cut.parts));
  if (cut.threads == 64)
    NT_LAUNCH(score_fwd_kernel, 64, a.dtype, grid, a, c2, cut.parts, cut.each, nt);
  else if (cut.threads == 256)
    NT_LAUNCH(score_fwd_kernel, 256, a.dtype, grid, a, c2, cut.parts, cut.each, nt);
  else
    NT_LAUNCH(score_fwd_kernel, 1024, a.dtype, grid, a, c2, cut.parts, cut.each, nt);
  if (cut.parts > 1) TYPE_LAUNCH(score_join_kernel, kJoin, a, c2, cut.parts);
  return LaunchStatus("TokenLogprobs");
}

// Workgroups per row of the gradient kernels: kBatch vectors a thread.
static uint32_t GradParts(uint64_t C, int dtype, int threads) {
  const uint64_t nv = C / (dtype == kF32 ? 4 : 8), each = static_cast<uint64_t>(threads) * kBatch;
  return static_cast<uint32_t>(nv <= each ? 1 : (nv + each - 1) / each);
}

Status TokenScoreBwd(const TokenScoreBwdArgs& a, const Ctx& c) {
  const TempScale c2 = ScaleOf(a.T);
  const int nt = StreamPolicy(2 * a.N * a.C * (a.dtype == kF32 ? 4 : 2)) ? 1 : 0;
  const int threads = a.C / (a.dtype == kF32 ? 4 : 8) <= 256 ? 64 : 256;
  const uint32_t parts = GradParts(a.C, a.dtype, threads);
  const dim3 grid(static_cast<unsigned>(a.N * parts));
  if (threads == 64) NT_LAUNCH(score_bwd_kernel, 64, a.dtype, grid, a, c2, parts, nt);
  else NT_LAUNCH(score_bwd_kernel, 256, a.dtype, grid, a, c2, parts, nt);
  return LaunchStatus("TokenLogprobsBwd");
}

static void DistillLoss(const TopkDistillArgs& a, const Ctx& c) {
  if (a.loss) hipLaunchKernelGGL(distill_loss_kernel, dim3(1), dim3(kLoss), 0, c.stream, a);
}

static void DistillRows(const TopkDistillArgs& a, const Ctx& c) {
  const TempScale c2 = ScaleOf(a.T);
  const int nt = StreamPolicy(a.N * a.C * (a.dtype == kF32 ? 4 : 2)) ? 1 : 0;
  const Cut cut = CutRows(a.N, a.C, a.dtype, 0);
  const dim3 grid(static_cast<unsigned>(a.N * cut.parts));
  if (cut.threads == 64)
    NT_LAUNCH(distill_fwd_kernel, 64, a.dtype, grid, a, c2, cut.parts, cut.each, nt);
  else if (cut.threads == 256)
    NT_LAUNCH(distill_fwd_kernel, 256, a.dtype, grid, a, c2, cut.parts, cut.each, nt);
  else
    NT_LAUNCH(distill_fwd_kernel, 1024, a.dtype, grid, a, c2, cut.parts, cut.each, nt);
  if (cut.parts > 1) TYPE_LAUNCH(distill_join_kernel, kWave, a, c2, cut.parts);
}

Status TopkDistillFwd(const TopkDistillArgs& a, const Ctx& c) {
  DistillRows(a, c);
  DistillLoss(a, c);
  return LaunchStatus("TopkDistill");
}

// With a.loss the gradient's launch also sums the rows' losses.
Status TopkDistillBwd(const TopkDistillArgs& a, const Ctx& c) {
  const TempScale c2 = ScaleOf(a.T);
  const int nt = StreamPolicy(2 * a.N * a.C * (a.dtype == kF32 ? 4 : 2)) ? 1 : 0;
  const int threads = a.C / (a.dtype == kF32 ? 4 : 8) <= 256 ? 64 : 256;
  const uint32_t parts = GradParts(a.C, a.dtype, threads);
  const dim3 grid(static_cast<unsigned>(a.N * parts + (a.loss ? 1 : 0)));
  if (threads == 64) NT_LAUNCH(distill_bwd_kernel, 64, a.dtype, grid, a, c2, parts, nt);
  else NT_LAUNCH(distill_bwd_kernel, 256, a.dtype, grid, a, c2, parts, nt);
  return LaunchStatus("TopkDistillBwd");
}

template <int DT, int NT, int R>
static void LaunchBoth(const TopkDistillArgs& a, const Ctx& c) {
  const int nt = StreamPolicy(2 * a.N * a.C * (DT == kF32 ? 4 : 2)) ? 1 : 0;
  hipLaunchKernelGGL((distill_both_kernel<DT, NT, R>), dim3(static_cast<unsigned>(a.N)),
                     dim3(NT + kWave), 0, c.stream, a, ScaleOf(a.T), nt);
}

// The widest row that distill_both_kernel holds, in vectors, and the shape for
// one of nv: the fewest registers that hold it. Measured in graphs, us, k 20:
//   many short rows to one wavefront each: 8192 rows of 2000 float32 28.8 with
//   64 x 8 against 35.6 with 256 x 4; 256 rows 7.8 against 6.6;
//   wide rows to 960 threads, two workgroups a CU: 8192 rows of 20000 float32
//   237 with 960 x 9 against 295 with 512 x 16, of 32000 393 against 409; 4096
//   rows of 50001 f16 221 against 290; 4096 of 32000 bf16 119 with 960 x 5
//   against 128 with 512 x 8, but 8192 of 17000 166 against 162.
constexpr uint64_t kBothVectors = 960 * 18;
template <int DT>
static void LaunchBothFor(uint64_t nv, const TopkDistillArgs& a, const Ctx& c) {
  if (nv <= 64 * 4) LaunchBoth<DT, 64, 4>(a, c);
  else if (nv <= 64 * 8 && a.N >= 1024) LaunchBoth<DT, 64, 8>(a, c);
  else if (nv <= 256 * 4) LaunchBoth<DT, 256, 4>(a, c);
  else if (nv <= 256 * 8) LaunchBoth<DT, 256, 8>(a, c);
  else if (DT != kF32 && nv > 960 * 3 && nv <= 960 * 5)
    LaunchBoth<DT == kF32 ? kBF16 : DT, 960, 5>(a, c);
  else if (nv <= 512 * 8) LaunchBoth<DT, 512, 8>(a, c);
  else if (nv <= 960 * 9) LaunchBoth<DT, 960, 9>(a, c);
  else LaunchBoth<DT, 960, 18>(a, c);
}

Status TopkDistillFwdBwd(const TopkDistillArgs& a, const Ctx& c) {
  const uint64_t nv = a.C / (a.dtype == kF32 ? 4 : 8);
  // The row fits no workgroup's registers, or rows are too few to fill the chip
  // (40 rows of 131072 bf16: 18.7 us in parts against 30.5).
  if (nv > kBothVectors || CutRows(a.N, a.C, a.dtype, 0).parts > 1) {
    TopkDistillArgs b = a;
    b.stats = static_cast<float*>(a.scratch);
    DistillRows(b, c);
    return TopkDistillBwd(b, c);
  }
  if (a.dtype == kF32) LaunchBothFor<kF32>(nv, a, c);
  else if (a.dtype == kBF16) LaunchBothFor<kBF16>(nv, a, c);
  else LaunchBothFor<kF16>(nv, a, c);
  DistillLoss(a, c);
  return LaunchStatus("TopkDistill");
}

}  // namespace seeml_hip
