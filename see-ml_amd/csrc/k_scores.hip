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
template <int DT> struct Elem;
template <> struct Elem<kF32> {
  using T = float;
  static __device__ float get(T v) { return v; }
  static __device__ T put(float v) { return v; }
};
template <> struct Elem<kBF16> {
  using T = __bf16;
  static __device__ float get(T v) { return static_cast<float>(v); }
  static __device__ T put(float v) { return static_cast<T>(v); }
};
template <> struct Elem<kF16> {
  using T = _Float16;
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

__device__ __forceinline__ uint64_t block_max_key(uint64_t v, uint64_t* scratch) {
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) {
    const uint64_t o = __shfl_xor(v, off, kWave);
    v = o > v ? o : v;
  }
  __syncthreads();
  if (threadIdx.x % kWave == 0) scratch[threadIdx.x / kWave] = v;
  __syncthreads();
  for (int i = 0; i < kBlock / kWave; ++i) v = scratch[i] > v ? scratch[i] : v;
  return v;
}

template <int DT>
__global__ __launch_bounds__(kBlock) void score_fwd_kernel(TokenScoreArgs a, TempScale c2) {
  __shared__ float fs[kBlock / kWave];
  __shared__ double ds[kBlock / kWave];
  __shared__ uint64_t ks[kBlock / kWave];
  using E = Elem<DT>;
  const size_t r = blockIdx.x;
  const typename E::T* x = static_cast<const typename E::T*>(a.logits) + r * a.stride;
  const uint32_t C = static_cast<uint32_t>(a.C);
  const double inv_T = 1.0 / a.T;
  float m = -FLT_MAX;
  for (uint32_t j = threadIdx.x; j < C; j += kBlock) m = fmaxf(m, E::get(x[j]));
  m = block_max<kBlock>(m, fs);
  double s = 0.0, w = 0.0;
  for (uint32_t j = threadIdx.x; j < C; j += kBlock) {
    const float d = scaled(E::get(x[j]), m, c2);
    const float e = exp2f(d);
    s += e;
    w += static_cast<double>(e) * fmaxf(d, kLow);
  }
  s = block_sum<double, kBlock>(s, ds);
  w = block_sum<double, kBlock>(w, ds) * M_LN2;
  const bool bad = s != s, empty = s == 0.0;
  const double ls = log(s);
  const double H = bad ? s : empty ? 0.0 : ls - w / s;
  if (threadIdx.x == 0) {
    if (a.logp) {
      const int32_t t = a.targets[r];
      float lp = 0.0f;
      if (t >= 0) {
        if (static_cast<uint32_t>(t) >= C || bad) lp = __builtin_nanf("");
        else if (empty) lp = -INFINITY;
        else lp = static_cast<float>((static_cast<double>(E::get(x[t])) - m) * inv_T - ls);
      }
      a.logp[r] = lp;
    }
    if (a.entropy) a.entropy[r] = static_cast<float>(H);
    if (a.stats) {
      float* o = a.stats + r * kScoreStats;
      o[0] = bad ? __builtin_nanf("") : empty ? 0.0f : m;
      o[1] = bad ? __builtin_nanf("") : empty ? INFINITY : static_cast<float>(ls);
      o[2] = static_cast<float>(H);
      o[3] = bad ? __builtin_nanf("") : empty ? 0.0f : static_cast<float>(1.0 / s);
    }
  }
  uint64_t last = ~uint64_t{0};
  for (uint32_t i = 0; i < a.k; ++i) {
    uint64_t best = 0;
    if (!bad)
      for (uint32_t j = threadIdx.x; j < C; j += kBlock) {
        const float v = E::get(x[j]);
        const uint64_t key = v > -INFINITY ? key_of(v, j) : 0;
        if (key < last && key > best) best = key;
      }
    best = block_max_key(best, ks);
    last = best ? best : 1;  // below 1 nothing is left
    if (threadIdx.x == 0) {
      const uint32_t col = 0xFFFFFFFFu - static_cast<uint32_t>(best);
      a.top_ids[r * a.k + i] = best ? static_cast<int32_t>(col) : -1;
      a.top_logp[r * a.k + i] =
          bad ? __builtin_nanf("")
              : best ? static_cast<float>((static_cast<double>(E::get(x[col])) - m) * inv_T - ls)
                     : -INFINITY;
    }
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

}  // namespace

uint64_t TokenScoreScratch(uint64_t, uint64_t, int, uint64_t) { return 0; }
uint64_t TopkDistillScratch(uint64_t N, uint64_t, int, uint64_t) {
  return N * kDistillStats * sizeof(float);
}

Status TokenScoreFwd(const TokenScoreArgs& a, const Ctx& c) {
  const TempScale c2 = ScaleOf(a.T);
  DTYPE_LAUNCH(score_fwd_kernel, a.dtype, dim3(static_cast<unsigned>(a.N)), dim3(kBlock), 0,
               c.stream, a, c2);
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
