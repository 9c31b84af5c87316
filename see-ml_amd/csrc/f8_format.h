// f8_format.h — the block-scaled 8-bit format of the F8 operators, on the device.
//
// A matrix [rows, cols] is one e4m3 code a value, rows padded with zeros to
// whole blocks of 128 columns, and one scale byte s a block, of value
// 2^(s - 127) (0 to 247). The scales lie block-major, [blocks of a row][rows,
// rounded up to 128], so that the rows of a tile, which a wavefront multiplies
// together, have theirs side by side; those of rows past the last are 0.
//
// A block's exponent is the least e with amax / 2^e <= 448, e4m3's largest
// number, amax over the block's finite values. A power of two costs nothing:
// e4m3 is a floating format, so a finer scale would gain no bit except in the
// lowest of its 17 binades, and multiplying by it is exact in every direction
// (a transposed weight has the same values, and the matrix cores apply it
// themselves). Rounding is to nearest, ties to even. Infinities and NaN become
// the NaN code and touch no other value of their block.
#pragma once

#include "device_common.h"
#include "kernels.h"

#include <cfloat>

namespace seeml_hip {
namespace f8 {

constexpr int kBlock = 128;
__host__ __device__ inline constexpr uint64_t Up128(uint64_t n) { return (n + 127) / 128 * 128; }

// The scale byte of a block whose largest finite magnitude is amax.
__device__ __forceinline__ uint32_t ScaleByte(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return e > 0 ? static_cast<uint32_t>(e) : 0u;
}
// 2^(s - 127), and its inverse (s <= 247), exactly; 2^-127 is subnormal.
__device__ __forceinline__ float ScaleValue(uint32_t s) {
  return __uint_as_float(s ? s << 23 : 0x400000u);
}
__device__ __forceinline__ float ScaleInverse(uint32_t s) { return __uint_as_float((254u - s) << 23); }

// The largest finite magnitude of n values: the rare infinity or NaN has mend() called,
// which may change them, and the values looked at again.
struct Nothing {
  __device__ __forceinline__ void operator()() const {}
};
template <int N, typename F = Nothing>
__device__ __forceinline__ float FiniteMax(const float (&v)[N], F&& mend = F()) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) top = __builtin_elementwise_maximum(top, fabsf(v[i]));
  if (__builtin_expect(!(top <= FLT_MAX), false)) {
    mend();
    top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, fabsf(v[i]) <= FLT_MAX ? fabsf(v[i]) : 0.0f);
  }
  return top;
}
// Four values, already in units of the scale, as codes. What passes 448 here is
// an infinity, which the conversion makes a NaN.
__device__ __forceinline__ uint32_t Pack4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  return static_cast<uint32_t>(w);
}
typedef float f32x2 __attribute__((ext_vector_type(2)));
// Four codes as numbers, without the scale.
__device__ __forceinline__ void Unpack4(uint32_t w, float* v) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
  const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
  v[0] = lo.x; v[1] = lo.y; v[2] = hi.x; v[3] = hi.y;
}

// One element of a float32, bfloat16 or half argument, and vectors of E of
// them (16 bytes) at the alignment of an element: rows of any stride keep the
// wide accesses.
typedef uint32_t u32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <int DT> struct Elem;
template <> struct Elem<kF32> {
  using T = float;
  using V = u32x4_at4;
  static constexpr int E = 4;
};
template <> struct Elem<kBF16> {
  using T = __bf16;
  using V = u32x4_at2;
  static constexpr int E = 8;
};
template <> struct Elem<kF16> {
  using T = _Float16;
  using V = u32x4_at2;
  static constexpr int E = 8;
};
template <int DT>
__device__ __forceinline__ void UnpackElems(u32x4 r, float* v) {
  using T = typename Elem<DT>::T;
  typedef T vec __attribute__((ext_vector_type(Elem<DT>::E)));
  const vec t = __builtin_bit_cast(vec, r);
#pragma unroll
  for (int i = 0; i < Elem<DT>::E; ++i) v[i] = static_cast<float>(t[i]);
}
template <int DT>
__device__ __forceinline__ u32x4 PackElems(const float* v) {
  using T = typename Elem<DT>::T;
  typedef T vec __attribute__((ext_vector_type(Elem<DT>::E)));
  vec t;
#pragma unroll
  for (int i = 0; i < Elem<DT>::E; ++i) t[i] = static_cast<T>(v[i]);
  return __builtin_bit_cast(u32x4, t);
}
// The E elements of a row from column c on; zeros from column `cols` on.
template <int DT>
__device__ __forceinline__ void LoadElems(const typename Elem<DT>::T* row, uint32_t c, uint32_t cols,
                                          float* v) {
  constexpr int E = Elem<DT>::E;
  if (c + E <= cols) {
    UnpackElems<DT>(*reinterpret_cast<const typename Elem<DT>::V*>(row + c), v);
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = c + i < cols ? static_cast<float>(row[c + i]) : 0.0f;
  }
}
// E elements, rounded once, to a row from column c on, short of `cols`.
template <int DT>
__device__ __forceinline__ void StoreElems(typename Elem<DT>::T* row, uint32_t c, uint32_t cols,
                                           const float* v) {
  constexpr int E = Elem<DT>::E;
  if (c + E <= cols) {
    *reinterpret_cast<typename Elem<DT>::V*>(row + c) = PackElems<DT>(v);
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (c + i < cols) row[c + i] = static_cast<typename Elem<DT>::T>(v[i]);
  }
}

// An activation a(x) and its derivative d(x). SiLU and GELU (its tanh form) both
// are x s with s = 1 / (1 + exp(-t)), t = x or 2u, and 1 - s is s at -t. From e =
// exp(-|t|), at most 1, they are 1 / (1 + e) and e / (1 + e): nothing overflows and
// nothing cancels, so that tails keep their digits. The hardware's exp2 (1 ulp) takes
// |t| log2(e) rounded to 24 bits; what the rounding left, times ln 2 in two parts, is
// made good behind it. With half ulps for that, for 1 + e and for the product, and the
// hardware's reciprocal's 1, s and 1 - s are off by less than 2^-21 of themselves; below
// 2^-126 they are 0. (A Newton step on the reciprocal: GELU's gradient of 8192x16384
// bfloat16 124 -> 128 us, errors of float32 results 6.5e-8 -> 6.4e-8 in the 2-norm.)
__device__ __forceinline__ void SigmoidParts(float t, float* s, float* rest) {
  constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f, kLn2Low = -1.90465421e-9f;
  const float n = fabsf(t) * -kLog2e;
  const float left = fmaf(n, -kLn2Low, fmaf(n, -kLn2, -fabsf(t)));
  float e = __builtin_amdgcn_exp2f(n);
  e = fmaf(e, left, e);
  const float d = 1.0f + e;
  const float r = __builtin_amdgcn_rcpf(d);
  const float er = e * r;
  *s = t >= 0.0f ? r : er;
  *rest = t >= 0.0f ? er : r;
}
// x held to [lo, hi] from one side; a NaN stays.
__device__ __forceinline__ float AtLeast(float x, float lo) { return __builtin_elementwise_maximum(x, lo); }
__device__ __forceinline__ float AtMost(float x, float hi) { return __builtin_elementwise_minimum(x, hi); }
template <int ACT>
__device__ __forceinline__ void ActAndSlope(float x, float* a, float* d) {
  if constexpr (ACT == 1) {
    const float low = x != x ? x : 0.0f;  // a NaN stays
    *a = x > 0.0f ? x : low;
    *d = x > 0.0f ? 1.0f : low;
  } else if constexpr (ACT == 3) {
    const float y = AtLeast(x, -128.0f);  // s is 0 from -88 on: no infinity meets it
    const float z = AtMost(y, 128.0f);    // 1 - s is 0 from 88 on
    float s, rest;
    SigmoidParts(z, &s, &rest);
    *a = y * s;
    *d = fmaf(z * s, rest, s);
  } else {
    constexpr float kC = 0.7978845608028654f, kA = 0.044715f;
    const float y = AtLeast(x, -16.0f);  // s is 0 from -11 on
    const float z = AtMost(y, 16.0f);
    const float q = z * z;
    float s, rest;
    SigmoidParts(2.0f * kC * z * fmaf(kA, q, 1.0f), &s, &rest);
    *a = y * s;
    *d = fmaf(z * s, rest * (2.0f * kC * fmaf(3.0f * kA, q, 1.0f)), s);
  }
}

}  // namespace f8
}  // namespace seeml_hip
