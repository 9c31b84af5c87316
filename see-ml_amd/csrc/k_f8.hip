// k_f8.hip — the row-wise kernels of the block-scaled 8-bit format (f8_format.h):
// quantising, reading back, and the backward passes that read a checkpoint.
//
//   dx = dy a'(x^)                                          (activation)
//   dx = r (gamma dy - r x^ mean(gamma dy r x^))            (RMS norm)
//   dg = dh u^ a'(g^), du = dh a(g^), both kept in 8 bits   (gated block)
//
// All are bound by memory, but for GELU's gradient in 16 bits, by its arithmetic. A unit is
// 16 bytes of the call's type (4 or 8 values) and as many codes; a thread has one of them:
// the CUs' many wavefronts keep memory busy, and more of them a thread was slower throughout
// (quantising 8192x2048 bfloat16 in 1, 2, 4, 8 units a thread 9.9, 10.2, 11.7, 12.2 us; GELU's
// gradient of 8192x16384 float32 196, 199, 209, 223). The lanes of a block of 128 are a row
// of 16 (16-bit types) or two (float32).
//
// Measured (kernel traces): quantising 8192x16384 float32 116 us (5.8 TB/s), 8192x2048 15.2
// (5.5), of bfloat16 10.2 (5.0); reading back 126 (5.3) and 10.2; a weight and its transpose,
// float32, 2048x5504 15.0 (4.5), 4096x16384 101 (4.0); GELU's gradient of 8192x16384 197 (6.1), of
// bfloat16 127 (5.3); the norm's of 8192x2048 27.6 (5.5), of bfloat16 17.6 (4.8); the gated block's
// of 8192x5504 bfloat16 53 (5.1), float32 63 (5.7). 777x1003 f16: 5.4, latency.
#include "f8_format.h"

#include <type_traits>

namespace seeml_hip {

using namespace f8;

namespace {

constexpr int kThreads = 256;

// n / d for n < 2^31 by a multiplication: d > 2^s, m = ceil(2^(32 + s) / d), so
// that m d - 2^(32 + s) < d <= 2^(s + 1).
struct Divider {
  uint32_t d, m, s;
};
Divider DividerOf(uint64_t d) {
  uint32_t s = 0;
  while ((uint64_t{2} << s) < d) ++s;
  return {static_cast<uint32_t>(d), static_cast<uint32_t>(((uint64_t{1} << (32 + s)) + d - 1) / d), s};
}
__device__ __forceinline__ uint32_t Quotient(uint32_t n, Divider v) { return __umulhi(n, v.m) >> v.s; }

// The largest of v over the lanes that share a block of 128.
template <int LANES>
__device__ __forceinline__ float LaneMax(float v) {
  // Rotations within a row of 16.
  auto ror = [](float x, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  v = fmaxf(v, ror(v, std::integral_constant<int, 0x128>()));
  v = fmaxf(v, ror(v, std::integral_constant<int, 0x124>()));
  v = fmaxf(v, ror(v, std::integral_constant<int, 0x122>()));
  v = fmaxf(v, ror(v, std::integral_constant<int, 0x121>()));
  if constexpr (LANES == 32) v = fmaxf(v, __shfl_xor(v, 16, kWave));
  return v;
}

// E values of a unit as codes with their block's scale byte, stored: unit q
// of `row`, whose codes are `code_row`. The last row's lanes also clear the
// scales of the rows past it. mend() is called where a value is not finite and may
// change it.
template <int E, typename F = Nothing>
__device__ __forceinline__ void StoreUnit(const float (&v)[E], uint8_t* code_row, uint8_t* scales,
                                          uint64_t rows128, uint32_t row, uint32_t rows, uint32_t q, F&& mend = F()) {
  constexpr int kLanes = kBlock / E;
  const uint32_t s = ScaleByte(LaneMax<kLanes>(FiniteMax(v, mend)));
  const float inv = ScaleInverse(s);
  uint32_t w[E / 4];
#pragma unroll
  for (int i = 0; i < E / 4; ++i)
    w[i] = Pack4(v[4 * i] * inv, v[4 * i + 1] * inv, v[4 * i + 2] * inv, v[4 * i + 3] * inv);
  if constexpr (E == 4) {
    reinterpret_cast<uint32_t*>(code_row)[q] = w[0];
  } else {
    reinterpret_cast<uint2*>(code_row)[q] = make_uint2(w[0], w[1]);
  }
  uint8_t* at = scales + (q / kLanes) * rows128;
  if (q % kLanes == 0) at[row] = static_cast<uint8_t>(s);
  if (row + 1 == rows)
    for (uint64_t r = rows + q % kLanes; r < rows128; r += kLanes) at[r] = 0;
}
template <int E>
__device__ __forceinline__ void LoadUnit(const uint8_t* code_row, const uint8_t* scales, uint64_t rows128,
                                         uint32_t row, uint32_t q, float (&v)[E]) {
  const float f = ScaleValue(scales[(q / (kBlock / E)) * rows128 + row]);
  if constexpr (E == 4) {
    Unpack4(reinterpret_cast<const uint32_t*>(code_row)[q], v);
  } else {
    const uint2 w = reinterpret_cast<const uint2*>(code_row)[q];
    Unpack4(w.x, v);
    Unpack4(w.y, v + 4);
  }
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] *= f;
}

struct UnitGrid {
  uint32_t units;  // of the whole matrix
  Divider per_row;
  uint32_t rows, cols;
  uint64_t cols128, rows128;
};
template <int DT>
UnitGrid GridOf(uint64_t rows, uint64_t cols) {
  const uint64_t per = Up128(cols) / Elem<DT>::E;
  return {static_cast<uint32_t>(rows * per), DividerOf(per), static_cast<uint32_t>(rows),
          static_cast<uint32_t>(cols), Up128(cols), Up128(rows)};
}
dim3 BlocksOf(const UnitGrid& g) { return dim3((g.units + kThreads - 1) / kThreads); }

// f(row, unit of the row) for this thread's unit. Whole lanes of a block are in
// range together (kBlock / E divides the units of a row).
template <typename F>
__device__ __forceinline__ void AtUnit(const UnitGrid& g, F&& f) {
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= g.units) return;
  const uint32_t row = Quotient(i, g.per_row);
  f(row, i - row * g.per_row.d);
}

template <int DT>
__global__ __launch_bounds__(kThreads) void f8_quantize_kernel(const typename Elem<DT>::T* x, uint64_t stride,
                                                               UnitGrid g, uint8_t* codes, uint8_t* scales) {
  constexpr int E = Elem<DT>::E;
  AtUnit(g, [&](uint32_t row, uint32_t q) {
    float v[E];
    LoadElems<DT>(x + row * stride, q * E, g.cols, v);
    StoreUnit<E>(v, codes + row * g.cols128, scales, g.rows128, row, g.rows, q);
  });
}

template <int DT>
__global__ __launch_bounds__(kThreads) void f8_dequantize_kernel(const uint8_t* codes, const uint8_t* scales,
                                                                 UnitGrid g, typename Elem<DT>::T* x,
                                                                 uint64_t stride) {
  constexpr int E = Elem<DT>::E;
  AtUnit(g, [&](uint32_t row, uint32_t q) {
    float v[E];
    LoadUnit<E>(codes + row * g.cols128, scales, g.rows128, row, q, v);
    StoreElems<DT>(x + row * stride, q * E, g.cols, v);
  });
}

// dy and dx may be the same.
template <int DT, int ACT>
__global__ __launch_bounds__(kThreads) void act_bwd_f8_kernel(const typename Elem<DT>::T* dy, uint64_t dy_stride,
                                                              const uint8_t* codes, const uint8_t* scales,
                                                              UnitGrid g, typename Elem<DT>::T* dx,
                                                              uint64_t dx_stride) {
  constexpr int E = Elem<DT>::E;
  AtUnit(g, [&](uint32_t row, uint32_t q) {
    float x[E], v[E];
    LoadUnit<E>(codes + row * g.cols128, scales, g.rows128, row, q, x);
    LoadElems<DT>(dy + row * dy_stride, q * E, g.cols, v);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      float a, d;
      ActAndSlope<ACT>(x[i], &a, &d);
      v[i] *= d;
    }
    StoreElems<DT>(dx + row * dx_stride, q * E, g.cols, v);
  });
}

// The gated block's elementwise backward. h, where asked for, is act(g^) u^.
template <int DT, int ACT, bool H>
__global__ __launch_bounds__(kThreads) void gated_bwd_f8_kernel(GatedF8BwdArgs p, UnitGrid g) {
  constexpr int E = Elem<DT>::E;
  using T = typename Elem<DT>::T;
  AtUnit(g, [&](uint32_t row, uint32_t q) {
    float dh[E], gv[E], uv[E], dg[E], du[E], hv[E], slope[E];
    LoadElems<DT>(static_cast<const T*>(p.dh) + row * p.dh_stride, q * E, g.cols, dh);
    LoadUnit<E>(p.g_codes + row * g.cols128, p.g_scales, g.rows128, row, q, gv);
    LoadUnit<E>(p.u_codes + row * g.cols128, p.u_scales, g.rows128, row, q, uv);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      float a;
      ActAndSlope<ACT>(gv[i], &a, &slope[i]);
      hv[i] = a * uv[i];
      du[i] = dh[i] * a;
      dg[i] = dh[i] * uv[i] * slope[i];
    }
    // Where dh u passes the range, the slope goes first: it is at most 1.13 and may be 0.
    // (Everywhere, dh act'(g) would be lost where u is large.)
    auto slope_first = [&] {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (!(fabsf(dh[i] * uv[i]) <= FLT_MAX)) dg[i] = dh[i] * slope[i] * uv[i];
    };
    if constexpr (H) StoreElems<DT>(static_cast<T*>(p.h) + row * p.h_stride, q * E, g.cols, hv);
    StoreUnit<E>(dg, p.dg_codes + row * g.cols128, p.dg_scales, g.rows128, row, g.rows, q, slope_first);
    StoreUnit<E>(du, p.du_codes + row * g.cols128, p.du_scales, g.rows128, row, g.rows, q);
  });
}

// One row per TPR threads, its units held in registers (HELD of them a thread),
// or read a second time (HELD = 0). dy and dx may be the same: a thread writes
// only what it alone has read.
template <int DT, int TPR, int HELD>
__global__ __launch_bounds__(kThreads) void rms_norm_bwd_f8_kernel(
    const typename Elem<DT>::T* dy, uint64_t dy_stride, const uint8_t* codes, const uint8_t* scales,
    const float* gamma, const float* rstd, typename Elem<DT>::T* dx, uint64_t dx_stride, uint32_t rows,
    uint32_t cols, uint32_t units, uint64_t rows128) {
  constexpr int E = Elem<DT>::E, kHold = HELD ? HELD : 1;
  __shared__ double part[kThreads / kWave];
  const uint32_t t = threadIdx.x % TPR;
  const uint32_t row = blockIdx.x * (kThreads / TPR) + threadIdx.x / TPR;
  if (TPR <= kWave && row >= rows) return;  // whole wavefronts, and no barrier follows
  const uint8_t* code_row = codes + static_cast<uint64_t>(row) * units * E;
  const auto* dy_row = dy + row * dy_stride;
  const float rf = rstd[row];
  float g[kHold][E], x[kHold][E];
  // gamma dy and x^ r. The normalised x is near 1 whatever x is, so that products with
  // it, their sum and the coefficient stay in float32's range where gamma dy does.
  auto load = [&](uint32_t q, float (&gv)[E], float (&xv)[E]) {
    float w[E];
    LoadUnit<E>(code_row, scales, rows128, row, q, xv);
    LoadElems<DT>(dy_row, q * E, cols, gv);
    LoadElems<kF32>(gamma, q * E, cols, w);
    if constexpr (E == 8) LoadElems<kF32>(gamma, q * E + 4, cols, w + 4);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      gv[i] *= w[i];
      xv[i] *= rf;
    }
  };
  // Partial sums of a thread in float32 (of a unit), then in 64 bits.
  double dot = 0.0;
  auto add = [&](const float (&gv)[E], const float (&xv)[E]) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) s = fmaf(gv[i], xv[i], s);
    dot += s;
  };
  if constexpr (HELD > 0) {
#pragma unroll
    for (int k = 0; k < kHold; ++k)
      if (t + k * TPR < units) load(t + k * TPR, g[k], x[k]);
#pragma unroll
    for (int k = 0; k < kHold; ++k)
      if (t + k * TPR < units) add(g[k], x[k]);
  } else {
    for (uint32_t q = t; q < units; q += TPR) {
      load(q, g[0], x[0]);
      add(g[0], x[0]);
    }
  }
  if constexpr (TPR <= kWave) {
    dot = wave_sum(dot);
  } else {
    dot = block_sum<double, kThreads>(dot, part);
  }
  const float c = static_cast<float>(dot / cols);
  auto store = [&](uint32_t q, float (&gv)[E], const float (&xv)[E]) {
#pragma unroll
    for (int i = 0; i < E; ++i) gv[i] = rf * (gv[i] - xv[i] * c);
    StoreElems<DT>(dx + row * dx_stride, q * E, cols, gv);
  };
  if constexpr (HELD > 0) {
#pragma unroll
    for (int k = 0; k < kHold; ++k)
      if (t + k * TPR < units) store(t + k * TPR, g[k], x[k]);
  } else {
    for (uint32_t q = t; q < units; q += TPR) {
      load(q, g[0], x[0]);
      store(q, g[0], x[0]);
    }
  }
}

// A 128 x 128 block of a weight, its codes as they lie and transposed. Run once
// per weight.
template <int DT>
__global__ __launch_bounds__(kThreads) void f8_quantize_weight_kernel(const typename Elem<DT>::T* w,
                                                                      uint64_t stride, uint32_t rows,
                                                                      uint32_t cols, uint32_t col_blocks,
                                                                      uint8_t* codes, uint8_t* scales,
                                                                      uint8_t* codes_t, uint8_t* scales_t) {
  constexpr int E = Elem<DT>::E, kPerRow = kBlock / E, kRows = kThreads / kPerRow, kSteps = kBlock / kRows;
  constexpr int kLd = kBlock + 4;
  __shared__ uint32_t tile[kBlock * kLd / 4];
  __shared__ float tops[kThreads / kWave];
  const uint32_t rb = blockIdx.x / col_blocks, cb = blockIdx.x % col_blocks;
  const uint32_t q = threadIdx.x % kPerRow, r0 = threadIdx.x / kPerRow;
  const uint32_t c = cb * kBlock + q * E;
  float v[kSteps][E];
  float top = 0.0f;
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const uint32_t row = rb * kBlock + r0 + k * kRows;
    if (row < rows) {
      LoadElems<DT>(w + row * stride, c, cols, v[k]);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) v[k][i] = 0.0f;
    }
    top = fmaxf(top, FiniteMax(v[k]));
  }
  const uint32_t s = ScaleByte(block_max<kThreads>(top, tops));
  const float inv = ScaleInverse(s);
  const uint64_t rows128 = Up128(rows), cols128 = Up128(cols);
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const uint32_t r = r0 + k * kRows, row = rb * kBlock + r;
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      const uint32_t p = Pack4(v[k][i] * inv, v[k][i + 1] * inv, v[k][i + 2] * inv, v[k][i + 3] * inv);
      tile[(r * kLd + q * E + i) / 4] = p;
      if (codes && row < rows) *reinterpret_cast<uint32_t*>(codes + row * cols128 + c + i) = p;
    }
  }
  if (threadIdx.x < kBlock) {
    const uint32_t i = threadIdx.x;
    const uint8_t byte = static_cast<uint8_t>(s);
    if (codes) scales[cb * rows128 + rb * kBlock + i] = rb * kBlock + i < rows ? byte : 0;
    if (codes_t) scales_t[rb * cols128 + cb * kBlock + i] = cb * kBlock + i < cols ? byte : 0;
  }
  if (!codes_t) return;
  __syncthreads();
  const uint8_t* bytes = reinterpret_cast<const uint8_t*>(tile);
  const uint32_t tc = threadIdx.x / 2, half = threadIdx.x % 2 * 64;
  if (cb * kBlock + tc >= cols) return;
  uint8_t* out = codes_t + (cb * kBlock + tc) * rows128 + rb * kBlock + half;
  for (int i = 0; i < 64; i += 4) {
    uint32_t p = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) p |= static_cast<uint32_t>(bytes[(half + i + j) * kLd + tc]) << (8 * j);
    *reinterpret_cast<uint32_t*>(out + i) = p;
  }
}

// f(type tag) for the runtime type / activation; arguments are checked before.
template <typename F>
void WithType(int dtype, F&& f) {
  if (dtype == kF32) f(std::integral_constant<int, kF32>());
  else if (dtype == kBF16) f(std::integral_constant<int, kBF16>());
  else f(std::integral_constant<int, kF16>());
}
template <typename F>
void WithAct(int act, F&& f) {
  if (act == 1) f(std::integral_constant<int, 1>());
  else if (act == 2) f(std::integral_constant<int, 2>());
  else f(std::integral_constant<int, 3>());
}

}  // namespace

Status F8Quantize(const void* x, int dtype, uint64_t stride, uint64_t rows, uint64_t cols, uint8_t* codes,
                  uint8_t* scales, const Ctx& c) {
  WithType(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const UnitGrid g = GridOf<DT>(rows, cols);
    hipLaunchKernelGGL((f8_quantize_kernel<DT>), BlocksOf(g), dim3(kThreads), 0, c.stream,
                       static_cast<const typename Elem<DT>::T*>(x), stride, g, codes, scales);
  });
  return LaunchStatus("F8Quantize");
}

Status F8QuantizeWeight(const void* w, int dtype, uint64_t stride, uint64_t rows, uint64_t cols,
                        uint8_t* codes, uint8_t* scales, uint8_t* codes_t, uint8_t* scales_t, const Ctx& c) {
  const uint32_t rb = static_cast<uint32_t>(Up128(rows) / kBlock), cb = static_cast<uint32_t>(Up128(cols) / kBlock);
  WithType(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    hipLaunchKernelGGL((f8_quantize_weight_kernel<DT>), dim3(rb * cb), dim3(kThreads), 0, c.stream,
                       static_cast<const typename Elem<DT>::T*>(w), stride, static_cast<uint32_t>(rows),
                       static_cast<uint32_t>(cols), cb, codes, scales, codes_t, scales_t);
  });
  return LaunchStatus("F8QuantizeWeight");
}

Status F8Dequantize(const uint8_t* codes, const uint8_t* scales, void* x, int dtype, uint64_t stride,
                    uint64_t rows, uint64_t cols, const Ctx& c) {
  WithType(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const UnitGrid g = GridOf<DT>(rows, cols);
    hipLaunchKernelGGL((f8_dequantize_kernel<DT>), BlocksOf(g), dim3(kThreads), 0, c.stream, codes, scales, g,
                       static_cast<typename Elem<DT>::T*>(x), stride);
  });
  return LaunchStatus("F8Dequantize");
}

Status ActBwdF8(const void* dy, int dtype, uint64_t dy_stride, const uint8_t* codes, const uint8_t* scales,
                int act, void* dx, uint64_t dx_stride, uint64_t rows, uint64_t cols, const Ctx& c) {
  WithType(dtype, [&](auto dt) {
    WithAct(act, [&](auto at) {
      constexpr int DT = decltype(dt)::value, ACT = decltype(at)::value;
      using T = typename Elem<DT>::T;
      const UnitGrid g = GridOf<DT>(rows, cols);
      hipLaunchKernelGGL((act_bwd_f8_kernel<DT, ACT>), BlocksOf(g), dim3(kThreads), 0, c.stream,
                         static_cast<const T*>(dy), dy_stride, codes, scales, g, static_cast<T*>(dx), dx_stride);
    });
  });
  return LaunchStatus("ActBwdF8");
}

Status RmsNormBwdF8(const void* dy, int dtype, uint64_t dy_stride, const uint8_t* codes, const uint8_t* scales,
                    const float* gamma, const float* rstd, void* dx, uint64_t dx_stride, uint64_t rows,
                    uint64_t cols, const Ctx& c) {
  WithType(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    using T = typename Elem<DT>::T;
    const uint32_t units = static_cast<uint32_t>(Up128(cols) / Elem<DT>::E);
    auto launch = [&](auto tpr, auto held) {
      constexpr int TPR = decltype(tpr)::value, HELD = decltype(held)::value;
      constexpr uint64_t kRows = kThreads / TPR;
      hipLaunchKernelGGL((rms_norm_bwd_f8_kernel<DT, TPR, HELD>),
                         dim3(static_cast<unsigned>((rows + kRows - 1) / kRows)), dim3(kThreads), 0, c.stream,
                         static_cast<const T*>(dy), dy_stride, codes, scales, gamma, rstd, static_cast<T*>(dx),
                         dx_stride, static_cast<uint32_t>(rows), static_cast<uint32_t>(cols), units, Up128(rows));
    };
    using std::integral_constant;
    if (units <= 64) launch(integral_constant<int, 64>(), integral_constant<int, 1>());
    else if (units <= 128) launch(integral_constant<int, 64>(), integral_constant<int, 2>());
    else if (units <= 256) launch(integral_constant<int, 256>(), integral_constant<int, 1>());
    else if (units <= 512) launch(integral_constant<int, 256>(), integral_constant<int, 2>());
    else if (units <= 1024) launch(integral_constant<int, 256>(), integral_constant<int, 4>());
    else launch(integral_constant<int, 256>(), integral_constant<int, 0>());
  });
  return LaunchStatus("RmsNormBwdF8");
}

Status GatedF8BwdRows(const GatedF8BwdArgs& a, const Ctx& c) {
  WithType(a.dtype, [&](auto dt) {
    WithAct(a.act, [&](auto at) {
      constexpr int DT = decltype(dt)::value, ACT = decltype(at)::value;
      const UnitGrid g = GridOf<DT>(a.T, a.F);
      if (a.h)
        hipLaunchKernelGGL((gated_bwd_f8_kernel<DT, ACT, true>), BlocksOf(g), dim3(kThreads), 0, c.stream, a, g);
      else
        hipLaunchKernelGGL((gated_bwd_f8_kernel<DT, ACT, false>), BlocksOf(g), dim3(kThreads), 0, c.stream, a, g);
    });
  });
  return LaunchStatus("GatedF8Bwd");
}

}  // namespace seeml_hip
