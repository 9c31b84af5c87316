// k_f8_lora.hip — a LoRA adapter's gradient from an activation kept in 8 bits:
//
//   out[d, j] = sum_t x^[t, d] dt[t, j]
//
// x^ is e4m3 times a power of two, exact in bfloat16 (below 2^-126 it may count
// as zero), and dt is cut into bfloat16 parts that sum to it exactly (one of
// bfloat16, two of half, three of float32), so the products on the bf16 matrix
// cores are exact and only their float32 sums round.
//
// Bound by reading x^ once: a workgroup takes a block of 128 columns and a range
// of rows, so that every CU has work, and a second kernel sums the ranges in
// order. Rows arrive in 16-byte loads, 64 to 256 of them ahead; the reduction runs along
// rows, so both operands pass through LDS as [t][column] and are read
// transposed (ds_read_b64_tr_b16).
//
// Measured: 8192x2048, rank 16, float32 10.2 us and the join 3.9 (16.8 MB; 11.3 and 8.3 with
// 32 rows between barriers and a join of one load at a time); 2047x1376, rank 64,
// bfloat16 9.1 and 3.4. Bound by latency: two loads' way from memory, then the write and
// the read of the ranges' results.
#include "f8_format.h"

#include <algorithm>

namespace seeml_hip {

using namespace f8;

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;
constexpr int kStep = 32;           // rows of one matrix instruction
constexpr int kRange = 128;         // rows of a range, at least
// Rows between barriers, with as many twice over in registers ahead: as many as
// leave LDS for two workgroups a CU.
constexpr int RowsFor(int tiles) { return tiles <= 2 ? 128 : tiles == 4 ? 64 : 32; }
constexpr int kXLd = kBlock + 32;   // 64 bytes past a multiple of the banks

struct LoraArgs {
  const uint8_t *codes, *scales;
  const void* dt;
  uint64_t dt_stride;
  float* out;  // [ranges][D][r]
  uint32_t T, D, r, rows_per_range;
  uint64_t cols128, rows128;
};

// x as PARTS bfloat16 values that sum to it, by truncation (nothing overflows).
// An infinity or NaN is all in the first.
template <int PARTS>
__device__ __forceinline__ void Parts(float x, uint16_t (&p)[PARTS]) {
  const uint32_t bits = __float_as_uint(x);
  const bool finite = (bits & 0x7F800000u) != 0x7F800000u;
  // A NaN keeps a bit of its payload.
  uint32_t top = bits & 0xFFFF0000u;
  if (!finite && bits & 0x7FFFFFu) top |= 0x400000u;
  p[0] = static_cast<uint16_t>(top >> 16);
  float rest = finite ? x - __uint_as_float(top) : 0.0f;
#pragma unroll
  for (int i = 1; i < PARTS; ++i) {
    const uint32_t b = __float_as_uint(rest) & 0xFFFF0000u;
    p[i] = static_cast<uint16_t>(b >> 16);
    rest -= __uint_as_float(b);
  }
}

typedef __attribute__((address_space(3))) bf16x4 LdsBf16x4;
// 4 rows of one column: 16 lanes name a [4 rows][16 columns] patch.
__device__ __forceinline__ bf16x4 ReadTr(const __bf16* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((LdsBf16x4*)p);
}

// RT column tiles of 16 of dt; wavefront w has columns 32 w .. 32 w + 31 of x^.
template <int DT, int RT>
__global__ __launch_bounds__(kThreads) void lora_grad_f8_kernel(LoraArgs p) {
  using T = typename Elem<DT>::T;
  constexpr int kParts = DT == kF32 ? 3 : DT == kF16 ? 2 : 1;
  constexpr int kRLd = RT * 16 + 32, kRows = RowsFor(RT), kSteps = kRows / kStep;
  __shared__ __align__(16) __bf16 xs[kRows * kXLd];
  __shared__ __align__(16) __bf16 ds[kParts * kRows * kRLd];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t b = blockIdx.x;
  const uint32_t t0 = blockIdx.y * p.rows_per_range, t1 = min(p.T, t0 + p.rows_per_range);

  // x^: a thread has 16 columns of every 32nd row.
  const uint32_t xr = threadIdx.x / 8, xc = threadIdx.x % 8 * 16;
  constexpr int kDt = kRows * RT * 16 / kThreads;  // values of dt a thread has
  struct Ahead {
    uint4 x[kSteps];
    uint32_t xscale[kSteps];
    float d[kDt];
  };
  Ahead a0, a1;
  auto load = [&](Ahead& a, uint32_t t) {
    auto& [x, xscale, d] = a;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const uint32_t row = t + i * kStep + xr;
      const bool in = row < t1;
      const uint32_t at = in ? row : t1 - 1;
      x[i] = *reinterpret_cast<const uint4*>(p.codes + at * p.cols128 + b * kBlock + xc);
      xscale[i] = p.scales[b * p.rows128 + at];
      if (!in) x[i] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kDt; ++i) {
      const uint32_t e = i * kThreads + threadIdx.x, row = t + e / (RT * 16), col = e % (RT * 16);
      const bool in = row < t1 && col < p.r;
      const T* at = static_cast<const T*>(p.dt) + (in ? row * p.dt_stride + col : 0);
      const float v = static_cast<float>(*at);
      d[i] = in ? v : 0.0f;
    }
  };
  auto store = [&](const Ahead& a) {
    const auto& [x, xscale, d] = a;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      float v[16];
      Unpack4(x[i].x, v);
      Unpack4(x[i].y, v + 4);
      Unpack4(x[i].z, v + 8);
      Unpack4(x[i].w, v + 12);
      const float f = ScaleValue(xscale[i]);
      bf16x8 lo, hi;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        lo[e] = static_cast<__bf16>(v[e] * f);
        hi[e] = static_cast<__bf16>(v[8 + e] * f);
      }
      *reinterpret_cast<bf16x8*>(xs + (i * kStep + xr) * kXLd + xc) = lo;
      *reinterpret_cast<bf16x8*>(xs + (i * kStep + xr) * kXLd + xc + 8) = hi;
    }
#pragma unroll
    for (int e = 0; e < kDt; ++e) {
      const uint32_t at = e * kThreads + threadIdx.x, row = at / (RT * 16), col = at % (RT * 16);
      uint16_t part[kParts];
      Parts<kParts>(d[e], part);
#pragma unroll
      for (int k = 0; k < kParts; ++k)
        ds[(k * kRows + row) * kRLd + col] = __builtin_bit_cast(__bf16, part[k]);
    }
  };
  floatx4 acc[2][RT];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int n = 0; n < RT; ++n) acc[i][n] = floatx4{};
  // k = 8 q + 0..7 of a 16 x 16 x 32 product.
  const int tr_row = lane / 16 * 8 + lane % 16 / 4, tr_col = lane % 4 * 4;
  auto fragment = [&](const __bf16* base, int ld) {
    const __bf16* at = base + tr_row * ld + tr_col;
    return __builtin_shufflevector(ReadTr(at), ReadTr(at + 4 * ld), 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto step = [&](Ahead& a, uint32_t t) {
    __syncthreads();
    store(a);
    __syncthreads();
    if (t + 2 * kRows < t1) load(a, t + 2 * kRows);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      bf16x8 fx[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) fx[i] = fragment(xs + s * kStep * kXLd + wave * 32 + i * 16, kXLd);
#pragma unroll
      for (int n = 0; n < RT; ++n)
#pragma unroll
        for (int k = kParts - 1; k >= 0; --k) {  // smallest first
          const bf16x8 fd = fragment(ds + (k * kRows + s * kStep) * kRLd + n * 16, kRLd);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            acc[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fx[i], fd, acc[i][n], 0, 0, 0);
        }
    }
  };
  load(a0, t0);
  if (t0 + kRows < t1) load(a1, t0 + kRows);
  for (uint32_t t = t0; t < t1; t += 2 * kRows) {
    step(a0, t);
    if (t + kRows < t1) step(a1, t + kRows);
  }
  // Rows of a result: d = 4 q + v; its column: j = lane % 16.
  float* out = p.out + static_cast<uint64_t>(blockIdx.y) * p.D * p.r;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int n = 0; n < RT; ++n)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const uint32_t dd = b * kBlock + wave * 32 + i * 16 + lane / 16 * 4 + v, col = n * 16 + lane % 16;
        if (dd < p.D && col < p.r) out[static_cast<uint64_t>(dd) * p.r + col] = acc[i][n][v];
      }
}

// Sums the ranges' results: 64 outputs a workgroup, each wavefront every fourth
// range, eight loads in flight, and the four sums in order.
__global__ __launch_bounds__(kThreads) void lora_join_kernel(const float* part, float* out, uint64_t n,
                                                             uint32_t ranges) {
  __shared__ float sums[kThreads];
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint64_t i = static_cast<uint64_t>(blockIdx.x) * kWave + lane, at = i < n ? i : n - 1;
  float v = 0.0f;
#pragma unroll 8
  for (uint32_t s = wave; s < ranges; s += kThreads / kWave) v += part[s * n + at];
  sums[threadIdx.x] = v;
  __syncthreads();
  if (wave == 0 && i < n) out[i] = sums[lane] + sums[64 + lane] + sums[128 + lane] + sums[192 + lane];
}

// Column tiles of 16 that a rank's kernel has.
uint32_t TilesOf(uint64_t r) { return r <= 16 ? 1 : r <= 32 ? 2 : r <= 64 ? 4 : 8; }
// Ranges of rows, two workgroups a CU, of at least what a workgroup loads ahead (kernel
// traces, us, rank 16: 256x2048 5.9 in one range, 4.4 and the join's 2.4 in two; 512x2048 6.2
// and 2.3 in two, 4.4 and 2.4 in four).
uint32_t RowsPerRange(uint64_t T, uint64_t D, uint64_t r) {
  const uint64_t least = std::max(kRange, 2 * RowsFor(static_cast<int>(TilesOf(r))));
  const uint64_t blocks = Up128(D) / kBlock, units = (T + least - 1) / least;
  const uint64_t want = std::max<uint64_t>(1, std::min<uint64_t>(units, (512 + blocks - 1) / blocks));
  return static_cast<uint32_t>((units + want - 1) / want * least);
}
uint32_t RangesOf(uint64_t T, uint64_t D, uint64_t r) {
  const uint32_t per = RowsPerRange(T, D, r);
  return static_cast<uint32_t>((T + per - 1) / per);
}

template <int DT>
void Launch(const LoraArgs& p, dim3 grid, hipStream_t s) {
  const uint32_t tiles = TilesOf(p.r);
  if (tiles == 1) hipLaunchKernelGGL((lora_grad_f8_kernel<DT, 1>), grid, dim3(kThreads), 0, s, p);
  else if (tiles == 2) hipLaunchKernelGGL((lora_grad_f8_kernel<DT, 2>), grid, dim3(kThreads), 0, s, p);
  else if (tiles == 4) hipLaunchKernelGGL((lora_grad_f8_kernel<DT, 4>), grid, dim3(kThreads), 0, s, p);
  else hipLaunchKernelGGL((lora_grad_f8_kernel<DT, 8>), grid, dim3(kThreads), 0, s, p);
}

}  // namespace

uint64_t GemmTnF8Scratch(uint64_t T, uint64_t D, uint64_t r) {
  const uint64_t n = RangesOf(T, D, r);
  return n > 1 ? n * D * r * sizeof(float) : 0;
}

Status GemmTnF8(const uint8_t* codes, const uint8_t* scales, const void* dt, int dtype, uint64_t dt_stride,
                float* out, uint64_t T, uint64_t D, uint64_t r, void* scratch, const Ctx& c) {
  const uint32_t ranges = RangesOf(T, D, r);
  const LoraArgs p{codes, scales, dt, dt_stride, ranges > 1 ? static_cast<float*>(scratch) : out,
                   static_cast<uint32_t>(T), static_cast<uint32_t>(D), static_cast<uint32_t>(r),
                   RowsPerRange(T, D, r), Up128(D), Up128(T)};
  const dim3 grid(static_cast<unsigned>(Up128(D) / kBlock), ranges);
  if (dtype == kF32) Launch<kF32>(p, grid, c.stream);
  else if (dtype == kBF16) Launch<kBF16>(p, grid, c.stream);
  else Launch<kF16>(p, grid, c.stream);
  if (Status s = LaunchStatus("GemmTnF8"); !s) return s;
  if (ranges == 1) return Status::Ok();
  const uint64_t n = D * r;
  hipLaunchKernelGGL(lora_join_kernel, dim3(static_cast<unsigned>((n + kWave - 1) / kWave)), dim3(kThreads),
                     0, c.stream, static_cast<const float*>(scratch), out, n, ranges);
  return LaunchStatus("GemmTnF8");
}

}  // namespace seeml_hip
