// k_f8_gemm.hip — products of block-scaled 8-bit matrices (f8_format.h) on the
// matrix cores, and the gated feed-forward block as one of them.
//
//   C[m, n] = sum_k a^[m, k] b^[n, k]            (one pair of operands or two, summed)
//   g = x^ Wg, u = x^ Wu, h = act(g) u           (both projections and the product)
//
// Both operands are k-contiguous (a weight is quantised with its transpose), so
// one product serves forward and backward. v_mfma_scale_f32_16x16x128 takes 128
// k of 16 rows a side, exactly a block, and applies both blocks' exponents
// itself: no scaling instruction, one accumulator.
//
// Precision. The 8-bit matrix instruction cuts a block's products about 16 bits
// below the largest (measured against 64 bits: relative 2-norm error 1.5e-5 for
// normal operands, 6e-5 where a row's magnitudes spread over 2^16, whatever K).
// That is well below a 16-bit output's rounding (2^-9 on average of bfloat16's
// 2^-8, 2e-4 of half's), and above a float32 output's, for which codes are
// widened to bfloat16 (exact with the scale, but below 2^-126, where bfloat16 has
// multiples of 2^-133) and multiplied there at half the rate: 1e-7.
#include "f8_format.h"

#include <algorithm>

namespace seeml_hip {

using namespace f8;

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));

constexpr int kXcds = 8;
constexpr int kGroupRows = 8;  // tile rows walked together (L2 panel sharing)

struct TileArgs {
  int pairs;
  const uint8_t *a_codes[2], *a_scales[2], *b_codes[2], *b_scales[2];  // gated: b of g, then of u
  uint32_t M, N;        // gated: N = F
  uint32_t k_blocks;    // of a pair
  uint64_t rows128, cols128;  // M and N rounded up: the scales' row counts
  uint32_t tiles_m, tiles_n;
  uint32_t blocks_per_split, splits;
  float* partial;       // splits > 1: [splits][gated: 2][M][N]
  void* C;
  uint64_t c_stride;
  int act;
  uint8_t *h_codes, *h_scales, *g_codes, *g_scales, *u_codes, *u_scales;
};

__device__ __forceinline__ uint32_t XcdOrder(uint32_t lin, uint32_t total) {
  const uint32_t per = total / kXcds, rem = total % kXcds;
  const uint32_t x = lin % kXcds, idx = lin / kXcds;
  return x < rem ? x * (per + 1) + idx : rem * (per + 1) + (x - rem) * per + idx;
}

// D += W A^T of one block: W supplies the result's rows (n), A its columns (m).
// OW and OA pick the byte of the scale registers.
template <int OW, int OA>
__device__ __forceinline__ floatx4 Mfma(intx8 w, intx8 a, floatx4 c, uint32_t ws, uint32_t as) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, c, 0, 0, OW, static_cast<int>(ws), OA,
                                                         static_cast<int>(as));
}
// The same by bfloat16 products: 32 codes of a lane as four vectors of 8.
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
struct Wide {
  bf16x8 v[4];
};
__device__ __forceinline__ Wide Widen(intx8 w, uint32_t scale_byte) {
  const float s = __uint_as_float(scale_byte << 23);  // its exponent is what counts
  Wide r;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], s, false);
    const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], s, true);
    r.v[i / 2][i % 2 * 4] = lo[0];
    r.v[i / 2][i % 2 * 4 + 1] = lo[1];
    r.v[i / 2][i % 2 * 4 + 2] = hi[0];
    r.v[i / 2][i % 2 * 4 + 3] = hi[1];
  }
  return r;
}
__device__ __forceinline__ floatx4 MfmaWide(const Wide& w, const Wide& a, floatx4 c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[i], a.v[i], c, 0, 0, 0);
  return c;
}
template <int N, typename F>
__device__ __forceinline__ void Static(F&& f) {
  [&]<int... I>(std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>()), ...); }
  (std::make_integer_sequence<int, N>());
}

typedef __attribute__((address_space(3))) uint32_t LdsWord;
typedef const __attribute__((address_space(1))) uint32_t GlobalWord;

// A workgroup of WM x WN wavefronts, each of MI x NI results of 16 x 16.
//
// Slots. LDS holds the tile's rows as 128-byte slots; slot 16 i + j of a
// wavefront's operand is its row j I + i (I = MI or NI), so that the I scales a
// lane needs are adjacent bytes, and a lane's results, (j = 4 q + v, i), are
// 4 I adjacent columns. The 16-byte chunks of slot s lie at chunk ^ (s / 2 % 8):
// the 16 lanes that read at once touch 16 different bank quads. Loads go
// straight to LDS; the permutations are in their global addresses.
//
// GATED: the first half of a wavefront's NI are columns of g, the second the
// same columns of u.
template <int MI, int NI, int WM, int WN, bool GATED>
struct Tile {
  static constexpr int kWaves = WM * WN, kThreads = kWaves * kWave;
  static constexpr int kM = WM * MI * 16, kSlotsN = WN * NI * 16;
  static constexpr int kN = GATED ? kSlotsN / 2 : kSlotsN;  // output columns
  static constexpr int kStage = (kM + kSlotsN) * kBlock;    // bytes
  static constexpr int kLoadsA = kM / 8 / kWaves, kLoadsN = kSlotsN / 8 / kWaves;
  static_assert(kM % (8 * kWaves) == 0 && kSlotsN % (8 * kWaves) == 0);
  static constexpr int kLds = 2 * kStage;
};

// FULL: float32 sums, by bfloat16 products.
template <int DT, bool FULL, int MI, int NI, int WM, int WN, bool GATED, bool SPLIT>
__global__ __launch_bounds__(WM* WN* kWave, 2) void f8_tile_kernel(TileArgs p) {
  using G = Tile<MI, NI, WM, WN, GATED>;
  __shared__ __align__(16) uint8_t smem[G::kLds];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int j = lane % 16, q = lane / 16;

  const uint32_t L = XcdOrder(blockIdx.x, gridDim.x);
  const uint32_t tiles = p.tiles_m * p.tiles_n;
  const uint32_t split = SPLIT ? L / tiles : 0, lt = SPLIT ? L % tiles : L;
  const uint32_t width = kGroupRows * p.tiles_n, group = lt / width;
  const uint32_t high = min(p.tiles_m - group * kGroupRows, static_cast<uint32_t>(kGroupRows));
  const uint32_t m0 = (group * kGroupRows + lt % width % high) * G::kM, n0 = lt % width / high * G::kN;
  const uint64_t ld = static_cast<uint64_t>(p.k_blocks) * kBlock;

  // Offsets of this lane's loads from their matrices; rows past the last are
  // the last's, and reach only outputs that are not stored.
  uint64_t a_at[G::kLoadsA], b_at[G::kLoadsN];
  bool b_u[G::kLoadsN];
#pragma unroll
  for (int i = 0; i < G::kLoadsA; ++i) {
    const uint32_t slot = (i * G::kWaves + wave) * 8 + lane / 8;
    const uint32_t s = slot % (MI * 16);
    const uint32_t row = min(m0 + slot - s + s % 16 * MI + s / 16, p.M - 1);
    a_at[i] = row * ld + ((lane % 8) ^ (slot / 2 % 8)) * 16;
  }
#pragma unroll
  for (int i = 0; i < G::kLoadsN; ++i) {
    const uint32_t slot = (i * G::kWaves + wave) * 8 + lane / 8;
    uint32_t s = slot % (NI * 16), col = slot - s;
    b_u[i] = false;
    if constexpr (GATED) {
      b_u[i] = s >= NI * 8;
      col = col / 2 + s % 16 * (NI / 2) + s / 16 % (NI / 2);
    } else {
      col += s % 16 * NI + s / 16;
    }
    b_at[i] = min(n0 + col, p.N - 1) * ld + ((lane % 8) ^ (slot / 2 % 8)) * 16;
  }
  auto issue = [&](uint32_t t, int buf) {
    const int pair = !GATED && t >= p.k_blocks ? 1 : 0;
    const uint64_t k = static_cast<uint64_t>(t - (pair ? p.k_blocks : 0)) * kBlock;
    uint8_t* lds = smem + buf * G::kStage;
#pragma unroll
    for (int i = 0; i < G::kLoadsA; ++i)
      __builtin_amdgcn_global_load_lds((GlobalWord*)(p.a_codes[pair] + k + a_at[i]),
                                       (LdsWord*)(lds + (i * G::kWaves + wave) * 1024), 16, 0, 0);
#pragma unroll
    for (int i = 0; i < G::kLoadsN; ++i) {
      const uint8_t* b = GATED ? (b_u[i] ? p.b_codes[1] : p.b_codes[0]) : p.b_codes[pair];
      __builtin_amdgcn_global_load_lds((GlobalWord*)(b + k + b_at[i]),
                                       (LdsWord*)(lds + G::kM * kBlock + (i * G::kWaves + wave) * 1024), 16, 0, 0);
    }
  };

  const int wm = wave / WN, wn = wave % WN;
  const uint32_t m_wave = m0 + wm * MI * 16, n_wave = n0 + wn * (GATED ? NI * 8 : NI * 16);
  // The scales of this lane's MI and NI rows; rows past the padding read others.
  constexpr int kNs = GATED ? NI / 2 : NI;  // adjacent ones
  const uint64_t as_at = min(static_cast<uint64_t>(m_wave + j * MI), p.rows128 - MI);
  const uint64_t bs_at = min(static_cast<uint64_t>(n_wave + j * kNs), p.cols128 - kNs);
  constexpr int kAw = (MI + 3) / 4, kBw = (NI + 3) / 4;
  auto scales = [&](uint32_t t, uint32_t (&sa)[kAw], uint32_t (&sb)[kBw]) {
    const int pair = !GATED && t >= p.k_blocks ? 1 : 0;
    const uint64_t k = t - (pair ? p.k_blocks : 0);
    auto get = [](const uint8_t* at, auto bytes, uint32_t* to) {
      if constexpr (decltype(bytes)::value == 8) {
        const uint2 w = *reinterpret_cast<const uint2*>(at);
        to[0] = w.x;
        to[1] = w.y;
      } else if constexpr (decltype(bytes)::value == 4) {
        to[0] = *reinterpret_cast<const uint32_t*>(at);
      } else {
        to[0] = *reinterpret_cast<const uint16_t*>(at);
      }
    };
    get(p.a_scales[pair] + k * p.rows128 + as_at, std::integral_constant<int, MI>(), sa);
    if constexpr (GATED) {
      static_assert(NI == 8);
      get(p.b_scales[0] + k * p.cols128 + bs_at, std::integral_constant<int, kNs>(), &sb[0]);
      get(p.b_scales[1] + k * p.cols128 + bs_at, std::integral_constant<int, kNs>(), &sb[1]);
    } else {
      get(p.b_scales[pair] + k * p.cols128 + bs_at, std::integral_constant<int, NI>(), sb);
    }
  };

  floatx4 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int n = 0; n < NI; ++n) acc[i][n] = floatx4{};

  const int frag0 = j * kBlock + ((q ^ (j >> 1)) * 16), frag1 = frag0 ^ 64;
  auto fragment = [&](const uint8_t* at) {
    const intx4 lo = *reinterpret_cast<const intx4*>(at + frag0);
    const intx4 hi = *reinterpret_cast<const intx4*>(at + frag1);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto compute = [&](int buf, const uint32_t (&sa)[kAw], const uint32_t (&sb)[kBw]) {
    const uint8_t* as = smem + buf * G::kStage + wm * MI * 16 * kBlock;
    const uint8_t* bs = smem + buf * G::kStage + (G::kM + wn * NI * 16) * kBlock;
    if constexpr (FULL) {
      Wide fa[MI];
#pragma unroll
      for (int i = 0; i < MI; ++i) fa[i] = Widen(fragment(as + i * 16 * kBlock), sa[i / 4] >> (i % 4 * 8) & 0xFF);
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        const Wide fb = Widen(fragment(bs + n * 16 * kBlock), sb[n / 4] >> (n % 4 * 8) & 0xFF);
#pragma unroll
        for (int i = 0; i < MI; ++i) acc[i][n] = MfmaWide(fb, fa[i], acc[i][n]);
      }
    } else {
      intx8 fa[MI];
#pragma unroll
      for (int i = 0; i < MI; ++i) fa[i] = fragment(as + i * 16 * kBlock);
      Static<NI>([&](auto n) {
        const intx8 fb = fragment(bs + n * 16 * kBlock);
        Static<MI>([&](auto i) {
          acc[i][n] = Mfma<decltype(n)::value % 4, decltype(i)::value % 4>(fb, fa[i], acc[i][n], sb[n / 4], sa[i / 4]);
        });
      });
    }
  };

  const uint32_t total = p.k_blocks * (GATED ? 1 : p.pairs);
  const uint32_t t0 = SPLIT ? split * p.blocks_per_split : 0;
  const uint32_t t1 = SPLIT ? min(total, t0 + p.blocks_per_split) : total;
  uint32_t sa[kAw], sb[kBw], sa_next[kAw] = {}, sb_next[kBw] = {};
  if (t0 < t1) {
    issue(t0, 0);
    scales(t0, sa, sb);
  }
  for (uint32_t t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    // This wavefront's loads have landed; behind the barrier everyone's have,
    // and everyone has read the other buffer.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t + 1 < t1) {
      issue(t + 1, buf ^ 1);
      scales(t + 1, sa_next, sb_next);
    }
    compute(buf, sa, sb);
#pragma unroll
    for (int i = 0; i < kAw; ++i) sa[i] = sa_next[i];
#pragma unroll
    for (int i = 0; i < kBw; ++i) sb[i] = sb_next[i];
  }

  using T = typename Elem<DT>::T;
  constexpr int kRun = 4 * kNs;  // adjacent columns of a lane
  const uint32_t n_lane = n_wave + q * kRun;
  // A lane's run of row i: half 0 or 1 (GATED: g or u).
  auto run = [&](auto i, int half, float (&v)[kRun]) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int n = 0; n < kNs; ++n) v[r * kNs + n] = acc[i][half * kNs + n][r];
  };
  auto store = [&](auto* row, const float (&v)[kRun], auto dt) {
    constexpr int D = decltype(dt)::value, kE = Elem<D>::E < kRun ? Elem<D>::E : kRun;
    if constexpr (kE == Elem<D>::E) {
#pragma unroll
      for (int c = 0; c < kRun; c += kE) StoreElems<D>(row, n_lane + c, p.N, v + c);
    } else {
#pragma unroll
      for (int c = 0; c < kRun; ++c)
        if (n_lane + c < p.N) row[n_lane + c] = static_cast<typename Elem<D>::T>(v[c]);
    }
  };
  if constexpr (SPLIT) {
    Static<MI>([&](auto i) {
      const uint32_t m = m_wave + j * MI + i;
      if (m >= p.M) return;
      const uint64_t plane = static_cast<uint64_t>(p.M) * p.N;
#pragma unroll
      for (int half = 0; half < (GATED ? 2 : 1); ++half) {
        float v[kRun];
        run(i, half, v);
        store(p.partial + (split * (GATED ? 2 : 1) + half) * plane + static_cast<uint64_t>(m) * p.N, v,
              std::integral_constant<int, kF32>());
      }
    });
  } else if constexpr (!GATED) {
    Static<MI>([&](auto i) {
      const uint32_t m = m_wave + j * MI + i;
      if (m >= p.M) return;
      float v[kRun];
      run(i, 0, v);
      store(static_cast<T*>(p.C) + m * p.c_stride, v, std::integral_constant<int, DT>());
    });
  } else {
    // Largest magnitudes of the tile's rows: a lane's run, the four lanes of a
    // row, the WN wavefronts through LDS.
    float* tops = reinterpret_cast<float*>(smem);  // [3][kM][WN]
    const bool keep = p.g_codes || p.u_codes || p.h_codes;
    auto gate = [&](auto i, float (&g)[kRun], float (&u)[kRun], float (&h)[kRun]) {
      run(i, 0, g);
      run(i, 1, u);
#pragma unroll
      for (int c = 0; c < kRun; ++c) {
        float d;
        if (p.act == 1) ActAndSlope<1>(g[c], &h[c], &d);
        else if (p.act == 2) ActAndSlope<2>(g[c], &h[c], &d);
        else ActAndSlope<3>(g[c], &h[c], &d);
        h[c] *= u[c];
      }
    };
    if (keep) {
      __syncthreads();
      Static<MI>([&](auto i) {
        float v[3][kRun];
        gate(i, v[0], v[1], v[2]);
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          float top = 0.0f;
#pragma unroll
          for (int c = 0; c < kRun; ++c) top = fmaxf(top, n_lane + c < p.N ? FiniteAbs(v[k][c]) : 0.0f);
          top = fmaxf(top, __shfl_xor(top, 16, kWave));
          top = fmaxf(top, __shfl_xor(top, 32, kWave));
          if (q == 0) tops[(k * G::kM + wm * MI * 16 + j * MI + i) * WN + wn] = top;
        }
      });
      __syncthreads();
    }
    Static<MI>([&](auto i) {
      const uint32_t m = m_wave + j * MI + i;
      if (m >= p.M) return;
      float v[3][kRun];
      gate(i, v[0], v[1], v[2]);
      if (p.C) store(static_cast<T*>(p.C) + m * p.c_stride, v[2], std::integral_constant<int, DT>());
      if (!keep) return;
      uint8_t* codes[3] = {p.g_codes, p.u_codes, p.h_codes};
      uint8_t* sc[3] = {p.g_scales, p.u_scales, p.h_scales};
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        if (!codes[k]) continue;
        const float* at = tops + (k * G::kM + wm * MI * 16 + j * MI + i) * WN;
        float top = at[0];
#pragma unroll
        for (int w = 1; w < WN; ++w) top = fmaxf(top, at[w]);
        const uint32_t s = ScaleByte(top);
        const float inv = ScaleInverse(s);
        uint32_t w[kRun / 4];
#pragma unroll
        for (int c = 0; c < kRun; ++c) v[k][c] = n_lane + c < p.N ? v[k][c] * inv : 0.0f;
#pragma unroll
        for (int c = 0; c < kRun / 4; ++c) w[c] = Pack4(v[k][4 * c], v[k][4 * c + 1], v[k][4 * c + 2], v[k][4 * c + 3]);
        uint8_t* to = codes[k] + m * p.cols128 + n_lane;
#pragma unroll
        for (int c = 0; c < kRun / 4; c += 4)
          *reinterpret_cast<uint4*>(to + 4 * c) = make_uint4(w[c], w[c + 1], w[c + 2], w[c + 3]);
        if (q == 0 && wn == 0) {
          uint8_t* row = sc[k] + n0 / kBlock * p.rows128;
          row[m] = static_cast<uint8_t>(s);
          if (m + 1 == p.M)
            for (uint64_t r = p.M; r < p.rows128; ++r) row[r] = 0;
        }
      }
    });
  }
}

// Few rows: a workgroup takes 16 weight rows (GATED: of g and of u) against all
// of A, its wavefronts every eighth block of k; their sums meet in LDS in
// wavefront order. Weights go straight to registers, each read once.
constexpr int kSkinnyWaves = 8;
template <int DT, int MT, bool GATED>
__global__ __launch_bounds__(kSkinnyWaves* kWave) void f8_skinny_kernel(TileArgs p) {
  constexpr bool kFull = DT == kF32;
  constexpr int kHalves = GATED ? 2 : 1;
  __shared__ floatx4 part[kSkinnyWaves][kHalves][MT][kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int j = lane % 16, q = lane / 16;
  const uint32_t n0 = blockIdx.x * 16;
  const uint64_t ld = static_cast<uint64_t>(p.k_blocks) * kBlock;
  const uint32_t n = min(n0 + j, p.N - 1);
  uint32_t m[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) m[i] = min(static_cast<uint32_t>(i * 16 + j), p.M - 1);
  floatx4 acc[kHalves][MT];
#pragma unroll
  for (int h = 0; h < kHalves; ++h)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[h][i] = floatx4{};
  auto load = [&](const uint8_t* at) {
    const intx4 lo = *reinterpret_cast<const intx4*>(at), hi = *reinterpret_cast<const intx4*>(at + 64);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  const uint32_t total = p.k_blocks * (GATED ? 1 : p.pairs);
  for (uint32_t t = wave; t < total; t += kSkinnyWaves) {
    const int pair = !GATED && t >= p.k_blocks ? 1 : 0;
    const uint64_t k = t - (pair ? p.k_blocks : 0);
    intx8 w[kHalves];
    uint32_t ws[kHalves];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      w[h] = load(p.b_codes[GATED ? h : pair] + n * ld + k * kBlock + q * 16);
      ws[h] = p.b_scales[GATED ? h : pair][k * p.cols128 + n];
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const intx8 a = load(p.a_codes[pair] + m[i] * ld + k * kBlock + q * 16);
      const uint32_t as = p.a_scales[pair][k * p.rows128 + m[i]];
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        if constexpr (kFull) acc[h][i] = MfmaWide(Widen(w[h], ws[h]), Widen(a, as), acc[h][i]);
        else acc[h][i] = Mfma<0, 0>(w[h], a, acc[h][i], ws[h], as);
      }
    }
  }
#pragma unroll
  for (int h = 0; h < kHalves; ++h)
#pragma unroll
    for (int i = 0; i < MT; ++i) part[wave][h][i][lane] = acc[h][i];
  __syncthreads();
  if (wave >= MT) return;
  floatx4 sum[kHalves];
#pragma unroll
  for (int h = 0; h < kHalves; ++h) {
    sum[h] = part[0][h][wave][lane];
#pragma unroll
    for (int w = 1; w < kSkinnyWaves; ++w) sum[h] += part[w][h][wave][lane];
  }
  const uint32_t row = wave * 16 + j, col = n0 + q * 4;
  if (row >= p.M) return;
  using T = typename Elem<DT>::T;
  T* out = static_cast<T*>(p.C) + row * p.c_stride;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    float y = sum[0][v];
    if constexpr (GATED) {
      float a, d;
      if (p.act == 1) ActAndSlope<1>(y, &a, &d);
      else if (p.act == 2) ActAndSlope<2>(y, &a, &d);
      else ActAndSlope<3>(y, &a, &d);
      y = a * sum[1][v];
    }
    if (col + v < p.N) out[col + v] = static_cast<T>(y);
  }
}

// Joins the slices of a split reduction, in slice order.
template <int DT>
__global__ __launch_bounds__(256) void f8_join_kernel(TileArgs p) {
  const uint64_t plane = static_cast<uint64_t>(p.M) * p.N;
  const uint64_t i = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= plane) return;
  float v = p.partial[i];
  for (uint32_t s = 1; s < p.splits; ++s) v += p.partial[s * plane + i];
  const uint64_t m = i / p.N;
  static_cast<typename Elem<DT>::T*>(p.C)[m * p.c_stride + (i - m * p.N)] = static_cast<typename Elem<DT>::T>(v);
}
// The same of g and u, with the gate: a wavefront has a block of 128 columns of
// a row, two adjacent ones a lane.
template <int DT>
__global__ __launch_bounds__(256) void f8_gated_join_kernel(TileArgs p) {
  const uint32_t blocks = static_cast<uint32_t>(p.cols128 / kBlock);
  const uint64_t unit = static_cast<uint64_t>(blockIdx.x) * 4 + threadIdx.x / kWave;
  const uint32_t lane = threadIdx.x % kWave;
  const uint64_t m = unit / blocks;
  if (m >= p.M) return;
  const uint32_t b = static_cast<uint32_t>(unit - m * blocks), c0 = b * kBlock + lane * 2;
  const uint64_t plane = static_cast<uint64_t>(p.M) * p.N;
  float v[3][2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const bool in = c0 + e < p.N;
    const uint64_t at = m * p.N + (in ? c0 + e : 0);
    float g = 0.0f, u = 0.0f;
    for (uint32_t s = 0; s < p.splits; ++s) {
      g += p.partial[2 * s * plane + at];
      u += p.partial[(2 * s + 1) * plane + at];
    }
    float a, d;
    if (p.act == 1) ActAndSlope<1>(g, &a, &d);
    else if (p.act == 2) ActAndSlope<2>(g, &a, &d);
    else ActAndSlope<3>(g, &a, &d);
    v[0][e] = in ? g : 0.0f;
    v[1][e] = in ? u : 0.0f;
    v[2][e] = in ? a * u : 0.0f;
    if (p.C && in)
      static_cast<typename Elem<DT>::T*>(p.C)[m * p.c_stride + c0 + e] = static_cast<typename Elem<DT>::T>(v[2][e]);
  }
  uint8_t* codes[3] = {p.g_codes, p.u_codes, p.h_codes};
  uint8_t* sc[3] = {p.g_scales, p.u_scales, p.h_scales};
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    if (!codes[k]) continue;
    const uint32_t s = ScaleByte(wave_max(fmaxf(FiniteAbs(v[k][0]), FiniteAbs(v[k][1]))));
    const float inv = ScaleInverse(s);
    const uint32_t w = Pack4(v[k][0] * inv, v[k][1] * inv, 0.0f, 0.0f);
    *reinterpret_cast<uint16_t*>(codes[k] + m * p.cols128 + c0) = static_cast<uint16_t>(w);
    uint8_t* row = sc[k] + b * p.rows128;
    if (lane == 0) row[m] = static_cast<uint8_t>(s);
    if (m + 1 == p.M)
      for (uint64_t r = p.M + lane; r < p.rows128; r += kWave) row[r] = 0;
  }
}

uint64_t CeilDiv(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// How a product runs. Few rows: the skinny kernel (row groups of 16). Tiles of
// 256 x 256 where they fill the chip, else 128 x 128 (gated: 64 rows of 128
// columns), their reduction split where they leave CUs idle.
struct Choice {
  int skinny = 0;  // 16-row groups: 1, 2 or 4
  bool big = false;
  uint32_t splits = 1, blocks_per_split = 0;
};
constexpr uint64_t kCus = 256;
Choice ChooseF8(uint64_t M, uint64_t N, uint64_t k_blocks, bool gated, bool keep) {
  Choice c;
  if (M <= 64 && !keep) {
    c.skinny = M <= 16 ? 1 : M <= 32 ? 2 : 4;
    return c;
  }
  const uint64_t big = CeilDiv(M, 256) * CeilDiv(N, gated ? 128 : 256);
  c.big = big * 2 >= kCus;
  if (c.big) return c;
  const uint64_t tiles = gated ? CeilDiv(M, 64) * CeilDiv(N, 128) : CeilDiv(M, 128) * CeilDiv(N, 128);
  const uint64_t want = std::min<uint64_t>({CeilDiv(2 * kCus, tiles), k_blocks / 4, 16});
  c.blocks_per_split = static_cast<uint32_t>(CeilDiv(k_blocks, std::max<uint64_t>(want, 1)));
  c.splits = static_cast<uint32_t>(CeilDiv(k_blocks, c.blocks_per_split));
  return c;
}

template <int DT, bool FULL, int MI, int NI, int WM, int WN, bool GATED, bool SPLIT>
Status LaunchTile(TileArgs& p, const Ctx& c, const char* what) {
  using G = Tile<MI, NI, WM, WN, GATED>;
  p.tiles_m = static_cast<uint32_t>(CeilDiv(p.M, G::kM));
  p.tiles_n = static_cast<uint32_t>(CeilDiv(p.N, G::kN));
  const uint64_t groups = static_cast<uint64_t>(p.tiles_m) * p.tiles_n * p.splits;
  if (groups * G::kThreads > 0xFFFFFFFFu) return Status::Fail(kUnitEngine, std::string(what) + ": grid exceeds launch limits");
  auto* kernel = f8_tile_kernel<DT, FULL, MI, NI, WM, WN, GATED, SPLIT>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(groups)), dim3(G::kThreads), 0, c.stream, p);
  return LaunchStatus(what);
}

template <int DT, bool GATED>
Status Run(TileArgs p, const Choice& ch, const Ctx& c, const char* what) {
  constexpr bool kFull = DT == kF32;
  p.splits = ch.splits;
  p.blocks_per_split = ch.blocks_per_split;
  if (ch.skinny) {
    const dim3 grid(static_cast<unsigned>(CeilDiv(p.N, 16))), block(kSkinnyWaves * kWave);
    if (ch.skinny == 1) hipLaunchKernelGGL((f8_skinny_kernel<DT, 1, GATED>), grid, block, 0, c.stream, p);
    else if (ch.skinny == 2) hipLaunchKernelGGL((f8_skinny_kernel<DT, 2, GATED>), grid, block, 0, c.stream, p);
    else hipLaunchKernelGGL((f8_skinny_kernel<DT, 4, GATED>), grid, block, 0, c.stream, p);
    return LaunchStatus(what);
  }
  if (ch.big) return LaunchTile<DT, kFull, 4, 8, 4, 2, GATED, false>(p, c, what);
  constexpr int MI = GATED ? 2 : 4, NI = GATED ? 8 : 4;
  if (ch.splits == 1) return LaunchTile<DT, kFull, MI, NI, 2, 2, GATED, false>(p, c, what);
  // Partials are float32 whatever the output's type.
  if (Status s = LaunchTile<kF32, kFull, MI, NI, 2, 2, GATED, true>(p, c, what); !s) return s;
  if constexpr (GATED) {
    const uint64_t units = static_cast<uint64_t>(p.M) * (p.cols128 / kBlock);
    hipLaunchKernelGGL((f8_gated_join_kernel<DT>), dim3(static_cast<unsigned>(CeilDiv(units, 4))), dim3(256), 0,
                       c.stream, p);
  } else {
    hipLaunchKernelGGL((f8_join_kernel<DT>), dim3(static_cast<unsigned>(CeilDiv(static_cast<uint64_t>(p.M) * p.N, 256))),
                       dim3(256), 0, c.stream, p);
  }
  return LaunchStatus(what);
}
template <bool GATED>
Status RunTyped(int dtype, const TileArgs& p, const Choice& ch, const Ctx& c, const char* what) {
  if (dtype == kF32) return Run<kF32, GATED>(p, ch, c, what);
  if (dtype == kBF16) return Run<kBF16, GATED>(p, ch, c, what);
  return Run<kF16, GATED>(p, ch, c, what);
}

}  // namespace

uint64_t GemmF8Scratch(uint64_t M, uint64_t N, uint64_t K, int pairs) {
  const Choice c = ChooseF8(M, N, Up128(K) / kBlock * pairs, false, false);
  return c.splits > 1 ? c.splits * M * N * sizeof(float) : 0;
}

Status GemmF8(const GemmF8Args& a, const Ctx& c) {
  TileArgs p{};
  p.pairs = a.pairs;
  for (int i = 0; i < a.pairs; ++i) {
    p.a_codes[i] = a.a_codes[i];
    p.a_scales[i] = a.a_scales[i];
    p.b_codes[i] = a.b_codes[i];
    p.b_scales[i] = a.b_scales[i];
  }
  p.M = static_cast<uint32_t>(a.M);
  p.N = static_cast<uint32_t>(a.N);
  p.k_blocks = static_cast<uint32_t>(Up128(a.K) / kBlock);
  p.rows128 = Up128(a.M);
  p.cols128 = Up128(a.N);
  p.partial = static_cast<float*>(a.scratch);
  p.C = a.C;
  p.c_stride = a.c_stride;
  return RunTyped<false>(a.dtype, p, ChooseF8(a.M, a.N, static_cast<uint64_t>(p.k_blocks) * a.pairs, false, false), c, "GemmF8");
}

uint64_t GatedF8Scratch(uint64_t T, uint64_t D, uint64_t F) {
  uint64_t most = GemmF8Scratch(T, D, F, 2);  // the backward's product
  for (const bool keep : {false, true}) {
    const Choice c = ChooseF8(T, F, Up128(D) / kBlock, true, keep);
    if (c.splits > 1) most = std::max<uint64_t>(most, 2 * c.splits * T * F * sizeof(float));
  }
  return most;
}

Status GatedF8Fwd(const GatedF8FwdArgs& a, const Ctx& c) {
  TileArgs p{};
  p.pairs = 1;
  p.a_codes[0] = a.x_codes;
  p.a_scales[0] = a.x_scales;
  p.b_codes[0] = a.wg_codes;
  p.b_scales[0] = a.wg_scales;
  p.b_codes[1] = a.wu_codes;
  p.b_scales[1] = a.wu_scales;
  p.M = static_cast<uint32_t>(a.T);
  p.N = static_cast<uint32_t>(a.F);
  p.k_blocks = static_cast<uint32_t>(Up128(a.D) / kBlock);
  p.rows128 = Up128(a.T);
  p.cols128 = Up128(a.F);
  p.partial = static_cast<float*>(a.scratch);
  p.C = a.h;
  p.c_stride = a.h_stride;
  p.act = a.act;
  p.h_codes = a.h_codes;
  p.h_scales = a.h_scales;
  p.g_codes = a.g_codes;
  p.g_scales = a.g_scales;
  p.u_codes = a.u_codes;
  p.u_scales = a.u_scales;
  const bool keep = a.h_codes || a.g_codes || a.u_codes;
  return RunTyped<true>(a.dtype, p, ChooseF8(a.T, a.F, p.k_blocks, true, keep), c, "GatedF8Fwd");
}

}  // namespace seeml_hip
