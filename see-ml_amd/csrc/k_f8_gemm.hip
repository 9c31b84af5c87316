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
// That is a hundredth of bfloat16's rounding (1.6e-3 in the 2-norm) and a tenth of
// half's (2e-4), up to a third of half's where magnitudes spread: 16-bit outputs take
// it, for twice the rate. A float32 output's rounding is far below, so for it codes are
// widened to bfloat16 (exact with the scale, but below 2^-126, where bfloat16 has
// multiples of 2^-133) and multiplied there at half the rate: 1e-7. So are products
// whose results are kept in 8 bits: 1.5e-5 moves one value in 7000 across the
// border between two codes, and a gated block's dx by 1.3e-3 in all.
//
// Measured (kernel traces, the card settled: the first thirty calls of a burst take up to
// 40% longer; largest library products 2711 TFLOP/s in 8 bits and 1439 in bfloat16):
// 8192x8192x8192 421 us (2613 TFLOP/s) and with float32 sums 772 (1424); 8192x2048x5504 (M, K,
// N) to bfloat16 91-94, to float32 162; two pairs of 8192x5504x2048 141-148; gated
// 8192x2048x5504 173 without checkpoints, 307 with. At 8192 cubed the matrix cores are busy
// 57% of the cycles (61% with float32 sums) at a clock that GRBM_GUI_ACTIVE puts at 1.9 GHz,
// of 2.4, and the library's rate is the same within 4%; at K = 2048 (40%) the end of each
// tile counts too: all CUs write 128 KiB at once, more than the L2s take (12% with the stores
// left out), and last rounds are partly filled. Small calls are bound by the latency of a
// step (0.6 us with the small tiles, 1.05 with float32 sums).
//
// Tried and not kept: persistent workgroups that load the next tile behind the
// write-back (8192x2048x5504 the same, gated 220 -> 244 us: their first step waits for the
// stores); non-temporal stores (float32 output 162 -> 226); asking for the lines of the
// step after the next, so that they come from the L2 (8192x8192x8192 430 -> 463); a fixed order of
// reads and products by the scheduler's group barriers (no change); two blocks of k ahead in
// the few-row kernel (5.9 -> 6.4).
#include "f8_choice.h"
#include "f8_format.h"

#include <type_traits>
#include <utility>

namespace seeml_hip {

using namespace f8;

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));

constexpr int kXcds = 8;
// Tile rows walked together, which share panels in an L2 (8192x8192x8192: 4, 8, 16, 32 rows 422,
// 418, 432, 545 us).
constexpr int kGroupRows = 8;

struct TileArgs {
  int pairs;
  const uint8_t *a_codes[2], *a_scales[2], *b_codes[2], *b_scales[2];  // gated: b of g, then of u
  uint32_t M, N;        // gated: N = F
  uint32_t k_blocks;    // of a pair
  uint64_t rows128, cols128;  // M and N rounded up: the scales' row counts
  uint32_t tiles_m, tiles_n;
  uint32_t first_n;     // column of the launch's first tile
  uint32_t blocks_per_split, splits;
  float* partial;       // splits > 1: [splits][M][N]
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
// BYTES a lane straight to LDS, lane after lane: one 64-bit base for all lanes, an
// offset for each.
template <int BYTES>
__device__ __forceinline__ void LoadToLds(const uint8_t* base, uint32_t at, uint8_t* to) {
#ifdef __HIP_DEVICE_COMPILE__
  const __amdgpu_buffer_rsrc_t r =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, 0xFFFFFFFFu, 0x00020000);
  static_assert(BYTES == 16 || BYTES == 4);
  if constexpr (BYTES == 16) __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LdsWord*)to, 16, at, 0, 0, 0);
  else __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LdsWord*)to, 4, at, 0, 0, 0);
#endif
}

// N adjacent elements of a row, short of column `cols`.
template <int DT, int N>
__device__ __forceinline__ void StoreRun(typename Elem<DT>::T* row, uint32_t c, uint32_t cols, const float (&v)[N]) {
  constexpr int E = Elem<DT>::E;
  if constexpr (N % E == 0) {
#pragma unroll
    for (int i = 0; i < N; i += E) StoreElems<DT>(row, c + i, cols, v + i);
  } else {
    using T = typename Elem<DT>::T;
    typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    if (c + N <= cols) {
      vec t;
#pragma unroll
      for (int i = 0; i < N; ++i) t[i] = static_cast<T>(v[i]);
      *reinterpret_cast<vec*>(row + c) = t;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (c + i < cols) row[c + i] = static_cast<T>(v[i]);
    }
  }
}

// A workgroup of WM x WN wavefronts, each of MI x NI results of 16 x 16.
//
// Slots. LDS holds the tile's rows as 128-byte slots. Slot 16 i + j of a
// wavefront's rows of A is its row j MI + i, so that the MI scales a lane needs are
// adjacent bytes. Of its rows of B (columns of C) slot 16 i + j, j = 4 q + v, is column
// 4 v I + q I + i (I = NI): the scales are adjacent too, a lane's results are four runs
// of I adjacent columns, and the four lanes of a row store 4 I adjacent ones at once.
// The 16-byte chunks of slot s lie at chunk ^ (s / 2 % 8): the 16 lanes that read at
// once touch 16 different bank quads: no conflicts are counted (3% of the LDS's cycles in
// the gated block with 8-bit outputs, where row maxima meet). Loads go straight to
// LDS; the permutations are in their global addresses.
//
// GATED: the first half of a wavefront's NI are columns of g, the second the
// same columns of u, and I = NI / 2 with column 4 q I + v I + i: one run of 4 I, whose codes
// are one store.
template <int MI, int NI, int WM, int WN, int STAGES, bool GATED>
struct Tile {
  static constexpr int kWaves = WM * WN, kThreads = kWaves * kWave;
  static constexpr int kM = WM * MI * 16, kSlotsN = WN * NI * 16;
  static constexpr int kN = GATED ? kSlotsN / 2 : kSlotsN;  // output columns
  static constexpr int kLoadsA = kM / 8 / kWaves, kLoadsN = kSlotsN / 8 / kWaves;
  static_assert(kM % (8 * kWaves) == 0 && kSlotsN % (8 * kWaves) == 0);
  static constexpr int kLoads = kLoadsA + kLoadsN + 1;  // of a wavefront and stage
  static constexpr int kScalesA = (kM + kSlotsN) * kBlock, kScalesN = kScalesA + 256;
  static_assert(kM <= 256 && kSlotsN <= 256 && kWaves % 2 == 0);
  static constexpr int kScalesU = kScalesN + 256;  // GATED
  static_assert(!GATED || kWaves % 4 == 0);
  static constexpr int kStage = kScalesU + (GATED ? 256 : 0);  // bytes
  static constexpr int kTops = STAGES * kStage;  // GATED: [3][kM][WN] float
  static constexpr int kLds = kTops + (GATED ? 3 * kM * WN * 4 : 0);
};

// FULL: float32 sums, by bfloat16 products.
//
// A workgroup has one tile (and, SPLIT, one range of k), its loads up to STAGES steps of
// 128 k ahead.
template <int DT, bool FULL, int MI, int NI, int WM, int WN, int STAGES, bool GATED, bool SPLIT>
__global__ __launch_bounds__(WM* WN* kWave, WM* WN / 4) void f8_tile_kernel(TileArgs p) {
  using G = Tile<MI, NI, WM, WN, STAGES, GATED>;
  __shared__ __align__(16) uint8_t smem[G::kLds];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int j = lane % 16, q = lane / 16;
  const int wm = wave / WN, wn = wave % WN;
  const uint32_t tiles = p.tiles_m * p.tiles_n, all = tiles * (SPLIT ? p.splits : 1);
  const uint64_t ld = static_cast<uint64_t>(p.k_blocks) * kBlock;
  const uint32_t k_steps = p.k_blocks * (GATED ? 1 : p.pairs);

  const uint32_t L = XcdOrder(blockIdx.x, all);
  const uint32_t split = SPLIT ? L / tiles : 0, lt = SPLIT ? L % tiles : L;
  const uint32_t width = kGroupRows * p.tiles_n, group = lt / width;
  const uint32_t high = min(p.tiles_m - group * kGroupRows, static_cast<uint32_t>(kGroupRows));
  const uint32_t m0 = (group * kGroupRows + lt % width % high) * G::kM, n0 = p.first_n + lt % width / high * G::kN;
  const uint32_t m_wave = m0 + wm * MI * 16, n_wave = n0 + wn * (GATED ? NI * 8 : NI * 16);

  // Loads. Offsets of this lane's loads from the tile's first rows (at most 255 rows of
  // 2^24 bytes); rows past the last are the last's, and reach only outputs that are
  // not stored. Scales: even wavefronts load A's, odd ones B's (every wavefront one
  // load, so that all count alike).
  uint32_t a_at[G::kLoadsA], b_at[G::kLoadsN];
  const bool scales_b = wave & 1;
#pragma unroll
  for (int i = 0; i < G::kLoadsA; ++i) {
    const uint32_t slot = (i * G::kWaves + wave) * 8 + lane / 8;
    const uint32_t s = slot % (MI * 16);
    const uint32_t row = min(m0 + slot - s + s % 16 * MI + s / 16, p.M - 1);
    a_at[i] = (row - m0) * static_cast<uint32_t>(ld) + ((lane % 8) ^ (slot / 2 % 8)) * 16;
  }
#pragma unroll
  for (int i = 0; i < G::kLoadsN; ++i) {
    const uint32_t slot = (i * G::kWaves + wave) * 8 + lane / 8;
    const uint32_t s = slot % (NI * 16);
    uint32_t col = slot - s;
    if constexpr (GATED) {
      col = col / 2 + s % 16 * (NI / 2) + s / 16 % (NI / 2);
    } else {
      col += s % 4 * (4 * NI) + s % 16 / 4 * NI + s / 16;
    }
    b_at[i] = (min(n0 + col, p.N - 1) - n0) * static_cast<uint32_t>(ld) + ((lane % 8) ^ (slot / 2 % 8)) * 16;
  }
  // Four scales a lane; those past the padding read others. GATED: g's and u's by
  // different wavefronts.
  const bool scales_u = GATED && wave % 4 == 3;
  const uint32_t s_ld = static_cast<uint32_t>(scales_b ? p.cols128 : p.rows128);
  const uint32_t s_at = min((scales_b ? n0 : m0) + lane * 4, s_ld - 4);
  const int s_to = scales_u ? G::kScalesU : scales_b ? G::kScalesN : G::kScalesA;
  uint32_t load_t = SPLIT ? split * p.blocks_per_split : 0;
  const uint32_t load_end = SPLIT ? min(k_steps, load_t + p.blocks_per_split) : k_steps;
  const uint32_t steps = load_end - load_t;
  auto issue = [&](int stage) {
    if (load_t == load_end) return;
    const int pair = !GATED && load_t >= p.k_blocks ? 1 : 0;
    const uint64_t kb = load_t - (pair ? p.k_blocks : 0), k = kb * kBlock;
    uint8_t* lds = smem + stage * G::kStage;
    const uint8_t* a = p.a_codes[pair] + m0 * ld + k;
#pragma unroll
    for (int i = 0; i < G::kLoadsA; ++i)
      LoadToLds<16>(a, a_at[i], lds + (i * G::kWaves + wave) * 1024);
#pragma unroll
    for (int i = 0; i < G::kLoadsN; ++i) {
      // GATED: whether the slots are u's, the same for all wavefronts.
      static_assert(!GATED || NI % G::kWaves == 0);
      const uint8_t* b = p.b_codes[GATED ? (i * G::kWaves % (2 * NI) >= NI ? 1 : 0) : pair] + n0 * ld + k;
      LoadToLds<16>(b, b_at[i], lds + G::kM * kBlock + (i * G::kWaves + wave) * 1024);
    }
    const uint8_t* sc = (scales_b ? p.b_scales[GATED ? (scales_u ? 1 : 0) : pair] : p.a_scales[pair]) + kb * s_ld;
    LoadToLds<4>(sc, s_at, lds + s_to);
    ++load_t;
  };

  floatx4 acc[MI][NI];

  const int frag0 = j * kBlock + ((q ^ (j >> 1)) * 16), frag1 = frag0 ^ 64;
  auto fragment = [&](const uint8_t* at) {
    const intx4 lo = *reinterpret_cast<const intx4*>(at + frag0);
    const intx4 hi = *reinterpret_cast<const intx4*>(at + frag1);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  constexpr int kNs = GATED ? NI / 2 : NI;  // adjacent columns
  constexpr int kBw = (NI + 3) / 4;
  const int as_at = G::kScalesA + wm * MI * 16 + j * MI;
  const int bs_at = G::kScalesN + (GATED ? wn * NI * 8 + j * kNs : wn * NI * 16 + j % 4 * (4 * kNs) + j / 4 * kNs);
  // A lane's operands of a step: MI rows of A, then NI of B one after another.
  auto read_a = [&](int stage, int i) { return fragment(smem + stage * G::kStage + (wm * MI + i) * 16 * kBlock); };
  auto read_b = [&](int stage, int n) {
    return fragment(smem + stage * G::kStage + (G::kM + (wn * NI + n) * 16) * kBlock);
  };
  struct Scales {
    uint32_t a, b[kBw];
  };
  auto read_scales = [&](int stage) {
    const uint8_t* lds = smem + stage * G::kStage;
    Scales r;
    if constexpr (MI == 4) r.a = *reinterpret_cast<const uint32_t*>(lds + as_at);
    else if constexpr (MI == 2) r.a = *reinterpret_cast<const uint16_t*>(lds + as_at);
    else r.a = lds[as_at];
#pragma unroll
    for (int i = 0; i < kBw; ++i) r.b[i] = *reinterpret_cast<const uint32_t*>(lds + bs_at + (GATED ? 256 : 4) * i);
    return r;
  };
  // Waits for this wavefront's loads of a step, of which at most `later` steps'
  // worth may be on their way behind it, and for its reads; behind the barrier
  // everyone's have landed, and everyone has read the stage before. (A
  // __syncthreads() would wait for all loads.)
  auto meet = [&](auto later, bool all) {
    constexpr int kLater = decltype(later)::value * G::kLoads;
    if (kLater > 0 && !all) {
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kLater) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
  };

#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int n = 0; n < NI; ++n) acc[i][n] = floatx4{};
  if constexpr (FULL) {
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) issue(s);
    int stage = 0;
    for (uint32_t t = 0; t < steps; ++t) {
      meet(std::integral_constant<int, STAGES - 2>(), t + STAGES - 1 > steps);
      issue(stage == 0 ? STAGES - 1 : stage - 1);
      const Scales sc = read_scales(stage);
      Wide fa[MI];
#pragma unroll
      for (int i = 0; i < MI; ++i) fa[i] = Widen(read_a(stage, i), sc.a >> (i * 8) & 0xFF);
      intx8 raw = read_b(stage, 0);
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        const Wide fb = Widen(raw, sc.b[n / 4] >> (n % 4 * 8) & 0xFF);
        if (n + 1 < NI) raw = read_b(stage, n + 1);
        // Consecutive products are independent.
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int i = 0; i < MI; ++i)
            acc[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb.v[k], fa[i].v[k], acc[i][n], 0, 0, 0);
      }
      stage = stage == STAGES - 1 ? 0 : stage + 1;
    }
  } else {
    // A row of B is read while the one before it is multiplied. All of a step's
    // are in registers when its last two are: there the wavefronts meet, the stage is
    // loaded again, and each row of A makes way for the next step's behind its last
    // product.
#pragma unroll
    for (int s = 0; s < STAGES; ++s) issue(s);
    meet(std::integral_constant<int, STAGES - 1>(), steps < STAGES);
    int stage = 0;
    intx8 fa[MI], fb[2];
    Scales sc = read_scales(0);
#pragma unroll
    for (int i = 0; i < MI; ++i) fa[i] = read_a(0, i);
    fb[0] = read_b(0, 0);
    auto multiply = [&](auto n, auto i) {
      acc[i][n] = Mfma<decltype(n)::value % 4, decltype(i)::value>(fb[n % 2], fa[i], acc[i][n], sc.b[n / 4], sc.a);
    };
    for (uint32_t t = 0; t < steps; ++t) {
      fb[1] = read_b(stage, 1);
      Static<NI - 2>([&](auto n) {
        Static<MI>([&](auto i) { multiply(n, i); });
        fb[n % 2] = read_b(stage, n + 2);
      });
      const bool more = t + 1 < steps;
      if (more) {
        meet(std::integral_constant<int, STAGES - 2>(), t + STAGES > steps);
        issue(stage);
        stage = stage == STAGES - 1 ? 0 : stage + 1;
      }
      // (After the last step these read what nothing uses.)
      const Scales next = read_scales(stage);
      Static<MI>([&](auto i) {
        multiply(std::integral_constant<int, NI - 2>(), i);
        multiply(std::integral_constant<int, NI - 1>(), i);
        fa[i] = read_a(stage, i);
      });
      fb[0] = read_b(stage, 0);
      sc = next;
    }
  }

  using T = typename Elem<DT>::T;
  if constexpr (!GATED) {
    using Out = std::conditional_t<SPLIT, float, T>;
    Static<MI>([&](auto i) {
      const uint32_t m = m_wave + j * MI + i;
      if (m >= p.M) return;
      Out* row = SPLIT ? reinterpret_cast<Out*>(p.partial) + (static_cast<uint64_t>(split) * p.M + m) * p.N
                       : static_cast<Out*>(p.C) + m * p.c_stride;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        float run[kNs];
#pragma unroll
        for (int n = 0; n < kNs; ++n) run[n] = acc[i][n][v];
        StoreRun<SPLIT ? kF32 : DT>(row, n_wave + v * 4 * kNs + q * kNs, p.N, run);
      }
    });
  } else {
    constexpr int kRun = 4 * kNs;  // adjacent columns of a lane
    static_assert(kRun == 16);
    const uint32_t n_lane = n_wave + q * kRun;
    // Columns past the last count as zeros.
    if (n0 + G::kN > p.N) {
#pragma unroll
      for (int n = 0; n < NI; ++n)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          if (n_lane + v * kNs + n % kNs >= p.N) {
#pragma unroll
            for (int i = 0; i < MI; ++i) acc[i][n][v] = 0.0f;
          }
    }
    auto run = [&](auto i, int half, float (&v)[kRun]) {
#pragma unroll
      for (int c = 0; c < kRun; ++c) v[c] = acc[i][half * kNs + c % kNs][c / kNs];
    };
    auto gate = [&](auto act, const float (&g)[kRun], const float (&u)[kRun], float (&h)[kRun]) {
#pragma unroll
      for (int c = 0; c < kRun; ++c) {
        float d;
        ActAndSlope<decltype(act)::value>(g[c], &h[c], &d);
        h[c] *= u[c];
      }
    };
    auto finish = [&](auto act) {
      // Largest magnitudes of the tile's rows: a lane's run, the four lanes of a
      // row, the WN wavefronts through LDS.
      float* tops = reinterpret_cast<float*>(smem + G::kTops);
      if (p.g_codes || p.u_codes || p.h_codes) {
        Static<MI>([&](auto i) {
          float g[kRun], u[kRun], h[kRun];
          run(i, 0, g);
          run(i, 1, u);
          float top[3] = {FiniteMax(g), FiniteMax(u), 0.0f};
          if (p.h_codes) {
            gate(act, g, u, h);
            top[2] = FiniteMax(h);
          }
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            top[k] = fmaxf(top[k], __shfl_xor(top[k], 16, kWave));
            top[k] = fmaxf(top[k], __shfl_xor(top[k], 32, kWave));
            if (q == 0) tops[(k * G::kM + wm * MI * 16 + j * MI + i) * WN + wn] = top[k];
          }
        });
        __syncthreads();
      }
      Static<MI>([&](auto i) {
        const uint32_t m = m_wave + j * MI + i;
        if (m >= p.M) return;
        auto keep = [&](int k, const float (&v)[kRun], uint8_t* codes, uint8_t* scales) {
          const float* at = tops + (k * G::kM + wm * MI * 16 + j * MI + i) * WN;
          float top = at[0];
#pragma unroll
          for (int w = 1; w < WN; ++w) top = fmaxf(top, at[w]);
          const uint32_t s = ScaleByte(top);
          const float inv = ScaleInverse(s);
          uint32_t w[4];
#pragma unroll
          for (int c = 0; c < 4; ++c)
            w[c] = Pack4(v[4 * c] * inv, v[4 * c + 1] * inv, v[4 * c + 2] * inv, v[4 * c + 3] * inv);
          *reinterpret_cast<uint4*>(codes + m * p.cols128 + n_lane) = make_uint4(w[0], w[1], w[2], w[3]);
          if (q == 0 && wn == 0) {
            uint8_t* row = scales + n0 / kBlock * p.rows128;
            row[m] = static_cast<uint8_t>(s);
            if (m + 1 == p.M)
              for (uint64_t r = p.M; r < p.rows128; ++r) row[r] = 0;
          }
        };
        float g[kRun], u[kRun];
        run(i, 0, g);
        run(i, 1, u);
        if (p.g_codes) keep(0, g, p.g_codes, p.g_scales);
        if (p.u_codes) keep(1, u, p.u_codes, p.u_scales);
        if (p.C || p.h_codes) {
          float h[kRun];
          gate(act, g, u, h);
          if (p.C) StoreRun<DT>(static_cast<T*>(p.C) + m * p.c_stride, n_lane, p.N, h);
          if (p.h_codes) keep(2, h, p.h_codes, p.h_scales);
        }
      });
    };
    if (p.act == 1) finish(std::integral_constant<int, 1>());
    else if (p.act == 2) finish(std::integral_constant<int, 2>());
    else finish(std::integral_constant<int, 3>());
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
template <int DT, bool FULL, int MI, int NI, int WM, int WN, int STAGES, bool GATED, bool SPLIT>
Status LaunchTile(TileArgs& p, const Ctx& c, const char* what, uint32_t first_tile = 0, uint32_t tiles_n = 0) {
  using G = Tile<MI, NI, WM, WN, STAGES, GATED>;
  p.tiles_m = static_cast<uint32_t>(CeilDiv(p.M, G::kM));
  p.tiles_n = tiles_n ? tiles_n : static_cast<uint32_t>(CeilDiv(p.N, G::kN)) - first_tile;
  p.first_n = first_tile * G::kN;
  const uint64_t groups = static_cast<uint64_t>(p.tiles_m) * p.tiles_n * p.splits;
  if (groups * G::kThreads > 0xFFFFFFFFu) return Status::Fail(kUnitEngine, std::string(what) + ": grid exceeds launch limits");
  auto* kernel = f8_tile_kernel<DT, FULL, MI, NI, WM, WN, STAGES, GATED, SPLIT>;
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
  // What is kept in 8 bits gets float32 sums whatever h's type (see Precision).
  constexpr bool kKeepFull = kFull || GATED;
  const bool full = kFull || p.g_codes || p.u_codes || p.h_codes;
  if (ch.big) {
    if (Status s = full ? LaunchTile<DT, kKeepFull, 4, 8, 4, 2, 2, GATED, false>(p, c, what, 0, ch.columns)
                        : LaunchTile<DT, kFull, 4, 8, 4, 2, 2, GATED, false>(p, c, what, 0, ch.columns);
        !s || ch.columns == 0)
      return s;
    return full ? LaunchTile<DT, kKeepFull, 2, 8, 4, 2, 3, GATED, false>(p, c, what, ch.columns)
                : LaunchTile<DT, kFull, 2, 8, 4, 2, 3, GATED, false>(p, c, what, ch.columns);
  }
  constexpr int MI = GATED ? 1 : 2, NI = GATED ? 8 : 4, kStages = GATED ? 3 : 4;  // of 160 KiB of LDS
  if (ch.splits == 1)
    return full ? LaunchTile<DT, kKeepFull, MI, NI, 4, 2, kStages, GATED, false>(p, c, what)
                : LaunchTile<DT, kFull, MI, NI, 4, 2, kStages, GATED, false>(p, c, what);
  if constexpr (!GATED) {
    // Partials are float32 whatever the output's type.
    if (Status s = LaunchTile<kF32, kFull, MI, NI, 4, 2, kStages, false, true>(p, c, what); !s) return s;
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
  return GemmF8Scratch(T, D, F, 2);  // the backward's product
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
