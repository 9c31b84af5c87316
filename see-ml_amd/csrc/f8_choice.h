// f8_choice.h — how an 8-bit product of given sizes runs (k_f8_gemm.hip). Plain C++:
// what it picks can be asked without a GPU.
#pragma once

#include <cstdint>

namespace seeml_hip {
namespace f8 {

inline uint64_t CeilDiv(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// How a product runs: few rows on the skinny kernel (in groups of 16), others on
// tiles of 256 x 256 or 128 x 128 (gated: 64 rows of 128 columns).
//
// A round of the chip (a tile a CU) costs about 1.4 us a step of 128 k with the large
// tiles and 0.55 with the small ones, whose loads run further ahead, so the large ones
// pay from three rounds of small ones on (us, large | small, bfloat16: 2048x2048x5504
// 32 | 39, 8192x512x1376 15 | 19, 4096x2048x2048 30 | 26, 2048x2048x2048 28 | 15; gated
// with checkpoints 1024x2048x5504 58 | 73, 4096x512x1376 23 | 27, 777x520x1003 26 | 12).
// Few rows: at 16 of 2048x5504 7.0 | 11.5 (skinny | small tiles), at 64 13.2 | 12.2,
// float32 13.2 | 20.1.
//
// Splitting a reduction saves steps where tiles leave CUs idle, and costs a launch and the
// partial sums' way through memory (about 4 us, and 8 bytes an output and slice): 128x5504x2048
// (M, K, N) 28 us in one slice, 15 in four; 515x1376x2000 10 in one, 15 in two. The gated
// block did not gain (300x2048x5504 20 in one, 37 in two).
struct Choice {
  int skinny = 0;  // 16-row groups: 1, 2 or 4
  bool big = false;
  uint32_t columns = 0;  // of large tiles, the rest half as high; 0: all
  uint32_t splits = 1, blocks_per_split = 0;
};
constexpr uint64_t kCus = 256;
inline Choice ChooseF8(uint64_t M, uint64_t N, uint64_t k_blocks, bool gated, bool keep) {
  Choice c;
  if (M <= 64 && !keep) {
    c.skinny = M <= 16 ? 1 : M <= 32 ? 2 : 4;
    return c;
  }
  const uint64_t big = CeilDiv(M, 256) * CeilDiv(N, gated ? 128 : 256);
  const uint64_t small = gated ? CeilDiv(M, 64) * CeilDiv(N, 128) : CeilDiv(M, 128) * CeilDiv(N, 128);
  c.big = CeilDiv(small, kCus) * 5 > CeilDiv(big, kCus) * 11;
  if (c.big) {
    // Whole rounds of large tiles; what is left over on tiles of half the height, where
    // those are one round (the same sums, so the same bits; us, all large | split: 4096x2048x5504
    // 60 | 55, gated with checkpoints 2048x2048x5504 104 | 90, 8192x2048x5504 323 | 321).
    const uint64_t high = CeilDiv(M, 256), wide = CeilDiv(N, gated ? 128 : 256), whole = big / kCus * kCus;
    const uint64_t columns = whole / high;
    if (whole < big && columns > 0 && CeilDiv(M, 128) * (wide - columns) <= kCus) c.columns = static_cast<uint32_t>(columns);
  }
  if (c.big || gated) return c;
  double least = 0.0;
  for (uint64_t s = 1; s <= 16 && (s == 1 || small * s <= kCus); s *= 2) {
    const uint64_t per = CeilDiv(k_blocks, s);
    const double us = 0.8 * per + (s > 1 ? 4.0 + 2e-6 * M * N * s : 0.0);
    if (s > 1 && us >= least) continue;
    least = us;
    c.blocks_per_split = static_cast<uint32_t>(per);
    c.splits = static_cast<uint32_t>(CeilDiv(k_blocks, per));
  }
  return c;
}

}  // namespace f8
}  // namespace seeml_hip
