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
// Times below are of the launches in a kernel trace (medians of 20), in us, sizes M x K x N,
// a split's with its join.
//
// Large or small. A round of the chip (a tile a CU) costs about 1.7 us a step of 128 k with
// the large tiles and 0.6 with the small ones (3.1 and 1.05 with float32 sums), whose
// loads run further ahead, so the large ones pay from three rounds of small ones on. Large |
// small, to bfloat16: 2048x2048x5504 33 | 40, 8192x512x1376 15.5 | 19.5, 4096x2048x2048 31.5 |
// 27.7, 2048x2048x2048 29 | 15, 4096x4096x4096 62 | 90; to float32, the same rule: 59 | 68, 24 |
// 26, 56 | 48, 53 | 26, 117 | 169; gated with checkpoints 1024x2048x5504 60 | 78, 4096x512x1376 26
// | 30, 777x520x1003 27 | 13.
//
// Few rows. Skinny | small tiles, split: 16x2048x5504 7.1 | 9.0 (float32 7.3 | 11.5), 64x2048x5504
// 13.2 | 11.9 (13.4 | 14.4), 64x5504x2048 16.5 | 14.0 (16.5 | 15.7), gated 64x2048x5504 15.1 |
// 14.7 (15.2 | 23.4): at 64 rows in 16 bits tiles would win by up to 2.5 us.
//
// Splitting a reduction saves steps where tiles leave CUs idle, and costs a launch and the
// partial sums' way through memory (about 4 us, and 8 bytes an output and slice). The step's
// 0.8 us lies between the two kinds of sums: one rule serves both, for the scratch sizes do
// not know the type. In 1, 2, 4, 8 slices, the one picked marked, to bfloat16 and to float32:
//   128x5504x2048   26.9 21.3 17.2 16.0*   48.2 31.9 21.9 18.4*
//   1000x4096x1000  21.3 20.8 21.1* 26.6   37.8 28.9 25.2* 30.6
//   777x2006x520    12.9 13.1 14.4* 18.5   20.6 18.2 15.9* 20.3
//   515x1376x2000   10.5* 16.4 20.8 23.6   16.7* 18.3 23.2 25.0
//   129x2048x5504   13.3* 16.9 21.4 25.9   21.7* 20.6 25.4 28.4
// It loses 1.6 us at most. The gated block did not gain (300x2048x5504: 17 us longer in two).
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
    // those are one round (the same sums, so the same bits; all large | with half tiles:
    // 4096x2048x5504 62 | 57, to float32 116 | 103, gated with checkpoints 2048x2048x5504 117 |
    // 103, 8192x2048x5504 385 | 387).
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
