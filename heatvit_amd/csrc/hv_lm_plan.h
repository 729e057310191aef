// hv_lm_plan.h -- which kernel an e4m3 block product takes. Host code without
// HIP, so that tests can ask which kernel their sizes reach.
#pragma once

#include <cstdint>

namespace hv {

enum class F8Kernel {
  kRows16,       // k_gemm_f8_rows: 16 rows by 16 channels
  kRows16x2,     //                 16 rows by 32 channels
  kRows32,       //                 32 rows by 16 channels
  kRows64,       //                 64 rows by 16 channels (float32 outputs)
  kTile64,       // k_gemm_f8_tile: 64 x 64
  kTile128Deep,  //                 128 x 128, four stages (16-bit outputs)
  kTile128,      //                 128 x 128, two stages
  kTile256,      //                 256 x 256 (16-bit outputs)
};

// m rows, n channels, rows of `lda` bytes; f32: a float32 output.
inline F8Kernel f8_kernel(bool f32, int m, int n, int64_t lda) {
  // Up to 16 rows (us at k = 4096): the weights' bytes bound them, and parts of
  // 16 channels leave a CU a workgroup up to 4096 channels; wider weights take two
  // parts a workgroup (1 row by 2048 channels 3.6, two parts 3.8; by 4096 5.2, 5.0,
  // and with weights from memory 6.4, 6.6, 16 rows 7.4, 8.3; by 8192 9.0, 7.2; by
  // 131072 104, 91; 16 rows to float32 by 2048 5.1, 5.6; by 8192 9.9, 8.5).
  const int parts = (n + 63) / 64 * 4;
  const bool near = lda < (int64_t)1 << 22;  // a tile's offsets into the rows are 32-bit
  if (m <= 16 || !near) return parts <= 256 ? F8Kernel::kRows16 : F8Kernel::kRows16x2;
  // More rows, few channels: 16 or 32 rows (float32 outputs, whose tiles' products
  // take longer, 64 too) by 16 channels while that is at most a workgroup a CU,
  // since its wavefronts share the blocks of k (us at k = 4096 by 16 rows, 32 and
  // 64, and tiles; bf16: 64 rows by 1000 channels 4.8, 6.7, 10.5, 8.7; by 2048 7.4,
  // 7.0, 11.0, 9.1; by 4096 13.2, 12.6, 11.4, 9.6; float32: 5.0, 7.2, 11.1, 19.3;
  // 7.7, 7.7, 11.8, 19.7; 13.9, 14.0, 12.4, 19.9; 100 by 4096 20.8, 23.8, 20.0,
  // 20.1).
  auto lone = [&](int rows) { return (int64_t)parts * ((m + rows - 1) / rows) <= 256; };
  if (lone(16)) return F8Kernel::kRows16;
  if (lone(32)) return F8Kernel::kRows32;
  if (f32 && lone(64)) return F8Kernel::kRows64;
  // Tiles by what a block of k costs (measured at k = 4096, us a round of
  // tiles): small ones, several to a CU, where there are few, large ones, which
  // read less for each product, where they fill the card.
  //   16-bit: 64 x 64 10 with one to a CU, 16 with two; 128 x 128 21 with one
  //   (four stages), 36 with two (two stages); 256 x 256 45
  //   float32: 64 x 64 21 and 28; 128 x 128 46 and 66
  // 1024 x 4096 outputs: 30.0, 21.4, 26.3, 43.9 us; 2048 x 4096: 56.8, 41.8,
  // 35.8, 45.3; 4096 x 4096: 115, 83, 74, 56.
  auto tiles = [&](int size) {
    return (int64_t)((m + size - 1) / size) * ((n + size - 1) / size);
  };
  auto cost = [&](int64_t t, int one, int two) {  // two to a CU: 512 a round
    return t <= 256 ? one : (t + 511) / 512 * two;
  };
  const int64_t c64 = cost(tiles(64), f32 ? 21 : 10, f32 ? 28 : 16);
  if (f32) return c64 <= cost(tiles(128), 46, 66) ? F8Kernel::kTile64 : F8Kernel::kTile128;
  const int64_t c128 = (tiles(128) + 511) / 512 * 36, c128deep = (tiles(128) + 255) / 256 * 21;
  const int64_t c256 = (tiles(256) + 255) / 256 * 45;
  if (c64 <= c128 && c64 <= c128deep && c64 <= c256) return F8Kernel::kTile64;
  if (c128deep <= c128 && c128deep <= c256) return F8Kernel::kTile128Deep;
  return c128 <= c256 ? F8Kernel::kTile128 : F8Kernel::kTile256;
}

}  // namespace hv
