// Which tile the products of kernels/block_tile.hpp take: rules on sizes, without HIP.
#pragma once
#include <cstdint>

namespace zluda_amd {

// Tiles of P x Q rows, waves along each, LDS stages of 128 bytes of K.  Of them a CU holds `per_cu` workgroups, and n of those take base + n * slope us a
// stage in a full chip (stage_us: 8-bit operands with their scales, 16-bit ones).  Measured on whole calls over 2048 of model, 5632 features, 16384
// rows of eight experts: 8-bit 210, 250, 391 and 511 us, 16-bit 354, 444, 591 and 763; and one workgroup a CU on calls of fewer tiles.
struct BlockTile { int bp, bq, wp, wq, stages, per_cu; float base8, slope8, base16, slope16; };
constexpr BlockTile kBlockTiles[] = {
    {256, 256, 2, 4, 2, 1, 0.0f, 1.82f, 0.0f, 1.69f},
    {128, 128, 2, 2, 2, 2, 0.45f, 0.33f, 0.45f, 0.30f},
    {64, 64, 2, 2, 4, 2, 0.13f, 0.163f, 0.13f, 0.123f},
    {64, 32, 2, 2, 4, 3, 0.13f, 0.108f, 0.13f, 0.08f},
};
constexpr int kBlockTileCount = 4;

// us until `tiles` workgroups of tile v are done on `cus` CUs, each with `stages` of K and the time of three for its start and end
inline float block_tiles_us(int v, uint64_t tiles, uint64_t stages, uint64_t cus, bool eight_bits) {
  const BlockTile &t = kBlockTiles[v];
  const float base = eight_bits ? t.base8 : t.base16, slope = eight_bits ? t.slope8 : t.slope16;
  const uint64_t slots = cus * t.per_cu, full = tiles / slots, rest = tiles % slots;
  float us = (float)full * (base + slope * t.per_cu);
  if (rest) us += base + slope * (float)((rest + cus - 1) / cus);
  return us * (float)(stages + 3);
}

} // namespace zluda_amd
