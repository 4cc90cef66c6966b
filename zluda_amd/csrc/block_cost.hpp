// Which tile the products of kernels/block_tile.hpp take: rules on sizes, without HIP.
#pragma once
#include <cstdint>

namespace zluda_amd {

// Tiles of P x Q rows, waves along each, LDS stages of 128 bytes of K.  Of them a CU holds `per_cu` workgroups, and n of those take base + n * slope us a
// stage (8-bit operands with their scales, 16-bit ones).  Measured on whole calls over 2048 of model, 5632 features, 16384 rows of eight experts: 8-bit 213, 259, 413,
// 533, 289 and 302 us, 16-bit 354, 441, 597, 764, 506 and 453 (the first six); and on calls that leave a CU one workgroup: 333 tokens, 5632 x 2000 31, 18.3, 17.9, 18.2,
// 17.2, 15.5 and 13.9, 1000, 2048 x 2048 26.5, 18.0, 11.4, 15.2, 10.4, 17.7 and 12.1, 700, 4096 x 4096 -, 25.9, 26.7, -, 22.0, 21.9 and 19.8.  (The last shape is there for
// what 128 x 128 leaves idle: 132 tiles of 5632 x 333 on 256 CUs are 176 of 96 columns.)
struct BlockTile { int bp, bq, wp, wq, stages, per_cu; float base8, slope8, base16, slope16, edge; };
constexpr BlockTile kBlockTiles[] = {
    {256, 256, 2, 4, 2, 1, 0.0f, 1.82f, 0.0f, 1.69f, 3.0f},
    {128, 128, 2, 2, 2, 2, 0.45f, 0.33f, 0.45f, 0.30f, 3.0f},
    {64, 64, 2, 2, 4, 2, 0.13f, 0.163f, 0.13f, 0.123f, 3.0f},
    {64, 32, 2, 2, 4, 3, 0.13f, 0.108f, 0.13f, 0.08f, 3.0f},
    {128, 64, 2, 2, 3, 2, 0.05f, 0.33f, 0.05f, 0.31f, 3.0f},
    {128, 128, 2, 2, 4, 1, 0.0f, 0.67f, 0.0f, 0.56f, 6.0f},
    {128, 96, 2, 2, 4, 1, 0.0f, 0.53f, 0.0f, 0.45f, 6.0f},
};
constexpr int kBlockTileCount = 7;

// us until `tiles` workgroups of tile v are done on `cus` CUs, each with `stages` of K and the time of `edge` more for its start and end (which nothing
// overlaps where a CU has one workgroup: 2559 tokens, 3264 x 320 with GELU 16.1 us on the second shape, 19.4 on the last, 21.8 on the one before it)
inline float block_tiles_us(int v, uint64_t tiles, uint64_t stages, uint64_t cus, bool eight_bits) {
  const BlockTile &t = kBlockTiles[v];
  const float base = eight_bits ? t.base8 : t.base16, slope = eight_bits ? t.slope8 : t.slope16;
  const uint64_t slots = cus * t.per_cu, full = tiles / slots, rest = tiles % slots;
  float us = (float)full * (base + slope * t.per_cu);
  if (rest) us += base + slope * (float)((rest + cus - 1) / cus);
  return us * ((float)stages + t.edge);
}

// Tile configurations of the products with a scale for each 128 of K (index = plan.variant for ZLUDA_KERNEL_MFMA_BLK8): workgroup tile, waves, LDS
// stages of 128 K bytes; uniform: only for P rows that share their scales (the accumulators of a wave leave no registers for more); exact: also for results in
// 32 bits (the widened operands take registers)
struct BlockVariant { int bp, bq, wp, wq, stages; bool uniform, exact; };
constexpr BlockVariant block_variant(int v, bool uniform, bool exact) {
  return {kBlockTiles[v].bp, kBlockTiles[v].bq, kBlockTiles[v].wp, kBlockTiles[v].wq, kBlockTiles[v].stages, uniform, exact};
}
constexpr BlockVariant kBlockVariants[] = {block_variant(0, true, false), block_variant(1, false, false), block_variant(2, false, true), block_variant(3, false, true),
                                           block_variant(4, false, true), block_variant(5, false, false), block_variant(6, false, false),
                                           {16, 16, 1, 8, 0, false, true}};  // kernels/block_decode.hpp: no tile of those
constexpr int kBlockDecode = kBlockTileCount;
static_assert(sizeof(kBlockVariants) / sizeof(kBlockVariants[0]) == kBlockDecode + 1, "a variant each");
constexpr int kNumBlockVariants = sizeof(kBlockVariants) / sizeof(kBlockVariants[0]);

} // namespace zluda_amd
