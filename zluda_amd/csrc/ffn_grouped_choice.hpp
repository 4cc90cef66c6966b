// Which tile the products by expert take: a rule on sizes, without HIP.
#pragma once
#include <algorithm>
#include <cmath>

#include "../../include/cublaslt_abi.h"
#include "../../include/zluda_ffn.h"
#include "block_cost.hpp"

namespace zluda_amd {

// The tile whose last workgroup is done first, if the rows are shared out about evenly, which only the device knows: a tile for each expert, and beyond that half
// of one that is not full for each, give or take `spread`: half of the estimate is the time with that much more, where a tile that fills the chip exactly goes into a
// second round (1001 rows of eight experts, 1024 x 2816, six draws of their counts: 14.4 to 15.2 us; without it 13.6 to 22.1).  Measured, us, in the order of
// kBlockTiles: 2048 of model, 5632 features, eight experts, bf16, 16 rows 53, 42, 37, 35, 39 and 46; 256 58, 45, 39, 41, 42 and 48; 1024 65, 68, 66, 78, 59, 59; 2048
// 94, 83, 108, 129, 91, 84; 4096 118, 140, 174, 220, 148, 142; 1024 of model, 2816 features, 64 experts, 4096 rows 103, 91, 97, 105, 87, 93.
inline int grouped_tile(const zluda_ffn_grouped *p, uint64_t cus) {
  const bool eight = p->x.type == CUDA_R_8F_E4M3, exact = eight && p->y.type == CUDA_R_32F;
  const uint64_t live = std::min(p->rows, p->experts), stages = (p->model * (eight ? 1 : 2) + 127) / 128;
  const uint64_t spread = live > 1 ? (uint64_t)std::ceil(0.29 * std::sqrt((double)live)) : 0;  // (a part of a tile each, even chances: 1 / sqrt(12) of a tile)
  int best = -1;
  float best_us = 0.0f;
  for (int v = 0; v < kBlockTileCount; v++) {
    if (exact && !kBlockVariants[v].exact) continue;
    const uint64_t q = std::max<uint64_t>(live, p->rows / kBlockTiles[v].bq + (live + 1) / 2), across = (p->features + kBlockTiles[v].bp - 1) / kBlockTiles[v].bp;
    float us = block_tiles_us(v, q * across, stages, cus, eight);
    if (q > live) us = 0.5f * (us + block_tiles_us(v, (q + spread) * across, stages, cus, eight));
    if (best < 0 || us < best_us) {
      best = v;
      best_us = us;
    }
  }
  return best;
}

} // namespace zluda_amd
