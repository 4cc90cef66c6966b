// Launchers of the products grouped by expert, one translation unit per kind of operands.
#pragma once
#include "block_cost.hpp"
#include "kernels/ffn_grouped_grad.hpp"
#include "launch_util.hpp"

namespace zluda_amd {

// row tiles there can be, whatever the counts
inline uint64_t most_row_tiles(uint64_t rows, uint64_t experts, uint64_t side) { return rows / side + std::min(experts, rows); }

uint32_t launch_grouped_bf16(const GroupedParams &p, int tile, hipStream_t s);
uint32_t launch_grouped_f16(const GroupedParams &p, int tile, hipStream_t s);
uint32_t launch_grouped_f8(const GroupedParams &p, int tile, hipStream_t s);
// the sums of dx's shares
uint32_t launch_grouped_round(const RoundParams &r, uint32_t type, const int32_t *offsets, int32_t experts, dim3 grid, hipStream_t s);
// side: of a tile, 128 or 256
uint32_t launch_grouped_grad(const GroupedGradParams &p, uint32_t type, int side, uint32_t groups, hipStream_t s);

template <int KIND, int DT, int V>
uint32_t launch_grouped_tile(const GroupedParams &p, hipStream_t s) {
  constexpr BlockTile t = kBlockTiles[V];
  const uint64_t groups = (uint64_t)((p.features + t.bp - 1) / t.bp) * most_row_tiles(p.rows, p.experts, t.bq);
  return launch_kernel(grouped_tile_kernel<KIND, DT, t.bp, t.bq, t.wp, t.wq, t.stages>, dim3((uint32_t)groups), dim3(t.wp * t.wq * 64), s, p);
}
template <int KIND, int DT>
uint32_t launch_grouped(const GroupedParams &p, int tile, hipStream_t s) {
  switch (tile) {
  case 0:
    if constexpr (KIND != KIND_F8_WIDE) return launch_grouped_tile<KIND, DT, 0>(p, s);
    break;
  case 1:
    if constexpr (KIND != KIND_F8_WIDE) return launch_grouped_tile<KIND, DT, 1>(p, s);
    break;
  case 2: return launch_grouped_tile<KIND, DT, 2>(p, s);
  case 3: return launch_grouped_tile<KIND, DT, 3>(p, s);
  case 4: return launch_grouped_tile<KIND, DT, 4>(p, s);
  case 5:
    if constexpr (KIND != KIND_F8_WIDE) return launch_grouped_tile<KIND, DT, 5>(p, s);
    break;
  case 6:
    if constexpr (KIND != KIND_F8_WIDE) return launch_grouped_tile<KIND, DT, 6>(p, s);
    break;
  }
  return CUBLAS_STATUS_INTERNAL_ERROR;
}

} // namespace zluda_amd
