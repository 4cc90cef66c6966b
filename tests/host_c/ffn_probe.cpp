// The choices of the feed-forward launches, for tests: built as a shared library of its own (the rules need no device).
#include "../../zluda_amd/csrc/ffn_launch.hpp"

using namespace zluda_amd;

#define PROBE extern "C" __attribute__((visibility("default")))

struct Gated {
  const void *x, *w;
  int64_t ldx, ldw;
  int32_t tokens, features, model;
};

PROBE uint32_t probe_column_strips(uint64_t cols) { return column_strips(cols); }
PROBE uint64_t probe_max_side() { return kMaxSide; }
// index of the tile of a gated product in kGatedTiles, -1: at any alignment
PROBE int probe_gated_tile(const Gated *p, int cus) { return gated_dma_operands(*p) ? gated_tile(*p, cus) : -1; }
PROBE int probe_gated_tile_shape(int tile, int *features, int *tokens) {
  if (tile < 0 || tile >= kGatedTileCount) return -1;
  *features = kGatedTiles[tile].features;
  *tokens = kGatedTiles[tile].tokens;
  return tile >= kGatedPersistent;
}
// shares of dX's K where dX and dW share a launch, 0: one after the other; x: as the product reads it
PROBE uint32_t probe_grad_splits(const zluda_ffn_gated_grad *p, const zluda_ffn_matrix *x, int64_t lddz, const void *dz, int cus, uint32_t *split_stages) {
  const GradTogether t = grad_together(p, cus);
  *split_stages = t.split_stages;
  return t.splits && grad_together_operands(p, *x, lddz, dz) ? t.splits : 0;
}
PROBE int probe_grad_largest_tiles(uint64_t m, uint64_t n, uint64_t cus) { return grad_largest_tiles(m, n, cus); }
PROBE uint64_t probe_rows_in_window(uint64_t rows, int64_t ld) { return rows_in_window(rows, ld); }
