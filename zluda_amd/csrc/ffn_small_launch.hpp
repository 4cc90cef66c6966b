// Gated feed-forward products in tiles that a workgroup takes one of, and at any alignment.
#pragma once
#include <cstring>

#include "ffn_launchers.hpp"
#include "kernels/ffn_gated_any.hpp"
#include "kernels/ffn_gated_tile.hpp"

namespace zluda_amd {

template <class E, int V>
inline uint32_t launch_gated_tile(const GatedParams &p, hipStream_t s) {
  constexpr GatedTile t = kGatedTiles[V];
  GatedTileParams m;
  memset((void *)&m, 0, sizeof(m));
  m.gated = p;
  m.g.batch = 1;
  m.tiles_p = (p.features + t.features - 1) / t.features; m.tiles_q = (p.tokens + t.tokens - 1) / t.tokens;
  m.group_p = 8;
  m.splits = 1;
  return launch_kernel(gated_tile_kernel<E, t.features, t.tokens, t.wp, t.wq, t.stages>, dim3(m.tiles_p * m.tiles_q), dim3(64 * t.wp * t.wq), s, m);
}

template <class E>
inline uint32_t launch_gated_small(const GatedParams &p, int tile, hipStream_t s) {
  switch (tile) {
  case 0: return launch_gated_tile<E, 0>(p, s);
  case 1: return launch_gated_tile<E, 1>(p, s);
  case 2: return launch_gated_tile<E, 2>(p, s);
  case 3: return launch_gated_tile<E, 3>(p, s);
  default: return launch_kernel(gated_any_kernel<E>, dim3((p.tokens + 63) / 64, (p.features + 31) / 32), dim3(256), s, p);
  }
}

} // namespace zluda_amd
