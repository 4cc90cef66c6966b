// Chooses the kernel of a gated feed-forward call.
#pragma once
#include <cstring>

#include "../../include/zluda_gemm_launch.h"
#include "ffn_launch.hpp"
#include "kernels/ffn_gated_w4.hpp"

namespace zluda_amd {

// 16-byte pieces of the operands' rows, through 2 GiB buffer windows
inline bool gated_dma_operands(const GatedParams &p) {
  return p.model % 8 == 0 && p.ldx % 8 == 0 && p.ldw % 8 == 0 && !(((uintptr_t)p.x | (uintptr_t)p.w) & 15) &&
         (2ll * p.features * p.ldw + p.model) * 2 < 0x7fffffffll && ((int64_t)p.tokens * p.ldx + p.model) * 2 < 0x7fffffffll;
}

template <class E, int BQ>
inline uint32_t launch_gated_w4(const GatedParams &p, int cus, hipStream_t s) {
  constexpr int KIND = E::type == CUDA_R_16BF ? KIND_BF16 : KIND_F16;
  GatedMfmaParams<E> m;
  memset((void *)&m, 0, sizeof(m));
  m.gated = p;
  m.g.A = p.w; m.g.B = p.x; m.g.bias = p.bias;
  m.g.M = p.features; m.g.N = p.tokens; m.g.K = p.model; m.g.batch = 1;
  m.g.a_si = p.ldw; m.g.a_sk = 1; m.g.b_sj = p.ldx; m.g.b_sk = 1;
  m.tiles_p = (p.features + 127) / 128; m.tiles_q = (p.tokens + BQ - 1) / BQ;
  m.group_p = 8;
  m.splits = 1;
  const int64_t tiles = (int64_t)m.tiles_p * m.tiles_q;
  const int slots = cus >= 8 ? cus / 8 * 8 : cus;  // (the kernel walks its tiles in steps of a multiple of 8)
  return launch_kernel(gemm_mfma_w4_kernel<KIND, 0, 0, W4_EPI_GATED, GatedMfmaParams<E>, BQ>, dim3((uint32_t)(tiles < slots ? tiles : slots)), dim3(256), s, m);
}

// The tile whose slowest CU is done first: rounds of tiles over the CUs, each the stages of K (and the time of three for its
// start and end).  All tiles share the bound of the one read of W, under which their differences vanish.
// Measured, us, in the order of kGatedTiles: 64 tokens, 4096 x 14336: 57, 48, 53, 64, 89, 96; 256: 133, 106, 89, 72, 92, 107; 384: 190, 142,
// 121, 119, 101, 108; 777: 450, 295, 239, 217, 219, 181; 300, 2048 x 5632: 34, 23, 37, 30, 37, 43; 2000: 171, 115, 109, 92, 76, 89.
inline int gated_tile(const GatedParams &p, int cus) {
  const int stages = (p.model + 63) / 64 + 3;
  int best = 0;
  float best_us = 0.0f;
  for (int v = 0; v < kGatedTileCount; v++) {
    const GatedTile &t = kGatedTiles[v];
    const int64_t n = ((p.features + t.features - 1) / t.features) * (int64_t)((p.tokens + t.tokens - 1) / t.tokens);
    const float us = (float)((n + cus - 1) / cus) * t.stage_us * stages;
    if (v == 0 || us < best_us) {
      best = v;
      best_us = us;
    }
  }
  return best;
}

template <class E>
inline uint32_t launch_gated(const GatedParams &p, hipStream_t s) {
  const int cus = (int)zluda_gemm_device_cu_count(), tile = gated_dma_operands(p) ? gated_tile(p, cus) : -1;
  if (tile >= kGatedPersistent) return kGatedTiles[tile].tokens == 192 ? launch_gated_w4<E, 192>(p, cus, s) : launch_gated_w4<E, 256>(p, cus, s);
  return E::type == CUDA_R_16BF ? launch_gated_small_bf16(p, tile, s) : launch_gated_small_f16(p, tile, s);
}

} // namespace zluda_amd
