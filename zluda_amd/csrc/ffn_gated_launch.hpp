// Chooses the kernel of a gated feed-forward call.
#pragma once
#include <cstring>

#include "../../include/zluda_gemm_launch.h"
#include "ffn_launchers.hpp"
#include "kernels/ffn_gated_w4.hpp"

namespace zluda_amd {

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

template <class E>
inline uint32_t launch_gated(const GatedParams &p, hipStream_t s) {
  const int cus = (int)zluda_gemm_device_cu_count(), tile = gated_dma_operands(p) ? gated_tile(p, cus) : -1;
  if (tile >= kGatedPersistent) return kGatedTiles[tile].tokens == 192 ? launch_gated_w4<E, 192>(p, cus, s) : launch_gated_w4<E, 256>(p, cus, s);
  return E::type == CUDA_R_16BF ? launch_gated_small_bf16(p, tile, s) : launch_gated_small_f16(p, tile, s);
}

} // namespace zluda_amd
