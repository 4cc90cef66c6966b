// The gated feed-forward products on the persistent four-wave kernel (gemm_mfma_w4.hpp, W4_EPI_GATED): 128 features and 256
// or 192 tokens a tile, 64 features of Wg and the same 64 of Wu in a wave's 128 rows.
//
// Bound by the matrix cores, as the plain product of X and [Wg; Wu]; the activation, the product and what is kept ride in the
// epilogue, from the accumulators, while the next tile's first stages are in flight.
#pragma once
#include "ffn_gated_store.hpp"
#include "gemm_mfma_w4.hpp"

namespace zluda_amd {

template <class E>
struct GatedMfmaParams : MfmaParams {
  GatedParams gated;

  // a wave's accumulators: tiles 0 .. 3 along P are G's, 4 .. 7 U's, for features f0 .. f0 + 63; TQ tiles of 16 tokens
  template <int TQ, class AccV>
  __device__ __forceinline__ void store_tile(AccV (&acc)[8][TQ], int f0, int t0, const W4Staged &staged) const {
    const int lane = lane_here(), l4 = 4 * (lane >> 4);
    float bg[4][4], bu[4][4];
#pragma unroll
    for (int a = 0; a < 4; a++)
#pragma unroll
      for (int e = 0; e < 4; e++) bg[a][e] = bu[a][e] = 0.0f;
    if (gated.bias) {
      const uint32_t odd = (uint32_t)(((uintptr_t)gated.bias >> 1) + f0) & 1;  // (the element the dword loads started at)
      const uint16_t *b = (const uint16_t *)staged.area + l4 + odd;
      const uint16_t *c = (const uint16_t *)(staged.area + W4Staged::WORDS) + l4 + ((odd + gated.features) & 1);
#pragma unroll
      for (int a = 0; a < 4; a++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          bg[a][e] = E::dec(b[16 * a + e]);
          bu[a][e] = E::dec(c[16 * a + e]);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    gated_with(gated, [&](auto kept, auto act) __attribute__((always_inline)) {
#pragma unroll
      for (int b = 0; b < TQ; b++) {
        // (one column of tiles at a time, read explicitly: see w4_store_f16)
        int raw[8][4];
#pragma unroll
        for (int a = 0; a < 8; a++)
#pragma unroll
          for (int e = 0; e < 4; e++) raw[a][e] = w4_acc_read(acc[a][b][e]);
        float g[4][4], u[4][4];
#pragma unroll
        for (int a = 0; a < 4; a++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            g[a][e] = bits2f((uint32_t)raw[a][e]) + bg[a][e];
            u[a][e] = bits2f((uint32_t)raw[a + 4][e]) + bu[a][e];
          }
        const int token = t0 + 16 * b + (lane & 15);
        gated_store<E, decltype(kept)::value, decltype(act)::value>(gated, f0, token, token < gated.tokens, g, u);
        __builtin_amdgcn_sched_barrier(0);
      }
    });
  }
};

} // namespace zluda_amd
