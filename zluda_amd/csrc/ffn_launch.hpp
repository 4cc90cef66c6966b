// Launchers of the gated feed-forward products, one translation unit per element type.
#pragma once
#include <hip/hip_runtime.h>

#include "kernels/ffn_gated_store.hpp"
#include "launch_util.hpp"

namespace zluda_amd {

uint32_t launch_gated_bf16(const GatedParams &p, hipStream_t s);
uint32_t launch_gated_f16(const GatedParams &p, hipStream_t s);

// The tiles of the gated products: `features` x `tokens` a workgroup, its waves wp x wq, LDS stages, and the time of a stage (of
// 64 K elements) in a full chip, us for each tile of a CU.  From whole calls of 4096 x 14336 and 1024 tokens: 437, 304, 262, 230 us, and
// 241 and 199 with the last two, the persistent four-wave kernel; smaller tiles are less work between two barriers and read more
// of LDS for each product.
struct GatedTile { int features, tokens, wp, wq, stages; float stage_us; };
constexpr GatedTile kGatedTiles[] = {{64, 32, 2, 2, 4, 0.24f},   {64, 64, 2, 2, 3, 0.335f},  {64, 128, 2, 2, 3, 0.58f},
                                     {128, 128, 4, 2, 3, 0.9f}, {128, 192, 2, 2, 2, 1.18f}, {128, 256, 2, 2, 2, 1.4f}};
constexpr int kGatedTileCount = 6, kGatedPersistent = 4;  // (from there on)
// in the first four of them, or (tile < 0) at any alignment
uint32_t launch_gated_small_bf16(const GatedParams &p, int tile, hipStream_t s);
uint32_t launch_gated_small_f16(const GatedParams &p, int tile, hipStream_t s);

// ---- the products of the backward pass in one launch (kernels/ffn_grad_products.hpp) ----------------------------------------------
// D[q][p] = sum over k of P[k][p] Q, Q as [q][k] (dX) or [k][q] (dW).  With `splits` > 1 share z of K writes 32-bit sums to
// part[z][q][p], q and p padded to whole tiles.
struct GradProduct {
  const void *p, *q;
  void *d;
  float *part;
  int64_t ldd;
  int32_t ldp, ldq;
  int32_t np, nq, k;
  int32_t tiles_p, tiles_q, splits, split_stages;
};
struct GradProductsParams {
  GradProduct dx, dw;
  uint32_t dx_groups;  // the first workgroups' product is dX, whose shares of K take longest
  // the bias gradient: the sum of `shares` rows of `sums`, at the end of the grid; NULL: none
  const float *sums;
  void *dbias;
  int32_t shares;
};
constexpr int kGradTile = 128, kGradStage = 64;
uint32_t launch_grad_products(uint32_t type, const GradProductsParams &p, hipStream_t s);

} // namespace zluda_amd
