// Launchers of the feed-forward products, one translation unit per element type.
#pragma once
#include <hip/hip_runtime.h>

#include "ffn_launch.hpp"
#include "kernels/ffn_gated_store.hpp"
#include "launch_util.hpp"

namespace zluda_amd {

uint32_t launch_gated_bf16(const GatedParams &p, hipStream_t s);
uint32_t launch_gated_f16(const GatedParams &p, hipStream_t s);

// in one of the first four of kGatedTiles, or (tile < 0) at any alignment
uint32_t launch_gated_small_bf16(const GatedParams &p, int tile, hipStream_t s);
uint32_t launch_gated_small_f16(const GatedParams &p, int tile, hipStream_t s);

// ---- the products of the backward pass in one launch (kernels/ffn_grad_products.hpp) ----------------------------------------------
// D[q][p] = sum over k of P[k][p] Q, Q as [q][k] (dX) or [k][q] (dW).  With `splits` > 1 share z of K writes 32-bit sums to
// part[z][q][p], p padded to whole tiles, part_rows rows of q, part_plane floats from share to share.
struct GradProduct {
  const void *p, *q;
  void *d;
  float *part;
  int64_t ldd;
  int32_t ldp, ldq;
  int32_t np, nq, k;
  int32_t tiles_p, tiles_q, splits, split_stages;
  int64_t part_plane;
  int32_t part_rows;
};
struct GradProductsParams {
  GradProduct dx, dw;
  uint32_t dx_groups;  // the first workgroups' product is dX, whose shares of K take longest
  // the bias gradient: the sum of `shares` rows of `sums`, at the end of the grid; NULL: none
  const float *sums;
  void *dbias;
  int32_t shares;
};
uint32_t launch_grad_products(uint32_t type, const GradProductsParams &p, hipStream_t s);

} // namespace zluda_amd
