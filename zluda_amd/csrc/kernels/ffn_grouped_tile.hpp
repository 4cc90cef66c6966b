// Products grouped by expert on the tiles of block_tile.hpp: P is an expert's matrix (features), Q its rows.
//
// A grid has a workgroup for each tile of features and each row tile that there can be; those without one end at once.  The tiles that there are get the
// order of the other products (work_item()): every XCD takes a contiguous range of row tiles, expert after expert, eight tiles of features at a
// time, so that what it reads of an expert's matrix serves all of the expert's rows from its L2.
#pragma once
#include "block_tile.hpp"
#include "ffn_grad_products.hpp"
#include "ffn_grouped.hpp"

namespace zluda_amd {

struct GroupedItem { RowTile rows; int p; };  // rows.e < 0: nothing to do
__device__ __forceinline__ GroupedItem grouped_item(const GroupedParams &p, int tiles_p, int side, uint32_t id, uint32_t groups) {
  GroupedItem it;
  it.rows = RowTile{-1, 0, 0, 0};
  it.p = 0;
  MfmaParams at;
  at.tiles_p = tiles_p; at.tiles_q = count_row_tiles(p.offsets, p.experts, p.rows, side, (int)(groups / (uint32_t)tiles_p)); at.g.batch = 1; at.splits = 1; at.group_p = 8;
  if (id >= (uint32_t)tiles_p * (uint32_t)at.tiles_q) return it;
  const WorkItem w = work_item(at, id);
  it.rows = find_row_tile(p.offsets, p.experts, p.rows, side, w.q);
  it.p = w.p;
  return it;
}

// KIND: that of block_tile.hpp; DT: of y, 0 bf16, 1 f16, 2 f32
template <int KIND, int DT, int BP, int BQ, int WP, int WQ, int NS>
__global__ __launch_bounds__(WP *WQ * 64, 2) void grouped_tile_kernel(GroupedParams p) {
  constexpr bool WIDE = BP == 256, F8 = kind_is_block8(KIND);
  using Ring = RingTile<KIND, 0, 0, true, WIDE ? 64 : BP, WIDE ? 64 : BQ, 2, 2, NS>;
  using Wide = WideTile<KIND == KIND_F8_WIDE ? KIND_F8 : KIND, 0, 0>;
  constexpr int TP = BP / WP / 16, TQ = BQ / WQ / 16, WORDS = WIDE ? Wide::WORDS : Ring::WORDS, ESZ = F8 ? 1 : 2;
  __shared__ v4i lds[WORDS];
  const int tiles_p = (p.features + BP - 1) / BP;
  const GroupedItem it = grouped_item(p, tiles_p, BQ, blockIdx.x, gridDim.x);
  if (it.rows.e < 0) return;
  const int p0 = it.p * BP, q0 = it.rows.at, kbytes = p.model * ESZ, stages = (kbytes + 127) / 128;
  TileSide P, Q;
  P.data = (const uint8_t *)p.b + ((int64_t)it.rows.e * p.features + p0) * p.ldb * ESZ;
  P.ld = (int)p.ldb * ESZ;
  P.rows = p.features - p0;
  Q.data = (const uint8_t *)p.a + ((int64_t)it.rows.first + q0) * p.lda * ESZ;
  Q.ld = (int)p.lda * ESZ;
  Q.rows = it.rows.n - q0;
  P.scales = p.b_scales; P.s_row = P.s_step = 0; P.per_row = false; P.s_at = p0 & 127;
  Q.scales = p.a_scales; Q.s_row = Q.s_step = 0; Q.per_row = true; Q.s_at = 0;
  if constexpr (F8) {
    P.scales += ((int64_t)it.rows.e * ((p.features + 127) >> 7) + (p0 >> 7)) * p.ldb_scales;
    P.s_row = (int)p.ldb_scales; P.s_step = 1;
    Q.scales += it.rows.first + q0;
    Q.s_row = 1; Q.s_step = (int)p.lda_scales;
  }
  v4f acc[TP][TQ];
  if constexpr (WIDE) Wide::run(P, Q, kbytes, 0, stages, lds, acc);
  else Ring::run(P, Q, kbytes, 0, stages, (it.p + it.rows.e) * 3 % stages, lds, acc);
  // y of the expert's rows as a column-major matrix of features x rows
  MfmaParams d;
  d.swapped = 0;
  d.g.alpha_mode = d.g.beta_mode = SCALAR_VALUE; d.g.alpha_val.f = 1.0f; d.g.beta_val.f = 0.0f; d.g.int_scale = 0;
  d.g.alpha_ptr = d.g.beta_ptr = d.g.a_scale = d.g.b_scale = d.g.c_scale = d.g.d_scale = d.g.bias = d.g.C = nullptr;
  d.g.a_scale_mode = d.g.b_scale_mode = SCALE_NONE;
  d.g.act = ACT_NONE;
  d.g.d_type = DT == 0 ? CUDA_R_16BF : DT == 1 ? CUDA_R_16F : CUDA_R_32F;
  d.g.d_si = 1; d.g.d_sj = p.ldd; d.g.d_sb = 0;
  d.g.alpha_sb = d.g.bias_sb = 0;
  d.g.D = (char *)p.d + it.rows.first * p.ldd * (DT == 2 ? 4 : 2);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (p0 + BP <= p.features) mfma16_store_f<KIND_F8, WP, WQ, TP, TQ, DT, ACT_NONE, false>(d, acc, p0, q0, p.features, it.rows.n, 0, wave);
  else mfma16_store_f<KIND_F8, WP, WQ, TP, TQ, DT, ACT_NONE, true>(d, acc, p0, q0, p.features, it.rows.n, 0, wave);
}

} // namespace zluda_amd
