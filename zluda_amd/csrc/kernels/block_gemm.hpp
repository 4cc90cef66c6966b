// cublasLtMatmul of 8-bit floats with a float scale for each 128 of K (SCALE_VEC128, SCALE_BLK128) on the tiles of block_tile.hpp; the epilogues are those
// of the other kernels on the 16x16 MFMA shapes.
#pragma once
#include "block_tile.hpp"

namespace zluda_amd {

// P and Q of the tile whose first rows are p0 and q0, in batch bt
__device__ __forceinline__ void block_sides(const MfmaParams &prm, int p0, int q0, int bt, TileSide &P, TileSide &Q) {
  const GemmArgs &g = prm.g;
  auto side = [&](bool of_a, int r0) {
    TileSide s;
    const int all = of_a ? g.M : g.N;
    const int64_t ld = of_a ? g.a_si : g.b_sj, blocks = blocks128(g.K), line = (blocks + 3) & ~3ll;
    s.data = (const uint8_t *)(of_a ? g.A : g.B) + (of_a ? g.a_sb : g.b_sb) * bt + r0 * ld;
    s.ld = (int)ld;
    s.rows = all - r0;
    const int mode = of_a ? g.a_scale_mode : g.b_scale_mode;
    const float *scales = (const float *)(of_a ? g.a_scale : g.b_scale) + scales128(mode, all, g.K) * bt;
    s.per_row = mode == SCALE_VEC128;
    s.scales = s.per_row ? scales + r0 : scales + (r0 >> 7) * line;
    s.s_row = s.per_row ? 1 : (int)line;
    s.s_step = s.per_row ? all : 1;
    s.s_at = r0 & 127;
    return s;
  };
  P = side(!prm.swapped, p0);
  Q = side(prm.swapped, q0);
}

// EXACT: results in 32 bits (KIND_F8_WIDE)
template <int FP, int FQ, bool SU, bool EXACT, int BP, int BQ, int WP, int WQ, int NS>
__global__ __launch_bounds__(WP *WQ * 64, 2) void block_gemm_kernel(MfmaParams prm) {
  constexpr bool WIDE = BP == 256;
  using Ring = RingTile<EXACT ? KIND_F8_WIDE : KIND_F8, FP, FQ, SU, WIDE ? 64 : BP, WIDE ? 64 : BQ, 2, 2, NS>;
  using Wide = WideTile<KIND_F8, FP, FQ>;
  constexpr int TP = BP / WP / 16, TQ = BQ / WQ / 16, WORDS = WIDE ? Wide::WORDS : Ring::WORDS;
  __shared__ v4i lds[WORDS];
  fetch_args(prm);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wp = wave % WP, wq = wave / WP;
  const WorkItem item = work_item(prm);
  const int p0 = item.p * BP, q0 = item.q * BQ;
  TileSide P, Q;
  block_sides(prm, p0, q0, item.bt, P, Q);
  const int all = (prm.g.K + 127) / 128;
  int first = 0, stages = all;
  if (prm.splits > 1) {
    first = item.z * prm.split_stages;
    stages = max(0, min(all - first, prm.split_stages));
  }
  v4f acc[TP][TQ];
  // (tiles start their walk along K apart from each other: rows a power of two apart share memory channels)
  if constexpr (WIDE) Wide::run(P, Q, prm.g.K, first, stages, lds, acc);
  else Ring::run(P, Q, prm.g.K, first, stages, stages > 0 ? item.p * 3 % stages : 0, lds, acc);
  const int NP = prm.swapped ? prm.g.N : prm.g.M, NQ = prm.swapped ? prm.g.M : prm.g.N;
  if (prm.splits > 1) {
    const int ws_np = prm.tiles_p * BP, ws_nq = prm.tiles_q * BQ;
    int32_t *ws_tile = (int32_t *)prm.ws + ((int64_t)item.z * prm.g.batch + item.bt) * ws_np * ws_nq + (int64_t)(q0 + wq * TQ * 16) * ws_np + p0 + wp * TP * 16;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)ws_tile, 0, 0xFFFFFFFF, 0x00020000);
    mfma16_store_raw<false>(rs, ws_np, acc, 1, 0);
    return;
  }
  mfma16_store_tile<KIND_F8, WP, WQ, TP, TQ, WORDS * 16, false>(prm, acc, (int *)&lds[0], p0, q0, NP, NQ, item.bt, wave);
}

} // namespace zluda_amd
