// Which kernel a feed-forward call takes, and in how many workgroups: rules on sizes, pitches and alignment, without HIP.
#pragma once
#include <algorithm>
#include <cstdint>

#include "../../include/zluda_ffn.h"
#include "kernels/store_window.hpp"

namespace zluda_amd {

constexpr uint64_t kMaxSide = 0x7fffff00;             // sizes are 32-bit numbers inside the kernels, with room to round up to 256
constexpr uint64_t kMaxFeatures = 1 << 20;            // (2^15 blocks of 32 along a grid's second dimension)

// strips of 512 columns: what a wave of the row-wise kernels takes, eight columns a thread (a width up to kMaxSide has no room for 511 more in 32 bits)
constexpr uint32_t column_strips(uint64_t cols) { return (uint32_t)((cols + 511) / 512); }

// ---- gated products -------------------------------------------------------------------------------------------------------------
// The tiles of the gated products: `features` x `tokens` a workgroup, its waves wp x wq, LDS stages, and the time of a stage (of
// 64 K elements) in a full chip, us for each tile of a CU.  From whole calls of 4096 x 14336 and 1024 tokens: 437, 304, 262, 230 us, and
// 241 and 199 with the last two, the persistent four-wave kernel; smaller tiles are less work between two barriers and read more
// of LDS for each product.
struct GatedTile { int features, tokens, wp, wq, stages; float stage_us; };
constexpr GatedTile kGatedTiles[] = {{64, 32, 2, 2, 4, 0.24f},   {64, 64, 2, 2, 3, 0.335f},  {64, 128, 2, 2, 3, 0.58f},
                                     {128, 128, 4, 2, 3, 0.9f}, {128, 192, 2, 2, 2, 1.18f}, {128, 256, 2, 2, 2, 1.4f}};
constexpr int kGatedTileCount = 6, kGatedPersistent = 4;  // (from there on)

// 16-byte pieces of the operands' rows, through 2 GiB buffer windows
template <class Params>
inline bool gated_dma_operands(const Params &p) {
  return p.model % 8 == 0 && p.ldx % 8 == 0 && p.ldw % 8 == 0 && !(((uintptr_t)p.x | (uintptr_t)p.w) & 15) &&
         (2ll * p.features * p.ldw + p.model) * 2 < 0x7fffffffll && ((int64_t)p.tokens * p.ldx + p.model) * 2 < 0x7fffffffll;
}

// The tile whose slowest CU is done first: rounds of tiles over the CUs, each the stages of K (and the time of three for its
// start and end).  All tiles share the bound of the one read of W, under which their differences vanish.
// Measured, us, in the order of kGatedTiles: 64 tokens, 4096 x 14336: 57, 48, 53, 64, 89, 96; 256: 133, 106, 89, 72, 92, 107; 384: 190, 142,
// 121, 119, 101, 108; 777: 450, 295, 239, 217, 219, 181; 300, 2048 x 5632: 34, 23, 37, 30, 37, 43; 2000: 171, 115, 109, 92, 76, 89.
template <class Params>
inline int gated_tile(const Params &p, int cus) {
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

// ---- the products of the gated layer's backward pass ----------------------------------------------------------------------------------
// The matmul kernels reach an operand through a window of 2 GiB.  Rows of one of pitch `ld` (16-bit elements) that lie inside one, what a kernel
// asks for past their end included; all of them where they are wider apart than that helps.  A call of more rows is run in parts of
// so many (40000 tokens, 2048 x 16384: dX 187 ms on the kernel without a window, 5.1 in two parts, dW 203 and 5.6; forward 300000 tokens,
// 4096 x 1024: 3.6 ms, 1390 TFLOP/s).
inline uint64_t rows_in_window(uint64_t rows, int64_t ld) {
  const int64_t most = ld < 1 ? 0 : (0x3fffffffll / ld - 256) & ~255ll;  // (a workspace is asked for before pitches are checked)
  return most > 0 && rows > (uint64_t)most ? (uint64_t)most : rows;
}
inline bool in_window(uint64_t rows, int64_t ld) { return (int64_t)(rows + 256) <= 0x3fffffffll / ld; }

constexpr int kGradTile = 128, kGradStage = 64;

// dX and dW in one launch of 128 x 128 tiles (kernels/ffn_grad_products.hpp), or one after the other on the framework's matmul kernels?  Together, us
// of whole backward passes and in brackets one after the other: 64 tokens, 4096 x 14336 118 (167), 300, 2048 x 5632 59 (70), 700, 4096 x 14336
// 399 (451), 1100 594 (663), 1001, 1024 x 2816 46 (55), 1500, 2048 x 8192 238 (270), 5000, 1024 x 8192 388 (465), 3000, 4096 x 2816 284 (286).
// One after the other
//  * where both fill the chip by themselves, dW twice with tiles of 256 x 256, which compute faster (2000, 4096 x 11008 758 and 709; 8192, 2048 x
//    8192 1152 and 925);
//  * where a tile of dW alone takes more than twice the time all tiles take the chip: its K is not shared out here (8192, 1024 x 512 105 and 60;
//    3000, 512 x 512 38 and 33; with as much as twice 4096, 1024 x 1024 61 and 64, 8192, 512 x 2048 148 and 131).
struct GradTogether {
  uint32_t splits, split_stages;  // shares of dX's K; 0: one after the other
  uint64_t part;                  // bytes of their sums
};
// Stages until the launch is done, of `slots` workgroups at a time that take dX's n_dx * s shares, then the tiles of dW: half way between an even load
// and one workgroup after the other at an even pace (one without a neighbour is faster, but not by as much).  A tile's start and end are as
// long as three stages; a stage of a share takes `pace` quarters more than one at an even load, as it waits for W; the shares' sums are written and
// read again, in a launch of their own.  Measured, us, shares of dX and times: 1001, 1024 x 2816 1: 71, 2: 49, 3: 46, 4: 49, 8: 49; 300, 2048 x 5632 3: 60,
// 5: 56, 8: 57; 700, 4096 x 14336 1: 459, 2: 393, 3: 415; 2000, 1024 x 1024 1: 32, 2: 41; W from memory: 150, 4096 x 14336 3: 195, 5: 169, 8: 168, 12: 176;
// 64, 4096 x 14336 3: 181, 8: 118, 12: 131; 100, 5120 x 13824 3: 198, 5: 164, 8: 168.
inline double grad_together_stages(uint64_t slots, uint64_t n_dx, uint64_t k_dx, uint64_t n_dw, uint64_t k_dw, uint64_t s, uint64_t pace) {
  const uint64_t l1 = (k_dx + s - 1) / s + 3, l2 = k_dw + 3, n1 = n_dx * s, even = (n1 * l1 + n_dw * l2) / slots, rounds = n1 / slots, rest = n1 % slots;
  uint64_t low = std::max(even, rounds * l1 + (rest ? l1 + l1 * pace / 4 : 0)), high = low + l1 + (n_dw / slots + 2) * l2;  // (dW's tiles fit behind `high`)
  while (low < high) {
    const uint64_t end = (low + high) / 2, early = end > rounds * l1 ? (end - rounds * l1) / l2 : 0, late = end > (rounds + 1) * l1 ? (end - (rounds + 1) * l1) / l2 : 0;
    if ((slots - rest) * early + rest * late >= n_dw) high = end;
    else low = end + 1;
  }
  return 0.5 * (double)(even + low) + (s > 1 ? 5.0 + 0.04 * (double)n1 : 0.0);
}
inline GradTogether grad_together(const zluda_ffn_gated_grad *p, int cus) {
  GradTogether g{0, 0, 0};
  if (!p->dx.data || !p->dw.data || !p->tokens || p->model % 8 || p->features % 4) return g;
  auto tiles = [](uint64_t a, uint64_t b, uint64_t side) { return ((a + side - 1) / side) * ((b + side - 1) / side); };
  const uint64_t f2 = 2 * p->features, slots = 2 * (uint64_t)cus, n_dx = tiles(p->model, p->tokens, kGradTile), n_dw = tiles(p->model, f2, kGradTile);
  const uint64_t k_dx = (f2 + kGradStage - 1) / kGradStage, k_dw = (p->tokens + kGradStage - 1) / kGradStage;
  const uint64_t all = (n_dx * k_dx + n_dw * k_dw + slots - 1) / slots;  // stages of a workgroup if they were shared out evenly
  if ((n_dx >= slots && tiles(p->model, f2, 256) >= slots) || k_dw > 2 * all) return g;
  const uint64_t pace = 8 * p->features * p->model > 256ull << 20 ? 2 : 1;  // (W and dW are more than the memory-side cache)
  uint64_t want = 1;
  double best = 0.0;
  for (uint64_t n = 1; n <= std::min<uint64_t>(16, k_dx); n++) {
    const double stages = grad_together_stages(slots, n_dx, k_dx, n_dw, k_dw, n, pace);
    if (n == 1 || stages < best) {
      want = n;
      best = stages;
    }
  }
  g.split_stages = (uint32_t)((k_dx + want - 1) / want);
  g.splits = (uint32_t)((k_dx + g.split_stages - 1) / g.split_stages);
  g.part = g.splits > 1 ? g.splits * n_dx * kGradTile * kGradTile * 4 : 0;
  return g;
}

// 16-byte pieces of all operands and results, through windows of 2 GiB
inline bool grad_together_operands(const zluda_ffn_gated_grad *p, const zluda_ffn_matrix &x, int64_t lddz, const void *dz) {
  return !((p->w.ld | x.ld | lddz | p->dx.ld | p->dw.ld) & 7) && p->dx.ld < kNarrowPitch && p->dw.ld < kNarrowPitch &&
         !(((uintptr_t)p->w.data | (uintptr_t)x.data | (uintptr_t)dz | (uintptr_t)p->dx.data | (uintptr_t)p->dw.data) & 15) && in_window(p->tokens, x.ld) &&
         in_window(p->tokens, lddz) && in_window(2 * p->features, p->w.ld);
}

// One after the other: tiles of 256 x 256 wherever they fill the chip twice; the planner's own choice, made from the time of a single stage, takes half-size
// ones for some of these (A:N B:T 2360 x 15440 x 6196, 610 tiles: 443 us on them, 557 on 128 x 128).
inline bool grad_largest_tiles(uint64_t m, uint64_t n, uint64_t cus) { return ((m + 255) / 256) * ((n + 255) / 256) >= 2 * cus; }

} // namespace zluda_amd
