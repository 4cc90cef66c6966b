// The entry points of include/zluda_ffn.h for products grouped by expert: argument checks, kernel choice and launches.
#include "../../include/zluda_ffn.h"

#include "ffn_checks.hpp"
#include "ffn_grouped_choice.hpp"
#include "ffn_grouped_launch.hpp"
#include "planner.hpp"

using namespace zluda_amd;

namespace {

uint32_t check_sizes(uint64_t rows, uint64_t experts, uint64_t features, uint64_t model, const int32_t *offsets) {
  if (!experts || !features || !model || ((uintptr_t)offsets & 3) || !offsets) return CUBLAS_STATUS_INVALID_VALUE;
  return rows > kMaxSide || experts > ZLUDA_FFN_MAX_EXPERTS || features > kMaxFeatures || model > kMaxFeatures ? CUBLAS_STATUS_NOT_SUPPORTED : CUBLAS_STATUS_SUCCESS;
}

uint32_t check_forward(const zluda_ffn_grouped *p) {
  if (!p) return CUBLAS_STATUS_INVALID_VALUE;
  FFN_CHECK(check_sizes(p->rows, p->experts, p->features, p->model, p->offsets));
  const uint32_t type = p->x.type;
  if (type == CUDA_R_8F_E4M3) {
    if (!is_h16(p->y.type) && p->y.type != CUDA_R_32F) return CUBLAS_STATUS_NOT_SUPPORTED;
    if ((!p->x.scales && p->rows) || ((uintptr_t)p->x.scales & 3) || p->x.ld_scales < (int64_t)p->rows) return CUBLAS_STATUS_INVALID_VALUE;
    if (!p->w.scales || ((uintptr_t)p->w.scales & 3) || p->w.ld_scales < (int64_t)((p->model + 127) / 128)) return CUBLAS_STATUS_INVALID_VALUE;
  } else if (!is_h16(type) || p->y.type != type) {
    return CUBLAS_STATUS_NOT_SUPPORTED;
  }
  FFN_CHECK(check_plain(p->x, p->rows, p->model, type));
  FFN_CHECK(check_plain(p->w, p->experts * p->features, p->model, type));
  return check_plain(p->y, p->rows, p->features, p->y.type);
}

uint32_t check_backward(const zluda_ffn_grouped_grad *p) {
  if (!p) return CUBLAS_STATUS_INVALID_VALUE;
  FFN_CHECK(check_sizes(p->rows, p->experts, p->features, p->model, p->offsets));
  const uint32_t type = p->dy.type;
  if (!is_h16(type)) return CUBLAS_STATUS_NOT_SUPPORTED;
  FFN_CHECK(check_plain(p->dy, p->rows, p->features, type));
  if (p->dx.data) {
    FFN_CHECK(check_plain(p->dx, p->rows, p->model, type));
    FFN_CHECK(check_plain(p->w, p->experts * p->features, p->model, type));
  }
  if (p->dw.data) {
    FFN_CHECK(check_plain(p->dw, p->experts * p->features, p->model, type));
    FFN_CHECK(check_plain(p->x, p->rows, p->model, type));
  }
  return !p->dx.data && !p->dw.data ? CUBLAS_STATUS_INVALID_VALUE : CUBLAS_STATUS_SUCCESS;
}

// the kernel for any alignment: `cols` of D in tiles of 64, and slots for the row tiles of 64
dim3 any_grid(uint64_t cols, uint64_t rows, uint64_t experts) {
  return dim3((uint32_t)((cols + 63) / 64), (uint32_t)std::min<uint64_t>((rows + 63) / 64 + std::min(experts, rows), kGridY));
}

// 16-byte pieces of the operands' rows; tiles whose rows, and the scales of a block of K, lie within reach of 32-bit offsets
bool tile_operands(const zluda_ffn_grouped *p) {
  const int64_t size = (int64_t)elem_size(p->x.type);
  const bool aligned = !(((uintptr_t)p->x.data | (uintptr_t)p->w.data | (uintptr_t)(p->x.ld * size) | (uintptr_t)(p->w.ld * size) | (p->model * size)) & 15);
  const bool near = p->x.ld < kNarrowPitch && p->w.ld < kNarrowPitch && p->y.ld < kNarrowPitch &&
                    (size != 1 || (p->x.ld_scales * (int64_t)((p->model + 127) / 128) < (1 << 28) && p->w.ld_scales < (1 << 28)));
  return aligned && near;
}

// Tiles of 128 x 128, two workgroups a CU, with dx's K in as many shares as grad_together_stages() has done first, or of 256 x 256; a stage takes 1.0 and 1.65 us.
// Measured, us, 1 share, 2, 4, 8, tiles of 256: 64 rows of eight experts, 2048 of model, 5632 features 106, 86, 98, 98, 149; 1024 123, 117, 127, 146, 160; 300,
// eight, 1024 x 2816 50, 37, 31, 31, 70; 692, two, 2688 x 4744 83, 68, 71, 84, 115; 64, one, 4096 x 4096 43, 29, 21, 23, 60; 600, 16, 2048 x 1408 46, 59, 65, 69, 49;
// 2000, two, 1024 x 1024 19, 25, 32, 45, 27; without shares and on 256: 2048 of model, 5632 features, eight experts, 4096 rows 261 and 223, 16384 821 and 668;
// 1024 x 2816, 64 experts, 16384 rows 356 and 309; 512 x 2048, 16, 16384 101 and 82.
struct GradChoice {
  uint64_t side;                    // of the tiles
  uint32_t splits, split_stages;    // shares of dx's K
  uint64_t part;                    // bytes of their sums
};
GradChoice pick_grad(const zluda_ffn_grouped_grad *p) {
  // (pace: a stage of a share waits for W, the longer where W and dW are more than the memory-side cache; as for the gated layer, grad_together())
  const uint64_t live = std::max<uint64_t>(1, std::min(p->rows, p->experts)), pace = 4 * p->experts * p->features * p->model > 256ull << 20 ? 2 : 1;
  GradChoice best{0, 1, 0, 0};
  double best_us = 0.0;
  for (uint64_t side : {128, 256}) {
    const uint64_t slots = (uint64_t)cus() * (side == 256 ? 1 : 2);
    auto tiles = [&](uint64_t n) { return (n + side - 1) / side; };
    auto stages = [](uint64_t k) { return (k + kGradStage - 1) / kGradStage; };
    const uint64_t n_dx = p->dx.data ? tiles(p->model) * std::max<uint64_t>(live, p->rows / side + (live + 1) / 2) : 0;
    const uint64_t n_dw = p->dw.data ? tiles(p->model) * tiles(p->features) * p->experts : 0, k_dx = stages(p->features);
    for (uint64_t n : {1, 2, 3, 4, 6, 8, 12, 16}) {
      if (n > 1 && (side == 256 || !n_dx || n_dx >= slots || n > k_dx)) break;
      const double us = grad_together_stages(slots, n_dx, k_dx, n_dw, stages(p->rows / p->experts), n, pace) * (side == 256 ? 1.65 : 1.0);
      if (best.side && us >= best_us) continue;
      best = {side, 1, (uint32_t)((k_dx + n - 1) / n), 0};
      best.splits = (uint32_t)((k_dx + best.split_stages - 1) / best.split_stages);
      best.part = best.splits > 1 ? best.splits * p->rows * tiles(p->model) * side * 4 : 0;
      best_us = us;
    }
  }
  return best;
}

// the same for the gradients, through windows of 2 GiB on an expert's matrices and rows; whole pieces of eight along every row
bool tile_shapes(const zluda_ffn_grouped_grad *p) {
  int64_t ld = p->dy.ld, most = p->dy.ld, least = p->dy.ld;  // (a workspace is asked for before pitches are checked)
  if (p->dx.data) { ld |= p->w.ld | p->dx.ld; most = std::max({most, p->w.ld, p->dx.ld}); least = std::min({least, p->w.ld, p->dx.ld}); }
  if (p->dw.data) { ld |= p->x.ld | p->dw.ld; most = std::max({most, p->x.ld, p->dw.ld}); least = std::min({least, p->x.ld, p->dw.ld}); }
  if ((ld & 7) || (p->model & 7) || (p->features & 7) || most >= kNarrowPitch || least < 1) return false;
  return in_window(p->rows, p->dy.ld) && (!p->dx.data || in_window(p->features, p->w.ld)) && (!p->dw.data || in_window(p->rows, p->x.ld));
}
bool tile_operands(const zluda_ffn_grouped_grad *p) {
  uintptr_t at = (uintptr_t)p->dy.data;
  if (p->dx.data) at |= (uintptr_t)p->w.data | (uintptr_t)p->dx.data;
  if (p->dw.data) at |= (uintptr_t)p->x.data | (uintptr_t)p->dw.data;
  return !(at & 15) && tile_shapes(p);
}

} // namespace

extern "C" uint32_t zluda_ffn_grouped_forward_workspace(const zluda_ffn_grouped *p, size_t *bytes) {
  if (!p || !bytes) return CUBLAS_STATUS_INVALID_VALUE;
  *bytes = 0;
  return CUBLAS_STATUS_SUCCESS;
}

extern "C" uint32_t zluda_ffn_grouped_forward(const zluda_ffn_grouped *p, void *workspace, size_t workspace_size, void *stream) {
  FFN_CHECK(check_forward(p));
  if (!p->rows) return CUBLAS_STATUS_SUCCESS;
  if (!zluda_gemm_device_cu_count()) return CUBLAS_STATUS_NOT_INITIALIZED;
  const GroupedParams g{p->offsets, p->x.data, p->w.data, p->y.data, (const float *)p->x.scales, (const float *)p->w.scales, p->x.ld, p->w.ld, p->y.ld,
                        p->x.ld_scales, p->w.ld_scales, (int32_t)p->rows, (int32_t)p->experts, (int32_t)p->features, (int32_t)p->model, p->x.type, p->y.type};
  if (tile_operands(p)) {
    const int tile = grouped_tile(p, (uint64_t)cus());
    if (((p->features + kBlockTiles[tile].bp - 1) / kBlockTiles[tile].bp) * most_row_tiles(p->rows, p->experts, kBlockTiles[tile].bq) < (1ull << 31))
      return (p->x.type == CUDA_R_16BF ? launch_grouped_bf16 : p->x.type == CUDA_R_16F ? launch_grouped_f16 : launch_grouped_f8)(g, tile, (hipStream_t)stream);
  }
  return launch_kernel(grouped_any_kernel<0>, any_grid(p->features, p->rows, p->experts), dim3(256), (hipStream_t)stream, g);
}

extern "C" uint32_t zluda_ffn_grouped_backward_workspace(const zluda_ffn_grouped_grad *p, size_t *bytes) {
  if (!p || !bytes) return CUBLAS_STATUS_INVALID_VALUE;
  *bytes = 0;
  if (check_sizes(p->rows, p->experts, p->features, p->model, (const int32_t *)16)) return check_sizes(p->rows, p->experts, p->features, p->model, (const int32_t *)16);
  if (tile_shapes(p)) *bytes = pick_grad(p).part;
  return CUBLAS_STATUS_SUCCESS;
}

extern "C" uint32_t zluda_ffn_grouped_backward(const zluda_ffn_grouped_grad *p, void *workspace, size_t workspace_size, void *stream) {
  FFN_CHECK(check_backward(p));
  const GradChoice pick = pick_grad(p);
  const uint64_t need = tile_shapes(p) ? pick.part : 0;
  if (need > workspace_size || (need && !workspace)) return CUBLAS_STATUS_ALLOC_FAILED;
  if (need && ((uintptr_t)workspace & 15)) return CUBLAS_STATUS_INVALID_VALUE;
  if (!zluda_gemm_device_cu_count()) return CUBLAS_STATUS_NOT_INITIALIZED;
  const hipStream_t s = (hipStream_t)stream;
  if (tile_operands(p)) {
    auto tiles = [&](uint64_t n) { return (n + pick.side - 1) / pick.side; };
    const uint64_t dx = p->dx.data && p->rows ? tiles(p->model) * most_row_tiles(p->rows, p->experts, pick.side) * pick.splits : 0;
    const uint64_t dw = p->dw.data ? tiles(p->model) * tiles(p->features) * p->experts : 0;
    if (dx + dw == 0) return CUBLAS_STATUS_SUCCESS;
    if (dx + dw < (1ull << 31)) {
      const GroupedGradParams q{p->offsets, p->dy.data, p->x.data, p->w.data, p->dx.data, p->dw.data, p->dx.ld, p->dw.ld, (int32_t)p->dy.ld, (int32_t)p->x.ld, (int32_t)p->w.ld,
                                (int32_t)p->rows, (int32_t)p->experts, (int32_t)p->features, (int32_t)p->model, (uint32_t)dx, (float *)workspace, (int32_t)pick.splits,
                                (int32_t)pick.split_stages};
      FFN_CHECK(launch_grouped_grad(q, p->dy.type, (int)pick.side, (uint32_t)(dx + dw), s));
      if (!dx || pick.splits == 1) return CUBLAS_STATUS_SUCCESS;
      const int64_t pitch = (int64_t)(tiles(p->model) * pick.side);
      const RoundParams r{q.part, p->dx.data, (int64_t)p->rows, pitch, p->dx.ld, (int64_t)p->rows * pitch, (int32_t)p->model, (int32_t)pick.splits};
      return launch_grouped_round(r, p->dy.type, p->offsets, q.experts, dim3(column_strips(p->model), (uint32_t)std::min<uint64_t>((p->rows + 3) / 4, kGridY)), s);
    }
  }
  GroupedParams g{p->offsets, p->dy.data, p->w.data, p->dx.data, nullptr, nullptr, p->dy.ld, p->w.ld, p->dx.ld, 0, 0, (int32_t)p->rows, (int32_t)p->experts,
                  (int32_t)p->features, (int32_t)p->model, p->dy.type, p->dy.type};
  if (p->dx.data && p->rows) FFN_CHECK(launch_kernel(grouped_any_kernel<1>, any_grid(p->model, p->rows, p->experts), dim3(256), s, g));
  if (!p->dw.data) return CUBLAS_STATUS_SUCCESS;
  g.b = p->x.data; g.ldb = p->x.ld; g.d = p->dw.data; g.ldd = p->dw.ld;
  const dim3 grid((uint32_t)((p->model + 63) / 64), (uint32_t)((p->features + 63) / 64), (uint32_t)p->experts);
  return launch_kernel(grouped_any_kernel<2>, grid, dim3(256), s, g);
}
