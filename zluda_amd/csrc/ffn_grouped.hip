// The entry points of include/zluda_ffn.h for products grouped by expert: argument checks, kernel choice and launches.
#include "../../include/zluda_ffn.h"

#include "ffn_checks.hpp"
#include "kernels/ffn_grouped.hpp"

using namespace zluda_amd;

namespace {

uint32_t check_sizes(uint64_t rows, uint64_t experts, uint64_t features, uint64_t model, const int32_t *offsets) {
  if (!experts || !features || !model || ((uintptr_t)offsets & 3) || !offsets) return CUBLAS_STATUS_INVALID_VALUE;
  return rows > kMaxSide || experts > ZLUDA_FFN_MAX_EXPERTS || features > kMaxFeatures || model > kMaxFeatures ? CUBLAS_STATUS_NOT_SUPPORTED : CUBLAS_STATUS_SUCCESS;
}
uint32_t check_plain(const zluda_ffn_matrix &m, uint64_t rows, uint64_t cols, uint32_t type) {
  if (!m.data && rows) return CUBLAS_STATUS_INVALID_VALUE;
  if (m.type != type) return CUBLAS_STATUS_NOT_SUPPORTED;
  return m.ld < (int64_t)cols || ((uintptr_t)m.data & (elem_size(type) - 1)) ? CUBLAS_STATUS_INVALID_VALUE : CUBLAS_STATUS_SUCCESS;
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
  return launch_kernel(grouped_any_kernel<0>, any_grid(p->features, p->rows, p->experts), dim3(256), (hipStream_t)stream, g);
}

extern "C" uint32_t zluda_ffn_grouped_backward_workspace(const zluda_ffn_grouped_grad *p, size_t *bytes) {
  if (!p || !bytes) return CUBLAS_STATUS_INVALID_VALUE;
  *bytes = 0;
  return CUBLAS_STATUS_SUCCESS;
}

extern "C" uint32_t zluda_ffn_grouped_backward(const zluda_ffn_grouped_grad *p, void *workspace, size_t workspace_size, void *stream) {
  FFN_CHECK(check_backward(p));
  if (!zluda_gemm_device_cu_count()) return CUBLAS_STATUS_NOT_INITIALIZED;
  const hipStream_t s = (hipStream_t)stream;
  GroupedParams g{p->offsets, p->dy.data, p->w.data, p->dx.data, nullptr, nullptr, p->dy.ld, p->w.ld, p->dx.ld, 0, 0, (int32_t)p->rows, (int32_t)p->experts,
                  (int32_t)p->features, (int32_t)p->model, p->dy.type, p->dy.type};
  if (p->dx.data && p->rows) FFN_CHECK(launch_kernel(grouped_any_kernel<1>, any_grid(p->model, p->rows, p->experts), dim3(256), s, g));
  if (!p->dw.data) return CUBLAS_STATUS_SUCCESS;
  g.b = p->x.data; g.ldb = p->x.ld; g.d = p->dw.data; g.ldd = p->dw.ld;
  const dim3 grid((uint32_t)((p->model + 63) / 64), (uint32_t)((p->features + 63) / 64), (uint32_t)p->experts);
  return launch_kernel(grouped_any_kernel<2>, grid, dim3(256), s, g);
}
