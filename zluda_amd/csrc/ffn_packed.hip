// The entry points of include/zluda_ffn.h for RMS norm and packed matrices: argument checks, kernel choice and launches.
#include "../../include/zluda_ffn.h"

#include "ffn_checks.hpp"
#include "kernels/ffn_elementwise.hpp"
#include "kernels/ffn_rms.hpp"

using namespace zluda_amd;

namespace {

bool plain_type(uint32_t type) { return is_h16(type) || type == CUDA_R_32F; }

uint32_t check_packed(const zluda_ffn_matrix &m, uint64_t rows, uint64_t cols, uint32_t block_rows) {
  if ((!m.data || !m.scales) && rows) return CUBLAS_STATUS_INVALID_VALUE;
  if (m.type != CUDA_R_8F_E4M3) return CUBLAS_STATUS_NOT_SUPPORTED;
  const uint64_t least = block_rows == 1 ? rows : (cols + kPack - 1) / kPack;
  return m.ld < (int64_t)cols || m.ld_scales < (int64_t)least || ((uintptr_t)m.scales & 3) ? CUBLAS_STATUS_INVALID_VALUE : CUBLAS_STATUS_SUCCESS;
}

// ---- RMS norm -------------------------------------------------------------------------------------------------------------------
uint32_t check_rms(uint64_t rows, uint64_t cols, uint32_t type, uint32_t weight_type) {
  if (!cols) return CUBLAS_STATUS_INVALID_VALUE;
  return cols > ZLUDA_FFN_NORM_MAX_COLS || rows > (uint64_t)INT64_MAX / 2 || !plain_type(type) || (weight_type != type && weight_type != CUDA_R_32F)
             ? CUBLAS_STATUS_NOT_SUPPORTED : CUBLAS_STATUS_SUCCESS;
}

template <class E>
uint32_t launch_rms(RmsParams p, hipStream_t s) {
  auto run = [&](auto kernel, int rows_each, int per_cu, int threads) {
    const int64_t rounds = (p.rows + rows_each - 1) / rows_each, each = (rounds + (int64_t)cus() * per_cu - 1) / ((int64_t)cus() * per_cu);
    p.per_group = (int32_t)std::min<int64_t>(each * rows_each, 1 << 30);
    return launch_kernel(kernel, dim3((uint32_t)((p.rows + p.per_group - 1) / p.per_group)), dim3(threads), s, p);
  };
  // Eight columns a thread as long as a workgroup has enough of them (sixteen and half the threads in brackets, us): 4 x 1024 2.9 (3.7), 777 x 1001 3.9 (4.8), 16384 x 1024
  // 26.7 (28.1); 4 x 4096 3.1 (4.0), 2048 x 4096 14.4 (16.9), 16384 x 4096 110 (107); 500 x 8192 9.1 (9.5), 8192 x 8192 106 (108), packed 97.1 (97.6).  Beyond that,
  // packed, what the many small workgroups overlap is worth more: 16384 x 8192 198 (191), plain 208 (210).
  if (p.cols <= 512) return run(rms_forward_kernel<E, 64, 4, 1>, 4, 8, 256);
  if (p.cols <= 1024) return run(rms_forward_kernel<E, 128, 2, 1>, 2, 8, 256);
  if (p.cols <= 2048) return run(rms_forward_kernel<E, 256, 1, 1>, 1, 8, 256);
  if (p.cols <= 4096) return run(rms_forward_kernel<E, 512, 1, 1>, 1, 4, 512);
  if (p.cols <= 8192) return p.codes && p.rows > 8192 ? run(rms_forward_kernel<E, 512, 1, 2>, 1, 4, 512) : run(rms_forward_kernel<E, 1024, 1, 1>, 1, 2, 1024);
  return run(rms_forward_kernel<E, 1024, 1, 2>, 1, 1, 1024);
}

// Rows a workgroup of the gradient kernel takes at a time, and workgroups: one round of rows while that leaves an eighth of the CUs idle, two beyond (300 x 1000 7.3 us
// in one, 8.3 in two; 777 x 1001 8.8 and 9.2; 2000 x 512, 250 workgroups, 7.4 and 7.2: the second kernel has their sums to read), and no more workgroups than are
// resident at once.
int rms_grad_rows_each(uint64_t cols) { return cols <= 512 ? 8 : cols <= 1024 ? 4 : cols <= 2048 ? 2 : 1; }
uint32_t rms_grad_groups(uint64_t rows, uint64_t cols) {
  const int each = rms_grad_rows_each(cols), least = rows <= (uint64_t)cus() * 7 / 8 * each ? each : 2 * each;
  if (rows <= 3ull * each) return 1;
  return (uint32_t)std::min<uint64_t>((rows + least - 1) / least, (uint64_t)cus() * (cols <= 4096 ? 2 : 1));
}
template <class E>
uint32_t launch_rms_grad(const RmsGradParams &p, uint32_t groups, hipStream_t s) {
  if (p.cols <= 512) return launch_kernel(rms_backward_kernel<E, 64, 8, 1>, dim3(groups), dim3(512), s, p);
  if (p.cols <= 1024) return launch_kernel(rms_backward_kernel<E, 128, 4, 1>, dim3(groups), dim3(512), s, p);
  if (p.cols <= 2048) return launch_kernel(rms_backward_kernel<E, 256, 2, 1>, dim3(groups), dim3(512), s, p);
  if (p.cols <= 4096) return launch_kernel(rms_backward_kernel<E, 512, 1, 1>, dim3(groups), dim3(512), s, p);
  if (p.cols <= 8192) return launch_kernel(rms_backward_kernel<E, 1024, 1, 1>, dim3(groups), dim3(1024), s, p);
  return launch_kernel(rms_backward_kernel<E, 1024, 1, 2>, dim3(groups), dim3(1024), s, p);
}

// ---- packing --------------------------------------------------------------------------------------------------------------------
template <class E>
uint32_t launch_activate(const ActivateParams &p, uint32_t block_rows, hipStream_t s) {
  if (block_rows != 1) {
    const dim3 grid((uint32_t)((p.cols + (int64_t)kPack - 1) / kPack), (uint32_t)std::min<int64_t>((p.rows + kPack - 1) / kPack, kGridY));
    return launch_kernel(activate_blocks_kernel<E>, grid, dim3(256), s, p);
  }
  const uint32_t strips = column_strips(p.cols);
  return launch_kernel(activate_kernel<E>, dim3(strips, (uint32_t)std::min<int64_t>((p.rows + 3) / 4, kGridY)), dim3(256), s, p);
}

} // namespace

extern "C" uint32_t zluda_ffn_rms_forward(const zluda_ffn_rms *p, void *stream) {
  if (!p) return CUBLAS_STATUS_INVALID_VALUE;
  const uint32_t type = p->x.type;
  FFN_CHECK(check_rms(p->rows, p->cols, type, p->weight_type));
  FFN_CHECK(check_plain(p->x, p->rows, p->cols, type));
  if (p->residual.data) FFN_CHECK(check_plain(p->residual, p->rows, p->cols, type));
  if (p->sum.data) FFN_CHECK(check_plain(p->sum, p->rows, p->cols, type));
  if (p->y.data) FFN_CHECK(check_plain(p->y, p->rows, p->cols, type));
  if (p->packed.data) FFN_CHECK(check_packed(p->packed, p->rows, p->cols, 1));
  if (p->rows && ((!p->sum.data && !p->y.data && !p->packed.data) || (p->sum.data && p->sum.data == p->y.data))) return CUBLAS_STATUS_INVALID_VALUE;
  FFN_CHECK(check_vector(p->weight, p->weight_type));
  FFN_CHECK(check_vector(p->rstd, CUDA_R_32F));
  if (!p->rows) return CUBLAS_STATUS_SUCCESS;
  if (!zluda_gemm_device_cu_count()) return CUBLAS_STATUS_NOT_INITIALIZED;
  const RmsParams r{p->x.data, p->residual.data, p->sum.data, p->y.data, (uint8_t *)p->packed.data, (float *)p->packed.scales, p->weight, p->rstd, (int64_t)p->rows,
                    p->x.ld, p->residual.ld, p->sum.ld, p->y.ld, p->packed.ld, p->packed.ld_scales, p->eps, (int32_t)p->cols, 0, p->weight_type};
  switch (type) {
  case CUDA_R_16BF: return launch_rms<ElemBF16>(r, (hipStream_t)stream);
  case CUDA_R_16F: return launch_rms<ElemF16>(r, (hipStream_t)stream);
  default: return launch_rms<ElemF32>(r, (hipStream_t)stream);
  }
}

extern "C" uint32_t zluda_ffn_rms_backward_workspace(const zluda_ffn_rms_grad *p, size_t *bytes) {
  if (!p || !bytes || !p->cols) return CUBLAS_STATUS_INVALID_VALUE;
  if (p->cols > ZLUDA_FFN_NORM_MAX_COLS) return CUBLAS_STATUS_NOT_SUPPORTED;
  const uint32_t groups = p->rows ? rms_grad_groups(p->rows, p->cols) : 1;
  *bytes = p->dweight && groups > 1 ? (size_t)groups * p->cols * 4 : 0;  // (a single workgroup has the sums themselves)
  return CUBLAS_STATUS_SUCCESS;
}

extern "C" uint32_t zluda_ffn_rms_backward(const zluda_ffn_rms_grad *p, void *workspace, size_t workspace_size, void *stream) {
  if (!p) return CUBLAS_STATUS_INVALID_VALUE;
  const uint32_t type = p->dy.type;
  FFN_CHECK(check_rms(p->rows, p->cols, type, p->weight_type));
  FFN_CHECK(check_plain(p->h, p->rows, p->cols, type));
  FFN_CHECK(check_plain(p->dy, p->rows, p->cols, type));
  if (p->add.data) FFN_CHECK(check_plain(p->add, p->rows, p->cols, type));
  if (p->dx.data) FFN_CHECK(check_plain(p->dx, p->rows, p->cols, type));
  if (p->rows && ((!p->dx.data && !p->dweight) || !p->rstd)) return CUBLAS_STATUS_INVALID_VALUE;
  FFN_CHECK(check_vector(p->weight, p->weight_type));
  FFN_CHECK(check_vector(p->dweight, p->weight_type));
  FFN_CHECK(check_vector(p->rstd, CUDA_R_32F));
  size_t need = 0;
  FFN_CHECK(zluda_ffn_rms_backward_workspace(p, &need));
  if (need > workspace_size || (need && !workspace)) return CUBLAS_STATUS_ALLOC_FAILED;
  if (need && ((uintptr_t)workspace & 15)) return CUBLAS_STATUS_INVALID_VALUE;
  if (!zluda_gemm_device_cu_count()) return CUBLAS_STATUS_NOT_INITIALIZED;
  const hipStream_t s = (hipStream_t)stream;
  if (!p->rows) {  // a sum of no terms
    if (!p->dweight) return CUBLAS_STATUS_SUCCESS;
    const ZeroParams z{p->dweight, 1, (int64_t)(p->cols * elem_size(p->weight_type)), 0};
    return launch_kernel(zero_rows_kernel, dim3((uint32_t)((p->cols + 255) / 256)), dim3(256), s, z);
  }
  const uint32_t groups = rms_grad_groups(p->rows, p->cols);
  const RmsGradParams r{p->h.data, p->dy.data, p->add.data, p->dx.data, p->weight, p->rstd, p->dweight && groups > 1 ? (float *)workspace : nullptr,
                        groups > 1 ? nullptr : p->dweight, (int64_t)p->rows, p->h.ld, p->dy.ld, p->add.ld, p->dx.ld, (int32_t)p->cols, p->weight_type};
  FFN_CHECK(type == CUDA_R_16BF  ? launch_rms_grad<ElemBF16>(r, groups, s)
            : type == CUDA_R_16F ? launch_rms_grad<ElemF16>(r, groups, s)
                                 : launch_rms_grad<ElemF32>(r, groups, s));
  if (!p->dweight || groups == 1) return CUBLAS_STATUS_SUCCESS;
  const NormFinishParams f{r.part, p->dweight, nullptr, (int32_t)groups, (int32_t)p->cols, p->weight_type};
  return launch_kernel(norm_finish_kernel<16, 64>, dim3((uint32_t)((p->cols + 15) / 16), 1), dim3(1024), s, f);
}

extern "C" uint32_t zluda_ffn_activate(const zluda_ffn_activation *p, void *stream) {
  if (!p || p->activation > ZLUDA_FFN_COPY || !p->cols || (p->block_rows != 1 && p->block_rows != kPack) || (p->activation == ZLUDA_FFN_COPY && p->up.data))
    return CUBLAS_STATUS_INVALID_VALUE;
  const uint32_t type = p->gate.type;
  if (!plain_type(type) || p->cols > kMaxSide || p->rows > (uint64_t)INT64_MAX / 2) return CUBLAS_STATUS_NOT_SUPPORTED;
  FFN_CHECK(check_plain(p->gate, p->rows, p->cols, type));
  if (p->up.data) FFN_CHECK(check_plain(p->up, p->rows, p->cols, type));
  if (p->y.data) FFN_CHECK(check_plain(p->y, p->rows, p->cols, type));
  if (p->packed.data) FFN_CHECK(check_packed(p->packed, p->rows, p->cols, p->block_rows));
  if (p->rows && !p->y.data && !p->packed.data) return CUBLAS_STATUS_INVALID_VALUE;
  if (!p->rows) return CUBLAS_STATUS_SUCCESS;
  if (!zluda_gemm_device_cu_count()) return CUBLAS_STATUS_NOT_INITIALIZED;
  const ActivateParams a{p->gate.data, p->up.data, p->y.data, (uint8_t *)p->packed.data, (float *)p->packed.scales, (int64_t)p->rows, p->gate.ld, p->up.ld, p->y.ld,
                         p->packed.ld, p->packed.ld_scales, (int32_t)p->cols, p->activation};
  switch (type) {
  case CUDA_R_16BF: return launch_activate<ElemBF16>(a, p->block_rows, (hipStream_t)stream);
  case CUDA_R_16F: return launch_activate<ElemF16>(a, p->block_rows, (hipStream_t)stream);
  default: return launch_activate<ElemF32>(a, p->block_rows, (hipStream_t)stream);
  }
}

extern "C" uint32_t zluda_ffn_unpack(uint64_t rows, uint64_t cols, uint32_t block_rows, const zluda_ffn_matrix *packed, const zluda_ffn_matrix *y, void *stream) {
  if (!packed || !y || !cols || (block_rows != 1 && block_rows != kPack)) return CUBLAS_STATUS_INVALID_VALUE;
  if (cols > kMaxSide || rows > (uint64_t)INT64_MAX / 2 || !plain_type(y->type)) return CUBLAS_STATUS_NOT_SUPPORTED;
  FFN_CHECK(check_packed(*packed, rows, cols, block_rows));
  FFN_CHECK(check_plain(*y, rows, cols, y->type));
  if (!rows) return CUBLAS_STATUS_SUCCESS;
  if (!zluda_gemm_device_cu_count()) return CUBLAS_STATUS_NOT_INITIALIZED;
  const UnpackParams u{(const uint8_t *)packed->data, (const float *)packed->scales, y->data, (int64_t)rows, packed->ld, packed->ld_scales, y->ld, (int32_t)cols, block_rows != 1};
  const dim3 grid(column_strips(cols), (uint32_t)std::min<uint64_t>((rows + 3) / 4, kGridY));
  switch (y->type) {
  case CUDA_R_16BF: return launch_kernel(unpack_kernel<ElemBF16>, grid, dim3(256), (hipStream_t)stream, u);
  case CUDA_R_16F: return launch_kernel(unpack_kernel<ElemF16>, grid, dim3(256), (hipStream_t)stream, u);
  default: return launch_kernel(unpack_kernel<ElemF32>, grid, dim3(256), (hipStream_t)stream, u);
  }
}
