// Argument checks that the feed-forward entry points share (include/zluda_ffn.h).
#pragma once
#include <algorithm>
#include <cstring>

#include "../../include/zluda_ffn.h"
#include "../../include/zluda_gemm_launch.h"
#include "ffn_launch.hpp"
#include "launch_util.hpp"

namespace zluda_amd {

constexpr int kGridY = 65535;

inline bool is_h16(uint32_t type) { return type == CUDA_R_16F || type == CUDA_R_16BF; }
inline uint64_t elem_size(uint32_t type) { return type == CUDA_R_32F ? 4 : type == CUDA_R_8F_E4M3 ? 1 : 2; }
inline int cus() {
  const int n = (int)zluda_gemm_device_cu_count();
  return n ? n : 256;
}

#define FFN_CHECK(expr)                            \
  do {                                             \
    const uint32_t st_ = (expr);                   \
    if (st_ != CUBLAS_STATUS_SUCCESS) return st_;  \
  } while (0)

inline uint32_t check_vector(const void *v, uint32_t type) { return ((uintptr_t)v & (elem_size(type) - 1)) ? CUBLAS_STATUS_INVALID_VALUE : CUBLAS_STATUS_SUCCESS; }
// a matrix of plain elements that has to be there
inline uint32_t check_plain(const zluda_ffn_matrix &m, uint64_t rows, uint64_t cols, uint32_t type) {
  if (!m.data && rows) return CUBLAS_STATUS_INVALID_VALUE;
  if (m.type != type) return CUBLAS_STATUS_NOT_SUPPORTED;
  return m.ld < (int64_t)cols || ((uintptr_t)m.data & (elem_size(type) - 1)) ? CUBLAS_STATUS_INVALID_VALUE : CUBLAS_STATUS_SUCCESS;
}

} // namespace zluda_amd
