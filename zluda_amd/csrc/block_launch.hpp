// Launchers of the products with a scale for each 128 of K; one translation unit per pair of formats.
#pragma once
#include "block_cost.hpp"
#include "kernels/block_decode.hpp"
#include "kernels/block_gemm.hpp"
#include "launch_util.hpp"
#include "planner.hpp"

namespace zluda_amd {

// plan.variant indexes kBlockVariants (planner.hpp); uniform: all P rows of a wave share their scales; exact: results in 32 bits
template <int FP, int FQ>
inline uint32_t launch_block_variant(const MfmaParams &prm, const zluda_gemm_plan &plan, bool uniform, bool exact, hipStream_t s) {
  const dim3 grid(plan.grid_x, plan.grid_y, plan.grid_z > 1 ? plan.grid_z : 1);  // z: split-K shares
  auto launch = [&](auto v_c, auto uniform_c, auto exact_c) -> uint32_t {
    constexpr BlockVariant v = kBlockVariants[decltype(v_c)::value];
    constexpr bool U = decltype(uniform_c)::value, X = decltype(exact_c)::value;
    if constexpr ((X && !v.exact) || (!U && v.uniform)) return CUBLAS_STATUS_INVALID_VALUE;
    else if constexpr (decltype(v_c)::value == kBlockDecode)
      return launch_kernel(block_decode_kernel<FP, FQ, U, X>, grid, dim3(512), s, prm);
    else return launch_kernel(block_gemm_kernel<FP, FQ, U, X, v.bp, v.bq, v.wp, v.wq, v.stages>, grid, dim3(v.wp * v.wq * 64), s, prm);
  };
  auto with = [&](auto v_c) -> uint32_t {
    using T = std::true_type;
    using F = std::false_type;
    return uniform ? (exact ? launch(v_c, T{}, T{}) : launch(v_c, T{}, F{})) : exact ? launch(v_c, F{}, T{}) : launch(v_c, F{}, F{});
  };
  switch (plan.variant) {
  case 0: return with(std::integral_constant<int, 0>{});
  case 1: return with(std::integral_constant<int, 1>{});
  case 2: return with(std::integral_constant<int, 2>{});
  case 3: return with(std::integral_constant<int, 3>{});
  case 4: return with(std::integral_constant<int, 4>{});
  case 5: return with(std::integral_constant<int, 5>{});
  case 6: return with(std::integral_constant<int, 6>{});
  case kBlockDecode: return with(std::integral_constant<int, kBlockDecode>{});
  }
  static_assert(kNumBlockVariants == 8, "a case each");
  return CUBLAS_STATUS_INVALID_VALUE;
}

} // namespace zluda_amd
