// The gradients of products grouped by expert.
#include "ffn_grouped_launch.hpp"
namespace zluda_amd {
template <class E>
static uint32_t launch_grad(const GroupedGradParams &p, int side, uint32_t groups, hipStream_t s) {
  return side == 256 ? launch_kernel(grouped_grad_kernel<E, 256>, dim3(groups), dim3(512), s, p) : launch_kernel(grouped_grad_kernel<E, 128>, dim3(groups), dim3(256), s, p);
}
uint32_t launch_grouped_round(const RoundParams &r, uint32_t type, const int32_t *offsets, int32_t experts, dim3 grid, hipStream_t s) {
  return type == CUDA_R_16BF ? launch_kernel(grouped_round_kernel<ElemBF16>, grid, dim3(256), s, r, offsets, experts)
                             : launch_kernel(grouped_round_kernel<ElemF16>, grid, dim3(256), s, r, offsets, experts);
}
uint32_t launch_grouped_grad(const GroupedGradParams &p, uint32_t type, int side, uint32_t groups, hipStream_t s) {
  return type == CUDA_R_16BF ? launch_grad<ElemBF16>(p, side, groups, s) : launch_grad<ElemF16>(p, side, groups, s);
}
} // namespace zluda_amd
