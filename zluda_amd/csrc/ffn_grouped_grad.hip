// The gradients of products grouped by expert.
#include "ffn_grouped_launch.hpp"
namespace zluda_amd {
uint32_t launch_grouped_grad(const GroupedGradParams &p, uint32_t type, uint32_t groups, hipStream_t s) {
  return type == CUDA_R_16BF ? launch_kernel(grouped_grad_kernel<ElemBF16>, dim3(groups), dim3(256), s, p) : launch_kernel(grouped_grad_kernel<ElemF16>, dim3(groups), dim3(256), s, p);
}
} // namespace zluda_amd
