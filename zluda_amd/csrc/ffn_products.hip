// The products of the gated layer's backward pass in one launch.
#include "kernels/ffn_grad_products.hpp"
namespace zluda_amd {
uint32_t launch_grad_products(uint32_t type, const GradProductsParams &p, hipStream_t s) {
  const dim3 grid(p.dx_groups + (uint32_t)(p.dw.tiles_p * p.dw.tiles_q) + (p.sums ? (uint32_t)(p.dw.nq + 63) / 64 : 0));
  return type == CUDA_R_16BF ? launch_kernel(grad_products_kernel<ElemBF16>, grid, dim3(256), s, p) : launch_kernel(grad_products_kernel<ElemF16>, grid, dim3(256), s, p);
}
} // namespace zluda_amd
