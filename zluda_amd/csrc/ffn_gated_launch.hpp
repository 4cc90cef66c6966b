// Chooses the kernel of a gated feed-forward call.
#pragma once
#include "ffn_launch.hpp"
#include "kernels/ffn_gated_any.hpp"

namespace zluda_amd {

template <class E>
inline uint32_t launch_gated(const GatedParams &p, hipStream_t s) {
  const dim3 grid((p.features + 31) / 32, (p.tokens + 63) / 64);
  return launch_kernel(gated_any_kernel<E>, grid, dim3(256), s, p);
}

} // namespace zluda_amd
