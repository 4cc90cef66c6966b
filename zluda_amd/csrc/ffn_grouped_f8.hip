// Products of packed operands grouped by expert.
#include "ffn_grouped_launch.hpp"
namespace zluda_amd {
uint32_t launch_grouped_f8(const GroupedParams &p, int tile, hipStream_t s) {
  switch (p.d_type) {
  case CUDA_R_16BF: return launch_grouped<KIND_F8, 0>(p, tile, s);
  case CUDA_R_16F: return launch_grouped<KIND_F8, 1>(p, tile, s);
  default: return launch_grouped<KIND_F8_WIDE, 2>(p, tile, s);
  }
}
} // namespace zluda_amd
