// Products of f16 operands grouped by expert.
#include "ffn_grouped_launch.hpp"
namespace zluda_amd {
uint32_t launch_grouped_f16(const GroupedParams &p, int tile, hipStream_t s) { return launch_grouped<KIND_F16, 1>(p, tile, s); }
} // namespace zluda_amd
