// Products of bf16 operands grouped by expert.
#include "ffn_grouped_launch.hpp"
namespace zluda_amd {
uint32_t launch_grouped_bf16(const GroupedParams &p, int tile, hipStream_t s) { return launch_grouped<KIND_BF16, 0>(p, tile, s); }
} // namespace zluda_amd
