// Gated feed-forward products of f16 operands on the four-wave persistent kernel, and the choice between it and the others.
#include "ffn_gated_launch.hpp"
namespace zluda_amd {
uint32_t launch_gated_f16(const GatedParams &p, hipStream_t s) { return launch_gated<ElemF16>(p, s); }
} // namespace zluda_amd
