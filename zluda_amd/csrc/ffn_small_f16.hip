// Gated feed-forward products of f16 operands: tiles, any alignment.
#include "ffn_small_launch.hpp"
namespace zluda_amd {
uint32_t launch_gated_small_f16(const GatedParams &p, int tile, hipStream_t s) { return launch_gated_small<ElemF16>(p, tile, s); }
} // namespace zluda_amd
