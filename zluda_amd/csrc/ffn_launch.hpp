// Launchers of the gated feed-forward products, one translation unit per element type.
#pragma once
#include <hip/hip_runtime.h>

#include "kernels/ffn_gated_store.hpp"
#include "launch_util.hpp"

namespace zluda_amd {

uint32_t launch_gated_bf16(const GatedParams &p, hipStream_t s);
uint32_t launch_gated_f16(const GatedParams &p, hipStream_t s);

} // namespace zluda_amd
