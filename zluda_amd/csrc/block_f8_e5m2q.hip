// Products with a scale for each 128 of K: formats of P and Q (0 E4M3, 1 E5M2) 0 and 1.
#include "block_launch.hpp"
namespace zluda_amd {
uint32_t launch_block_f8_e5m2q(const MfmaParams &prm, const zluda_gemm_plan &plan, bool uniform, bool exact, hipStream_t s) { return launch_block_variant<0, 1>(prm, plan, uniform, exact, s); }
} // namespace zluda_amd
