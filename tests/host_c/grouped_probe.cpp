// The tile that a product by expert takes, for tests: built as a shared library of its own (the rule needs no device).
#include "../../zluda_amd/csrc/ffn_grouped_choice.hpp"

extern "C" __attribute__((visibility("default"))) int probe_grouped_tile(const zluda_ffn_grouped *p, uint64_t cus) { return zluda_amd::grouped_tile(p, cus); }
extern "C" __attribute__((visibility("default"))) int probe_grouped_tiles() { return zluda_amd::kBlockTileCount; }
