// Attention over packed sequences: the instances for head dimension 64.
#include "flash_attention_packed_kernel.hpp"

int tfk::run_attention_packed_d64(const PackedCall& c) { return run_packed<64>(c); }
