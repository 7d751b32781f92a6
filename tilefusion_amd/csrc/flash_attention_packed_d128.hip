// Attention over packed sequences: the instances for head dimension 128.
#include "flash_attention_packed_kernel.hpp"

int tfk::run_attention_packed_d128(const PackedCall& c) { return run_packed<128>(c); }
