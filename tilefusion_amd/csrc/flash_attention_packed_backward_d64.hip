// Gradients of attention over packed sequences: the instances for head dimension 64.
#include "flash_attention_packed_backward.hpp"

int tfk::run_attention_packed_backward_d64(const PackedGradCall& c) { return run_grad<64>(c); }
