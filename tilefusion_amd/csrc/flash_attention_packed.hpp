// Attention over packed sequences: what the C entry points (flash_attention_packed.hip) and the kernels' source files share.
#pragma once

#include "packed_sequences.hpp"

namespace tfk {

struct PackedCall {
  const void *query, *key, *value;
  void* out;
  PackedArgs args;
  float scale_log2;
  bool bf16, causal;
  int rows;   // per workgroup: 256, 128 or 64
  hipStream_t stream;
};
int run_attention_packed_d64(const PackedCall& c);
int run_attention_packed_d128(const PackedCall& c);

struct PackedGradCall {
  const void *query, *key, *value, *out, *grad_out;
  const float* lse;
  void *grad_query, *grad_key, *grad_value;   // grad_query, or grad_key and grad_value, may be null
  void* stats;     // room for 16 bytes a row
  void* partial;   // parts > 1: room for parts times dK and dV in fp32
  int parts;       // that the rows behind a tile of keys are cut into
  PackedArgs args;
  float scale;
  bool bf16, causal;
  hipStream_t stream;
};
constexpr int kGradKeys = 128;   // keys of a workgroup that makes dK and dV
int run_attention_packed_backward_d64(const PackedGradCall& c);
int run_attention_packed_backward_d128(const PackedGradCall& c);

// Tiles of `rows` that sequences of `all` rows together can make.
inline int64_t most_tiles(int64_t all, int64_t sequences, int64_t rows) { return (all + sequences * (rows - 1)) / rows; }

}  // namespace tfk
