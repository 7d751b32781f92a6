// Attention over packed sequences: the C entry points, and which instance of the kernels a call runs.
#include <algorithm>

#include "flash_attention.hpp"
#include "flash_attention_packed.hpp"

namespace tfk {
namespace {

int check_packed(const char* who, const tf_packed_attention_t* p) {
  TFK_REQUIRE(p, TF_ERR_INVALID_ARG, "%s: null pointer", who);
  TFK_REQUIRE(p->dtype == TF_DTYPE_F16 || p->dtype == TF_DTYPE_BF16, TF_ERR_UNSUPPORTED, "%s: dtype must be TF_DTYPE_F16 or TF_DTYPE_BF16", who);
  TFK_REQUIRE(p->D == 64 || p->D == 128, TF_ERR_UNSUPPORTED, "%s: head dim must be 64 or 128 (got %lld)", who, (long long)p->D);
  TFK_REQUIRE(p->tokens >= 0 && p->kv_tokens >= 0 && p->tokens < (1 << 24) && p->kv_tokens < (1 << 24) && p->sequences >= 0 && p->sequences <= 65536,
              TF_ERR_INVALID_ARG, "%s: tokens and kv_tokens must be below 2^24, sequences at most 65536", who);
  TFK_REQUIRE(p->heads > 0 && p->heads <= 1024 && p->kv_heads > 0 && p->heads % p->kv_heads == 0, TF_ERR_INVALID_ARG,
              "%s: heads must be a multiple of kv_heads, at most 1024 (got %lld and %lld)", who, (long long)p->heads, (long long)p->kv_heads);
  TFK_REQUIRE(std::max(p->tokens, p->kv_tokens) * (p->heads / p->kv_heads) < (1ll << 30), TF_ERR_INVALID_ARG,
              "%s: tokens times the heads of a group must be below 2^30", who);
  TFK_REQUIRE(is_softmax_scale(p->softmax_scale), TF_ERR_INVALID_ARG, "%s: softmax_scale must be finite, times log2(e) in fp32 too", who);
  if (p->tokens == 0 && p->kv_tokens == 0) return TF_OK;
  TFK_REQUIRE(p->offsets && (p->query || p->tokens == 0) && ((p->key && p->value) || p->kv_tokens == 0), TF_ERR_INVALID_ARG, "%s: null pointer", who);
  TFK_REQUIRE(p->kv_offsets || p->tokens == p->kv_tokens, TF_ERR_INVALID_ARG, "%s: keys of another number than queries need kv_offsets", who);
  // A tile of up to 64 tokens is addressed in 32 bits from its first one, and its head in 64.
  const int64_t* strides[] = {p->query_strides, p->key_strides, p->value_strides};
  for (const int64_t* s : strides)
    TFK_REQUIRE(s[0] >= 0 && s[0] % 8 == 0 && s[0] < (1 << 24) && s[1] >= 0 && s[1] % 8 == 0 && s[1] < (1ll << 40), TF_ERR_INVALID_ARG,
                "%s: strides must be multiples of 8 elements, from token to token below 2^24 and from head to head below 2^40", who);
  // (the backward pass addresses a tile of 32 rows, whose tokens are 33 at most, in 32 bits from the first one's; one head alone is no step further)
  const int64_t group = p->heads / p->kv_heads;
  TFK_REQUIRE(33 * p->query_strides[0] + (group > 1 ? group * p->query_strides[1] : 0) < (1ll << 31) - p->D, TF_ERR_INVALID_ARG,
              "%s: the heads of a group must lie within 2^31 elements", who);
  TFK_REQUIRE(((reinterpret_cast<uintptr_t>(p->query) | reinterpret_cast<uintptr_t>(p->key) | reinterpret_cast<uintptr_t>(p->value)) & 15) == 0,
              TF_ERR_INVALID_ARG, "%s: operands must begin at 16-byte boundaries", who);
  return TF_OK;
}
PackedArgs packed_args(const tf_packed_attention_t& p) {
  const int64_t group = p.heads / p.kv_heads;
  return {p.offsets, p.kv_offsets ? p.kv_offsets : p.offsets, (int)p.sequences, (int)p.tokens, (int)p.kv_tokens, (int)p.heads, (int)p.kv_heads,
          make_divider((unsigned)group), (int)p.query_strides[0], (int)p.key_strides[0], (int)p.value_strides[0],
          group > 1 ? (int)p.query_strides[1] : 0, group * p.query_strides[1], p.key_strides[1], p.value_strides[1], nullptr};
}

// Rows per workgroup, from the sequences' mean length, which is all that the host knows of them.  A tile of 64 keys takes 1.45 us with 256 rows, 1.0 with
// 128 and 0.77 with 64 (D = 128), and a CU has room for one workgroup (two with 64 rows and D = 64): the largest for which the next smaller
// one would go round more than once, or whose rows sequences fill.  us with 256 / 128 / 64 rows, 32 heads x 128: 858 tokens behind 6000 keys 144 / 102 / 147, 512
// of them 148 / 102 / 79; 60 texts of 20 to 400 in groups of 4 heads 70 / 86 / 121; 37 of 1 to 300, 16/4 heads x 64: 12.1 / 9.8 / 10.9.
int packed_rows(int64_t tokens, int64_t sequences, int64_t heads, int64_t kv_heads, int64_t D) {
  const int64_t mean = sequences > 0 ? tokens / sequences * (heads / kv_heads) : 0;
  const auto tiles = [&](int64_t rows) { return tokens * heads / rows + sequences / 2 * kv_heads; };
  if (tiles(128) > kCUs && mean >= 256) return 256;
  if (tiles(64) > (D == 64 ? 2 : 1) * kCUs && mean >= 64) return 128;
  return 64;
}

// Parts that the rows behind a tile of keys are cut into: where there are fewer tiles than the chip runs workgroups at a time (512), and rows enough.
// 11 texts of 30 to 1001 tokens, 16/4 heads x 64: 156 us in one part, 102 in 2, 70 in 4, 85 in 8; 4 of 1500: 154 in 2, 174 in 4 or 5.
int grad_parts(const tf_packed_attention_t& p) {
  const int64_t tiles = std::max<int64_t>(1, (p.kv_tokens / kGradKeys + p.sequences / 2) * p.kv_heads);
  const int64_t rows = p.sequences > 0 ? p.tokens / p.sequences * (p.heads / p.kv_heads) : 0;
  return (int)std::max<int64_t>(1, std::min<int64_t>({512 / tiles, rows / 256, 8}));
}
size_t stats_bytes(const tf_packed_attention_t& p) { return ((size_t)p.tokens * (size_t)p.heads * 16 + 255) / 256 * 256; }

}  // namespace
}  // namespace tfk

extern "C" int tf_flash_attention_packed(const tf_packed_attention_t* p, void* out, float* lse, void* stream) {
  using namespace tfk;
  constexpr const char* who = "tf_flash_attention_packed";
  if (int rc = check_packed(who, p)) return rc;
  if (p->tokens == 0) return TF_OK;
  TFK_REQUIRE(out && (reinterpret_cast<uintptr_t>(out) & 15) == 0, TF_ERR_INVALID_ARG, "%s: out must begin at a 16-byte boundary", who);
  PackedCall c = {p->query, p->key, p->value, out, packed_args(*p), (float)(p->softmax_scale * 1.4426950408889634), p->dtype == TF_DTYPE_BF16,
                  p->causal != 0, packed_rows(p->tokens, p->sequences, p->heads, p->kv_heads, p->D), static_cast<hipStream_t>(stream)};
  c.args.lse = lse;
  return p->D == 128 ? run_attention_packed_d128(c) : run_attention_packed_d64(c);
}

extern "C" size_t tf_flash_attention_packed_backward_workspace_bytes(const tf_packed_attention_t* p) {
  using namespace tfk;
  if (!p || p->tokens < 0 || p->kv_tokens < 0 || p->sequences < 0 || p->kv_heads <= 0 || p->heads < p->kv_heads || p->D <= 0) return 0;
  const int parts = grad_parts(*p);
  return stats_bytes(*p) + (parts > 1 ? (size_t)parts * 2 * (size_t)p->kv_tokens * (size_t)p->kv_heads * (size_t)p->D * sizeof(float) : 0);
}

extern "C" int tf_flash_attention_packed_backward(const tf_packed_attention_t* p, const void* grad_out, const void* out, const float* lse,
                                                  void* grad_query, void* grad_key, void* grad_value, void* workspace, size_t workspace_bytes,
                                                  void* stream) {
  using namespace tfk;
  constexpr const char* who = "tf_flash_attention_packed_backward";
  if (int rc = check_packed(who, p)) return rc;
  TFK_REQUIRE((grad_key == nullptr) == (grad_value == nullptr) || p->kv_tokens == 0, TF_ERR_INVALID_ARG, "%s: grad_key and grad_value are both asked for or neither", who);
  if (p->tokens == 0 && p->kv_tokens == 0) return TF_OK;
  TFK_REQUIRE((grad_out && out && lse) || p->tokens == 0, TF_ERR_INVALID_ARG, "%s: null pointer", who);
  TFK_REQUIRE(((reinterpret_cast<uintptr_t>(grad_out) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(grad_query) |
                reinterpret_cast<uintptr_t>(grad_key) | reinterpret_cast<uintptr_t>(grad_value) | reinterpret_cast<uintptr_t>(workspace)) & 15) == 0,
              TF_ERR_INVALID_ARG, "%s: operands must begin at 16-byte boundaries", who);
  const size_t need = tf_flash_attention_packed_backward_workspace_bytes(p);
  TFK_REQUIRE((workspace && workspace_bytes >= need) || need == 0, TF_ERR_INVALID_ARG, "%s: workspace holds %zu bytes, %zu needed", who, workspace_bytes, need);
  const PackedGradCall c = {p->query, p->key, p->value, out, grad_out, lse, grad_query, grad_key, grad_value, workspace,
                            static_cast<char*>(workspace) + stats_bytes(*p), grad_parts(*p), packed_args(*p),
                            (float)p->softmax_scale, p->dtype == TF_DTYPE_BF16, p->causal != 0, static_cast<hipStream_t>(stream)};
  return p->D == 128 ? run_attention_packed_backward_d128(c) : run_attention_packed_backward_d64(c);
}

extern "C" int tf_flash_attention_packed_rows(int64_t tokens, int64_t sequences, int64_t heads, int64_t kv_heads, int64_t D) {
  if (tokens < 0 || sequences < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || (D != 64 && D != 128)) return 0;
  return tfk::packed_rows(tokens, sequences, heads, kv_heads, D);
}
