// New tokens enter a paged cache: queries and keys are rotated by their positions, keys and values go to their pages.
//
// No counterpart in the reference.  A pair (a, b) of a head's first `rotated` elements becomes (a cos - b sin, a sin + b cos) with the
// angle of the token's position and the pair's number; a pair is either two neighbours or elements i and i + rotated / 2.  In fp32, rounded once.
//
// Every byte is read and written once, with nothing to share but a token's row of cos and sin: bound by HBM for prompts and by a chain of
// dependent loads (sequence, length, page and angles, store) for a step of a few tokens.
// 9 prompts of 77 to 2999, 32/8 heads x 128, fp16: 39 us, 5.2 TB/s (one row a thread 45, two 42, three 39, four 39); a token each of 64: 3.7 us one after
// another in a graph, of which a token alone takes 3.4; 4.4 from the kernel's first to its last signal.
#include <algorithm>
#include <iterator>
#include <limits>
#include <utility>

#include "paged_cache.hpp"

namespace tfk {
namespace {

constexpr int kThreads = 256;

struct AppendArgs {
  const void *query, *key, *value;
  int64_t query_token, query_head, key_token, key_head, value_token, value_head;   // strides in elements
  const float *cos, *sin;   // [positions][half]
  int64_t positions;
  int half;
  const int *offsets, *lengths;   // no offsets: token b is the one new token of sequence b
  int sequences, heads, kv_heads;
  PageTable table;
  void *key_cache, *value_cache;
  int64_t key_cache_strides[3], value_cache_strides[3];   // page, token, head
  void *query_out, *key_out;   // [tokens][heads][D]; no key_out: the rotated keys are in the cache only
};

// What becomes of a token: kKept has a place in the cache, kLost should have one and has none (its rotated rows are NaN), kNone
// belongs to no sequence, or its sequence is not as long as its new tokens (zeros).
enum TokenState { kKept, kLost, kNone };

// One workgroup per token and kRows head rows of it (queries, then keys, then values); a thread takes 8 elements of
// every kThreads / (D / 8)-th row, so that one set of angles serves all of its rows.
// kVector: `half` and the tables' beginning let the angles, and the partner of eight elements, be loaded in 16-byte pieces.
template <typename T, int D, bool kNeighbours, bool kVector, int kUnroll>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a) {
  using V8 = T __attribute__((ext_vector_type(8)));
  constexpr int kVecs = D / 8, kRowsPerPass = kThreads / kVecs, kRows = kRowsPerPass * kUnroll;
  const int t = blockIdx.x, vec = threadIdx.x % kVecs, rows = a.heads + 2 * a.kv_heads;
  const int row0 = blockIdx.y * kRows + threadIdx.x / kVecs;

  // ---- the rows themselves, in flight while the token's place is found ------------------------
  V8 x[kUnroll], partner[kUnroll];
  const int half = a.half, first = 8 * vec;
  // (kVector, halves: all eight are in the first half, the second half or behind the rotated part)
  const int partner_at = first < half ? first + half : first - half;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int row = row0 + u * kRowsPerPass;
    if (row >= rows) break;
    const T* src;
    if (row < a.heads) src = static_cast<const T*>(a.query) + t * a.query_token + row * a.query_head;
    else if (row < a.heads + a.kv_heads) src = static_cast<const T*>(a.key) + t * a.key_token + (row - a.heads) * a.key_head;
    else src = static_cast<const T*>(a.value) + t * a.value_token + (row - a.heads - a.kv_heads) * a.value_head;
    x[u] = *reinterpret_cast<const V8*>(src + first);
    if (!kNeighbours && row < a.heads + a.kv_heads && first < 2 * half) {
      if constexpr (kVector) {
        partner[u] = *reinterpret_cast<const V8*>(src + partner_at);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int e = first + i;
          partner[u][i] = e < half ? src[e + half] : e < 2 * half ? src[e - half] : (T)0.f;
        }
      }
    }
  }

  // ---- the token's place -----------------------------------------------------------------------
  TokenState state = kNone;
  int64_t position = -1;
  int page = -1;
  const int b = a.offsets ? __builtin_amdgcn_readfirstlane(find_sequence(a.offsets, a.sequences, t)) : t;
  if (b >= 0 && b < a.sequences) {
    const int64_t after = a.offsets ? (int64_t)read_uniform(a.offsets + b + 1) - t : 1;   // new tokens from this one on
    const int64_t before = a.offsets ? (int64_t)t - read_uniform(a.offsets + b) : 0;
    position = (int64_t)read_uniform(a.lengths + b) - after;
    if (position >= before) {
      page = page_of(a.table, b, position);
      state = page >= 0 && position < a.positions ? kKept : kLost;
    }
  }

  float c[8], s[8];   // of this thread's elements, the sines signed for element and partner
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    c[i] = 1.f;
    s[i] = 0.f;
  }
  if (state == kKept && first < 2 * half) {
    const float *cos = a.cos + position * half, *sin = a.sin + position * half;
    if constexpr (kVector) {
      constexpr int kAngles = kNeighbours ? 4 : 8;
      const int at = kNeighbours ? first / 2 : first < half ? first : first - half;
      float ca[kAngles], sa[kAngles];
#pragma unroll
      for (int i = 0; i < kAngles; i += 4) {
        const float4_t c4 = *reinterpret_cast<const float4_t*>(cos + at + i), s4 = *reinterpret_cast<const float4_t*>(sin + at + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          ca[i + j] = c4[j];
          sa[i + j] = s4[j];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        c[i] = ca[kNeighbours ? i / 2 : i];
        const float v = sa[kNeighbours ? i / 2 : i];
        s[i] = (kNeighbours ? i % 2 == 0 : first < half) ? -v : v;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = first + i;
        if (e >= 2 * half) break;
        const int at = kNeighbours ? e / 2 : e < half ? e : e - half;
        c[i] = cos[at];
        s[i] = (kNeighbours ? e % 2 == 0 : e < half) ? -sin[at] : sin[at];
      }
    }
  }

  const int in_page = state == kKept ? (int)position - divide(a.table.page, (int)position) * (int)a.table.page.d : 0;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int row = row0 + u * kRowsPerPass;
    if (row >= rows) break;
    if (row >= a.heads + a.kv_heads) {
      if (state == kKept) {
        const int64_t* st = a.value_cache_strides;
        T* to = static_cast<T*>(a.value_cache) + page * st[0] + in_page * st[1] + (row - a.heads - a.kv_heads) * st[2];
        *reinterpret_cast<V8*>(to + first) = x[u];
      }
      continue;
    }
    V8 y = x[u];
    if (state != kKept) {
      const float v = state == kLost ? std::numeric_limits<float>::quiet_NaN() : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = (T)v;
    } else if (first < 2 * half) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (!kVector && first + i >= 2 * half) break;   // (1 * x + 0 * x would lose an infinity)
        y[i] = (T)(c[i] * (float)x[u][i] + s[i] * (float)(kNeighbours ? x[u][i ^ 1] : partner[u][i]));
      }
    }
    if (row < a.heads) {
      *reinterpret_cast<V8*>(static_cast<T*>(a.query_out) + ((int64_t)t * a.heads + row) * D + first) = y;
      continue;
    }
    const int head = row - a.heads;
    if (a.key_out) *reinterpret_cast<V8*>(static_cast<T*>(a.key_out) + ((int64_t)t * a.kv_heads + head) * D + first) = y;
    if (state == kKept) {
      const int64_t* st = a.key_cache_strides;
      *reinterpret_cast<V8*>(static_cast<T*>(a.key_cache) + page * st[0] + in_page * st[1] + head * st[2] + first) = y;
    }
  }
}

template <typename T, int D, bool kNeighbours, bool kVector>
int launch_append(const AppendArgs& a, int64_t tokens, hipStream_t st) {
  constexpr int kUnroll = 3, kRows = kThreads / (D / 8) * kUnroll;
  const int rows = a.heads + 2 * a.kv_heads;
  return launch_kernel(append_kernel<T, D, kNeighbours, kVector, kUnroll>, dim3((unsigned)tokens, (unsigned)((rows + kRows - 1) / kRows)),
                       dim3(kThreads), 0, st, a);
}
template <typename T, int D>
int launch_append(const AppendArgs& a, int64_t tokens, bool neighbours, hipStream_t st) {
  const bool at_16 = ((reinterpret_cast<uintptr_t>(a.cos) | reinterpret_cast<uintptr_t>(a.sin)) & 15) == 0;
  const bool vector = at_16 && a.half % (neighbours ? 4 : 8) == 0;
  if (neighbours) return vector ? launch_append<T, D, true, true>(a, tokens, st) : launch_append<T, D, true, false>(a, tokens, st);
  return vector ? launch_append<T, D, false, true>(a, tokens, st) : launch_append<T, D, false, false>(a, tokens, st);
}

// No row of a cache lies on another: every dimension's steps lead past all that those with smaller steps reach, as in whatever order and slice of a
// tensor (not every cache without overlaps is of this kind, but all that are made by turning and cutting are).
bool rows_apart(const tf_paged_cache_t& c, const int64_t (&strides)[3]) {
  std::pair<int64_t, int64_t> steps[] = {{strides[0], c.pages}, {strides[1], c.page_size}, {strides[2], c.kv_heads}};
  std::sort(std::begin(steps), std::end(steps));
  __int128 reach = c.D;
  for (const auto& [stride, count] : steps) {
    if (count == 1) continue;
    if (stride < reach) return false;
    reach += (__int128)stride * (count - 1);
  }
  return true;
}

}  // namespace

int check_paged_cache(const char* who, const tf_paged_cache_t* c) {
  TFK_REQUIRE(c && c->key && c->value && c->page_table && c->lengths, TF_ERR_INVALID_ARG, "%s: null pointer", who);
  TFK_REQUIRE(c->dtype == TF_DTYPE_F16 || c->dtype == TF_DTYPE_BF16, TF_ERR_UNSUPPORTED, "%s: dtype must be TF_DTYPE_F16 or TF_DTYPE_BF16", who);
  TFK_REQUIRE(c->D == 64 || c->D == 128, TF_ERR_UNSUPPORTED, "%s: head dim must be 64 or 128 (got %lld)", who, (long long)c->D);
  TFK_REQUIRE(c->pages > 0 && c->pages < (1ll << 31) && c->kv_heads > 0 && c->kv_heads <= 65536, TF_ERR_INVALID_ARG,
              "%s: pages and kv_heads must be positive and below 2^31 and 2^16 + 1", who);
  TFK_REQUIRE(c->page_size > 0 && c->page_size <= 65536, TF_ERR_INVALID_ARG, "%s: page_size must be 1 .. 65536 (got %lld)", who, (long long)c->page_size);
  TFK_REQUIRE(c->sequences >= 0 && c->sequences <= (1 << 20) && c->table_width >= 0 && c->table_width < (1ll << 31) && c->table_stride >= 0,
              TF_ERR_INVALID_ARG, "%s: at most 2^20 sequences, table_width below 2^31", who);
  for (int i = 0; i < 3; ++i)
    for (const int64_t stride : {c->key_strides[i], c->value_strides[i]})
      TFK_REQUIRE((stride == 0 || stride >= c->D) && stride % 8 == 0, TF_ERR_INVALID_ARG,
                  "%s: the cache's strides must be multiples of 8 elements and no less than a row, or zero where there is one", who);
  TFK_REQUIRE(((reinterpret_cast<uintptr_t>(c->key) | reinterpret_cast<uintptr_t>(c->value)) & 15) == 0, TF_ERR_INVALID_ARG,
              "%s: the cache must begin at a 16-byte boundary", who);
  return TF_OK;
}
PageTable page_table(const tf_paged_cache_t& c) {
  return {c.page_table, c.table_stride, (int)c.table_width, (int)c.pages, make_divider((unsigned)c.page_size)};
}

}  // namespace tfk

extern "C" int tf_append_paged_kv(const tf_paged_cache_t* cache, const void* query, const void* key, const void* value, const int64_t* strides,
                                  const float* cos, const float* sin, int64_t positions, int64_t rotated, int interleaved, const int32_t* offsets,
                                  int64_t tokens, int64_t heads, void* query_out, void* key_out, void* stream) {
  using namespace tfk;
  constexpr const char* who = "tf_append_paged_kv";
  if (int rc = check_paged_cache(who, cache)) return rc;
  TFK_REQUIRE(rows_apart(*cache, cache->key_strides) && rows_apart(*cache, cache->value_strides), TF_ERR_INVALID_ARG,
              "%s: rows of the cache lie on each other", who);
  TFK_REQUIRE(tokens >= 0 && tokens < (1 << 24) && heads > 0 && heads <= 65536, TF_ERR_INVALID_ARG, "%s: tokens below 2^24, heads 1 .. 65536", who);
  TFK_REQUIRE(rotated > 0 && rotated % 2 == 0 && rotated <= cache->D && positions >= 0, TF_ERR_INVALID_ARG,
              "%s: rotated must be even and at most the head dim (got %lld)", who, (long long)rotated);
  if (tokens == 0) return TF_OK;
  TFK_REQUIRE(query && key && value && strides && cos && sin && query_out, TF_ERR_INVALID_ARG, "%s: null pointer", who);
  for (int i = 0; i < 6; ++i)
    TFK_REQUIRE(strides[i] >= 0 && strides[i] % 8 == 0, TF_ERR_INVALID_ARG, "%s: strides must be multiples of 8 elements", who);
  TFK_REQUIRE(((reinterpret_cast<uintptr_t>(query) | reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value) |
                reinterpret_cast<uintptr_t>(query_out) | reinterpret_cast<uintptr_t>(key_out)) & 15) == 0,
              TF_ERR_INVALID_ARG, "%s: operands must begin at 16-byte boundaries", who);
  AppendArgs a = {query, key, value, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], cos, sin, positions, (int)(rotated / 2),
                  offsets, cache->lengths, (int)cache->sequences, (int)heads, (int)cache->kv_heads, page_table(*cache), cache->key, cache->value,
                  {}, {}, query_out, key_out};
  std::copy_n(cache->key_strides, 3, a.key_cache_strides);
  std::copy_n(cache->value_strides, 3, a.value_cache_strides);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const bool bf16 = cache->dtype == TF_DTYPE_BF16, neighbours = interleaved != 0;
  if (cache->D == 128) return bf16 ? launch_append<bf16_t, 128>(a, tokens, neighbours, st) : launch_append<half_t, 128>(a, tokens, neighbours, st);
  return bf16 ? launch_append<bf16_t, 64>(a, tokens, neighbours, st) : launch_append<half_t, 64>(a, tokens, neighbours, st);
}
