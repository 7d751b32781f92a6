// Sequences packed one behind the other, for attention: which rows of queries, and which keys, a workgroup takes.
//
// The query heads of a group read the same keys: they are rows of one problem, row r being head r % group of token r / group, so that a tile of rows
// spans few tokens (less of a causal tile is masked, short sequences fill theirs) and keys are fetched once for a group.
//
// Sequence b is tokens offsets[b] .. offsets[b + 1] - 1 of the queries and kv_offsets[b] .. of the keys.  The host does not know them: a launch has
// as many workgroups as there can be tiles, and each finds its own.  Offsets are in device memory and may hold anything; what they
// name beyond the tensors is cut off.
#pragma once

#include "common.hpp"
#include "paged_cache.hpp"

namespace tfk {

struct PackedArgs {
  const int *offsets, *kv_offsets;   // [sequences + 1]
  int sequences, tokens, kv_tokens, heads, kv_heads;
  Divider group;   // query heads that share a head of keys
  int query_row, key_row, value_row, query_head;   // strides in elements; query_head: from one to the next of the heads of a group
  int64_t query_group, key_head, value_head;       // ... from one head of keys to the next (that of a long text's head-major tensor is its tokens * D)
  float* lse;   // [heads][tokens], or null
};

struct PackedTile {
  int sequence;   // -1: none
  int from_end;   // tiles of the sequence behind it
  int q0, lq, k0, lkv;   // tokens and keys: the first, how many
};

// rows [begin, begin + length) of a sequence, within `rows`
struct PackedRange { int begin, length; };
__host__ __device__ inline PackedRange packed_range(int begin, int end, int rows) {
  const int b = begin < 0 ? 0 : begin < rows ? begin : rows, e = end < rows ? end : rows;
  return {b, e > b ? e - b : 0};   // (compared first: an end near -2^31 less b is a large number)
}

// A sequence's queries and keys, the tiles of `rows` rows (or keys) that it makes, and how far its last (first) one counts: see find_tile.
struct SequenceTiles {
  PackedRange q, k;
  int tiles, level;
};
template <bool kKeys>
__host__ __device__ inline SequenceTiles sequence_tiles(PackedRange q, PackedRange k, int group, int rows) {
  const auto tiles_of = [&](int n) { return (n + rows - 1) / rows; };
  return {q, k, kKeys ? tiles_of(k.length) : tiles_of(q.length * group), kKeys ? tiles_of(k.length) : tiles_of(k.length * group)};
}

// The `rank`-th of the tiles of `rows` rows that the sequences make, most keys first.  Tile e from a sequence's end ends
// e * rows rows in front of it and counts as ceil(lkv * group / rows) - e (causal or not: the longest sequences first, and their last
// tokens).  The largest number that more tiles reach than come before this one is found by halving, each step a
// sum over the sequences, 64 at a time: a hundred cycles a step with up to 64 sequences, where a sorted list would be a launch of its own.  (Of more
// sequences all offsets are read again in each step, by every workgroup: 256 texts of 10 to 200 tokens, 16/4 heads x 64, take 61 us, 1000 of them 571, of whose bytes 66 are.)
template <bool kKeys>
TFK_DEVICE PackedTile find_tile(const PackedArgs& a, int rows, int rank) {
  const int lane = threadIdx.x % kWaveSize;
  auto own = [&](int b) __attribute__((always_inline)) -> SequenceTiles {   // a lane's
    if (b >= a.sequences) return {};
    return sequence_tiles<kKeys>(packed_range(a.offsets[b], a.offsets[b + 1], a.tokens), packed_range(a.kv_offsets[b], a.kv_offsets[b + 1], a.kv_tokens),
                                 (int)a.group.d, rows);
  };
  const SequenceTiles first = own(lane);   // (kept: mostly all there are)
  auto of = [&](int b0) __attribute__((always_inline)) -> SequenceTiles { return b0 == 0 ? first : own(b0 + lane); };
  int most = -0x7fffffff, least = 0x7fffffff;
  for (int b0 = 0; b0 < a.sequences; b0 += kWaveSize) {
    const SequenceTiles o = of(b0);
    if (o.tiles > 0) {
      most = max(most, o.level);
      least = min(least, o.level - o.tiles + 1);
    }
  }
  int high = wave_max(most) + 1, low = -wave_max(-least);   // none reaches `high`, all reach `low`
  auto count = [&](int level) __attribute__((always_inline)) {
    int n = 0;
    for (int b0 = 0; b0 < a.sequences; b0 += kWaveSize) {
      const SequenceTiles o = of(b0);
      n += min(max(o.level - level + 1, 0), o.tiles);
    }
    return wave_sum(n);
  };
  constexpr PackedTile none = {-1, 0, 0, 0, 0, 0};
  if (low >= high || count(low) <= rank) return none;
  int above = 0;   // tiles that reach `high`
  while (high - low > 1) {
    const int middle = low + (high - low) / 2, n = count(middle);
    if (n > rank) {
      low = middle;
    } else {
      high = middle;
      above = n;
    }
  }
  int left = rank - above;   // of the tiles that count `low`, one a sequence
  for (int b0 = 0; b0 < a.sequences; b0 += kWaveSize) {
    const SequenceTiles o = of(b0);
    const bool has = o.level >= low && o.level - low < o.tiles;
    const unsigned long long all = __builtin_amdgcn_ballot_w64(has);
    const int n = __builtin_popcountll(all);
    if (left >= n) {
      left -= n;
      continue;
    }
    const bool mine = has && __builtin_popcountll(all & ((1ull << lane) - 1)) == left;
    const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(mine));
    // (the ranges that the tile has been counted by: of ones that are read again, and that a program has changed meanwhile, it may be no tile)
    const auto of_lane = [&](int x) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(x, at); };
    return {b0 + at, of_lane(o.level) - low, of_lane(o.q.begin), of_lane(o.q.length), of_lane(o.k.begin), of_lane(o.k.length)};
  }
  return none;
}
TFK_DEVICE PackedTile packed_tile(const PackedArgs& a, int rows, int rank) { return find_tile<false>(a, rows, rank); }
// The same of the tiles of `keys` keys, from_end counted from a sequence's first key, which the most rows see.
TFK_DEVICE PackedTile packed_key_tile(const PackedArgs& a, int keys, int rank) { return find_tile<true>(a, keys, rank); }

// Rows in front of the first sequence and behind the last: `use` for each of them, `groups` workgroups sharing them out.
template <typename Use>
TFK_DEVICE void rows_outside(const int* offsets, int sequences, int rows, int group_no, int groups, Use use) {
  const int from = min(max(read_uniform(offsets), 0), rows), to = min(max(read_uniform(offsets + sequences), from), rows);
  const int outside = from + rows - to;
  for (int i = group_no; i < outside; i += groups) use(i < from ? i : to + i - from);
}
template <typename T>
TFK_DEVICE void clear_row(T* row, int elements) {
  using V8 = T __attribute__((ext_vector_type(8)));
  for (int c = threadIdx.x; c < elements / 8; c += blockDim.x) *reinterpret_cast<V8*>(row + 8 * c) = V8{};
}
}  // namespace tfk
