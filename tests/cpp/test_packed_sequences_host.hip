// Host-run checks of csrc/packed_sequences.hpp: ranges that offsets name, whatever those are, and the tiles that sequences make.
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

#include "packed_sequences.hpp"

#define CHECK(x)                                            \
  do {                                                      \
    if (!(x)) {                                             \
      std::printf("line %d: %s\n", __LINE__, #x);           \
      std::exit(1);                                         \
    }                                                       \
  } while (0)

int main() {
  using namespace tfk;
  const int odd[] = {-2147483647 - 1, -70, -1, 0, 1, 30, 99, 100, 101, 2147483647};
  for (int begin : odd)
    for (int end : odd) {
      const PackedRange r = packed_range(begin, end, 100);
      CHECK(r.begin >= 0 && r.length >= 0 && r.begin + r.length <= 100);
      if (0 <= begin && begin <= end && end <= 100) CHECK(r.begin == begin && r.length == end - begin);
    }

  // Every tile that a sequence has: the rows (in tiles from the front, or in 64s from the end for causal attention) and keys that the kernels take for its
  // number begin in front of the last and not a tile in front of the first.
  for (int group : {1, 3, 4, 8, 100})
    for (int lq : {0, 1, 31, 64, 129, 300, 1000})
      for (int lkv : {0, 1, 127, 128, 400, 4000}) {
        const PackedRange q = {5, lq}, k = {7, lkv};
        for (int rows : {64, 128, 256}) {
          const SequenceTiles s = sequence_tiles<false>(q, k, group, rows);
          CHECK(s.q.begin == 5 && s.q.length == lq && s.k.begin == 7 && s.k.length == lkv && (s.tiles == 0) == (lq == 0));
          CHECK(s.tiles * rows >= lq * group && s.level * rows >= lkv * group && (s.level - 1) * rows < lkv * group);
          for (int e = 0; e < s.tiles; ++e) {
            const int all = lq * group, first = (s.tiles - 1 - e) * rows, first_causal = (all + 63) / 64 * 64 - (e + 1) * rows;
            CHECK(first >= 0 && first < all && first_causal > -rows && first_causal < all);
          }
        }
        const SequenceTiles s = sequence_tiles<true>(q, k, group, 128);
        CHECK(s.level == s.tiles && s.tiles * 128 >= lkv && (s.tiles == 0) == (lkv == 0));
        for (int e = 0; e < s.tiles; ++e) CHECK(e * 128 < lkv);
      }
  std::printf("ok\n");
  return 0;
}
