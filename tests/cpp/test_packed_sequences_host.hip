// Host-run checks of csrc/packed_sequences.hpp: ranges that offsets name, whatever those are.
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
  std::printf("ok\n");
  return 0;
}
