// Host-run checks of csrc/paged_cache.hpp: ranges of equal cost that workgroups take, and which of them has a unit.
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

#include "paged_cache.hpp"

#define CHECK(x)                                            \
  do {                                                      \
    if (!(x)) {                                             \
      std::printf("line %d: %s\n", __LINE__, #x);           \
      std::exit(1);                                         \
    }                                                       \
  } while (0)

int main() {
  using namespace tfk;
  for (unsigned groups : {1u, 2u, 3u, 255u, 256u})
    for (unsigned cost : {256u, 257u, 300u, 511u, 512u, 5000u, 100003u}) {
      const EqualRanges r = equal_ranges(cost, groups);
      CHECK(range_begin(r, 0) == 0 && range_begin(r, groups) == cost);
      for (unsigned i = 0; i < groups; ++i) {
        const unsigned begin = range_begin(r, i), end = range_begin(r, i + 1);
        CHECK(end - begin == cost / groups || end - begin == cost / groups + 1);
        CHECK(range_of(r, begin) == i && range_of(r, end - 1) == i);
      }
      // units that there are not, as they are counted of lengths that have grown meanwhile
      for (unsigned at : {cost, cost + 1, 2 * cost, 1u << 30, 0x7fffffffu, 0xffffffffu}) CHECK(range_of(r, at) < groups);
    }
  const EqualRanges most = equal_ranges(0x7fffffffu, 256);
  CHECK(range_begin(most, 256) == 0x7fffffffu && range_of(most, 0x7ffffffeu) == 255);
  std::printf("ok\n");
  return 0;
}
