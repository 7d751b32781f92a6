// Host-run checks of csrc/paged_cache.hpp: divisions by a multiplication, and which page holds a position of a sequence.
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
  // quotients around every multiple that is near a power of two, and at the ends
  for (unsigned d : {1u, 2u, 3u, 5u, 7u, 16u, 48u, 63u, 64u, 65u, 100u, 255u, 1000u, 1023u, 1024u, 4097u, 65535u, 65536u, 0x7fffffffu}) {
    const Divider by = make_divider(d);
    auto same = [&](long long n) {
      if (n >= 0 && n <= 0x7fffffffll) CHECK(divide(by, (int)n) == n / (long long)d);
    };
    for (long long n = 0; n < 70000; ++n) same(n);
    for (int bit = 0; bit < 31; ++bit)
      for (long long off = -2; off <= 2; ++off) {
        const long long at = ((1ll << bit) / d + 1) * d + off;
        same(at);
        same(at - d);
        same((1ll << bit) + off);
      }
    for (long long n = 0x7fffffffll; n > 0x7fffffffll - 70000; --n) same(n);
  }

  // two sequences with room for three pages of 48 tokens, rows of the table 5 apart; pages -7 and 9 are not the cache's
  int entries[10] = {4, -7, 8, 99, 99, 0, 9, 1, 99, 99};
  const PageTable t = {entries, 5, 3, 9, make_divider(48)};
  CHECK(page_of(t, 0, 0) == 4 && page_of(t, 0, 47) == 4 && page_of(t, 0, 96) == 8 && page_of(t, 0, 143) == 8);
  CHECK(page_of(t, 1, 0) == 0 && page_of(t, 1, 100) == 1);
  CHECK(page_of(t, 0, 48) == -1 && page_of(t, 0, 95) == -1 && page_of(t, 1, 48) == -1);   // pages that there are not
  CHECK(page_of(t, 0, 144) == -1 && page_of(t, 1, 144) == -1);                              // behind the table's last
  CHECK(page_of(t, 0, -1) == -1 && page_of(t, 1, -1000) == -1);
  CHECK(page_of(t, 0, 0x7fffffffll) == -1 && page_of(t, 0, 1ll << 40) == -1);
  const PageTable none = {nullptr, 0, 0, 9, make_divider(16)};   // a table of no entries is not read
  CHECK(page_of(none, 0, 0) == -1);
  std::printf("ok\n");
  return 0;
}
