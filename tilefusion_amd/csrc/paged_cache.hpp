// A cache of keys and values in pages, as append_paged_kv.hip writes and flash_decode_paged.hip reads it, and sequences packed one
// behind the other.
//
// Token `position` of sequence b is row position % page_size of page table[b][position / page_size].  The host does not see tables, lengths
// and offsets, which are in device memory: the kernels take whatever they hold.  A page that is not one of the cache's is
// never read or written.
#pragma once

#include "common.hpp"

namespace tfk {

// n / d and n % d for 0 <= n < 2^31, 0 < d < 2^31: n * ceil(2^(31 + l) / d) >> (31 + l) with l = ceil(log2 d).  The multiplier is
// too large by less than d / 2^(31 + l) of itself at most, which moves the quotient by less than n / 2^(31 + l) <= 1 / d, and below 2^32.
struct Divider {
  unsigned d, factor;
  int shift;
};
inline Divider make_divider(unsigned d) {
  int l = 0;
  while ((1ull << l) < d) ++l;
  return {d, (unsigned)(((1ull << (31 + l)) + d - 1) / d), 31 + l};
}
__host__ __device__ inline int divide(const Divider& by, int n) {
  return (int)(((unsigned long long)(unsigned)n * by.factor) >> by.shift);
}

// A value that all lanes of a wavefront read at one address and no kernel of the launch writes, through the scalar cache.
__host__ __device__ inline int read_uniform(const int* p) {
#if defined(__HIP_DEVICE_COMPILE__)
  return *(const __attribute__((address_space(4))) int*)(uintptr_t)p;
#else
  return *p;
#endif
}

// `cost` units in `groups` ranges of equal length, the first `longer` of them longer by one; 0 < groups <= cost.
struct EqualRanges {
  unsigned groups, quota, longer;
};
__host__ __device__ inline EqualRanges equal_ranges(unsigned cost, unsigned groups) { return {groups, cost / groups, cost % groups}; }
__host__ __device__ inline unsigned range_begin(const EqualRanges& r, unsigned no) { return no * r.quota + (no < r.longer ? no : r.longer); }
// The range that holds a unit, the last one for units that there are not.
__host__ __device__ inline unsigned range_of(const EqualRanges& r, unsigned at) {
  const unsigned split = r.longer * (r.quota + 1), no = at < split ? at / (r.quota + 1) : r.longer + (at - split) / r.quota;
  return no < r.groups ? no : r.groups - 1;
}

struct PageTable {
  const int* pages;   // [sequences][stride], `width` of each row
  int64_t stride;
  int width, cache_pages;
  Divider page;
};
// Page that holds `position` of sequence b, -1 where there is none (a position before the first or behind the table's last, a page
// that the cache does not have).
__host__ __device__ inline int page_of(const PageTable& t, int64_t b, int64_t position) {
  if (position < 0 || position >= (int64_t)t.width * t.page.d || position >= 0x7fffffff) return -1;
  const int page = read_uniform(t.pages + b * t.stride + divide(t.page, (int)position));
  return page >= 0 && page < t.cache_pages ? page : -1;
}

// `use` of what all lanes up to one's own have, in steps that stay within registers (rows of 16 lanes by shifts of 1, 2, 4 and 8, then a row's
// last lane to the next row, and the 32nd to the upper half): a tenth of the time of six exchanges through LDS.  All lanes call.
template <typename Use>
TFK_DEVICE int wave_scan(int x, int identity, Use use) {
#if defined(__HIP_DEVICE_COMPILE__)
  x = use(x, __builtin_amdgcn_update_dpp(identity, x, 0x111, 0xf, 0xf, false));
  x = use(x, __builtin_amdgcn_update_dpp(identity, x, 0x112, 0xf, 0xf, false));
  x = use(x, __builtin_amdgcn_update_dpp(identity, x, 0x114, 0xf, 0xf, false));
  x = use(x, __builtin_amdgcn_update_dpp(identity, x, 0x118, 0xf, 0xf, false));
  x = use(x, __builtin_amdgcn_update_dpp(identity, x, 0x142, 0xa, 0xf, false));
  x = use(x, __builtin_amdgcn_update_dpp(identity, x, 0x143, 0xc, 0xf, false));
#endif
  return x;
}
TFK_DEVICE int wave_prefix(int x) {   // sum up to a lane, its own included
  return wave_scan(x, 0, [](int a, int b) { return a + b; });
}
TFK_DEVICE int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_prefix(x), kWaveSize - 1); }
TFK_DEVICE int wave_max(int x) {
  return __builtin_amdgcn_readlane(wave_scan(x, -0x7fffffff, [](int a, int b) { return max(a, b); }), kWaveSize - 1);
}

// The sequence that holds token t of packed ones, those before it ending at or in front of t: -1 in front of the first, n behind the last.
// A wavefront looks at 64 ends at a time (all lanes call).  Offsets that do not ascend give some number within -1 .. n.
TFK_DEVICE int find_sequence(const int* __restrict__ offsets, int n, int t) {
  const int lane = threadIdx.x % kWaveSize;
  const bool before = offsets[0] > t;
  int low = 0, count = n;   // the ends offsets[low + 1 .. low + count] are left
  while (count > kWaveSize) {
    const int step = (count + kWaveSize - 1) / kWaveSize;
    const bool passed = (lane + 1) * step <= count && offsets[low + (lane + 1) * step] <= t;
    const int groups = __builtin_popcountll(__builtin_amdgcn_ballot_w64(passed));
    low += groups * step;
    count = min(step, count - groups * step);
  }
  const bool passed = lane < count && offsets[low + lane + 1] <= t;
  low += __builtin_popcountll(__builtin_amdgcn_ballot_w64(passed));
  return before ? -1 : low;
}

// Arguments of the entry points (append_paged_kv.hip).
int check_paged_cache(const char* who, const tf_paged_cache_t* cache);
PageTable page_table(const tf_paged_cache_t& cache);

}  // namespace tfk
