// One new token of every sequence against a paged cache, with grouped heads: out[b][h] = softmax(scale q K^T) V over the
// lengths[b] keys of the sequence, which lie in the pages that its row of the table names.
//
// No counterpart in the reference.  HBM-bound: every key and value is read once, for all query heads of its group together (4 G flops a
// byte for a group of G), so the products run on the matrix pipe whatever G is: S^T = K Q^T and O^T = V^T P^T with a block of 16 queries, of
// which a group fills G columns (a larger group is several blocks, which read the keys again).
//   * Work is cut without the host knowing the lengths: all (sequence, key head) items are laid end to end, in blocks of kBlockKeys keys and what
//     an item costs besides, and every workgroup takes an equal range of that, whatever items that range cuts through.  An item in one workgroup's range is
//     written by it, of any other every workgroup leaves its part (fp32 rows, maximum, sum) and the last to arrive puts the
//     parts together.  A workgroup has at most two parts, so the workspace depends on the sequences' number alone.
//   * A wavefront takes every kWaves-th tile of 16 keys of the range and shares nothing with the others up to the end of an item: tiles of K and V
//     go from their pages to registers, 24 KiB ahead, which with 8 wavefronts on a CU is what its share of HBM needs on the way; keys are fragments
//     as they are loaded, values pass through 4 KiB of LDS for their transposition, with no barrier.
//   * Pages are whole tiles: a tile's page is looked up with a scalar load, one tile before it is needed, and the lanes' offsets
//     within a tile are constants of the launch.
// 16 texts of 32768 keys, 8 heads x 128: 343 us, 6.3 TB/s, where the same bytes from one dense cache come at 6.7 (flash_decode.hip); 60 texts of 17 to 8001
// keys, 8 x 64: 43 us, 3.7 TB/s, of which 12 go to the launch, the ranges, the first pages and the last parts, as one text of 1999 keys shows, which takes
// no less.  That much is this kernel's arrangement for many texts, and no bound of one: the dense kernel reads as many bytes in 6.3.
#include <algorithm>

#include "flash_attention.hpp"
#include "paged_cache.hpp"

namespace tfk {
namespace {

constexpr int kWaves = 8, kThreads = kWaves * kWaveSize, kTileKeys = 16;
constexpr int kBlockKeys = kWaves * kTileKeys;   // a tile each
constexpr int tiles_ahead(int d) { return d == 128 ? 3 : 4; }   // of a wavefront, in registers: 24 or 16 KiB
constexpr int kQueries = 16;   // of an item: one block of MFMA columns
// Workgroups of a launch, one on a CU.  (Two of half the size: the older one is served first and is done at two thirds of the time, the other
// goes on alone and takes in less than the CU's share: they were done at 235 and 343 us with 16 of 8 heads x 32768 x 128.)
constexpr int kGroups = kCUs;

struct DecodeArgs {
  const void* query;
  int64_t query_token, query_head;
  void* out;   // [sequences][heads][D]
  const void *key, *value;
  int64_t key_strides[3], value_strides[3];   // page, token, head
  PageTable table;
  const int* lengths;
  int sequences, heads, kv_heads, group, blocks_of_group;   // blocks_of_group: blocks of kQueries in a group
  float scale_log2;
  float* part;         // [workgroups][2]: rows [kQueries][D], then maximum and sum [kQueries][2]
  arrivals_t *arrivals, tag;   // a word an item
};

// Keys of a sequence of `length` that are looked at; -1: that is beyond the table.
TFK_DEVICE int keys_of(const DecodeArgs& a, int length) {
  return length > (int64_t)a.table.width * a.table.page.d ? -1 : max(length, 0);
}
TFK_DEVICE int blocks_of(int keys) { return (max(keys, 0) + kBlockKeys - 1) / kBlockKeys; }
// An item costs the time of its blocks and of kOverhead more: to begin with new queries and pages, and to come together.  Ranges are of equal
// cost (60 texts of 17 to 8001 keys, 8 heads x 64: the workgroups with many short ones were done at 60 us, the others at 30).
__host__ __device__ constexpr int overhead(int d) { return d == 128 ? 1 : 2; }
template <int D>
TFK_DEVICE int cost_of(int keys) { return keys > 0 ? blocks_of(keys) + overhead(D) : 0; }

// 16 bytes at base + offset, zeros where that is not within `bytes`; `base` and `bytes` are wavefront-uniform.  kOnce: whole lines, which no
// cache need keep (a key's line is loaded in two halves: 16 of 8 heads x 32768 x 128 341 us with the hint, 335 without).
template <typename V, bool kOnce>
TFK_DEVICE V load_below(const void* base, unsigned bytes, unsigned offset) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int kRaw32Bit = 0x00020000, kStreaming = kOnce ? 2 : 0;
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, kRaw32Bit);
  return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(rsrc, offset, 0, kStreaming));
#else
  return V{};
#endif
}

// Position of (query, element) in a workgroup's part.
template <int D>
constexpr int part_floats() { return kQueries * (D + 2); }

// O^T += V^T P^T over 16 keys: lane l supplies V^T[l%16][4*(l/16)+t] and P^T[4*(l/16)+t][l%16].
template <typename T>
TFK_DEVICE float4_t mfma_16x16x16(typename Vec<T>::v4 a, typename Vec<T>::v4 b, float4_t c) {
  using Short4 = short __attribute__((ext_vector_type(4)));
  if constexpr (std::is_same_v<T, bf16_t>)
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(Short4, a), __builtin_bit_cast(Short4, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0);
}

// Two numbers that another workgroup of the launch has left; `from` wavefront-uniform, offset in bytes.
TFK_DEVICE float2_t load_shared_8B(const void* from, unsigned offset) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int kRaw32Bit = 0x00020000, kAgent = 16;   // sc1
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(from), 0, 0x7fffffff, kRaw32Bit);
  return __builtin_bit_cast(float2_t, __builtin_amdgcn_raw_buffer_load_b64(rsrc, offset, 0, kAgent));
#else
  return float2_t{};
#endif
}

// A sum of weights and the rows that they weigh, against a maximum.
struct Weighed {
  float m = -INFINITY, l = 0.f;
  float4_t o = {0.f, 0.f, 0.f, 0.f};
};
TFK_DEVICE void add_weighed(Weighed& w, float m, float l, float4_t o) {
  const float top = fmaxf(w.m, m);
  const float a = w.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(w.m - top), b = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
  w.o = a * w.o + b * o;
  // (a sum that is NaN, for a page that is not there, stays it with whatever weight)
  w.l = (w.l == 0.f ? 0.f : a * w.l) + (l == 0.f ? 0.f : b * l);
  w.m = top;
}
template <typename T>
TFK_DEVICE void store_weighed(const Weighed& w, T* to) {
  const float inv = w.l == 0.f ? 0.f : 1.f / w.l;
  typename Vec<T>::v4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = (T)(w.o[e] * inv);
  *reinterpret_cast<typename Vec<T>::v4*>(to) = y;
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads, 2) void flash_decode_paged_kernel(DecodeArgs a) {
  using V4 = typename Vec<T>::v4;
  using V8 = typename Vec<T>::v8;
  constexpr int kChunks = D / 8, kRowsPerLoad = kWaveSize / kChunks;   // 16-byte pieces of a row; rows of one load
  constexpr int kLoads = kTileKeys / kRowsPerLoad;                      // ... of a tile's keys, as of its values
  constexpr int kKK = D / 32, kDB = D / 16, kColumns = D / 4, kAhead = tiles_ahead(D);
  constexpr int kRoom = kQueries * D * 4;   // bytes of LDS of a wavefront: its rows at the end, before that a tile of values
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  __shared__ float s_stats[kWaves][kQueries][2];
  __shared__ bool s_last[2];

  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int items_of = a.kv_heads * a.blocks_of_group;   // of a sequence

  // ---- this workgroup's range of the items' costs ---------------------------------------------------------
  auto own_cost = [&](int b) __attribute__((always_inline)) { return b < a.sequences ? cost_of<D>(keys_of(a, a.lengths[b])) : 0; };
  const int first_own = wave_prefix(own_cost(lane));   // (kept: mostly all there are)
  int total = __builtin_amdgcn_readlane(first_own, 63);
  for (int b0 = kWaveSize; b0 < a.sequences; b0 += kWaveSize) total += __builtin_amdgcn_readlane(wave_prefix(own_cost(b0 + lane)), 63);
  const unsigned cost = (unsigned)total * (unsigned)items_of;   // (below 2^31: the host has seen the tables' width)
  // sequences without a key, and those that the table cannot hold
  for (int b = blockIdx.x; b < a.sequences; b += gridDim.x) {
    const int n = keys_of(a, read_uniform(a.lengths + b));
    if (n > 0) continue;
    const float v = n < 0 ? __builtin_nanf("") : 0.f;
    for (int i = tid; i < a.heads * D; i += kThreads) static_cast<T*>(a.out)[(int64_t)b * a.heads * D + i] = (T)v;
  }
  const unsigned groups = min(gridDim.x, cost);
  if (blockIdx.x >= groups) return;
  const EqualRanges ranges = equal_ranges(cost, groups);
  const unsigned begin = range_begin(ranges, blockIdx.x), end = range_begin(ranges, blockIdx.x + 1);
  // the sequence in which the range begins
  int b = 0;
  unsigned before = 0;   // the cost of the sequences in front of it
  for (int b0 = 0; b0 < a.sequences; b0 += kWaveSize) {
    const int up_to = b0 == 0 ? first_own : wave_prefix(own_cost(b0 + lane));
    const bool passed = before + (unsigned)up_to * (unsigned)items_of <= begin;
    const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(passed));
    b = b0 + n;
    if (n > 0) before += (unsigned)__builtin_amdgcn_readlane(up_to, n - 1) * (unsigned)items_of;
    if (n < kWaveSize) break;
  }

  // ---- what a lane loads of a tile, bytes from its first row in memory, and where the values go in LDS ----
  const int key_step = (int)a.key_strides[1] * 2, value_step = (int)a.value_strides[1] * 2;
  const unsigned key_off = (unsigned)(lr * key_step + 16 * lg);   // chunk 4 kk + lg of key lr: a fragment as it is
  unsigned value_off[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) value_off[i] = (unsigned)((i * kRowsPerLoad + lane / kChunks) * value_step + lane % kChunks * 16);
  const unsigned room = lds_address(smem) + wave * kRoom;
  // (the swizzle is an exclusive or of chunk numbers: rows of one load to the next, and columns 16 db, differ by constants)
  unsigned v_to[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int row = i * kRowsPerLoad + lane / kChunks;
    v_to[i] = room + row * D * 2 + swz_v<kChunks>(row, lane % kChunks) * 16;
  }
  const int v_row = 4 * lg + (lr >> 2), v_col = 4 * (lr & 3);
  const unsigned v_at = room + v_row * D * 2 + swz_v<kChunks>(v_row, v_col / 8) * 16 + (v_col % 8) * 2;

  // Items of which this workgroup has a part, the range's first and last at most: they are put together when all else is done, so
  // that nothing waits for stores and counts in between.
  struct Part {
    int parts = 0, first = 0, h0 = 0, queries = 0, b = 0;   // workgroups, the first of them; heads; sequence
    arrivals_t* word = nullptr;
  } mine[2];   // [1]: of an item that begins in this range

  // One item, or what of it is in the range: blocks [first, first + blocks).
  struct Segment {
    int b, h0, queries, head, keys, first, blocks;
    unsigned begin, cost;   // where the item begins, and what it costs
  };
  // The next segment of the range from `at` on, which is moved behind it; no blocks: there is none.  An item's overhead stands in front of its
  // blocks, and a range may end in it.  b and `before` are those of the segment in front, or of the range's beginning.
  unsigned at = begin;
  auto next_segment = [&]() __attribute__((always_inline)) -> Segment {
    Segment g = {};
    while (at < end && g.blocks == 0) {
      int keys = keys_of(a, read_uniform(a.lengths + b));
      unsigned of_item = cost_of<D>(keys);
      // (the range is within the sum; bounded all the same, for lengths that a program changes while they are read)
      while (at >= before + of_item * (unsigned)items_of && b + 1 < a.sequences) {
        before += of_item * (unsigned)items_of;
        keys = keys_of(a, read_uniform(a.lengths + ++b));
        of_item = cost_of<D>(keys);
      }
      if (at - before >= of_item * (unsigned)items_of) break;
      const unsigned item = (at - before) / of_item, item_begin = before + item * of_item, stop = min(item_begin + of_item, end);
      const int head = (int)item / a.blocks_of_group, query0 = (int)item % a.blocks_of_group * kQueries;
      const int first = max((int)(at - item_begin) - overhead(D), 0), last = max((int)(stop - item_begin) - overhead(D), 0);
      g = {b, head * a.group + query0, min(kQueries, a.group - query0), head, keys, first, last - first, item_begin, of_item};
      at = stop;
    }
    return g;
  };

  V8 qf[kKK], k[kAhead][kKK], v[kAhead][kLoads];
  bool lost = false, next_lost = false;   // a page that the cache does not have
  int next_page = 0;
  // This wavefront's tile of a block of a segment.
  auto page_for = [&](const Segment& g, int block) __attribute__((always_inline)) {
    // (within the table: keys_of; what the entry holds is looked at when it is needed, so that nothing waits for it here)
    return read_uniform(a.table.pages + g.b * a.table.stride + divide(a.table.page, min((g.first + block) * kWaves + wave, (g.keys - 1) / kTileKeys) * kTileKeys));
  };
  // Tiles past the end are asked for as well, and rows behind the last key: the bounds check of a buffer load returns zeros there and fetches nothing.
  // (With a branch around loads the compiler waits for all of them where its two ways meet.  Zeros, because what the cache holds behind
  // the last key may be infinite, and its weight of zero would make NaN of it.)
  auto load = [&](const Segment& g, int n, int block, int page, bool& none) __attribute__((always_inline)) {
    const int tile = (g.first + block) * kWaves + wave, key0 = min(tile, (g.keys - 1) / kTileKeys) * kTileKeys;
    const int rows = block < g.blocks ? min(kTileKeys, g.keys - tile * kTileKeys) : 0;
    const bool there = page >= 0 && page < a.table.cache_pages;
    none |= rows > 0 && !there;
    page = there ? page : 0;
    const int row = key0 - divide(a.table.page, key0) * (int)a.table.page.d;
    const T* kp = static_cast<const T*>(a.key) + page * a.key_strides[0] + row * a.key_strides[1] + g.head * a.key_strides[2];
    const T* vp = static_cast<const T*>(a.value) + page * a.value_strides[0] + row * a.value_strides[1] + g.head * a.value_strides[2];
    const unsigned key_bytes = rows > 0 ? (unsigned)((rows - 1) * key_step + D * 2) : 0u;
    const unsigned value_bytes = rows > 0 ? (unsigned)((rows - 1) * value_step + D * 2) : 0u;
#pragma unroll
    for (int kk = 0; kk < kKK; ++kk) k[n][kk] = load_below<V8, false>(kp, key_bytes, key_off + 64 * kk);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) v[n][i] = load_below<V8, true>(vp, value_bytes, value_off[i]);
    __builtin_amdgcn_sched_barrier(0);   // the requests leave before the next tile is consumed
  };
  // What a segment's first blocks need, asked for.
  auto start = [&](const Segment& g) __attribute__((always_inline)) {
    const T* q = static_cast<const T*>(a.query) + g.b * a.query_token + (g.h0 + min(lr, g.queries - 1)) * a.query_head;
    int pages[kAhead];
#pragma unroll
    for (int n = 0; n < kAhead; ++n) pages[n] = page_for(g, n);
    next_page = page_for(g, kAhead);   // (asked for a tile before it is needed)
#pragma unroll
    for (int kk = 0; kk < kKK; ++kk) qf[kk] = *reinterpret_cast<const V8*>(q + 32 * kk + 8 * lg);
#pragma unroll
    for (int n = 0; n < kAhead; ++n) load(g, n, n, pages[n], next_lost);
  };

  Segment now = next_segment();
  if (now.blocks > 0) start(now);
  while (now.blocks > 0) {
    lost = next_lost;
    next_lost = false;
    float4_t o[kDB];
#pragma unroll
    for (int db = 0; db < kDB; ++db) o[db] = float4_t{0.f, 0.f, 0.f, 0.f};
    // Weights are taken 2^kUp times as large in fp16 and enter the product as a number and its remainder: a weight's smallest remainder is
    // then 2^-31 of the largest weight.
    constexpr float kUp = std::is_same_v<T, bf16_t> ? 0.f : 7.f, kLazy = kUp + 8.f;
    float top = -INFINITY, sum = 0.f;   // reference of query lr; this lane's part of its weights' sum

    auto consume = [&](int n, int left) __attribute__((always_inline)) {   // left: keys of the tile; it may have none
      float4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < kKK; ++kk) s = mfma_t<T>(k[n][kk], qf[kk], s);
      // (LDS serves a wavefront in order: what the last tile has read is read)
#pragma unroll
      for (int i = 0; i < kLoads; ++i) *(__attribute__((address_space(3))) V8*)(size_t)v_to[i] = v[n][i];
      V4 vf[kDB];
#pragma unroll
      for (int db = 0; db < kDB; ++db) vf[db] = lds_read_tr4<V4>(v_at ^ (db << 5));
      float big = -INFINITY;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[r] = 4 * lg + r < left ? s[r] * a.scale_log2 : -INFINITY;
        big = fmaxf(big, s[r]);
      }
      if (__builtin_amdgcn_ballot_w64(big > top + kLazy) != 0) {   // (the first finite score, too)
        const float higher = fmaxf(top, quad_max(big) - kUp);
        const float factor = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top - higher);
        top = higher;
        sum *= factor;
#pragma unroll
        for (int db = 0; db < kDB; ++db) o[db] *= factor;
      }
      const float reference = top == -INFINITY ? 0.f : top;
      V4 p, rest;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float w = __builtin_amdgcn_exp2f(s[r] - reference);
        sum += w;
        const SplitWeight<T> two = split_weight<T>(w);
        p[r] = two.whole;
        rest[r] = two.rest;
      }
#pragma unroll
      for (int db = 0; db < kDB; ++db) {
        o[db] = mfma_16x16x16<T>(vf[db], p, o[db]);
        o[db] = mfma_16x16x16<T>(vf[db], rest, o[db]);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    // (the queries came first: waited for here, they are not waited for among the tiles, and all that is ahead with them)
#pragma unroll
    for (int kk = 0; kk < kKK; ++kk) asm volatile("" : "+v"(qf[kk]));
    auto consume_block = [&](int n, int block) __attribute__((always_inline)) {
      consume(n, now.keys - ((now.first + block) * kWaves + wave) * kTileKeys);
    };
    // (whole rounds, and then what is left: the loads on their way at a loop's beginning are always the same, and the compiler waits for no more
    // than it needs)
    int block = 0;
    for (; block + kAhead <= now.blocks; block += kAhead) {
#pragma unroll
      for (int n = 0; n < kAhead; ++n) {
        consume_block(n, block + n);
        load(now, n, block + n + kAhead, next_page, lost);
        next_page = page_for(now, block + n + 1 + kAhead);
      }
      barrier_only();   // (the wavefronts in step: the older ones are served first, and would leave the others behind)
    }
#pragma unroll
    for (int n = 0; n < kAhead - 1; ++n)
      if (block + n < now.blocks) consume_block(n, block + n);

    // ---- the next segment is on its way while this one's wavefronts come together ---------------
    const Segment done = now;
    now = next_segment();
    if (now.blocks > 0) start(now);
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (lost) sum = __builtin_nanf("");
    if (lg == 0) {
      s_stats[wave][lr][0] = top;
      s_stats[wave][lr][1] = sum;
    }
    float* const s_rows = reinterpret_cast<float*>(smem + wave * kRoom);   // [kQueries][D]
#pragma unroll
    for (int db = 0; db < kDB; ++db) *reinterpret_cast<float4_t*>(s_rows + lr * D + ((db ^ (lr & (kDB - 1))) * 16 + 4 * lg)) = o[db];
    barrier_lds_only();
    // the workgroups that have a part of the item
    const bool whole = done.first == 0 && done.blocks + overhead(D) == (int)done.cost;
    // (workgroups that there are, also for lengths that a program changes while they are read)
    const unsigned part_first = whole ? blockIdx.x : range_of(ranges, done.begin + overhead(D));
    const int parts = whole ? 1 : (int)(range_of(ranges, done.begin + done.cost - 1) - part_first) + 1;
    const bool begins = blockIdx.x == part_first;
    T* const out = static_cast<T*>(a.out) + ((int64_t)done.b * a.heads + done.h0) * D;
    float* const part = a.part + ((int64_t)blockIdx.x * 2 + (begins ? 1 : 0)) * part_floats<D>();
    if (parts > 1) {
      arrivals_t* const word = a.arrivals + ((int64_t)done.b * items_of + done.h0 / a.group * a.blocks_of_group + done.h0 % a.group / kQueries) * kArrivalsPitch;
      if (begins && tid == 0) open_arrivals(word, a.tag);
      const Part p = {parts, (int)part_first, done.h0, done.queries, done.b, word};
      if (begins) mine[1] = p;
      else mine[0] = p;
    }
    for (int i = tid; i < done.queries * kColumns; i += kThreads) {
      const int qi = i / kColumns, c = i % kColumns;
      Weighed w;
#pragma unroll
      for (int x = 0; x < kWaves; ++x)
        add_weighed(w, s_stats[x][qi][0], s_stats[x][qi][1],
                    *reinterpret_cast<const float4_t*>(reinterpret_cast<const float*>(smem + x * kRoom) + qi * D +
                                                       (((c / 4) ^ (qi & (kDB - 1))) * 16 + 4 * (c % 4))));
      if (parts == 1) {
        store_weighed(w, out + qi * D + 4 * c);
        continue;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) store_shared(part + qi * D + 4 * c + e, w.o[e]);
      if (c == 0) {
        store_shared(part + kQueries * D + 2 * qi, w.m);
        store_shared(part + kQueries * D + 2 * qi + 1, w.l);
      }
    }
    barrier_lds_only();   // the room is the next item's
  }

  if (mine[0].parts + mine[1].parts == 0) return;
  wait_vmem_all();
  __syncthreads();
  if (lane == 0 && wave < 2) s_last[wave] = mine[wave].parts > 0 && arrive(mine[wave].word, a.tag, (unsigned)mine[wave].parts);
  __syncthreads();
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (!s_last[which]) continue;
    // The parts lie in the second room of the first workgroup and in the first rooms of the others.  kBatch of them are on their way at a
    // time, and where an item has few queries several threads share the parts of a column.
    constexpr int kBatch = 8;
    constexpr unsigned kPitch = 2 * part_floats<D>() * 4, kSecond = part_floats<D>() * 4;
    const Part& p = mine[which];
    const float* const from = a.part + (int64_t)p.first * 2 * part_floats<D>();
    T* const out = static_cast<T*>(a.out) + ((int64_t)p.b * a.heads + p.h0) * D;
    const int units = p.queries * kColumns, parts = p.parts;
    const int sharing = units * 8 <= kThreads ? 8 : units * 4 <= kThreads ? 4 : units * 2 <= kThreads ? 2 : 1;
    Weighed* const s_shared = reinterpret_cast<Weighed*>(smem);   // [sharing][units]
    for (int i = tid; i < units * sharing; i += kThreads) {
      const int unit = i % units, share = i / units, qi = unit / kColumns, c = unit % kColumns;
      Weighed w;
      for (int s0 = share; s0 < parts; s0 += kBatch * sharing) {
        float2_t ml[kBatch];
        float4_t x[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int s = min(s0 + u * sharing, parts - 1);
          const unsigned slot = (unsigned)s * kPitch + (s == 0 ? kSecond : 0u);
          ml[u] = load_shared_8B(from, slot + (kQueries * D + 2 * qi) * 4);
          x[u] = load_shared_16B<float4_t>(from, slot + (qi * D + 4 * c) * 4);
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
          if (s0 + u * sharing < parts) add_weighed(w, ml[u][0], ml[u][1], x[u]);
      }
      if (sharing == 1) store_weighed(w, out + qi * D + 4 * c);
      else s_shared[share * units + unit] = w;
    }
    if (sharing > 1) {
      __syncthreads();
      if (tid < units) {
        Weighed w = s_shared[tid];
        for (int k = 1; k < sharing; ++k) {
          const Weighed& x = s_shared[k * units + tid];
          add_weighed(w, x.m, x.l, x.o);
        }
        store_weighed(w, out + tid / kColumns * D + 4 * (tid % kColumns));
      }
      __syncthreads();
    }
  }
}

int blocks_of_group(int64_t heads, int64_t kv_heads) { return (int)((heads / kv_heads + kQueries - 1) / kQueries); }
size_t part_bytes(int64_t D) { return (size_t)kGroups * 2 * kQueries * (size_t)(D + 2) * sizeof(float); }

template <typename T, int D>
int launch_decode_paged(const DecodeArgs& a, hipStream_t st) {
  auto kern = flash_decode_paged_kernel<T, D>;
  constexpr int lds = kWaves * kQueries * D * 4;
  TFK_LDS_OPT_IN(kern, lds);
  // (what there can be: a launch of a few sequences with short tables asks for no more workgroups than that)
  const int64_t most = (int64_t)a.sequences * a.kv_heads * a.blocks_of_group * (((int64_t)a.table.width * a.table.page.d + kBlockKeys - 1) / kBlockKeys + overhead(D));
  return launch_kernel(kern, dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(most, kGroups))), dim3(kThreads), lds, st, a);
}

}  // namespace

}  // namespace tfk

extern "C" size_t tf_flash_decode_paged_workspace_bytes(int64_t sequences, int64_t heads, int64_t kv_heads, int64_t D) {
  if (sequences <= 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads != 0 || (D != 64 && D != 128)) return 0;
  return tfk::part_bytes(D) + (size_t)sequences * kv_heads * tfk::blocks_of_group(heads, kv_heads) * tfk::kArrivalsPitch * sizeof(tfk::arrivals_t);
}

extern "C" int tf_flash_decode_paged(const tf_paged_cache_t* cache, const void* query, const int64_t* query_strides, void* out, int64_t heads,
                                     double softmax_scale, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace tfk;
  constexpr const char* who = "tf_flash_decode_paged";
  if (int rc = check_paged_cache(who, cache)) return rc;
  TFK_REQUIRE(heads > 0 && heads <= 65536 && heads % cache->kv_heads == 0, TF_ERR_INVALID_ARG, "%s: heads must be a multiple of kv_heads, at most 65536", who);
  TFK_REQUIRE(cache->page_size % 16 == 0, TF_ERR_UNSUPPORTED, "%s: page_size must be a multiple of 16 (got %lld)", who, (long long)cache->page_size);
  TFK_REQUIRE(cache->key_strides[1] < (1 << 26) && cache->value_strides[1] < (1 << 26), TF_ERR_UNSUPPORTED,
              "%s: the cache's strides from token to token must be below 2^26 elements", who);
  TFK_REQUIRE(is_softmax_scale(softmax_scale), TF_ERR_INVALID_ARG, "%s: softmax_scale must be finite, times log2(e) in fp32 too", who);
  if (cache->sequences == 0) return TF_OK;
  TFK_REQUIRE(cache->table_width < (1ll << 31) / cache->page_size &&
                  cache->sequences * (cache->table_width * cache->page_size / kBlockKeys + 3) <
                      (1ll << 31) / (cache->kv_heads * blocks_of_group(heads, cache->kv_heads)),
              TF_ERR_INVALID_ARG, "%s: the table has room for 2^31 tokens a sequence, or 2^31 blocks of 128 keys in all", who);
  TFK_REQUIRE(cache->sequences * heads < (1 << 24), TF_ERR_INVALID_ARG, "%s: sequences * heads must be below 2^24", who);
  TFK_REQUIRE(query && query_strides && out && workspace, TF_ERR_INVALID_ARG, "%s: null pointer", who);
  TFK_REQUIRE(query_strides[0] >= 0 && query_strides[1] >= 0 && query_strides[0] % 8 == 0 && query_strides[1] % 8 == 0, TF_ERR_INVALID_ARG,
              "%s: strides must be multiples of 8 elements", who);
  TFK_REQUIRE(((reinterpret_cast<uintptr_t>(query) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15) == 0, TF_ERR_INVALID_ARG,
              "%s: operands must begin at 16-byte boundaries", who);
  const size_t need = tf_flash_decode_paged_workspace_bytes(cache->sequences, heads, cache->kv_heads, cache->D);
  TFK_REQUIRE(workspace_bytes >= need, TF_ERR_INVALID_ARG, "%s: workspace holds %zu bytes, %zu needed", who, workspace_bytes, need);
  TFK_REQUIRE(is_ordinary_device_memory(workspace), TF_ERR_INVALID_ARG, "%s: the workspace must be ordinary memory of the current device", who);
  DecodeArgs a = {query, query_strides[0], query_strides[1], out, cache->key, cache->value, {}, {}, page_table(*cache), cache->lengths,
                  (int)cache->sequences, (int)heads, (int)cache->kv_heads, (int)(heads / cache->kv_heads), blocks_of_group(heads, cache->kv_heads),
                  (float)(softmax_scale * 1.4426950408889634), static_cast<float*>(workspace),
                  reinterpret_cast<arrivals_t*>(static_cast<char*>(workspace) + part_bytes(cache->D)), next_arrivals_tag()};
  std::copy_n(cache->key_strides, 3, a.key_strides);
  std::copy_n(cache->value_strides, 3, a.value_strides);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const bool bf16 = cache->dtype == TF_DTYPE_BF16;
  if (cache->D == 128) return bf16 ? launch_decode_paged<bf16_t, 128>(a, st) : launch_decode_paged<half_t, 128>(a, st);
  return bf16 ? launch_decode_paged<bf16_t, 64>(a, st) : launch_decode_paged<half_t, 64>(a, st);
}
