// One new token of every sequence against a paged cache, with grouped heads: out[b][h] = softmax(scale q K^T) V over the
// lengths[b] keys of the sequence, which lie in the pages that its row of the table names.
//
// No counterpart in the reference.  HBM-bound: every key and value is read once, for all query heads of its group together (4 G flops a
// byte for a group of G), so the products run on the matrix pipe whatever G is: S^T = K Q^T and O^T = V^T P^T with a block of 16 queries, of
// which a group fills G columns (a larger group is several blocks, which read the keys again).
//   * Work is cut without the host knowing the lengths: all (sequence, key head) items are laid end to end in blocks of kBlockKeys keys and
//     every workgroup takes an equal range of them, whatever items that range cuts through.  An item in one workgroup's range is
//     written by it, of any other every workgroup leaves its part (fp32 rows, maximum, sum) and the last to arrive puts the
//     parts together.  A workgroup has at most two parts, so the workspace depends on the sequences' number alone.
//   * A wavefront takes every kWaves-th tile of 16 keys of the range and shares nothing with the others up to the end of an item: tiles of K and V
//     go from their pages to LDS directly, three tiles ahead, and are waited for by count, with no barrier.
//   * Pages are whole tiles: a tile's page is looked up with a scalar load, one tile before it is needed, and the lanes' offsets
//     within a tile are constants of the launch.
#include <algorithm>

#include "flash_attention.hpp"
#include "paged_cache.hpp"

namespace tfk {
namespace {

constexpr int kWaves = 4, kThreads = kWaves * kWaveSize, kTileKeys = 16, kStages = 4;
constexpr int kTilesPerBlock = 8, kBlockKeys = kTilesPerBlock * kTileKeys;
constexpr int kQueries = 16;   // of an item: one block of MFMA columns
// Workgroups of a launch: those that LDS lets run at once.
__host__ __device__ constexpr int tile_bytes(int d) { return 2 * kTileKeys * d * 2; }
__host__ __device__ constexpr int resident(int d) { return kCUs * (kMaxLdsBytes / (kStages * kWaves * tile_bytes(d))); }

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

TFK_DEVICE int wave_prefix(int x) {   // inclusive sum over the lanes
  const int lane = threadIdx.x % kWaveSize;
#pragma unroll
  for (int d = 1; d < kWaveSize; d *= 2) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  return x;
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
__global__ __launch_bounds__(kThreads, 1) void flash_decode_paged_kernel(DecodeArgs a) {
  using V4 = typename Vec<T>::v4;
  using V8 = typename Vec<T>::v8;
  constexpr int kChunks = D / 8, kRowsPerLoad = kWaveSize / kChunks;   // 16-byte pieces of a row; rows of one load
  constexpr int kLoads = kTileKeys / kRowsPerLoad;                      // ... of a tile's keys, as of its values
  constexpr int kKK = D / 32, kDB = D / 16, kColumns = D / 4;
  constexpr int kKeyBytes = kTileKeys * D * 2, kStage = tile_bytes(D);
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  __shared__ float s_stats[kWaves][kQueries][2];
  __shared__ bool s_last;

  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int items_of = a.kv_heads * a.blocks_of_group;   // of a sequence

  // ---- this workgroup's range of blocks ---------------------------------------------------------
  auto own_blocks = [&](int b) __attribute__((always_inline)) { return b < a.sequences ? blocks_of(keys_of(a, a.lengths[b])) : 0; };
  const int first_own = wave_prefix(own_blocks(lane));   // (kept: mostly all there are)
  int total = __builtin_amdgcn_readlane(first_own, 63);
  for (int b0 = kWaveSize; b0 < a.sequences; b0 += kWaveSize) total += __builtin_amdgcn_readlane(wave_prefix(own_blocks(b0 + lane)), 63);
  const unsigned blocks = (unsigned)total * (unsigned)items_of;   // (below 2^31: the host has seen the tables' width)
  // sequences without a key, and those that the table cannot hold
  for (int b = blockIdx.x; b < a.sequences; b += gridDim.x) {
    const int n = keys_of(a, read_uniform(a.lengths + b));
    if (n > 0) continue;
    const float v = n < 0 ? __builtin_nanf("") : 0.f;
    for (int i = tid; i < a.heads * D; i += kThreads) static_cast<T*>(a.out)[(int64_t)b * a.heads * D + i] = (T)v;
  }
  // (no more workgroups than blocks; the first `longer` have one block more)
  const unsigned groups = min(gridDim.x, blocks);
  if (blockIdx.x >= groups) return;
  const unsigned quota = blocks / groups, longer = blocks - quota * groups;
  const unsigned begin = blockIdx.x * quota + min(blockIdx.x, longer), end = begin + quota + (blockIdx.x < longer ? 1 : 0);
  auto group_of = [&](unsigned block) __attribute__((always_inline)) {
    const unsigned split = longer * (quota + 1);
    return block < split ? block / (quota + 1) : longer + (block - split) / quota;
  };
  // the sequence in which the range begins
  int b = 0;
  unsigned before = 0;   // blocks of the sequences in front of it
  for (int b0 = 0; b0 < a.sequences; b0 += kWaveSize) {
    const int up_to = b0 == 0 ? first_own : wave_prefix(own_blocks(b0 + lane));
    const bool passed = before + (unsigned)up_to * (unsigned)items_of <= begin;
    const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(passed));
    b = b0 + n;
    if (n > 0) before += (unsigned)__builtin_amdgcn_readlane(up_to, n - 1) * (unsigned)items_of;
    if (n < kWaveSize) break;
  }

  // ---- LDS: where loads leave their rows and fragments find them ------------------------------
  const unsigned wave_base = lds_address(smem) + wave * kStages * kStage;
  unsigned key_off[kLoads], value_off[kLoads];   // bytes from a tile's first row in memory
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int row = i * kRowsPerLoad + lane / kChunks;
    key_off[i] = (unsigned)(row * (int)a.key_strides[1] + swz_k<kChunks>(row, lane % kChunks) * 8) * 2u;
    value_off[i] = (unsigned)(row * (int)a.value_strides[1] + swz_v<kChunks>(row, lane % kChunks) * 8) * 2u;
  }
  // (the swizzles are exclusive ors of chunk numbers: fragment kk of the keys is 64 kk further in that sense, db of the values 32 db)
  const unsigned k_at = lr * D * 2 + swz_k<kChunks>(lr, lg) * 16;
  const int v_row = 4 * lg + (lr >> 2), v_col = 4 * (lr & 3);
  const unsigned v_at = kKeyBytes + v_row * D * 2 + swz_v<kChunks>(v_row, v_col / 8) * 16 + (v_col % 8) * 2;

  for (unsigned at = begin; at < end; ++b) {
    const int keys = keys_of(a, read_uniform(a.lengths + b));
    const unsigned of_item = blocks_of(keys), of_sequence = of_item * (unsigned)items_of;
    while (at < end && at < before + of_sequence) {
      // ---- one item, or what of it is in the range: blocks [first, last) --------------------
      const int item = (int)((at - before) / of_item);
      const unsigned item_begin = before + (unsigned)item * of_item;
      const int first = (int)(at - item_begin), last = (int)min(of_item, end - item_begin);
      at = item_begin + last;
      const int head = item / a.blocks_of_group, query0 = item % a.blocks_of_group * kQueries;
      const int queries = min(kQueries, a.group - query0);
      const int h0 = head * a.group + query0;
      arrivals_t* const word = a.arrivals + ((int64_t)b * items_of + item) * kArrivalsPitch;
      // the workgroups that have a part of it
      const bool whole = first == 0 && last == (int)of_item;
      const unsigned part_first = whole ? blockIdx.x : group_of(item_begin);
      const int parts = whole ? 1 : (int)(group_of(item_begin + of_item - 1) - part_first) + 1;
      if (parts > 1 && tid == 0 && blockIdx.x == part_first) open_arrivals(word, a.tag);

      V8 qf[kKK];
      const T* q = static_cast<const T*>(a.query) + b * a.query_token + (h0 + min(lr, queries - 1)) * a.query_head;
#pragma unroll
      for (int kk = 0; kk < kKK; ++kk) qf[kk] = *reinterpret_cast<const V8*>(q + 32 * kk + 8 * lg);

      const int tile_end = min(last * kTilesPerBlock, (keys + kTileKeys - 1) / kTileKeys);
      bool lost = false;   // a page that the cache does not have
      const T* const keys_at = static_cast<const T*>(a.key) + head * a.key_strides[2];
      const T* const values_at = static_cast<const T*>(a.value) + head * a.value_strides[2];
      auto page_for = [&](int tile) __attribute__((always_inline)) { return page_of(a.table, b, min(tile, tile_end - 1) * kTileKeys); };
      auto request = [&](int tile, int page, int stage) __attribute__((always_inline)) {
        const unsigned dst = wave_base + stage * kStage;
        lost |= page < 0;
        page = max(page, 0);
        const int key0 = tile * kTileKeys, row = key0 - divide(a.table.page, key0) * (int)a.table.page.d;
        const T* k = keys_at + page * a.key_strides[0] + row * a.key_strides[1];
        const T* v = values_at + page * a.value_strides[0] + row * a.value_strides[1];
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
          asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(key_off[i]), "s"(k), "{m0}"(dst + i * 1024) : "memory");
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
          asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(value_off[i]), "s"(v), "{m0}"(dst + kKeyBytes + i * 1024) : "memory");
      };

      float4_t o[kDB];
#pragma unroll
      for (int db = 0; db < kDB; ++db) o[db] = float4_t{0.f, 0.f, 0.f, 0.f};
      // Weights are taken 2^kUp times as large in fp16 and enter the product as a number and its remainder: a weight's smallest remainder is
      // then 2^-31 of the largest weight.
      constexpr float kUp = std::is_same_v<T, bf16_t> ? 0.f : 7.f, kLazy = kUp + 8.f;
      float top = -INFINITY, sum = 0.f;   // reference of query lr; this lane's part of its weights' sum

      int tile = first * kTilesPerBlock + wave, ahead = tile;   // the next to compute, to request
      int pages[kStages - 1];
#pragma unroll
      for (int n = 0; n < kStages - 1; ++n) pages[n] = page_for(tile + n * kWaves);
      int next_page = page_for(tile + (kStages - 1) * kWaves);
#pragma unroll
      for (int kk = 0; kk < kKK; ++kk) asm volatile("" : "+v"(qf[kk]));   // (waited for here, not among the tiles)
#pragma unroll
      for (int n = 0; n < kStages - 1; ++n, ahead += kWaves)
        if (ahead < tile_end) request(ahead, pages[n], n);
      for (int n = 0; tile < tile_end; ++n, tile += kWaves) {
        const unsigned stage = wave_base + n % kStages * kStage;
        if (ahead < tile_end) {
          request(ahead, next_page, (n + kStages - 1) % kStages);
          ahead += kWaves;
          next_page = page_for(ahead);
          wait_vmem<(kStages - 1) * 2 * kLoads>();
        } else {   // (the last tiles have all been asked for)
          const int behind = (tile_end - 1 - tile) / kWaves;
          if (behind >= 2) wait_vmem<2 * 2 * kLoads>();
          else if (behind == 1) wait_vmem<2 * kLoads>();
          else wait_vmem_all();
        }
        const int left = keys - tile * kTileKeys;   // keys of the tile, one at least
        if (left < kTileKeys) {
          // rows behind the last key hold anything: their weight is zero, and zero times an infinity is none
          const V8 zeros = {};
#pragma unroll
          for (int i = 0; i < kLoads; ++i)
            if (i * kRowsPerLoad + lane / kChunks >= left)
              *(__attribute__((address_space(3))) V8*)(size_t)(stage + kKeyBytes + i * 1024 + lane * 16) = zeros;
        }
        const unsigned ka = opaque(stage + k_at), va = opaque(stage + v_at);
        float4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < kKK; ++kk) s = mfma_t<T>(lds_read_b128<V8>(ka ^ (kk << 6)), qf[kk], s);
        V4 vf[kDB];
#pragma unroll
        for (int db = 0; db < kDB; ++db) vf[db] = lds_read_tr4<V4>(va ^ (db << 5));
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
        // the tile's reads are done before its room is asked for again
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }

      // ---- the wavefronts together, in their tiles' room ------------------------------------------
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      if (lost) sum = __builtin_nanf("");
      if (lg == 0) {
        s_stats[wave][lr][0] = top;
        s_stats[wave][lr][1] = sum;
      }
      float* const s_rows = reinterpret_cast<float*>(smem + wave * kStages * kStage);   // [kQueries][D]
#pragma unroll
      for (int db = 0; db < kDB; ++db) *reinterpret_cast<float4_t*>(s_rows + lr * D + ((db ^ (lr & (kDB - 1))) * 16 + 4 * lg)) = o[db];
      __syncthreads();
      T* const out = static_cast<T*>(a.out) + ((int64_t)b * a.heads + h0) * D;
      float* const part = a.part + ((int64_t)blockIdx.x * 2 + (blockIdx.x == part_first ? 1 : 0)) * part_floats<D>();
      for (int i = tid; i < queries * kColumns; i += kThreads) {
        const int qi = i / kColumns, c = i % kColumns;
        Weighed w;
#pragma unroll
        for (int v = 0; v < kWaves; ++v)
          add_weighed(w, s_stats[v][qi][0], s_stats[v][qi][1],
                      *reinterpret_cast<const float4_t*>(reinterpret_cast<const float*>(smem + v * kStages * kStage) + qi * D +
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
      if (parts > 1) {
        wait_vmem_all();
        __syncthreads();
        if (tid == 0) s_last = arrive(word, a.tag, (unsigned)parts);
        __syncthreads();
        if (s_last) {
          // The parts lie in the second room of the first workgroup and in the first rooms of the others.  kBatch of them are on their way at a
          // time, and where an item has few queries several threads share the parts of a column.
          constexpr int kBatch = 8;
          constexpr unsigned kPitch = 2 * part_floats<D>() * 4, kSecond = part_floats<D>() * 4;
          const float* const from = a.part + (int64_t)part_first * 2 * part_floats<D>();
          const int units = queries * kColumns;
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
          }
        }
      }
      __syncthreads();   // the room is the next item's
    }
    before += of_sequence;
  }
}

int blocks_of_group(int64_t heads, int64_t kv_heads) { return (int)((heads / kv_heads + kQueries - 1) / kQueries); }
size_t part_bytes(int64_t D) { return (size_t)resident((int)D) * 2 * kQueries * (size_t)(D + 2) * sizeof(float); }

template <typename T, int D>
int launch_decode_paged(const DecodeArgs& a, hipStream_t st) {
  auto kern = flash_decode_paged_kernel<T, D>;
  constexpr int lds = kStages * kWaves * tile_bytes(D);
  TFK_LDS_OPT_IN(kern, lds);
  // (blocks that there can be: a launch of a few sequences with short tables asks for no more workgroups than those)
  const int64_t most = (int64_t)a.sequences * a.kv_heads * a.blocks_of_group * (((int64_t)a.table.width * a.table.page.d + kBlockKeys - 1) / kBlockKeys);
  return launch_kernel(kern, dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(most, resident(D)))), dim3(kThreads), lds, st, a);
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
  TFK_REQUIRE(softmax_scale == softmax_scale && softmax_scale - softmax_scale == 0.0, TF_ERR_INVALID_ARG, "%s: softmax_scale must be finite", who);
  if (cache->sequences == 0) return TF_OK;
  TFK_REQUIRE(cache->table_width < (1ll << 31) / cache->page_size &&
                  cache->sequences * (cache->table_width * cache->page_size / kBlockKeys + 1) <
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
