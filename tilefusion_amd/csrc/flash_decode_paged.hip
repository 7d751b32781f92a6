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
//   * A wavefront takes every kWaves-th 32 keys of the range and shares nothing with the others up to the end of an item: tiles of K and V go
//     from their pages to LDS directly, two tiles deep, and are waited for by count, with no barrier.
//   * Pages are whole 16-key blocks: a block's page is looked up with scalar loads, a tile ahead, and the lanes' offsets
//     within a block are constants of the launch.
#include <algorithm>

#include "flash_attention.hpp"
#include "paged_cache.hpp"

namespace tfk {
namespace {

constexpr int kWaves = 4, kTileKeys = 32, kBlockKeys = kWaves * kTileKeys;
constexpr int kQueries = 16;   // of an item: one block of MFMA columns
// Workgroups of a launch: those that LDS lets run at once.
__host__ __device__ constexpr int tile_bytes(int d) { return 2 * kTileKeys * d * 2; }
__host__ __device__ constexpr int resident(int d) { return kCUs * (kMaxLdsBytes / (2 * kWaves * tile_bytes(d))); }

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

template <typename T, int D>
__global__ __launch_bounds__(kWaves * kWaveSize, 1) void flash_decode_paged_kernel(DecodeArgs a) {
  using V4 = typename Vec<T>::v4;
  using V8 = typename Vec<T>::v8;
  constexpr int kChunks = D / 8, kRowsPerLoad = kWaveSize / kChunks;   // 16-byte pieces of a row; rows of one load
  constexpr int kLoads = kTileKeys / kRowsPerLoad, kLoadsPer16 = kLoads / 2;   // ... of a tile's keys, as of its values
  constexpr int kKK = D / 32, kDB = D / 16;
  constexpr int kKeyBytes = kTileKeys * D * 2, kStage = tile_bytes(D), kStages = 2;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  __shared__ float s_stats[kWaves][kQueries][2];
  __shared__ bool s_last;

  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int items_of = a.kv_heads * a.blocks_of_group;   // of a sequence

  // ---- this workgroup's range of blocks ---------------------------------------------------------
  int total = 0;
  for (int b0 = 0; b0 < a.sequences; b0 += kWaveSize) total += b0 + lane < a.sequences ? blocks_of(keys_of(a, a.lengths[b0 + lane])) : 0;
  total = __builtin_amdgcn_readlane(wave_prefix(total), 63);
  const long long blocks = (long long)total * items_of;
  // (no more workgroups than blocks)
  const int groups = (int)min((long long)gridDim.x, blocks);
  // sequences without a key, and those that the table cannot hold
  for (int b = blockIdx.x; b < a.sequences; b += gridDim.x) {
    const int n = keys_of(a, read_uniform(a.lengths + b));
    if (n > 0) continue;
    const float v = n < 0 ? __builtin_nanf("") : 0.f;
    for (int i = tid; i < a.heads * D; i += kWaves * kWaveSize) static_cast<T*>(a.out)[(int64_t)b * a.heads * D + i] = (T)v;
  }
  if ((int)blockIdx.x >= groups) return;
  const long long begin = blocks * blockIdx.x / groups, end = blocks * (blockIdx.x + 1) / groups;
  // the sequence in which the range begins
  int b = 0;
  long long before = 0;   // blocks of the sequences in front of it
  for (int b0 = 0; b0 < a.sequences; b0 += kWaveSize) {
    const int own = b0 + lane < a.sequences ? blocks_of(keys_of(a, a.lengths[b0 + lane])) : 0;
    const int up_to = wave_prefix(own);
    const bool passed = before + (long long)up_to * items_of <= begin;
    const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(passed));
    b = b0 + n;
    if (n == kWaveSize) {
      before += (long long)__builtin_amdgcn_readlane(up_to, 63) * items_of;
      continue;
    }
    if (n > 0) before += (long long)__builtin_amdgcn_readlane(up_to, n - 1) * items_of;
    break;
  }

  // ---- LDS: where loads leave their rows and fragments find them ------------------------------
  const unsigned wave_base = lds_address(smem) + wave * kStages * kStage;
  unsigned key_off[kLoadsPer16], value_off[kLoadsPer16];   // bytes from a 16-key block's first row in memory
#pragma unroll
  for (int i = 0; i < kLoadsPer16; ++i) {
    const int row = i * kRowsPerLoad + lane / kChunks;
    key_off[i] = (unsigned)(row * (int)a.key_strides[1] + swz_k<kChunks>(row, lane % kChunks) * 8) * 2u;
    value_off[i] = (unsigned)(row * (int)a.value_strides[1] + swz_v<kChunks>(row, lane % kChunks) * 8) * 2u;
  }
  unsigned k_at[kKK], v_at[kDB];
#pragma unroll
  for (int kk = 0; kk < kKK; ++kk) k_at[kk] = lr * D * 2 + swz_k<kChunks>(lr, 4 * kk + lg) * 16;
#pragma unroll
  for (int db = 0; db < kDB; ++db) {
    const int row = 4 * lg + (lr >> 2), col = db * 16 + 4 * (lr & 3);
    v_at[db] = kKeyBytes + row * D * 2 + swz_v<kChunks>(row, col / 8) * 16 + (col % 8) * 2;
  }

  for (long long at = begin; at < end; ++b) {
    const int keys = keys_of(a, read_uniform(a.lengths + b));
    const int of_item = blocks_of(keys);
    const long long of_sequence = (long long)of_item * items_of;
    while (at < end && at < before + of_sequence) {
      // ---- one item, or what of it is in the range: blocks [first, last) --------------------
      const int item = (int)((at - before) / of_item);
      const long long item_begin = before + (long long)item * of_item;
      const int first = (int)(at - item_begin), last = (int)min((long long)of_item, end - item_begin);
      at = item_begin + last;
      const int head = item / a.blocks_of_group, query0 = item % a.blocks_of_group * kQueries;
      const int queries = min(kQueries, a.group - query0);
      const int h0 = head * a.group + query0;
      const int item_id = b * items_of + item;
      // the workgroups that have a part of it
      const long long part_first = ((item_begin + 1) * groups - 1) / blocks, part_last = ((item_begin + of_item) * groups - 1) / blocks;
      const int parts = (int)(part_last - part_first) + 1;
      if (parts > 1 && tid == 0 && blockIdx.x == part_first) open_arrivals(a.arrivals + (int64_t)item_id * kArrivalsPitch, a.tag);

      V8 qf[kKK];
      const T* q = static_cast<const T*>(a.query) + b * a.query_token + (h0 + min(lr, queries - 1)) * a.query_head;
#pragma unroll
      for (int kk = 0; kk < kKK; ++kk) qf[kk] = *reinterpret_cast<const V8*>(q + 32 * kk + 8 * lg);
#pragma unroll
      for (int kk = 0; kk < kKK; ++kk) asm volatile("" : "+v"(qf[kk]));   // (waited for here, not among the tiles)

      const int tile_end = last * kWaves, last16 = (keys - 1) / 16;
      bool lost = false;   // a page that the cache does not have
      const T* const keys_at = static_cast<const T*>(a.key) + head * a.key_strides[2];
      const T* const values_at = static_cast<const T*>(a.value) + head * a.value_strides[2];
      auto request = [&](int tile, int stage) __attribute__((always_inline)) {
        const unsigned dst = wave_base + stage * kStage;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int key0 = min(2 * tile + h, last16) * 16;
          int page = page_of(a.table, b, key0);
          lost |= page < 0;
          page = max(page, 0);
          const int row = key0 - divide(a.table.page, key0) * (int)a.table.page.d;
          const T* k = keys_at + page * a.key_strides[0] + row * a.key_strides[1];
          const T* v = values_at + page * a.value_strides[0] + row * a.value_strides[1];
#pragma unroll
          for (int i = 0; i < kLoadsPer16; ++i) {
            asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(key_off[i]), "s"(k), "{m0}"(dst + (h * kLoadsPer16 + i) * 1024) : "memory");
          }
#pragma unroll
          for (int i = 0; i < kLoadsPer16; ++i) {
            asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                         : : "v"(value_off[i]), "s"(v), "{m0}"(dst + kKeyBytes + (h * kLoadsPer16 + i) * 1024) : "memory");
          }
        }
      };

      float4_t o[kDB];
#pragma unroll
      for (int db = 0; db < kDB; ++db) o[db] = float4_t{0.f, 0.f, 0.f, 0.f};
      // Weights are taken 2^kUp times as large in fp16 and enter the product as a number and its remainder: a weight's smallest remainder is
      // then 2^-31 of the largest weight.
      constexpr float kUp = std::is_same_v<T, bf16_t> ? 0.f : 7.f, kLazy = kUp + 8.f;
      float top = -INFINITY, sum = 0.f;   // reference of query lr; this lane's part of its weights' sum

      int tile = first * kWaves + wave;
      if (tile < tile_end) request(tile, 0);
      for (int n = 0; tile < tile_end; ++n, tile += kWaves) {
        const unsigned stage = wave_base + (n & 1) * kStage;
        if (tile + kWaves < tile_end) {
          request(tile + kWaves, (n + 1) & 1);
          wait_vmem<2 * kLoads>();
        } else {
          wait_vmem_all();
        }
        const int left = keys - tile * kTileKeys;   // keys of the tile; it may have none
        if (left < kTileKeys) {
          // rows behind the last key hold anything: their weight is zero, and zero times an infinity is none
          const V8 zeros = {};
#pragma unroll
          for (int i = 0; i < kLoads; ++i)
            if (i * kRowsPerLoad + lane / kChunks >= left)
              *(__attribute__((address_space(3))) V8*)(size_t)(stage + kKeyBytes + i * 1024 + lane * 16) = zeros;
        }
        float4_t s[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          s[kb] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kk = 0; kk < kKK; ++kk) s[kb] = mfma_t<T>(lds_read_b128<V8>(stage + k_at[kk] + kb * 16 * D * 2), qf[kk], s[kb]);
        }
        float big = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            s[kb][r] = 16 * kb + 4 * lg + r < left ? s[kb][r] * a.scale_log2 : -INFINITY;
            big = fmaxf(big, s[kb][r]);
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
        V8 p, rest;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float w = __builtin_amdgcn_exp2f(s[kb][r] - reference);
            sum += w;
            const SplitWeight<T> two = split_weight<T>(w);
            p[4 * kb + r] = two.whole;
            rest[4 * kb + r] = two.rest;
          }
#pragma unroll
        for (int db = 0; db < kDB; ++db) {
          const V4 lo = lds_read_tr4<V4>(stage + v_at[db]), hi = lds_read_tr4<V4>(stage + v_at[db] + 16 * D * 2);
          V8 vf;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            vf[t] = lo[t];
            vf[4 + t] = hi[t];
          }
          o[db] = mfma_t<T>(vf, p, o[db]);
          o[db] = mfma_t<T>(vf, rest, o[db]);
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
      const int64_t slot = ((int64_t)blockIdx.x * 2 + (blockIdx.x == part_first ? 1 : 0)) * part_floats<D>();
      for (int i = tid; i < queries * (D / 4); i += kWaves * kWaveSize) {
        const int qi = i / (D / 4), c = i % (D / 4);
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) m = fmaxf(m, s_stats[w][qi][0]);
        float l = 0.f;
        float4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const float f = s_stats[w][qi][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_stats[w][qi][0] - m);
          const float* rows = reinterpret_cast<const float*>(smem + w * kStages * kStage);
          acc += f * *reinterpret_cast<const float4_t*>(rows + qi * D + (((c / 4) ^ (qi & (kDB - 1))) * 16 + 4 * (c % 4)));
          const float own = s_stats[w][qi][1];
          l += own == 0.f ? 0.f : f * own;
        }
        if (parts == 1) {
          const float inv = l == 0.f ? 0.f : 1.f / l;
          V4 y;
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = (T)(acc[e] * inv);
          *reinterpret_cast<V4*>(static_cast<T*>(a.out) + ((int64_t)b * a.heads + h0 + qi) * D + 4 * c) = y;
        } else {
          float* to = a.part + slot;
#pragma unroll
          for (int e = 0; e < 4; ++e) store_shared(to + qi * D + 4 * c + e, acc[e]);
          if (c == 0) {
            store_shared(to + kQueries * D + 2 * qi, m);
            store_shared(to + kQueries * D + 2 * qi + 1, l);
          }
        }
      }
      if (parts > 1) {
        wait_vmem_all();
        __syncthreads();
        if (tid == 0) s_last = arrive(a.arrivals + (int64_t)item_id * kArrivalsPitch, a.tag, (unsigned)parts);
        __syncthreads();
        if (s_last) {
          // (a part's beginning: 16-byte pieces of the first workgroup's second room, then of the others' first)
          const unsigned pitch = 2 * part_floats<D>() * 4;
          const float* const from = a.part + part_first * 2 * part_floats<D>();
          for (int i = tid; i < queries * (D / 4); i += kWaves * kWaveSize) {
            const int qi = i / (D / 4), c = i % (D / 4);
            float m = -INFINITY;
            for (int s = 0; s < parts; ++s)
              m = fmaxf(m, load_shared(from + (int64_t)s * 2 * part_floats<D>() + (s == 0 ? part_floats<D>() : 0) + kQueries * D + 2 * qi));
            float l = 0.f;
            float4_t acc = {0.f, 0.f, 0.f, 0.f};
            for (int s = 0; s < parts; ++s) {
              const float* part = from + (int64_t)s * 2 * part_floats<D>() + (s == 0 ? part_floats<D>() : 0);
              const float pm = load_shared(part + kQueries * D + 2 * qi), pl = load_shared(part + kQueries * D + 2 * qi + 1);
              const float4_t x = load_shared_16B<float4_t>(from, s * pitch + ((s == 0 ? part_floats<D>() : 0) + qi * D + 4 * c) * 4);
              const float f = pm == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(pm - m);
              l += pl == 0.f ? 0.f : f * pl;
              acc += f * x;
            }
            const float inv = l == 0.f ? 0.f : 1.f / l;
            V4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = (T)(acc[e] * inv);
            *reinterpret_cast<V4*>(static_cast<T*>(a.out) + ((int64_t)b * a.heads + h0 + qi) * D + 4 * c) = y;
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
  constexpr int lds = 2 * kWaves * tile_bytes(D);
  TFK_LDS_OPT_IN(kern, lds);
  // (blocks that there can be: a launch of a few sequences with short tables asks for no more workgroups than those)
  const int64_t most = (int64_t)a.sequences * a.kv_heads * a.blocks_of_group * (((int64_t)a.table.width * a.table.page.d + kBlockKeys - 1) / kBlockKeys);
  return launch_kernel(kern, dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(most, resident(D)))), dim3(kWaves * kWaveSize), lds, st, a);
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
  TFK_REQUIRE(cache->table_width * cache->page_size < (1ll << 31) && cache->sequences * (cache->table_width * cache->page_size / kBlockKeys + 1) < (1ll << 31),
              TF_ERR_INVALID_ARG, "%s: the table holds more than 2^31 tokens a sequence, or 2^31 blocks of 128", who);
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
