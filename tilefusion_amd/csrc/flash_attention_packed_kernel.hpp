// Attention over packed sequences, causal or not, with grouped heads: O = softmax(scale Q K^T) V for the rows of one
// sequence and one head of keys at a time, in a source file per head dimension.
//
// The matrix products, tiles and schedule are those of flash_attention.hpp (S^T = K Q^T and O^T = V^T P^T, keys and values in a ring of tiles of
// 64 in LDS, two sets of wavefronts half a tile apart).  Of its own it has
//   * rows that are the heads of a group of one token after the other (packed_sequences.hpp), and tiles that the device deals out;
//   * scores that are scaled in fp32, and weights that are summed in fp32 before they are rounded for the product: the log-sum-exp leaves in
//     fp32 for the backward pass, and a rounding of scaled queries, or a sum of rounded weights, would put 2^-9 (bf16) into it;
//   * weights that enter the product as one number of the type, which half a step each puts into the result: 2.0e-3 from 64 bits in bf16 (relative, over the
//     tensor), 1.6e-3 of them the result's own rounding, and 2.2e-4 against 1.9e-4 in fp16.  A number and its remainder, as decoding over pages has
//     it, whose products are free beside its loads, would be half as many matrix instructions again where those are what bounds;
//   * rows without a key (more queries than keys), which are zero;
//   * infinities and NaN among the values of a tile that is masked in part reach the rows that see them and no others.
// A fragment's address is the first one's, exclusive or a constant, which leaves the registers that masked tiles need.  Bound by the products with the exponentials beside them
// on long sequences (one of 8192, 32/8 heads x 128, bf16: 448 to 469 us, 1.2 PFLOP/s, as the board's clock is), by what a workgroup takes to begin and end, 8 us, on ragged ones
// (14 of 64 to 4001: 257 to 269 us).
#pragma once

#include "flash_attention.hpp"
#include "flash_attention_packed.hpp"

namespace tfk {
namespace {

// One in the sign's place of each 16-bit half that is an infinity or a NaN: an exponent of ones, into which one more carries.
template <typename T>
TFK_DEVICE unsigned not_finite(unsigned two) {
  return ((two & 0x7fff7fffu) + (std::is_same_v<T, bf16_t> ? 0x00800080u : 0x04000400u)) & 0x80008000u;
}

// kWavesT wavefronts x 16 * kQB rows per workgroup.
template <typename T, int D, bool kCausal, int kWavesT, int kQB>
__global__ __launch_bounds__(kWavesT * 64, 1) void flash_attention_packed_kernel(const T* __restrict__ Q, const T* __restrict__ K,
                                                                                 const T* __restrict__ V, T* __restrict__ O, float scale_log2,
                                                                                 PackedArgs a) {
  using V2 = typename Vec<T>::v2;
  using V4 = typename Vec<T>::v4;
  using V8 = typename Vec<T>::v8;
  constexpr int kBN = 64, kStages = ring_stages(kWavesT, D);
  constexpr int kRowsPerWave = 16 * kQB, kBM = kWavesT * kRowsPerWave;
  constexpr int kChunks = D / 8, kRowsPerInstr = 64 / kChunks;   // 16-byte pieces of a row; rows of a 1 KiB request
  constexpr int kTileBytes = kBN * D * 2, kStageBytes = 2 * kTileBytes;
  constexpr int kKB = kBN / 16, kKK = D / 32, kDB = D / 16, kJ = kBN / 32;
  constexpr int kPerWave = kTileBytes / 1024 / kWavesT, kLoadsPerTile = 2 * kPerWave;   // requests of a wavefront: keys, then values
  static_assert(kPerWave * kWavesT * 1024 == kTileBytes, "");
  extern __shared__ __attribute__((aligned(1024))) char smem[];

  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  rows_outside(a.offsets, a.sequences, a.tokens, (int)blockIdx.x, (int)gridDim.x, [&](int row) {
    clear_row(O + (size_t)row * a.heads * D, a.heads * D);
    if (!a.lse) return;
    for (int h = tid; h < a.heads; h += kWavesT * 64) a.lse[(size_t)h * a.tokens + row] = -INFINITY;
  });
  const PackedTile tile = packed_tile(a, kBM, (int)blockIdx.x / a.kv_heads);
  if (tile.sequence < 0) return;
  // Neighbours in the grid, which run on different XCDs, are of different heads of keys: with 8 of them the tiles of a
  // sequence that read the same keys read them from one L2.
  const int head = (int)blockIdx.x % a.kv_heads, group = (int)a.group.d;
  const int Lkv = tile.lkv, shift = tile.lkv - tile.lq, rows = tile.lq * group;
  // Causal tiles end at the last row, in 64s: the tile that is not full is the one with the fewest keys.  Rows in front of the first are none.
  const int tile_row0 = kCausal ? (rows + 63) / 64 * 64 - (tile.from_end + 1) * kBM : ((rows + kBM - 1) / kBM - 1 - tile.from_end) * kBM;
  const int q_row0 = tile_row0 + wave * kRowsPerWave;
  Q += (size_t)tile.q0 * a.query_row + head * a.query_group;
  K += (size_t)tile.k0 * a.key_row + head * a.key_head;
  V += (size_t)tile.k0 * a.value_row + head * a.value_head;
  const size_t o_row = (size_t)a.heads * D;
  O += tile.q0 * o_row + (size_t)head * group * D;
  float* const lse = a.lse ? a.lse + (size_t)head * group * a.tokens + tile.q0 : nullptr;

  // the last key that a row sees, -1 in front of the first
  auto limit_of = [&](int row) __attribute__((always_inline)) {
    return kCausal ? min(Lkv - 1, divide(a.group, min(max(row, 0), rows - 1)) + shift) : Lkv - 1;
  };
  const int n_end = limit_of(tile_row0 + kBM - 1) + 1;
  if (n_end <= 0) {   // no row of the tile has a key
    for (int i = tid; i < kBM * kChunks; i += kWavesT * 64) {
      const int row = tile_row0 + i / kChunks;
      if ((unsigned)row >= (unsigned)rows) continue;
      const int token = divide(a.group, row), g = row - token * group;
      *reinterpret_cast<V8*>(O + token * o_row + g * D + i % kChunks * 8) = V8{};
      if (lse && i % kChunks == 0) lse[(size_t)g * a.tokens + token] = -INFINITY;
    }
    return;
  }
  const int num_tiles = (n_end + kBN - 1) / kBN;

  // ---- Q^T fragments (B operand): lane holds Q[row][32*kk + 8*lg .. +7] ----------------------
  V8 qf[kKK][kQB];
  int limit[kQB];
#pragma unroll
  for (int qb = 0; qb < kQB; ++qb) {
    const int row = min(max(q_row0 + 16 * qb + lr, 0), rows - 1), token = divide(a.group, row);
    limit[qb] = kCausal ? min(Lkv - 1, token + shift) : Lkv - 1;
    const T* q = Q + (size_t)token * a.query_row + (size_t)(row - token * group) * a.query_head;
#pragma unroll
    for (int kk = 0; kk < kKK; ++kk) qf[kk][qb] = *reinterpret_cast<const V8*>(q + kk * 32 + lg * 8);
  }

  // ---- global -> LDS: request r of a wavefront is 1 KiB of a tile of keys (r < kPerWave) or values ----
  const unsigned smem_base = lds_address(smem);
  unsigned req_off[kLoadsPerTile];   // per-lane byte offset inside the tile in memory
#pragma unroll
  for (int t = 0; t < kPerWave; ++t) {
    const int row = (wave + kWavesT * t) * kRowsPerInstr + lane / kChunks;
    req_off[t] = (unsigned)(row * a.key_row + swz_k<kChunks>(row, lane % kChunks) * 8) * 2u;
    req_off[kPerWave + t] = (unsigned)(row * a.value_row + swz_v<kChunks>(row, lane % kChunks) * 8) * 2u;
  }
  auto destination = [&](int tile_no, int r) __attribute__((always_inline)) {
    return smem_base + (tile_no % kStages) * kStageBytes + (r < kPerWave ? 0 : kTileBytes) + (wave + kWavesT * (r % kPerWave)) * 1024;
  };
  // a whole tile within the keys
  auto issue_request_lean = [&](int tile_no, int r) __attribute__((always_inline)) {
    const char* base = r < kPerWave ? reinterpret_cast<const char*>(K) + (size_t)tile_no * (size_t)(kBN * 2 * a.key_row)
                                    : reinterpret_cast<const char*>(V) + (size_t)tile_no * (size_t)(kBN * 2 * a.value_row);
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(req_off[r]), "s"(base), "{m0}"(destination(tile_no, r)) : "memory");
  };
  // any tile: past the last one that is needed it is that one again, rows behind the last key are the last key's
  auto issue_request = [&](int tile_no, int r) __attribute__((always_inline)) {
    const int n0 = min(tile_no, num_tiles - 1) * kBN;
    const int row = (wave + kWavesT * (r % kPerWave)) * kRowsPerInstr + lane / kChunks;
    const size_t at = min(n0 + row, Lkv - 1);
    const T* from = r < kPerWave ? K + at * a.key_row + swz_k<kChunks>(row, lane % kChunks) * 8
                                 : V + at * a.value_row + swz_v<kChunks>(row, lane % kChunks) * 8;
    lds_dma_16B(from, destination(tile_no, r));
  };
  auto issue_tile_loads = [&](int tile_no) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < kLoadsPerTile; ++r) issue_request(tile_no, r);
  };

  // ---- LDS -> registers (see flash_attention.hpp for which lane holds what) ------------------
  // (a swizzle is an exclusive or of chunk numbers: kk and db are one more of the address of the first)
  const int v_row = 4 * lg + (lr >> 2), v_col = 4 * (lr & 3);
  const unsigned k_off = lr * D * 2 + swz_k<kChunks>(lr, lg) * 16;
  const unsigned v_off = v_row * D * 2 + swz_v<kChunks>(v_row, v_col / 8) * 16 + (v_col % 8) * 2 + kTileBytes;
  float4_t o_acc[kDB][kQB];
  float neg_m[kQB], l_sum[kQB];   // minus a row's reference; this lane's part of its weights' sum
  bool unset[kQB];                // no score above -inf seen yet
#pragma unroll
  for (int qb = 0; qb < kQB; ++qb) {
    unset[qb] = true;
    neg_m[qb] = l_sum[qb] = 0.f;
#pragma unroll
    for (int db = 0; db < kDB; ++db) o_acc[db][qb] = float4_t{0.f, 0.f, 0.f, 0.f};
  }
  float4_t s[kKB][kQB];
  V8 kf[2][kKB];   // K fragments of reduction step kk (buffer kk & 1)
  V8 vf[kJ][kDB];  // V fragments of reduction step j
  V8 pb[kJ][kQB];  // weights, B operand of the second product
  auto stage_of = [&](int it) __attribute__((always_inline)) { return smem_base + (it % kStages) * kStageBytes; };
  auto k_reads = [&](int buf, int it, int kk) __attribute__((always_inline)) {
    const unsigned ka = opaque((stage_of(it) + k_off) ^ (kk << 6));
#pragma unroll
    for (int kb = 0; kb < kKB; ++kb) kf[buf][kb] = lds_read_b128<V8>(ka + kb * 16 * D * 2);
  };
  auto v_frag = [&](unsigned va, int j) __attribute__((always_inline)) {
    const V4 lo = lds_read_tr4<V4>(va + (32 * j) * D * 2), hi = lds_read_tr4<V4>(va + (32 * j + 16) * D * 2);
    V8 f;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f[t] = lo[t];
      f[4 + t] = hi[t];
    }
    return f;
  };
  auto v_reads = [&](int it, int j) __attribute__((always_inline)) {
#pragma unroll
    for (int db = 0; db < kDB; ++db) vf[j][db] = v_frag(opaque((stage_of(it) + v_off) ^ (db << 5)), j);
  };
  // S^T = K Q^T; the fragments of step 0 are on their way.  req_tile >= 0: its requests go out between the products.
  auto qk_tile = [&](int it, int req_tile, auto lean_c) __attribute__((always_inline)) {
#pragma unroll
    for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
      for (int qb = 0; qb < kQB; ++qb) s[kb][qb] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < kKK; ++kk) {
      const unsigned ka = kk + 1 < kKK ? opaque((stage_of(it) + k_off) ^ ((kk + 1) << 6)) : 0u;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kb = 0; kb < kKB; ++kb) {
#pragma unroll
        for (int qb = 0; qb < kQB; ++qb) s[kb][qb] = mfma_t<T>(kf[kk & 1][kb], qf[kk][qb], s[kb][qb]);
        if (kk + 1 < kKK) kf[(kk + 1) & 1][kb] = lds_read_b128<V8>(ka + kb * 16 * D * 2);
#pragma unroll
        for (int r = 0; r < kLoadsPerTile; ++r)
          if ((r * kKK * kKB) / kLoadsPerTile == kk * kKB + kb) {
            if constexpr (decltype(lean_c)::value) issue_request_lean(req_tile, r);
            else issue_request(req_tile, r);
          }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  auto softmax_tile = [&](int it, auto mask_c) __attribute__((always_inline)) {
    v_reads(it, 0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
      for (int qb = 0; qb < kQB; ++qb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[kb][qb][r] = fmaf(s[kb][qb][r], scale_log2, neg_m[qb]);
          if constexpr (decltype(mask_c)::value)
            if (it * kBN + kb * 16 + 4 * lg + r > limit[qb]) s[kb][qb][r] = -INFINITY;
        }
    // The reference is set 2^kUp below the largest score and raised when some score is more than kLazy (log2 units) above it; weights reach 2^kLazy until
    // then.  In fp16, whose smallest number is 2^-24, a weight's smallest step is so 2^-31 of the largest weight or less; bf16 has the range.
    constexpr float kUp = std::is_same_v<T, bf16_t> ? 0.f : 7.f, kLazy = kUp + 8.f;
    float mx[kQB];
    bool grow = false;
#pragma unroll
    for (int qb = 0; qb < kQB; ++qb) {
      mx[qb] = s[0][qb][0];
#pragma unroll
      for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx[qb] = fmaxf(mx[qb], s[kb][qb][r]);
      grow |= mx[qb] > kLazy || unset[qb];
    }
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
#pragma unroll
      for (int qb = 0; qb < kQB; ++qb) {
        const float qmax = quad_max(mx[qb]);
        float shift_m = unset[qb] ? qmax - kUp : fmaxf(0.f, qmax - kUp);
        const float alpha = unset[qb] ? 1.f : __builtin_amdgcn_exp2f(-shift_m);
        if (unset[qb] && qmax == -INFINITY) shift_m = 0.f;
        else unset[qb] = false;
        l_sum[qb] *= alpha;
#pragma unroll
        for (int db = 0; db < kDB; ++db) o_acc[db][qb] *= alpha;
#pragma unroll
        for (int kb = 0; kb < kKB; ++kb) s[kb][qb] -= shift_m;
        neg_m[qb] -= shift_m;
      }
    }
#pragma unroll
    for (int qb = 0; qb < kQB; ++qb) {
#pragma unroll
      for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[kb][qb][r] = __builtin_amdgcn_exp2f(s[kb][qb][r]);
      float4_t sum = s[0][qb];
#pragma unroll
      for (int kb = 1; kb < kKB; ++kb) sum += s[kb][qb];
      l_sum[qb] += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
      for (int j = 0; j < kJ; ++j)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          pb[j][qb][t] = (T)s[2 * j][qb][t];
          pb[j][qb][4 + t] = (T)s[2 * j + 1][qb][t];
        }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // O^T += V^T P^T; the K fragments of the next tile's first step are requested during the last step.
  // clean: zeros in the place of values that are not finite.
  auto pv_tile = [&](int it, int it_next, bool clean) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      if (j + 1 < kJ) v_reads(it, j + 1);
      else k_reads(0, it_next, 0);
      if (clean) {
#pragma unroll
        for (int db = 0; db < kDB; ++db) {
          uint4_t x = __builtin_bit_cast(uint4_t, vf[j][db]);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] &= ~((not_finite<T>(x[e]) >> 15) * 0xffffu);
          vf[j][db] = __builtin_bit_cast(V8, x);
        }
      }
#pragma unroll
      for (int db = 0; db < kDB; ++db)
#pragma unroll
        for (int qb = 0; qb < kQB; ++qb) o_acc[db][qb] = mfma_t<T>(vf[j][db], pb[j][qb], o_acc[db][qb]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // A value that is not finite, in a tile that is masked in part: it goes to the rows that see it one by one, and is zero in the
  // product, where a weight of zero would make a NaN of it for the rows that do not.
  auto add_not_finite = [&](int it) __attribute__((always_inline)) {
    const unsigned at = stage_of(it) + kTileBytes + lane * 16;
    for (int i = 0; i < kTileBytes / 1024; ++i) {
      const uint4_t x = lds_read_b128<uint4_t>(at + i * 1024);
      unsigned mine = 0;   // a bit for each of the eight
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned bits = not_finite<T>(x[e]);
        mine |= ((bits >> 15 & 1u) | (bits >> 30 & 2u)) << (2 * e);
      }
      for (;;) {
        const unsigned long long lanes = __builtin_amdgcn_ballot_w64(mine != 0);
        if (lanes == 0) break;
        const int from = __builtin_ctzll(lanes), e = __builtin_ctz(__builtin_amdgcn_readlane(mine, from));
        const unsigned pair = e < 4 ? (e < 2 ? x[0] : x[1]) : (e < 6 ? x[2] : x[3]);
        const unsigned short bits = (unsigned short)(__builtin_amdgcn_readlane(pair, from) >> (e % 2 * 16));
        const float value = (float)__builtin_bit_cast(T, bits);
        const int row = i * kRowsPerInstr + from / kChunks, col = swz_v<kChunks>(row, from % kChunks) * 8 + e;
#pragma unroll
        for (int qb = 0; qb < kQB; ++qb) {
          const float to_row = it * kBN + row <= limit[qb] ? value : 0.f;
#pragma unroll
          for (int db = 0; db < kDB; ++db)
#pragma unroll
            for (int r = 0; r < 4; ++r) o_acc[db][qb][r] += 16 * db + 4 * lg + r == col ? to_row : 0.f;
        }
        if (lane == from) mine &= mine - 1;
      }
    }
  };
  auto pv = [&](int it, auto mask_c) __attribute__((always_inline)) {
    bool found = false;
    if constexpr (decltype(mask_c)::value) {
      unsigned seen = 0;
#pragma unroll
      for (int i = 0; i < kTileBytes / 1024; ++i) {
        const uint4_t x = lds_read_b128<uint4_t>(stage_of(it) + kTileBytes + lane * 16 + i * 1024);
#pragma unroll
        for (int e = 0; e < 4; ++e) seen |= not_finite<T>(x[e]);
      }
      found = __builtin_amdgcn_ballot_w64(seen != 0) != 0;
      if (found) add_not_finite(it);
    }
    pv_tile(it, it + 1, found);
  };
  // Q is waited for here, and not at its first use among the tiles (where the wait would drain the requests ahead)
  auto q_is_there = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int kk = 0; kk < kKK; ++kk)
#pragma unroll
      for (int qb = 0; qb < kQB; ++qb) asm volatile("" : "+v"(qf[kk][qb]));
  };

  // Tiles [0, n_plain) need no mask for this wavefront's rows, those from n_compute on have nothing for it: it only keeps the ring going.
  int n_plain = n_end / kBN, n_compute = num_tiles;
  if (kCausal) {
    n_plain = max(0, min(n_plain, (__builtin_amdgcn_readfirstlane(limit_of(q_row0)) + 1) / kBN));
    const int last = __builtin_amdgcn_readfirstlane(limit_of(q_row0 + kRowsPerWave - 1));
    n_compute = last < 0 ? 0 : last / kBN + 1;
  }
  if (q_row0 + kRowsPerWave <= 0 || q_row0 >= rows) n_plain = n_compute = 0;   // (all rows in front of the first or behind the last)
  const int n_fast = min(num_tiles, Lkv / kBN);   // whole tiles (lean request form)
  if constexpr (kWavesT == 8) {
#pragma unroll
    for (int t = 0; t < 3; ++t) issue_tile_loads(t);
    barrier_keep_vmem<2 * kLoadsPerTile>();   // tile 0 has landed
    q_is_there();
    const bool second_set = wave >= 4;
    if (second_set) barrier_only();   // slot 0: set 0 alone
    k_reads(0, 0, 0);
    if (n_compute > 0) qk_tile(0, 3, std::false_type{});
    else issue_tile_loads(3);
    auto tile_step = [&](int t, auto mask_c, auto lean_c) __attribute__((always_inline)) {
      barrier_keep_vmem<2 * kLoadsPerTile>();   // tile t+1 has landed
      softmax_tile(t, mask_c);
      barrier_only();
      __builtin_amdgcn_s_setprio(2);
      pv(t, mask_c);
      if (t + 1 < n_compute) qk_tile(t + 1, t + 4, lean_c);
      else issue_tile_loads(t + 4);
      __builtin_amdgcn_s_setprio(0);
    };
    const int n_lean = min(min(n_plain, n_compute - 1), n_fast - 4);
    int t = 0;
    for (; t < n_lean; ++t) tile_step(t, std::false_type{}, std::true_type{});
    for (; t < n_plain; ++t) tile_step(t, std::false_type{}, std::false_type{});
    for (; t < n_compute; ++t) tile_step(t, std::true_type{}, std::false_type{});
    for (; t < num_tiles; ++t) {
      barrier_keep_vmem<2 * kLoadsPerTile>();
      barrier_only();
      issue_tile_loads(t + 4);
    }
    if (!second_set) barrier_only();   // the slot in which set 1 finishes its last tile
  } else {
#pragma unroll
    for (int t = 0; t < kStages - 1; ++t) issue_tile_loads(t);
    barrier_keep_vmem<(kStages - 2) * kLoadsPerTile>();   // tile 0 has landed
    q_is_there();
    auto tile_step = [&](int t, auto mask_c, auto lean_c) __attribute__((always_inline)) {
      barrier_keep_vmem<(kStages - 3) * kLoadsPerTile>();
      qk_tile(t, t + kStages - 1, lean_c);
      softmax_tile(t, mask_c);
      pv(t, mask_c);
    };
    const int n_lean = min(n_plain, n_fast - (kStages - 1));
    int t = 0;
    k_reads(0, 0, 0);
    for (; t < n_lean; ++t) tile_step(t, std::false_type{}, std::true_type{});
    for (; t < n_plain; ++t) tile_step(t, std::false_type{}, std::false_type{});
    for (; t < n_compute; ++t) tile_step(t, std::true_type{}, std::false_type{});
    for (; t < num_tiles; ++t) {
      barrier_keep_vmem<(kStages - 3) * kLoadsPerTile>();
      issue_tile_loads(t + kStages - 1);
    }
  }
  wait_vmem_all();   // the requests past the last tile must not outlive the workgroup's LDS

  // ---- O[row][16*db + 4*lg + r] = O^T / l, re-dealt so that four adjacent lanes store 64 contiguous bytes of a row ----
  const int st_row = lane >> 2, st_seg = lane & 3, src_lane = st_row + 16 * (((st_seg & 1) << 1) | (st_seg >> 1));
#pragma unroll
  for (int qb = 0; qb < kQB; ++qb) {
    float l = l_sum[qb];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int own = q_row0 + 16 * qb + lr;
    if (lse && lg == 0 && (unsigned)own < (unsigned)rows) {
      const int token = divide(a.group, own);
      lse[(size_t)(own - token * group) * a.tokens + token] = l == 0.f ? -INFINITY : (__builtin_amdgcn_logf(l) - neg_m[qb]) * 0.6931471805599453f;
    }
    const int row = q_row0 + 16 * qb + st_row;   // the row this lane stores
    const bool there = (unsigned)row < (unsigned)rows;
    const int token = divide(a.group, there ? row : 0), g = (there ? row : 0) - token * group;
    T* o_lane = O + token * o_row + g * D + 8 * st_seg;
#pragma unroll
    for (int db = 0; db < kDB; db += 2) {
      unsigned x[2], y[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const V2 hx = {(T)(o_acc[db][qb][2 * h] * inv), (T)(o_acc[db][qb][2 * h + 1] * inv)};
        const V2 hy = {(T)(o_acc[db + 1][qb][2 * h] * inv), (T)(o_acc[db + 1][qb][2 * h + 1] * inv)};
        x[h] = __builtin_bit_cast(unsigned, hx);
        y[h] = __builtin_bit_cast(unsigned, hy);
#if defined(__HIP_DEVICE_COMPILE__)
        auto sw = __builtin_amdgcn_permlane16_swap(x[h], y[h], false, false);   // x of the odd groups <-> y of the even groups
        x[h] = sw[0];
        y[h] = sw[1];
#endif
      }
      uint4_t v;
      v[0] = (unsigned)__builtin_amdgcn_ds_bpermute(4 * src_lane, (int)x[0]);
      v[1] = (unsigned)__builtin_amdgcn_ds_bpermute(4 * src_lane, (int)x[1]);
      v[2] = (unsigned)__builtin_amdgcn_ds_bpermute(4 * src_lane, (int)y[0]);
      v[3] = (unsigned)__builtin_amdgcn_ds_bpermute(4 * src_lane, (int)y[1]);
      if (there) *reinterpret_cast<uint4_t*>(o_lane + 16 * db) = v;
    }
  }
}

template <typename T, int D, bool kCausal, int kWavesT, int kQB>
int launch_packed(const PackedCall& c) {
  auto kern = flash_attention_packed_kernel<T, D, kCausal, kWavesT, kQB>;
  constexpr int lds = ring_stages(kWavesT, D) * 2 * 64 * D * 2;
  static_assert(lds <= kMaxLdsBytes, "tiles do not fit in LDS");
  TFK_LDS_OPT_IN(kern, lds);
  const int64_t tiles = most_tiles((int64_t)c.args.tokens * c.args.group.d, c.args.sequences, 16 * kQB * kWavesT) * c.args.kv_heads;
  // (tokens of no sequence are cleared by whatever workgroups there are)
  return launch_kernel(kern, dim3((unsigned)std::max<int64_t>(tiles, 1)), dim3(kWavesT * 64), lds, c.stream, static_cast<const T*>(c.query),
                       static_cast<const T*>(c.key), static_cast<const T*>(c.value), static_cast<T*>(c.out), c.scale_log2, c.args);
}
template <typename T, int D, bool kCausal>
int launch_packed_rows(const PackedCall& c) {
  if (c.rows == 256) return launch_packed<T, D, kCausal, 8, 2>(c);
  if (c.rows == 128) return launch_packed<T, D, kCausal, 8, 1>(c);
  return launch_packed<T, D, kCausal, 4, 1>(c);
}
template <int D>
int run_packed(const PackedCall& c) {
  if (c.bf16) return c.causal ? launch_packed_rows<bf16_t, D, true>(c) : launch_packed_rows<bf16_t, D, false>(c);
  return c.causal ? launch_packed_rows<half_t, D, true>(c) : launch_packed_rows<half_t, D, false>(c);
}

}  // namespace
}  // namespace tfk
