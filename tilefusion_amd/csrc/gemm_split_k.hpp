// The main loop of the small matrix products: few rows, few columns or few tiles of A * B^T.  gemm.hip stores its results as they are; the
// kernels of product.hpp do more with them.
#pragma once

#include <type_traits>

#include "common.hpp"

namespace tfk {

using int4v_t = int __attribute__((ext_vector_type(4)));

// One k-step of 16-byte fragments: lane l supplies 16 bytes of row l % 16 of either operand (8 16-bit elements, 16 of 8 bits), the
// (l / 16)-th of the step.  Sums of 8-bit products are int32, in the same registers.
template <typename InT>
TFK_DEVICE float4_t mfma_rows(uint4_t a, uint4_t b, float4_t c) {
  if constexpr (std::is_same_v<InT, int8_t>) {
    return __builtin_bit_cast(float4_t, __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(int4v_t, b), __builtin_bit_cast(int4v_t, a),
                                                                               __builtin_bit_cast(int4v_t, c), 0, 0, 0));
  } else if constexpr (std::is_same_v<InT, bf16_t>) {
    using bf8_t = bf16_t __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8_t, b), __builtin_bit_cast(bf8_t, a), c, 0, 0, 0);
  } else {
    return mfma_16x16x32(__builtin_bit_cast(half8_t, b), __builtin_bit_cast(half8_t, a), c);
  }
}

namespace {

// ------------------------------------------------------------------------------------------
// Few rows, few columns or few tiles: the wavefronts of a workgroup share ONE output tile of
// 16*TM x 16*TN and split K among themselves (k-tile t goes to wavefront t % kWaves), each streaming
// its own part of both operands through an LDS ring of its own: no barrier until the partial tiles
// are added up in LDS at the end.
//
// Such problems are bound by how fast a CU takes in its operands: a tile of 32 x 16 does 21 flops per
// byte.  Operand fragments read straight from memory into registers run into the address unit, which
// merges only ADJACENT lanes - the sixteen rows of a fragment lie 16 lanes apart, 64 accesses per
// KiB, a quarter of the L1's rate (32 x 4096 x 4096: 12.7 us).  LDS-direct requests of 8 rows x 128 bytes
// are whole lines: 7.8 us, 4.4 TB/s (the 64 x 64 bounds-checked kernel that ran before: 68.6).
// ------------------------------------------------------------------------------------------
template <int TM_, int TN_, int WAVES_>
struct SplitKShape {
  static constexpr int TM = TM_, TN = TN_, kWaves = WAVES_;
  static constexpr int kStages = 2;                           // k-tiles in a wavefront's ring
  static constexpr int BM = 16 * TM, BN = 16 * TN, BK = 64;
  static constexpr int kThreads = kWaves * kWaveSize;
  static constexpr int kFrags = TM + TN;                      // 16-row operand fragments per 32-deep step
  static constexpr int kLoads = 2 * kFrags;                   // 1 KiB requests (8 rows x 128 bytes) per k-tile
  static constexpr int kStageBytes = kLoads * 1024;
  static constexpr int kPitch = BN + 4;                       // floats per row of a partial tile in LDS
  static constexpr int kRingBytes = kWaves * kStages * kStageBytes;
  static constexpr int kPartBytes = kWaves * BM * kPitch * 4;
  static constexpr int kLdsBytes = kRingBytes > kPartBytes ? kRingBytes : kPartBytes;
  static_assert(kLoads < 64, "vmcnt is a 6-bit counter");
  // the same swizzle as the big kernel's: conflict-free fragment reads of 128-byte rows
  __host__ __device__ static constexpr int swizzle(int row, int c) { return c ^ ((row / 2) % 8); }
};

// Leaves the partial tiles of the wavefronts in LDS, [wave][row][kPitch] (int32 where InT is int8_t), behind a barrier: their sum is the
// tile of A * B^T whose first row and column are m0 and n0, of which M x N exist.  K counts 16 bits (half the elements of 8), K % 8 == 0.
// kTwo: the tile's columns alternate between rows of B and of B1 in blocks of 16, from row n0 of either on, BN / 2 of each, of which N exist.
template <typename S, typename InT, bool kTwo = false>
TFK_DEVICE void split_k_multiply(const uint16_t* A, const uint16_t* B, const uint16_t* B1, int M, int N, int K, int m0, int n0, int lane, int wave,
                                 char* smem) {
  const int lr = lane & 15, lg = lane >> 4;
  // Request n of a k-tile: rows 8n .. 8n+7 of A (n < 2 TM) or B, lane l fills physical chunk l % 8 of
  // row l / 8.  Rows past the edge re-fetch the last one.  The chunks of the last k-tile that lie
  // behind K fetch that tile's first chunk instead; their products are masked below.
  const char* a_tile = reinterpret_cast<const char*>(A + (size_t)m0 * K);
  const char* b_tile = reinterpret_cast<const char*>(B + (size_t)n0 * K);
  const char* b1_tile = kTwo ? reinterpret_cast<const char*>(B1 + (size_t)n0 * K) : nullptr;
  const int num_k_tiles = (K + S::BK - 1) / S::BK, last_tile = num_k_tiles - 1;
  unsigned off[S::kLoads], off_last[S::kLoads];
#pragma unroll
  for (int n = 0; n < S::kLoads; ++n) {
    const bool of_a = n < 2 * S::TM;
    const int row = (of_a ? n : n - 2 * S::TM) * 8 + lane / 8;
    const int c = S::swizzle(row, lane % 8);
    // (kTwo: blocks of 16 rows are of B and of B1 in turn)
    const int in_b = kTwo ? row / 32 * 16 + row % 16 : row;
    const unsigned base = (unsigned)min(of_a ? row : in_b, (of_a ? M - m0 : N - n0) - 1) * (unsigned)K * 2u;
    off[n] = base + 16u * c;
    off_last[n] = last_tile * S::BK + 8 * c < K ? off[n] : base;
  }
  const unsigned ring = lds_address(smem) + wave * S::kStages * S::kStageBytes;
  auto request = [&](int stage, int kt) __attribute__((always_inline)) {
    const bool last = kt == last_tile;
#pragma unroll
    for (int n = 0; n < S::kLoads; ++n) {
      const char* src = (n < 2 * S::TM ? a_tile : kTwo && (n - 2 * S::TM) / 2 % 2 ? b1_tile : b_tile) + (size_t)kt * (S::BK * 2);
      // (the LDS destination is an M0 input of the statement, the s_nop the wait state behind an M0 write)
      asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                   :
                   : "v"(last ? off_last[n] : off[n]), "s"(src), "{m0}"(ring + stage * S::kStageBytes + n * 1024)
                   : "memory");
    }
  };
  unsigned rd[2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) rd[ks] = ring + lr * 128 + S::swizzle(lr, 4 * ks + lg) * 16;

  float4_t acc[S::TM][S::TN];
#pragma unroll
  for (int i = 0; i < S::TM; ++i)
#pragma unroll
    for (int j = 0; j < S::TN; ++j) acc[i][j] = float4_t{0.f, 0.f, 0.f, 0.f};

  uint4_t fr[2][2][S::kFrags];   // [set][32-deep step][fragments of A, then of B]
  auto read = [&](int set, int stage) __attribute__((always_inline)) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int f = 0; f < S::kFrags; ++f)
        fr[set][ks][f] =
            *(__attribute__((address_space(3))) const uint4_t*)(size_t)(rd[ks] + stage * S::kStageBytes + f * 2048);
  };
  auto mask_behind_k = [&](int set) __attribute__((always_inline)) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
      if (last_tile * S::BK + (4 * ks + lg) * 8 >= K) {
#pragma unroll
        for (int f = 0; f < S::kFrags; ++f) fr[set][ks][f] = uint4_t{0u, 0u, 0u, 0u};
      }
  };
  // waits until at most this wavefront's youngest k-tile, if there is one behind the awaited, is still in flight
  auto wait_for_tile = [&](bool one_behind) __attribute__((always_inline)) {
    if (one_behind) wait_vmem<S::kLoads>();
    else wait_vmem<0>();
  };
  const int mine = wave < num_k_tiles ? (last_tile - wave) / S::kWaves + 1 : 0;   // k-tiles of this wavefront
  auto tile_of = [&](int t) __attribute__((always_inline)) { return wave + t * S::kWaves; };
#pragma unroll
  for (int t = 0; t < S::kStages; ++t)
    if (t < mine) request(t, tile_of(t));
  if (mine > 0) {
    wait_for_tile(mine > 1);
    read(0, 0);
  }
  int stage = 0;   // of tile t
  // Tile t: its fragments are on their way into set t % 2; once they have arrived its stage takes tile
  // t + kStages, and the fragments of tile t + 1 are requested under the products of tile t.
  auto step = [&](int t, auto set_c) __attribute__((always_inline)) {
    constexpr int set = decltype(set_c)::value;
    __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
    __builtin_amdgcn_sched_barrier(0);
    if (t + S::kStages < mine) request(stage, tile_of(t + S::kStages));
    stage = stage + 1 == S::kStages ? 0 : stage + 1;
    if (t + 1 < mine) {
      wait_for_tile(t + 2 < mine);
      read(set ^ 1, stage);
    }
    if (K % S::BK != 0 && tile_of(t) == last_tile) mask_behind_k(set);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < S::TM; ++i)
#pragma unroll
        for (int j = 0; j < S::TN; ++j) acc[i][j] = mfma_rows<InT>(fr[set][ks][i], fr[set][ks][S::TM + j], acc[i][j]);
    __builtin_amdgcn_sched_barrier(0);
  };
  for (int t = 0; t < mine; t += 2) {
    step(t, std::integral_constant<int, 0>{});
    if (t + 1 < mine) step(t + 1, std::integral_constant<int, 1>{});
  }
  __syncthreads();   // every ring has been read: the partial tiles take their place

  float* s_part = reinterpret_cast<float*>(smem);
  float* own = s_part + wave * S::BM * S::kPitch;
#pragma unroll
  for (int i = 0; i < S::TM; ++i)
#pragma unroll
    for (int j = 0; j < S::TN; ++j)
      *reinterpret_cast<float4_t*>(own + (16 * i + lr) * S::kPitch + 16 * j + 4 * lg) = acc[i][j];
  __syncthreads();
}

}  // namespace
}  // namespace tfk
