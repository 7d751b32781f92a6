// Products A * B^T whose results do not go to memory as they are: what the operators of gemm_int8.hip, gated_ffn.hip and
// linear_cross_entropy.hip share.  A is [M, K], B [N, K], both row-major; a kernel computes tiles of the product in registers and hands
// them to an EPILOGUE, a struct of pointers and sizes that is called once for every wavefront's tile.
//
// A wavefront's tile is TM x TN blocks of 16 x 16, as v_mfma_*_16x16x* leaves them with its operands swapped: element r of
// acc[i][j] of lane l is row 16 * i + l % 16, column 16 * j + 4 * (l / 16) + r.
#pragma once

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "common.hpp"
#include "gemm_ring64_cols.hpp"
#include "gemm_split_k.hpp"

namespace tfk {

// The operands of a product, at 16-byte boundaries, K a multiple of 16 bytes (copy_rows makes such rows of others).  With two matrices B (gate and up) the columns of the product alternate between them in blocks of 16:
// block 2 * j is columns 16 * j .. of b[0], block 2 * j + 1 the same columns of b[1].
struct Operands {
  const void* a;
  const void* b[2];
  int M, N;          // rows of a, rows of each b
  int K;
  int tile_row = 0;  // of the result's rows of tiles, the first that a launch does
};

// Where a wavefront's tile lies: its first row and column (of b[0] where there are two), and the first that no tile in front of it
// has: tiles at an edge may overlap their neighbours, and what is added up or counted must be so once.
struct TileAt {
  int row, col;
  int row_from, col_from;
  int lane;
  int slot;          // of the row's partial results: one for each wavefront that works on the row
};

// ---- stores ---------------------------------------------------------------------------------
// An epilogue is called as epilogue.run<kInside>(acc, at): kInside says that the whole tile lies inside the result.
//
// Two blocks side by side, columns `col` .. col + 31, rounded to T: 16 bytes a lane, four adjacent lanes a row, which is what leaves a wavefront as
// one access (as gemm.hip's own store, with its reasons).  us of the gated block in bf16, 16 bytes from where they are / with lanes traded first: 4096 x 2816 x 1024
// 49.4 / 50.1, with rows of 2815 58.6 / 50.0, and gate and up kept 88.5 / 57.6.  Rows and columns from `rows` and `cols` on are left out,
// and rows in front of `from`.
template <bool kInside, typename T>
TFK_DEVICE void store_block_pair(T* c, size_t pitch, int row, int col, int rows, int cols, int lane, float4_t left, float4_t right,
                                 int from) {
  typedef uint4_t out16B_t __attribute__((aligned(2)));
  typedef T two_t __attribute__((ext_vector_type(2)));
  const int st_row = lane >> 2, st_seg = lane & 3;
  const int src_lane = st_row + 16 * (((st_seg & 1) << 1) | (st_seg >> 1));
  unsigned x[2], y[2];
#pragma unroll
  for (int d = 0; d < 2; ++d) {
    x[d] = __builtin_bit_cast(unsigned, two_t{(T)left[2 * d], (T)left[2 * d + 1]});
    y[d] = __builtin_bit_cast(unsigned, two_t{(T)right[2 * d], (T)right[2 * d + 1]});
#if defined(__HIP_DEVICE_COMPILE__)
    auto sw = __builtin_amdgcn_permlane16_swap(x[d], y[d], false, false);
    x[d] = sw[0];
    y[d] = sw[1];
#endif
  }
  uint4_t v;
  v[0] = (unsigned)__builtin_amdgcn_ds_bpermute(4 * src_lane, (int)x[0]);
  v[1] = (unsigned)__builtin_amdgcn_ds_bpermute(4 * src_lane, (int)x[1]);
  v[2] = (unsigned)__builtin_amdgcn_ds_bpermute(4 * src_lane, (int)y[0]);
  v[3] = (unsigned)__builtin_amdgcn_ds_bpermute(4 * src_lane, (int)y[1]);
  const int r = row + st_row, at = col + 8 * st_seg;
  if (!kInside && (r >= rows || r < from)) return;
  T* const to = c + (size_t)r * pitch + at;
  if (kInside || at + 8 <= cols) {
    *reinterpret_cast<out16B_t*>(to) = v;
  } else {
    uint16_t* const p = reinterpret_cast<uint16_t*>(to);
#pragma unroll
    for (int t = 0; t < 8; ++t)
      if (at + t < cols) p[t] = (uint16_t)(v[t / 2] >> (16 * (t % 2)));
  }
}
// One block, rounded to T: four columns a lane.
template <bool kInside, typename T>
TFK_DEVICE void store_block(T* c, size_t pitch, int row, int col, int rows, int cols, int lane, float4_t v, int from) {
  typedef T four_t __attribute__((ext_vector_type(4)));
  typedef four_t four_any_t __attribute__((aligned(sizeof(T))));
  const int r = row + (lane & 15), at = col + 4 * (lane >> 4);
  if (!kInside && (r >= rows || r < from)) return;
  T* const to = c + (size_t)r * pitch + at;
  if (kInside || at + 4 <= cols) {
    *reinterpret_cast<four_any_t*>(to) = four_t{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
  } else {
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (at + t < cols) to[t] = (T)v[t];
  }
}
// Row i of a wavefront's blocks: v[0 .. n)
template <bool kInside, typename T, int kBlocks>
TFK_DEVICE void store_blocks(T* c, size_t pitch, int row, int col, int rows, int cols, int lane, const float4_t (&v)[kBlocks], int from = 0) {
  constexpr int kPairs = sizeof(T) == 2 ? kBlocks / 2 : 0;
  if constexpr (kPairs > 0) {
#pragma unroll
    for (int j = 0; j < kPairs; ++j) store_block_pair<kInside>(c, pitch, row, col + 32 * j, rows, cols, lane, v[2 * j], v[2 * j + 1], from);
  }
#pragma unroll
  for (int j = 2 * kPairs; j < kBlocks; ++j) store_block<kInside>(c, pitch, row, col + 16 * j, rows, cols, lane, v[j], from);
}

// ------------------------------------------------------------------------------------------
// A * B^T: the main loops of the GEMM.
// ------------------------------------------------------------------------------------------
// M >= BM (kFew: M < BM), N >= BN (kTwo: BN / 2), K >= 128 bytes.  The last tile of a row or column of tiles ends where the result does: it
// overlaps its neighbour.
template <typename S, typename InT, bool kTwo, bool kFew, typename Epilogue>
__global__ __launch_bounds__(S::kThreads) void product_ring64_kernel(Operands x, int tiles_m, int tiles_n, Epilogue epilogue) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int kCols = kTwo ? S::BN / 2 : S::BN;   // columns of the result
  int tile_m, tile_n;
  tile_of_block(blockIdx.x, gridDim.x, tiles_m, tiles_n, tile_m, tile_n);
  tile_m += x.tile_row;
  const int m0 = kFew ? 0 : min(tile_m * S::BM, x.M - S::BM), n0 = min(tile_n * kCols, x.N - kCols);
  const int wm = wave / S::WAVES_N, wn = wave % S::WAVES_N;
  float4_t acc[S::TM][S::TN];
  ring64_multiply<S, InT, kTwo, kFew>(static_cast<const uint16_t*>(x.a), static_cast<const uint16_t*>(x.b[0]), static_cast<const uint16_t*>(x.b[1]),
                                      x.K * (int)sizeof(InT) / 2, m0, n0, lane, wave, smem, acc, x.M);
  // nothing of the epilogue is worth a register of the main loop
  int again = lane;
  asm volatile("" : "+v"(again));
  epilogue.template run<!kFew>(acc, TileAt{m0 + wm * S::WM, n0 + wn * (kCols / S::WAVES_N), tile_m * S::BM, tile_n * kCols, again,
                                          tile_n * S::WAVES_N + wn});
}

// Any M and N.  Wavefront w finishes the rows of blocks w, w + kWaves, ... of the tile that all of them added up.
template <typename S, typename InT, bool kTwo, typename Epilogue>
__global__ __launch_bounds__(S::kThreads) void product_split_k_kernel(Operands x, int tiles_m, int tiles_n, Epilogue epilogue) {
  static_assert(!kTwo || S::TN % 2 == 0, "gate and up side by side");
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int kCols = kTwo ? S::BN / 2 : S::BN;
  const int pid = xcd_major(blockIdx.x, tiles_m * tiles_n);
  const int m0 = (x.tile_row + pid % tiles_m) * S::BM, n0 = pid / tiles_m * kCols;
  split_k_multiply<S, InT, kTwo>(static_cast<const uint16_t*>(x.a), static_cast<const uint16_t*>(x.b[0]), static_cast<const uint16_t*>(x.b[1]), x.M,
                                 x.N, x.K * (int)sizeof(InT) / 2, m0, n0, lane, wave, smem);
  const float* const parts = reinterpret_cast<const float*>(smem);
  for (int i = wave; i < S::TM; i += S::kWaves) {
    float4_t sum[1][S::TN];
#pragma unroll
    for (int j = 0; j < S::TN; ++j) {
      const int at = (16 * i + (lane & 15)) * S::kPitch + 16 * j + 4 * (lane >> 4);
      sum[0][j] = *reinterpret_cast<const float4_t*>(parts + at);
#pragma unroll
      for (int w = 1; w < S::kWaves; ++w) {
        const float4_t more = *reinterpret_cast<const float4_t*>(parts + w * S::BM * S::kPitch + at);
        if constexpr (std::is_same_v<InT, int8_t>)
          sum[0][j] = __builtin_bit_cast(float4_t, __builtin_bit_cast(int4v_t, sum[0][j]) + __builtin_bit_cast(int4v_t, more));
        else
          sum[0][j] += more;
      }
    }
    epilogue.template run<false>(sum, TileAt{m0 + 16 * i, n0, m0, n0, lane, pid / tiles_m});
  }
}

// ---- host side ---------------------------------------------------------------------------
inline int64_t tiles_of(int64_t extent, int64_t tile) { return (extent + tile - 1) / tile; }
inline int64_t round_up_to(int64_t x, int64_t to) { return tiles_of(x, to) * to; }
inline bool at_16B(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

constexpr int64_t kMaxTiles = ((int64_t)1 << 23) - 1;   // of a launch: it has less than 2^32 threads, of which a workgroup has 512 at most

// The kernel that gemm.hip's cost model expects to be done first with M x N outputs over K 16-bit elements, out of those of `allowed` (a bit per row of
// its table kGemmKernels): its position there.
int pick_table_kernel(int64_t M, int64_t N, int64_t K, unsigned allowed, float* expected_us);
// What it expects of a kernel of its table, in us.
float expected_table_us(int kernel, int64_t tiles, int64_t K);

// Positions in that table, and the kernels here.  With two matrices B, tiles have an even number of 16-column blocks to a wavefront, a
// wavefront's requests begin with a block (no tiles of 192 columns), and the smallest tile is 16 x 32.
constexpr unsigned kOneAllowed = 0x7fff, kTwoAllowed = 0x7fff & ~(1u << 1 | 1u << 2 | 1u << 11 | 1u << 13);

struct ProductPlan {
  int kernel;       // position
  int64_t slots;    // of a row's partial results (TileAt)
};
// Behind the table's end: its tiles of 128 x 128 (requests 4 k-tiles ahead; in pairs on a CU) for fewer than 128 rows.
constexpr int kFewAlone = 15, kFewPaired = 16;
// slots of a row's partial results
inline int64_t product_slots(int kernel, int64_t N) {
  constexpr int kColumns[] = {16, 16, 16, 32, 32, 32, 64, 64, 64, 64, 64, 96, 64, 96, 128, 64, 64};   // a wavefront's (split K: a tile's)
  // (the last tile has a slot for each of its wavefronts)
  return kernel < 7 ? tiles_of(N, kColumns[kernel]) : 2 * tiles_of(N, 2 * kColumns[kernel]);
}
// K: 16-bit elements (half the elements of 8)
inline ProductPlan plan_product(int64_t M, int64_t N, int64_t K, bool two) {
  const int64_t columns = two ? 2 * N : N;
  // (the table has no tile of 16 x 32: up to 16 rows it is ahead of 32 x 32, 1 x 4096 x 11264 of two matrices 33.2 us / 38.4)
  if (two && M <= 16) return {0, product_slots(0, N)};
  float us;
  const unsigned allowed = two ? kTwoAllowed & ~1u : kOneAllowed;
  int kernel = pick_table_kernel(M, columns, K, allowed, &us);
  // More tiles than a launch has, of whatever size: what is best for as many rows as a launch does.
  for (int64_t m = M; !(us < INFINITY) && m > 64;) {
    m = round_up_to(m / 2, 64);
    kernel = pick_table_kernel(m, columns, K, allowed, &us);
  }
  // Fewer than 128 rows and many columns: large tiles all the same where the model expects them sooner than the small ones, which read the
  // weights once for every 32 or 64 rows.  us, small / large: loss of 100 x 1024 over 32000 words 33 / 20.5, of 37 22.3 / 19.4, gated
  // block 100 x 4096 x 11264 57 / 44.5; 64 x 2048 x 8192 17.7 / 21.3 (where the small ones stay).
  if (M < 128 && columns >= 128 && K >= 64) {
    const int64_t tiles = tiles_of(columns, 128);
    const int few = tiles <= 256 ? kFewAlone : kFewPaired;
    if (tiles <= kMaxTiles && expected_table_us(few == kFewAlone ? 7 : 9, tiles, K) < us) kernel = few;
  }
  return {kernel, product_slots(kernel, N)};
}

// As many rows of tiles at a time as a launch has room for: all of them where the result is not enormous.
template <typename S, typename Epilogue>
int launch_tiles(const char* who, void (*kern)(Operands, int, int, Epilogue), Operands x, int64_t tiles_m, int64_t tiles_n, const Epilogue& epilogue,
                 hipStream_t st) {
  TFK_REQUIRE(tiles_n <= kMaxTiles, TF_ERR_INVALID_ARG, "%s: result too large", who);
  const int64_t most = kMaxTiles / tiles_n;
  for (int64_t from = 0; from < tiles_m; from += most) {
    const int64_t rows = std::min(most, tiles_m - from);
    x.tile_row = (int)from;
    if (int rc = launch_kernel(kern, dim3((unsigned)(rows * tiles_n)), dim3(S::kThreads), S::kLdsBytes, st, x, (int)rows, (int)tiles_n, epilogue)) return rc;
  }
  return TF_OK;
}
template <typename S, typename InT, bool kTwo, typename Epilogue, bool kFew = false>
int launch_ring64_product(const char* who, const Operands& x, const Epilogue& epilogue, hipStream_t st) {
  auto kern = product_ring64_kernel<S, InT, kTwo, kFew, Epilogue>;
  static_assert(S::kLdsBytes <= kMaxLdsBytes, "ring does not fit in LDS");
  TFK_LDS_OPT_IN(kern, S::kLdsBytes);
  return launch_tiles<S>(who, kern, x, tiles_of(x.M, S::BM), tiles_of(x.N, kTwo ? S::BN / 2 : S::BN), epilogue, st);
}
template <typename S, typename InT, bool kTwo, typename Epilogue>
int launch_split_k_product(const char* who, const Operands& x, const Epilogue& epilogue, hipStream_t st) {
  auto kern = product_split_k_kernel<S, InT, kTwo, Epilogue>;
  static_assert(S::kLdsBytes <= kMaxLdsBytes, "rings do not fit in LDS");
  if constexpr (S::kLdsBytes > 64 * 1024) TFK_LDS_OPT_IN(kern, S::kLdsBytes);
  return launch_tiles<S>(who, kern, x, tiles_of(x.M, S::BM), tiles_of(x.N, kTwo ? S::BN / 2 : S::BN), epilogue, st);
}

template <typename InT, bool kTwo, typename Epilogue>
int launch_product(const char* who, const Operands& x, const ProductPlan& plan, const Epilogue& epilogue, hipStream_t st) {
  using Launcher = int (*)(const char*, const Operands&, const Epilogue&, hipStream_t);
  if constexpr (kTwo) {
    static constexpr Launcher kLaunchers[] = {
        launch_split_k_product<SplitKShape<1, 2, 4>, InT, kTwo, Epilogue>, nullptr, nullptr,
        launch_split_k_product<SplitKShape<2, 2, 1>, InT, kTwo, Epilogue>, launch_split_k_product<SplitKShape<2, 2, 4>, InT, kTwo, Epilogue>,
        launch_split_k_product<SplitKShape<4, 2, 4>, InT, kTwo, Epilogue>, launch_split_k_product<SplitKShape<4, 4, 4>, InT, kTwo, Epilogue>,
        launch_ring64_product<Ring64Shape<128, 128, 4>, InT, kTwo, Epilogue>, launch_ring64_product<Ring64Shape<128, 128, 2>, InT, kTwo, Epilogue>,
        launch_ring64_product<Ring64Shape<128, 128, 2>, InT, kTwo, Epilogue>, launch_ring64_product<Ring64Shape<192, 128, 2>, InT, kTwo, Epilogue>,
        nullptr, launch_ring64_product<Ring64Shape<256, 128, 2>, InT, kTwo, Epilogue>, nullptr,
        launch_ring64_product<Ring64Shape<256, 256, 2>, InT, kTwo, Epilogue>,
        launch_ring64_product<Ring64Shape<128, 128, 4>, InT, kTwo, Epilogue, true>, launch_ring64_product<Ring64Shape<128, 128, 2>, InT, kTwo, Epilogue, true>};
    return kLaunchers[plan.kernel](who, x, epilogue, st);
  } else {
    static constexpr Launcher kLaunchers[] = {
        launch_split_k_product<SplitKShape<1, 1, 4>, InT, kTwo, Epilogue>, launch_split_k_product<SplitKShape<1, 1, 8>, InT, kTwo, Epilogue>,
        launch_split_k_product<SplitKShape<2, 1, 4>, InT, kTwo, Epilogue>, launch_split_k_product<SplitKShape<2, 2, 1>, InT, kTwo, Epilogue>,
        launch_split_k_product<SplitKShape<2, 2, 4>, InT, kTwo, Epilogue>, launch_split_k_product<SplitKShape<4, 2, 4>, InT, kTwo, Epilogue>,
        launch_split_k_product<SplitKShape<4, 4, 4>, InT, kTwo, Epilogue>,
        launch_ring64_product<Ring64Shape<128, 128, 4>, InT, kTwo, Epilogue>, launch_ring64_product<Ring64Shape<128, 128, 2>, InT, kTwo, Epilogue>,
        launch_ring64_product<Ring64Shape<128, 128, 2>, InT, kTwo, Epilogue>, launch_ring64_product<Ring64Shape<192, 128, 2>, InT, kTwo, Epilogue>,
        launch_ring64_product<Ring64Shape<192, 192, 2>, InT, kTwo, Epilogue>, launch_ring64_product<Ring64Shape<256, 128, 2>, InT, kTwo, Epilogue>,
        launch_ring64_product<Ring64Shape<256, 192, 2>, InT, kTwo, Epilogue>, launch_ring64_product<Ring64Shape<256, 256, 2>, InT, kTwo, Epilogue>,
        launch_ring64_product<Ring64Shape<128, 128, 4>, InT, kTwo, Epilogue, true>, launch_ring64_product<Ring64Shape<128, 128, 2>, InT, kTwo, Epilogue, true>};
    return kLaunchers[plan.kernel](who, x, epilogue, st);
  }
}

// ------------------------------------------------------------------------------------------
// A * B and A^T * B: the products of a backward pass, summed over tokens or over rows of a weight.
// ------------------------------------------------------------------------------------------
struct ColsProduct {
  ColsOperand a, b;         // extents: rows and columns of the result
  const uint16_t* b1;       // where b's rows continue from k-tile `turn` on
  int turn;
  int k_tiles, k_pad;       // 64 summed rows each; zeros in front of the first ones
  int row_from;             // the result's first row that is stored
};
struct ColsPlan {
  int shape;                // into kColsShapes
  int splits, per_split;    // the sum is cut into that many parts of so many k-tiles (the last may be shorter)
  float us;                 // expected
};
struct ColsSize {
  int64_t M, N, k_tiles;    // rows and columns of the result, 64 summed rows each
};
struct ColsShape {
  int bm, bn, table;        // tile, position in gemm.hip's table
};
constexpr ColsShape kColsShapes[] = {{256, 256, 14}, {256, 128, 12}, {128, 128, 7}, {128, 128, 9}};

// Cut, a product costs a launch more and its parts' way through memory (4 bytes written and read for each element and part, at 4 TB/s).
// (Twelve numbers of parts are looked at, not all 64: choosing among these takes the calling thread 10 us a product.  Forced choices, backward pass of the
// gated block and of the head over 11 problems: at most 10% ahead of it.)
inline ColsPlan plan_cols(const ColsSize& of) {
  const auto [M, N, k_tiles] = of;
  constexpr int kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
  ColsPlan best = {0, 1, (int)k_tiles, INFINITY};
  for (int s = 0; s < (int)(sizeof(kColsShapes) / sizeof(kColsShapes[0])); ++s) {
    const int64_t tiles = tiles_of(M, kColsShapes[s].bm) * tiles_of(N, kColsShapes[s].bn);
    for (int64_t splits : kSplits) {
      const int64_t per = tiles_of(k_tiles, splits);
      if (splits > 1 && (tiles * splits > 1024 || per < 4 || tiles_of(k_tiles, per) != splits)) continue;
      const float parts = splits > 1 ? 3.f + (float)(8 * splits * M * N) / 4e6f : 0.f;
      const float us = expected_table_us(kColsShapes[s].table, tiles * splits, 64 * per) + parts;
      if (us < best.us) best = {s, (int)splits, (int)per, us};
    }
  }
  return best;
}

// Both products of a backward pass in one launch (product_pair_kernel), or one after the other as `x` and `w` are planned.  A launch's last round of tiles
// leaves CUs idle, and together there is one such round.  us of the gated block's backward pass in bf16, one after the other / together: 100 x 2816 x 1024
// (tokens x F x K) 25.6 / 18.8, 1337 x 1544 x 1032 52.7 / 42.8, 2048 x 1024 x 1024 42.8 / 28.3, 4096 x 5632 x 2048 360 / 325; 4096 x 2816 x 1024 135 / 133.
// Of the head's in fp16: 1024 tokens x 8192 words x 512 55.4 / 48.4, 613 x 32003 x 1024 181 / 180.  Sums may be cut otherwise than in a product
// that runs alone.
struct PairPlan {
  bool together;
  ColsPlan x, w;            // where they run together
};
inline PairPlan plan_pair(const ColsPlan& x, const ColsSize& of_x, const ColsPlan& w, const ColsSize& of_w) {
  constexpr int kXSplits[] = {1, 2, 3, 4, 6, 8}, kWSplits[] = {1, 2, 3, 4};
  PairPlan best = {false, x, w};
  float best_us = x.us + w.us;
  const auto parts_us = [](const ColsSize& of, int splits) { return splits > 1 ? 3.f + (float)(8 * splits * of.M * of.N) / 4e6f : 0.f; };
  const auto per_split = [](const ColsSize& of, int splits) -> int64_t {   // 0: not cut so
    const int64_t per = tiles_of(of.k_tiles, splits);
    return splits == 1 || (per >= 4 && tiles_of(of.k_tiles, per) == splits) ? per : 0;
  };
  for (int s = 0; s < (int)(sizeof(kColsShapes) / sizeof(kColsShapes[0])); ++s) {
    const int bm = kColsShapes[s].bm, bn = kColsShapes[s].bn;
    const int64_t x_tiles = tiles_of(of_x.M, bm) * tiles_of(of_x.N, bn), w_tiles = tiles_of(of_w.M, bm) * tiles_of(of_w.N, bn);
    const int64_t at_once = s == 3 ? 512 : 256;
    for (int xs : kXSplits) {
      const int64_t x_per = per_split(of_x, xs);
      if (x_per == 0 || x_tiles * xs > 8 * at_once || parts_us(of_x, xs) >= best_us) continue;
      for (int ws : kWSplits) {
        const int64_t w_per = per_split(of_w, ws), blocks = x_tiles * xs + w_tiles * ws;
        // (the last of more than eight rounds does not pay, and parts of so many tiles are half a gigabyte)
        if (w_per == 0 || blocks > 8 * at_once || (s == 3 && blocks <= 256)) continue;
        // what a workgroup of each takes where so many run at a time; the longest, or the whole work and half a workgroup more for the end
        const int64_t round = std::min(blocks, at_once);
        const float x_us = expected_table_us(kColsShapes[s].table, round, 64 * x_per), w_us = expected_table_us(kColsShapes[s].table, round, 64 * w_per);
        const float longest = std::max(x_us, w_us), rounds_us = (x_tiles * xs * x_us + w_tiles * ws * w_us) / at_once + 0.5f * std::min(x_us, w_us);
        const float us = (blocks > at_once ? std::max(longest, rounds_us) : longest) + parts_us(of_x, xs) + parts_us(of_w, ws);
        if (us < best_us) {
          best = {true, {s, xs, (int)x_per, us}, {s, ws, (int)w_per, us}};
          best_us = us;
        }
      }
    }
  }
  return best;
}

struct PartEpilogue;   // below; takes whole tiles

template <typename S, typename InT, bool kColA, typename Epilogue>
TFK_DEVICE void product_cols_tile(const ColsProduct& x, int index, int tiles_m, int tiles_n, int per_split, const Epilogue& epilogue, char* smem) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = tiles_m * tiles_n, split = index / tiles;
  int tile_m, tile_n;
  tile_of_block(index - split * tiles, tiles, tiles_m, tiles_n, tile_m, tile_n);
  const int m0 = tile_m * S::BM, n0 = tile_n * S::BN, t0 = split * per_split;
  const int wm = wave / S::WAVES_N, wn = wave % S::WAVES_N;
  float4_t acc[S::TM][S::TN];
  ring64_multiply_cols<S, InT, kColA>(x.a, x.b, x.b1, x.turn, m0, n0, t0, min(per_split, x.k_tiles - t0), x.k_pad, lane, wave, smem, acc);
  int again = lane;
  asm volatile("" : "+v"(again));
  const TileAt at = {m0 + wm * S::WM, n0 + wn * S::WN, x.row_from, n0, again, split};
  if (std::is_same_v<Epilogue, PartEpilogue>) epilogue.template run<true>(acc, at);
  else if (m0 >= x.row_from && m0 + S::BM <= x.a.extent && n0 + S::BN <= x.b.extent) epilogue.template run<true>(acc, at);
  else epilogue.template run<false>(acc, at);
}
template <typename S, typename InT, bool kColA, typename Epilogue>
__global__ __launch_bounds__(S::kThreads) void product_cols_kernel(ColsProduct x, int tiles_m, int tiles_n, int per_split, Epilogue epilogue) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  product_cols_tile<S, InT, kColA>(x, blockIdx.x, tiles_m, tiles_n, per_split, epilogue, smem);
}

// Whether 32-bit offsets reach the operands of a tile.
template <typename S, bool kColA>
bool cols_reach(const ColsProduct& x) {
  constexpr uint64_t kEnd = (uint64_t)1 << 32;
  return cols_farthest(kColA ? S::BK : std::min(S::BM, x.a.extent), x.a.pitch) < kEnd && cols_farthest(S::BK, x.b.pitch) < kEnd;
}

template <typename S, typename InT, bool kColA, typename Epilogue>
int launch_cols_shape(const char* who, const ColsProduct& x, const ColsPlan& plan, const Epilogue& epilogue, hipStream_t st) {
  auto kern = product_cols_kernel<S, InT, kColA, Epilogue>;
  TFK_LDS_OPT_IN(kern, S::kLdsBytes);
  const int64_t tiles_m = tiles_of(x.a.extent, S::BM), tiles_n = tiles_of(x.b.extent, S::BN);
  TFK_REQUIRE(tiles_m * tiles_n * plan.splits <= kMaxTiles, TF_ERR_INVALID_ARG, "%s: result too large", who);
  TFK_REQUIRE((cols_reach<S, kColA>(x)), TF_ERR_INVALID_ARG, "%s: rows too long", who);
  return launch_kernel(kern, dim3((unsigned)(tiles_m * tiles_n * plan.splits)), dim3(S::kThreads), S::kLdsBytes, st, x, (int)tiles_m, (int)tiles_n,
                       plan.per_split, epilogue);
}
template <typename InT, bool kColA, typename Epilogue>
int launch_cols(const char* who, const ColsProduct& x, const ColsPlan& plan, const Epilogue& epilogue, hipStream_t st) {
  switch (plan.shape) {
    case 0: return launch_cols_shape<Ring64Shape<256, 256, 2>, InT, kColA>(who, x, plan, epilogue, st);
    case 1: return launch_cols_shape<Ring64Shape<256, 128, 2>, InT, kColA>(who, x, plan, epilogue, st);
    case 2: return launch_cols_shape<Ring64Shape<128, 128, 4>, InT, kColA>(who, x, plan, epilogue, st);
    default: return launch_cols_shape<Ring64Shape<128, 128, 2>, InT, kColA>(who, x, plan, epilogue, st);
  }
}

// ---- what gradients end in -----------------------------------------------------------------
struct Scale {
  float in, out;   // operands were multiplied by `in` where they were made, sums are by `out`
};
// What sums are multiplied by, where it is not null: a scale, one number for all, one for each row.
struct Factors {
  const Scale* scale = nullptr;
  const float *all = nullptr, *rows = nullptr;

  TFK_DEVICE float common() const { return (scale != nullptr ? scale->out : 1.f) * (all != nullptr ? *all : 1.f); }
  TFK_DEVICE float of_row(int64_t row) const { return rows != nullptr ? rows[row] : 1.f; }
};
// A sum that is complete: multiplied by its factors, rounded to T.
template <typename T>
struct WholeEpilogue {
  T* out;                  // [M][N]
  Factors factors;
  int M, N;

  template <bool kInside, int TM, int TN>
  TFK_DEVICE void run(float4_t (&acc)[TM][TN], const TileAt& at) const {
    const float common = factors.common();
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int row = at.row + 16 * i + (at.lane & 15);
      const float by = common * factors.of_row(kInside ? row : min(row, M - 1));
      float4_t v[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) v[j] = acc[i][j] * by;
      store_blocks<kInside>(out, (size_t)N, at.row + 16 * i, at.col, M, N, at.lane, v, at.row_from);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};
// A part of a sum: fp32, whole tiles (what lies behind the result's rows and columns is not looked at again), added to what an earlier launch left
// there or in its place.
struct PartEpilogue {
  float* parts;
  int64_t rows, pitch;     // whole tiles
  bool add;

  template <bool, int TM, int TN>
  TFK_DEVICE void run(float4_t (&acc)[TM][TN], const TileAt& at) const {
    if (add) leave<true>(acc, at);
    else leave<false>(acc, at);
  }
  template <bool kAdd, int TM, int TN>
  TFK_DEVICE void leave(float4_t (&acc)[TM][TN], const TileAt& at) const {
    float* const mine = parts + (at.slot * rows + at.row + (at.lane & 15)) * pitch + at.col + 4 * (at.lane >> 4);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        float4_t* const to = reinterpret_cast<float4_t*>(mine + 16 * i * pitch + 16 * j);
        *to = kAdd ? acc[i][j] + *to : acc[i][j];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};
// Either of them.
template <typename Whole>
struct CutEpilogue {
  Whole whole;
  PartEpilogue part;
  bool cut;

  template <bool kInside, int TM, int TN>
  TFK_DEVICE void run(float4_t (&acc)[TM][TN], const TileAt& at) const {
    if (cut) part.template run<true>(acc, at);
    else whole.template run<kInside>(acc, at);
  }
};

// Both products of a backward pass in one launch.
template <typename Epilogue>
struct ColsLaunch {
  ColsProduct x;
  int tiles_m, tiles_n, per_split, blocks;
  Epilogue epilogue;
};
// Workgroups begin in the order of their numbers: those with the longer sums first.
template <typename S, typename InT, typename RowsEpilogue, typename ColsEpilogue>
__global__ __launch_bounds__(S::kThreads) void product_pair_kernel(ColsLaunch<RowsEpilogue> rows, ColsLaunch<ColsEpilogue> cols) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  int index = blockIdx.x;
  bool of_rows;
  if (rows.per_split >= cols.per_split) {
    of_rows = index < rows.blocks;
    if (!of_rows) index -= rows.blocks;
  } else {
    of_rows = index >= cols.blocks;
    if (of_rows) index -= cols.blocks;
  }
  if (of_rows) product_cols_tile<S, InT, false>(rows.x, index, rows.tiles_m, rows.tiles_n, rows.per_split, rows.epilogue, smem);
  else product_cols_tile<S, InT, true>(cols.x, index, cols.tiles_m, cols.tiles_n, cols.per_split, cols.epilogue, smem);
}
template <typename S, typename InT, typename RowsEpilogue, typename ColsEpilogue>
int launch_pair_shape(const char* who, const ColsProduct& x, const ColsPlan& x_plan, const RowsEpilogue& x_epilogue, const ColsProduct& w,
                      const ColsPlan& w_plan, const ColsEpilogue& w_epilogue, hipStream_t st) {
  auto kern = product_pair_kernel<S, InT, RowsEpilogue, ColsEpilogue>;
  TFK_LDS_OPT_IN(kern, S::kLdsBytes);
  const auto tiles = [](const ColsOperand& t, int tile) { return tiles_of(t.extent, tile); };
  const int64_t x_blocks = tiles(x.a, S::BM) * tiles(x.b, S::BN) * x_plan.splits, w_blocks = tiles(w.a, S::BM) * tiles(w.b, S::BN) * w_plan.splits;
  TFK_REQUIRE(x_blocks + w_blocks <= kMaxTiles, TF_ERR_INVALID_ARG, "%s: result too large", who);
  TFK_REQUIRE((cols_reach<S, false>(x) && cols_reach<S, true>(w)), TF_ERR_INVALID_ARG, "%s: rows too long", who);
  return launch_kernel(
      kern, dim3((unsigned)(x_blocks + w_blocks)), dim3(S::kThreads), S::kLdsBytes, st,
      ColsLaunch<RowsEpilogue>{x, (int)tiles(x.a, S::BM), (int)tiles(x.b, S::BN), x_plan.per_split, (int)x_blocks, x_epilogue},
      ColsLaunch<ColsEpilogue>{w, (int)tiles(w.a, S::BM), (int)tiles(w.b, S::BN), w_plan.per_split, (int)w_blocks, w_epilogue});
}
template <typename InT, typename RowsEpilogue, typename ColsEpilogue>
int launch_pair(const char* who, const ColsProduct& x, const ColsPlan& x_plan, const RowsEpilogue& x_epilogue, const ColsProduct& w,
                const ColsPlan& w_plan, const ColsEpilogue& w_epilogue, hipStream_t st) {
  if (x_plan.shape == 0) return launch_pair_shape<Ring64Shape<256, 256, 2>, InT>(who, x, x_plan, x_epilogue, w, w_plan, w_epilogue, st);
  if (x_plan.shape == 1) return launch_pair_shape<Ring64Shape<256, 128, 2>, InT>(who, x, x_plan, x_epilogue, w, w_plan, w_epilogue, st);
  if (x_plan.shape == 2) return launch_pair_shape<Ring64Shape<128, 128, 4>, InT>(who, x, x_plan, x_epilogue, w, w_plan, w_epilogue, st);
  return launch_pair_shape<Ring64Shape<128, 128, 2>, InT>(who, x, x_plan, x_epilogue, w, w_plan, w_epilogue, st);
}

// The room that the parts of a product with M x N results take, in floats, and its rows and pitch.
struct PartsRoom {
  int64_t rows, pitch, floats;
  PartsRoom(const ColsPlan& plan, int64_t M, int64_t N)
      : rows(round_up_to(M, kColsShapes[plan.shape].bm)), pitch(round_up_to(N, kColsShapes[plan.shape].bn)), floats(plan.splits * rows * pitch) {}
};
// out = T(the sum of the parts, times its factors): rows `first` .. M - 1, of which the first is out's and the factors'; N columns
template <typename T>
int launch_sum_parts(const float* parts, const PartsRoom& room, int splits, int64_t first, int64_t M, int64_t N, T* out, const Factors& factors,
                     hipStream_t st);

// ------------------------------------------------------------------------------------------
// Layout
// ------------------------------------------------------------------------------------------
// `padded_rows` rows of `pitch` bytes (a multiple of 16, from a 16-byte boundary on) with the `bytes` bytes of each of `rows` rows of src in
// front, zeros behind them and in the rows that follow: up to three matrices in one launch.
struct RowsToCopy {
  const void* src;
  int64_t rows;
  void* dst;
  int64_t padded_rows;
};
int launch_copy_rows(const RowsToCopy* matrices, int count, int64_t bytes, int64_t pitch, hipStream_t st);
// count 16-bit elements of zero
int launch_zero_16bit(void* dst, int64_t count, hipStream_t st);

}  // namespace tfk
