// Products A * B^T whose results do not go to memory as they are: what the operators of gemm_int8.hip, gated_ffn.hip and
// linear_cross_entropy.hip share.  A is [M, K], B [N, K], both row-major; a kernel computes tiles of the product in registers and hands
// them to an EPILOGUE, a struct of pointers and sizes that is called once for every wavefront's tile.
//
// A wavefront's tile is TM x TN blocks of 16 x 16, as v_mfma_*_16x16x* leaves them with its operands swapped: element r of
// acc[i][j] of lane l is row 16 * i + l % 16, column 16 * j + 4 * (l / 16) + r.
#pragma once

#include <algorithm>
#include <climits>
#include <type_traits>

#include "common.hpp"
#include "gemm_ring64.hpp"
#include "gemm_split_k.hpp"

namespace tfk {

// The operands of a product.  With two matrices B (gate and up) the columns of the product alternate between them in blocks of 16:
// block 2 * j is columns 16 * j .. of b[0], block 2 * j + 1 the same columns of b[1].
struct Operands {
  const void* a;
  const void* b[2];
  int M, N;          // rows of a, rows of each b
  int K;
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
// one access (as gemm.hip's own store, with its reasons).  Rows and columns from `rows` and `cols` on are left out.
template <bool kInside, typename T>
TFK_DEVICE void store_block_pair(T* c, size_t pitch, int row, int col, int rows, int cols, int lane, float4_t left, float4_t right) {
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
  if (!kInside && r >= rows) return;
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
TFK_DEVICE void store_block(T* c, size_t pitch, int row, int col, int rows, int cols, int lane, float4_t v) {
  typedef T four_t __attribute__((ext_vector_type(4)));
  typedef four_t four_any_t __attribute__((aligned(sizeof(T))));
  const int r = row + (lane & 15), at = col + 4 * (lane >> 4);
  if (!kInside && r >= rows) return;
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
TFK_DEVICE void store_blocks(T* c, size_t pitch, int row, int col, int rows, int cols, int lane, const float4_t (&v)[kBlocks]) {
  constexpr int kPairs = sizeof(T) == 2 ? kBlocks / 2 : 0;
  if constexpr (kPairs > 0) {
#pragma unroll
    for (int j = 0; j < kPairs; ++j) store_block_pair<kInside>(c, pitch, row, col + 32 * j, rows, cols, lane, v[2 * j], v[2 * j + 1]);
  }
#pragma unroll
  for (int j = 2 * kPairs; j < kBlocks; ++j) store_block<kInside>(c, pitch, row, col + 16 * j, rows, cols, lane, v[j]);
}

// ------------------------------------------------------------------------------------------
// Any M, N, K and any alignment: tiles of 64 x 64, 128 bytes of K at a time through registers into one LDS stage, every access checked.
// What the other kernels' requests cannot fetch runs here: rows that do not start at 16-byte boundaries.
// ------------------------------------------------------------------------------------------
constexpr int kAnyTile = 64, kAnyThreads = 256;

TFK_DEVICE int row_swizzle(int row, int c) { return c ^ ((row / 2) % 8); }   // 128-byte rows, 16-byte chunks: no bank conflicts

template <typename InT>
TFK_DEVICE uint4_t load_chunk_any(const InT* row, int k, int K, bool whole) {
  constexpr int kElems = 16 / sizeof(InT);
  uint4_t v = {0u, 0u, 0u, 0u};
  if (whole) {
    if (k < K) v = *reinterpret_cast<const uint4_t*>(row + k);
    return v;
  }
  using bits_t = std::conditional_t<sizeof(InT) == 1, uint8_t, uint16_t>;
  const bits_t* p = reinterpret_cast<const bits_t*>(row);
#pragma unroll
  for (int t = 0; t < kElems; ++t)
    if (k + t < K) v[t * sizeof(InT) / 4] |= (unsigned)p[k + t] << (8 * (t * sizeof(InT) % 4));
  return v;
}

template <typename InT, bool kTwo, typename Epilogue>
__global__ __launch_bounds__(kAnyThreads) void product_any_kernel(Operands x, bool whole, int tiles_m, Epilogue epilogue) {
  constexpr int kStep = 128 / sizeof(InT);   // elements of K at a time
  __shared__ __attribute__((aligned(16))) char sa[kAnyTile * 128];
  __shared__ __attribute__((aligned(16))) char sb[kAnyTile * 128];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tile_m = blockIdx.x % tiles_m, tile_n = blockIdx.x / tiles_m;
  constexpr int kCols = kTwo ? kAnyTile / 2 : kAnyTile;   // columns of the result
  const int m0 = tile_m * kAnyTile, n0 = tile_n * kCols;
  const int wm = wave / 2, wn = wave % 2, fr = lane & 15, fg = lane >> 4;
  const InT* const a = static_cast<const InT*>(x.a);

  float4_t acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = float4_t{0.f, 0.f, 0.f, 0.f};

  for (int k0 = 0; k0 < x.K; k0 += kStep) {
    for (int f = tid; f < kAnyTile * 8; f += kAnyThreads) {
      const int row = f / 8, c = f % 8;
      const int k = k0 + c * (16 / (int)sizeof(InT));
      uint4_t va = {0u, 0u, 0u, 0u}, vb = {0u, 0u, 0u, 0u};
      if (m0 + row < x.M) va = load_chunk_any(a + (size_t)(m0 + row) * x.K, k, x.K, whole);
      const int n = n0 + (kTwo ? row / 32 * 16 + row % 16 : row);
      const InT* const b = static_cast<const InT*>(kTwo && row / 16 % 2 ? x.b[1] : x.b[0]);
      if (n < x.N) vb = load_chunk_any(b + (size_t)n * x.K, k, x.K, whole);
      *reinterpret_cast<uint4_t*>(sa + row * 128 + row_swizzle(row, c) * 16) = va;
      *reinterpret_cast<uint4_t*>(sb + row * 128 + row_swizzle(row, c) * 16) = vb;
    }
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      uint4_t af[2], bf[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int ra = wm * 32 + i * 16 + fr, rb = wn * 32 + i * 16 + fr;
        af[i] = *reinterpret_cast<const uint4_t*>(sa + ra * 128 + row_swizzle(ra, 4 * ks + fg) * 16);
        bf[i] = *reinterpret_cast<const uint4_t*>(sb + rb * 128 + row_swizzle(rb, 4 * ks + fg) * 16);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma_rows<InT>(af[i], bf[j], acc[i][j]);
    }
    __syncthreads();
  }
  const int col = n0 + wn * (kTwo ? 16 : 32);
  epilogue.template run<false>(acc, TileAt{m0 + wm * 32, col, m0, n0, lane, tile_n * 2 + wn});
}

// ------------------------------------------------------------------------------------------
// Rows that start at 16-byte boundaries: the main loops of the GEMM.
// ------------------------------------------------------------------------------------------
// M >= BM, N >= BN (kTwo: BN / 2), K >= 128 bytes.  The last tile of a row or column of tiles ends where the result does: it overlaps its neighbour.
template <typename S, typename InT, bool kTwo, typename Epilogue>
__global__ __launch_bounds__(S::kThreads) void product_ring64_kernel(Operands x, int tiles_m, int tiles_n, Epilogue epilogue) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int kCols = kTwo ? S::BN / 2 : S::BN;   // columns of the result
  int tile_m, tile_n;
  tile_of_block(blockIdx.x, gridDim.x, tiles_m, tiles_n, tile_m, tile_n);
  const int m0 = min(tile_m * S::BM, x.M - S::BM), n0 = min(tile_n * kCols, x.N - kCols);
  const int wm = wave / S::WAVES_N, wn = wave % S::WAVES_N;
  float4_t acc[S::TM][S::TN];
  ring64_multiply<S, InT, kTwo>(static_cast<const uint16_t*>(x.a), static_cast<const uint16_t*>(x.b[0]), static_cast<const uint16_t*>(x.b[1]),
                                x.K * (int)sizeof(InT) / 2, m0, n0, lane, wave, smem, acc);
  // nothing of the epilogue is worth a register of the main loop
  int again = lane;
  asm volatile("" : "+v"(again));
  epilogue.template run<true>(acc, TileAt{m0 + wm * S::WM, n0 + wn * (kCols / S::WAVES_N), tile_m * S::BM, tile_n * kCols, again,
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
  const int m0 = pid % tiles_m * S::BM, n0 = pid / tiles_m * kCols;
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

// The kernel that gemm.hip's cost model expects to be done first with M x N outputs over K 16-bit elements, out of those of `allowed` (a bit per row of
// its table kGemmKernels; bit 0 is among them): its position there.
int pick_table_kernel(int64_t M, int64_t N, int64_t K, unsigned allowed);

// Positions in that table, and the kernels here.  With two matrices B, tiles have an even number of 16-column blocks to a wavefront, a
// wavefront's requests begin with a block (no tiles of 192 columns), and the smallest tile is 16 x 32.
constexpr int kAnyKernel = -1;
constexpr unsigned kOneAllowed = 0x7fff, kTwoAllowed = 0x7fff & ~(1u << 1 | 1u << 2 | 1u << 11 | 1u << 13);

struct ProductPlan {
  int kernel;       // position, or kAnyKernel
  int64_t slots;    // of a row's partial results (TileAt)
};
// slots of a row's partial results
inline int64_t product_slots(int kernel, int64_t N) {
  constexpr int kColumns[] = {16, 16, 16, 32, 32, 32, 64, 64, 64, 64, 64, 96, 64, 96, 128};   // a wavefront's (split K: a tile's)
  if (kernel == kAnyKernel) return 2 * tiles_of(N, kAnyTile);
  // (the last tile has a slot for each of its wavefronts)
  return kernel < 7 ? tiles_of(N, kColumns[kernel]) : 2 * tiles_of(N, 2 * kColumns[kernel]);
}

template <typename InT>
ProductPlan plan_product(const Operands& x, bool two) {
  // rows that 16-byte requests can walk
  const bool whole = x.K % (16 / (int)sizeof(InT)) == 0 && at_16B(x.a) && at_16B(x.b[0]) && (!two || at_16B(x.b[1]));
  const int kernel = whole ? pick_table_kernel(x.M, two ? 2 * (int64_t)x.N : x.N, (int64_t)x.K * (int)sizeof(InT) / 2, two ? kTwoAllowed : kOneAllowed)
                           : kAnyKernel;
  return {kernel, product_slots(kernel, x.N)};
}

template <typename S, typename InT, bool kTwo, typename Epilogue>
int launch_ring64_product(const Operands& x, const Epilogue& epilogue, hipStream_t st) {
  auto kern = product_ring64_kernel<S, InT, kTwo, Epilogue>;
  static_assert(S::kLdsBytes <= kMaxLdsBytes, "ring does not fit in LDS");
  TFK_LDS_OPT_IN(kern, S::kLdsBytes);
  const int64_t tiles_m = tiles_of(x.M, S::BM), tiles_n = tiles_of(x.N, kTwo ? S::BN / 2 : S::BN);
  return launch_kernel(kern, dim3((unsigned)(tiles_m * tiles_n)), dim3(S::kThreads), S::kLdsBytes, st, x, (int)tiles_m, (int)tiles_n, epilogue);
}
template <typename S, typename InT, bool kTwo, typename Epilogue>
int launch_split_k_product(const Operands& x, const Epilogue& epilogue, hipStream_t st) {
  auto kern = product_split_k_kernel<S, InT, kTwo, Epilogue>;
  static_assert(S::kLdsBytes <= kMaxLdsBytes, "rings do not fit in LDS");
  if constexpr (S::kLdsBytes > 64 * 1024) TFK_LDS_OPT_IN(kern, S::kLdsBytes);
  const int64_t tiles_m = tiles_of(x.M, S::BM), tiles_n = tiles_of(x.N, kTwo ? S::BN / 2 : S::BN);
  return launch_kernel(kern, dim3((unsigned)(tiles_m * tiles_n)), dim3(S::kThreads), S::kLdsBytes, st, x, (int)tiles_m, (int)tiles_n, epilogue);
}

template <typename InT, bool kTwo, typename Epilogue>
int launch_product(const char* who, const Operands& x, const ProductPlan& plan, const Epilogue& epilogue, hipStream_t st) {
  // (a launch has less than 2^32 threads: 2^24 workgroups of 256; no tile has fewer than 256 elements, or 512 of two matrices)
  TFK_REQUIRE(tiles_of(x.M, 16) * tiles_of(x.N, 16) < (int64_t)1 << 27, TF_ERR_INVALID_ARG, "%s: result too large", who);
  if (plan.kernel == kAnyKernel) {
    const int64_t tiles_m = tiles_of(x.M, kAnyTile), tiles_n = tiles_of(x.N, kTwo ? kAnyTile / 2 : kAnyTile);
    const bool whole = x.K % (16 / (int)sizeof(InT)) == 0 && at_16B(x.a) && at_16B(x.b[0]) && (!kTwo || at_16B(x.b[1]));
    return launch_kernel(product_any_kernel<InT, kTwo, Epilogue>, dim3((unsigned)(tiles_m * tiles_n)), dim3(kAnyThreads), 0, st, x, whole, (int)tiles_m,
                         epilogue);
  }
  using Launcher = int (*)(const Operands&, const Epilogue&, hipStream_t);
  if constexpr (kTwo) {
    static constexpr Launcher kLaunchers[] = {
        launch_split_k_product<SplitKShape<1, 2, 4>, InT, kTwo, Epilogue>, nullptr, nullptr,
        launch_split_k_product<SplitKShape<2, 2, 1>, InT, kTwo, Epilogue>, launch_split_k_product<SplitKShape<2, 2, 4>, InT, kTwo, Epilogue>,
        launch_split_k_product<SplitKShape<4, 2, 4>, InT, kTwo, Epilogue>, launch_split_k_product<SplitKShape<4, 4, 4>, InT, kTwo, Epilogue>,
        launch_ring64_product<Ring64Shape<128, 128, 4>, InT, kTwo, Epilogue>, launch_ring64_product<Ring64Shape<128, 128, 2>, InT, kTwo, Epilogue>,
        launch_ring64_product<Ring64Shape<128, 128, 2>, InT, kTwo, Epilogue>, launch_ring64_product<Ring64Shape<192, 128, 2>, InT, kTwo, Epilogue>,
        nullptr, launch_ring64_product<Ring64Shape<256, 128, 2>, InT, kTwo, Epilogue>, nullptr,
        launch_ring64_product<Ring64Shape<256, 256, 2>, InT, kTwo, Epilogue>};
    return kLaunchers[plan.kernel](x, epilogue, st);
  } else {
    static constexpr Launcher kLaunchers[] = {
        launch_split_k_product<SplitKShape<1, 1, 4>, InT, kTwo, Epilogue>, launch_split_k_product<SplitKShape<1, 1, 8>, InT, kTwo, Epilogue>,
        launch_split_k_product<SplitKShape<2, 1, 4>, InT, kTwo, Epilogue>, launch_split_k_product<SplitKShape<2, 2, 1>, InT, kTwo, Epilogue>,
        launch_split_k_product<SplitKShape<2, 2, 4>, InT, kTwo, Epilogue>, launch_split_k_product<SplitKShape<4, 2, 4>, InT, kTwo, Epilogue>,
        launch_split_k_product<SplitKShape<4, 4, 4>, InT, kTwo, Epilogue>,
        launch_ring64_product<Ring64Shape<128, 128, 4>, InT, kTwo, Epilogue>, launch_ring64_product<Ring64Shape<128, 128, 2>, InT, kTwo, Epilogue>,
        launch_ring64_product<Ring64Shape<128, 128, 2>, InT, kTwo, Epilogue>, launch_ring64_product<Ring64Shape<192, 128, 2>, InT, kTwo, Epilogue>,
        launch_ring64_product<Ring64Shape<192, 192, 2>, InT, kTwo, Epilogue>, launch_ring64_product<Ring64Shape<256, 128, 2>, InT, kTwo, Epilogue>,
        launch_ring64_product<Ring64Shape<256, 192, 2>, InT, kTwo, Epilogue>, launch_ring64_product<Ring64Shape<256, 256, 2>, InT, kTwo, Epilogue>};
    return kLaunchers[plan.kernel](x, epilogue, st);
  }
}

// ------------------------------------------------------------------------------------------
// Layout: what the products of a backward pass take transposed
// ------------------------------------------------------------------------------------------
// dst[c * pitch + r] = src[r * src_pitch + c] of 16-bit elements, for c < cols and r < padded_rows, zeros from `rows` on.
int launch_transpose_padded(const char* who, const void* src, int64_t src_pitch, void* dst, int64_t pitch, int64_t rows, int64_t cols,
                            int64_t padded_rows, hipStream_t st);
// zeros in columns from .. to - 1 of rows of 16-bit elements
int launch_zero_columns(const char* who, void* dst, int64_t pitch, int64_t rows, int64_t from, int64_t to, hipStream_t st);
// count 16-bit elements of zero
int launch_zero_16bit(void* dst, int64_t count, hipStream_t st);

}  // namespace tfk
