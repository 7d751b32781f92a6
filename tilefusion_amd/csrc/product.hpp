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
  epilogue(acc, TileAt{m0 + wm * 32, col, m0, n0, lane, tile_n * 2 + wn});
}

// ---- host side ---------------------------------------------------------------------------
inline int64_t tiles_of(int64_t extent, int64_t tile) { return (extent + tile - 1) / tile; }
inline int64_t round_up_to(int64_t x, int64_t to) { return tiles_of(x, to) * to; }
inline bool at_16B(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// rows that 16-byte accesses can walk
template <typename InT>
bool whole_chunks(const Operands& x, bool two) {
  return x.K % (16 / (int)sizeof(InT)) == 0 && at_16B(x.a) && at_16B(x.b[0]) && (!two || at_16B(x.b[1]));
}

// slots of a row's partial results in the kernel above
inline int64_t any_slots(int64_t N) { return 2 * tiles_of(N, kAnyTile); }

template <typename InT, bool kTwo, typename Epilogue>
int launch_product_any(const char* who, const Operands& x, const Epilogue& epilogue, hipStream_t st) {
  const int64_t tiles_m = tiles_of(x.M, kAnyTile), tiles_n = tiles_of(x.N, kTwo ? kAnyTile / 2 : kAnyTile);
  // (a launch has less than 2^32 threads)
  TFK_REQUIRE(tiles_m * tiles_n < (int64_t)1 << 24, TF_ERR_INVALID_ARG, "%s: result too large", who);
  return launch_kernel(product_any_kernel<InT, kTwo, Epilogue>, dim3((unsigned)(tiles_m * tiles_n)), dim3(kAnyThreads), 0, st, x,
                       whole_chunks<InT>(x, kTwo), (int)tiles_m, epilogue);
}

// ------------------------------------------------------------------------------------------
// Layout: what the products of a backward pass take transposed
// ------------------------------------------------------------------------------------------
// dst[c * pitch + r] = src[r * src_pitch + c] of 16-bit elements, for c < cols and r < padded_rows, zeros from `rows` on.
int launch_transpose_padded(const char* who, const void* src, int64_t src_pitch, void* dst, int64_t pitch, int64_t rows, int64_t cols,
                            int64_t padded_rows, hipStream_t st);
// count 16-bit elements of zero
int launch_zero_16bit(void* dst, int64_t count, hipStream_t st);

}  // namespace tfk
