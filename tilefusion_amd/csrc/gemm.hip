// GEMM macro kernel for gfx950: C[M,N] = A[M,K] * B[K,N] with A row-major and B handed over
// as its [N,K] buffer (column-major K x N), fp16 in, fp32 accumulate, fp32 or fp16 out.
//
// Counterpart of the reference's ke_gemm / ke_gemm_level1_pipeline / ke_gemm_level2_pipeline
// (include/kernels/gemm_device.cuh:110-419) and its host launcher (src/kernels/gemm.cu:63-142),
// re-designed for CDNA4:
//   * 64-lane wavefronts, v_mfma_f32_16x16x32_f16 base tiles, accumulators in the unified
//     512-entry register file (one wavefront per SIMD, 128x128 per wavefront at the big tile);
//   * both operands are K-contiguous, so an MFMA operand fragment is one 16-byte LDS read;
//   * tiles go global -> LDS without passing through VGPRs (global_load_lds_dwordx4) into an
//     XOR-swizzled LDS ring: a wavefront instruction always writes 1 KiB of consecutive LDS,
//     so the swizzle is applied on the global (source) side;
//   * the main kernel (gemm_ring64_kernel) uses 64-deep k-tiles so that every request fetches
//     whole 128-byte lines, keeps the ring in units of one operand, and issues its MFMAs from
//     assembly with a hand-placed instruction order (a lone wavefront issues one instruction
//     per 4 cycles: at most three others fit behind a 16-cycle MFMA); it comes with tiles from
//     128 x 128 to 256 x 256, for any M and N from one tile on and any K % 8 == 0 from 64 on;
//   * problems of few rows, columns or tiles run gemm_split_k_kernel, whose wavefronts share one small
//     tile and split K; a measured cost model picks the kernel and the tile;
//   * workgroup -> tile map keeps the workgroups of one XCD (one L2) on a compact block of
//     output tiles.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "product.hpp"

namespace tfk {
namespace {

template <int BM_, int BN_, int BK_, int WAVES_M_, int WAVES_N_>
struct GemmShape {
  static constexpr int BM = BM_, BN = BN_, BK = BK_;
  static constexpr int WAVES_M = WAVES_M_, WAVES_N = WAVES_N_;
  static constexpr int kWaves = WAVES_M * WAVES_N;
  static constexpr int kThreads = kWaves * kWaveSize;
  static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N;  // tile of one wavefront
  static constexpr int TM = WM / 32, TN = WN / 32;            // 32x32 MFMA tiles per wavefront
  static constexpr int kKSteps = BK / 16;
  static constexpr int kChunks = BK / 8;              // 16-byte chunks per tile row
  static constexpr int kRowsPer256B = 16 / kChunks;   // rows that share one pass over all banks
  static constexpr int kABytes = BM * BK * 2;
  static constexpr int kBBytes = BN * BK * 2;
  static_assert(WM % 32 == 0 && WN % 32 == 0 && BK % 16 == 0, "wavefront tile must be MFMA-sized");

  // Physical 16-byte chunk of logical chunk `c` in tile row `row`.  Sixteen consecutive rows
  // reading the same logical chunk land in sixteen different 16-byte bank groups.
  __host__ __device__ static constexpr int swizzle(int row, int c) {
    return c ^ ((row / kRowsPer256B) % kChunks);
  }
};

template <typename OutT>
TFK_DEVICE void store_out(OutT* p, float v) {
  if constexpr (sizeof(OutT) == 2) {
    *p = (OutT)v;
  } else {
    *p = v;
  }
}

template <typename InT> using in8_t = InT __attribute__((ext_vector_type(8)));
// MFMAs by operand type (half_t or bf16_t) for the bounds-checked kernel
template <typename InT>
TFK_DEVICE float16_t mfma32_t(in8_t<InT> a, in8_t<InT> b, float16_t c) {
  if constexpr (std::is_same_v<InT, bf16_t>) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  else return mfma_32x32x16(a, b, c);
}

// The kernel of large problems: M >= BM, N >= BN, and what ring64_multiply asks of K.
template <typename S, typename InT, typename OutT>
__global__ __launch_bounds__(S::kThreads) void gemm_ring64_kernel(
    const InT* __restrict__ A, const InT* __restrict__ B, OutT* __restrict__ C, int M,
    int N, int K, int tiles_m, int tiles_n) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int tile_m, tile_n;
  tile_of_block(blockIdx.x, gridDim.x, tiles_m, tiles_n, tile_m, tile_n);
  // The last tile of a row or column of tiles ends where C ends: it overlaps its neighbour, and the rows
  // and columns both compute are written twice with the same bits.  No request, product or store has
  // to know about edges.
  const int m0 = min(tile_m * S::BM, M - S::BM), n0 = min(tile_n * S::BN, N - S::BN);
  const int wm = wave / S::WAVES_N, wn = wave % S::WAVES_N, fr = lane & 15, fg = lane >> 4;
  float4_t acc[S::TM][S::TN];
  ring64_multiply<S, InT>(reinterpret_cast<const uint16_t*>(A), reinterpret_cast<const uint16_t*>(B), nullptr, K, m0, n0, lane, wave, smem, acc);
  // --- epilogue -----------------------------------------------------------------------------
  // acc[i][j][r] = C[.. + 16*i + l%16][.. + 16*j + 4*(l/16) + r].  For fp16 output the data is
  // re-dealt so that a store instruction writes 16 rows x 64 contiguous bytes with FOUR
  // ADJACENT lanes per row: the address unit merges adjacent lanes into one 64-byte access,
  // whereas lanes 16 apart cost one access each (measured: 64 accesses per instruction and
  // 9 k cycles of epilogue per wavefront).  Step 1: the 16-lane groups g and g^1 trade halves
  // of a pair of tiles (v_permlane16_swap), after which group 0/2 holds columns 0-7 / 8-15 of
  // tile j and group 1/3 the same of tile j+1, 16 bytes per lane.  Step 2: ds_bpermute moves
  // the 16 bytes of (row r, segment s) to lane 4*r + s.
  // (An odd N leaves the rows of C, and then the vectors of a store, without alignment.)
  typedef uint4_t out16B_t __attribute__((aligned(2)));
  typedef float4_t out4f_t __attribute__((aligned(4)));
  const int c_row0 = m0 + wm * S::WM;
  if constexpr (sizeof(OutT) == 2) {
    const int st_row = lane >> 2, st_seg = lane & 3;
    // segment s of a row lives in group {0, 2, 1, 3}[s] after step 1
    const int src_lane = st_row + 16 * (((st_seg & 1) << 1) | (st_seg >> 1));
    OutT* c_lane = C + (size_t)(c_row0 + st_row) * N + n0 + wn * S::WN + 8 * st_seg;
#pragma unroll
    for (int i = 0; i < S::TM; ++i)
#pragma unroll
      for (int j = 0; j < S::TN; j += 2) {
        typedef InT h2_t __attribute__((ext_vector_type(2)));
        unsigned x[2], y[2];
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          const h2_t hx = {(InT)acc[i][j][2 * d], (InT)acc[i][j][2 * d + 1]};
          const h2_t hy = {(InT)acc[i][j + 1][2 * d], (InT)acc[i][j + 1][2 * d + 1]};
          x[d] = __builtin_bit_cast(unsigned, hx);
          y[d] = __builtin_bit_cast(unsigned, hy);
#if defined(__HIP_DEVICE_COMPILE__)
          // x of the odd groups <-> y of the even groups
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
        *reinterpret_cast<out16B_t*>(c_lane + (size_t)(16 * i) * N + 16 * j) = v;
      }
  } else {
    const int c_col0 = n0 + wn * S::WN + 4 * fg;
#pragma unroll
    for (int i = 0; i < S::TM; ++i)
#pragma unroll
      for (int j = 0; j < S::TN; ++j)
        *reinterpret_cast<out4f_t*>(C + (size_t)(c_row0 + fr + 16 * i) * N + c_col0 + 16 * j) = acc[i][j];
  }
}

template <typename S, typename OutT, typename InT>
int launch_ring64(const void* A, const void* B, void* C, int M, int N, int K, hipStream_t st) {
  auto kern = gemm_ring64_kernel<S, InT, OutT>;
  constexpr int lds = S::kLdsBytes;
  static_assert(lds <= kMaxLdsBytes, "ring does not fit in LDS");
  TFK_LDS_OPT_IN(kern, lds);
  const int tiles_m = (M + S::BM - 1) / S::BM, tiles_n = (N + S::BN - 1) / S::BN;
  return launch_kernel(kern, dim3(tiles_m * tiles_n), dim3(S::kThreads), lds, st,
                       static_cast<const InT*>(A), static_cast<const InT*>(B),
                       static_cast<OutT*>(C), M, N, K, tiles_m, tiles_n);
}

template <typename S, typename InT, typename OutT>
__global__ __launch_bounds__(S::kThreads) void gemm_split_k_kernel(
    const InT* __restrict__ A, const InT* __restrict__ B, OutT* __restrict__ C, int M, int N, int K, int tiles_m,
    int tiles_n) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // consecutive tiles of one XCD share columns of B (m runs fastest)
  const int pid = xcd_major(blockIdx.x, tiles_m * tiles_n);
  const int m0 = pid % tiles_m * S::BM, n0 = pid / tiles_m * S::BN;
  split_k_multiply<S, InT>(reinterpret_cast<const uint16_t*>(A), reinterpret_cast<const uint16_t*>(B), nullptr, M, N, K, m0, n0, lane, wave, smem);
  const float* s_part = reinterpret_cast<const float*>(smem);
  for (int f = tid; f < S::BM * S::BN / 4; f += S::kThreads) {
    const int row = f / (S::BN / 4), col = f % (S::BN / 4) * 4;
    float4_t sum = *reinterpret_cast<const float4_t*>(s_part + row * S::kPitch + col);
#pragma unroll
    for (int w = 1; w < S::kWaves; ++w)
      sum += *reinterpret_cast<const float4_t*>(s_part + (w * S::BM + row) * S::kPitch + col);
    if (m0 + row >= M) continue;
    OutT* dst = C + (size_t)(m0 + row) * N + n0 + col;
    if (n0 + col + 4 <= N) {
      typedef OutT out4_t __attribute__((ext_vector_type(4)));
      typedef out4_t out4_any_t __attribute__((aligned(sizeof(OutT))));   // rows of an odd N have no alignment
      *reinterpret_cast<out4_any_t*>(dst) = out4_t{(OutT)sum[0], (OutT)sum[1], (OutT)sum[2], (OutT)sum[3]};
    } else {
#pragma unroll
      for (int r = 0; r < 3; ++r)
        if (n0 + col + r < N) dst[r] = (OutT)sum[r];
    }
  }
}

template <typename S, typename OutT, typename InT>
int launch_split_k(const void* A, const void* B, void* C, int M, int N, int K, hipStream_t st) {
  auto kern = gemm_split_k_kernel<S, InT, OutT>;
  static_assert(S::kLdsBytes <= kMaxLdsBytes, "rings do not fit in LDS");
  if constexpr (S::kLdsBytes > 64 * 1024) TFK_LDS_OPT_IN(kern, S::kLdsBytes);
  const int tiles_m = (M + S::BM - 1) / S::BM, tiles_n = (N + S::BN - 1) / S::BN;
  return launch_kernel(kern, dim3(tiles_m * tiles_n), dim3(S::kThreads), S::kLdsBytes, st, static_cast<const InT*>(A),
                       static_cast<const InT*>(B), static_cast<OutT*>(C), M, N, K, tiles_m, tiles_n);
}

// ------------------------------------------------------------------------------------------
// Operands that do not start at a 16-byte boundary, and short K with many outputs: any M, N; K % 8 == 0.  Register-staged,
// bounds-checked, one LDS stage.
// ------------------------------------------------------------------------------------------
template <typename S, typename OutT, typename InT>
__global__ __launch_bounds__(S::kThreads) void gemm_guarded_kernel(
    const InT* __restrict__ A, const InT* __restrict__ B, OutT* __restrict__ C, int M,
    int N, int K) {
  __shared__ __attribute__((aligned(16))) char sa[S::kABytes];
  __shared__ __attribute__((aligned(16))) char sb[S::kBBytes];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int m0 = blockIdx.x * S::BM, n0 = blockIdx.y * S::BN;
  const int wm = wave / S::WAVES_N, wn = wave % S::WAVES_N;
  const int fr = lane & 31, fg = lane >> 5;

  float16_t acc[S::TM][S::TN];
#pragma unroll
  for (int i = 0; i < S::TM; ++i)
#pragma unroll
    for (int j = 0; j < S::TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  for (int k0 = 0; k0 < K; k0 += S::BK) {
    for (int f = tid; f < S::BM * S::kChunks; f += S::kThreads) {
      const int row = f / S::kChunks, c = f % S::kChunks;
      const int gr = m0 + row, gk = k0 + c * 8;
      uint4_t v = {0u, 0u, 0u, 0u};
      if (gr < M && gk < K) v = *reinterpret_cast<const uint4_t*>(A + (size_t)gr * K + gk);
      *reinterpret_cast<uint4_t*>(sa + row * S::BK * 2 + S::swizzle(row, c) * 16) = v;
    }
    for (int f = tid; f < S::BN * S::kChunks; f += S::kThreads) {
      const int row = f / S::kChunks, c = f % S::kChunks;
      const int gr = n0 + row, gk = k0 + c * 8;
      uint4_t v = {0u, 0u, 0u, 0u};
      if (gr < N && gk < K) v = *reinterpret_cast<const uint4_t*>(B + (size_t)gr * K + gk);
      *reinterpret_cast<uint4_t*>(sb + row * S::BK * 2 + S::swizzle(row, c) * 16) = v;
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < S::kKSteps; ++kk) {
      in8_t<InT> af[S::TM], bf[S::TN];
#pragma unroll
      for (int i = 0; i < S::TM; ++i) {
        const int row = wm * S::WM + i * 32 + fr;
        af[i] = *reinterpret_cast<const in8_t<InT>*>(sa + row * S::BK * 2 + S::swizzle(row, 2 * kk + fg) * 16);
      }
#pragma unroll
      for (int j = 0; j < S::TN; ++j) {
        const int row = wn * S::WN + j * 32 + fr;
        bf[j] = *reinterpret_cast<const in8_t<InT>*>(sb + row * S::BK * 2 + S::swizzle(row, 2 * kk + fg) * 16);
      }
#pragma unroll
      for (int i = 0; i < S::TM; ++i)
#pragma unroll
        for (int j = 0; j < S::TN; ++j) acc[i][j] = mfma32_t<InT>(af[i], bf[j], acc[i][j]);
    }
    __syncthreads();
  }

#pragma unroll
  for (int i = 0; i < S::TM; ++i)
#pragma unroll
    for (int j = 0; j < S::TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = m0 + wm * S::WM + i * 32 + 8 * (r / 4) + 4 * fg + (r % 4);
        const int col = n0 + wn * S::WN + j * 32 + fr;
        if (row < M && col < N) store_out(C + (size_t)row * N + col, acc[i][j][r]);
      }
}

using ShapeSmall = GemmShape<64, 64, 32, 2, 2>;    // bounds-checked path

template <typename S, typename OutT, typename InT>
int launch_guarded(const void* A, const void* B, void* C, int M, int N, int K, hipStream_t st) {
  dim3 grid((M + S::BM - 1) / S::BM, (N + S::BN - 1) / S::BN);
  return launch_kernel(gemm_guarded_kernel<S, OutT, InT>, grid, dim3(S::kThreads), 0, st,
                       static_cast<const InT*>(A), static_cast<const InT*>(B),
                       static_cast<OutT*>(C), M, N, K);
}

// ------------------------------------------------------------------------------------------
// Which kernel: the one that a cost model expects to be done first.
//
// The tiles of a problem, the rounds in which 256 CUs do them and the k-tiles of each are known; what
// a k-tile costs is measured.  Microseconds, fitted to 264 problems (M 1-8192, N and K 64-8192, bf16, three
// to eight rotating operand sets; root mean square error 8-16% a kernel).  Taking the expected best is
// 3.5% behind taking the measured best of all kernels on average, and never 2x.
//   ring kernels:    start + rounds * (round + ktiles * (step + shared * fill + unaligned))
//     `shared` is what a CU pays for the others' requests, times how much of the chip a round fills: a
//     128 x 128 tile's k-tile takes 0.30 us with few workgroups, 0.56 with one on every CU (its
//     32 KiB a k-tile then ask 15 TB/s of the L2s), a 256 x 256 tile's 0.85 and 1.6 for four times the work.
//   split-K kernels: start + max(rounds * ktiles of one wavefront * step,
//                                tiles per CU * ktiles * (shared + unaligned)) + tiles per CU * round
//     the latency of one workgroup's chain, or the rate at which a CU takes in all of its workgroups.
// `unaligned` applies where K is no multiple of 64: rows then start anywhere in a 128-byte line.
// ------------------------------------------------------------------------------------------
struct GemmKernel {
  int bm, bn, waves;        // output tile; wavefronts that share its K (ring kernels: 1)
  int per_cu;               // workgroups that a CU holds
  bool ring;
  float start, round, step, shared, unaligned;
  int64_t min_tiles = 0, max_tiles = INT64_MAX;   // where the figures apply
};
constexpr GemmKernel kGemmKernels[] = {
    {16, 16, 4, 4, false, 2.25f, 0.18f, 0.208f, 0.056f, 0.005f},
    {16, 16, 8, 2, false, 2.32f, 0.42f, 0.279f, 0.057f, 0.005f},
    {32, 16, 4, 3, false, 2.36f, 0.28f, 0.259f, 0.089f, 0.009f},
    {32, 32, 1, 8, false, 2.41f, 0.13f, 0.294f, 0.100f, 0.050f},
    {32, 32, 4, 2, false, 2.30f, 0.50f, 0.342f, 0.128f, 0.012f},
    {64, 32, 4, 1, false, 2.42f, 1.44f, 0.527f, 0.235f, 0.042f},
    {64, 64, 4, 1, false, 2.87f, 2.12f, 0.785f, 0.324f, 0.092f},
    {128, 128, 1, 1, true, 0.58f, 3.23f, 0.298f, 0.260f, 0.205f},              // requests 4 tiles ahead
    {128, 128, 1, 1, true, 0.92f, 2.29f, 0.386f, 0.284f, 0.129f, 0, 256},      // 2 tiles ahead: starts sooner
    {128, 128, 1, 2, true, 2.30f, 1.51f, 0.160f, 0.349f, 0.176f, 257},         // ... and shares a CU in pairs
    {192, 128, 1, 1, true, 0.21f, 3.75f, 0.426f, 0.331f, 0.212f},
    {192, 192, 1, 1, true, 0.00f, 4.93f, 0.529f, 0.509f, 0.233f},
    {256, 128, 1, 1, true, 0.00f, 4.60f, 0.496f, 0.447f, 0.266f},
    {256, 192, 1, 1, true, 0.00f, 5.84f, 0.670f, 0.583f, 0.240f},
    {256, 256, 1, 1, true, 0.00f, 6.63f, 0.851f, 0.729f, 0.216f},
};
constexpr int kNumGemmKernels = sizeof(kGemmKernels) / sizeof(kGemmKernels[0]);

// Rows that start anywhere in a line: from K = 328 on these ring kernels fetch whole lines (Ring64Shape::kLines), which costs them a
// segment more at first and saves them 0.13-0.27 us a k-tile. Microseconds as above, fitted to 60 problems (M, N 128-8192, K
// 328-8192; 4-5% root mean square); picks are 2% behind the best of all kernels on average. us, k-tiles that start where rows
// start / whole lines: 1500 x 1500 x 3000, 128 x 128 31.0 / 22.6; 700 x 4096 x 4104 40.2 / 30.5; 2999 x 1544 x 1032,
// 192 x 128 18.7 / 17.3; 3333 x 2288 x 1944, 256 x 128 39.3 / 33.5, 192 x 192 35.3 / 33.6. (The larger tiles leave no room for a third
// segment, and two workgroups of 128 x 128 none for each other; below K = 328 the further segment costs as much as it saves:
// 8192 x 1000 x 328 14.0 / 13.5.)
constexpr int kLinesFrom = 328;
bool takes_lines(int K) { return K % 64 != 0 && K >= kLinesFrom; }
struct LinesKernel {
  int index;                // into kGemmKernels
  float start, round, step, shared;
};
constexpr LinesKernel kLinesKernels[] = {
    {7, 1.63f, 3.67f, 0.317f, 0.139f},
    {10, 1.32f, 4.65f, 0.430f, 0.167f},
    {11, 0.60f, 5.44f, 0.695f, 0.269f},
    {12, 1.36f, 4.11f, 0.660f, 0.281f},
};

// A tile of 160 x 128, figures between those of 128 x 128 and 192 x 128, for grids that the one gives a second round and the
// other leaves CUs idle on (2999 x 1544 x 1032: 208 tiles of 192 rows, 247 of 160). It takes the place of one of these two where it is
// expected to be done sooner. us, the pick / it, of one run each: 2999 x 1544 x 1032 17.3 / 16.6, 613 x 7874 x 2040 26.1 / 22.9, 2547 x
// 1739 x 6712 63.5 / 59.1; 56 such problems take 0.923 of the time (1.00 at most). Of K a multiple of 64, from 256 on: 0.961 over 119
// (1.02 at most): 2466 x 1722 x 256 8.4 / 7.8, 1571 x 3014 x 3008 33.3 / 30.0, 587 x 7483 x 2496 28.3 / 25.8. Not in place of the larger
// tiles: whole lines of 192 x 192, which the model would have it replace now and then, are ahead of it by 5% on average (10% at most)
// over 52 problems (5288 x 4630 x 1768, fp32 result, 94.8 / 104.4).
constexpr LinesKernel kBetween = {-1, 1.45f, 4.15f, 0.373f, 0.153f};
constexpr int kBetweenRows = 160, kBetweenColumns = 128;
constexpr GemmKernel kBetweenWhole = {kBetweenRows, kBetweenColumns, 1, 1, true, 0.40f, 3.49f, 0.362f, 0.296f, 0.f};

float expected_us(const GemmKernel& g, int64_t tiles, int ktiles, bool unaligned_rows, const LinesKernel* lines) {
  const int64_t rounds = (tiles + 256 * g.per_cu - 1) / (256 * g.per_cu);
  const float unaligned = unaligned_rows ? g.unaligned : 0.f;
  const float per_cu = tiles / 256.f;
  if (g.ring) {
    const float fill = std::min(1.f, per_cu / (rounds * g.per_cu));
    if (lines != nullptr) return lines->start + rounds * (lines->round + ktiles * (lines->step + lines->shared * fill));
    return g.start + rounds * g.per_cu * (g.round + ktiles * (g.step + g.shared * fill + unaligned));
  }
  const int chain = (ktiles + g.waves - 1) / g.waves;
  return g.start + std::max(rounds * chain * g.step, per_cu * ktiles * (g.shared + unaligned)) + per_cu * g.round;
}

// Up to K = 128 (16-bit results: 120) with many outputs, what counts is how C leaves, in which the table above does not go by the type (it was
// fitted to 16-bit results), and the bounds-checked kernel is in the race: its k-tiles are 32 deep, and
// several of its workgroups share a CU.  Microseconds, fitted to 521 problems (7 to 13% root mean square): start +
// round per round of the chip + per tile of a CU: tile, depth a k-tile, wide for an fp32 result, odd_k where K is no
// multiple of 64, odd_n where rows of C do not start at 16-byte boundaries.  Picks are 1.6% behind the best
// of all kernels on average and 20% at most; those of the table above 8% and 83% (517 x 3008 x 64, fp32 result:
// 128 x 128 ring 5.9 us, bounds-checked kernel 4.05; 1664 x 1472 x 64 6.2 and 4.8).
struct ShortKKernel {
  int index;                // into kGemmKernels; behind its end: the bounds-checked kernel
  int bm, bn, k_tile;
  float start, round, tile, depth, wide, odd_k, odd_n;
};
constexpr ShortKKernel kShortKKernels[] = {
    {3, 32, 32, 64, 2.93f, 0.f, 0.163f, 0.064f, 0.070f, 0.f, 0.010f},
    {8, 128, 128, 64, 3.34f, 1.31f, 0.303f, 0.415f, 1.54f, 0.178f, 0.277f},
    {11, 192, 192, 64, 2.83f, 3.90f, 0.288f, 0.896f, 3.32f, 0.584f, 0.811f},
    {12, 256, 128, 64, 2.54f, 3.80f, 0.153f, 0.853f, 3.18f, 0.559f, 0.640f},
    {13, 256, 192, 64, 2.68f, 5.32f, 0.f, 1.262f, 4.89f, 0.768f, 0.871f},
    {kNumGemmKernels, 64, 64, 32, 3.23f, 0.f, 0.254f, 0.168f, 0.296f, 0.f, 0.139f},
};

int pick_short_k_kernel(int M, int N, int K, bool c_is_f32) {
  const int64_t row_bytes = (int64_t)N * (c_is_f32 ? 4 : 2);
  int best = 3;
  float best_us = INFINITY;
#pragma unroll
  for (const ShortKKernel& g : kShortKKernels) {
    if (kGemmKernels[g.index % kNumGemmKernels].ring && (M < g.bm || N < g.bn || K < 64)) continue;
    if (g.index == kNumGemmKernels) {
      if (N > 65535 * 64) continue;   // its grid has columns of tiles in y
      // Its tiles are 64 columns wide, so rows of C that are no whole 128-byte lines leave it in parts of lines, which
      // costs from ~32 MiB of C on (5898 x 5498 x 64, fp32 result: 58 us, 128 x 128 ring 33; 8192 x 4160 x 64 33 and 36).
      if (K >= 64 && row_bytes % 128 != 0 && M * row_bytes > (int64_t)32 << 20) continue;
    }
    const int64_t tiles = (int64_t)((M + g.bm - 1) / g.bm) * ((N + g.bn - 1) / g.bn);
    const float per_tile = g.tile + (K + g.k_tile - 1) / g.k_tile * g.depth + (c_is_f32 ? g.wide : 0.f) +
                           (K % 64 != 0 ? g.odd_k : 0.f) + (row_bytes % 16 != 0 ? g.odd_n : 0.f);
    const float us = g.start + (tiles + 255) / 256 * g.round + tiles / 256.f * per_tile;
    if (us < best_us) {
      best = g.index;
      best_us = us;
    }
  }
  return best;
}

// What runs in place of `pick`, a kernel of the table: the tile between where it is ahead of a ring kernel of its kind, the same tile with whole
// lines where rows start anywhere in one. Their positions are those behind the bounds-checked kernel's.
constexpr int kLinesAt = kNumGemmKernels + 1, kBetweenWholeAt = kLinesAt + sizeof(kLinesKernels) / sizeof(kLinesKernels[0]),
              kBetweenLinesAt = kBetweenWholeAt + 1, kNumGemmLaunchers = kBetweenLinesAt + 1;
int stand_in(int pick, int M, int N, int K) {
  const bool lines = takes_lines(K);
  int at = pick;
  const LinesKernel* of_pick = nullptr;
  if (lines) {
    for (const LinesKernel& l : kLinesKernels)
      if (l.index == pick) {
        of_pick = &l;
        at = kLinesAt + (int)(&l - kLinesKernels);
      }
    if (of_pick == nullptr) return pick;
  } else if (K % 64 != 0 || K < 256 || pick < 7) {
    return pick;
  }
  if (pick > 10) return at;   // (tiles that are larger both ways)
  if (M < kBetweenRows || N < kBetweenColumns) return at;
  const GemmKernel& g = kGemmKernels[pick];
  const int ktiles = (K + 63) / 64;
  auto expected = [&](const GemmKernel& k, const LinesKernel* l) {
    return expected_us(k, (int64_t)((M + k.bm - 1) / k.bm) * ((N + k.bn - 1) / k.bn), ktiles, lines, l);
  };
  if (expected(kBetweenWhole, lines ? &kBetween : nullptr) < expected(g, of_pick)) return lines ? kBetweenLinesAt : kBetweenWholeAt;
  return at;
}

// The kernel of a call whose operands start at 16-byte boundaries: a position in the launchers of dispatch().
int pick_gemm_kernel(int M, int N, int K, bool c_is_f32) {
  // (2^35 elements of C with a K below the ring kernels' are more threads than a launch of the split-K kernels may have)
  if (K < 64 && (int64_t)M * N >= (int64_t)1 << 35) return kNumGemmKernels;
  if (K <= (c_is_f32 ? 128 : 120) && (int64_t)((M + 63) / 64) * ((N + 63) / 64) >= 96) return pick_short_k_kernel(M, N, K, c_is_f32);
  int best = 0, best_plain = 0;
  float best_us = INFINITY, best_plain_us = INFINITY;
  const int ktiles = (K + 63) / 64;
#pragma unroll   // the divisions are by constants then
  for (int i = 0; i < kNumGemmKernels; ++i) {
    const GemmKernel& g = kGemmKernels[i];
    if (g.ring && (M < g.bm || N < g.bn || K < 64)) continue;   // (what gemm_ring64_kernel asks for)
    const int64_t tiles = (int64_t)((M + g.bm - 1) / g.bm) * ((N + g.bn - 1) / g.bn);
    if (tiles < g.min_tiles || tiles > g.max_tiles) continue;
    const float plain_us = expected_us(g, tiles, ktiles, K % 64 != 0, nullptr);
    float us = plain_us;
    if (takes_lines(K))
      for (const LinesKernel& l : kLinesKernels)
        if (l.index == i) us = expected_us(g, tiles, ktiles, true, &l);
    if (us < best_us) {
      best = i;
      best_us = us;
    }
    if (plain_us < best_plain_us) {
      best_plain = i;
      best_plain_us = plain_us;
    }
  }
  // Where tiles of 256 x 192 or 256 x 256 would be picked if there were no whole lines they are: the two fits do not compare well there
  // (us, those / the whole-line tile that is expected to be ahead: 5530 x 3814 x 1184 55.0 / 68.5, 7568 x 5021 x 1424 113 / 135, 3727 x 6430 x
  // 1256 66 / 76; 80 such problems 1.077 of the time with whole lines, those tiles 0.3% behind the best of all).
  if (best_plain == 13 || best_plain == 14) return best_plain;
  return stand_in(best, M, N, K);
}

}  // namespace

int pick_table_kernel(int64_t M, int64_t N, int64_t K, unsigned allowed, float* expected) {
  int best = 0;
  float best_us = INFINITY;
  const int ktiles = (int)((K + 63) / 64);
#pragma unroll
  for (int i = 0; i < kNumGemmKernels; ++i) {
    const GemmKernel& g = kGemmKernels[i];
    if (!(allowed >> i & 1) || (g.ring && (M < g.bm || N < g.bn || K < 64))) continue;
    const int64_t tiles = ((M + g.bm - 1) / g.bm) * ((N + g.bn - 1) / g.bn);
    if (tiles < g.min_tiles || tiles > std::min(g.max_tiles, kMaxTiles)) continue;
    const float us = expected_us(g, tiles, ktiles, K % 64 != 0, nullptr);
    if (us < best_us) {
      best = i;
      best_us = us;
    }
  }
  *expected = best_us;
  return best;
}

float expected_table_us(int kernel, int64_t tiles, int64_t K) {
  return expected_us(kGemmKernels[kernel], tiles, (int)((K + 63) / 64), K % 64 != 0, nullptr);
}

namespace {

template <typename OutT, typename InT>
int dispatch(const void* A, const void* B, void* C, int M, int N, int K, hipStream_t st) {
  using Launcher = int (*)(const void*, const void*, void*, int, int, int, hipStream_t);
  static constexpr Launcher kLaunchers[] = {
      launch_split_k<SplitKShape<1, 1, 4>, OutT, InT>, launch_split_k<SplitKShape<1, 1, 8>, OutT, InT>,
      launch_split_k<SplitKShape<2, 1, 4>, OutT, InT>, launch_split_k<SplitKShape<2, 2, 1>, OutT, InT>,
      launch_split_k<SplitKShape<2, 2, 4>, OutT, InT>, launch_split_k<SplitKShape<4, 2, 4>, OutT, InT>,
      launch_split_k<SplitKShape<4, 4, 4>, OutT, InT>,
      launch_ring64<Ring64Shape<128, 128, 4>, OutT, InT>, launch_ring64<Ring64Shape<128, 128, 2>, OutT, InT>,
      launch_ring64<Ring64Shape<128, 128, 2>, OutT, InT>, launch_ring64<Ring64Shape<192, 128, 2>, OutT, InT>,
      launch_ring64<Ring64Shape<192, 192, 2>, OutT, InT>, launch_ring64<Ring64Shape<256, 128, 2>, OutT, InT>,
      launch_ring64<Ring64Shape<256, 192, 2>, OutT, InT>, launch_ring64<Ring64Shape<256, 256, 2>, OutT, InT>,
      launch_guarded<ShapeSmall, OutT, InT>,
      launch_ring64<Ring64Shape<128, 128, 2, 5>, OutT, InT>, launch_ring64<Ring64Shape<192, 128, 2, 4>, OutT, InT>,
      launch_ring64<Ring64Shape<192, 192, 2, 3>, OutT, InT>, launch_ring64<Ring64Shape<256, 128, 2, 3>, OutT, InT>,
      launch_ring64<Ring64Shape<kBetweenRows, kBetweenColumns, 2>, OutT, InT>,
      launch_ring64<Ring64Shape<kBetweenRows, kBetweenColumns, 2, 4>, OutT, InT>,
  };
  static_assert(sizeof(kLaunchers) / sizeof(kLaunchers[0]) == kNumGemmLaunchers,
                "a launcher per row of kGemmKernels, the bounds-checked kernel, one per row of kLinesKernels, the two of 160 rows");
  // LDS-direct requests take 16 bytes at a 16-byte boundary.
  if ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(B)) % 16 != 0)
    return kLaunchers[kNumGemmKernels](A, B, C, M, N, K, st);
  return kLaunchers[pick_gemm_kernel(M, N, K, sizeof(OutT) == 4)](A, B, C, M, N, K, st);
}

}  // namespace
}  // namespace tfk

namespace tfk {
namespace {
int check_gemm_args(const char* who, const void* A, const void* B, const void* C, int64_t M, int64_t N, int64_t K,
                    int tm, int tn, int tk, int num_stages, int pipeline_level) {
  TFK_REQUIRE(A && B && C, TF_ERR_INVALID_ARG, "%s: null pointer", who);
  TFK_REQUIRE(M > 0 && N > 0 && K > 0, TF_ERR_INVALID_ARG, "%s: M, N, K must be positive", who);
  TFK_REQUIRE(M < (1 << 30) && N < (1 << 30) && K < (1 << 22), TF_ERR_INVALID_ARG, "%s: dimension too large", who);
  TFK_REQUIRE(tm > 0 && tn > 0 && tk > 0, TF_ERR_INVALID_ARG, "%s: tile sizes must be positive", who);
  TFK_REQUIRE(M % tm == 0 && N % tn == 0 && K % tk == 0, TF_ERR_INVALID_ARG,
              "%s: tile [%d,%d,%d] does not divide problem [%lld,%lld,%lld]", who, tm, tn, tk,
              (long long)M, (long long)N, (long long)K);
  TFK_REQUIRE(num_stages >= 1 && num_stages <= 3, TF_ERR_INVALID_ARG, "%s: num_stages must be 1, 2 or 3", who);
  TFK_REQUIRE(pipeline_level >= 0 && pipeline_level <= 2, TF_ERR_INVALID_ARG,
              "%s: pipeline_level must be 0, 1 or 2", who);
  return TF_OK;
}
}  // namespace
}  // namespace tfk

extern "C" int tf_gemm_f16(const void* A, const void* B, void* C, int c_is_f16, int64_t M,
                           int64_t N, int64_t K, int tm, int tn, int tk, int num_stages,
                           int pipeline_level, void* stream) {
  using namespace tfk;
  if (int rc = check_gemm_args("tf_gemm_f16", A, B, C, M, N, K, tm, tn, tk, num_stages, pipeline_level)) return rc;
  TFK_REQUIRE(K % 8 == 0, TF_ERR_UNSUPPORTED, "tf_gemm_f16: K (%lld) must be a multiple of 8",
              (long long)K);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (c_is_f16) return dispatch<half_t, half_t>(A, B, C, (int)M, (int)N, (int)K, st);
  return dispatch<float, half_t>(A, B, C, (int)M, (int)N, (int)K, st);
}

extern "C" int tf_gemm(const void* A, const void* B, void* C, int dtype, int c_is_f32, int64_t M, int64_t N,
                       int64_t K, int tm, int tn, int tk, int num_stages, int pipeline_level, void* stream) {
  using namespace tfk;
  if (dtype == TF_DTYPE_F16)
    return tf_gemm_f16(A, B, C, c_is_f32 ? 0 : 1, M, N, K, tm, tn, tk, num_stages, pipeline_level, stream);
  TFK_REQUIRE(dtype == TF_DTYPE_BF16, TF_ERR_UNSUPPORTED, "tf_gemm: dtype must be TF_DTYPE_F16 or TF_DTYPE_BF16");
  if (int rc = check_gemm_args("tf_gemm", A, B, C, M, N, K, tm, tn, tk, num_stages, pipeline_level)) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  // bf16: the same kernels with the bf16 MFMAs (every kernel of this file is a template of the
  // operand type)
  TFK_REQUIRE(K % 8 == 0, TF_ERR_UNSUPPORTED, "tf_gemm: K (%lld) must be a multiple of 8", (long long)K);
  if (c_is_f32) return dispatch<float, bf16_t>(A, B, C, (int)M, (int)N, (int)K, st);
  return dispatch<bf16_t, bf16_t>(A, B, C, (int)M, (int)N, (int)K, st);
}

extern "C" int tf_gemm_kernel_index(int64_t M, int64_t N, int64_t K, int c_is_f32) {
  if (M <= 0 || N <= 0 || K <= 0 || M >= (1 << 30) || N >= (1 << 30) || K >= (1 << 22)) return -1;
  return tfk::pick_gemm_kernel((int)M, (int)N, (int)K, c_is_f32 != 0);
}

extern "C" int tf_product_kernel_index(int64_t M, int64_t N, int64_t K, int two) {
  if (M <= 0 || N <= 0 || K <= 0 || M >= (1 << 30) || N >= (1 << 30) || K >= (1 << 22)) return -1;
  return tfk::plan_product(M, N, K, two != 0).kernel;
}

extern "C" int tf_product_cols_plan(int64_t M, int64_t N, int64_t rows, int* parts) {
  if (M <= 0 || N <= 0 || rows <= 0 || parts == nullptr) return -1;
  const tfk::ColsPlan plan = tfk::plan_cols({M, N, tfk::tiles_of(rows, 64)});
  *parts = plan.splits;
  return plan.shape;
}

extern "C" int tf_product_pair_plan(int64_t M, int64_t N, int64_t rows, int64_t M2, int64_t N2, int64_t rows2, int* parts, int* parts2) {
  if (M <= 0 || N <= 0 || rows <= 0 || M2 <= 0 || N2 <= 0 || rows2 <= 0 || parts == nullptr || parts2 == nullptr) return -1;
  const tfk::ColsSize one = {M, N, tfk::tiles_of(rows, 64)}, other = {M2, N2, tfk::tiles_of(rows2, 64)};
  const tfk::PairPlan plan = tfk::plan_pair(tfk::plan_cols(one), one, tfk::plan_cols(other), other);
  *parts = plan.x.splits;
  *parts2 = plan.w.splits;
  return plan.together ? plan.x.shape : -1;
}
