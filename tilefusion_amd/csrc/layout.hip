// Transposed copies with their rows completed by zeros: what the products of a backward pass, which sum over tokens or over columns
// of a weight, take as rows.
#include "product.hpp"

namespace tfk {
namespace {

constexpr int kTile = 64, kThreads = 256;

// Bound by memory: 64 x 64 elements of 16 bits through LDS, rows of 128 bytes on either side.  A pitch of 66 elements (33 words)
// puts the words that the lanes of a wavefront read down a column into different banks.
__global__ __launch_bounds__(kThreads) void transpose_padded_kernel(const uint16_t* __restrict__ src, int64_t src_pitch,
                                                                    uint16_t* __restrict__ dst, int64_t pitch, int rows, int cols, int padded_rows,
                                                                    int tiles_c) {
  __shared__ uint16_t tile[kTile][kTile + 2];
  const int r0 = blockIdx.x / tiles_c * kTile, c0 = blockIdx.x % tiles_c * kTile;
  for (int f = threadIdx.x; f < kTile * kTile; f += kThreads) {
    const int r = f / kTile, c = f % kTile;
    tile[r][c] = r0 + r < rows && c0 + c < cols ? src[(size_t)(r0 + r) * src_pitch + c0 + c] : 0;
  }
  __syncthreads();
  for (int f = threadIdx.x; f < kTile * kTile; f += kThreads) {
    const int c = f / kTile, r = f % kTile;
    if (c0 + c < cols && r0 + r < padded_rows) dst[(size_t)(c0 + c) * pitch + r0 + r] = tile[r][c];
  }
}

__global__ __launch_bounds__(kThreads) void zero_kernel(uint16_t* dst, int64_t count) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < count; i += (int64_t)gridDim.x * kThreads) dst[i] = 0;
}

__global__ __launch_bounds__(kThreads) void zero_columns_kernel(uint16_t* dst, int64_t pitch, int64_t rows, int from, int width) {
  const int64_t count = rows * width;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < count; i += (int64_t)gridDim.x * kThreads)
    dst[i / width * pitch + from + i % width] = 0;
}

}  // namespace

int launch_transpose_padded(const char* who, const void* src, int64_t src_pitch, void* dst, int64_t pitch, int64_t rows, int64_t cols,
                            int64_t padded_rows, hipStream_t st) {
  const int64_t tiles_r = tiles_of(padded_rows, kTile), tiles_c = tiles_of(cols, kTile);
  TFK_REQUIRE(tiles_r * tiles_c < (int64_t)1 << 24, TF_ERR_INVALID_ARG, "%s: matrix too large", who);
  return launch_kernel(transpose_padded_kernel, dim3((unsigned)(tiles_r * tiles_c)), dim3(kThreads), 0, st, static_cast<const uint16_t*>(src),
                       src_pitch, static_cast<uint16_t*>(dst), pitch, (int)rows, (int)cols, (int)padded_rows, (int)tiles_c);
}

int launch_zero_16bit(void* dst, int64_t count, hipStream_t st) {
  if (count == 0) return TF_OK;
  const int64_t blocks = std::min<int64_t>(tiles_of(count, kThreads), 4096);
  return launch_kernel(zero_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, st, static_cast<uint16_t*>(dst), count);
}

int launch_zero_columns(const char*, void* dst, int64_t pitch, int64_t rows, int64_t from, int64_t to, hipStream_t st) {
  const int64_t blocks = std::min<int64_t>(tiles_of(rows * (to - from), kThreads), 4096);
  return launch_kernel(zero_columns_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, st, static_cast<uint16_t*>(dst), pitch, rows, (int)from,
                       (int)(to - from));
}

}  // namespace tfk
