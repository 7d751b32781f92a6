// What the products of product.hpp need beside themselves: rows that 16-byte requests can walk, zeros, sums of partial results.
#include "product.hpp"

namespace tfk {
namespace {

constexpr int kThreads = 256;

struct CopyArgs {
  const char* src[3];
  uint4_t* dst[3];
  int64_t rows[3], end[3];   // rows of src; chunks of all matrices up to and with this one
};
// Bound by memory; 16 bytes a lane.  (Unaligned 16-byte loads are one instruction, of one or two lines.)
__global__ __launch_bounds__(kThreads) void copy_rows_kernel(CopyArgs x, int64_t bytes, int chunks, int64_t count) {
  typedef uint4_t any16B_t __attribute__((aligned(1)));
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < count; i += (int64_t)gridDim.x * kThreads) {
    const int which = i < x.end[0] ? 0 : i < x.end[1] ? 1 : 2;
    const int64_t in = which == 0 ? i : i - x.end[which - 1];
    const int64_t row = in / chunks, at = (in - row * chunks) * 16;
    const char* const from = x.src[which] + row * bytes + at;
    uint4_t v = {0u, 0u, 0u, 0u};
    if (row < x.rows[which] && at + 16 <= bytes) {
      v = *reinterpret_cast<const any16B_t*>(from);
    } else if (row < x.rows[which]) {
#pragma unroll
      for (int t = 0; t < 16; ++t)
        if (at + t < bytes) v[t / 4] |= (unsigned)(uint8_t)from[t] << (8 * (t % 4));
    }
    x.dst[which][in] = v;
  }
}

__global__ __launch_bounds__(kThreads) void zero_kernel(uint16_t* dst, int64_t count) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < count; i += (int64_t)gridDim.x * kThreads) dst[i] = 0;
}

// Four columns a lane.  A wavefront takes every fourth part, several on their way at a time (21 x 256 sums of 64 parts: 20 us a part after the other, 5
// so); the four sums are added in their order.
constexpr int kSumChunks = 64, kSumWays = kThreads / kSumChunks;
template <typename T>
__global__ __launch_bounds__(kThreads) void sum_parts_kernel(const float* __restrict__ parts, int64_t part, int64_t pitch, int splits, int64_t first,
                                                             int64_t count, int N, int chunks, T* __restrict__ out, Factors factors) {
  __shared__ float4_t s_sum[kSumWays][kSumChunks];
  const float common = factors.common();
  typedef T out4_t __attribute__((ext_vector_type(4)));
  typedef out4_t out4_any_t __attribute__((aligned(sizeof(T))));
  const int lane = threadIdx.x % kSumChunks, way = threadIdx.x / kSumChunks;
  for (int64_t base = (int64_t)blockIdx.x * kSumChunks; base < count; base += (int64_t)gridDim.x * kSumChunks) {
    const int64_t i = min(base + lane, count - 1), row = i / chunks;
    const int col = (int)(i - row * chunks) * 4;
    const float* const from = parts + (first + row) * pitch + col;
    float4_t v = {0.f, 0.f, 0.f, 0.f};
    int s = way;
    for (; s + 3 * kSumWays < splits; s += 4 * kSumWays) {
      float4_t x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) x[u] = *reinterpret_cast<const float4_t*>(from + (s + u * kSumWays) * part);
#pragma unroll
      for (int u = 0; u < 4; ++u) v += x[u];
    }
    for (; s < splits; s += kSumWays) v += *reinterpret_cast<const float4_t*>(from + s * part);
    s_sum[way][lane] = v;
    __syncthreads();
    if (way == 0 && base + lane < count) {
#pragma unroll
      for (int w = 1; w < kSumWays; ++w) v += s_sum[w][lane];
      v *= common * factors.of_row(row);
      T* const to = out + row * N + col;
      if (col + 4 <= N) {
        *reinterpret_cast<out4_any_t*>(to) = out4_t{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
      } else {
#pragma unroll
        for (int t = 0; t < 3; ++t)
          if (col + t < N) to[t] = (T)v[t];
      }
    }
    __syncthreads();
  }
}

unsigned blocks_for(int64_t items) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>(tiles_of(items, kThreads), 8192)); }

}  // namespace

int launch_copy_rows(const RowsToCopy* matrices, int count, int64_t bytes, int64_t pitch, hipStream_t st) {
  CopyArgs x{};
  int64_t end = 0;
  for (int m = 0; m < 3; ++m) {
    if (m < count) {
      x.src[m] = static_cast<const char*>(matrices[m].src);
      x.dst[m] = static_cast<uint4_t*>(matrices[m].dst);
      x.rows[m] = matrices[m].rows;
      end += matrices[m].padded_rows * (pitch / 16);
    }
    x.end[m] = end;
  }
  return launch_kernel(copy_rows_kernel, dim3(blocks_for(end)), dim3(kThreads), 0, st, x, bytes, (int)(pitch / 16), end);
}

int launch_zero_16bit(void* dst, int64_t count, hipStream_t st) {
  if (count == 0) return TF_OK;
  return launch_kernel(zero_kernel, dim3(blocks_for(count)), dim3(kThreads), 0, st, static_cast<uint16_t*>(dst), count);
}

template <typename T>
int launch_sum_parts(const float* parts, const PartsRoom& room, int splits, int64_t first, int64_t M, int64_t N, T* out, const Factors& factors,
                     hipStream_t st) {
  const int64_t chunks = tiles_of(N, 4), count = (M - first) * chunks;
  return launch_kernel(sum_parts_kernel<T>, dim3(blocks_for(tiles_of(count, kSumChunks) * kThreads)), dim3(kThreads), 0, st, parts, room.rows * room.pitch, room.pitch, splits, first, count,
                       (int)N, (int)chunks, out, factors);
}
template int launch_sum_parts<half_t>(const float*, const PartsRoom&, int, int64_t, int64_t, int64_t, half_t*, const Factors&, hipStream_t);
template int launch_sum_parts<bf16_t>(const float*, const PartsRoom&, int, int64_t, int64_t, int64_t, bf16_t*, const Factors&, hipStream_t);

}  // namespace tfk
