// What the products of product.hpp need beside themselves: rows that 16-byte requests can walk, zeros, sums of partial results.
#include "product.hpp"

namespace tfk {
namespace {

constexpr int kThreads = 256;

// Bound by memory; 16 bytes a lane.  (Unaligned 16-byte loads are one instruction, of one or two lines.)
__global__ __launch_bounds__(kThreads) void copy_rows_kernel(const char* __restrict__ src, int64_t bytes, int64_t rows, uint4_t* __restrict__ dst,
                                                             int chunks, int64_t count) {
  typedef uint4_t any16B_t __attribute__((aligned(1)));
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < count; i += (int64_t)gridDim.x * kThreads) {
    const int64_t row = i / chunks, at = (i - row * chunks) * 16;
    const char* const from = src + row * bytes + at;
    uint4_t v = {0u, 0u, 0u, 0u};
    if (row < rows && at + 16 <= bytes) {
      v = *reinterpret_cast<const any16B_t*>(from);
    } else if (row < rows) {
#pragma unroll
      for (int t = 0; t < 16; ++t)
        if (at + t < bytes) v[t / 4] |= (unsigned)(uint8_t)from[t] << (8 * (t % 4));
    }
    dst[i] = v;
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

// Four columns a lane; the parts are added in their order.
template <typename T>
__global__ __launch_bounds__(kThreads) void sum_parts_kernel(const float* __restrict__ parts, int64_t part, int64_t pitch, int splits, int64_t first,
                                                             int64_t count, int N, int chunks, T* __restrict__ out, const Scale* scale) {
  const float by = scale != nullptr ? scale->out : 1.f;
  typedef T out4_t __attribute__((ext_vector_type(4)));
  typedef out4_t out4_any_t __attribute__((aligned(sizeof(T))));
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < count; i += (int64_t)gridDim.x * kThreads) {
    const int64_t row = i / chunks;
    const int col = (int)(i - row * chunks) * 4;
    const float* const from = parts + (first + row) * pitch + col;
    float4_t v = *reinterpret_cast<const float4_t*>(from);
    for (int s = 1; s < splits; ++s) v += *reinterpret_cast<const float4_t*>(from + s * part);
    v *= by;
    T* const to = out + row * N + col;
    if (col + 4 <= N) {
      *reinterpret_cast<out4_any_t*>(to) = out4_t{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    } else {
#pragma unroll
      for (int t = 0; t < 3; ++t)
        if (col + t < N) to[t] = (T)v[t];
    }
  }
}

unsigned blocks_for(int64_t items) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>(tiles_of(items, kThreads), 8192)); }

}  // namespace

int launch_copy_rows(const char*, const void* src, int64_t bytes, int64_t rows, void* dst, int64_t pitch, int64_t padded_rows, hipStream_t st) {
  const int64_t count = padded_rows * (pitch / 16);
  return launch_kernel(copy_rows_kernel, dim3(blocks_for(count)), dim3(kThreads), 0, st, static_cast<const char*>(src), bytes, rows,
                       static_cast<uint4_t*>(dst), (int)(pitch / 16), count);
}

int launch_zero_16bit(void* dst, int64_t count, hipStream_t st) {
  if (count == 0) return TF_OK;
  return launch_kernel(zero_kernel, dim3(blocks_for(count)), dim3(kThreads), 0, st, static_cast<uint16_t*>(dst), count);
}

int launch_zero_columns(void* dst, int64_t pitch, int64_t rows, int64_t from, int64_t to, hipStream_t st) {
  return launch_kernel(zero_columns_kernel, dim3(blocks_for(rows * (to - from))), dim3(kThreads), 0, st, static_cast<uint16_t*>(dst), pitch, rows,
                       (int)from, (int)(to - from));
}

template <typename T>
int launch_sum_parts(const float* parts, const PartsRoom& room, int splits, int64_t first, int64_t M, int64_t N, T* out, const Scale* scale,
                     hipStream_t st) {
  const int64_t chunks = tiles_of(N, 4), count = (M - first) * chunks;
  return launch_kernel(sum_parts_kernel<T>, dim3(blocks_for(count)), dim3(kThreads), 0, st, parts, room.rows * room.pitch, room.pitch, splits, first, count,
                       (int)N, (int)chunks, out, scale);
}
template int launch_sum_parts<half_t>(const float*, const PartsRoom&, int, int64_t, int64_t, int64_t, half_t*, const Scale*, hipStream_t);
template int launch_sum_parts<bf16_t>(const float*, const PartsRoom&, int, int64_t, int64_t, int64_t, bf16_t*, const Scale*, hipStream_t);

}  // namespace tfk
