// Products of 8-bit integers with a scale for each row of either operand, and the quantisation of rows that makes the first of them:
//
//   C[m, n] = (sum_k A[m, k] * B[n, k]) * scale_a[m] * scale_b[n]
//
// The sum is exact in int32 (|A|, |B| <= 128: K <= 131071); it is converted to fp32, scaled, and rounded once to the result's type.
#include "product.hpp"

namespace tfk {
namespace {

template <typename OutT>
struct Int8Epilogue {
  OutT* c;
  const float *scale_a, *scale_b;
  int M, N;

  template <bool kInside, int TM, int TN>
  TFK_DEVICE void run(float4_t (&acc)[TM][TN], const TileAt& at) const {
    const int lr = at.lane & 15, lg = at.lane >> 4;
    // the lane's scales: of one row in each row of blocks, of four columns in each column of them
    float4_t sb[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) sb[j][r] = scale_b[kInside ? at.col + 16 * j + 4 * lg + r : min(at.col + 16 * j + 4 * lg + r, N - 1)];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int row = at.row + 16 * i;
      const float sa = scale_a[kInside ? row + lr : min(row + lr, M - 1)];
      float4_t v[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int4v_t sum = __builtin_bit_cast(int4v_t, acc[i][j]);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[j][r] = (float)sum[r] * sa * sb[j][r];
      }
      store_blocks<kInside>(c, (size_t)N, row, at.col, M, N, at.lane, v);
      __builtin_amdgcn_sched_barrier(0);   // (a row of blocks at a time: registers)
    }
  }
};

// K is no multiple of 16: rows are copied, completed by zeros to whole lines.  2999 x 1544 x 1032: 7 us for the copies and 13 for the product, 131 by a kernel
// that checks every access.
struct CopyPlan {
  int64_t pitch = 0;
  size_t b = 0, bytes = 0;
  CopyPlan(int64_t M, int64_t N, int64_t K) {
    if (K % 16 == 0) return;
    pitch = round_up_to(K, 128);
    b = M * pitch;
    bytes = b + N * pitch;
  }
};

template <typename OutT>
int gemm_int8(const void* A, const void* B, const float* sa, const float* sb, void* C, int64_t M, int64_t N, int64_t K, hipStream_t st) {
  const Operands x = {A, {B, nullptr}, (int)M, (int)N, (int)K};
  return launch_product<int8_t, false>("tf_gemm_int8", x, plan_product(M, N, K / 2, false),
                                       Int8Epilogue<OutT>{static_cast<OutT*>(C), sa, sb, (int)M, (int)N}, st);
}

// ---- quantize_rows -------------------------------------------------------------------------
// scale = max|x| / 127 of a row, q the whole number nearest to x / scale, in the middle of two the even one.  x times the reciprocal of the
// scale, rounded, is that number or, next to a middle, one beside it; what is left, x - q * scale, decides: it is exact there (x has at most 11
// significant bits and is a multiple of scale's last one).  Where half a step or more is left, which is rare, the element is looked at again.
//
// Bound by memory, in both directions: a workgroup a row, which it keeps in registers from the search for the maximum to the rounding (rows of more than
// kQuantThreads * 8 * 8 elements are read twice).  4096 x 4096 fp16: 30 us an element at a time with a division each, 12 so.
constexpr int kQuantThreads = 256;

template <typename T>
struct Eight {
  typedef T any_t __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  typedef T type __attribute__((ext_vector_type(8)));
};
// elements k .. k + 7 of a row, zeros from K on
template <typename T>
TFK_DEVICE typename Eight<T>::type load_eight(const T* row, int k, int K) {
  if (k + 8 <= K) return *reinterpret_cast<const typename Eight<T>::any_t*>(row + k);
  typename Eight<T>::type v;
#pragma unroll
  for (int t = 0; t < 8; ++t) v[t] = k + t < K ? row[k + t] : (T)0.f;
  return v;
}
template <typename T>
TFK_DEVICE unsigned top_of(typename Eight<T>::type v, unsigned top) {
#pragma unroll
  for (int t = 0; t < 8; ++t) top = max(top, __float_as_uint((float)v[t]) & 0x7fffffffu);   // (a NaN is larger than everything)
  return top;
}
TFK_DEVICE float quantize_again(float x, float q, float scale) {
  const float left = __builtin_fmaf(-q, scale, x), half = 0.5f * scale;
  const bool odd = ((int)q & 1) != 0;
  if (left > half || (left == half && odd)) q += 1.f;
  else if (left < -half || (left == -half && odd)) q -= 1.f;
  return fminf(fmaxf(q, -127.f), 127.f);   // (a scale below the normal numbers has few bits left)
}
// Eight elements to eight bytes.
template <typename T>
TFK_DEVICE uint2_t quantize_eight(typename Eight<T>::type v, float inverse, float scale) {
  constexpr float kWhole = 12582912.f;   // 1.5 * 2^23: a number added to it is rounded to a whole one, in the sum's low bits
  const float half = 0.5f * scale;
  unsigned bits[8];
  bool look = false;
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const float x = (float)v[t], r = __builtin_fmaf(x, inverse, kWhole);
    bits[t] = __float_as_uint(r);
    look |= !(fabsf(__builtin_fmaf(-(r - kWhole), scale, x)) < half);
  }
  if (look) {
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const float x = (float)v[t];
      bits[t] = (unsigned)(int)quantize_again(x, fminf(fmaxf(__builtin_rintf(x / scale), -128.f), 128.f), scale);
    }
  }
  uint2_t out;
#pragma unroll
  for (int w = 0; w < 2; ++w)
    out[w] = (bits[4 * w] & 0xff) | (bits[4 * w + 1] & 0xff) << 8 | (bits[4 * w + 2] & 0xff) << 16 | bits[4 * w + 3] << 24;
  return out;
}
TFK_DEVICE void store_eight(int8_t* row, int k, int K, uint2_t v) {
  typedef uint2_t any_t __attribute__((aligned(1)));
  if (k + 8 <= K) {
    *reinterpret_cast<any_t*>(row + k) = v;
    return;
  }
#pragma unroll
  for (int t = 0; t < 8; ++t)
    if (k + t < K) row[k + t] = (int8_t)(v[t / 4] >> (8 * (t % 4)));
}

// kHeld: groups of eight that a thread keeps; 0: it reads the row again.
template <typename T, int kHeld>
__global__ __launch_bounds__(kQuantThreads) void quantize_rows_kernel(const T* __restrict__ x, int8_t* __restrict__ q, float* __restrict__ scales, int K) {
  __shared__ unsigned s_top[kQuantThreads / 64];
  const size_t row = blockIdx.x;
  const T* const src = x + row * K;
  int8_t* const dst = q + row * K;
  typename Eight<T>::type held[kHeld > 0 ? kHeld : 1];
  unsigned top = 0;
  if constexpr (kHeld > 0) {
#pragma unroll
    for (int h = 0; h < kHeld; ++h) held[h] = load_eight(src, (h * kQuantThreads + (int)threadIdx.x) * 8, K);
#pragma unroll
    for (int h = 0; h < kHeld; ++h) top = top_of<T>(held[h], top);
  } else {
    for (int k = threadIdx.x * 8; k < K; k += kQuantThreads * 8) top = top_of<T>(load_eight(src, k, K), top);
  }
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) top = max(top, (unsigned)__shfl_xor((int)top, d));
  if (threadIdx.x % 64 == 0) s_top[threadIdx.x / 64] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kQuantThreads / 64; ++w) top = max(top, s_top[w]);
  // a row with an infinity or a NaN has no scale, and its products shall say so
  const bool finite = top < 0x7f800000u;
  const float scale = finite ? __uint_as_float(top) / 127.f : __uint_as_float(0x7fc00000u);
  if (threadIdx.x == 0) scales[row] = scale;
  const bool none = !(scale > 0.f);
  const float inverse = 1.f / scale;
  auto leave = [&](int k, typename Eight<T>::type v) __attribute__((always_inline)) {
    store_eight(dst, k, K, none ? uint2_t{0u, 0u} : quantize_eight<T>(v, inverse, scale));
  };
  if constexpr (kHeld > 0) {
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
      const int k = (h * kQuantThreads + (int)threadIdx.x) * 8;
      if (k < K) leave(k, held[h]);
    }
  } else {
    for (int k = threadIdx.x * 8; k < K; k += kQuantThreads * 8) leave(k, load_eight(src, k, K));
  }
}

template <typename T>
int quantize_rows(const void* x, void* q, float* scales, int64_t rows, int64_t K, hipStream_t st) {
  const int64_t held = tiles_of(K, kQuantThreads * 8);
  const auto kern = held <= 1   ? quantize_rows_kernel<T, 1>
                    : held <= 2 ? quantize_rows_kernel<T, 2>
                    : held <= 4 ? quantize_rows_kernel<T, 4>
                    : held <= 8 ? quantize_rows_kernel<T, 8>
                                : quantize_rows_kernel<T, 0>;
  return launch_kernel(kern, dim3((unsigned)rows), dim3(kQuantThreads), 0, st, static_cast<const T*>(x), static_cast<int8_t*>(q), scales, (int)K);
}

}  // namespace
}  // namespace tfk

extern "C" size_t tf_gemm_int8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || K > 131071 || M >= (1 << 30) || N > (1 << 29) - 64) return 0;
  return tfk::CopyPlan(M, N, K).bytes;
}

extern "C" int tf_gemm_int8(const void* A, const void* B, const float* scale_a, const float* scale_b, void* C, int c_dtype, int64_t M, int64_t N,
                            int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace tfk;
  TFK_REQUIRE(M >= 0 && N >= 0 && K > 0, TF_ERR_INVALID_ARG, "tf_gemm_int8: negative extent, or no K");
  TFK_REQUIRE(c_dtype >= TF_DTYPE_F32 && c_dtype <= TF_DTYPE_BF16, TF_ERR_UNSUPPORTED,
              "tf_gemm_int8: the result must be TF_DTYPE_F32, TF_DTYPE_F16 or TF_DTYPE_BF16");
  TFK_REQUIRE(K <= 131071, TF_ERR_INVALID_ARG, "tf_gemm_int8: a sum of more than 131071 products does not fit 32 bits (K = %lld)", (long long)K);
  TFK_REQUIRE(M < (1 << 30) && N <= (1 << 29) - 64, TF_ERR_INVALID_ARG, "tf_gemm_int8: dimension too large");   // (tiles of 64 columns: kMaxTiles)
  if (M == 0 || N == 0) return TF_OK;
  TFK_REQUIRE(A && B && scale_a && scale_b && C, TF_ERR_INVALID_ARG, "tf_gemm_int8: null pointer");
  const CopyPlan copy(M, N, K);
  TFK_REQUIRE(copy.bytes > 0 || (at_16B(A) && at_16B(B)), TF_ERR_INVALID_ARG, "tf_gemm_int8: A and B must begin at 16-byte boundaries");
  TFK_REQUIRE(copy.bytes == 0 || (workspace && workspace_bytes >= copy.bytes && at_16B(workspace)), TF_ERR_INVALID_ARG,
              "tf_gemm_int8: workspace of %zu bytes at a 16-byte boundary needed, got %zu", copy.bytes, workspace_bytes);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (copy.bytes > 0) {
    char* const ws = static_cast<char*>(workspace);
    const RowsToCopy both[] = {{A, M, ws, M}, {B, N, ws + copy.b, N}};
    if (int rc = launch_copy_rows(both, 2, K, copy.pitch, st)) return rc;
    A = ws;
    B = ws + copy.b;
    K = copy.pitch;
  }
  if (c_dtype == TF_DTYPE_F32) return gemm_int8<float>(A, B, scale_a, scale_b, C, M, N, K, st);
  if (c_dtype == TF_DTYPE_F16) return gemm_int8<half_t>(A, B, scale_a, scale_b, C, M, N, K, st);
  return gemm_int8<bf16_t>(A, B, scale_a, scale_b, C, M, N, K, st);
}

extern "C" int tf_quantize_rows(const void* x, void* q, float* scales, int dtype, int64_t rows, int64_t K, void* stream) {
  using namespace tfk;
  TFK_REQUIRE(rows >= 0 && K > 0, TF_ERR_INVALID_ARG, "tf_quantize_rows: negative number of rows, or no columns");
  TFK_REQUIRE(dtype == TF_DTYPE_F16 || dtype == TF_DTYPE_BF16, TF_ERR_UNSUPPORTED, "tf_quantize_rows: dtype must be TF_DTYPE_F16 or TF_DTYPE_BF16");
  TFK_REQUIRE(rows < (1 << 24) && K < (1 << 30), TF_ERR_INVALID_ARG, "tf_quantize_rows: dimension too large");
  if (rows == 0) return TF_OK;
  TFK_REQUIRE(x && q && scales, TF_ERR_INVALID_ARG, "tf_quantize_rows: null pointer");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == TF_DTYPE_F16) return quantize_rows<half_t>(x, q, scales, rows, K, st);
  return quantize_rows<bf16_t>(x, q, scales, rows, K, st);
}
