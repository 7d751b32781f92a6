// Products of 8-bit integers with a scale for each row of either operand, and the quantisation of rows that makes the first of them:
//
//   C[m, n] = scale_a[m] * scale_b[n] * sum_k A[m, k] * B[n, k]
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

// K is no multiple of 16: rows are copied, completed by zeros to whole lines (131 us instead of 140 for 2999 x 1544 x 1032).
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
// scale = max|x| / 127 of a row, q the whole number nearest to x / scale, in the middle of two the even one.  The quotient is rounded
// twice on the way (to 32 bits, to a whole number), which can go wrong by one next to a middle, so what is left, x - q * scale, decides:
// it is exact there (x has at most 11 significant bits and is a multiple of scale's last one), and more than half a step is another q.
TFK_DEVICE int quantize(float x, float scale) {
  float q = __builtin_rintf(x / scale);
  const float left = __builtin_fmaf(-q, scale, x), half = 0.5f * scale;
  const bool odd = ((int)q & 1) != 0;
  if (left > half || (left == half && odd)) q += 1.f;
  else if (left < -half || (left == -half && odd)) q -= 1.f;
  // (a scale below the normal numbers has few bits left)
  return (int)fminf(fmaxf(q, -127.f), 127.f);
}

constexpr int kQuantThreads = 256;

template <typename T>
__global__ __launch_bounds__(kQuantThreads) void quantize_rows_kernel(const T* __restrict__ x, int8_t* __restrict__ q, float* __restrict__ scales, int K) {
  __shared__ float s_top[kQuantThreads / 64];
  const size_t row = blockIdx.x;
  const T* const src = x + row * K;
  int8_t* const dst = q + row * K;
  // (a NaN is larger than everything: the integer order of the bits of |x|)
  unsigned top = 0;
  for (int k = threadIdx.x; k < K; k += kQuantThreads) top = max(top, __float_as_uint((float)src[k]) & 0x7fffffffu);
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) top = max(top, (unsigned)__shfl_xor((int)top, d));
  if (threadIdx.x % 64 == 0) s_top[threadIdx.x / 64] = __uint_as_float(top);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kQuantThreads / 64; ++w) top = max(top, __float_as_uint(s_top[w]));
  // a row with an infinity or a NaN has no scale, and its products shall say so
  const bool finite = top < 0x7f800000u;
  const float scale = finite ? __uint_as_float(top) / 127.f : __uint_as_float(0x7fc00000u);
  if (threadIdx.x == 0) scales[row] = scale;
  for (int k = threadIdx.x; k < K; k += kQuantThreads) dst[k] = finite && scale > 0.f ? (int8_t)quantize((float)src[k], scale) : (int8_t)0;
}

}  // namespace
}  // namespace tfk

extern "C" size_t tf_gemm_int8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || K > 131071 || M >= (1 << 30) || N >= (1 << 30)) return 0;
  return tfk::CopyPlan(M, N, K).bytes;
}

extern "C" int tf_gemm_int8(const void* A, const void* B, const float* scale_a, const float* scale_b, void* C, int c_dtype, int64_t M, int64_t N,
                            int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace tfk;
  TFK_REQUIRE(M >= 0 && N >= 0 && K > 0, TF_ERR_INVALID_ARG, "tf_gemm_int8: negative extent, or no K");
  TFK_REQUIRE(c_dtype >= TF_DTYPE_F32 && c_dtype <= TF_DTYPE_BF16, TF_ERR_UNSUPPORTED,
              "tf_gemm_int8: the result must be TF_DTYPE_F32, TF_DTYPE_F16 or TF_DTYPE_BF16");
  TFK_REQUIRE(K <= 131071, TF_ERR_INVALID_ARG, "tf_gemm_int8: a sum of more than 131071 products does not fit 32 bits (K = %lld)", (long long)K);
  TFK_REQUIRE(M < (1 << 30) && N < (1 << 30), TF_ERR_INVALID_ARG, "tf_gemm_int8: dimension too large");
  if (M == 0 || N == 0) return TF_OK;
  TFK_REQUIRE(A && B && scale_a && scale_b && C, TF_ERR_INVALID_ARG, "tf_gemm_int8: null pointer");
  const CopyPlan copy(M, N, K);
  TFK_REQUIRE(copy.bytes > 0 || (at_16B(A) && at_16B(B)), TF_ERR_INVALID_ARG, "tf_gemm_int8: A and B must begin at 16-byte boundaries");
  TFK_REQUIRE(copy.bytes == 0 || (workspace && workspace_bytes >= copy.bytes && at_16B(workspace)), TF_ERR_INVALID_ARG,
              "tf_gemm_int8: workspace of %zu bytes at a 16-byte boundary needed, got %zu", copy.bytes, workspace_bytes);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (copy.bytes > 0) {
    char* const ws = static_cast<char*>(workspace);
    if (int rc = launch_copy_rows("tf_gemm_int8", A, K, M, ws, copy.pitch, M, st)) return rc;
    if (int rc = launch_copy_rows("tf_gemm_int8", B, K, N, ws + copy.b, copy.pitch, N, st)) return rc;
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
  if (dtype == TF_DTYPE_F16)
    return launch_kernel(quantize_rows_kernel<half_t>, dim3((unsigned)rows), dim3(kQuantThreads), 0, st, static_cast<const half_t*>(x),
                         static_cast<int8_t*>(q), scales, (int)K);
  return launch_kernel(quantize_rows_kernel<bf16_t>, dim3((unsigned)rows), dim3(kQuantThreads), 0, st, static_cast<const bf16_t*>(x),
                       static_cast<int8_t*>(q), scales, (int)K);
}
