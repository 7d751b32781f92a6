// The gated feed-forward block: h = act(x * Wg^T) * (x * Wu^T) in one kernel, and its backward pass.
//
// Forward.  The two projections are one product whose columns alternate between the two weights in blocks of 16 (Operands), so
// that a lane holds the gate and the up value of an element in the same place of two neighbouring blocks, and the activation and the
// product are done on the accumulators: one rounding, to h.  For training gate and up are kept as well, rounded to the type.
//
// Backward, from the gate and up values that were kept:
//   dg = dh * up * act'(gate), du = dh * act(gate)
//   dx = dg * Wg + du * Wu,  dWg = dg^T * x,  dWu = du^T * x
// One pass over dh, gate and up leaves [dg | du] twice, as rows of tokens and transposed, both completed by zeros to multiples of 64; then
// dx is one product over 2F and the weights' gradients are one (or two) over the tokens.  dg and du are rounded to the type once, as the operands of
// the matrix instructions have to be.
#include "product.hpp"

namespace tfk {
namespace {

// act(g) = g * phi(g)
TFK_DEVICE float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + __expf(-x)); }
constexpr float kGeluCubic = 0.044715f;
constexpr float kGeluTwice = 1.5957691216057308f;   // 2 * sqrt(2 / pi): (1 + tanh(y)) / 2 = sigmoid(2y)

TFK_DEVICE float act_phi(float g, int activation) {
  if (activation == TF_ACT_SILU) return sigmoid(g);
  if (activation == TF_ACT_GELU) return 0.5f + 0.5f * erff(g * 0.7071067811865476f);
  return sigmoid(kGeluTwice * (g + kGeluCubic * g * g * g));
}
TFK_DEVICE float act(float g, int activation) { return g * act_phi(g, activation); }
// act and its derivative
TFK_DEVICE void act_both(float g, int activation, float& value, float& slope) {
  const float p = act_phi(g, activation);
  value = g * p;
  if (activation == TF_ACT_GELU) {
    slope = p + g * 0.3989422804014327f * __expf(-0.5f * g * g);
    return;
  }
  const float inner = activation == TF_ACT_SILU ? 1.f : kGeluTwice * (1.f + 3.f * kGeluCubic * g * g);
  const float both = p * (1.f - p);
  slope = both > 0.f ? p + g * both * inner : p;   // (far out the square may be infinite; a NaN stays one)
}

template <typename T>
struct GatedEpilogue {
  T *h, *gate, *up;   // gate, up: null where they are not kept
  int M, F, activation;

  template <bool kInside, int TM, int TN>
  TFK_DEVICE void run(float4_t (&acc)[TM][TN], const TileAt& at) const {
    if (activation == TF_ACT_SILU) finish<kInside, TF_ACT_SILU>(acc, at);
    else if (activation == TF_ACT_GELU) finish<kInside, TF_ACT_GELU>(acc, at);
    else finish<kInside, TF_ACT_GELU_TANH>(acc, at);
  }
  template <bool kInside, int kActivation, int TM, int TN>
  TFK_DEVICE void finish(float4_t (&acc)[TM][TN], const TileAt& at) const {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int row = at.row + 16 * i;
      float4_t v[TN / 2];
      if (gate != nullptr) {
#pragma unroll
        for (int j = 0; j < TN / 2; ++j) v[j] = acc[i][2 * j];
        store_blocks<kInside>(gate, (size_t)F, row, at.col, M, F, at.lane, v);
#pragma unroll
        for (int j = 0; j < TN / 2; ++j) v[j] = acc[i][2 * j + 1];
        store_blocks<kInside>(up, (size_t)F, row, at.col, M, F, at.lane, v);
      }
#pragma unroll
      for (int j = 0; j < TN / 2; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) v[j][r] = act(acc[i][2 * j][r], kActivation) * acc[i][2 * j + 1][r];
      store_blocks<kInside>(h, (size_t)F, row, at.col, M, F, at.lane, v);
      __builtin_amdgcn_sched_barrier(0);   // (a row of blocks at a time: registers)
    }
  }
};

template <typename T>
int gated_ffn(const void* x, const void* w_gate, const void* w_up, void* h, void* gate, void* up, int activation, int64_t M, int64_t F, int64_t K,
              hipStream_t st) {
  const Operands operands = {x, {w_gate, w_up}, (int)M, (int)F, (int)K};
  return launch_product<T, true>(
      "tf_gated_ffn", operands, plan_product<T>(operands, true),
      GatedEpilogue<T>{static_cast<T*>(h), static_cast<T*>(gate), static_cast<T*>(up), (int)M, (int)F, activation}, st);
}

// ---- backward ------------------------------------------------------------------------------
constexpr int kTile = 64, kThreads = 256;

// One 64 x 64 tile of dh, gate and up: dg and du to rows [dg | du] of pitch 2 * Fp, and transposed to rows of pitch Mp.
template <typename T>
__global__ __launch_bounds__(kThreads) void gated_ffn_grads_kernel(const T* __restrict__ dh, const T* __restrict__ gate, const T* __restrict__ up,
                                                                  T* __restrict__ rows, T* __restrict__ cols, int M, int F, int Mp, int Fp, int tiles_f,
                                                                  int activation) {
  __shared__ T s_dg[kTile][kTile + 2], s_du[kTile][kTile + 2];
  const int m0 = blockIdx.x / tiles_f * kTile, f0 = blockIdx.x % tiles_f * kTile;
  for (int e = threadIdx.x; e < kTile * kTile; e += kThreads) {
    const int r = e / kTile, c = e % kTile;
    float dg = 0.f, du = 0.f;
    if (m0 + r < M && f0 + c < F) {
      const size_t at = (size_t)(m0 + r) * F + f0 + c;
      float value, slope;
      act_both((float)gate[at], activation, value, slope);
      const float d = (float)dh[at];
      dg = d * (float)up[at] * slope;
      du = d * value;
    }
    s_dg[r][c] = (T)dg;
    s_du[r][c] = (T)du;
    if (m0 + r < M) {
      T* const to = rows + (size_t)(m0 + r) * 2 * Fp + f0 + c;
      to[0] = (T)dg;
      to[Fp] = (T)du;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < kTile * kTile; e += kThreads) {
    const int c = e / kTile, r = e % kTile;
    if (f0 + c < F) {
      cols[(size_t)(f0 + c) * Mp + m0 + r] = s_dg[r][c];
      cols[(size_t)(F + f0 + c) * Mp + m0 + r] = s_du[r][c];
    }
  }
}

struct BackwardPlan {
  int64_t Mp, Fp;
  size_t rows, cols, weights, x, bytes;   // offsets in the workspace, its size
  BackwardPlan(int64_t M, int64_t F, int64_t K) {
    Mp = round_up_to(M, 64);
    Fp = round_up_to(F, 64);
    size_t at = 0;
    auto take = [&](int64_t elements) {
      const size_t from = at;
      at += round_up_to(2 * elements, 256);
      return from;
    };
    rows = take(M * 2 * Fp);      // [dg | du]
    cols = take(2 * F * Mp);      // the same transposed
    weights = take(K * 2 * Fp);   // [Wg^T | Wu^T]
    x = take(K * Mp);             // x^T
    bytes = at;
  }
};

template <typename T>
int gated_ffn_backward(const void* dh, const void* x, const void* w_gate, const void* w_up, const void* gate, const void* up, void* dx, void* dw_gate,
                       void* dw_up, int dtype, int activation, int64_t M, int64_t F, int64_t K, char* ws, hipStream_t st) {
  constexpr const char* who = "tf_gated_ffn_backward";
  if (M == 0) {
    if (int rc = launch_zero_16bit(dw_gate, F * K, st)) return rc;
    return launch_zero_16bit(dw_up, F * K, st);
  }
  const BackwardPlan p(M, F, K);
  T* const rows = reinterpret_cast<T*>(ws + p.rows);
  T* const cols = reinterpret_cast<T*>(ws + p.cols);
  const int64_t tiles_f = p.Fp / kTile, tiles = tiles_f * (p.Mp / kTile);
  TFK_REQUIRE(tiles < (int64_t)1 << 24, TF_ERR_INVALID_ARG, "%s: gradient too large", who);
  if (int rc = launch_kernel(gated_ffn_grads_kernel<T>, dim3((unsigned)tiles), dim3(kThreads), 0, st, static_cast<const T*>(dh),
                             static_cast<const T*>(gate), static_cast<const T*>(up), rows, cols, (int)M, (int)F, (int)p.Mp, (int)p.Fp, (int)tiles_f,
                             activation))
    return rc;
  T* const weights = reinterpret_cast<T*>(ws + p.weights);
  if (int rc = launch_transpose_padded(who, w_gate, K, weights, 2 * p.Fp, F, K, p.Fp, st)) return rc;
  if (int rc = launch_transpose_padded(who, w_up, K, weights + p.Fp, 2 * p.Fp, F, K, p.Fp, st)) return rc;
  if (int rc = launch_transpose_padded(who, x, K, ws + p.x, p.Mp, M, K, p.Mp, st)) return rc;
  if (int rc = tf_gemm(rows, weights, dx, dtype, 0, M, K, 2 * p.Fp, 1, 1, 1, 1, 0, st)) return rc;
  // (one product where the two gradients lie one behind the other)
  const bool together = static_cast<char*>(dw_up) == static_cast<char*>(dw_gate) + 2 * F * K && 2 * F < (1 << 30);
  if (together) return tf_gemm(cols, ws + p.x, dw_gate, dtype, 0, 2 * F, K, p.Mp, 1, 1, 1, 1, 0, st);
  if (int rc = tf_gemm(cols, ws + p.x, dw_gate, dtype, 0, F, K, p.Mp, 1, 1, 1, 1, 0, st)) return rc;
  return tf_gemm(cols + F * p.Mp, ws + p.x, dw_up, dtype, 0, F, K, p.Mp, 1, 1, 1, 1, 0, st);
}

int check_sizes(const char* who, int dtype, int activation, int64_t M, int64_t F, int64_t K) {
  TFK_REQUIRE(dtype == TF_DTYPE_F16 || dtype == TF_DTYPE_BF16, TF_ERR_UNSUPPORTED, "%s: dtype must be TF_DTYPE_F16 or TF_DTYPE_BF16", who);
  TFK_REQUIRE(activation >= TF_ACT_SILU && activation <= TF_ACT_GELU_TANH, TF_ERR_INVALID_ARG, "%s: unknown activation %d", who, activation);
  TFK_REQUIRE(M >= 0 && F > 0 && K > 0, TF_ERR_INVALID_ARG, "%s: M must not be negative, F and K must be positive", who);
  // (sums run over 2 F and over M as well as over K, and a sum has at most 2^22 - 64 terms)
  TFK_REQUIRE(M <= (1 << 22) - 64 && F <= (1 << 21) - 64 && K <= (1 << 22) - 64, TF_ERR_INVALID_ARG, "%s: dimension too large", who);
  return TF_OK;
}

}  // namespace
}  // namespace tfk

extern "C" int tf_gated_ffn(const void* x, const void* w_gate, const void* w_up, void* h, void* gate, void* up, int dtype, int activation, int64_t M,
                            int64_t F, int64_t K, void* stream) {
  using namespace tfk;
  if (int rc = check_sizes("tf_gated_ffn", dtype, activation, M, F, K)) return rc;
  if (M == 0) return TF_OK;
  TFK_REQUIRE(x && w_gate && w_up && h, TF_ERR_INVALID_ARG, "tf_gated_ffn: null pointer");
  TFK_REQUIRE((gate == nullptr) == (up == nullptr), TF_ERR_INVALID_ARG, "tf_gated_ffn: gate and up are kept both or neither");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == TF_DTYPE_F16) return gated_ffn<half_t>(x, w_gate, w_up, h, gate, up, activation, M, F, K, st);
  return gated_ffn<bf16_t>(x, w_gate, w_up, h, gate, up, activation, M, F, K, st);
}

extern "C" size_t tf_gated_ffn_backward_workspace_bytes(int64_t M, int64_t F, int64_t K) {
  using namespace tfk;
  if (M <= 0 || check_sizes("tf_gated_ffn_backward_workspace_bytes", TF_DTYPE_F16, TF_ACT_SILU, M, F, K) != TF_OK) return 0;
  return BackwardPlan(M, F, K).bytes;
}

extern "C" int tf_gated_ffn_backward(const void* dh, const void* x, const void* w_gate, const void* w_up, const void* gate, const void* up, void* dx,
                                     void* dw_gate, void* dw_up, int dtype, int activation, int64_t M, int64_t F, int64_t K, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  using namespace tfk;
  if (int rc = check_sizes("tf_gated_ffn_backward", dtype, activation, M, F, K)) return rc;
  TFK_REQUIRE(dw_gate && dw_up, TF_ERR_INVALID_ARG, "tf_gated_ffn_backward: null pointer");
  if (M > 0) {
    TFK_REQUIRE(dh && x && w_gate && w_up && gate && up && dx, TF_ERR_INVALID_ARG, "tf_gated_ffn_backward: null pointer");
    const size_t want = BackwardPlan(M, F, K).bytes;
    TFK_REQUIRE(workspace && workspace_bytes >= want && at_16B(workspace), TF_ERR_INVALID_ARG,
                "tf_gated_ffn_backward: workspace of %zu bytes at a 16-byte boundary needed, got %zu", want, workspace_bytes);
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* const ws = static_cast<char*>(workspace);
  if (dtype == TF_DTYPE_F16)
    return gated_ffn_backward<half_t>(dh, x, w_gate, w_up, gate, up, dx, dw_gate, dw_up, dtype, activation, M, F, K, ws, st);
  return gated_ffn_backward<bf16_t>(dh, x, w_gate, w_up, gate, up, dx, dw_gate, dw_up, dtype, activation, M, F, K, ws, st);
}
