// Softmax cross entropy of a linear head over a large vocabulary, without its logits z = H * W^T ever being in memory:
//
//   lse[t] = log sum_v exp(z[t, v]),   loss[t] = lse[t] - z[t, target[t]]
//
// Forward.  A tile of the product is reduced, in the registers it was computed in, to a maximum and a sum of exp(z - maximum) for each of
// its rows, and the lane that holds the target's logit writes that down; a second kernel merges the parts of a row.
//
// Backward, a piece of the vocabulary at a time: the product is computed again, and from lse
//   P[t, v] = grad_loss[t] * (exp(z[t, v] - lse[t]) - [v = target[t]]),   dH += P * W,   dW = P^T * H.
// P of a piece is rounded to 16 bits, as the operand of a matrix instruction has to be, divided by the smallest power of two that no
// |grad_loss| is above (times 2^14 for fp16), so that the weights of a mean over many tokens do not fall below fp16's range; the sums are
// multiplied by it again in 32 bits.  dH is summed over the pieces in fp32 and rounded once.
#include <cmath>

#include "product.hpp"

namespace tfk {
namespace {

struct Part {
  float top, sum;   // a maximum, and the sum of exp(z - maximum)
};
// what a maximum is subtracted as: where there is none (every logit -inf), zero, so that the sum is zero and not a NaN
TFK_DEVICE float as_origin(float top) { return top == -INFINITY ? 0.f : top; }

constexpr float kLog2e = 1.4426950408889634f;

struct LseEpilogue {
  Part* parts;            // [T][slots]
  int slots;
  float* at_target;       // [T]
  const int64_t* target;
  int M, N;

  template <bool kInside, int TM, int TN>
  TFK_DEVICE void run(float4_t (&acc)[TM][TN], const TileAt& at) const {
    if (kInside && at.col >= at.col_from) reduce<false>(acc, at);
    else reduce<true>(acc, at);
  }
  // kSome: columns in front of col_from and from N on do not count
  template <bool kSome, int TM, int TN>
  TFK_DEVICE void reduce(float4_t (&acc)[TM][TN], const TileAt& at) const {
    const int lr = at.lane & 15, lg = at.lane >> 4;
    const auto counts = [&](int j, int r) __attribute__((always_inline)) {
      const int col = at.col + 16 * j + 4 * lg + r;
      return !kSome || (col >= at.col_from && col < N);
    };
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int row = at.row + 16 * i + lr;
      const int64_t wanted = (row < M ? target[row] : -1) - at.col;   // counted from the tile's first column
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (counts(j, r)) top = fmaxf(top, acc[i][j][r]);
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float origin = as_origin(top) * kLog2e;
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (counts(j, r)) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][r], kLog2e, -origin));
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      if (lg == 0 && row < M) parts[(size_t)row * slots + at.slot] = Part{top, sum};
      // few tiles hold a target of theirs
      if (__any(wanted >= 0 && wanted < 16 * TN)) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (wanted == 16 * j + 4 * lg + r && counts(j, r)) at_target[row] = acc[i][j][r];
      }
      __builtin_amdgcn_sched_barrier(0);   // (a row of blocks at a time: registers)
    }
  }
};

// One wavefront a row.
constexpr int kMergeThreads = 256, kMergeRows = kMergeThreads / 64;
__global__ __launch_bounds__(kMergeThreads) void merge_parts_kernel(const Part* __restrict__ parts, int slots, const float* __restrict__ at_target,
                                                                    const int64_t* __restrict__ target, int64_t ignore_index, int T, int V,
                                                                    float* __restrict__ loss, float* __restrict__ lse) {
  const int row = blockIdx.x * kMergeRows + threadIdx.x / 64, lane = threadIdx.x % 64;
  if (row >= T) return;
  const Part* const mine = parts + (size_t)row * slots;
  float top = -INFINITY, sum = 0.f;
  for (int s = lane; s < slots; s += 64) {
    const Part p = mine[s];
    const float next = fmaxf(top, p.top), origin = as_origin(next);
    sum = sum * __expf(top - origin) + p.sum * __expf(p.top - origin);
    top = next;
  }
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) {
    const float other_top = __shfl_xor(top, d), other_sum = __shfl_xor(sum, d);
    const float next = fmaxf(top, other_top), origin = as_origin(next);
    sum = sum * __expf(top - origin) + other_sum * __expf(other_top - origin);
    top = next;
  }
  if (lane != 0) return;
  const float value = as_origin(top) + logf(sum);
  const int64_t wanted = target[row];
  lse[row] = value;
  // a target outside the vocabulary is a mistake that must not pass for a number
  loss[row] = wanted == ignore_index ? 0.f : wanted >= 0 && wanted < V ? value - at_target[row] : __uint_as_float(0x7fc00000u);
}

// ---- backward ------------------------------------------------------------------------------
struct Scale {
  float in, out;   // P holds grad_loss * in, sums are multiplied by out
};

constexpr int kScaleThreads = 1024;
__global__ __launch_bounds__(kScaleThreads) void find_scale_kernel(const float* __restrict__ grad_loss, const int64_t* __restrict__ target,
                                                                   int64_t ignore_index, int T, int headroom, Scale* scale) {
  __shared__ float s_top[kScaleThreads / 64];
  float top = 0.f;
  for (int t = threadIdx.x; t < T; t += kScaleThreads)
    if (target[t] != ignore_index) top = fmaxf(top, fabsf(grad_loss[t]));
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) top = fmaxf(top, __shfl_xor(top, d));
  if (threadIdx.x % 64 == 0) s_top[threadIdx.x / 64] = top;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < kScaleThreads / 64; ++w) top = fmaxf(top, s_top[w]);
  int e = 0;
  if (top > 0.f && top < INFINITY) {
    const float m = frexpf(top, &e);   // top = m * 2^e, 0.5 <= m < 1
    if (m == 0.5f) --e;
  }
  e = max(e, -110);   // (2^-e and the headroom have to fit as well)
  *scale = Scale{ldexpf(1.f, headroom - e), ldexpf(1.f, e - headroom)};
}

template <typename T>
struct ProbEpilogue {
  T* p;                    // [tokens][pitch]
  int64_t pitch;
  const float *lse, *grad_loss;
  const Scale* scale;
  const int64_t* target;
  int64_t ignore_index;
  int M, N;                // tokens, columns of the piece
  int first, V;            // the piece's first column, columns of all

  template <bool kInside, int TM, int TN>
  TFK_DEVICE void run(float4_t (&acc)[TM][TN], const TileAt& at) const {
    const int lr = at.lane & 15, lg = at.lane >> 4;
    const float in = scale->in;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int row = kInside ? at.row + 16 * i + lr : min(at.row + 16 * i + lr, M - 1);
      const int64_t wanted = target[row];
      const bool ignored = wanted == ignore_index;
      const float origin = lse[row];
      // (a target outside the vocabulary: as the loss)
      const float weight = wanted >= 0 && wanted < V ? grad_loss[row] * in : __uint_as_float(0x7fc00000u);
      const int64_t hot = wanted - first - at.col;   // counted from the tile's first column
      const float from = origin * kLog2e;
      float4_t v[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) v[j][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][r], kLog2e, -from)) * weight;
      if (__any(hot >= 0 && hot < 16 * TN)) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (hot == 16 * j + 4 * lg + r) v[j][r] = (__builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][r], kLog2e, -from)) - 1.f) * weight;
      }
      if (__any(ignored)) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) v[j][r] = ignored ? 0.f : v[j][r];
      }
      store_blocks<kInside>(p, (size_t)pitch, at.row + 16 * i, at.col, M, N, at.lane, v);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// A product that is scaled and rounded.
template <typename T>
struct ScaledEpilogue {
  T* out;                  // [M][N]
  const Scale* scale;
  int M, N;

  template <bool kInside, int TM, int TN>
  TFK_DEVICE void run(float4_t (&acc)[TM][TN], const TileAt& at) const {
    const float by = scale->out;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      float4_t v[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) v[j] = acc[i][j] * by;
      store_blocks<kInside>(out, (size_t)N, at.row + 16 * i, at.col, M, N, at.lane, v);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// One of several products that are summed in fp32; the last call scales and rounds the sum.
template <typename T>
struct SumEpilogue {
  float* sum;              // [M][N]
  T* out;                  // [M][N]
  const Scale* scale;
  bool first, last;
  int M, N;

  template <bool kInside, int TM, int TN>
  TFK_DEVICE void run(float4_t (&acc)[TM][TN], const TileAt& at) const {
    if (kInside && at.row >= at.row_from && at.col >= at.col_from) add<true>(acc, at);
    else add<false>(acc, at);
  }
  // kWhole: the tile overlaps none in front of it, and ends inside
  template <bool kWhole, int TM, int TN>
  TFK_DEVICE void add(float4_t (&acc)[TM][TN], const TileAt& at) const {
    typedef float4_t four_any_t __attribute__((aligned(4)));
    const int lr = at.lane & 15, lg = at.lane >> 4;
    const float by = last ? scale->out : 1.f;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int row = at.row + 16 * i + lr;
      if (kWhole) {
        float* const from = sum + (size_t)row * N + at.col + 4 * lg;
        float4_t v[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          v[j] = acc[i][j];
          if (!first) v[j] += *reinterpret_cast<const four_any_t*>(from + 16 * j);
          v[j] *= by;
        }
        if (last) {
          store_blocks<true>(out, (size_t)N, at.row + 16 * i, at.col, M, N, at.lane, v);
        } else {
#pragma unroll
          for (int j = 0; j < TN; ++j) *reinterpret_cast<four_any_t*>(from + 16 * j) = v[j];
        }
      } else if (row < M && row >= at.row_from) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int col = at.col + 16 * j + 4 * lg + r;
            if (col >= N || col < at.col_from) continue;
            const size_t to = (size_t)row * N + col;
            const float value = (first ? acc[i][j][r] : acc[i][j][r] + sum[to]) * by;
            if (last) out[to] = (T)value;
            else sum[to] = value;
          }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

struct ForwardPlan {
  int64_t slots;
  size_t at_target, bytes;
  ForwardPlan(int64_t T, int64_t V, int64_t K) {
    // (which kernel runs also depends on where the operands start)
    slots = std::max(product_slots(kAnyKernel, V), product_slots(pick_table_kernel(T, V, K, kOneAllowed), V));
    at_target = round_up_to(sizeof(Part) * T * slots, 256);
    bytes = at_target + round_up_to(sizeof(float) * T, 256);
  }
};

// What is held for a piece of the vocabulary: P as it is and transposed, and W transposed; beside them H transposed and the sums of dH.
struct BackwardPlan {
  int64_t Tp, piece;   // tokens completed to a multiple of 64, columns of a piece
  int64_t pieces;
  size_t p, pt, wt, ht, sum, scale, bytes;
  BackwardPlan(int64_t T, int64_t V, int64_t K) {
    Tp = round_up_to(T, 64);
    piece = std::min(round_up_to(V, 64), std::max<int64_t>(4096, ((int64_t)1 << 27) / Tp / 256 * 256));
    pieces = tiles_of(V, piece);
    size_t at = 0;
    auto take = [&](int64_t bytes_) {
      const size_t from = at;
      at += round_up_to(bytes_, 256);
      return from;
    };
    p = take(2 * T * piece);
    pt = take(2 * piece * Tp);
    wt = take(2 * K * piece);
    ht = take(2 * K * Tp);
    sum = take(pieces > 1 ? 4 * T * K : 0);
    scale = take(sizeof(Scale));
    bytes = at;
  }
};

template <typename T>
int forward(const void* hidden, const void* weight, const int64_t* target, float* loss, float* lse, int64_t tokens, int64_t V, int64_t K,
            int64_t ignore_index, char* ws, hipStream_t st) {
  const ForwardPlan plan(tokens, V, K);
  Part* const parts = reinterpret_cast<Part*>(ws);
  float* const at_target = reinterpret_cast<float*>(ws + plan.at_target);
  const Operands x = {hidden, {weight, nullptr}, (int)tokens, (int)V, (int)K};
  const ProductPlan product = plan_product<T>(x, false);
  if (int rc = launch_product<T, false>("tf_linear_cross_entropy", x, product,
                                        LseEpilogue{parts, (int)product.slots, at_target, target, (int)tokens, (int)V}, st))
    return rc;
  return launch_kernel(merge_parts_kernel, dim3((unsigned)tiles_of(tokens, kMergeRows)), dim3(kMergeThreads), 0, st, parts, (int)product.slots,
                       at_target, target, ignore_index, (int)tokens, (int)V, loss, lse);
}

template <typename T>
int backward(const float* grad_loss, const void* hidden, const void* weight, const int64_t* target, const float* lse, void* grad_hidden,
             void* grad_weight, int64_t tokens, int64_t V, int64_t K, int64_t ignore_index, char* ws, hipStream_t st) {
  constexpr const char* who = "tf_linear_cross_entropy_backward";
  if (tokens == 0) return launch_zero_16bit(grad_weight, V * K, st);
  const BackwardPlan plan(tokens, V, K);
  T* const p = reinterpret_cast<T*>(ws + plan.p);
  Scale* const scale = reinterpret_cast<Scale*>(ws + plan.scale);
  float* const sum = reinterpret_cast<float*>(ws + plan.sum);
  constexpr int kHeadroom = std::is_same_v<T, half_t> ? 14 : 0;
  if (int rc = launch_kernel(find_scale_kernel, dim3(1), dim3(kScaleThreads), 0, st, grad_loss, target, ignore_index, (int)tokens, kHeadroom, scale))
    return rc;
  if (int rc = launch_transpose_padded(who, hidden, K, ws + plan.ht, plan.Tp, tokens, K, plan.Tp, st)) return rc;
  for (int64_t first = 0; first < V; first += plan.piece) {
    const int64_t columns = std::min(plan.piece, V - first), pitch = round_up_to(columns, 64);
    const char* const w = static_cast<const char*>(weight) + 2 * first * K;
    const Operands logits = {hidden, {w, nullptr}, (int)tokens, (int)columns, (int)K};
    if (int rc = launch_product<T, false>(who, logits, plan_product<T>(logits, false),
                                              ProbEpilogue<T>{p, pitch, lse, grad_loss, scale, target, ignore_index, (int)tokens, (int)columns,
                                                              (int)first, (int)V},
                                              st))
      return rc;
    if (pitch > columns)
      if (int rc = launch_zero_columns(who, p, pitch, tokens, columns, pitch, st)) return rc;
    if (int rc = launch_transpose_padded(who, p, pitch, ws + plan.pt, plan.Tp, tokens, columns, plan.Tp, st)) return rc;
    if (int rc = launch_transpose_padded(who, w, K, ws + plan.wt, pitch, columns, K, pitch, st)) return rc;
    const Operands of_hidden = {p, {ws + plan.wt, nullptr}, (int)tokens, (int)K, (int)pitch};
    const ProductPlan hidden_plan = plan_product<T>(of_hidden, false);
    T* const to_hidden = static_cast<T*>(grad_hidden);
    const int rc = plan.pieces == 1
                       ? launch_product<T, false>(who, of_hidden, hidden_plan, ScaledEpilogue<T>{to_hidden, scale, (int)tokens, (int)K}, st)
                       : launch_product<T, false>(who, of_hidden, hidden_plan,
                                                  SumEpilogue<T>{sum, to_hidden, scale, first == 0, first + columns == V, (int)tokens, (int)K}, st);
    if (rc) return rc;
    const Operands of_weight = {ws + plan.pt, {ws + plan.ht, nullptr}, (int)columns, (int)K, (int)plan.Tp};
    if (int rc = launch_product<T, false>(who, of_weight, plan_product<T>(of_weight, false),
                                          ScaledEpilogue<T>{static_cast<T*>(grad_weight) + first * K, scale, (int)columns, (int)K}, st))
      return rc;
  }
  return TF_OK;
}

int check_sizes(const char* who, int dtype, int64_t T, int64_t V, int64_t K) {
  TFK_REQUIRE(dtype == TF_DTYPE_F16 || dtype == TF_DTYPE_BF16, TF_ERR_UNSUPPORTED, "%s: dtype must be TF_DTYPE_F16 or TF_DTYPE_BF16", who);
  TFK_REQUIRE(T >= 0 && V > 0 && K > 0, TF_ERR_INVALID_ARG, "%s: T must not be negative, V and K must be positive", who);
  TFK_REQUIRE(T <= (1 << 22) - 64 && V <= (1 << 30) - 64 && K <= (1 << 22) - 64, TF_ERR_INVALID_ARG, "%s: dimension too large", who);
  return TF_OK;
}

}  // namespace
}  // namespace tfk

extern "C" size_t tf_linear_cross_entropy_workspace_bytes(int64_t T, int64_t V, int64_t K) {
  using namespace tfk;
  if (T <= 0 || check_sizes("tf_linear_cross_entropy_workspace_bytes", TF_DTYPE_F16, T, V, K) != TF_OK) return 0;
  return ForwardPlan(T, V, K).bytes;
}

extern "C" int tf_linear_cross_entropy(const void* hidden, const void* weight, const int64_t* target, float* loss, float* lse, int dtype, int64_t T,
                                       int64_t V, int64_t K, int64_t ignore_index, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace tfk;
  if (int rc = check_sizes("tf_linear_cross_entropy", dtype, T, V, K)) return rc;
  if (T == 0) return TF_OK;
  TFK_REQUIRE(hidden && weight && target && loss && lse, TF_ERR_INVALID_ARG, "tf_linear_cross_entropy: null pointer");
  const size_t want = ForwardPlan(T, V, K).bytes;
  TFK_REQUIRE(workspace && workspace_bytes >= want && at_16B(workspace), TF_ERR_INVALID_ARG,
              "tf_linear_cross_entropy: workspace of %zu bytes at a 16-byte boundary needed, got %zu", want, workspace_bytes);
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* const ws = static_cast<char*>(workspace);
  if (dtype == TF_DTYPE_F16) return forward<half_t>(hidden, weight, target, loss, lse, T, V, K, ignore_index, ws, st);
  return forward<bf16_t>(hidden, weight, target, loss, lse, T, V, K, ignore_index, ws, st);
}

extern "C" size_t tf_linear_cross_entropy_backward_workspace_bytes(int64_t T, int64_t V, int64_t K) {
  using namespace tfk;
  if (T <= 0 || check_sizes("tf_linear_cross_entropy_backward_workspace_bytes", TF_DTYPE_F16, T, V, K) != TF_OK) return 0;
  return BackwardPlan(T, V, K).bytes;
}

extern "C" int tf_linear_cross_entropy_backward(const float* grad_loss, const void* hidden, const void* weight, const int64_t* target, const float* lse,
                                                void* grad_hidden, void* grad_weight, int dtype, int64_t T, int64_t V, int64_t K, int64_t ignore_index,
                                                void* workspace, size_t workspace_bytes, void* stream) {
  using namespace tfk;
  if (int rc = check_sizes("tf_linear_cross_entropy_backward", dtype, T, V, K)) return rc;
  TFK_REQUIRE(grad_weight, TF_ERR_INVALID_ARG, "tf_linear_cross_entropy_backward: null pointer");
  if (T > 0) {
    TFK_REQUIRE(grad_loss && hidden && weight && target && lse && grad_hidden, TF_ERR_INVALID_ARG,
                "tf_linear_cross_entropy_backward: null pointer");
    const size_t want = BackwardPlan(T, V, K).bytes;
    TFK_REQUIRE(workspace && workspace_bytes >= want && at_16B(workspace), TF_ERR_INVALID_ARG,
                "tf_linear_cross_entropy_backward: workspace of %zu bytes at a 16-byte boundary needed, got %zu", want, workspace_bytes);
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* const ws = static_cast<char*>(workspace);
  if (dtype == TF_DTYPE_F16)
    return backward<half_t>(grad_loss, hidden, weight, target, lse, grad_hidden, grad_weight, T, V, K, ignore_index, ws, st);
  return backward<bf16_t>(grad_loss, hidden, weight, target, lse, grad_hidden, grad_weight, T, V, K, ignore_index, ws, st);
}
