// Softmax cross entropy of a linear head over a large vocabulary, without its logits z = H * W^T ever being in memory:
//
//   lse[t] = log sum_v exp(z[t, v]),   loss[t] = lse[t] - z[t, target[t]]
//
// Forward.  A tile of the product is reduced, in the registers it was computed in, to a maximum and a sum of exp(z - maximum) for each of
// its rows, and the lane that holds the target's logit writes that down; a second kernel merges the parts of a row.
//
// (rows of K that is no multiple of 8 are copied first, completed by zeros to whole lines)
//
// Backward, a piece of the vocabulary at a time: the product is computed again, and from lse
//   P[t, v] = w[t] * (exp(z[t, v] - lse[t]) - [v = target[t]]),   dH[t] += m[t] * (P * W)[t],   dW = P^T * (m * H),   grad_loss = w * m.
// P of a piece is rounded to 16 bits, as the operand of a matrix instruction has to be.  At the target it is nearly -w[t], the largest part of both
// gradients by far: with all of grad_loss in w, what 16 bits leave out of that one number would be an error of everything that a token (and with a
// mean every token) adds, up to 2.5 times in all what rounding the results leaves out.  So w is a power of two, and m in (0.5, 1]: dH is
// multiplied by it in 32 bits, and the rounding of m * H is another one for each element (1.4 times as much).  What m takes out of all tokens
// is the mantissa of the grad_loss of the last one that counts (of the last 8192): where they have the same, m is 1 and nothing is rounded.
// In fp16 P is multiplied by a power of two as well by which the largest is 2^15 at most, so that the weights of a mean over many tokens do not fall
// below the type's range; the sums are divided by it in 32 bits.  (bf16 has the range of fp32.)  dH is summed over the pieces in fp32 and rounded once.
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

// A workgroup a row: the largest maximum first, then the sums relative to it.
constexpr int kMergeThreads = 256;
__global__ __launch_bounds__(kMergeThreads) void merge_parts_kernel(const Part* __restrict__ parts, int slots, const float* __restrict__ at_target,
                                                                    const int64_t* __restrict__ target, int64_t ignore_index, int V,
                                                                    float* __restrict__ loss, float* __restrict__ lse) {
  __shared__ float s_top[kMergeThreads / 64], s_sum[kMergeThreads / 64];
  const size_t row = blockIdx.x;
  const Part* const mine = parts + row * slots;
  const int tid = threadIdx.x;
  float top = -INFINITY, sum = 0.f;
  for (int s = tid; s < slots; s += kMergeThreads) top = fmaxf(top, mine[s].top);
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) top = fmaxf(top, __shfl_xor(top, d));
  if (tid % 64 == 0) s_top[tid / 64] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kMergeThreads / 64; ++w) top = fmaxf(top, s_top[w]);
  const float origin = as_origin(top);
  for (int s = tid; s < slots; s += kMergeThreads) {
    const Part p = mine[s];
    sum += p.sum * __expf(p.top - origin);
  }
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) sum += __shfl_xor(sum, d);
  if (tid % 64 == 0) s_sum[tid / 64] = sum;
  __syncthreads();
  if (tid != 0) return;
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kMergeThreads / 64; ++w) sum += s_sum[w];
  const float value = origin + logf(sum);
  const int64_t wanted = target[row];
  lse[row] = value;
  // a target outside the vocabulary is a mistake that must not pass for a number
  loss[row] = wanted == ignore_index ? 0.f : wanted >= 0 && wanted < V ? value - at_target[row] : __uint_as_float(0x7fc00000u);
}

// ---- backward ------------------------------------------------------------------------------
// x = power * m, power a power of two with x's sign and m in (0.5, 1]; numbers without a mantissa of their own (0, those below the normal ones,
// infinities, NaN) keep m = 1.
struct Split {
  float power, m;
};
TFK_DEVICE Split split(float x) {
  const unsigned bits = __float_as_uint(x), exponent = bits >> 23 & 0xff;
  if (exponent == 0 || exponent == 0xff || (bits & 0x7fffffu) == 0) return {x, 1.f};
  return {__uint_as_float((bits & 0x80000000u) | min(exponent + 1, 254u) << 23), __uint_as_float((bits & 0x7fffffu) | 126u << 23)};
}

// What a backward pass takes from grad_loss: w (0 for ignored tokens, NaN for targets outside the vocabulary, as the loss), m, and m * H in rows of `width`,
// zeros for ignored tokens.
// Everything is a quarter of grad_loss, divided by that mantissa: factors[tokens] makes up for that, factors[t] has m as well.
// The first workgroup looks for the largest finite one as well, where there is a scale.
constexpr int kWeighThreads = 256;
constexpr int kSearched = 8192;   // tokens at the end of which one is to count
template <typename T>
__global__ __launch_bounds__(kWeighThreads) void weigh_tokens_kernel(const float* __restrict__ grad_loss, const int64_t* __restrict__ target,
                                                                     int64_t ignore_index, int tokens, int V, Scale* scale, float* __restrict__ weights,
                                                                     float* __restrict__ factors, const T* __restrict__ hidden, T* __restrict__ weighted,
                                                                     int K, int width) {
  typedef T eight_t __attribute__((ext_vector_type(8)));
  typedef eight_t eight_any_t __attribute__((aligned(2)));
  const auto counts = [&](int64_t wanted) __attribute__((always_inline)) { return wanted != ignore_index && wanted >= 0 && wanted < V; };
  // The mantissa of the last token that counts: the batch may be padded behind it.  A wavefront looks at 256 tokens at a time.
  float common = 1.f;
  for (int end = tokens; end > 0 && end > tokens - kSearched; end -= 256) {
    const int t = end - 4 * (int)(threadIdx.x % 64) - 1;   // the lane's last one
    int64_t wanted[4];
    float grad[4], mine = 0.f;
#pragma unroll
    for (int n = 0; n < 4; ++n) wanted[n] = target[max(t - n, 0)], grad[n] = grad_loss[max(t - n, 0)];
    bool found = false;
#pragma unroll
    for (int n = 3; n >= 0; --n)
      if (t - n >= 0 && counts(wanted[n])) found = true, mine = grad[n];
    const unsigned long long lanes = __ballot(found);
    if (lanes != 0) {
      common = split(__shfl(mine, __ffsll(lanes) - 1)).m;
      break;
    }
  }
  const int64_t first = (int64_t)blockIdx.x * kWeighThreads + threadIdx.x, step = (int64_t)gridDim.x * kWeighThreads;
  if (weighted != nullptr) {
    const unsigned chunks = (unsigned)width / 8;
    const int64_t count = (int64_t)tokens * chunks;
    for (int64_t i = first; i < count; i += step) {
      const int64_t row = count < ((int64_t)1 << 32) ? (unsigned)i / chunks : i / chunks;
      const int col = (int)(i - row * chunks) * 8;
      const int64_t wanted = target[row];
      const float grad = grad_loss[row];
      eight_t v;
      if (col + 8 <= K) {
        v = *reinterpret_cast<const eight_any_t*>(hidden + row * K + col);
      } else {
#pragma unroll
        for (int t = 0; t < 8; ++t) v[t] = col + t < K ? hidden[row * K + col + t] : (T)0.f;
      }
      const float m = counts(wanted) ? split(grad * 0.25f / common).m : 1.f;
      // (an ignored token's row is what its P, zeros, are multiplied by: it may hold anything, and zero times a NaN is one)
      const bool ignored = wanted == ignore_index;
#pragma unroll
      for (int t = 0; t < 8; ++t) v[t] = ignored ? (T)0.f : (T)((float)v[t] * m);
      *reinterpret_cast<eight_t*>(weighted + i * 8) = v;
    }
  }
  for (int64_t t = first; t < tokens; t += step) {
    const int64_t wanted = target[t];
    const float grad = grad_loss[t];
    const Split s = counts(wanted) ? split(grad * 0.25f / common) : Split{wanted == ignore_index ? 0.f : __uint_as_float(0x7fc00000u), 1.f};
    weights[t] = s.power;
    factors[t] = 4.f * common * s.m;
    if (t == 0) factors[tokens] = 4.f * common;
  }
  if (scale == nullptr || blockIdx.x != 0) return;
  __shared__ float s_top[kWeighThreads / 64];
  float top = 0.f;
  for (int t = threadIdx.x; t < tokens; t += kWeighThreads)
    if (target[t] != ignore_index && fabsf(grad_loss[t]) < INFINITY) top = fmaxf(top, fabsf(grad_loss[t]));
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) top = fmaxf(top, __shfl_xor(top, d));
  if (threadIdx.x % 64 == 0) s_top[threadIdx.x / 64] = top;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < kWeighThreads / 64; ++w) top = fmaxf(top, s_top[w]);
  int e = 0;
  if (top > 0.f) {
    const float m = frexpf(top, &e);   // top = m * 2^e, 0.5 <= m < 1
    if (m == 0.5f) --e;
  }
  // A quarter of the largest, divided by a mantissa, is 2^(e - 1) at most, and so is its power of two.
  e = max(e, -110);   // (2^(16 - e) has to fit as well)
  *scale = Scale{ldexpf(1.f, 16 - e), ldexpf(1.f, e - 16)};
}

template <typename T>
struct ProbEpilogue {
  T* p;                    // [tokens][pitch], the piece's first column
  int64_t pitch;
  int pad;                 // columns of zeros in front of it
  const float *lse, *weights;
  const Scale* scale;      // null: 1
  const int64_t* target;
  int64_t ignore_index;
  int M, N;                // tokens, columns of the piece
  int first;               // the piece's first column

  template <bool kInside, int TM, int TN>
  TFK_DEVICE void run(float4_t (&acc)[TM][TN], const TileAt& at) const {
    const int lr = at.lane & 15, lg = at.lane >> 4;
    const float in = scale != nullptr ? scale->in : 1.f;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int row = kInside ? at.row + 16 * i + lr : min(at.row + 16 * i + lr, M - 1);
      const int64_t wanted = target[row];
      const bool ignored = wanted == ignore_index;
      const float origin = lse[row] * kLog2e;
      const float weight = weights[row] * in;
      const int64_t hot = wanted - first - at.col;   // counted from the tile's first column
      float4_t v[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) v[j][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][r], kLog2e, -origin)) * weight;
      if (__any(hot >= 0 && hot < 16 * TN)) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (hot == 16 * j + 4 * lg + r) v[j][r] = (__builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][r], kLog2e, -origin)) - 1.f) * weight;
      }
      if (__any(ignored)) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) v[j][r] = ignored ? 0.f : v[j][r];
      }
      store_blocks<kInside>(p, (size_t)pitch, at.row + 16 * i, at.col, M, N, at.lane, v);
      if (at.col == 0)
        for (int z = lg; z < pad; z += 4) p[(int64_t)row * pitch - 1 - z] = (T)0.f;   // (the last row again where the tile ends behind it)
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

int64_t aligned_width(int64_t K) { return K % 8 == 0 ? K : round_up_to(K, 64); }

struct ForwardPlan {
  ProductPlan product;
  size_t at_target, hidden, weight, bytes;   // offsets in the workspace (of the parts: 0; hidden, weight: copies), its size
  ForwardPlan(int64_t T, int64_t V, int64_t K) {
    const int64_t width = aligned_width(K);
    product = plan_product(T, V, width, false);
    size_t at = 0;
    auto take = [&](int64_t bytes_) {
      const size_t from = at;
      at += round_up_to(bytes_, 256);
      return from;
    };
    take(sizeof(Part) * T * product.slots);
    at_target = take(sizeof(float) * T);
    hidden = take(width != K ? 2 * T * width : 0);
    weight = take(width != K ? 2 * V * width : 0);
    bytes = at;
  }
};

// What is held for a piece of the vocabulary: P, completed by zeros in front of its columns to a multiple of 64 (they meet the rows of zeros that
// the product over them begins with); and parts of the sums.
struct BackwardPlan {
  int64_t width, piece, pieces;      // K with its zeros, columns of a piece (the last may have fewer)
  ColsPlan of_hidden, of_weight;     // (the last piece's are as those of the others)
  PairPlan both;                     // where both are asked for
  size_t scale, weights, factors, weighted, hidden, weight, hidden_parts, weight_parts, bytes;   // offsets in the workspace (of P: 0), its size
  BackwardPlan(int64_t T, int64_t V, int64_t K) {
    width = aligned_width(K);
    piece = piece_of(T, V);
    pieces = tiles_of(V, piece);
    const ColsSize hidden_size = {T, K, piece / 64}, weight_size = {piece, K, tiles_of(T, 64)};
    of_hidden = plan_cols(hidden_size);
    of_weight = plan_cols(weight_size);
    both = plan_pair(of_hidden, hidden_size, of_weight, weight_size);
    size_t at = 0;
    auto take = [&](int64_t bytes_) {
      const size_t from = at;
      at += round_up_to(bytes_, 256);
      return from;
    };
    take(2 * T * piece);
    scale = take(sizeof(Scale));
    weights = take(4 * T);
    factors = take(4 * (T + 1));
    weighted = take(2 * T * width);
    hidden = take(width != K ? 2 * T * width : 0);
    weight = take(width != K ? 2 * piece * width : 0);
    const auto floats = [K](const ColsPlan& plan, bool cut, int64_t rows) { return cut ? PartsRoom(plan, rows, K).floats : 0; };
    const auto hidden_floats = [&](const ColsPlan& plan) { return floats(plan, pieces > 1 || plan.splits > 1, T); };
    const auto weight_floats = [&](const ColsPlan& plan) { return floats(plan, plan.splits > 1, piece); };
    hidden_parts = take(4 * std::max(hidden_floats(of_hidden), hidden_floats(both.x)));
    weight_parts = take(4 * std::max(weight_floats(of_weight), weight_floats(both.w)));
    bytes = at;
  }
  static int64_t piece_of(int64_t T, int64_t V) {
    return std::min(round_up_to(V, 64), std::min(kPieceColumns, std::max<int64_t>(4096, kPieceElements / T / 256 * 256)));
  }
  static constexpr int64_t kPieceElements = (int64_t)1 << 27;   // of P, 256 MiB
  static constexpr int64_t kPieceColumns = (int64_t)1 << 25;    // P's rows are walked 64 at a time, by 32-bit offsets
  static_assert(cols_farthest(64, kPieceColumns) < (uint64_t)1 << 32);
};

template <typename T>
int forward(const void* hidden, const void* weight, const int64_t* target, float* loss, float* lse, int64_t tokens, int64_t V, int64_t K,
            int64_t ignore_index, char* ws, hipStream_t st) {
  constexpr const char* who = "tf_linear_cross_entropy";
  const ForwardPlan plan(tokens, V, K);
  const int64_t width = aligned_width(K);
  if (width != K) {
    const RowsToCopy both[] = {{hidden, tokens, ws + plan.hidden, tokens}, {weight, V, ws + plan.weight, V}};
    if (int rc = launch_copy_rows(both, 2, 2 * K, 2 * width, st)) return rc;
    hidden = ws + plan.hidden;
    weight = ws + plan.weight;
  }
  Part* const parts = reinterpret_cast<Part*>(ws);
  float* const at_target = reinterpret_cast<float*>(ws + plan.at_target);
  const Operands x = {hidden, {weight, nullptr}, (int)tokens, (int)V, (int)width};
  if (int rc = launch_product<T, false>(who, x, plan.product, LseEpilogue{parts, (int)plan.product.slots, at_target, target, (int)tokens, (int)V}, st))
    return rc;
  return launch_kernel(merge_parts_kernel, dim3((unsigned)tokens), dim3(kMergeThreads), 0, st, parts, (int)plan.product.slots, at_target, target,
                       ignore_index, (int)V, loss, lse);
}

template <typename T>
int backward(const float* grad_loss, const void* hidden, const void* weight, const int64_t* target, const float* lse, void* grad_hidden,
             void* grad_weight, int64_t tokens, int64_t V, int64_t K, int64_t ignore_index, char* ws, hipStream_t st) {
  constexpr const char* who = "tf_linear_cross_entropy_backward";
  if (tokens == 0) return grad_weight != nullptr ? launch_zero_16bit(grad_weight, V * K, st) : TF_OK;
  const BackwardPlan plan(tokens, V, K);
  T* const p = reinterpret_cast<T*>(ws);
  constexpr bool kScaled = std::is_same_v<T, half_t>;
  Scale* const scale = kScaled ? reinterpret_cast<Scale*>(ws + plan.scale) : nullptr;
  float* const hidden_parts = reinterpret_cast<float*>(ws + plan.hidden_parts);
  float* const weight_parts = reinterpret_cast<float*>(ws + plan.weight_parts);
  float *const weights = reinterpret_cast<float*>(ws + plan.weights), *const factors = reinterpret_cast<float*>(ws + plan.factors);
  T* const weighted = grad_weight != nullptr ? reinterpret_cast<T*>(ws + plan.weighted) : nullptr;
  const int64_t items = weighted != nullptr ? tokens * (plan.width / 8) : tokens;
  if (int rc = launch_kernel(weigh_tokens_kernel<T>, dim3((unsigned)std::min<int64_t>(tiles_of(items, kWeighThreads), 4096)), dim3(kWeighThreads), 0, st, grad_loss,
                             target, ignore_index, (int)tokens, (int)V, scale, weights, factors, static_cast<const T*>(hidden), weighted, (int)K, (int)plan.width))
    return rc;
  if (plan.width != K) {
    const RowsToCopy copy = {hidden, tokens, ws + plan.hidden, tokens};
    if (int rc = launch_copy_rows(&copy, 1, 2 * K, 2 * plan.width, st)) return rc;
    hidden = ws + plan.hidden;
  }
  const auto bits = [](const void* t) { return static_cast<const uint16_t*>(t); };
  const int width = (int)plan.width;
  const int t_tiles = (int)tiles_of(tokens, 64), t_pad = (int)(t_tiles * 64 - tokens);
  const ColsOperand of_tokens = {bits(weighted), width, width, (int)K};
  const Factors by_hidden = {scale, nullptr, factors}, by_weight = {scale, factors + tokens, nullptr};
  const bool together = grad_hidden != nullptr && grad_weight != nullptr && plan.both.together;
  const ColsPlan &of_hidden = together ? plan.both.x : plan.of_hidden, &of_weight = together ? plan.both.w : plan.of_weight;
  const PartsRoom hidden_room(of_hidden, tokens, K), weight_room(of_weight, plan.piece, K);
  const bool cut_hidden = plan.pieces > 1 || of_hidden.splits > 1, cut_weight = of_weight.splits > 1;
  for (int64_t first = 0; first < V; first += plan.piece) {
    const int64_t columns = std::min(plan.piece, V - first), pitch = round_up_to(columns, 64);
    const int pad = (int)(pitch - columns);
    const char* w = static_cast<const char*>(weight) + 2 * first * K;
    if (plan.width != K) {
      const RowsToCopy copy = {w, columns, ws + plan.weight, columns};
      if (int rc = launch_copy_rows(&copy, 1, 2 * K, 2 * plan.width, st)) return rc;
      w = ws + plan.weight;
    }
    const Operands logits = {hidden, {w, nullptr}, (int)tokens, (int)columns, width};
    if (int rc = launch_product<T, false>(who, logits, plan_product(tokens, columns, width, false),
                                          ProbEpilogue<T>{p + pad, pitch, pad, lse, weights, scale, target, ignore_index, (int)tokens, (int)columns,
                                                          (int)first},
                                          st))
      return rc;

    // dH += P * W (a short last piece may have fewer parts), dW = P^T * H: the columns of P in front of the piece's are rows that are not stored
    ColsPlan hidden_plan = of_hidden;
    hidden_plan.per_split = (int)tiles_of(pitch / 64, of_hidden.splits);
    hidden_plan.splits = (int)tiles_of(pitch / 64, hidden_plan.per_split);
    const ColsProduct hidden_product = {{bits(p), pitch, (int)pitch, (int)tokens}, {bits(w), width, width, (int)K}, bits(w), INT_MAX, (int)(pitch / 64), pad, 0};
    const ColsProduct weight_product = {{bits(p), pitch, (int)pitch, (int)pitch}, of_tokens, of_tokens.x, INT_MAX, t_tiles, t_pad, pad};
    T* const out = grad_weight != nullptr ? static_cast<T*>(grad_weight) + first * K : nullptr;
    const WholeEpilogue<T> whole_hidden = {static_cast<T*>(grad_hidden), by_hidden, (int)tokens, (int)K};
    const WholeEpilogue<T> whole_weight = {out != nullptr ? out - (int64_t)pad * K : nullptr, by_weight, (int)pitch, (int)K};
    const PartEpilogue part_hidden = {hidden_parts, hidden_room.rows, hidden_room.pitch, first > 0};
    const PartEpilogue part_weight = {weight_parts, weight_room.rows, weight_room.pitch, false};
    int rc = TF_OK;
    if (together) {
      rc = launch_pair<T>(who, hidden_product, hidden_plan, CutEpilogue<WholeEpilogue<T>>{whole_hidden, part_hidden, cut_hidden}, weight_product, of_weight,
                          CutEpilogue<WholeEpilogue<T>>{whole_weight, part_weight, cut_weight}, st);
    } else {
      if (grad_hidden != nullptr)
        rc = cut_hidden ? launch_cols<T, false>(who, hidden_product, hidden_plan, part_hidden, st)
                        : launch_cols<T, false>(who, hidden_product, hidden_plan, whole_hidden, st);
      if (rc == TF_OK && grad_weight != nullptr)
        rc = cut_weight ? launch_cols<T, true>(who, weight_product, of_weight, part_weight, st)
                        : launch_cols<T, true>(who, weight_product, of_weight, whole_weight, st);
    }
    if (rc == TF_OK && grad_weight != nullptr && cut_weight)
      rc = launch_sum_parts<T>(weight_parts, weight_room, of_weight.splits, pad, pitch, K, out, by_weight, st);
    if (rc) return rc;
  }
  if (grad_hidden == nullptr || !cut_hidden) return TF_OK;
  return launch_sum_parts<T>(hidden_parts, hidden_room, of_hidden.splits, 0, tokens, K, static_cast<T*>(grad_hidden), by_hidden, st);
}

int check_sizes(const char* who, int dtype, int64_t T, int64_t V, int64_t K) {
  TFK_REQUIRE(dtype == TF_DTYPE_F16 || dtype == TF_DTYPE_BF16, TF_ERR_UNSUPPORTED, "%s: dtype must be TF_DTYPE_F16 or TF_DTYPE_BF16", who);
  TFK_REQUIRE(T >= 0 && V > 0 && K > 0, TF_ERR_INVALID_ARG, "%s: T must not be negative, V and K must be positive", who);
  TFK_REQUIRE(T <= (1 << 22) - 64 && V <= (1 << 28) - 64 && K <= (1 << 22) - 64, TF_ERR_INVALID_ARG, "%s: dimension too large", who);
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
  TFK_REQUIRE(K % 8 != 0 || (at_16B(hidden) && at_16B(weight)), TF_ERR_INVALID_ARG,
              "tf_linear_cross_entropy: hidden and weight must begin at 16-byte boundaries");
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
  if (T > 0) {   // (grad_hidden of no tokens may be null all the same)
    TFK_REQUIRE(grad_weight || grad_hidden, TF_ERR_INVALID_ARG, "tf_linear_cross_entropy_backward: no gradient asked for");
    TFK_REQUIRE(grad_loss && hidden && weight && target && lse, TF_ERR_INVALID_ARG,
                "tf_linear_cross_entropy_backward: null pointer");
    TFK_REQUIRE(K % 8 != 0 || (at_16B(hidden) && at_16B(weight)), TF_ERR_INVALID_ARG,
                "tf_linear_cross_entropy_backward: hidden and weight must begin at 16-byte boundaries");
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

extern "C" int64_t tf_linear_cross_entropy_backward_piece(int64_t T, int64_t V, int64_t K) {
  using namespace tfk;
  if (T <= 0 || check_sizes("tf_linear_cross_entropy_backward_piece", TF_DTYPE_F16, T, V, K) != TF_OK) return -1;
  return BackwardPlan::piece_of(T, V);
}
