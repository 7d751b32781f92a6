// The gated feed-forward block: h = act(x * Wg^T) * (x * Wu^T) in one kernel, and its backward pass.
//
// Forward.  The two projections are one product whose columns alternate between the two weights in blocks of 16 (Operands), so
// that a lane holds the gate and the up value of an element in the same place of two neighbouring blocks, and the activation and the
// product are done on the accumulators: one rounding, to h.  For training gate and up are kept as well, rounded to the type.
//
// Backward, from the gate and up values that were kept:
//   dg = dh * up * act'(gate), du = dh * act(gate)
//   dx = dg * Wg + du * Wu,  dWg = dg^T * x,  dWu = du^T * x
// One pass over dh, gate and up leaves [dg | du] as rows of tokens, each half completed by zeros to a multiple of 64 columns; dx is one product over the
// 2F columns, the weights' gradients are one over the tokens.  dg and du are rounded to the type once, as operands of
// matrix instructions have to be; in fp16 times a power of two where their own range is not the type's, by which the sums are divided in fp32.
#include "product.hpp"

namespace tfk {
namespace {

// act(g) = g * phi(g), and phi's derivative
TFK_DEVICE float exp_of(float x) { return __builtin_amdgcn_exp2f(1.4426950408889634f * x); }
TFK_DEVICE float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + exp_of(-x)); }
constexpr float kGeluCubic = 0.044715f;
constexpr float kGeluTwice = 1.5957691216057308f;   // 2 * sqrt(2 / pi): (1 + tanh(y)) / 2 = sigmoid(2y)

// The normal distribution's weight below -|g|, from exp(-g^2 / 2): bell * t * p(t), t = 1 / (1 + 0.28 |g|), where t * p(t) stands for
// erfcx(|g| / sqrt(2)) / 2.  p is the polynomial of degree 8 whose largest relative error over all g is least (Remez' exchange): 1.7e-7, so that the
// tail, which is not taken from 1, is right in its leading digits as far out as it is a number of the type.  In fp32 5e-7 up to |g| = 1, and g^2 * 2^-23 further
// out, by the argument of bell.  The library's erff takes both of its branches for every wavefront (2999 x 1032 x 1544 with gate and up kept, fp16:
// 43 us with it, 33 so).
TFK_DEVICE float normal_tail(float g, float bell) {
  const float t = __builtin_amdgcn_rcpf(1.f + 0.28f * fabsf(g));
  float p = 0.024719954f;
  p = __builtin_fmaf(p, t, -0.093593046f);
  p = __builtin_fmaf(p, t, 0.092428006f);
  p = __builtin_fmaf(p, t, -0.0064490973f);
  p = __builtin_fmaf(p, t, 0.072774976f);
  p = __builtin_fmaf(p, t, 0.0836308f);
  p = __builtin_fmaf(p, t, 0.10308466f);
  p = __builtin_fmaf(p, t, 0.1116998f);
  p = __builtin_fmaf(p, t, 0.11170386f);
  return p * t * bell;
}
TFK_DEVICE float act_phi(float g, int activation) {
  if (activation == TF_ACT_SILU) return sigmoid(g);
  if (activation == TF_ACT_GELU) {
    const float tail = normal_tail(g, exp_of(-0.5f * g * g));
    return g < 0.f ? tail : 1.f - tail;
  }
  return sigmoid(kGeluTwice * (g + kGeluCubic * g * g * g));
}
TFK_DEVICE float act(float g, int activation) { return g * act_phi(g, activation); }
// act and its derivative; at infinities, which a kept gate beyond the largest number of its type has become, their limits
TFK_DEVICE void act_both(float g, int activation, float& value, float& slope) {
  if (activation == TF_ACT_GELU) {
    const float bell = exp_of(-0.5f * g * g), tail = normal_tail(g, bell);
    const float p = g < 0.f ? tail : 1.f - tail;
    value = g == -INFINITY ? 0.f : g * p;
    slope = bell > 0.f ? p + g * 0.3989422804014327f * bell : p;
    return;
  }
  const float p = act_phi(g, activation);
  value = g == -INFINITY ? 0.f : g * p;
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

// K is no multiple of 8: rows are copied, completed by zeros to whole lines.
int64_t aligned_width(int64_t K) { return K % 8 == 0 ? K : round_up_to(K, 64); }

struct ForwardPlan {
  size_t w_gate = 0, w_up = 0, bytes = 0;   // copies: offsets (of x: 0), all
  ForwardPlan(int64_t M, int64_t F, int64_t K) {
    if (K % 8 == 0) return;
    w_gate = 2 * M * aligned_width(K);
    w_up = w_gate + 2 * F * aligned_width(K);
    bytes = w_up + 2 * F * aligned_width(K);
  }
};

template <typename T>
int gated_ffn(const void* x, const void* w_gate, const void* w_up, void* h, void* gate, void* up, int activation, int64_t M, int64_t F, int64_t K,
              char* ws, hipStream_t st) {
  constexpr const char* who = "tf_gated_ffn";
  const ForwardPlan copy(M, F, K);
  if (copy.bytes > 0) {
    const int64_t pitch = 2 * aligned_width(K);
    const RowsToCopy all[] = {{x, M, ws, M}, {w_gate, F, ws + copy.w_gate, F}, {w_up, F, ws + copy.w_up, F}};
    if (int rc = launch_copy_rows(all, 3, 2 * K, pitch, st)) return rc;
    x = ws;
    w_gate = ws + copy.w_gate;
    w_up = ws + copy.w_up;
  }
  const Operands operands = {x, {w_gate, w_up}, (int)M, (int)F, (int)aligned_width(K)};
  return launch_product<T, true>(
      who, operands, plan_product(M, F, aligned_width(K), true),
      GatedEpilogue<T>{static_cast<T*>(h), static_cast<T*>(gate), static_cast<T*>(up), (int)M, (int)F, activation}, st);
}

// ---- backward ------------------------------------------------------------------------------
constexpr int kThreads = 256;
// dg and du have a power of two in common.  (bf16 has the range of fp32.)
template <typename T>
constexpr bool kScaled = std::is_same_v<T, half_t>;
constexpr int kMostTops = 1024;   // workgroups that look for the largest

// The largest of the workgroup's numbers, in every thread.
TFK_DEVICE float largest_of_block(float top) {
  __shared__ float s_top[kThreads / 64];
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) top = fmaxf(top, __shfl_xor(top, d));
  if (threadIdx.x % 64 == 0) s_top[threadIdx.x / 64] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) top = fmaxf(top, s_top[w]);
  return top;
}

// Elements i * 8 .. of dg and du to rows [dg | du] of pitch 2 * Fp, zeros behind F columns of each, times `in`; the largest finite one of them in `top`.
template <typename T, int kActivation>
TFK_DEVICE void leave_grads(const T* __restrict__ dh, const T* __restrict__ gate, const T* __restrict__ up, T* __restrict__ rows, int64_t i, int chunks, int F,
                            int Fp, float in, float& top) {
  typedef T eight_t __attribute__((ext_vector_type(8)));
  typedef eight_t eight_any_t __attribute__((aligned(2)));
  const int64_t row = i / chunks;
  const int col = (int)(i - row * chunks) * 8;
  const size_t at = (size_t)row * F + col;
  eight_t d, g, u, dg, du;
  if (col + 8 <= F) {
    d = *reinterpret_cast<const eight_any_t*>(dh + at);
    g = *reinterpret_cast<const eight_any_t*>(gate + at);
    u = *reinterpret_cast<const eight_any_t*>(up + at);
  } else {
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const bool inside = col + t < F;
      d[t] = inside ? dh[at + t] : (T)0.f;
      g[t] = inside ? gate[at + t] : (T)0.f;
      u[t] = inside ? up[at + t] : (T)0.f;
    }
  }
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    float value, slope;
    act_both((float)g[t], kActivation, value, slope);
    const float of_gate = (float)d[t] * (float)u[t] * slope, of_up = (float)d[t] * value;
    if constexpr (kScaled<T>) {
      const float most = fmaxf(fabsf(of_gate), fabsf(of_up)), least = fminf(fabsf(of_gate), fabsf(of_up));
      top = fmaxf(top, most < INFINITY ? most : least < INFINITY ? least : 0.f);
    }
    dg[t] = (T)(of_gate * in);
    du[t] = (T)(of_up * in);
  }
  T* const to = rows + (size_t)row * 2 * Fp + col;
  *reinterpret_cast<eight_t*>(to) = dg;
  *reinterpret_cast<eight_t*>(to + Fp) = du;
}

// [dg | du].  Eight elements a lane; bound by memory (five streams of 16 bits an element).  fp16: tops, the largest of each workgroup.
template <typename T, int kActivation>
__global__ __launch_bounds__(kThreads) void gated_ffn_grads_kernel(const T* __restrict__ dh, const T* __restrict__ gate, const T* __restrict__ up,
                                                                  T* __restrict__ rows, float* __restrict__ tops, int64_t count, int F, int Fp) {
  float top = 0.f;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < count; i += (int64_t)gridDim.x * kThreads)
    leave_grads<T, kActivation>(dh, gate, up, rows, i, Fp / 8, F, Fp, 1.f, top);
  if constexpr (kScaled<T>) {
    top = largest_of_block(top);
    if (threadIdx.x == 0) tops[blockIdx.x] = top;
  }
}

// fp16: where the largest is beyond the type, or so small (below 2^-6) that numbers a 256th of it are below fp16's normal ones, [dg | du] once more, times a
// power of two by which the largest is 2^14 to 2^15.  In between, fp16's smallest number leaves 2^-19 of the largest out of the others at most: less than rounding
// leaves out of numbers that are a 64th of it.  Elsewhere, as with a loss whose scale
// suits the type, there is nothing to do, and the launch is what it costs: backward passes of 1337 x 1544 x 1032 42.8 -> 46.6 us, 2048 x 1024 x 1024 28.4 -> 31.8,
// 8192 x 11264 x 4096 2374 -> 2391 (with 4096 workgroups looking and 2048 here 2435: each of these reads what all of those found).
template <typename T, int kActivation>
__global__ __launch_bounds__(kThreads) void gated_ffn_rescale_kernel(const T* __restrict__ dh, const T* __restrict__ gate, const T* __restrict__ up,
                                                                    T* __restrict__ rows, const float* __restrict__ tops, int num_tops, Scale* scale,
                                                                    int64_t count, int F, int Fp) {
  float top = 0.f;
  for (int i = threadIdx.x; i < num_tops; i += kThreads) top = fmaxf(top, tops[i]);
  top = largest_of_block(top);
  const bool again = top > 0.f && (top < 0.015625f || top > 65504.f);
  int e = 0;
  frexpf(top, &e);                                  // top = m * 2^e, 0.5 <= m < 1
  const int by = again ? min(15 - e, 110) : 0;      // (2^-by has to be a number as well)
  const float in = ldexpf(1.f, by);
  if (blockIdx.x == 0 && threadIdx.x == 0) *scale = Scale{in, ldexpf(1.f, -by)};
  if (!again) return;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < count; i += (int64_t)gridDim.x * kThreads)
    leave_grads<T, kActivation>(dh, gate, up, rows, i, Fp / 8, F, Fp, in, top);
}

template <typename T>
struct GradsKernels {
  decltype(&gated_ffn_grads_kernel<T, TF_ACT_SILU>) grads;
  void (*rescale)(const T*, const T*, const T*, T*, const float*, int, Scale*, int64_t, int, int);   // null: not scaled
};
template <typename T, int kActivation>
GradsKernels<T> grads_kernels_of() {
  if constexpr (kScaled<T>) return {gated_ffn_grads_kernel<T, kActivation>, gated_ffn_rescale_kernel<T, kActivation>};
  else return {gated_ffn_grads_kernel<T, kActivation>, nullptr};
}
template <typename T>
GradsKernels<T> grads_kernels(int activation) {
  if (activation == TF_ACT_SILU) return grads_kernels_of<T, TF_ACT_SILU>();
  if (activation == TF_ACT_GELU) return grads_kernels_of<T, TF_ACT_GELU>();
  return grads_kernels_of<T, TF_ACT_GELU_TANH>();
}

struct BackwardPlan {
  int64_t Fp, Kp;
  bool copy_weights, copy_x;
  ColsPlan of_x, of_w;            // products: dx, the weights' gradients
  PairPlan both;                  // where both are asked for
  int64_t x_floats;               // of dx's parts, which those of the weights' gradients lie behind
  size_t tops, scale, weights, x, parts, bytes;   // offsets in the workspace ([dg | du]: 0), its size
  BackwardPlan(int64_t M, int64_t F, int64_t K) {
    Fp = round_up_to(F, 64);
    Kp = aligned_width(K);
    // the sum over F goes on in the second weight at a whole k-tile
    copy_weights = Kp != K || Fp != F;
    copy_x = Kp != K;
    const ColsSize x_size = {M, K, 2 * Fp / 64}, w_size = {Fp + F, K, tiles_of(M, 64)};
    of_x = plan_cols(x_size);
    of_w = plan_cols(w_size);
    both = plan_pair(of_x, x_size, of_w, w_size);
    size_t at = 0;
    auto take = [&](int64_t bytes_) {
      const size_t from = at;
      at += round_up_to(bytes_, 256);
      return from;
    };
    take(2 * M * 2 * Fp);
    tops = take(sizeof(float) * kMostTops);
    scale = take(sizeof(Scale));
    weights = take(copy_weights ? 2 * 2 * Fp * Kp : 0);
    x = take(copy_x ? 2 * M * Kp : 0);
    const auto floats = [K](const ColsPlan& plan, int64_t rows) { return plan.splits > 1 ? PartsRoom(plan, rows, K).floats : 0; };
    x_floats = floats(both.x, M);
    parts = take(4 * std::max({floats(of_x, M), floats(of_w, Fp + F), both.together ? x_floats + floats(both.w, Fp + F) : 0}));
    bytes = at;
  }
};

// The weights' gradients out of one product over the columns of [dg | du]: rows from Fp on are the second one's.
template <typename T>
struct BothEpilogue {
  WholeEpilogue<T> gate, up;   // M: F, Fp + F; up's `out` is Fp rows in front of it
  int Fp;

  template <bool kInside, int TM, int TN>
  TFK_DEVICE void run(float4_t (&acc)[TM][TN], const TileAt& at) const {
    constexpr int kRows = 16 * TM;
    if (at.row + kRows <= Fp) {
      if (kInside && at.row + kRows <= gate.M) gate.template run<kInside>(acc, at);
      else gate.template run<false>(acc, at);
    } else if (at.row >= Fp) {
      up.template run<kInside>(acc, at);
    } else {
      gate.template run<false>(acc, at);
      TileAt behind = at;
      behind.row_from = Fp;
      up.template run<false>(acc, behind);
    }
  }
};

template <typename T>
int gated_ffn_backward(const void* dh, const void* x, const void* w_gate, const void* w_up, const void* gate, const void* up, void* dx, void* dw_gate,
                       void* dw_up, int activation, int64_t M, int64_t F, int64_t K, char* ws, hipStream_t st) {
  constexpr const char* who = "tf_gated_ffn_backward";
  if (M == 0) {
    if (dw_gate == nullptr) return TF_OK;
    if (int rc = launch_zero_16bit(dw_gate, F * K, st)) return rc;
    return launch_zero_16bit(dw_up, F * K, st);
  }
  const BackwardPlan p(M, F, K);
  T* const rows = reinterpret_cast<T*>(ws);
  const int64_t chunks = M * (p.Fp / 8);
  float* const tops = reinterpret_cast<float*>(ws + p.tops);
  Scale* const scale = kScaled<T> ? reinterpret_cast<Scale*>(ws + p.scale) : nullptr;
  const GradsKernels<T> kernels = grads_kernels<T>(activation);
  const T *const of_h = static_cast<const T*>(dh), *const of_gate = static_cast<const T*>(gate), *const of_up = static_cast<const T*>(up);
  const int64_t blocks = std::min<int64_t>(tiles_of(chunks, kThreads), kScaled<T> ? kMostTops : 65536);
  if (int rc = launch_kernel(kernels.grads, dim3((unsigned)blocks), dim3(kThreads), 0, st, of_h, of_gate, of_up, rows, tops, chunks, (int)F, (int)p.Fp))
    return rc;
  if (scale != nullptr)
    if (int rc = launch_kernel(kernels.rescale, dim3((unsigned)std::min<int64_t>(blocks, 512)), dim3(kThreads), 0, st, of_h, of_gate, of_up, rows, tops,
                               (int)blocks, scale, chunks, (int)F, (int)p.Fp))
      return rc;
  RowsToCopy copies[3];
  int count = 0;
  if (p.copy_weights && dx != nullptr) {
    char* const to = ws + p.weights;
    copies[count++] = {w_gate, F, to, p.Fp};
    copies[count++] = {w_up, F, to + 2 * p.Fp * p.Kp, p.Fp};
    w_gate = to;
    w_up = to + 2 * p.Fp * p.Kp;
  }
  if (p.copy_x && dw_gate != nullptr) {
    copies[count++] = {x, M, ws + p.x, M};
    x = ws + p.x;
  }
  if (count > 0)
    if (int rc = launch_copy_rows(copies, count, 2 * K, 2 * p.Kp, st)) return rc;
  float* const parts = reinterpret_cast<float*>(ws + p.parts);
  const auto bits = [](const void* t) { return static_cast<const uint16_t*>(t); };
  const uint16_t* const grads_at = bits(ws);
  const ColsProduct of_x = {{grads_at, 2 * p.Fp, (int)(2 * p.Fp), (int)M}, {bits(w_gate), p.Kp, (int)p.Kp, (int)K}, bits(w_up), (int)(p.Fp / 64), (int)(2 * p.Fp / 64), 0, 0};
  const int m_tiles = (int)tiles_of(M, 64), m_pad = (int)(m_tiles * 64 - M);
  const ColsOperand tokens = {bits(x), p.Kp, (int)p.Kp, (int)K};
  const ColsProduct of_w = {{grads_at, 2 * p.Fp, (int)(2 * p.Fp), (int)(p.Fp + F)}, tokens, tokens.x, INT_MAX, m_tiles, m_pad, 0};
  T *const to_x = static_cast<T*>(dx), *const to_gate = static_cast<T*>(dw_gate), *const to_up = static_cast<T*>(dw_up);
  const Factors by = {scale, nullptr, nullptr};
  const WholeEpilogue<T> whole_x = {to_x, by, (int)M, (int)K};
  const BothEpilogue<T> whole_w = {{to_gate, by, (int)F, (int)K}, {to_up != nullptr ? to_up - p.Fp * K : nullptr, by, (int)(p.Fp + F), (int)K}, (int)p.Fp};
  const bool together = dx != nullptr && dw_gate != nullptr && p.both.together;
  const ColsPlan &x_plan = together ? p.both.x : p.of_x, &w_plan = together ? p.both.w : p.of_w;
  const PartsRoom x_room(x_plan, M, K), w_room(w_plan, p.Fp + F, K);
  float* const w_parts = together ? parts + p.x_floats : parts;
  const PartEpilogue part_x = {parts, x_room.rows, x_room.pitch, false}, part_w = {w_parts, w_room.rows, w_room.pitch, false};
  if (together)
    if (int rc = launch_pair<T>(who, of_x, x_plan, CutEpilogue<WholeEpilogue<T>>{whole_x, part_x, x_plan.splits > 1}, of_w, w_plan,
                                CutEpilogue<BothEpilogue<T>>{whole_w, part_w, w_plan.splits > 1}, st))
      return rc;
  if (dx != nullptr) {
    if (!together)
      if (int rc = x_plan.splits == 1 ? launch_cols<T, false>(who, of_x, x_plan, whole_x, st) : launch_cols<T, false>(who, of_x, x_plan, part_x, st)) return rc;
    if (x_plan.splits > 1)
      if (int rc = launch_sum_parts<T>(parts, x_room, x_plan.splits, 0, M, K, to_x, by, st)) return rc;
  }
  if (dw_gate == nullptr) return TF_OK;
  if (!together)
    if (int rc = w_plan.splits == 1 ? launch_cols<T, true>(who, of_w, w_plan, whole_w, st) : launch_cols<T, true>(who, of_w, w_plan, part_w, st)) return rc;
  if (w_plan.splits == 1) return TF_OK;
  if (int rc = launch_sum_parts<T>(w_parts, w_room, w_plan.splits, 0, F, K, to_gate, by, st)) return rc;
  return launch_sum_parts<T>(w_parts, w_room, w_plan.splits, p.Fp, p.Fp + F, K, to_up, by, st);
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

extern "C" size_t tf_gated_ffn_workspace_bytes(int64_t M, int64_t F, int64_t K) {
  using namespace tfk;
  if (M <= 0 || check_sizes("tf_gated_ffn_workspace_bytes", TF_DTYPE_F16, TF_ACT_SILU, M, F, K) != TF_OK) return 0;
  return ForwardPlan(M, F, K).bytes;
}

extern "C" int tf_gated_ffn(const void* x, const void* w_gate, const void* w_up, void* h, void* gate, void* up, int dtype, int activation, int64_t M,
                            int64_t F, int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace tfk;
  if (int rc = check_sizes("tf_gated_ffn", dtype, activation, M, F, K)) return rc;
  if (M == 0) return TF_OK;
  TFK_REQUIRE(x && w_gate && w_up && h, TF_ERR_INVALID_ARG, "tf_gated_ffn: null pointer");
  TFK_REQUIRE((gate == nullptr) == (up == nullptr), TF_ERR_INVALID_ARG, "tf_gated_ffn: gate and up are kept both or neither");
  const size_t want = ForwardPlan(M, F, K).bytes;
  TFK_REQUIRE(want > 0 || (at_16B(x) && at_16B(w_gate) && at_16B(w_up)), TF_ERR_INVALID_ARG,
              "tf_gated_ffn: x and the weights must begin at 16-byte boundaries");
  TFK_REQUIRE(want == 0 || (workspace && workspace_bytes >= want && at_16B(workspace)), TF_ERR_INVALID_ARG,
              "tf_gated_ffn: workspace of %zu bytes at a 16-byte boundary needed, got %zu", want, workspace_bytes);
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* const ws = static_cast<char*>(workspace);
  if (dtype == TF_DTYPE_F16) return gated_ffn<half_t>(x, w_gate, w_up, h, gate, up, activation, M, F, K, ws, st);
  return gated_ffn<bf16_t>(x, w_gate, w_up, h, gate, up, activation, M, F, K, ws, st);
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
  TFK_REQUIRE((dw_gate == nullptr) == (dw_up == nullptr), TF_ERR_INVALID_ARG, "tf_gated_ffn_backward: the gradients of both weights or of neither");
  if (M > 0) {   // (dx of no tokens may be null all the same)
    TFK_REQUIRE(dx || dw_gate, TF_ERR_INVALID_ARG, "tf_gated_ffn_backward: no gradient asked for");
    TFK_REQUIRE(dh && x && w_gate && w_up && gate && up, TF_ERR_INVALID_ARG, "tf_gated_ffn_backward: null pointer");
    TFK_REQUIRE(K % 8 != 0 || (at_16B(x) && at_16B(w_gate) && at_16B(w_up)), TF_ERR_INVALID_ARG,
                "tf_gated_ffn_backward: x and the weights must begin at 16-byte boundaries");
    const size_t want = BackwardPlan(M, F, K).bytes;
    TFK_REQUIRE(workspace && workspace_bytes >= want && at_16B(workspace), TF_ERR_INVALID_ARG,
                "tf_gated_ffn_backward: workspace of %zu bytes at a 16-byte boundary needed, got %zu", want, workspace_bytes);
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* const ws = static_cast<char*>(workspace);
  if (dtype == TF_DTYPE_F16)
    return gated_ffn_backward<half_t>(dh, x, w_gate, w_up, gate, up, dx, dw_gate, dw_up, activation, M, F, K, ws, st);
  return gated_ffn_backward<bf16_t>(dh, x, w_gate, w_up, gate, up, dx, dw_gate, dw_up, activation, M, F, K, ws, st);
}
