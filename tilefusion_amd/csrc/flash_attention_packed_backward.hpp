// Gradients of attention over packed sequences (the forward pass: flash_attention_packed_kernel.hpp), in a source file per head dimension.
//
// With P = exp(scale Q K^T - lse) and delta = rowsum(dO o O):   dV = P^T dO,   dS = P o (dO V^T - delta),   dQ = scale dS K,   dK = scale dS^T Q.
// P is made again from the forward pass's log-sum-exp.  No atomics, so that the same bits come out every time:
//   * a first kernel leaves delta, and lse in units of log2, beside each other in the order of rows that the second reads them in;
//   * of the second's workgroups some take 128 keys and walk the rows that see them (all heads of a group are rows, so a group's sum is the same sum), or,
//     where there would be few of those, a part of the rows, and a third kernel adds the parts up;
//   * the others take 128 rows and walk their keys.  That makes P and dO V^T twice, 7 products instead of 5; sums of dQ from the
//     key side would need atomics in fp32, whose order changes results, and a pass of their own over 4 bytes an element.
// Both walk tiles of 32 in a ring in LDS (global_load_lds), their own 32 keys or rows of a wavefront in registers as the second operand of the
// first two products, whose accumulators are the second operand of the last ones as they are, P and dS rounded to the type for that (gradients 2.3e-3 to 2.4e-3 from 64 bits in bf16
// and 2.9e-4 in fp16, relative, over the tensor, where the results' own rounding is 1.7e-3 and 2.1e-4): a lane holds one key (row), its registers
// four rows (keys).  The tile is read from LDS as rows and, transposed, as columns; one swizzle serves both.  Two workgroups of four wavefronts share a
// CU, so that one's exponentials run beside the other's products.
// 4 texts of 2048, 32/8 heads x 128, causal, bf16: 487 to 515 us (as the board's clock is), of which 28 are the first kernel's (HBM) and the rest the second's (7 products at 1.0
// PFLOP/s); fp16 628 to 647, bound by the questions for powers of two between its products.  11 texts of 30 to 1001, 16/4 heads x 64, fp16: 66 us, 5 + 54 + 6.
#pragma once

#include "flash_attention.hpp"
#include "flash_attention_packed.hpp"

namespace tfk {
namespace {

constexpr int kGradWaves = 4, kGradTile = 32;
static_assert(kGradKeys == kGradWaves * 16 * 2, "");
constexpr float kLog2E = 1.4426950408889634f;

// 16 rows that read one logical 16-byte chunk hit 16 different bank groups, and 8 rows that read 32 bytes transposed hit 8 different windows.
template <int CH>
__host__ __device__ constexpr int swz_both(int row, int c) {
  const int pair = CH >= 16 ? row & 7 : (row >> 1) & 3;
  return c ^ (pair << 1 | ((row >> 3) & 1));
}

// Where a lane finds its part of a fragment in a tile [rows][D]: rows lr, chunk 4 kk + lg (rows), or rows 4 lg .. + 3 and 16 more, columns
// 16 db .. + 15, transposed (columns).  The swizzle is an exclusive or of chunk numbers, so that kk and db are one more of the offset in a tile at a multiple of 256 bytes.
struct FragmentOffsets { unsigned row, column; };
template <int D>
TFK_DEVICE FragmentOffsets fragment_offsets() {
  const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4, row = 4 * lg + (lr >> 2), col = 4 * (lr & 3);
  return {(unsigned)(lr * D * 2 + swz_both<D / 8>(lr, lg) * 16), (unsigned)(row * D * 2 + swz_both<D / 8>(row, col / 8) * 16 + (col % 8) * 2)};
}
// (`at`: the tile plus one of the offsets, exclusive or 64 kk or 32 db; the rest is constant)
template <typename T, int D>
TFK_DEVICE typename Vec<T>::v8 column_fragment(unsigned at) {
  using V4 = typename Vec<T>::v4;
  const V4 lo = lds_read_tr4<V4>(at), hi = lds_read_tr4<V4>(at + 16 * D * 2);
  typename Vec<T>::v8 f;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    f[t] = lo[t];
    f[4 + t] = hi[t];
  }
  return f;
}

// One in the sign's place of each 16-bit half that is an infinity or a NaN: an exponent of ones, into which one more carries.
template <typename T>
TFK_DEVICE unsigned not_finite_halves(unsigned two) {
  return ((two & 0x7fff7fffu) + (std::is_same_v<T, bf16_t> ? 0x00800080u : 0x04000400u)) & 0x80008000u;
}
// Zeros in the place of what is not finite.
template <typename T>
TFK_DEVICE void clean(typename Vec<T>::v8& f) {
  uint4_t x = __builtin_bit_cast(uint4_t, f);
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] &= ~((not_finite_halves<T>(x[e]) >> 15) * 0xffffu);
  f = __builtin_bit_cast(typename Vec<T>::v8, x);
}

// fp16: P is taken 2^15 times as large (its smallest number is then 2^-39), and dS times a power of two a lane, by which the largest so far is
// 2^14 to 2^15; both are divided out of the fp32 sums.  bf16 has the range.
template <typename T>
constexpr float kUpP = std::is_same_v<T, bf16_t> ? 0.f : 15.f;
TFK_DEVICE float power_for(float largest) {   // 2^(14 - floor(log2 largest)), within fp32
  const int e = (int)(__builtin_bit_cast(unsigned, largest) >> 23 & 255u);
  return __builtin_bit_cast(float, (unsigned)min(max(127 + 14 + 127 - e, 27), 227) << 23);
}

// 16 bytes a lane from base + offset to LDS; base is wavefront-uniform.
TFK_DEVICE void lds_dma_from(const void* base, unsigned offset, unsigned lds_addr) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "{m0}"(lds_addr) : "memory");
}

struct GradArgs {
  PackedArgs packed;      // of query, key and value
  const void *query, *key, *value, *out, *grad_out;   // out, grad_out [tokens][heads][D]
  const float* lse;       // [heads][tokens]
  // [kv_heads][tokens * group]: lse * log2 e, delta, and nothing, so that a row is 16 bytes: all requests to LDS are of one size (requests of 4
  // bytes are done before older ones of 16, and a count of those on their way would not tell which have landed)
  float4_t* stats;
  void *grad_query, *grad_key, *grad_value;            // contiguous
  float scale, scale_log2;
  int key_groups, parts;   // workgroups for dK and dV; parts that the rows of each of their tiles are cut into
  float* partial;          // parts > 1: [parts][dK, dV][kv_tokens][kv_heads][D] in fp32
  unsigned group_factor;   // ceil(2^32 / group): the high half of n * it is n / group for n < 2^22, where group is not 1
};

// Every row of a tile is 16 lanes wide at most; a thread takes 8 elements of a row of out and grad_out.
template <typename T, int D>
__global__ __launch_bounds__(256) void packed_stats_kernel(GradArgs a) {
  using V8 = typename Vec<T>::v8;
  constexpr int kLanes = D / 8;
  const int64_t row = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes, all = (int64_t)a.packed.tokens * a.packed.heads;
  const int64_t at = (row < all ? row : all - 1) * D + threadIdx.x % kLanes * 8;
  const V8 o = *reinterpret_cast<const V8*>(static_cast<const T*>(a.out) + at), g = *reinterpret_cast<const V8*>(static_cast<const T*>(a.grad_out) + at);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum = fmaf((float)o[i], (float)g[i], sum);
#pragma unroll
  for (int d = 1; d < kLanes; d *= 2) sum += __shfl_xor(sum, d);
  if (row >= all || threadIdx.x % kLanes != 0) return;
  const int token = (int)(row / a.packed.heads), head = (int)(row % a.packed.heads), group = (int)a.packed.group.d;
  const float4_t x = {a.lse[(size_t)head * a.packed.tokens + token] * kLog2E, sum, 0.f, 0.f};
  a.stats[((size_t)(head / group) * a.packed.tokens + token) * group + head % group] = x;
}

// Columns 16 db + 4 lg .. of row lr, times `factor` (of the lane's row lr), to row st_row of `to` (the lane's pointer to that row's segment).
template <typename T, int kDB>
TFK_DEVICE void store_transposed(const float4_t (&acc)[kDB], float factor, T* to, bool there) {
  using V2 = typename Vec<T>::v2;
  const int lane = threadIdx.x & 63, st_row = lane >> 2, st_seg = lane & 3, src_lane = st_row + 16 * (((st_seg & 1) << 1) | (st_seg >> 1));
#pragma unroll
  for (int db = 0; db < kDB; db += 2) {
    unsigned x[2], y[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const V2 hx = {(T)(acc[db][2 * h] * factor), (T)(acc[db][2 * h + 1] * factor)};
      const V2 hy = {(T)(acc[db + 1][2 * h] * factor), (T)(acc[db + 1][2 * h + 1] * factor)};
      x[h] = __builtin_bit_cast(unsigned, hx);
      y[h] = __builtin_bit_cast(unsigned, hy);
#if defined(__HIP_DEVICE_COMPILE__)
      auto sw = __builtin_amdgcn_permlane16_swap(x[h], y[h], false, false);
      x[h] = sw[0];
      y[h] = sw[1];
#endif
    }
    uint4_t v;
    v[0] = (unsigned)__builtin_amdgcn_ds_bpermute(4 * src_lane, (int)x[0]);
    v[1] = (unsigned)__builtin_amdgcn_ds_bpermute(4 * src_lane, (int)x[1]);
    v[2] = (unsigned)__builtin_amdgcn_ds_bpermute(4 * src_lane, (int)y[0]);
    v[3] = (unsigned)__builtin_amdgcn_ds_bpermute(4 * src_lane, (int)y[1]);
    if (there) *reinterpret_cast<uint4_t*>(to + 16 * db + 8 * st_seg) = v;
  }
}

// What a lane's dS are multiplied by (fp16): at first as much as numbers can be, so that nothing has to be known of whether there were any.
struct Power {
  float up = 0x1p100f;
};
// Four dS of a lane for each of kN operands, times its power of two, into halves `h`, of which the first may be there; `acc` are the sums that hold them.
// (One question for all of them: in fp16 every branch here parts the products in front of it from those behind.)
template <typename T, int kN, int kDB>
TFK_DEVICE void to_operands(const float4_t (&ds)[kN], int h, typename Vec<T>::v8 (&f)[kN], Power (&power)[kN], float4_t (&acc)[kN][kDB]) {
  if constexpr (!std::is_same_v<T, bf16_t>) {
    bool beyond = false;
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const float4_t& d = ds[n];
      beyond |= fmaxf(fmaxf(__builtin_fabsf(d[0]), __builtin_fabsf(d[1])), fmaxf(__builtin_fabsf(d[2]), __builtin_fabsf(d[3]))) * power[n].up > 32768.f;
    }
    if (__builtin_amdgcn_ballot_w64(beyond) != 0) {
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        // (infinities and NaN go through as they are, and do not count for those beside them)
        float finite = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t) finite = fmaxf(finite, __builtin_fabsf(ds[n][t]) < INFINITY ? __builtin_fabsf(ds[n][t]) : 0.f);
        const float largest = quad_max(finite);
        if (largest * power[n].up > 32768.f) {
          const float up = power_for(largest), factor = up / power[n].up;
          power[n].up = up;
#pragma unroll
          for (int db = 0; db < kDB; ++db) acc[n][db] *= factor;
          if (h == 1) {
#pragma unroll
            for (int t = 0; t < 4; ++t) f[n][t] = (T)((float)f[n][t] * factor);
          }
        }
      }
    }
  }
#pragma unroll
  for (int n = 0; n < kN; ++n)
#pragma unroll
    for (int t = 0; t < 4; ++t) f[n][4 * h + t] = (T)(std::is_same_v<T, bf16_t> ? ds[n][t] : ds[n][t] * power[n].up);
}

template <int D>
constexpr int grad_stage_bytes() { return 2 * kGradTile * D * 2 + kGradTile * 16; }
constexpr int kGradStages = 4;
// Fragments of a wavefront's own values that stay in LDS behind the ring and are read again for each 16 rows, with D = 128: the powers of two (fp16) and masks
// (causal) leave too few registers for all of them, and what the compiler put into scratch instead was fetched behind a wait for every request of
// the ring (4 x 2048 x 32 heads, causal: fp16 787 us, 672 so, bf16 523 and 504; not causal, bf16: 825 and 830).  Two workgroups share a CU's LDS, which has
// room for three.
template <typename T, int D, bool kCausal>
constexpr int kGradHeld = D == 128 && (kCausal || !std::is_same_v<T, bf16_t>) ? 3 : 0;
template <typename T, int D, bool kCausal>
constexpr int grad_lds_bytes() { return kGradStages * grad_stage_bytes<D>() + kGradWaves * kGradHeld<T, D, kCausal> * 1024; }

// ---- dK and dV of 128 keys ------------------------------------------------------------------------
// `group_no` of `groups` workgroups.
template <typename T, int D, bool kCausal, int kKB>
TFK_DEVICE void grad_keys(const GradArgs& g, char* smem, int group_no, int groups) {
  using V8 = typename Vec<T>::v8;
  constexpr int kChunks = D / 8, kRowsPerInstr = 64 / kChunks, kTileBytes = kGradTile * D * 2;
  constexpr int kStage = grad_stage_bytes<D>(), kPerWave = kTileBytes / 1024 / kGradWaves, kRequests = 2 * kPerWave + 1;
  constexpr int kKK = D / 32, kDB = D / 16, kGradOwn = kGradWaves * 16 * kKB;
  const PackedArgs& a = g.packed;
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  T* const grad_key = static_cast<T*>(g.grad_key);
  T* const grad_value = static_cast<T*>(g.grad_value);
  if (g.parts == 1) {
    rows_outside(a.kv_offsets, a.sequences, a.kv_tokens, group_no, groups, [&](int row) {
      clear_row(grad_key + (size_t)row * a.kv_heads * D, a.kv_heads * D);
      clear_row(grad_value + (size_t)row * a.kv_heads * D, a.kv_heads * D);
    });
  }
  const int part = group_no / a.kv_heads % g.parts, head = group_no % a.kv_heads, group = (int)a.group.d;
  const PackedTile tile = packed_key_tile(a, kGradOwn, group_no / a.kv_heads / g.parts);
  if (tile.sequence < 0) return;
  const int shift = tile.lkv - tile.lq, rows = tile.lq * group, key0 = tile.from_end * kGradOwn;   // (counted from the front)
  const T* const Q = static_cast<const T*>(g.query) + (size_t)tile.q0 * a.query_row + head * a.query_group;
  const T* const dO = static_cast<const T*>(g.grad_out) + ((size_t)tile.q0 * a.heads + (size_t)head * group) * D;
  const float4_t* const stats = g.stats + ((size_t)head * a.tokens + tile.q0) * group;

  // ---- this wavefront's keys: blocks wave and wave + 4 of 16 (so that all have as much behind the diagonal) ----
  V8 kf[kKB][kKK], vf[kKB][kKK];
#pragma unroll
  for (int kb = 0; kb < kKB; ++kb) {
    const int key = key0 + 16 * (kGradWaves * kb + wave) + lr;
    const size_t at = tile.k0 + min(key, tile.lkv - 1);
    const T* k = static_cast<const T*>(g.key) + at * a.key_row + head * a.key_head;
    const T* v = static_cast<const T*>(g.value) + at * a.value_row + head * a.value_head;
#pragma unroll
    for (int kk = 0; kk < kKK; ++kk) {
      kf[kb][kk] = *reinterpret_cast<const V8*>(k + 32 * kk + 8 * lg);
      vf[kb][kk] = *reinterpret_cast<const V8*>(v + 32 * kk + 8 * lg);
    }
  }
  constexpr int kHeld = kGradHeld<T, D, kCausal>;   // the last ones of the last block
  const unsigned smem_base = lds_address(smem), held = smem_base + kGradStages * kStage + wave * kHeld * 1024;
  auto held_at = [&]() __attribute__((always_inline)) { return held + opaque((unsigned)tid & 63u) * 16; };
#pragma unroll
  for (int i = 0; i < kHeld; ++i) *(__attribute__((address_space(3))) V8*)(size_t)(held_at() + i * 1024) = vf[kKB - 1][kKK - kHeld + i];
  const int tiles = (rows + kGradTile - 1) / kGradTile;
  const int all_first = kCausal ? min(tiles, max(key0 - shift, 0) * group / kGradTile) : 0;
  // of the tiles that see these keys, this part's
  const int first = all_first + (int)((int64_t)(tiles - all_first) * part / g.parts), end = all_first + (int)((int64_t)(tiles - all_first) * (part + 1) / g.parts);
  // tiles from here on are masked for none of this wavefront's keys, but for the last one's rows behind the last
  const int last_min = __builtin_amdgcn_readfirstlane(kCausal ? max(key0 + 16 * (kGradWaves * (kKB - 1) + wave) + 15 - shift, 0) * group : 0);
  const int n_masked = min(tiles, (last_min + kGradTile - 1) / kGradTile), n_full = rows / kGradTile;
  const int first_min = __builtin_amdgcn_readfirstlane(kCausal ? max(key0 + 16 * wave - shift, 0) * group : 0);

  auto request_tile = [&](int t) __attribute__((always_inline)) {
    const unsigned stage = smem_base + t % kGradStages * kStage;
    const int lane = (int)opaque((unsigned)tid & 63u);   // (what follows from it is made again for each tile: registers are short)
    // (from the token of the tile's first row, behind which 32 bits reach any row of it)
    const int r0 = min(t, tiles - 1) * kGradTile, token0 = divide(a.group, r0), skipped = token0 * group, last = rows - 1 - skipped;
    const T* const q = Q + (size_t)token0 * a.query_row;
    const T* const o = dO + (size_t)token0 * a.heads * D;
#pragma unroll
    for (int i = 0; i < kPerWave; ++i) {
      const int instr = wave + kGradWaves * i, row_l = instr * kRowsPerInstr + lane / kChunks;
      const int row = min(r0 - skipped + row_l, last), token = group == 1 ? row : (int)__umulhi((unsigned)row, g.group_factor), hg = row - token * group;
      const int col = swz_both<kChunks>(row_l, lane % kChunks) * 8;
      lds_dma_from(q, (unsigned)(token * a.query_row + hg * a.query_head + col) * 2u, stage + instr * 1024);
      lds_dma_from(o, (unsigned)((token * a.heads + hg) * D + col) * 2u, stage + kTileBytes + instr * 1024);
    }
    // 8 rows' statistics
    if (lane < 8) lds_dma_from(stats + r0, (unsigned)min(8 * wave + lane, rows - 1 - r0) * 16u, stage + 2 * kTileBytes + wave * 128);
  };

  const FragmentOffsets off = fragment_offsets<D>();
  float4_t dk[kKB][kDB], dv[kKB][kDB];
  Power power[kKB];
#pragma unroll
  for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
    for (int db = 0; db < kDB; ++db) dk[kb][db] = dv[kb][db] = float4_t{0.f, 0.f, 0.f, 0.f};

  auto compute = [&](int t, auto mask_c) __attribute__((always_inline)) {
    constexpr bool kMask = decltype(mask_c)::value;
    const unsigned stage = smem_base + t % kGradStages * kStage;
    V8 pf[kKB], sf[kKB];
    [[maybe_unused]] int row_min[kKB];   // the first row of the tile that sees key lr of a block
    if constexpr (kMask) {
      const int own = (int)opaque((unsigned)lr);
#pragma unroll
      for (int kb = 0; kb < kKB; ++kb)
        row_min[kb] = (kCausal ? max(key0 + 16 * (kGradWaves * kb + wave) + own - shift, 0) * group : 0) - t * kGradTile;
    }
    [[maybe_unused]] float odd = 0.f;   // NaN where a score or dP is not finite, as all are of a row of Q or dO with an infinity or a NaN
    const unsigned row_at = opaque(stage + off.row), column_at = opaque(stage + off.column);
    [[maybe_unused]] const unsigned held_from = kHeld > 0 ? held_at() : 0u;
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      float4_t s[kKB], dp[kKB];
#pragma unroll
      for (int kb = 0; kb < kKB; ++kb) s[kb] = dp[kb] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < kKK; ++kk) {
        const unsigned at = row_at ^ (kk << 6);
        const V8 q = lds_read_b128<V8>(at + rb * 16 * D * 2), o = lds_read_b128<V8>(at + rb * 16 * D * 2 + kTileBytes);
#pragma unroll
        for (int kb = 0; kb < kKB; ++kb) s[kb] = mfma_t<T>(q, kf[kb][kk], s[kb]);
#pragma unroll
        for (int kb = 0; kb < kKB; ++kb)
          dp[kb] = mfma_t<T>(o, kb == kKB - 1 && kk >= kKK - kHeld ? lds_read_b128<V8>(held_from + (kk - kKK + kHeld) * 1024) : vf[kb][kk], dp[kb]);
        if (kk % 2 == 1) __builtin_amdgcn_sched_barrier(0);   // (more of them ahead cost registers that there are not)
      }
      float4_t ds[kKB];
      // rows 16 rb + 4 lg + r: their lse and delta
      float base[4], delta[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float2_t x = lds_read_b64<float2_t>(stage + 2 * kTileBytes + (16 * rb + 4 * lg + r) * 16);
        base[r] = kUpP<T> - x[0];
        delta[r] = x[1];
      }
#pragma unroll
      for (int kb = 0; kb < kKB; ++kb) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float p = __builtin_amdgcn_exp2f(fmaf(s[kb][r], g.scale_log2, base[r])), d = p * (dp[kb][r] - delta[r]);
          if constexpr (kMask) {
            odd = fmaf(s[kb][r], 0.f, fmaf(dp[kb][r], 0.f, odd));
            const int row = 16 * rb + 4 * lg + r;
            const bool sees = row >= row_min[kb] && row < rows - t * kGradTile;
            p = sees ? p : 0.f;
            d = sees ? d : 0.f;
          }
          pf[kb][4 * rb + r] = (T)p;
          ds[kb][r] = d;
        }
      }
      to_operands<T, kKB, kDB>(ds, rb, sf, power, dk);
      __builtin_amdgcn_sched_barrier(0);
    }
    // Infinities and NaN in rows that a part of the keys does not see (there a weight of zero would make NaN of them) are taken out of the products.  Of Q
    // that leaves the right NaN: a row with them has NaN weights.  Those of dO go to the keys that see them one by one.
    bool found = false;
    if constexpr (kMask) {
      found = __builtin_amdgcn_ballot_w64(odd != 0.f) != 0;
      for (int i = 0; found && i < kTileBytes / 1024; ++i) {
        const uint4_t x = lds_read_b128<uint4_t>(stage + kTileBytes + lane * 16 + i * 1024);
        unsigned mine = 0;   // a bit for each of the eight
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned bits = not_finite_halves<T>(x[e]);
          mine |= ((bits >> 15 & 1u) | (bits >> 30 & 2u)) << (2 * e);
        }
        for (;;) {
          const unsigned long long lanes = __builtin_amdgcn_ballot_w64(mine != 0);
          if (lanes == 0) break;
          const int from = __builtin_ctzll(lanes), e = __builtin_ctz(__builtin_amdgcn_readlane(mine, from));
          const unsigned pair = e < 4 ? (e < 2 ? x[0] : x[1]) : (e < 6 ? x[2] : x[3]);
          const unsigned short bits = (unsigned short)(__builtin_amdgcn_readlane(pair, from) >> (e % 2 * 16));
          const float value = (float)__builtin_bit_cast(T, bits);
          const int row_l = i * kRowsPerInstr + from / kChunks, col = swz_both<kChunks>(row_l, from % kChunks) * 8 + e;
#pragma unroll
          for (int kb = 0; kb < kKB; ++kb) {
            const float to_key = row_l >= row_min[kb] && row_l < rows - t * kGradTile ? value : 0.f;
#pragma unroll
            for (int db = 0; db < kDB; ++db)
#pragma unroll
              for (int r = 0; r < 4; ++r) dv[kb][db][r] += 16 * db + 4 * lg + r == col ? to_key : 0.f;
          }
          if (lane == from) mine &= mine - 1;
        }
      }
    }
#pragma unroll
    for (int db = 0; db < kDB; ++db) {
      const unsigned at = column_at ^ (db << 5);
      V8 o = column_fragment<T, D>(at + kTileBytes), q = column_fragment<T, D>(at);
      if (found) {
        clean<T>(o);
        clean<T>(q);
      }
#pragma unroll
      for (int kb = 0; kb < kKB; ++kb) dv[kb][db] = mfma_t<T>(o, pf[kb], dv[kb][db]);
#pragma unroll
      for (int kb = 0; kb < kKB; ++kb) dk[kb][db] = mfma_t<T>(q, sf[kb], dk[kb][db]);
      if (db % 2 == 1) __builtin_amdgcn_sched_barrier(0);
    }
  };

  if (first < end) {
#pragma unroll
    for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
      for (int kk = 0; kk < kKK; ++kk) {   // (waited for here, not among the tiles)
        asm volatile("" : "+v"(kf[kb][kk]));
        if (kb < kKB - 1 || kk < kKK - kHeld) asm volatile("" : "+v"(vf[kb][kk]));
      }
#pragma unroll
    for (int t = 0; t < kGradStages - 1; ++t) request_tile(first + t);
    auto next_tile = [&](int t) __attribute__((always_inline)) {
      barrier_keep_vmem<(kGradStages - 2) * kRequests>();   // tile t has landed, tile t-1 has been read
      request_tile(t + kGradStages - 1);
    };
    for (int t = first; t < end; ++t) {
      for (; t >= n_masked && t < min(n_full, end); ++t) {
        next_tile(t);
        compute(t, std::false_type{});
      }
      if (t >= end) break;
      next_tile(t);
      // (otherwise none of the rows sees a key of this wavefront's)
      if ((t + 1) * kGradTile > first_min) compute(t, std::true_type{});
    }
    wait_vmem_all();   // the requests past the last tile must not outlive the workgroup's LDS
  }

  const int st_row = lane >> 2;
#pragma unroll
  for (int kb = 0; kb < kKB; ++kb) {
    if (g.parts > 1) {
      const int key = key0 + 16 * (kGradWaves * kb + wave) + lr;
      if (key >= tile.lkv) continue;
      const float down_k = std::is_same_v<T, bf16_t> ? 1.f : 1.f / power[kb].up;
      const size_t all = (size_t)a.kv_tokens * a.kv_heads * D, at = ((size_t)(tile.k0 + key) * a.kv_heads + head) * D + 4 * lg;
      float* to = g.partial + 2 * part * all + at;
#pragma unroll
      for (int db = 0; db < kDB; ++db) {
        *reinterpret_cast<float4_t*>(to + 16 * db) = dk[kb][db] * down_k;
        *reinterpret_cast<float4_t*>(to + all + 16 * db) = dv[kb][db];
      }
      continue;
    }
    const int key = key0 + 16 * (kGradWaves * kb + wave) + st_row;
    const bool there = key < tile.lkv;
    const size_t at = ((size_t)(tile.k0 + (there ? key : 0)) * a.kv_heads + head) * D;
    constexpr float kDownP = std::is_same_v<T, bf16_t> ? 1.f : 1.f / 32768.f;
    float down = g.scale * kDownP;
    if constexpr (!std::is_same_v<T, bf16_t>) {
      // (in two steps: the power alone may be beyond what is left of fp32's range)
#pragma unroll
      for (int db = 0; db < kDB; ++db) dk[kb][db] *= 1.f / power[kb].up;
    }
    store_transposed<T, kDB>(dk[kb], down, grad_key + at, there);
    store_transposed<T, kDB>(dv[kb], kDownP, grad_value + at, there);
  }
}

// ---- dQ of 128 rows --------------------------------------------------------------------------------
template <typename T, int D, bool kCausal, int kQB>
TFK_DEVICE void grad_queries(const GradArgs& g, char* smem, int group_no, int groups) {
  using V8 = typename Vec<T>::v8;
  constexpr int kChunks = D / 8, kRowsPerInstr = 64 / kChunks, kTileBytes = kGradTile * D * 2;
  constexpr int kStage = 2 * kTileBytes, kPerWave = kTileBytes / 1024 / kGradWaves, kRequests = 2 * kPerWave;
  constexpr int kKK = D / 32, kDB = D / 16, kGradOwn = kGradWaves * 16 * kQB;
  const PackedArgs& a = g.packed;
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  T* const grad_query = static_cast<T*>(g.grad_query);
  rows_outside(a.offsets, a.sequences, a.tokens, group_no, groups, [&](int row) { clear_row(grad_query + (size_t)row * a.heads * D, a.heads * D); });
  const PackedTile tile = packed_tile(a, kGradOwn, group_no / a.kv_heads);
  if (tile.sequence < 0) return;
  const int head = group_no % a.kv_heads, group = (int)a.group.d;
  const int Lkv = tile.lkv, shift = tile.lkv - tile.lq, rows = tile.lq * group;
  const int tile_row0 = ((rows + kGradOwn - 1) / kGradOwn - 1 - tile.from_end) * kGradOwn;
  const T* const Q = static_cast<const T*>(g.query) + (size_t)tile.q0 * a.query_row + head * a.query_group;
  const size_t at_head = ((size_t)tile.q0 * a.heads + (size_t)head * group) * D;
  const T* const dO = static_cast<const T*>(g.grad_out) + at_head;
  const T* const K = static_cast<const T*>(g.key) + (size_t)tile.k0 * a.key_row + head * a.key_head;
  const T* const V = static_cast<const T*>(g.value) + (size_t)tile.k0 * a.value_row + head * a.value_head;
  const float4_t* const stats = g.stats + ((size_t)head * a.tokens + tile.q0) * group;
  auto limit_of = [&](int row) __attribute__((always_inline)) { return kCausal ? min(Lkv - 1, divide(a.group, min(row, rows - 1)) + shift) : Lkv - 1; };

  // ---- this wavefront's rows: blocks wave and wave + 4 of 16 ----------------------------------
  V8 qf[kQB][kKK], of[kQB][kKK];
  float base[kQB], delta[kQB];
  int limit[kQB];
#pragma unroll
  for (int qb = 0; qb < kQB; ++qb) {
    const int row = min(tile_row0 + 16 * (kGradWaves * qb + wave) + lr, rows - 1), token = divide(a.group, row), hg = row - token * group;
    limit[qb] = limit_of(row);
    const float4_t x = stats[row];
    base[qb] = kUpP<T> - x[0];
    delta[qb] = x[1];
#pragma unroll
    for (int kk = 0; kk < kKK; ++kk) {
      qf[qb][kk] = *reinterpret_cast<const V8*>(Q + (size_t)token * a.query_row + (size_t)hg * a.query_head + 32 * kk + 8 * lg);
      of[qb][kk] = *reinterpret_cast<const V8*>(dO + ((size_t)token * a.heads + hg) * D + 32 * kk + 8 * lg);
    }
  }
  const int n_end = limit_of(tile_row0 + kGradOwn - 1) + 1, tiles = n_end <= 0 ? 0 : (n_end + kGradTile - 1) / kGradTile;
  // of this wavefront: tiles that every row sees whole, and those that any row sees
  const int n_plain = max(0, (__builtin_amdgcn_readfirstlane(limit_of(tile_row0 + 16 * wave)) + 1) / kGradTile);
  const int last = __builtin_amdgcn_readfirstlane(limit_of(tile_row0 + 16 * (kGradWaves * (kQB - 1) + wave) + 15));
  const int n_compute = last < 0 ? 0 : last / kGradTile + 1;

  const unsigned smem_base = lds_address(smem);
  auto request_tile = [&](int t) __attribute__((always_inline)) {
    const unsigned stage = smem_base + t % kGradStages * kStage;
    const int n0 = min(t, tiles - 1) * kGradTile;
    const T* const k = K + (size_t)n0 * a.key_row;
    const T* const v = V + (size_t)n0 * a.value_row;
#pragma unroll
    for (int i = 0; i < kPerWave; ++i) {
      const int instr = wave + kGradWaves * i, row_l = instr * kRowsPerInstr + lane / kChunks, key = min(row_l, Lkv - 1 - n0);
      const int col = swz_both<kChunks>(row_l, lane % kChunks) * 8;
      lds_dma_from(k, (unsigned)(key * a.key_row + col) * 2u, stage + instr * 1024);
      lds_dma_from(v, (unsigned)(key * a.value_row + col) * 2u, stage + kTileBytes + instr * 1024);
    }
  };
  const FragmentOffsets off = fragment_offsets<D>();
  float4_t dq[kQB][kDB];
  Power power[kQB];
#pragma unroll
  for (int qb = 0; qb < kQB; ++qb)
#pragma unroll
    for (int db = 0; db < kDB; ++db) dq[qb][db] = float4_t{0.f, 0.f, 0.f, 0.f};

  auto compute = [&](int t, auto mask_c) __attribute__((always_inline)) {
    constexpr bool kMask = decltype(mask_c)::value;
    const unsigned stage = smem_base + t % kGradStages * kStage;
    V8 sf[kQB];
    [[maybe_unused]] float odd = 0.f;   // NaN where a score is not finite, as all are of a key with an infinity or a NaN
    const unsigned row_at = opaque(stage + off.row), column_at = opaque(stage + off.column);
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      float4_t s[kQB], dp[kQB];
#pragma unroll
      for (int qb = 0; qb < kQB; ++qb) s[qb] = dp[qb] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < kKK; ++kk) {
        const unsigned at = row_at ^ (kk << 6);
        const V8 k = lds_read_b128<V8>(at + kb * 16 * D * 2), v = lds_read_b128<V8>(at + kb * 16 * D * 2 + kTileBytes);
#pragma unroll
        for (int qb = 0; qb < kQB; ++qb) s[qb] = mfma_t<T>(k, qf[qb][kk], s[qb]);
#pragma unroll
        for (int qb = 0; qb < kQB; ++qb) dp[qb] = mfma_t<T>(v, of[qb][kk], dp[qb]);
      }
      float4_t ds[kQB];
#pragma unroll
      for (int qb = 0; qb < kQB; ++qb) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float d = __builtin_amdgcn_exp2f(fmaf(s[qb][r], g.scale_log2, base[qb])) * (dp[qb][r] - delta[qb]);
          if constexpr (kMask) {
            odd = fmaf(s[qb][r], 0.f, odd);
            if (t * kGradTile + 16 * kb + 4 * lg + r > limit[qb]) d = 0.f;
          }
          ds[qb][r] = d;
        }
      }
      to_operands<T, kQB, kDB>(ds, kb, sf, power, dq);
    }
    // Infinities and NaN in keys that a part of the rows does not see are taken out of the product: the rows that see them have NaN weights.
    bool found = false;
    if constexpr (kMask) found = __builtin_amdgcn_ballot_w64(odd != 0.f) != 0;
#pragma unroll
    for (int db = 0; db < kDB; ++db) {
      V8 k = column_fragment<T, D>(column_at ^ (db << 5));
      if (found) clean<T>(k);
#pragma unroll
      for (int qb = 0; qb < kQB; ++qb) dq[qb][db] = mfma_t<T>(k, sf[qb], dq[qb][db]);
    }
  };

  if (tiles > 0) {
#pragma unroll
    for (int qb = 0; qb < kQB; ++qb) {
#pragma unroll
      for (int kk = 0; kk < kKK; ++kk) asm volatile("" : "+v"(qf[qb][kk]), "+v"(of[qb][kk]));   // (waited for here, not among the tiles)
      asm volatile("" : "+v"(base[qb]), "+v"(delta[qb]));
    }
#pragma unroll
    for (int t = 0; t < kGradStages - 1; ++t) request_tile(t);
    auto next_tile = [&](int t) __attribute__((always_inline)) {
      barrier_keep_vmem<(kGradStages - 2) * kRequests>();   // tile t has landed, tile t-1 has been read
      request_tile(t + kGradStages - 1);
    };
    int t = 0;
    for (; t < min(n_plain, tiles); ++t) {
      next_tile(t);
      compute(t, std::false_type{});
    }
    for (; t < tiles; ++t) {
      next_tile(t);
      if (t < n_compute) compute(t, std::true_type{});
    }
    wait_vmem_all();
  }

  const int st_row = lane >> 2;
#pragma unroll
  for (int qb = 0; qb < kQB; ++qb) {
    const int row = tile_row0 + 16 * (kGradWaves * qb + wave) + st_row;
    const bool there = row < rows;
    const int token = divide(a.group, there ? row : 0), hg = (there ? row : 0) - token * group;
    float down = g.scale;
    if constexpr (!std::is_same_v<T, bf16_t>) {
      down *= 1.f / 32768.f;
#pragma unroll
      for (int db = 0; db < kDB; ++db) dq[qb][db] *= 1.f / power[qb].up;
    }
    store_transposed<T, kDB>(dq[qb], down, grad_query + at_head + ((size_t)token * a.heads + hg) * D, there);
  }
}

// Both in one launch: the keys' workgroups first, which take longer, and the queries' where CUs have room.
template <typename T, int D, bool kCausal, int kKB, int kQB>
__global__ __launch_bounds__(kGradWaves * 64, 2) void packed_grad_kernel(GradArgs g) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int no = (int)blockIdx.x;
  if (no < g.key_groups) grad_keys<T, D, kCausal, kKB>(g, smem, no, g.key_groups);
  else grad_queries<T, D, kCausal, kQB>(g, smem, no - g.key_groups, (int)gridDim.x - g.key_groups);
}

// dK and dV: the sums of the parts' sums.  A thread takes 4 elements.
template <typename T>
__global__ __launch_bounds__(256) void packed_grad_parts_kernel(GradArgs g, int d) {
  using V4 = typename Vec<T>::v4;
  const PackedArgs& a = g.packed;
  const size_t all = (size_t)a.kv_tokens * a.kv_heads * d, at = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= all) return;
  const int row = (int)(at / ((size_t)a.kv_heads * d)), from = read_uniform(a.kv_offsets), to = read_uniform(a.kv_offsets + a.sequences);
  const bool there = row >= from && row < to;   // (rows of no sequence have no parts)
  float4_t dk = {0.f, 0.f, 0.f, 0.f}, dv = dk;
  for (int p = 0; p < (there ? g.parts : 0); ++p) {
    dk += *reinterpret_cast<const float4_t*>(g.partial + 2 * p * all + at);
    dv += *reinterpret_cast<const float4_t*>(g.partial + (2 * p + 1) * all + at);
  }
  constexpr float kDownP = std::is_same_v<T, bf16_t> ? 1.f : 1.f / 32768.f;
  V4 k, v;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    k[e] = (T)(dk[e] * (g.scale * kDownP));
    v[e] = (T)(dv[e] * kDownP);
  }
  *reinterpret_cast<V4*>(static_cast<T*>(g.grad_key) + at) = k;
  *reinterpret_cast<V4*>(static_cast<T*>(g.grad_value) + at) = v;
}

template <typename T, int D, bool kCausal>
int launch_grad(GradArgs g, hipStream_t st) {
  const PackedArgs& a = g.packed;
  const int64_t all = (int64_t)a.tokens * a.heads;
  constexpr int kRows = 256 / (D / 8);
  if (all > 0)
    if (int rc = launch_kernel(packed_stats_kernel<T, D>, dim3((unsigned)((all + kRows - 1) / kRows)), dim3(256), 0, st, g)) return rc;
  const bool of_keys = g.grad_key && a.kv_tokens > 0, of_queries = g.grad_query && a.tokens > 0;
  constexpr int kKB = 2, kQB = 2;
  auto kern = packed_grad_kernel<T, D, kCausal, kKB, kQB>;
  constexpr int lds = grad_lds_bytes<T, D, kCausal>();
  static_assert(2 * lds <= kMaxLdsBytes, "two workgroups do not fit in a CU's LDS");
  TFK_LDS_OPT_IN(kern, lds);
  // (rows of no sequence are cleared by whatever workgroups there are)
  g.key_groups = of_keys ? (int)std::max<int64_t>(most_tiles(a.kv_tokens, a.sequences, kGradKeys) * a.kv_heads * g.parts, 1) : 0;
  const int64_t query_groups = of_queries ? std::max<int64_t>(most_tiles((int64_t)a.tokens * a.group.d, a.sequences, kGradWaves * 16 * kQB) * a.kv_heads, 1) : 0;
  if (g.key_groups + query_groups > 0)
    if (int rc = launch_kernel(kern, dim3((unsigned)(g.key_groups + query_groups)), dim3(kGradWaves * 64), lds, st, g)) return rc;
  if (of_keys && g.parts > 1) {
    const int64_t threads = (int64_t)a.kv_tokens * a.kv_heads * D / 4;
    return launch_kernel(packed_grad_parts_kernel<T>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, g, D);
  }
  return TF_OK;
}
template <int D>
int run_grad(const PackedGradCall& c) {
  const GradArgs g = {c.args, c.query, c.key, c.value, c.out, c.grad_out, c.lse, static_cast<float4_t*>(c.stats), c.grad_query, c.grad_key, c.grad_value,
                      c.scale, c.scale * kLog2E, 0, c.parts, static_cast<float*>(c.partial), (unsigned)(((1ull << 32) + c.args.group.d - 1) / c.args.group.d)};
  if (c.bf16) return c.causal ? launch_grad<bf16_t, D, true>(g, c.stream) : launch_grad<bf16_t, D, false>(g, c.stream);
  return c.causal ? launch_grad<half_t, D, true>(g, c.stream) : launch_grad<half_t, D, false>(g, c.stream);
}

}  // namespace
}  // namespace tfk
