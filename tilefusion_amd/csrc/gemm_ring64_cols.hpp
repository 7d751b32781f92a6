// The main loop of gemm_ring64.hpp for operands that are summed over their ROWS: what the gradients of a product are.  With A [M, K] (rows) or
// [K, M] (columns) and B [K, N], both row-major, a tile of A * B or A^T * B.
//
// An operand whose columns count is kept in LDS as it lies in memory, 64 rows of a tile's width, and transposed on its way to registers: a
// ds_read_b64_tr_b16 hands each lane of a group of 16 one column of a block of 4 rows x 16 columns, two of them are a fragment.  The same bytes leave
// LDS as with rows; what is paid for the transposition is one more read instruction and one addition a fragment, between matrix
// instructions that have room for them.  Without it every operand of a backward pass would be copied transposed first: 28% of the time of the
// gradients of 8192 tokens x 1024 over 131072 words (7.3 ms), 14% of the gated block's of 8192 x 4096 x 11264.
//
// Rows of a tile lie one behind the other (512 bytes for 256 columns: all in the same banks), so blocks of 16 columns, 32 bytes, trade places with an XOR
// by the row: the 8 rows that two groups of lanes read at a time then lie in 8 different eighths of the banks.
#pragma once

#include "gemm_ring64.hpp"

namespace tfk {
namespace {

// x: rows of 16-bit elements, `pitch` (a multiple of 8) apart, from a 16-byte boundary on.
struct ColsOperand {
  const uint16_t* x;
  int64_t pitch;
  int width;             // columns that may be read, a multiple of 8
  int extent;            // rows (A by rows) or columns of the result
};

// Lanes' offsets are counted from that many bytes in front: what an immediate offset takes off may be more than a row has.
constexpr int kColsLead = 4096;
// The farthest of them where `rows` rows of a tile are walked, `pitch` elements apart; it has to stay below 2^32.
__host__ __device__ constexpr uint64_t cols_farthest(int64_t rows, int64_t pitch) { return 2 * (uint64_t)(rows - 1) * (uint64_t)pitch + 512 + kColsLead; }

// The 16-column block that lies in place of block b in row `row` of a tile, and the other way round.
__host__ __device__ constexpr int cols_swizzle(int row) { return (row & 3) | (row >> 3 & 1) << 2; }

// acc += tile (m0, n0) over the k-tiles t0 .. t0 + num - 1 of 64; m0 and n0 are multiples of 8, and what lies behind the operands' extents
// is some of theirs again (not to be stored).  The first k-tile begins k_pad rows in front of B (and of A, kColA;
// otherwise A's rows hold zeros there), which are taken for zeros.  B's rows continue in `b1` from k-tile `turn` on.
// cols_farthest of 64 rows of an operand by columns, and of the tile's rows of A by rows, is below 2^32.
template <typename S, typename InT, bool kColA>
TFK_DEVICE void ring64_multiply_cols(const ColsOperand& a, const ColsOperand& b, const uint16_t* b1, int turn, int m0, int n0, int t0, int num, int k_pad,
                                     int lane, int wave, char* smem, float4_t (&acc)[S::TM][S::TN]) {
  static_assert(S::kLines == 0 && (S::TM == 8 || S::TM == 4) && (S::TN == 8 || S::TN == 4), "blocks of 4 or 8 to a wavefront");
  static_assert(S::free_gaps() >= 8, "a gap for every piece");
  constexpr int kPitchA = S::BM * 2, kPitchB = S::BN * 2;                 // bytes of a row in LDS
  constexpr int kRowsA = 1024 / kPitchA, kRowsB = 1024 / kPitchB;         // rows of a request
  constexpr int kLead = kColsLead;
  const int wm = wave / S::WAVES_N, wn = wave % S::WAVES_N;
  const int fr = lane & 15, fg = lane >> 4;

  // ---- global -> LDS: as in gemm_ring64.hpp, 1 KiB a request ---------------------------------
  const bool padded = k_pad != 0 && t0 == 0;
  const bool only = padded && num == 1;   // requests behind the last k-tile ask for it again: not in front of the operand
  unsigned off_a[S::kLoadsA], off_b[S::kLoadsB];
#pragma unroll
  for (int n = 0; n < S::kLoadsA; ++n) {
    if constexpr (kColA) {
      const int row = (wave * S::kLoadsA + n) * kRowsA + lane / (64 / kRowsA), c = lane % (64 / kRowsA);
      const int chunk = min(((c >> 1) ^ cols_swizzle(row)) * 2 + (c & 1), (a.width - m0) / 8 - 1);
      off_a[n] = (unsigned)(only ? max(row, k_pad) : row) * (unsigned)a.pitch * 2u + 16u * chunk + kLead - 1024u * (n % 4);
    } else {
      const int row = wave * 8 * S::kLoadsA + 8 * n + lane / 8;
      off_a[n] = (unsigned)min(row, a.extent - 1 - m0) * (unsigned)a.pitch * 2u + (unsigned)S::swizzle(row, lane % 8) * 16u + kLead - 1024u * (n % 4);
    }
  }
#pragma unroll
  for (int n = 0; n < S::kLoadsB; ++n) {
    const int row = (wave * S::kLoadsB + n) * kRowsB + lane / (64 / kRowsB), c = lane % (64 / kRowsB);
    const int chunk = min(((c >> 1) ^ cols_swizzle(row)) * 2 + (c & 1), (b.width - n0) / 8 - 1);
    off_b[n] = (unsigned)(only ? max(row, k_pad) : row) * (unsigned)b.pitch * 2u + 16u * chunk + kLead - 1024u * (n % 4);
  }
  // a k-tile's address in front of the lanes' offsets
  const char* const a_tile = reinterpret_cast<const char*>(a.x + (kColA ? m0 - k_pad * a.pitch : m0 * a.pitch)) - kLead;
  const char* const b_tile = reinterpret_cast<const char*>(b.x + n0 - k_pad * b.pitch) - kLead;
  const char* const b1_tile = reinterpret_cast<const char*>(b1 + n0) - kLead;
  const uint64_t a_step = kColA ? 128 * (uint64_t)a.pitch : 128, b_step = 128 * (uint64_t)b.pitch;   // bytes from k-tile to k-tile
  const int last = t0 + num - 1;
  auto a_src = [&](int t) __attribute__((always_inline)) { return a_tile + (uint64_t)(unsigned)min(t, last) * a_step; };
  auto b_src = [&](int t) __attribute__((always_inline)) {
    const int at = min(t, last);
    return at < turn ? b_tile + (uint64_t)(unsigned)at * b_step : b1_tile + (uint64_t)(unsigned)(at - turn) * b_step;
  };
  const unsigned smem_addr = lds_address(smem);
  const unsigned lds_wave_a = smem_addr + wave * S::kLoadsA * 1024, lds_wave_b = smem_addr + wave * S::kLoadsB * 1024;
  auto request = [&](unsigned off, const char* src, unsigned lds_unit, int n) __attribute__((always_inline)) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 offset:%2"
                 :
                 : "v"(off), "s"(src), "n"(1024 * (n % 4)), "{m0}"(lds_unit + (n - n % 4) * 1024)
                 : "memory");
  };

  // ---- LDS -> fragments ----------------------------------------------------------------------
  // By columns: lane r of a group of 16 addresses row r / 4 of a block, columns 4 * (r % 4) ..; block f of the wavefront lies at
  // base[f / 4] + block[f % 4].  By rows: as in gemm_ring64.hpp, a base for each k-step.
  const int row_l = 8 * fg + (fr >> 2), x = cols_swizzle(row_l);
  unsigned block[4];
#pragma unroll
  for (int f = 0; f < 4; ++f) block[f] = (unsigned)((f ^ x) & 3) * 32u;
  auto cols_base = [&](int wave_at, int blocks, int pitch, int half) __attribute__((always_inline)) {
    return (unsigned)(row_l * pitch + (((wave_at * blocks + 4 * half) ^ (x & 4)) * 32) + (fr & 3) * 8);
  };
  unsigned base_a[2], base_b[2];
  if constexpr (kColA) {
    base_a[0] = smem_addr + cols_base(wm, S::TM, kPitchA, 0);
    base_a[1] = smem_addr + cols_base(wm, S::TM, kPitchA, 1);
  } else {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) base_a[ks] = smem_addr + (wm * S::WM + fr) * S::kRowBytes + S::swizzle(fr, 4 * ks + fg) * 16;
  }
  base_b[0] = smem_addr + cols_base(wn, S::TN, kPitchB, 0);
  base_b[1] = smem_addr + cols_base(wn, S::TN, kPitchB, 1);

  half8_t afx[2][S::TM], bf[2][S::TN];
  auto read_cols = [&](const unsigned (&base)[2], int f, int ks, int pitch) __attribute__((always_inline)) {
    typedef __fp16 fp16x4_t __attribute__((ext_vector_type(4)));
    const unsigned at = base[f / 4] + block[f % 4] + ks * 32 * pitch;
    const half4_t lo = __builtin_bit_cast(half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4_t*)(size_t)at));
    const half4_t hi =
        __builtin_bit_cast(half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4_t*)(size_t)(at + 4 * pitch)));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto read_a = [&](const unsigned (&base)[2], int f, int ks) __attribute__((always_inline)) {
    if constexpr (kColA) return read_cols(base, f, ks, kPitchA);
    else return *(__attribute__((address_space(3))) const half8_t*)(size_t)(base[ks] + f * 16 * S::kRowBytes);
  };
  auto read_b = [&](const unsigned (&base)[2], int f, int ks) __attribute__((always_inline)) { return read_cols(base, f, ks, kPitchB); };

#pragma unroll
  for (int i = 0; i < S::TM; ++i)
#pragma unroll
    for (int j = 0; j < S::TN; ++j) acc[i][j] = float4_t{0.f, 0.f, 0.f, 0.f};

  // slot i of k-step ks: its MFMAs, and the reads of the next k-step (of the unit bases rd_a, rd_b) where they have their place
  auto slot = [&](int ks, int i, const unsigned (&rd_a)[2], const unsigned (&rd_b)[2], auto&& between) __attribute__((always_inline)) {
    const int first = S::reads_first(i), n_reads = S::reads_in(i);
    int done = 0;
#pragma unroll
    for (int j = 0; j < S::TN; ++j) {
      if constexpr (std::is_same_v<InT, bf16_t>)
        asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc[i][j]) : "v"(bf[ks][j]), "v"(afx[ks][i]));
      else
        asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(acc[i][j]) : "v"(bf[ks][j]), "v"(afx[ks][i]));
      if (done < n_reads && j == (done * S::TN) / n_reads + 1) {
        const int q = first + done;
        __builtin_amdgcn_sched_barrier(0);
        if (q < S::TN) bf[ks ^ 1][q] = read_b(rd_b, q, ks ^ 1);
        else afx[ks ^ 1][q - S::TN] = read_a(rd_a, q - S::TN, ks ^ 1);
        __builtin_amdgcn_sched_barrier(0);
        ++done;
      } else {
        between(S::kPrep.piece[i * S::TN + j]);
      }
    }
  };
  auto ring_barrier = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt((S::kInFlight & 15) | 0x70 | ((S::kInFlight >> 4) << 14));   // vmcnt(kInFlight) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  // prologue: k-tiles 0 .. kAhead-1, rows in front of the sum from a block of zeros
#pragma unroll
  for (int u = 0; u < 2 * S::kAhead; ++u) {
    const bool of_b = u % 2;
    const char* const src = of_b ? b_src(t0 + u / 2) : a_src(t0 + u / 2);
    const unsigned unit = (of_b ? lds_wave_b : lds_wave_a) + u * S::kUnitBytes;
#pragma unroll
    for (int n = 0; n < (of_b ? S::kLoadsB : S::kLoadsA); ++n) {
      const unsigned off = of_b ? off_b[n] : off_a[n];
      if (u < 2 && (kColA || of_b) && padded) {
        const int rows = of_b ? kRowsB : kRowsA;
        const int row = (wave * (of_b ? S::kLoadsB : S::kLoadsA) + n) * rows + lane / (64 / rows);
        lds_dma_16B(row < k_pad ? reinterpret_cast<const char*>(kZeros) : src + (off + 1024u * (n % 4)), unit + n * 1024);
      } else {
        request(off, src, unit, n);
      }
    }
  }
  wait_vmem<(S::kAhead - 1) * (S::kLoadsA + S::kLoadsB)>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  unsigned rd_a[2] = {base_a[0], base_a[1]}, rd_b[2] = {base_b[0] + S::kUnitBytes, base_b[1] + S::kUnitBytes};   // of k-tile t
#pragma unroll
  for (int f = 0; f < S::TN; ++f) bf[0][f] = read_b(rd_b, f, 0);
#pragma unroll
  for (int i = 0; i < S::TM; ++i) afx[0][i] = read_a(rd_a, i, 0);
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
  __builtin_amdgcn_sched_barrier(0);

  constexpr unsigned kRingBytes = S::kUnits * S::kUnitBytes;
  auto ring = [](unsigned o) __attribute__((always_inline)) { return o >= kRingBytes ? o - kRingBytes : o; };
  unsigned oa = 0, oa1 = 0, ob1 = 0;                               // A of k-tile t; A, B of t+1
  unsigned next_a[2], next_b[2];                                   // rd_a, rd_b of k-tile t+1
  unsigned req_a = lds_wave_a + 2 * S::kAhead * S::kUnitBytes, req_b = 0;
  const char *src_a = a_src(t0 + S::kAhead), *src_b = nullptr, *from = nullptr;
  int kt = 0;
#define TFK_PIN_S(x) asm volatile("" : "+s"(x))
#define TFK_PIN_V(x) asm volatile("" : "+v"(x))
  // bookkeeping of k-step 0: where k-tile t+1 is read, B of t+kAhead is requested (into the unit of A of t)
  auto prep0 = [&](int piece, int t) __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    switch (piece) {
      case 0: TFK_PIN_S(oa); oa1 = ring(oa + 2 * S::kUnitBytes); TFK_PIN_S(oa1); break;
      case 1: ob1 = ring(oa1 + S::kUnitBytes); TFK_PIN_S(ob1); break;
      case 2: next_a[0] = base_a[0] + oa1; TFK_PIN_V(next_a[0]); next_a[1] = base_a[1] + oa1; TFK_PIN_V(next_a[1]); break;
      case 3: next_b[0] = base_b[0] + ob1; TFK_PIN_V(next_b[0]); next_b[1] = base_b[1] + ob1; TFK_PIN_V(next_b[1]); break;
      case 4: req_b = lds_wave_b + oa; TFK_PIN_S(req_b); break;
      case 5: kt = t; TFK_PIN_S(kt); kt = min(kt + S::kAhead, last); TFK_PIN_S(kt); break;
      case 6:
        from = kt < turn ? b_tile : b1_tile;
        TFK_PIN_S(from);
        if (kt >= turn) kt -= turn;
        TFK_PIN_S(kt);
        break;
      case 7: src_b = from + (uint64_t)(unsigned)kt * b_step; TFK_PIN_S(src_b); break;
      default: break;
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // of k-step 1: A of t+kAhead+1 (into the unit behind the ring's last)
  auto prep1 = [&](int piece, int t) __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    switch (piece) {
      case 0: oa = oa1; TFK_PIN_S(oa); break;
      case 1: rd_a[0] = next_a[0]; TFK_PIN_V(rd_a[0]); rd_a[1] = next_a[1]; TFK_PIN_V(rd_a[1]); break;
      case 2: rd_b[0] = next_b[0]; TFK_PIN_V(rd_b[0]); rd_b[1] = next_b[1]; TFK_PIN_V(rd_b[1]); break;
      case 3: req_a = ring(oa + 2 * S::kAhead * S::kUnitBytes); TFK_PIN_S(req_a); break;
      case 4: req_a += lds_wave_a; TFK_PIN_S(req_a); break;
      case 5: kt = t; TFK_PIN_S(kt); kt = min(kt + S::kAhead + 1, last); TFK_PIN_S(kt); break;
      case 6: src_a = a_tile + (uint64_t)(unsigned)kt * a_step; TFK_PIN_S(src_a); break;
      default: break;
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  for (int t = t0; t <= last; ++t) {
#pragma unroll
    for (int i = 0; i < S::TM; ++i) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < S::kLoadsA; ++n)
        if ((n * S::TM) / S::kLoadsA == i) request(off_a[n], src_a, req_a, n);
      slot(0, i, rd_a, rd_b, [&](int piece) __attribute__((always_inline)) { prep0(piece, t); });
    }
    __builtin_amdgcn_sched_barrier(0);
    ring_barrier();
#pragma unroll
    for (int i = 0; i < S::TM; ++i) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < S::kLoadsB; ++n)
        if ((n * S::TM) / S::kLoadsB == i) request(off_b[n], src_b, req_b, n);
      slot(1, i, next_a, next_b, [&](int piece) __attribute__((always_inline)) { prep1(piece, t); });
    }
    // (the wait states behind the last MFMAs, as in gemm_ring64.hpp)
    int t_seen = t;
    asm volatile("" : "+s"(t_seen));
    if (t_seen == last) asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
  }
#undef TFK_PIN_S
#undef TFK_PIN_V
  __builtin_amdgcn_sched_barrier(0);
  wait_vmem_all();   // the requests behind the last k-tile must not outlive the workgroup's LDS
}

}  // namespace
}  // namespace tfk
