// The main loop of the large matrix products: tiles of A * B^T of 128 x 128 to 256 x 256, both operands in rows that are contiguous in K.
// gemm.hip stores them as they are; the kernels of product.hpp do more with them.
#pragma once

#include <type_traits>

#include "common.hpp"

namespace tfk {
namespace {

// Workgroup ids are dealt round-robin to the 8 XCDs, so ids that are equal mod 8 share an L2.  This
// gives each XCD a run of consecutive positions out of 0 .. nblocks-1.
TFK_DEVICE int xcd_major(int bid, int nblocks) {
  const int xcd = bid & 7;
  return xcd * (nblocks >> 3) + min(xcd, nblocks & 7) + (bid >> 3);
}
// XCD-aware tile order: a grouped (4 tile-rows at a time) walk of the output, so that the workgroups
// of an XCD re-use A and B panels.
TFK_DEVICE void tile_of_block(int bid, int nblocks, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int pid = xcd_major(bid, nblocks);
  constexpr int kGroup = 4;
  const int group_size = kGroup * tiles_n;
  const int gid = pid / group_size;
  const int first_m = gid * kGroup;
  const int rows = min(tiles_m - first_m, kGroup);
  const int in_group = pid - gid * group_size;
  tm = first_m + in_group % rows;
  tn = in_group / rows;
}

// ------------------------------------------------------------------------------------------
// 256 x 256 x 64 path: same 2 x 2 wavefronts of 128 x 128, but k-tiles of 64 so that every
// global->LDS instruction fetches whole 128-byte lines (8 rows x 128 bytes).  The vector L1
// moves full lines, so the 64-byte row segments of a 32-deep tile spend half of the L2->L1
// bandwidth on bytes that are dropped and requested again one k-tile later.
//
// A 64-deep tile is 64 KiB and only 160 KiB of LDS exist, so the ring is kept in UNITS of one
// operand of one tile (32 KiB, five of them): unit u lives in ring slot u % 5, A of tile t is
// unit 2t and B of tile t unit 2t+1.  Iteration t:
//   k-step 0: multiplies fragments (t, 0), reads fragments (t, 1), requests A of tile t+2 into
//             the slot B of tile t-1 left;
//   barrier:  tile t is read out (both its units are free) and tile t+1 has landed
//             (vmcnt leaves only the 8 requests of k-step 0 outstanding);
//   k-step 1: multiplies (t, 1), reads fragments (t+1, 0), requests B of tile t+2 into the
//             slot A of tile t left.
// Every request has at least 8 MFMA slots (1024 MFMA cycles) to land.
// ------------------------------------------------------------------------------------------
//
// The same kernel serves smaller tiles (2 x 2 wavefronts of half a tile each way), for grids that 256 x 256
// tiles would leave CUs idle on: 3333 x 2288 x 1944 takes 45.5 us with 126 tiles of 256 x 256, 36.7 with
// 216 of 192 x 192 and 36.4 with 252 of 256 x 128; 2999 x 1544 x 1032 27.6 and, with 192 x 128, 18.7 (the bounds-checked kernel that ran
// these shapes before: 37.8; whole lines, below, 17.3, and with 160 x 128 16.6).  Units then have the size of the larger operand.  128 x 128 tiles have k-steps
// four times shorter; where a workgroup has its CU to itself their requests run kAhead = 4 tiles
// ahead (a ring of 2 * kAhead + 1 = 9 units).
//
// K that is no multiple of 64 (kLines): rows start anywhere in a 128-byte line, and k-tiles that start where a row starts
// would fetch every line twice, for two tiles (8 rows x 128 bytes are 16 lines instead of 8: 0.13 to 0.27 us more a k-tile).
// So what is fetched are SEGMENTS of whole lines: segment u of a row is its u-th line, and in it k-tile t of the row takes
// the end of segment t and the front of segment t + 1, by an amount that only depends on the row. Rows 8 apart start at
// the same place in a line, so a lane's fragments all are shifted alike, and what a lane pays is the choice between
// the two segments (one v_and and one v_add3 an address). The ring is kept in whole tiles then, kLines of them: two are
// read, the others in flight. 2999 x 1544 x 1032 18.7 -> 17.3 us (K = 1024: 14.7).
template <int BM_, int BN_, int AHEAD_, int LINES_ = 0>
struct Ring64Shape {
  static constexpr int BM = BM_, BN = BN_, BK = 64;
  static constexpr int WAVES_M = 2, WAVES_N = 2;
  static constexpr int kWaves = WAVES_M * WAVES_N, kThreads = kWaves * kWaveSize;
  static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N;
  static constexpr int TM = WM / 16, TN = WN / 16;          // 16x16 MFMA tiles per wavefront
  static constexpr int kRowBytes = BK * 2;                  // 128
  static constexpr int kUnitBytes = (BM > BN ? BM : BN) * kRowBytes;   // one operand of one tile
  static constexpr int kAhead = AHEAD_;                     // tiles between a request and its use
  static constexpr int kUnits = 2 * kAhead + 1;
  static constexpr int kLoadsA = BM / 8 / kWaves, kLoadsB = BN / 8 / kWaves;   // 1 KiB requests per wavefront and unit
  static constexpr int kLoadsMax = kLoadsA > kLoadsB ? kLoadsA : kLoadsB;
  static constexpr int kLoads = kLoadsA + kLoadsB;
  static constexpr int kLines = LINES_;                     // segments in the ring, 0: k-tiles start where rows start
  static constexpr int kTileBytes = (BM + BN) * kRowBytes;
  static constexpr int kLdsBytes = kLines ? kLines * kTileBytes : kUnits * kUnitBytes;
  // slot schedule of a k-step (TM slots of TN MFMAs): the TM + TN fragment reads of the next
  // k-step are dealt to the first kReadSlots slots; the scalar bookkeeping runs in the gaps
  // without a read from slot kPrepSlot on
  static constexpr int kReads = TM + TN;
  static constexpr int kReadSlots = TM == 8 ? 6 : TM - 1;
  static constexpr int kPrepSlot = TM == 8 ? 6 : 0;
  static constexpr int reads_first(int i) { return i < kReadSlots ? (i * kReads) / kReadSlots : kReads; }
  static constexpr int reads_in(int i) { return reads_first(i + 1) - reads_first(i); }
  // read number d of a slot follows MFMA (d * TN) / n of that slot (gap j = that + 1)
  static constexpr bool gap_has_read(int i, int j) {
    const int n = reads_in(i);
    for (int d = 0; d < n; ++d)
      if (j == (d * TN) / n + 1) return true;
    return false;
  }
  // which bookkeeping piece runs in gap j of slot i (-1: none); a table, so that the unrolled
  // slots index it with constants
  struct PrepTable {
    int piece[TM * TN];
  };
  static constexpr PrepTable make_prep_table() {
    PrepTable t{};
    int rank = 0;
    for (int i = 0; i < TM; ++i)
      for (int j = 0; j < TN; ++j) t.piece[i * TN + j] = (i < kPrepSlot || gap_has_read(i, j)) ? -1 : rank++;
    return t;
  }
  static constexpr PrepTable kPrep = make_prep_table();
  static constexpr int free_gaps() { return kPrep.piece[TM * TN - 1] + 1; }
  static constexpr bool reads_fit() {
    for (int i = 0; i < TM; ++i) {
      if (reads_in(i) > TN - 1) return false;
      for (int d = 1; d < reads_in(i); ++d)   // two reads never share a gap
        if ((d * TN) / reads_in(i) == ((d - 1) * TN) / reads_in(i)) return false;
    }
    return true;
  }
  static_assert(BM % 32 == 0 && BN % 64 == 0, "whole MFMA tile pairs; an even request count of B (see the swizzle of g_off)");
  static constexpr bool kOwnOffsetsB = kLines > 0 || kLoadsA % 2 != 0;   // requests of B do not lie as those of A
  static_assert(reads_fit() && free_gaps() >= 7,
                "slot schedule: every read and bookkeeping piece needs its own gap");
  // requests in flight behind the barrier in the middle of a tile: A of tile t+kAhead, all of the
  // tiles t+2 .. t+kAhead-1
  // (kLines: the segments t+3 .. t+kLines-1)
  static constexpr int kInFlight = kLines ? (kLines - 3) * kLoads : kLoadsA + (kAhead - 2) * kLoads;
  static_assert((kAhead - 1) * kLoads < 64 && (kLines - 2) * kLoads < 64, "vmcnt is a 6-bit counter");
  static_assert(kLines == 0 || (kLines >= 3 && free_gaps() >= 8), "two segments are read, one is in flight; a gap for every piece");
  // 128-byte rows: two rows per pass over the banks; chunk ^ (row / 2) % 8 keeps every
  // ds_read_b128 lane pass on 16 different bank groups
  __host__ __device__ static constexpr int swizzle(int row, int c) { return c ^ ((row / 2) % 8); }
};

__device__ const uint4_t kZeros[1] = {};   // what the chunks in front of a row are fetched from

// acc = the tile of A * B^T whose first row and column are m0 and n0, by the whole workgroup; the requests are done and LDS is free behind a
// barrier.  M >= m0 + BM, N >= n0 + BN, and K >= BK (kLines: K > 64 * kLines): requests past the last k-tile ask for that tile again, which
// must not be the one completed with zeros.
// InT is half_t, bf16_t or int8_t: they differ in the MFMA mnemonic, everything else moves 16 bits at a time without looking at them.
// K counts these: half the elements of 8 bits.  int8_t: the accumulators are int32.
// kTwo: the tile's columns alternate between rows of B and of B1 in blocks of 16, from row n0 of either on, BN / 2 of each.
// kFew: A has only `rows` < BM rows (m0 = 0); what lies behind them in the tile is the last one again.
template <typename S, typename InT, bool kTwo = false, bool kFew = false>
TFK_DEVICE void ring64_multiply(const uint16_t* A, const uint16_t* B, const uint16_t* B1, int K, int m0, int n0, int lane, int wave, char* smem,
                                float4_t (&acc)[S::TM][S::TN], int rows = 0) {
  const int wm = wave / S::WAVES_N, wn = wave % S::WAVES_N;
  // global -> LDS plan: request n of a wavefront covers rows (wave * kLoads + n) * 8 .. +7 of a
  // unit (consecutive 1 KiB blocks of LDS, so four requests share one M0 base and differ in the
  // instruction's immediate offset); lane l fills physical chunk l % 8 of row l / 8 and fetches the logical chunk the
  // swizzle maps there.  A and B share the per-lane offsets (same row stride K); the address
  // is a scalar base (tile origin + k offset) plus this 32-bit per-lane offset, so a request
  // needs no vector arithmetic.
  const int ld_row = lane / 8, ld_c = lane % 8;
  // K is completed to whole k-tiles at its FRONT: k-tile t starts at element 64 * t - k_pad of a row, and
  // the chunks of tile 0 that lie in front of the row are fetched from a block of zeros.  Only the
  // prologue knows about it.
  const int num_k_tiles = (K + S::BK - 1) / S::BK;
  const int k_pad = num_k_tiles * S::BK - K;
  // kLines: chunk c of row r, counted from the completed front, is chunk (c + shift(r)) % 8 of segment (c + shift(r)) / 8,
  // shift(r) = 1 .. 8. In LDS it lies where it would without a shift, so that reads see the same banks.
  constexpr bool kShift = S::kLines > 0;
  constexpr int kLead = kShift ? 256 : 0;   // (keeps lane offsets positive: up to 15 chunks in front of a row)
  const int pad_chunks = k_pad / 8;
  auto shift_of = [&](const uint16_t* X, int row) __attribute__((always_inline)) {
    const unsigned in_line = (unsigned)(reinterpret_cast<uintptr_t>(X) >> 4) + (unsigned)row * (unsigned)(K / 8);
    return (int)((in_line - (unsigned)pad_chunks - 1u) & 7u) + 1;
  };
  const int a_shift = shift_of(A, m0 + ld_row), b_shift = shift_of(B, n0 + ld_row);   // of the rows that this lane fetches
  // (kTwo, kFew: offsets are counted from kLeadFar bytes in front: what an immediate offset takes off may be more than a row has)
  constexpr int kLeadFar = 4096;
  const char* a_tile = kFew ? reinterpret_cast<const char*>(A) - 2 * k_pad - kLeadFar
                            : reinterpret_cast<const char*>(A + (size_t)(m0 + wave * 8 * S::kLoadsA) * K) - (kShift ? kLead : 2 * k_pad);
  // kTwo: block 2 * j of 16 rows of the unit are rows of B, block 2 * j + 1 the same rows of B1; a request's 8 rows are of one
  // of them.
  const char* b_tile = kTwo ? reinterpret_cast<const char*>(B + (size_t)(n0 + wave * 4 * S::kLoadsB) * K) - 2 * k_pad - kLeadFar
                            : reinterpret_cast<const char*>(B + (size_t)(n0 + wave * 8 * S::kLoadsB) * K) - (kShift ? kLead : 2 * k_pad);
  const char* b1_tile = kTwo ? reinterpret_cast<const char*>(B1 + (size_t)(n0 + wave * 4 * S::kLoadsB) * K) - 2 * k_pad - kLeadFar : nullptr;
  unsigned g_off[S::kLoadsMax];
  constexpr bool kOwnOffsetsB = S::kOwnOffsetsB || kTwo || kFew;
  unsigned g_off_b[kOwnOffsetsB ? S::kLoadsB : 1];
  // (an odd number of requests: every other wavefront's rows begin in the middle of the swizzle's sixteen)
  const int a_odd = S::kLoadsA % 2 ? wave & 1 : 0;
  // the chunk of a segment that this lane fetches with request n
  auto segment_chunk = [&](int n, int shift) __attribute__((always_inline)) { return (S::swizzle(ld_row + 8 * n, ld_c) + shift) & 7; };
  auto segment_off = [&](int n, int odd, int shift) __attribute__((always_inline)) {
    return (unsigned)(ld_row + 8 * n) * (unsigned)K * 2u + (unsigned)(kLead + 16 * (segment_chunk(n + odd, shift) - shift - pad_chunks)) -
           1024u * (n % 4);
  };
  auto tile_off = [&](int n, int odd) __attribute__((always_inline)) {
    return (unsigned)(ld_row + 8 * n) * (unsigned)K * 2u + (unsigned)S::swizzle(ld_row + 8 * (n + odd), ld_c) * 16u -
           1024u * (n % 4);   // the instruction's immediate offset (added to both addresses) gives it back
  };
#pragma unroll
  for (int n = 0; n < S::kLoadsMax; ++n)
    g_off[n] = kShift ? segment_off(n, a_odd, a_shift)
                      : tile_off(n, a_odd);
  if constexpr (kFew) {
    static_assert(S::kLines == 0 && S::kLoadsA % 2 == 0, "");
#pragma unroll
    for (int n = 0; n < S::kLoadsA; ++n)
      g_off[n] = (unsigned)min(wave * 8 * S::kLoadsA + ld_row + 8 * n, rows - 1) * (unsigned)K * 2u + (unsigned)S::swizzle(ld_row + 8 * n, ld_c) * 16u +
                 kLeadFar - 1024u * (n % 4);
  }
  if constexpr (kTwo) {
    static_assert(S::kLines == 0 && S::kLoadsB % 4 == 0, "a wavefront's requests begin with a block of B");
#pragma unroll
    for (int n = 0; n < S::kLoadsB; ++n)
      g_off_b[n] = (unsigned)(ld_row + n / 4 * 16 + n % 2 * 8) * (unsigned)K * 2u + (unsigned)S::swizzle(ld_row + 8 * n, ld_c) * 16u + kLeadFar -
                   1024u * (n % 4);
  } else if constexpr (kOwnOffsetsB) {
#pragma unroll
    for (int n = 0; n < S::kLoadsB; ++n) g_off_b[n] = kShift ? segment_off(n, 0, b_shift) : tile_off(n, 0);
  }
  // LDS -> fragment plan: fragment i of k-step ks: row 16*i + l%16 of the wavefront's rows,
  // logical chunk 4*ks + l/16
  const int fr = lane & 15, fg = lane >> 4;
  unsigned a_rd[2], b_rd[2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    a_rd[ks] = (wm * S::WM + fr) * S::kRowBytes + S::swizzle(fr, 4 * ks + fg) * 16;
    b_rd[ks] = (wn * S::WN + fr) * S::kRowBytes + S::swizzle(fr, 4 * ks + fg) * 16;
  }

#pragma unroll
  for (int i = 0; i < S::TM; ++i)
#pragma unroll
    for (int j = 0; j < S::TN; ++j) acc[i][j] = float4_t{0.f, 0.f, 0.f, 0.f};

  const unsigned smem_addr = lds_address(smem);
  // Slot i of a k-step multiplies A fragment i with all B fragments; both operands have two
  // register sets (this k-step's and the next one's).
  half8_t afx[2][S::TM], bf[2][S::TN];
  // The requests are issued from inline assembly: the compiler then keeps exact counts for the
  // fragment reads (a direct-to-LDS load it knows about makes every LDS wait a full drain),
  // and the vector-memory waits are placed by hand below.
  // src: tile origin + k offset (scalar); lds_unit: LDS byte address of this wavefront's first
  // 1 KiB block in the destination unit.
  // M0 - the LDS destination of requests n .. n+3 (n % 4 == 0), which differ in the immediate
  // offset - is an INPUT of every request statement: the compiler writes it (once per group of
  // four: the statements do not change it) and cannot use the register for anything else between
  // that write and a request.  The s_nop is the wait state an M0 write needs in front of an
  // LDS-direct load; next to a request at the head of a slot it costs no issue time.
  auto request_at = [&](unsigned off, const char* src, unsigned lds_unit, int n) __attribute__((always_inline)) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 offset:%2"
                 :
                 : "v"(off), "s"(src), "n"(1024 * (n % 4)), "{m0}"(lds_unit + (n - n % 4) * 1024)
                 : "memory");
  };
  auto request = [&](const char* src, unsigned lds_unit, int n, auto of_b) __attribute__((always_inline)) {
    if constexpr (kOwnOffsetsB && decltype(of_b)::value) request_at(g_off_b[n], src, lds_unit, n);
    else request_at(g_off[n], src, lds_unit, n);
  };
  auto k_src = [&](const char* tile, int t) __attribute__((always_inline)) {
    return tile + (size_t)min(t, num_k_tiles - 1) * S::BK * 2;   // clamped past the end
  };
  const unsigned lds_wave_a = smem_addr + wave * S::kLoadsA * 1024, lds_wave_b = smem_addr + wave * S::kLoadsB * 1024;
  // Slot with the MFMAs issued from inline assembly, accumulators pinned to AGPRs, and the
  // slot's fragment reads placed by hand between them.  (With compiler-issued MFMAs the
  // register allocator, at exactly 256 live accumulators, shuffles accumulators through VGPRs
  // whenever the schedule changes slightly.)
  auto lds_read_b128 = [](unsigned addr) __attribute__((always_inline)) {
    return *(__attribute__((address_space(3))) const half8_t*)(size_t)addr;
  };
  // rd_a / rd_b: this lane's LDS byte address of fragment 0 of the next k-step's A / B operand
  // (unit base + row + swizzled chunk); fragment f is f * 2 KiB further, in the offset field.
  auto slot_pinned = [&](int buf, int i, unsigned rd_a, unsigned rd_b, auto&& between) __attribute__((always_inline)) {
    // The TN + TM fragment reads of the next k-step, B fragments first, are dealt to the first
    // kReadSlots slots; the last slot(s) read nothing, so the drain in front of the barrier
    // (and the one at the head of the next k-step) finds the reads already returned.
    const int first = S::reads_first(i);
    const int n_reads = S::reads_in(i);
    int done = 0;
#pragma unroll
    for (int j = 0; j < S::TN; ++j) {
      if constexpr (std::is_same_v<InT, int8_t>)
        asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(acc[i][j]) : "v"(bf[buf][j]), "v"(afx[buf][i]));
      else if constexpr (std::is_same_v<InT, bf16_t>)
        asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc[i][j]) : "v"(bf[buf][j]), "v"(afx[buf][i]));
      else
        asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(acc[i][j]) : "v"(bf[buf][j]), "v"(afx[buf][i]));
      // after MFMA j: issue the next read if j is its position (reads spread evenly over the slot)
      if (done < n_reads && j == (done * S::TN) / n_reads + 1) {
        const int q = first + done;
        __builtin_amdgcn_sched_barrier(0);
        if (q < S::TN) bf[buf ^ 1][q] = lds_read_b128(rd_b + q * 16 * S::kRowBytes);
        else afx[buf ^ 1][q - S::TN] = lds_read_b128(rd_a + (q - S::TN) * 16 * S::kRowBytes);
        __builtin_amdgcn_sched_barrier(0);
        ++done;
      } else {
        between(j);   // a piece of scalar bookkeeping, if this gap has one
      }
    }
  };
  // Workgroup barrier in the middle of tile t: tile t+1 must have landed, the requests of
  // tiles t+2 .. t+kAhead-1 and of this tile's k-step 0 stay in flight.  The LDS wait and the
  // barrier are builtins so that the compiler knows every earlier fragment read has returned.
  constexpr int kInFlight = S::kInFlight;
  auto ring_barrier = [&]() __attribute__((always_inline)) {
    // one s_waitcnt: vmcnt(kInFlight) lgkmcnt(0); a builtin, so the compiler knows the LDS part
    __builtin_amdgcn_s_waitcnt((kInFlight & 15) | 0x70 | ((kInFlight >> 4) << 14));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // the requests of a k-step sit at the heads of its slots, evenly spread
  auto request_slot = [&](int i, const char* src, const char* src1, unsigned lds_unit, auto loads_c, auto of_b) __attribute__((always_inline)) {
    constexpr int kLoads = decltype(loads_c)::value;
#pragma unroll
    for (int n = 0; n < kLoads; ++n)
      if ((n * S::TM) / kLoads == i) request(kTwo && decltype(of_b)::value && n / 2 % 2 ? src1 : src, lds_unit, n, of_b);
  };
  constexpr std::integral_constant<int, S::kLoadsA> kOfA{};
  constexpr std::integral_constant<int, S::kLoadsB> kOfB{};

  // The compiler does not know that the accumulators are written by MFMAs (they are issued
  // from assembly), so nothing would keep it from reading the youngest results right behind
  // the loop without the wait states the matrix pipe needs.  The delay therefore sits inside
  // the last iteration, in front of anything the register allocator may put on the exit
  // edge.  The iteration count is laundered through an empty asm so that the test is not
  // recognised as the exit condition and sunk out of the loop.
  auto settle_behind_last = [&](int t) __attribute__((always_inline)) {
    int t_seen = t;
    asm volatile("" : "+s"(t_seen));
    if (t_seen + 1 == num_k_tiles) asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
  };
#define TFK_PIN_S(x) asm volatile("" : "+s"(x))
#define TFK_PIN_V(x) asm volatile("" : "+v"(x))
  if constexpr (kShift) {
    // prologue: segments 0 .. kLines-1; the chunks in front of a row, in segments 0 and 1, are zeros
#pragma unroll
    for (int u = 0; u < S::kLines; ++u)
#pragma unroll
      for (int q = 0; q < S::kLoads; ++q) {
        const bool of_a = q < S::kLoadsA;
        const int n = of_a ? q : q - S::kLoadsA;
        const int shift = of_a ? a_shift : b_shift;
        const unsigned off = of_a ? g_off[n] : g_off_b[n];
        const char* tile = (of_a ? a_tile : b_tile) + u * (S::BK * 2);
        const unsigned unit = (of_a ? lds_wave_a : lds_wave_b + S::BM * S::kRowBytes) + u * S::kTileBytes;
        if (u < 2) {
          const bool in_front = 8 * u + segment_chunk(of_a ? n + a_odd : n, shift) - shift < pad_chunks;
          lds_dma_16B(in_front ? reinterpret_cast<const char*>(kZeros) : tile + (off + 1024u * (n % 4)), unit + n * 1024);
        } else {
          request_at(off, tile, unit, n);
        }
      }
    // all ones where this lane's chunk of a k-step lies in the second of the two segments
    int a_next[2], b_next[2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      a_next[ks] = 4 * ks + fg + shift_of(A, m0 + fr) >= 8 ? -1 : 0;
      b_next[ks] = 4 * ks + fg + shift_of(B, n0 + fr) >= 8 ? -1 : 0;
    }
    constexpr unsigned kRingBytes = S::kLines * S::kTileBytes;
    auto ring = [](unsigned o) __attribute__((always_inline)) { return o >= kRingBytes ? o - kRingBytes : o; };
    const unsigned rdbase_a0 = smem_addr + a_rd[0], rdbase_a1 = smem_addr + a_rd[1];
    const unsigned rdbase_b0 = smem_addr + S::BM * S::kRowBytes + b_rd[0], rdbase_b1 = smem_addr + S::BM * S::kRowBytes + b_rd[1];
    const unsigned lds_b = lds_wave_b + S::BM * S::kRowBytes;
    wait_vmem<(S::kLines - 2) * S::kLoads>();   // segments 0 and 1 have landed
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    unsigned rd_a0 = rdbase_a0 + (a_next[0] & S::kTileBytes), rd_b0 = rdbase_b0 + (b_next[0] & S::kTileBytes);
#pragma unroll
    for (int f = 0; f < S::TN; ++f) bf[0][f] = lds_read_b128(rd_b0 + f * 16 * S::kRowBytes);
#pragma unroll
    for (int i = 0; i < S::TM; ++i) afx[0][i] = lds_read_b128(rd_a0 + i * 16 * S::kRowBytes);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_sched_barrier(0);
    unsigned s0 = 0, s1 = S::kTileBytes, s2 = 0;   // segments t, t+1 and t+2 in the ring
    unsigned step = S::kTileBytes;                 // from a segment to the next one's
    unsigned rd_a1 = rdbase_a1 + (a_next[1] & S::kTileBytes), rd_b1 = rdbase_b1 + (b_next[1] & S::kTileBytes);
    unsigned req_a = 0, req_b = 0;
    const char *src_a = a_tile, *src_b = b_tile;
    int kt = 0;
    // during k-step 0: where the fragments of (t+1, 0) are, and segment t+kLines, which takes the place of segment t in k-step 1
    auto prep0 = [&](int piece, int t) __attribute__((always_inline)) {
      __builtin_amdgcn_sched_barrier(0);
      switch (piece) {
        case 0: s1 = ring(s0 + S::kTileBytes); TFK_PIN_S(s1); break;
        case 1: s2 = ring(s1 + S::kTileBytes); TFK_PIN_S(s2); break;
        case 2: step = s2 - s1; TFK_PIN_S(step); rd_a0 = rdbase_a0 + s1 + (a_next[0] & step); TFK_PIN_V(rd_a0); break;
        case 3: rd_b0 = rdbase_b0 + s1 + (b_next[0] & step); TFK_PIN_V(rd_b0); break;
        case 4: req_a = lds_wave_a + s0; TFK_PIN_S(req_a); req_b = lds_b + s0; TFK_PIN_S(req_b); break;
        case 5: kt = t; TFK_PIN_S(kt); kt = min(kt + S::kLines, num_k_tiles); TFK_PIN_S(kt); break;
        case 6: src_a = a_tile + (size_t)(unsigned)(kt * (S::BK * 2)); TFK_PIN_S(src_a); break;
        case 7: src_b = b_tile + (size_t)(unsigned)(kt * (S::BK * 2)); TFK_PIN_S(src_b); break;
        default: break;
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    auto prep1 = [&](int piece) __attribute__((always_inline)) {
      __builtin_amdgcn_sched_barrier(0);
      switch (piece) {
        case 0: rd_a1 = rdbase_a1 + s1 + (a_next[1] & step); TFK_PIN_V(rd_a1); break;
        case 1: rd_b1 = rdbase_b1 + s1 + (b_next[1] & step); TFK_PIN_V(rd_b1); break;
        case 2: s0 = s1; TFK_PIN_S(s0); break;
        default: break;
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    for (int t = 0; t < num_k_tiles; ++t) {
      // The last segment ends behind the row: what lies there is never read, and not fetched either (the row's last chunk is,
      // again). Requests from here on ask for no other segment.
      if (t + S::kLines == num_k_tiles) {
#pragma unroll
        for (int n = 0; n < S::kLoadsA; ++n) g_off[n] -= 16u * (unsigned)max(0, segment_chunk(n + a_odd, a_shift) - (a_shift - 1));
#pragma unroll
        for (int n = 0; n < S::kLoadsB; ++n) g_off_b[n] -= 16u * (unsigned)max(0, segment_chunk(n, b_shift) - (b_shift - 1));
      }
#pragma unroll
      for (int i = 0; i < S::TM; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        slot_pinned(0, i, rd_a1, rd_b1, [&](int j) __attribute__((always_inline)) { prep0(S::kPrep.piece[i * S::TN + j], t); });
      }
      __builtin_amdgcn_sched_barrier(0);
      ring_barrier();   // segment t is read out, segment t+2 has landed
#pragma unroll
      for (int i = 0; i < S::TM; ++i) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < S::kLoads; ++q)
          if ((q * S::TM) / S::kLoads == i) {
            if (q < S::kLoadsA) request_at(g_off[q], src_a, req_a, q);
            else request_at(g_off_b[q - S::kLoadsA], src_b, req_b, q - S::kLoadsA);
          }
        slot_pinned(1, i, rd_a0, rd_b0, [&](int j) __attribute__((always_inline)) { prep1(S::kPrep.piece[i * S::TN + j]); });
      }
      settle_behind_last(t);
    }
  } else {
    // prologue: tiles 0 .. kAhead-1 into the first 2 * kAhead units; fragments (0, 0) once
    // tile 0 is there
#pragma unroll
    for (int u = 0; u < 2 * S::kAhead; ++u)
#pragma unroll
      for (int n = 0; n < (u % 2 ? S::kLoadsB : S::kLoadsA); ++n) {
        const char* tile = u % 2 ? (kTwo && n / 2 % 2 ? b1_tile : b_tile) : a_tile;
        const unsigned unit = (u % 2 ? lds_wave_b : lds_wave_a) + u * S::kUnitBytes;
        if (u < 2 && k_pad != 0) {
          const bool in_front = S::swizzle(ld_row + 8 * (u % 2 ? n : n + a_odd), ld_c) * 8 < k_pad;
          const char* src = tile + ((kOwnOffsetsB && u % 2 ? g_off_b[n] : g_off[n]) + 1024u * (n % 4));
          lds_dma_16B(in_front ? reinterpret_cast<const char*>(kZeros) : src, unit + n * 1024);
        } else {
          if (u % 2) request(k_src(tile, u / 2), unit, n, std::true_type{});
          else request(k_src(tile, u / 2), unit, n, std::false_type{});
        }
      }
    wait_vmem<(S::kAhead - 1) * (S::kLoadsA + S::kLoadsB)>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int f = 0; f < S::TN; ++f)
      bf[0][f] = *reinterpret_cast<const half8_t*>(smem + S::kUnitBytes + b_rd[0] + f * 16 * S::kRowBytes);
#pragma unroll
    for (int i = 0; i < S::TM; ++i)
      afx[0][i] = *reinterpret_cast<const half8_t*>(smem + a_rd[0] + i * 16 * S::kRowBytes);
    // drained here, visibly to the compiler, so that the waits it places at the head of the loop
    // only have to cover the loop's own reads
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_sched_barrier(0);

    // Ring bookkeeping, in bytes: oa = LDS offset of the unit holding A of tile t; B of tile t is
    // one unit further, A of t+1 two, ... (mod kUnits units).  A wavefront alone on its SIMD issues one
    // instruction every 4 cycles, so a 16-cycle MFMA hides at most three other instructions:
    // everything an iteration needs (fragment read bases, request destinations and sources) is
    // therefore computed during the previous k-step in pieces of at most three instructions,
    // each pinned into its own gap between two MFMAs of the slots that carry no fragment reads.
    constexpr unsigned kRingBytes = S::kUnits * S::kUnitBytes;
    auto ring = [](unsigned o) __attribute__((always_inline)) { return o >= kRingBytes ? o - kRingBytes : o; };
    const unsigned rdbase_a0 = smem_addr + a_rd[0], rdbase_a1 = smem_addr + a_rd[1];
    const unsigned rdbase_b0 = smem_addr + b_rd[0], rdbase_b1 = smem_addr + b_rd[1];
    const int last_tile = num_k_tiles - 1;
    unsigned oa = 0;                                             // A of tile t
    unsigned oa1 = 2 * S::kUnitBytes, ob1 = 3 * S::kUnitBytes;   // A, B of tile t+1
    unsigned rd_a1 = rdbase_a1, rd_b1 = rdbase_b1 + S::kUnitBytes;   // reads of (t, k-step 1)
    unsigned req_a = lds_wave_a + 2 * S::kAhead * S::kUnitBytes;       // A of t+kAhead
    const char* src_a = k_src(a_tile, S::kAhead);
    unsigned rd_a0 = 0, rd_b0 = 0, req_b = 0;                        // set during k-step 0
    const char *src_b = b_tile, *src_b1 = b1_tile;
    int kt = 0;
    // pieces run in the read-free gaps from slot kPrepSlot on of k-step 0 / k-step 1
    auto prep0 = [&](int step, int t) __attribute__((always_inline)) {
      __builtin_amdgcn_sched_barrier(0);
      switch (step) {
        case 0: TFK_PIN_S(oa); oa1 = ring(oa + 2 * S::kUnitBytes); TFK_PIN_S(oa1); break;
        case 1: ob1 = ring(oa1 + S::kUnitBytes); TFK_PIN_S(ob1); break;
        case 2: rd_a0 = rdbase_a0 + oa1; TFK_PIN_V(rd_a0); break;
        case 3: rd_b0 = rdbase_b0 + ob1; TFK_PIN_V(rd_b0); break;
        case 4: req_b = lds_wave_b + oa; TFK_PIN_S(req_b); break;
        case 5: kt = t; TFK_PIN_S(kt); kt = min(kt + S::kAhead, last_tile); TFK_PIN_S(kt); break;
        case 6: src_b = b_tile + (size_t)(unsigned)(kt * (S::BK * 2)); TFK_PIN_S(src_b); break;
        case 7:
          if constexpr (kTwo) {
            static_assert(S::free_gaps() >= 8, "a gap for every piece");
            src_b1 = b1_tile + (size_t)(unsigned)(kt * (S::BK * 2));
            TFK_PIN_S(src_b1);
          }
          break;
        default: break;
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    auto prep1 = [&](int step, int t) __attribute__((always_inline)) {
      __builtin_amdgcn_sched_barrier(0);
      switch (step) {
        case 0: oa = oa1; TFK_PIN_S(oa); rd_a1 = rdbase_a1 + oa; TFK_PIN_V(rd_a1); break;
        case 1: rd_b1 = rdbase_b1 + ob1; TFK_PIN_V(rd_b1); break;
        case 2: req_a = ring(oa + 2 * S::kAhead * S::kUnitBytes); TFK_PIN_S(req_a); break;
        case 3: req_a += lds_wave_a; TFK_PIN_S(req_a); break;
        case 4: kt = t; TFK_PIN_S(kt); kt = min(kt + S::kAhead + 1, last_tile); TFK_PIN_S(kt); break;
        case 5: src_a = a_tile + (size_t)(unsigned)(kt * (S::BK * 2)); TFK_PIN_S(src_a); break;
        default: break;
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    for (int t = 0; t < num_k_tiles; ++t) {
#pragma unroll
      for (int i = 0; i < S::TM; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        request_slot(i, src_a, src_a, req_a, kOfA, std::false_type{});
        slot_pinned(0, i, rd_a1, rd_b1, [&](int j) __attribute__((always_inline)) {
          prep0(S::kPrep.piece[i * S::TN + j], t);
        });
      }
      __builtin_amdgcn_sched_barrier(0);
      ring_barrier();
#pragma unroll
      for (int i = 0; i < S::TM; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        request_slot(i, src_b, src_b1, req_b, kOfB, std::true_type{});
        slot_pinned(1, i, rd_a0, rd_b0, [&](int j) __attribute__((always_inline)) {
          prep1(S::kPrep.piece[i * S::TN + j], t);
        });
      }
      settle_behind_last(t);
    }
  }
  __builtin_amdgcn_sched_barrier(0);
  wait_vmem_all();  // the clamped tail requests must not outlive the workgroup's LDS
#undef TFK_PIN_S
#undef TFK_PIN_V
}

}  // namespace
}  // namespace tfk
