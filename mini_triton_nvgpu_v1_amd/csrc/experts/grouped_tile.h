// Products grouped by expert on v_mfma_f32_16x16x32 (f16, bf16) tiles.
//
// A workgroup computes a BM x BN tile of one group's result with the depth in
// k-tiles of BK = 64. An operand lies in memory with the depth along its rows
// (KC: A of kind rows, B stored n x k) or across them (KS: B stored k x n, both
// operands of kind wgrad); it goes to LDS as it lies (direct loads of 16 bytes
// a lane) and becomes fragments by ds_read_b128 (KC) or two transposing
// ds_read_b64_tr_b16 (KS). The product is C^T += B^T A^T, so a lane ends with
// four consecutive columns of a row.
//
// The groups' sizes are known to the GPU only: the grid has a workgroup for
// every tile that the sizes could need, each wave counts the groups' row tiles
// and finds its own, and the workgroups past the last tile end at once.
// Rows that A's indices gather are loaded straight from their places: a lane
// holds the offset of each row that it loads (kind rows), or reads the indices
// of the next k-tile's rows from LDS, where a load two k-tiles ahead put them
// (kind wgrad).
//
// The loop is the one of the dense 16x16x32 tiles: every slot of it is one
// MFMA (inline assembly, accumulator tied in place) followed by the fragment
// reads and loads placed there at compile time; one barrier per k-tile. The
// rules that the inline assembly depends on:
//  (a) each accumulator's first MFMA takes a zero;
//  (b) 24 wait states between the last MFMA and the first accumulator read;
//  (c) a fragment register is rewritten at least 8 slots after its last read;
//  and no instruction but an MFMA touches an accumulator before (b), which the
//  build checks (csrc/tools/mfma_order.py).
//
// 32768 rows x 4096 x 4096 in bf16: one group 816 us (1348 TFLOP/s, the library's
// dense product 824), 16 even groups 847, their rows gathered 876, 16 uneven groups
// 915: 2304 tiles, of which 144 are the groups' ragged ends, go 9 rounds over the
// 256 compute units where 2048 go 8. Bound by the matrix units at the clock the
// power allows. 32-deep k-tiles in 4 or 5 stages instead of 64-deep ones in 2: 961
// and 955 us at 931.
#pragma once

#include "experts_device.h"

namespace tbk {

constexpr int gt_gcd(int a, int b) { return b == 0 ? a : gt_gcd(b, a % b); }
constexpr int gt_min(int a, int b) { return a < b ? a : b; }
constexpr int gt_max(int a, int b) { return a > b ? a : b; }

// Past every record: operands of gathered rows span less than this (the host
// checks), all others less than 2 GiB from their window's base.
constexpr uint32_t kFar = 0xF0000000u;

// One operand: BX rows of C (A) or columns of C (B) by BK of the depth.
template <int BX, int BK, int NT, bool KC>
struct GroupedOperand {
  static constexpr int RB = (KC ? BK : BX) * 2;  // LDS row bytes
  static constexpr int CPR = RB / 16;            // 16-byte chunks per row
  static constexpr int BYTES = BX * BK * 2;
  static constexpr int ROUNDS = BYTES / (NT * 16); // loads per lane per k-tile
  static constexpr int RPR = NT * 16 / RB;         // LDS rows a round covers
  static constexpr int READS = KC ? 1 : 2;         // LDS reads per fragment
  // chunk' = chunk ^ swizzle(row), 256-byte bank period: the b128 reads take
  // 16 rows at one chunk, the transposing reads 4 rows at two 64-byte segments
  static constexpr int PP = KC ? 256 / RB : (RB >= 256 ? 1 : 256 / RB);
  static constexpr int MAXPH = KC ? CPR : gt_min(CPR / 4, 4);
  static constexpr int swizzle(int row) {
    return KC ? (row / PP) % MAXPH : ((4 * ((row / PP) % MAXPH)) ^ (2 * ((row / 8) % 2)));
  }
  // the swizzle repeats every 16 rows: rounds between two of the same phase
  static constexpr int PHASES = 16 / gt_gcd(RPR, 16);
  static_assert(ROUNDS >= 1 && ROUNDS * NT * 16 == BYTES, "whole load rounds");
  static_assert(RPR >= 1 && RB >= 128, "rounds of whole rows, rows of 128 bytes or more");
};

// INDEXED: kind wgrad with gathered rows of A.
template <int BM, int BN, int WGM, int WGN, int STAGES, bool AKC, bool BKC, bool INDEXED>
struct GroupedTile {
  static constexpr int BK = 64, KS = 2;
  static constexpr int NW = WGM * WGN, NT = NW * 64;
  static constexpr int WTM = BM / WGM, WTN = BN / WGN;
  static constexpr int TI = WTM / 16, TJ = WTN / 16, NM = TI * TJ;
  typedef GroupedOperand<BM, BK, NT, AKC> A;
  typedef GroupedOperand<BN, BK, NT, BKC> B;
  static constexpr int RA = A::READS, RB = B::READS;
  static constexpr int NR = RA * TI + RB * TJ; // fragment reads per k step
  static constexpr int STAGE = A::BYTES + B::BYTES;
  // indices of the rows of the k-tiles ahead, a copy per wave
  static constexpr int IDX_AHEAD = 2 * STAGES - 1;
  static constexpr int IDX_SLOTS = 2 * STAGES;
  static constexpr int IDX_BYTES = INDEXED ? NW * IDX_SLOTS * 256 : 0;
  static constexpr int LDS_BYTES = STAGES * STAGE + IDX_BYTES;
  static constexpr int LA = A::ROUNDS, LB = B::ROUNDS;
  static constexpr int LPT = LA + LB + (INDEXED ? 1 : 0); // loads per lane per k-tile
  // MFMA m of a k step: tile (m / TJ, m % TJ). Reads in the order of first
  // use: A0, B0 .. B(TJ-1), A1 .. A(TI-1)
  static constexpr bool op_is_a(int o) { return o < RA || o >= RA + RB * TJ; }
  static constexpr int op_index(int o) {
    return o < RA ? 0 : (o >= RA + RB * TJ ? (o - RB * TJ) / RA : (o - RA) / RB);
  }
  static constexpr int op_half(int o) {
    return o < RA ? o : (o >= RA + RB * TJ ? (o - RB * TJ) % RA : (o - RA) % RB);
  }
  static constexpr int BQ = NM >= 64 ? 8 : (NM >= 32 ? 4 : 2); // the barrier's slot
  static constexpr int last_use(int o) {
    return op_is_a(o) ? op_index(o) * TJ + TJ - 1 : (TI - 1) * TJ + op_index(o);
  }
  static constexpr int spread_slot(int s0, int o) { return s0 + o * (NM - s0) / NR; }
  static constexpr int first_start(int lo) {
    for (int s0 = lo; s0 < NM; ++s0) {
      bool ok = true;
      for (int o = 0; o < NR; ++o)
        ok = ok && NM - last_use(o) + spread_slot(s0, o) >= 8;
      if (ok)
        return s0;
    }
    return NM;
  }
  static constexpr int S0_MID = first_start(0), S0_LAST = first_start(BQ);
  static constexpr int slot_mid(int o) { return spread_slot(S0_MID, o); }
  static constexpr int slot_last(int o) { return spread_slot(S0_LAST, o); }
  static constexpr int NSLOT = KS * NM;
  static constexpr int SPREAD = STAGES == 2 ? NSLOT * 5 / 8 : NSLOT - NSLOT / 8;
  static constexpr int load_slot(int l) { return l * SPREAD / LPT; }
  static constexpr int PER_SLOT = 3;
  static constexpr int mid_op(int m, int k) {
    for (int o = 0, c = 0; o < NR; ++o)
      if (slot_mid(o) == m && c++ == k)
        return o;
    return -1;
  }
  static constexpr int last_op(int m, int k) {
    for (int o = 0, c = 0; o < NR; ++o)
      if (slot_last(o) == m && c++ == k)
        return o;
    return -1;
  }
  static constexpr int load_at(int s, int k) {
    for (int l = 0, c = 0; l < LPT; ++l)
      if (load_slot(l) == s && c++ == k)
        return l;
    return -1;
  }
  // vmcnt at the prologue's wait and at a k-tile's barrier: the operands'
  // loads of the k-tiles that may still be on their way
  static constexpr int VM_PROLOGUE = (STAGES - 1) * (LA + LB);
  static constexpr int VM_LOOP = (STAGES - 2) * (LA + LB);
  static constexpr int U = STAGES;
  static constexpr int min_rewrite_distance() {
    int d = 1 << 30;
    for (int o = 0; o < NR; ++o) {
      d = gt_min(d, NM - last_use(o) + slot_mid(o));
      d = gt_min(d, NM - last_use(o) + slot_last(o));
    }
    return d;
  }
  static constexpr bool tables_cover() {
    for (int o = 0; o < NR; ++o)
      if (slot_mid(o) >= NM || slot_last(o) < BQ || slot_last(o) >= NM)
        return false;
    for (int m = 0; m < NM; ++m)
      if (mid_op(m, PER_SLOT) >= 0 || last_op(m, PER_SLOT) >= 0)
        return false;
    for (int s = 0; s < NSLOT; ++s)
      if (load_at(s, PER_SLOT) >= 0)
        return false;
    return true;
  }
  // epilogue staging: 16-row blocks of the wave tile through LDS, f32
  static constexpr int E_ROWB = WTN * 4;
  static constexpr int EPI_REGION = 16 * E_ROWB;

  static_assert(BM % (16 * WGM) == 0 && BN % (32 * WGN) == 0, "16x16 tiles, in column pairs");
  static_assert(NM >= 16 && NM <= 64, "16..64 MFMA tiles per wave");
  static_assert(LDS_BYTES <= 160 * 1024, "160 KiB of LDS");
  static_assert(NW * EPI_REGION <= STAGES * STAGE, "the epilogue's staging fits the ring");
  static_assert(VM_PROLOGUE < 64, "vmcnt range");
  static_assert(tables_cover(), "every read and load has its slot");
  static_assert(min_rewrite_distance() >= 8, "(c)");
};

// 4 bytes per lane into LDS at lds_base + 4 * lane (load_lds16).
__device__ __forceinline__ void load_lds4(u32x4 rsrc, uint32_t lds_base, uint32_t voff) {
  lds_base = __builtin_amdgcn_readfirstlane(lds_base);
  asm volatile("s_mov_b32 m0, %0\n\t"
               "buffer_load_dword %1, %2, 0 offen lds"
               :
               : "s"(lds_base), "v"(voff), "s"(rsrc)
               : "memory");
}

template <int T>
__device__ __forceinline__ void mfma_first(f32x4 &acc, const half8 &b, const half8 &a) {
  if constexpr (T == kElemF16)
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, 0" : "=a"(acc) : "v"(b), "v"(a));
  else
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=a"(acc) : "v"(b), "v"(a));
}
template <int T>
__device__ __forceinline__ void mfma_next(f32x4 &acc, const half8 &b, const half8 &a) {
  if constexpr (T == kElemF16)
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(acc) : "v"(b), "v"(a));
  else
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(b), "v"(a));
}

// Where a tile lies. Rows: slots [row0, row_end) of the result's rows, the
// depth k. Wgrad: rows [row0, row_end) of C_e, the depth the slots
// [slot0, slot0 + depth).
struct TilePlace {
  int group, row0, row_end, col0, slot0, depth;
};

// The tile's result, staged through LDS 16 rows at a time: lane l holds row
// l % 16 of block i, columns 16 j + 4 (l / 16) .. +3. In LDS a row is its f32
// columns in 16-byte chunks, chunk ^ (row % 16); whole rows come back, 4
// columns a lane, are rounded and stored.
template <class T, int TC, int ACT, bool WGRAD, bool AGPR = true>
__device__ __forceinline__ void grouped_store(const GroupedParams &p, const TilePlace &at,
                                              f32x4 (&acc)[T::TI][T::TJ], TBK_LDS char *wl,
                                              int wm, int wn) {
  constexpr bool GATED = ACT == kActSwiglu;
  constexpr int WIDTH = GATED ? T::WTN / 2 : T::WTN; // result columns of a wave
  constexpr int CPR = WIDTH / 4;                     // lanes per row
  constexpr int RPI = 64 / CPR, NLD = 16 / RPI;
  constexpr int XM = gt_min(16, CPR);
  constexpr int ES = TC == kElemF32 ? 4 : 2;
  const int el = lane_id_fresh();
  const int r = el & 15, g = el >> 4;
  const int q = el % CPR, rr0 = el / CPR;
  const int col = at.col0 + wn * WIDTH + 4 * q;
  const int64_t first = (int64_t)at.row0 * p.ldc + (WGRAD ? at.group * p.stride : 0);
  const int rows = at.row_end - at.row0;
  const uint64_t span = (uint64_t)rows * (uint64_t)p.ldc * ES;
  const __amdgpu_buffer_rsrc_t rc = make_rsrc(static_cast<char *>(p.C) + first * ES,
                                              span < kOob ? (uint32_t)span : kOob - 16u);
  static_for<T::TI>([&](auto i_c) {
    constexpr int i = decltype(i_c)::value;
    // an asm (no instruction) that differs per activation: the variants of the
    // dispatch then share no accumulator read, which the compiler would hoist
    // above it and hold in VGPRs for the whole tile
#pragma unroll
    for (int j = 0; j < T::TJ; ++j)
      if constexpr (AGPR)
        asm volatile("; activation %1" : "+a"(acc[i][j]) : "i"(ACT));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < T::TJ; j += GATED ? 2 : 1) {
      f32x4 x = acc[i][j];
      if constexpr (GATED) {
        const f32x4 u = acc[i][j + 1];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[e] = epi_activation(x[e], 3) * u[e];
      } else if constexpr (ACT != 0) {
        x = epi_apply4_t<ACT, false>(x, (f32x4)0.f, 0.f, 0.f);
      }
      const int chunk = (GATED ? 2 * j : 4 * j) + g;
      *(TBK_LDS f32x4 *)(wl + r * (WIDTH * 4) + ((chunk ^ (r % XM)) * 16)) = x;
      if (j & 1)
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int s = 0; s < NLD; ++s) {
      const int rr = s * RPI + rr0;
      f32x4 v = *(const TBK_LDS f32x4 *)(wl + rr * (WIDTH * 4) + ((q ^ (rr % XM)) * 16));
      const int trow = wm * T::WTM + 16 * i + rr;
      const uint32_t off = trow < rows && col < p.n
                               ? ((uint32_t)trow * (uint32_t)p.ldc + (uint32_t)col) * ES
                               : kOob;
      if constexpr (TC == kElemF32) {
        if constexpr (WGRAD)
          if (p.load_c)
            v += __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rc, off, 0, 0));
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), rc, off, 0, kStoreNT);
      } else {
        u32x2 h;
        if constexpr (TC == kElemF16) {
          h[0] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[0]) |
                 ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[1]) << 16);
          h[1] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2]) |
                 ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[3]) << 16);
        } else {
          h[0] = (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v[0]) |
                 ((uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v[1]) << 16);
          h[1] = (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v[2]) |
                 ((uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v[3]) << 16);
        }
        __builtin_amdgcn_raw_buffer_store_b64(h, rc, off, 0, 0);
      }
    }
    // the next block's writes go to the addresses just read
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  });
}

// A T-typed tile; TC: the result's type. WGRAD: kind wgrad (both operands KS).
template <int T, int TC, int BM, int BN, int WGM, int WGN, int STAGES, bool BKC, bool WGRAD,
          bool INDEXED>
__device__ __forceinline__ void grouped_tile(const GroupedParams &p, const TilePlace &at,
                                             u32x4 *lds) {
  typedef GroupedTile<BM, BN, WGM, WGN, STAGES, !WGRAD, BKC, INDEXED> G;
  typedef typename G::A OA;
  typedef typename G::B OB;
  static_assert(!(WGRAD && BKC) && (WGRAD || !INDEXED), "kind wgrad: depth across the rows");
  constexpr int TI = G::TI, TJ = G::TJ, NM = G::NM, NR = G::NR, BQ = G::BQ, KS = 2;
  constexpr int LA = G::LA, LPT = G::LPT, U = G::U, BK = G::BK;
  constexpr int L0A = INDEXED ? 1 : 0; // load 0 is the index load
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WGN, wn = wave % WGN;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(TBK_LDS void *)lds;
  const bool gated = !WGRAD && p.act == kActSwiglu;
  const int nk = (at.depth + BK - 1) / BK;
  const int kfull = at.depth / BK;
  const int krem = at.depth - kfull * BK;
  const int t = wave * 64 + lane;
  const int a_r0 = t / OA::CPR, a_pc = t % OA::CPR;
  const int b_r0 = t / OB::CPR, b_pc = t % OB::CPR;
  const uint32_t wlds = lds0 + wave * 1024u;
  const uint32_t lda2 = (uint32_t)p.lda * 2u, ldb2 = (uint32_t)p.ldb * 2u;

  // ---- A -------------------------------------------------------------------
  // Rows: the offset of each row that the lane loads, from A's base (gathered)
  // or from the tile's first row; a slot past the group or without a row of A
  // reads zeros. Wgrad: per phase the offset of the lane's columns.
  uint32_t va[WGRAD ? OA::PHASES : LA];
  const char *a_base_ptr = static_cast<const char *>(p.A);
  uint32_t a_records = 0;
  if constexpr (!WGRAD) {
    const bool gather = p.rows != nullptr;
    const uint64_t span = (uint64_t)p.a_rows * lda2;
    if (!gather) {
      a_base_ptr += (int64_t)at.row0 * lda2;
      const int64_t rows_here = gt_min((int)p.a_rows, at.row_end) - at.row0;
      a_records = rows_here > 0 ? gt_min((int)rows_here, BM) * lda2 : 0u;
    } else {
      a_records = (uint32_t)span; // below kFar: the host checks
    }
#pragma unroll
    for (int R = 0; R < LA; ++R) {
      const int row = a_r0 + R * OA::RPR, slot = at.row0 + row;
      const int lc = a_pc ^ OA::swizzle(row);
      int64_t src = -1;
      if (slot < at.row_end)
        src = slot_row(p, slot);
      if (!gather)
        src -= src >= 0 ? at.row0 : 0;
      va[R] = src >= 0 ? (uint32_t)src * lda2 + (uint32_t)lc * 16u : kFar;
    }
  } else {
#pragma unroll
    for (int ph = 0; ph < OA::PHASES; ++ph) {
      const int col = at.row0 + 8 * (a_pc ^ OA::swizzle(a_r0 + ph * OA::RPR));
      va[ph] = col < at.row_end ? (uint32_t)col * 2u + (INDEXED ? 0u : (uint32_t)a_r0 * lda2)
                                : kFar;
    }
  }
  // chunk of the depth in the partial last k-tile (KC operands)
  auto past_k = [&](int row, int pc, auto op) {
    return 8 * (pc ^ decltype(op)::swizzle(row)) >= krem;
  };

  // ---- B -------------------------------------------------------------------
  uint32_t vb[OB::PHASES];
  const char *b_base_ptr = static_cast<const char *>(p.B);
  uint32_t b_records = 0;
  uint32_t b_round = (uint32_t)OB::RPR * ldb2; // bytes between rounds of rows
  if constexpr (WGRAD) {
    b_base_ptr += (int64_t)at.slot0 * ldb2;
#pragma unroll
    for (int ph = 0; ph < OB::PHASES; ++ph) {
      const int col = at.col0 + 8 * (b_pc ^ OB::swizzle(b_r0 + ph * OB::RPR));
      vb[ph] = col < p.n ? (uint32_t)col * 2u + (uint32_t)b_r0 * ldb2 : kFar;
    }
  } else {
    b_base_ptr += (int64_t)at.group * p.stride * 2;
    const int bn = gated ? 2 * p.n : p.n; // columns of B_e
    if constexpr (BKC) {
      // LDS row r holds column r of the tile; gated: 16 of the gate, then the
      // same 16 of the other half
      b_base_ptr += (int64_t)at.col0 * ldb2;
      b_records = (uint32_t)(bn - at.col0) * ldb2;
      const int row = gated ? (b_r0 >> 5) * 16 + (b_r0 & 15) + ((b_r0 >> 4) & 1) * p.n : b_r0;
      b_round = gated ? b_round / 2 : b_round;
      static_assert(OB::PHASES == 1 && OB::RPR % 32 == 0, "a round is whole column pairs");
      vb[0] = (uint32_t)row * ldb2 + (uint32_t)(b_pc ^ OB::swizzle(b_r0)) * 16u;
    } else {
      b_records = (uint32_t)p.k * ldb2;
#pragma unroll
      for (int ph = 0; ph < OB::PHASES; ++ph) {
        const int r = b_r0 + ph * OB::RPR;
        const int c = 8 * (b_pc ^ OB::swizzle(r)); // column of the tile
        int col = at.col0 + c;
        bool in = col < p.n;
        if (gated) {
          col = at.col0 + (c >> 5) * 16 + (c & 15);
          in = col < p.n;
          col += ((c >> 4) & 1) * p.n;
        }
        vb[ph] = in ? (uint32_t)b_r0 * ldb2 + (uint32_t)col * 2u : kOob;
      }
    }
  }

  // ---- loads -----------------------------------------------------------------
  // the rows' indices in LDS (gathered rows of kind wgrad)
  const uint32_t idx0 = lds0 + STAGES * G::STAGE + wave * (G::IDX_SLOTS * 256);
  const int *rows_base = INDEXED ? p.rows + at.slot0 : nullptr;
  auto load_index = [&](int kt) {
    load_lds4(rsrc_dwords(rows_base, kt < nk ? (uint32_t)at.depth * 4u : 0u),
              idx0 + (uint32_t)(kt % G::IDX_SLOTS) * 256u,
              kt < nk ? ((uint32_t)kt * BK + lane) * 4u : 0u);
  };
  // kind wgrad: rows of k-tile kt that the group has
  auto rows_of = [&](int kt) { return kt < kfull ? BK : (kt == kfull ? krem : 0); };
  // the row of A that the lane loads in round R, a_rows where there is none; read
  // some slots before it is used
  static_assert(!INDEXED || (LA == G::LB && OA::RPR == OB::RPR), "one index for A and B");
  uint32_t src_row[INDEXED ? LA : 1];
  auto read_index = [&](int kt, auto r_c) {
    constexpr int R = decltype(r_c)::value;
    src_row[R] =
        *(const TBK_LDS uint32_t *)(uintptr_t)(idx0 + (uint32_t)(kt % G::IDX_SLOTS) * 256u +
                                               (uint32_t)(a_r0 + R * OA::RPR) * 4u);
  };
  const uint32_t a_rows = (uint32_t)p.a_rows;
  uint32_t lda_of[INDEXED ? OA::PHASES : 1]; // 0 for columns past the last
#pragma unroll
  for (int ph = 0; ph < (INDEXED ? OA::PHASES : 0); ++ph)
    lda_of[ph] = va[ph] == kFar ? 0u : lda2;
  auto rsrc_a = [&](int kt) {
    if constexpr (WGRAD) {
      if constexpr (INDEXED)
        return rsrc_dwords(a_base_ptr, kt < nk ? a_rows * lda2 : 0u);
      else
        return rsrc_dwords(a_base_ptr + ((int64_t)at.slot0 + (int64_t)kt * BK) * lda2,
                           kt < nk ? kFar : 0u);
    } else {
      return rsrc_dwords(a_base_ptr, kt < nk ? a_records : 0u);
    }
  };
  auto rsrc_b = [&](int kt) {
    if constexpr (WGRAD)
      return rsrc_dwords(b_base_ptr + (int64_t)kt * BK * ldb2, kt < nk ? kFar : 0u);
    else
      return rsrc_dwords(b_base_ptr, kt < nk ? b_records : 0u);
  };
  // load l of k-tile kt into stage ST
  auto load = [&](const u32x4 &ra, const u32x4 &rb, int kt, auto st_c, auto l_c) {
    constexpr int ST = decltype(st_c)::value, L = decltype(l_c)::value;
    const bool kpart = kt == kfull, live = kt < nk;
    if constexpr (L < L0A) {
      load_index(kt + G::IDX_AHEAD - STAGES);
    } else if constexpr (L - L0A < LA) {
      constexpr int R = L - L0A;
      uint32_t v;
      uint32_t so = 0;
      if constexpr (INDEXED) {
        const uint32_t row = a_r0 + R * OA::RPR < rows_of(kt) ? src_row[R] : ~0u;
        src_row[R] = row < a_rows ? row : a_rows;
        v = src_row[R] * lda_of[R % OA::PHASES] + va[R % OA::PHASES];
      } else if constexpr (WGRAD) {
        v = a_r0 + R * OA::RPR < rows_of(kt) ? va[R % OA::PHASES] : kFar;
        so = live ? (uint32_t)(R * OA::RPR) * lda2 : 0u;
      } else {
        v = kpart && past_k(a_r0 + R * OA::RPR, a_pc, OA{}) ? kFar : va[R];
        so = live ? (uint32_t)kt * (BK * 2u) : 0u;
      }
      load_lds16_at<ST * G::STAGE + R * G::NW * 1024>(ra, wlds, v, so);
    } else {
      constexpr int R = L - L0A - LA;
      uint32_t v = vb[R % OB::PHASES], so = 0;
      if constexpr (WGRAD) {
        if constexpr (INDEXED)
          v = src_row[R] < a_rows ? v : kFar;
        else
          v = b_r0 + R * OB::RPR < rows_of(kt) ? v : kFar;
        so = live ? (uint32_t)(R * OB::RPR) * ldb2 : 0u;
      } else if constexpr (BKC) {
        v = kpart && past_k(b_r0, b_pc, OB{}) ? kOob : v;
        so = live ? (uint32_t)kt * (BK * 2u) + (uint32_t)R * b_round : 0u;
      } else {
        const int lim = kpart ? krem - R * OB::RPR : (1 << 30);
        v = b_r0 >= lim ? kOob : v;
        so = live ? ((uint32_t)kt * BK + (uint32_t)(R * OB::RPR)) * ldb2 : 0u;
      }
      load_lds16_at<ST * G::STAGE + OA::BYTES + R * G::NW * 1024>(rb, wlds, v, so);
    }
  };

  // ---- fragment reads ----------------------------------------------------------
  const int g = lane >> 4, ta = (lane >> 2) & 3, tb = lane & 3;
  // KC: one base per k step; KS: one per fragment
  uint32_t a_base[STAGES][WGRAD ? TI : KS], b_base[STAGES][BKC ? KS : TJ];
#pragma unroll
  for (int st = 0; st < STAGES; ++st) {
    const uint32_t sa = lds0 + st * G::STAGE, sb = sa + OA::BYTES;
    if constexpr (!WGRAD) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int row = wm * G::WTM + (lane & 15);
        a_base[st][ks] = sa + row * OA::RB + (((4 * ks + g) ^ OA::swizzle(row)) * 16);
      }
    } else {
#pragma unroll
      for (int i = 0; i < TI; ++i) {
        const int k = 8 * g + ta, c = (wm * G::WTM + 16 * i) / 8 + (tb >> 1);
        a_base[st][i] = sa + k * OA::RB + ((c ^ OA::swizzle(k)) * 16) + 8 * (tb & 1);
      }
    }
    if constexpr (BKC) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int row = wn * G::WTN + (lane & 15);
        b_base[st][ks] = sb + row * OB::RB + (((4 * ks + g) ^ OB::swizzle(row)) * 16);
      }
    } else {
#pragma unroll
      for (int j = 0; j < TJ; ++j) {
        const int k = 8 * g + ta, c = (wn * G::WTN + 16 * j) / 8 + (tb >> 1);
        b_base[st][j] = sb + k * OB::RB + ((c ^ OB::swizzle(k)) * 16) + 8 * (tb & 1);
      }
    }
  }
  f32x4 acc[TI][TJ];
  half8 fa[2][TI], fb[2][TJ];
  auto read_kc = [](uint32_t addr) {
    return __builtin_bit_cast(half8, *(const TBK_LDS u32x4 *)(uintptr_t)addr);
  };
  auto read_ks = [](uint32_t addr) {
    return __builtin_bit_cast(
        half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((TBK_LDS short4 *)(uintptr_t)addr));
  };
  auto rd = [&](auto buf_c, auto st_c, auto ks_c, auto o_c) {
    constexpr int BUF = decltype(buf_c)::value, ST = decltype(st_c)::value;
    constexpr int KSI = decltype(ks_c)::value, O = decltype(o_c)::value;
    constexpr int I = G::op_index(O), H = G::op_half(O);
    if constexpr (G::op_is_a(O)) {
      if constexpr (!WGRAD) {
        fa[BUF][I] = read_kc(a_base[ST][KSI] + I * 16 * OA::RB);
      } else {
        const half4 h = read_ks(a_base[ST][I] + KSI * 32 * OA::RB + H * 4 * OA::RB);
        if constexpr (H == 0)
          fa[BUF][I].lo = h;
        else
          fa[BUF][I].hi = h;
      }
    } else {
      if constexpr (BKC) {
        fb[BUF][I] = read_kc(b_base[ST][KSI] + I * 16 * OB::RB);
      } else {
        const half4 h = read_ks(b_base[ST][I] + KSI * 32 * OB::RB + H * 4 * OB::RB);
        if constexpr (H == 0)
          fb[BUF][I].lo = h;
        else
          fb[BUF][I].hi = h;
      }
    }
  };
  auto barrier = [&]() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  using F = std::integral_constant<bool, false>;
  using Z = std::integral_constant<int, 0>;
  using ONE = std::integral_constant<int, 1>;
  using LAST = std::integral_constant<int, KS - 1>;
  using QB = std::integral_constant<int, BQ>;
  using ENDS = std::integral_constant<int, NM>;
  // the table's k-th entries of a slot, k < PER_SLOT
  auto each = [](auto table, auto &&f) {
    static_for<G::PER_SLOT>([&](auto k_c) {
      constexpr int O = decltype(table)::at(decltype(k_c)::value);
      if constexpr (O >= 0)
        f(std::integral_constant<int, O>{});
    });
  };
  // slots [LO, HI) of k step ks, stage st: the MFMAs, the reads of the k-tile's
  // next k step, and `extra`
  auto kstep = [&](auto st_c, auto ks_c, auto lo_c, auto hi_c, auto first_c, auto &&extra) {
    constexpr int KSI = decltype(ks_c)::value;
    static_for<NM>([&](auto m_c) {
      constexpr int M = decltype(m_c)::value;
      if constexpr (M >= decltype(lo_c)::value && M < decltype(hi_c)::value) {
        constexpr int i = M / TJ, j = M % TJ;
        if constexpr (decltype(first_c)::value)
          mfma_first<T>(acc[i][j], fb[KSI][j], fa[KSI][i]);
        else
          mfma_next<T>(acc[i][j], fb[KSI][j], fa[KSI][i]);
        if constexpr (KSI + 1 < KS) {
          struct Table {
            static constexpr int at(int k) { return G::mid_op(M, k); }
          };
          each(Table{}, [&](auto o_c) { rd(ONE{}, st_c, ONE{}, o_c); });
        }
        extra(m_c);
        __builtin_amdgcn_sched_barrier(0);
      }
    });
  };
  auto nothing = [](auto) {};
  // from the barrier of k-tile it to just before the barrier of k-tile it + 1;
  // stage Q (k-tile it) is refilled with k-tile it + STAGES
  auto body = [&](int it, auto q_c) {
    constexpr int Q = decltype(q_c)::value, SN = (Q + 1) % STAGES;
    using SNEXT = std::integral_constant<int, SN>;
    const u32x4 ra = rsrc_a(it + STAGES), rb = rsrc_b(it + STAGES);
    wait_vmcnt_lgkm0<G::VM_LOOP>();
    barrier();
    auto refill_at = [&](auto s_c) {
      constexpr int S = decltype(s_c)::value;
      struct Table {
        static constexpr int at(int k) { return G::load_at(S, k); }
      };
      each(Table{}, [&](auto l_c) {
        constexpr int L = decltype(l_c)::value;
        load(ra, rb, it + STAGES, q_c, l_c);
        if constexpr (INDEXED && L < LA) { // two loads ahead of load L0A + R
          constexpr int R = L + L0A;
          if constexpr (R < LA)
            read_index(it + STAGES, std::integral_constant<int, R>{});
        }
      });
    };
    if constexpr (INDEXED)
      read_index(it + STAGES, std::integral_constant<int, 0>{});
    kstep(q_c, LAST{}, QB{}, ENDS{}, F{}, [&](auto m_c) {
      constexpr int M = decltype(m_c)::value;
      struct Table {
        static constexpr int at(int k) { return G::last_op(M, k); }
      };
      each(Table{}, [&](auto o_c) { rd(Z{}, SNEXT{}, Z{}, o_c); });
      refill_at(std::integral_constant<int, M - BQ>{});
    });
    static_for<KS>([&](auto ks_c) {
      constexpr int KSI = decltype(ks_c)::value;
      using HI = std::integral_constant<int, KSI + 1 < KS ? NM : BQ>;
      kstep(SNEXT{}, ks_c, Z{}, HI{}, F{}, [&](auto m_c) {
        refill_at(std::integral_constant<int, NM - BQ + KSI * NM + decltype(m_c)::value>{});
      });
    });
  };

  // ---- prologue ------------------------------------------------------------------
  if constexpr (INDEXED) {
    static_for<G::IDX_AHEAD>([&](auto kt_c) { load_index(decltype(kt_c)::value); });
    wait_vmcnt<0>();
    asm volatile("" ::: "memory");
  }
  static_for<STAGES>([&](auto st_c) {
    constexpr int ST = decltype(st_c)::value;
    const u32x4 ra = rsrc_a(ST), rb = rsrc_b(ST);
    if constexpr (INDEXED)
      static_for<LA>([&](auto r_c) { read_index(ST, r_c); });
    static_for<LPT>([&](auto l_c) {
      if constexpr (decltype(l_c)::value >= L0A)
        load(ra, rb, ST, st_c, l_c);
    });
  });
  wait_vmcnt<G::VM_PROLOGUE>();
  barrier();
  static_for<NR>([&](auto o_c) { rd(Z{}, Z{}, Z{}, o_c); });
  kstep(Z{}, Z{}, Z{}, ENDS{}, std::integral_constant<bool, true>{}, nothing);
  kstep(Z{}, ONE{}, Z{}, QB{}, F{}, nothing);
  // bodies of k-tiles 0 .. nk - 2; the tail is the last k-tile after its
  // barrier point
  int it = 0;
  if (it < nk - 1) {
    for (;;) {
      bool done = false;
      static_for<U>([&](auto q_c) {
        if (!done) {
          body(it, q_c);
          ++it;
          done = it >= nk - 1;
        }
      });
      if (done)
        break;
    }
  }
  kstep(Z{}, LAST{}, QB{}, ENDS{}, F{}, nothing);
  acc_read_fence(acc); // (b)
  wait_vmcnt<0>();     // the loads past the end have landed too

  // ---- result -----------------------------------------------------------------------
  barrier(); // every wave is past its last fragment read
  TBK_LDS char *wl = (TBK_LDS char *)(TBK_LDS void *)lds + wave * G::EPI_REGION;
  if constexpr (WGRAD) {
    grouped_store<G, TC, 0, true>(p, at, acc, wl, wm, wn);
  } else {
    // dispatched once for the tile
    auto variant = [&](auto act_c) {
      grouped_store<G, TC, decltype(act_c)::value, false>(p, at, acc, wl, wm, wn);
    };
    switch (p.act) {
    case 1: variant(std::integral_constant<int, 1>{}); break;
    case 2: variant(std::integral_constant<int, 2>{}); break;
    case 3: variant(std::integral_constant<int, 3>{}); break;
    case 4: variant(std::integral_constant<int, 4>{}); break;
    default: variant(std::integral_constant<int, 0>{}); break;
    }
  }
}

// Tile `w` of `rows` x `cols` tiles in runs of `gm` row tiles: within a run the
// rows come first, so that tiles running together share both operands.
__device__ __forceinline__ void tile_order(int w, int rows, int cols, int gm, int &r, int &c) {
  const int run = gm * cols, first = w / run * gm;
  const int here = min(gm, rows - first), in = w % run;
  r = first + in % here;
  c = in / here;
}

// The tile of kind rows that block `block` takes: an XCD takes a run of
// neighbouring tiles, and a run goes through a group's row tiles (8 of them at
// most) before it moves on to the next columns, so that the group's weights are
// read once. False: no tile is left.
__device__ __forceinline__ bool rows_place(const GroupedParams &p, int block, int bm, int cols,
                                           int tiles_n, TilePlace &at) {
  GroupTile g{-1, 0, 0, 0, 0};
  int w;
  if (p.groups <= 64) { // one count serves the total and the search
    const GroupScan c(p, bm, 0);
    const int total = last_lane(c.upto) * tiles_n;
    if (block >= total)
      return false;
    w = program_of_block(block, total, 8);
    c.find(w / tiles_n, bm, 0, g);
  } else {
    const int total = group_tiles(p, bm) * tiles_n;
    if (block >= total)
      return false;
    w = program_of_block(block, total, 8);
    g = group_tile(p, bm, w / tiles_n);
  }
  if (g.group < 0)
    return false;
  int tm, tn;
  tile_order(g.index * tiles_n + w % tiles_n, g.tiles, tiles_n, 8, tm, tn);
  at = TilePlace{g.group, g.begin + (tm - g.index) * bm, g.end, tn * cols, 0, p.k};
  return true;
}

template <int T, int TC, int BM, int BN, int WGM, int WGN, int STAGES, bool BKC>
__global__ __launch_bounds__(WGM *WGN * 64, 1) void grouped_rows(GroupedParams p, int tiles_n) {
  typedef GroupedTile<BM, BN, WGM, WGN, STAGES, true, BKC, false> G;
  __shared__ u32x4 lds[G::LDS_BYTES / 16];
  TilePlace at;
  if (rows_place(p, blockIdx.x, BM, p.act == kActSwiglu ? BN / 2 : BN, tiles_n, at))
    grouped_tile<T, TC, BM, BN, WGM, WGN, STAGES, BKC, false, false>(p, at, lds);
}

template <int T, int TC, int BM, int BN, int WGM, int WGN, int STAGES, bool INDEXED>
__global__ __launch_bounds__(WGM *WGN * 64, 1) void grouped_wgrad(GroupedParams p, int tiles_m,
                                                                  int tiles_n, int gm) {
  typedef GroupedTile<BM, BN, WGM, WGN, STAGES, false, false, INDEXED> G;
  __shared__ u32x4 lds[G::LDS_BYTES / 16];
  // The groups' depths differ, so every XCD (blocks go round them) takes an eighth
  // of each group's tiles rather than whole groups: 8192 tokens of 2 of 16 experts,
  // C 4096 x 2048 in f32, 361 us against 408 with whole groups (with later steps
  // 298-310 at its fastest and 323-339 on average: 811-922 TFLOP/s, and 537 MB of C
  // written after the products).
  const int per = tiles_m * tiles_n, per_xcd = (per + 7) / 8;
  const int i = blockIdx.x / 8, group = i / per_xcd;
  const int w = (int)(blockIdx.x % 8) * per_xcd + i % per_xcd;
  if (w >= per)
    return;
  int tm, tn;
  tile_order(w, tiles_m, tiles_n, gm, tm, tn);
  const int begin = __builtin_amdgcn_readfirstlane(group_at(p, group));
  const int end = __builtin_amdgcn_readfirstlane(group_at(p, group + 1));
  const TilePlace at{group, tm * BM, p.k, tn * BN, begin, end > begin ? end - begin : 0};
  grouped_tile<T, TC, BM, BN, WGM, WGN, STAGES, false, true, INDEXED>(p, at, lds);
}

} // namespace tbk
