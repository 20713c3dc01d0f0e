// Products of e4m3 operands with block scales, on v_mfma_f32_16x16x128_f8f6f4:
//   C[i] = act(sum over blocks b of 128 of the depth:
//              a_scale[row][b] b_scale[column / 128][b] (A_b[row] . B_b[column]))
// One such MFMA takes a whole block of the depth, so its result, from a zero
// accumulator, is one block's product: it is scaled and added to the tile's f32
// accumulators by the vector unit (one product of scales and four
// multiply-adds per MFMA, less than the MFMA's own time).
// The instruction keeps, of each 8 neighbouring products, what lies above 2^-13 of
// the largest power of two among them, and sums the groups of 8 as f32: up to
// 2^-10 of the sum of the magnitudes is lost, and of ordinary activations and
// weights 1e-5 of the result, which is below the rounding of 16-bit results and
// far below the 2^-4 of the operands. Exact sums would need the f16 instruction
// on converted values, at half the rate.
//
// A k-tile is one block. Rows of 128 bytes lie in LDS as in memory, 16-byte
// chunk ^ (row / 2) % 8; lane l of a fragment takes chunks l / 16 and
// 4 + l / 16 of row l % 16: the depth's order within a block does not matter as
// long as A and B have the same.
//
// A wave tile's rows go in pairs of 16. While a pair's MFMAs run, the next
// pair's fragments are read. The barrier of a k-tile comes before its last
// pair, whose fragments are in registers by then: behind it the freed stage is
// refilled two k-tiles ahead, and the next k-tile's first pair and B's
// fragments, each after its last use, are read.
//
// 8192 x 8192 x 4096 on 256 x 256 tiles: 256-268 us, 2.05-2.15 PFLOP/s. At 265 us it took 180
// with the MFMAs alone (3.05 PFLOP/s, the clock the power allows), 238 without the
// loads, 252 without the scaling: no one of them bounds it, they share a compute
// unit whose 8 waves meet at a barrier every 128 of the depth. By count LDS is a
// bound of the same size as the matrix unit: a k-tile's 192 KB of fragment reads and
// 64 KB of loads are 2048 clocks at 128 bytes each, its MFMAs 2048 clocks too. Three stages on 256 x
// 128 tiles took 328 us, four on 128 x 128 463: the loads are not late.
#pragma once

#include "grouped_tile.h"

namespace tbk {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

template <int BM, int BN, int WGM, int WGN, int STAGES>
struct ScaledTile {
  static constexpr int BK = 128;
  static constexpr int NW = WGM * WGN, NT = NW * 64;
  static constexpr int WTM = BM / WGM, WTN = BN / WGN;
  static constexpr int TI = WTM / 16, TJ = WTN / 16, NM = TI * TJ;
  static constexpr int NP = TI / 2;    // pairs of fragment rows
  static constexpr int PS = 2 * TJ;    // MFMA slots of a pair
  static constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  // Scales, in units of 64: the rows', then the columns' (one for 8). Those of
  // four k-tiles lie side by side in memory and are loaded together, each unit's
  // by four waves in the same k-tile, so that a row's cache line is asked for once
  // and not four times (it does not stay there: 8192 x 8192 x 4096 265 -> 256 us).
  static constexpr int UNITS = BM / 64 + 1;
  static constexpr int KT_BYTES = UNITS * 256;          // of a k-tile
  static constexpr int RING = 4 * STAGES;               // k-tiles of scales in LDS
  static constexpr int SCALES = STAGES * STAGE;         // where they are
  static constexpr int TABLE = SCALES + RING * KT_BYTES; // the units' offsets
  static constexpr int SPARE = TABLE + UNITS * 256;     // what no wave needs
  static constexpr int LDS_BYTES = SPARE + 256;
  static constexpr int LA = A_BYTES / (NT * 16), LB = B_BYTES / (NT * 16);
  static constexpr int LPT = LA + LB + 1;
  static constexpr int RPR = NT * 16 / BK; // rows a round covers
  static constexpr int swizzle(int row) { return (row / 2) % 8; }
  // epilogue staging
  static constexpr int E_ROWB = WTN * 4, EPI_REGION = 16 * E_ROWB;
  // refill load l goes body slot load_slot(l): slots from the barrier on
  static constexpr int load_slot(int l) { return l * (NM * 3 / 8) / LPT; }
  static_assert(load_slot(LPT - 1) < NM, "a k-tile's loads are issued before the next barrier");
  static_assert(TI % 4 == 0 && WTN % 32 == 0, "pairs of rows, two buffers of them");
  static_assert(LA * NT * 16 == A_BYTES && LB * NT * 16 == B_BYTES, "whole load rounds");
  static_assert(RPR % 32 == 0, "rounds of whole swizzle periods and column pairs");
  static_assert(UNITS <= NW && NW % 4 == 0 && BN / 8 <= 64, "four waves per unit");
  static_assert(LDS_BYTES <= 160 * 1024, "160 KiB of LDS");
  static_assert((STAGES - 1) * LPT < 64, "vmcnt range");
  static_assert(NW * EPI_REGION <= LDS_BYTES, "the epilogue's staging fits");
};

// Inline assembly, so that the slots stay in order. What the compiler then does
// not know about it holds by the schedule: a result is read three MFMAs later
// (each takes the matrix unit for at least 8 passes of 4 clocks; a result is
// there 5 passes after its last), and a fragment's registers are rewritten by
// LDS reads that are issued two MFMAs after its last use.
__device__ __forceinline__ void mfma_f8(f32x4 &d, const i32x8 &b, const i32x8 &a) {
  asm volatile("v_mfma_f32_16x16x128_f8f6f4 %0, %1, %2, 0" : "=&v"(d) : "v"(b), "v"(a));
}

template <int TC, int BM, int BN, int WGM, int WGN, int STAGES>
__device__ __forceinline__ void scaled_tile(const GroupedParams &p, const TilePlace &at,
                                            u32x4 *lds) {
  typedef ScaledTile<BM, BN, WGM, WGN, STAGES> G;
  constexpr int TI = G::TI, TJ = G::TJ, NM = G::NM, NP = G::NP, PS = G::PS;
  constexpr int LA = G::LA, LB = G::LB, LPT = G::LPT, BK = G::BK;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WGN, wn = wave % WGN;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(TBK_LDS void *)lds;
  const uint32_t wlds = lds0 + wave * 1024u;
  const bool gated = p.act == kActSwiglu;
  const int bn = gated ? 2 * p.n : p.n;
  const int nk = (at.depth + BK - 1) / BK, kfull = at.depth / BK;
  const int krem = at.depth - kfull * BK;
  const int t = wave * 64 + lane;
  const int r0 = t / 8, pc = t % 8; // the lane's row and chunk of a load round
  const int lc = pc ^ G::swizzle(r0);
  const bool past = lc * 16 >= krem; // in the partial last k-tile
  const uint32_t lda = (uint32_t)p.lda, ldb = (uint32_t)p.ldb;

  // ---- A: the offset of each row that the lane loads -----------------------------
  const char *a_ptr = static_cast<const char *>(p.A);
  const char *sa_ptr = reinterpret_cast<const char *>(p.a_scale);
  const uint32_t a_records = (uint32_t)((uint64_t)p.a_rows * lda); // gathered: below kFar
  const int64_t window = p.rows ? 0 : at.row0;                     // else from the tile's row
  auto source_row = [&](int row) -> int64_t {
    const int slot = at.row0 + row;
    const int64_t src = slot < at.row_end ? slot_row(p, slot) : -1;
    return src >= 0 ? src - window : -1;
  };
  uint32_t va[LA];
#pragma unroll
  for (int R = 0; R < LA; ++R) {
    const int64_t src = source_row(r0 + R * G::RPR);
    va[R] = src >= 0 ? (uint32_t)src * lda + (uint32_t)lc * 16u : kFar;
  }
  a_ptr += window * lda;
  sa_ptr += window * nk * 4;
  const uint32_t a_rec = p.rows ? a_records : kFar;

  // ---- B: LDS row r holds column r of the tile; gated: 16 of the gate, then the
  // same 16 of the other half
  const char *b_ptr = static_cast<const char *>(p.B) + (int64_t)at.group * p.stride +
                      (int64_t)at.col0 * ldb;
  const uint32_t b_records = (uint32_t)(bn - at.col0) * ldb;
  const int brow = gated ? (r0 >> 5) * 16 + (r0 & 15) + ((r0 >> 4) & 1) * p.n : r0;
  const uint32_t b_round = (uint32_t)G::RPR * ldb / (gated ? 2u : 1u);
  const uint32_t vb = (uint32_t)brow * ldb + (uint32_t)lc * 16u;

  // ---- scales: every unit's offsets in a table, an entry a lane ------------------
  const int nbt = (bn + 127) / 128;
  const char *sb_ptr =
      reinterpret_cast<const char *>(p.b_scale) + (int64_t)at.group * nbt * nk * 4;
  if (wave < G::UNITS) {
    uint32_t v = kFar;
    if (wave < G::UNITS - 1) {
      const int64_t src = source_row(wave * 64 + lane);
      v = src >= 0 ? (uint32_t)src * (uint32_t)nk * 4u : kFar;
    } else {
      const int c = 8 * lane;
      int col = at.col0 + c;
      bool in = col < p.n && c < BN;
      if (gated) {
        col = at.col0 + (c >> 5) * 16 + (c & 15);
        in = col < p.n && c < BN;
        col += ((c >> 4) & 1) * p.n;
      }
      v = in ? (uint32_t)(col / 128) * (uint32_t)nk * 4u : kFar;
    }
    *(TBK_LDS uint32_t *)(uintptr_t)(lds0 + G::TABLE + t * 4u) = v;
  }
  // Step x: in phase x % 4, units x % 4 and x % 4 + 4 of k-tiles 4 (x / 4) .. + 3, a
  // wave each. The last step of a group of four k-tiles, 4 g + 3, is the last load of
  // k-tile 4 g: issued before the barrier that ends the wait for that k-tile (the
  // static_assert on its slot), waited for with it and read right behind. So
  // STAGES - 1 barriers lie between, one with two stages: no step may come later.
  // The group whose place the first step takes was read before the barrier that this
  // step is issued behind.
  auto load_scales = [&](int x) {
    const int u = x % 4 + (wave / 4) * 4, kt = (x & ~3) + wave % 4;
    const bool live = u < G::UNITS && kt < nk;
    const uint32_t v = *(const TBK_LDS uint32_t *)(uintptr_t)(
        lds0 + G::TABLE + (uint32_t)(live ? u : 0) * 256u + lane * 4u);
    const char *q = (u == G::UNITS - 1 ? sb_ptr : sa_ptr) + (live ? (int64_t)kt * 4 : 0);
    load_lds4(rsrc_dwords(q, live ? kFar : 0u),
              lds0 + (live ? G::SCALES + (uint32_t)(kt % G::RING) * G::KT_BYTES + u * 256u
                           : (uint32_t)G::SPARE),
              v);
  };

  auto load = [&](int kt, auto st_c, auto l_c) {
    constexpr int ST = decltype(st_c)::value, L = decltype(l_c)::value;
    const bool live = kt < nk;
    if constexpr (L < LA) {
      const uint32_t v = kt == kfull && past ? kFar : va[L];
      load_lds16_at<ST * G::STAGE + L * G::NW * 1024>(rsrc_dwords(a_ptr, live ? a_rec : 0u), wlds,
                                                      v, live ? (uint32_t)kt * BK : 0u);
    } else if constexpr (L < LA + LB) {
      constexpr int R = L - LA;
      const uint32_t v = kt == kfull && past ? kOob : vb;
      load_lds16_at<ST * G::STAGE + G::A_BYTES + R * G::NW * 1024>(
          rsrc_dwords(b_ptr, live ? b_records : 0u), wlds, v,
          live ? (uint32_t)kt * BK + (uint32_t)R * b_round : 0u);
    } else {
      load_scales(kt + 3);
    }
  };

  // ---- fragments --------------------------------------------------------------------
  const int g = lane >> 4, l16 = lane & 15;
  uint32_t a_base[2], b_base[2]; // per half of the fragment
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int ra = wm * G::WTM + l16, rb = wn * G::WTN + l16;
    a_base[h] = lds0 + ra * BK + (((4 * h + g) ^ G::swizzle(ra)) * 16);
    b_base[h] = lds0 + G::A_BYTES + rb * BK + (((4 * h + g) ^ G::swizzle(rb)) * 16);
  }
  const uint32_t sa_base = lds0 + G::SCALES + (wm * G::WTM + l16) * 4;
  const uint32_t sb_base = lds0 + G::SCALES + BM * 4 + (wn * G::WTN + 4 * g) / 8 * 4;
  // where the scales of this k-tile and of the next are in their ring
  uint32_t here = 0, next = G::KT_BYTES;
  f32x4 acc[TI][TJ];
  i32x8 fa[2][2], fb[TJ]; // [buffer][row of the pair], [column]
  float sa[2][2], sb[STAGES][TJ];
  auto lds128 = [](uint32_t a) { return *(const TBK_LDS i32x4 *)(uintptr_t)a; };
  auto lds32 = [](uint32_t a) { return *(const TBK_LDS float *)(uintptr_t)a; };
  // read q of pair pr (stage st, buffer pr % 2): 4 halves, then 2 scales
  auto read_a = [&](auto st_c, auto pr_c, auto q_c, uint32_t scales) {
    constexpr int ST = decltype(st_c)::value, PR = decltype(pr_c)::value;
    constexpr int Q = decltype(q_c)::value;
    if constexpr (Q < 4 && Q % 2 == 0)
      fa[PR % 2][Q / 2].lo = lds128(a_base[0] + ST * G::STAGE + (2 * PR + Q / 2) * 16 * BK);
    else if constexpr (Q < 4)
      fa[PR % 2][Q / 2].hi = lds128(a_base[1] + ST * G::STAGE + (2 * PR + Q / 2) * 16 * BK);
    else
      sa[PR % 2][Q - 4] = lds32(sa_base + scales + (2 * PR + Q - 4) * 64);
  };
  auto read_b = [&](auto st_c, auto j_c, uint32_t scales) {
    constexpr int ST = decltype(st_c)::value, J = decltype(j_c)::value;
    fb[J].lo = lds128(b_base[0] + ST * G::STAGE + J * 16 * BK);
    fb[J].hi = lds128(b_base[1] + ST * G::STAGE + J * 16 * BK);
    sb[ST][J] = lds32(sb_base + scales + J * 8);
  };
  auto barrier = [&]() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // the MFMAs' results on their way to the accumulators
  constexpr int RING = 4;
  f32x4 res[RING];
  float scale[RING];
  auto add = [&](int m) { // tile m of a k-tile
    const int i = 2 * (m / PS) + (m & 1), j = (m % PS) / 2;
    asm volatile("" : "+v"(res[m % RING])); // not before the MFMAs issued by now
#pragma unroll
    for (int e = 0; e < 4; ++e)
      acc[i][j][e] = __builtin_fmaf(res[m % RING][e], scale[m % RING], acc[i][j][e]);
    asm volatile("" : "+v"(acc[i][j])); // nor later than here
  };
  using Z = std::integral_constant<int, 0>;
  // one k-tile in stage ST: from its first slot to its last
  auto ktile = [&](int kt, auto st_c) {
    constexpr int ST = decltype(st_c)::value;
    using NEXT = std::integral_constant<int, (ST + 1) % STAGES>;
    using BEFORE = std::integral_constant<int, (ST + STAGES - 1) % STAGES>;
    static_for<NM>([&](auto m_c) {
      constexpr int M = decltype(m_c)::value;
      constexpr int PR = M / PS, S = M % PS, J = S / 2, I = M & 1;
      if constexpr (M == (NP - 1) * PS) {
        // the k-tile's fragments are all in registers; the next has landed
        wait_vmcnt_lgkm0<(STAGES - 2) * LPT>();
        barrier();
      }
      mfma_f8(res[M % RING], fb[J], fa[PR % 2][I]);
      scale[M % RING] = sa[PR % 2][I] * sb[ST][J];
      if constexpr (M >= RING - 1)
        add(M - (RING - 1));
      // the next pair: two reads in every slot from the second on (of the next
      // k-tile behind the barrier)
      if constexpr (S >= 1 && S <= 3) {
        constexpr int Q = 2 * (S - 1);
        using Q0 = std::integral_constant<int, Q>;
        using Q1 = std::integral_constant<int, Q + 1>;
        if constexpr (PR + 1 < NP) {
          using P1 = std::integral_constant<int, PR + 1>;
          read_a(st_c, P1{}, Q0{}, here);
          read_a(st_c, P1{}, Q1{}, here);
        } else {
          read_a(NEXT{}, Z{}, Q0{}, next);
          read_a(NEXT{}, Z{}, Q1{}, next);
        }
      }
      // B's fragments of the next k-tile, two slots after their last use
      if constexpr (PR == NP - 1 && S >= 3 && I == 1)
        read_b(NEXT{}, std::integral_constant<int, J - 1>{}, next);
      if constexpr (M == 1)
        read_b(st_c, std::integral_constant<int, TJ - 1>{}, here);
      // refill: behind the barrier k-tile kt + STAGES into this stage, which goes on
      // in the next k-tile's slots (here for the stage before)
      constexpr int BODY = M >= (NP - 1) * PS ? M - (NP - 1) * PS : M + PS;
      static_for<LPT>([&](auto l_c) {
        if constexpr (G::load_slot(decltype(l_c)::value) == BODY) {
          if constexpr (M >= (NP - 1) * PS)
            load(kt + STAGES, st_c, l_c);
          else
            load(kt + STAGES - 1, BEFORE{}, l_c);
        }
      });
      __builtin_amdgcn_sched_barrier(0);
    });
    // the last results: each MFMA behind them is done before it is read
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7");
#pragma unroll
    for (int m = NM - (RING - 1); m < NM; ++m)
      add(m);
    here = next;
    next = next == (G::RING - 1) * G::KT_BYTES ? 0u : next + G::KT_BYTES;
  };

  // ---- prologue: all k-tiles of the ring, of the last one what the first k-tile's
  // slots do not load
  __syncthreads(); // the table
  for (int x = 0; x < 3; ++x)
    load_scales(x); // step 3 comes with k-tile 0
  static_for<STAGES>([&](auto st_c) {
    static_for<LPT>([&](auto l_c) {
      if constexpr (decltype(st_c)::value < STAGES - 1 ||
                    G::load_slot(decltype(l_c)::value) < PS)
        load(decltype(st_c)::value, st_c, l_c);
    });
  });
#pragma unroll
  for (int i = 0; i < TI; ++i)
#pragma unroll
    for (int j = 0; j < TJ; ++j)
      acc[i][j] = (f32x4){};
  constexpr int AHEAD = [] {
    int c = 0;
    for (int l = 0; l < LPT; ++l)
      c += G::load_slot(l) < PS;
    return c;
  }();
  wait_vmcnt<(STAGES - 2) * LPT + AHEAD>();
  barrier();
  static_for<6>([&](auto q_c) { read_a(Z{}, Z{}, q_c, 0u); });
  static_for<TJ - 1>([&](auto j_c) { read_b(Z{}, j_c, 0u); });
  for (int kt = 0; kt < nk; kt += STAGES)
    static_for<STAGES>([&](auto st_c) {
      if (kt + decltype(st_c)::value < nk)
        ktile(kt + decltype(st_c)::value, st_c);
    });
  wait_vmcnt_lgkm0<0>(); // the loads and reads past the end have landed too
  barrier();

  TBK_LDS char *wl = (TBK_LDS char *)(TBK_LDS void *)lds + wave * G::EPI_REGION;
  auto variant = [&](auto act_c) {
    grouped_store<G, TC, decltype(act_c)::value, false, false>(p, at, acc, wl, wm, wn);
  };
  switch (p.act) {
  case 1: variant(std::integral_constant<int, 1>{}); break;
  case 2: variant(std::integral_constant<int, 2>{}); break;
  case 3: variant(std::integral_constant<int, 3>{}); break;
  case 4: variant(std::integral_constant<int, 4>{}); break;
  default: variant(std::integral_constant<int, 0>{}); break;
  }
}

template <int TC, int BM, int BN, int WGM, int WGN, int STAGES>
__global__ __launch_bounds__(WGM *WGN * 64, (WGM * WGN + 3) / 4) void scaled_rows(GroupedParams p,
                                                                                  int tiles_n) {
  typedef ScaledTile<BM, BN, WGM, WGN, STAGES> G;
  __shared__ u32x4 lds[G::LDS_BYTES / 16];
  TilePlace at;
  if (rows_place(p, blockIdx.x, BM, p.act == kActSwiglu ? BN / 2 : BN, tiles_n, at))
    scaled_tile<TC, BM, BN, WGM, WGN, STAGES>(p, at, lds);
}

} // namespace tbk
