// Grouped products of kind rows where the groups have few rows each (single
// tokens, decoding steps): bound by reading each group's weights once.
//
// A workgroup takes 16 RT rows of one group and a run of columns; its waves
// share the depth, a chunk each in turn, and their sums meet in LDS at the end.
// Weights go straight from memory to registers, several chunks ahead, with no
// LDS and no barrier on the way:
//  * stored n x k: lane l loads 16 bytes of column l % 16 at depth 8 (l / 16),
//    which is a fragment of the matrix instruction as it stands;
//  * stored k x n: lane l loads 8 columns (block l % 16) of each of 8 rows
//    (block l / 16 of 4): 32 x 128 of the weights in 8 loads of 4 whole
//    256-byte pieces. One byte permute per register turns the 8 x 8 values that
//    a lane holds into 8 fragments, column 8 (l % 16) + j for the j-th.
// One token's 8 of 128 experts, 4096 x 2048 bf16 n x k: 28-30 us, 4.5-4.8 TB/s of
// weights (64 workgroups of 128 x 128 tiles 54 us); 13 tokens, 6 of 64, 2048 x 2048 f16 k x
// n: 62-68 us, 5.7-6.3 TB/s with the last-level cache; e4m3, 16 x 8192 x 4096: 13 us, four
// chunks a wave, so latency.
// Rows of A that a tile lacks read nothing. Products and sums are f32 (e4m3: the
// instruction's own sums within a block, scaled_tile.h says how exact); the
// waves' sums are added in wave order, so results do not vary from run to run.
#pragma once

#include "experts_device.h"

namespace tbk {

typedef int fr_i32x8 __attribute__((ext_vector_type(8)));
typedef int fr_i32x4 __attribute__((ext_vector_type(4)));

constexpr int kFewWaves = 8;
constexpr uint32_t kFewFar = 0xF0000000u; // past every record

// f32 sums of a wave for 16 rows, staged for the other waves: row stride in
// floats, padded so that 16 rows start in different banks
constexpr int few_stride(int cols) { return cols + 4; }

// chunks in flight per wave: what the registers hold
constexpr int few_ahead(int fit) { return fit < 2 ? 2 : (fit > 4 ? 4 : fit); }

template <int T>
__device__ __forceinline__ f32x4 few_mfma(u32x4 b, u32x4 a, f32x4 c) {
  if constexpr (T == kElemF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, b),
                                                  __builtin_bit_cast(half8, a), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bhalf8, b),
                                                   __builtin_bit_cast(bhalf8, a), c, 0, 0, 0);
}

// What a workgroup computes and where A's rows are.
template <int ES, int RT>
struct FewPlace {
  int group, row0, row_end;
  __amdgpu_buffer_rsrc_t a, b;
  uint32_t arow[RT]; // the lane's row (l % 16) of each row tile, kFewFar: none
  int64_t src[RT];   // its row of A, -1: none
  __device__ __forceinline__ bool find(const GroupedParams &p, int tile) {
    const GroupTile g = group_tile(p, 16 * RT, tile);
    if (g.group < 0)
      return false;
    group = g.group, row0 = g.begin, row_end = g.end;
    const int64_t window = p.rows ? 0 : row0;
    const int l16 = threadIdx.x & 15;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int slot = row0 + 16 * i + l16;
      src[i] = slot < row_end ? slot_row(p, slot) : -1;
      arow[i] = src[i] >= 0 ? (uint32_t)((src[i] - window) * p.lda * ES) : kFewFar;
    }
    a = make_rsrc(static_cast<const char *>(p.A) + window * p.lda * ES, kFewFar);
    b = make_rsrc(static_cast<const char *>(p.B) + group * p.stride * ES, kOob);
    return true;
  }
};

// The waves' sums of row tile i (COLS columns, the gated half second) to C.
// `stage`: kFewWaves x 16 x few_stride(COLS) floats, which this wave has written
// its own part of. col0: the first result column.
template <int TC, int COLS>
__device__ __forceinline__ void few_store(const GroupedParams &p, const float *stage, int row0,
                                          int row_end, int col0) {
  constexpr int LD = few_stride(COLS);
  const bool gated = p.act == kActSwiglu;
  const int width = gated ? COLS / 2 : COLS;
  __syncthreads();
  for (int q = threadIdx.x; q < 16 * width / 4; q += kFewWaves * 64) {
    const int r = q / (width / 4), c = q % (width / 4) * 4;
    auto total = [&](int col) {
      f32x4 s = *reinterpret_cast<const f32x4 *>(stage + r * LD + col);
#pragma unroll
      for (int w = 1; w < kFewWaves; ++w)
        s += *reinterpret_cast<const f32x4 *>(stage + (w * 16 + r) * LD + col);
      return s;
    };
    f32x4 v = total(c);
    if (gated) {
      const f32x4 u = total(width + c);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[e] = epi_activation(v[e], 3) * u[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[e] = epi_activation(v[e], p.act);
    }
    if (row0 + r < row_end && col0 + c < p.n) {
      const int64_t at = (int64_t)(row0 + r) * p.ldc + col0 + c;
      if constexpr (TC == kElemF32) {
        *reinterpret_cast<f32x4 *>(static_cast<float *>(p.C) + at) = v;
      } else {
        store4<TC>(p.C, at, v);
      }
    }
  }
  __syncthreads();
}

// ---- weights k x n -----------------------------------------------------------------
template <int T, int TC, int RT>
__global__ __launch_bounds__(kFewWaves * 64, RT > 2 ? 1 : 2) void few_rows_kn(GroupedParams p,
                                                                             int tiles_n) {
  constexpr int COLS = 128, CK = 32;      // columns; depth of a chunk
  constexpr int AHEAD = RT > 2 ? 2 : 3;   // chunks in flight per wave
  __shared__ float stage[kFewWaves * 16 * few_stride(COLS)];
  FewPlace<2, RT> at;
  if (!at.find(p, blockIdx.x / tiles_n))
    return;
  const bool gated = p.act == kActSwiglu;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col0 = (blockIdx.x % tiles_n) * (gated ? COLS / 2 : COLS);
  // the lane's 8 columns; gated: blocks 0..7 of the gate, 8..15 of the other half
  int col = col0 + 8 * (gated ? l16 & 7 : l16);
  const bool in = col < p.n;
  col += gated && l16 >= 8 ? p.n : 0;
  const uint32_t ldb2 = (uint32_t)p.ldb * 2u;
  const uint32_t vb = (uint32_t)(8 * g) * ldb2 + (uint32_t)col * 2u;
  const int chunks = (p.k + CK - 1) / CK;
  u32x4 b[AHEAD][8], a[AHEAD][RT];
  auto load = [&](int u, int chunk) {
    // whole blocks of 8 of the depth: k is a multiple of 8
    const bool live = chunk * CK + 8 * g < p.k;
    const uint32_t v = live && in ? vb + (uint32_t)chunk * CK * ldb2 : kFewFar;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      b[u][i] = __builtin_amdgcn_raw_buffer_load_b128(at.b, v + (uint32_t)i * ldb2, 0, 0);
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const uint32_t x = live && at.arow[i] != kFewFar
                             ? at.arow[i] + (uint32_t)(chunk * CK + 8 * g) * 2u
                             : kFewFar;
      a[u][i] = __builtin_amdgcn_raw_buffer_load_b128(at.a, x, 0, 0);
    }
  };
  f32x4 acc[RT][8] = {};
#pragma unroll
  for (int u = 0; u < AHEAD; ++u)
    load(u, wave + u * kFewWaves);
  for (int c = wave; c < chunks; c += AHEAD * kFewWaves) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        u32x4 f; // column j of the lane's block, its 8 rows
        const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          f[q] = __builtin_amdgcn_perm(b[u][2 * q + 1][j / 2], b[u][2 * q][j / 2], sel);
#pragma unroll
        for (int i = 0; i < RT; ++i)
          acc[i][j] = few_mfma<T>(f, a[u][i], acc[i][j]);
      }
      load(u, c + (u + AHEAD) * kFewWaves);
    }
  }
  // lane l: row l % 16, columns 32 (l / 16) + 8 r + j of acc[.][j][r]
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    float *mine = stage + (wave * 16 + l16) * few_stride(COLS) + 32 * g;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      *reinterpret_cast<f32x4 *>(mine + 8 * r) =
          (f32x4){acc[i][0][r], acc[i][1][r], acc[i][2][r], acc[i][3][r]};
      *reinterpret_cast<f32x4 *>(mine + 8 * r + 4) =
          (f32x4){acc[i][4][r], acc[i][5][r], acc[i][6][r], acc[i][7][r]};
    }
    few_store<TC, COLS>(p, stage, at.row0 + 16 * i, at.row_end, col0);
  }
}

// ---- weights n x k -----------------------------------------------------------------
// NB: fragments of 16 columns; gated: the second half of them is the other half's
template <int NB>
__device__ __forceinline__ int few_column(const GroupedParams &p, int col0, int s, int l16,
                                          bool gated, bool &in) {
  const int half = gated ? NB / 2 : NB;
  const int col = col0 + 16 * (s % half) + l16;
  in = col < p.n;
  return col + (gated && s >= half ? p.n : 0);
}

template <int T, int TC, int RT, int NB>
__global__ __launch_bounds__(kFewWaves * 64, RT > 2 ? 1 : 2) void few_rows_nk(GroupedParams p,
                                                                             int tiles_n) {
  constexpr int COLS = 16 * NB, CK = 64; // two MFMAs deep: whole 128-byte lines
  constexpr int AHEAD = few_ahead(144 / (8 * (NB + RT)));
  __shared__ float stage[kFewWaves * 16 * few_stride(COLS)];
  FewPlace<2, RT> at;
  if (!at.find(p, blockIdx.x / tiles_n))
    return;
  const bool gated = p.act == kActSwiglu;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col0 = (blockIdx.x % tiles_n) * (gated ? COLS / 2 : COLS);
  uint32_t vb[NB];
#pragma unroll
  for (int s = 0; s < NB; ++s) {
    bool in;
    const int col = few_column<NB>(p, col0, s, l16, gated, in);
    vb[s] = in ? (uint32_t)col * (uint32_t)p.ldb * 2u : kFewFar;
  }
  const int chunks = (p.k + CK - 1) / CK;
  u32x4 b[AHEAD][2][NB], a[AHEAD][2][RT];
  auto load = [&](int u, int chunk) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = chunk * CK + 32 * h + 8 * g;
      const bool live = k < p.k;
      const uint32_t off = (uint32_t)k * 2u;
#pragma unroll
      for (int s = 0; s < NB; ++s)
        b[u][h][s] = __builtin_amdgcn_raw_buffer_load_b128(
            at.b, live && vb[s] != kFewFar ? vb[s] + off : kFewFar, 0, 0);
#pragma unroll
      for (int i = 0; i < RT; ++i)
        a[u][h][i] = __builtin_amdgcn_raw_buffer_load_b128(
            at.a, live && at.arow[i] != kFewFar ? at.arow[i] + off : kFewFar, 0, 0);
    }
  };
  f32x4 acc[RT][NB] = {};
#pragma unroll
  for (int u = 0; u < AHEAD; ++u)
    load(u, wave + u * kFewWaves);
  for (int c = wave; c < chunks; c += AHEAD * kFewWaves) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int s = 0; s < NB; ++s)
#pragma unroll
          for (int i = 0; i < RT; ++i)
            acc[i][s] = few_mfma<T>(b[u][h][s], a[u][h][i], acc[i][s]);
      load(u, c + (u + AHEAD) * kFewWaves);
    }
  }
  // lane l: row l % 16, columns 16 s + 4 (l / 16) + r of acc[.][s][r]
#pragma unroll
  for (int i = 0; i < RT; ++i) {
#pragma unroll
    for (int s = 0; s < NB; ++s)
      *reinterpret_cast<f32x4 *>(stage + (wave * 16 + l16) * few_stride(COLS) + 16 * s + 4 * g) =
          acc[i][s];
    few_store<TC, COLS>(p, stage, at.row0 + 16 * i, at.row_end, col0);
  }
}

// ---- e4m3 weights n x k, block scales -------------------------------------------------
// A chunk is one block of 128 of the depth: one MFMA from a zero accumulator per
// fragment, scaled and added.
template <int TC, int RT, int NB>
__global__ __launch_bounds__(kFewWaves * 64, RT > 2 ? 1 : 2) void few_rows_f8(GroupedParams p,
                                                                             int tiles_n) {
  constexpr int COLS = 16 * NB, CK = 128;
  constexpr int AHEAD = few_ahead(120 / (8 * (NB + RT)));
  __shared__ float stage[kFewWaves * 16 * few_stride(COLS)];
  FewPlace<1, RT> at;
  if (!at.find(p, blockIdx.x / tiles_n))
    return;
  const bool gated = p.act == kActSwiglu;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col0 = (blockIdx.x % tiles_n) * (gated ? COLS / 2 : COLS);
  const int chunks = (p.k + CK - 1) / CK;
  const int nbt = ((gated ? 2 * p.n : p.n) + 127) / 128;
  const float *b_scale = p.b_scale + (int64_t)at.group * nbt * chunks;
  uint32_t vb[NB], vsb[NB], vsa[RT];
#pragma unroll
  for (int s = 0; s < NB; ++s) {
    bool in;
    int col = few_column<NB>(p, col0, s, l16, gated, in);
    vb[s] = in ? (uint32_t)col * (uint32_t)p.ldb : kFewFar;
    // the scale of the columns that the lane holds results of (four in a row
    // within a block)
    col = few_column<NB>(p, col0, s, 4 * g, gated, in);
    vsb[s] = in ? (uint32_t)(col / 128) * (uint32_t)chunks * 4u : kFewFar;
  }
  const __amdgpu_buffer_rsrc_t rsb = make_rsrc(b_scale, (uint32_t)nbt * (uint32_t)chunks * 4u);
  const int64_t window = p.rows ? 0 : at.row0;
  const __amdgpu_buffer_rsrc_t rsa = make_rsrc(p.a_scale + window * chunks, kFewFar);
#pragma unroll
  for (int i = 0; i < RT; ++i)
    vsa[i] = at.src[i] >= 0 ? (uint32_t)(at.src[i] - window) * (uint32_t)chunks * 4u : kFewFar;
  fr_i32x8 b[AHEAD][NB], a[AHEAD][RT];
  float sa[AHEAD][RT], sb[AHEAD][NB];
  auto load16 = [](const __amdgpu_buffer_rsrc_t &r, uint32_t v) {
    return __builtin_bit_cast(fr_i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, v, 0, 0));
  };
  auto load4 = [](const __amdgpu_buffer_rsrc_t &r, uint32_t v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, v, 0, 0));
  };
  auto load = [&](int u, int chunk) {
    const int k = chunk * CK + 16 * g; // and 64 further on
    const bool live0 = k < p.k, live1 = k + 64 < p.k, any = chunk < chunks;
#pragma unroll
    for (int s = 0; s < NB; ++s) {
      const bool in = vb[s] != kFewFar;
      b[u][s].lo = load16(at.b, in && live0 ? vb[s] + (uint32_t)k : kFewFar);
      b[u][s].hi = load16(at.b, in && live1 ? vb[s] + (uint32_t)k + 64u : kFewFar);
      sb[u][s] = load4(rsb, any && vsb[s] != kFewFar ? vsb[s] + (uint32_t)chunk * 4u : kFewFar);
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const bool in = at.arow[i] != kFewFar;
      a[u][i].lo = load16(at.a, in && live0 ? at.arow[i] + (uint32_t)k : kFewFar);
      a[u][i].hi = load16(at.a, in && live1 ? at.arow[i] + (uint32_t)k + 64u : kFewFar);
      sa[u][i] = load4(rsa, any && in ? vsa[i] + (uint32_t)chunk * 4u : kFewFar);
    }
  };
  f32x4 acc[RT][NB] = {};
#pragma unroll
  for (int u = 0; u < AHEAD; ++u)
    load(u, wave + u * kFewWaves);
  for (int c = wave; c < chunks; c += AHEAD * kFewWaves) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int s = 0; s < NB; ++s) {
          const f32x4 d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
              b[u][s], a[u][i], (f32x4){}, 0, 0, 0, 0, 0, 0);
          const float f = sa[u][i] * sb[u][s];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[i][s][e] = __builtin_fmaf(d[e], f, acc[i][s][e]);
        }
      load(u, c + (u + AHEAD) * kFewWaves);
    }
  }
#pragma unroll
  for (int i = 0; i < RT; ++i) {
#pragma unroll
    for (int s = 0; s < NB; ++s)
      *reinterpret_cast<f32x4 *>(stage + (wave * 16 + l16) * few_stride(COLS) + 16 * s + 4 * g) =
          acc[i][s];
    few_store<TC, COLS>(p, stage, at.row0 + 16 * i, at.row_end, col0);
  }
}

} // namespace tbk
