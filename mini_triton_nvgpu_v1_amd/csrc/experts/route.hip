// The router of a mixture-of-experts layer: each token's top_k experts, their
// softmax weights and the stable order of the (token, expert) pairs by expert;
// and the gradient of the logits.
//
// For a token's logits x (experts e): the chosen set S holds the top_k largest
// x_e, ties to the lowest e; an expert at -inf or NaN is never chosen. Weights
// are the softmax over S (renormalize) or over all experts:
//   w_e = exp(x_e - m) / sum exp(x_f - m),  m the largest logit,
// in f32 whatever the logits' type. Gradient, with g the weights' gradients on
// S and 0 elsewhere, p the same softmax (0 outside S when renormalized):
//   dx_e = p_e (g_e - sum_f g_f w_f).
//
// Order: pair (t, j) goes to its expert's run, after the expert's pairs of all
// earlier tokens. A token names an expert at most once, so the pair's rank
// within 64 tokens is the number of earlier tokens among them that name the
// expert: one bit a token in a 64-bit mask per expert, set with LDS atomics
// (OR: their order does not matter), counted with popcounts.
//
// A token's experts lie over 16 lanes, so a wave chooses for 4 tokens at a
// time: per choice a scan of the lane's own experts and a 4-step exchange.
//
// Bound by latency, not by its few megabytes: the choices of a token depend on
// each other. Up to 256 tokens one workgroup does all of it (13 tokens x 64
// experts, top 6: 4.5 us); beyond, one launch chooses and counts and a second
// places, since the places need every block's counts (16384 x 128 f32, top 8:
// 10.0-10.4 + 6.5 us, the gradient 7.2-7.6).
#include "experts_device.h"

#include <math.h>

namespace tbk {

namespace {

constexpr int kSmallTokens = 256; // tokens that one workgroup routes by itself
constexpr int kTokenBlock = 64;   // tokens of a workgroup otherwise
constexpr int kSumBlocks = 512;   // blocks whose counts the placing step sums

template <int T> struct RouteElem { typedef float type; };
template <> struct RouteElem<kElemF16> { typedef _Float16 type; };
template <> struct RouteElem<kElemBF16> { typedef __bf16 type; };

// e^x for x <= 0 (a difference from the largest logit): 2^(x log2 e) with the
// hardware's exponential, the product's rounding error put back, 2 units in the
// last place. 0 below -150; NaN counts as below (the callers look for infinities).
__device__ __forceinline__ float exp_below(float x) {
  const float y = fmaxf(x, -150.f), L = 1.44269504088896341f;
  const float t = y * L;
  // log2 e - L = 1.9259629911e-8; 2^(t + d) = 2^t (1 + d ln 2) for a small d
  const float d = __builtin_fmaf(y, 1.9259629911e-8f, __builtin_fmaf(y, L, -t));
  const float e = __builtin_amdgcn_exp2f(t);
  return __builtin_fmaf(e, d * 0.69314718055994531f, e);
}

// The value of another lane of the 16 that hold a token: neighbours, pairs,
// halves of 8 and of 16 mirrored, in the vector unit's own lane moves. After
// each step the lanes that were joined hold the same, so mirrored is as good as
// swapped.
template <int STEP>
__device__ __forceinline__ int other_lane(int v) {
  constexpr int CTRL = STEP == 0 ? 0xB1 : STEP == 1 ? 0x4E : STEP == 2 ? 0x141 : 0x140;
  return __builtin_amdgcn_update_dpp(v, v, CTRL, 0xf, 0xf, false);
}
template <int STEP>
__device__ __forceinline__ float other_lane(float v) {
  return __builtin_bit_cast(float, other_lane<STEP>(__builtin_bit_cast(int, v)));
}
// sum and maximum over the 16 lanes of a token
__device__ __forceinline__ float row_max(float v) {
  static_for<4>([&](auto d) { v = fmaxf(v, other_lane<decltype(d)::value>(v)); });
  return v;
}
__device__ __forceinline__ float row_sum(float v) {
  static_for<4>([&](auto d) { v += other_lane<decltype(d)::value>(v); });
  return v;
}

// Elements of a vector access: 16 bytes, or the lane's whole share if that is less.
template <int T, int EPL>
constexpr int kVec = (T == kElemF32 ? 4 : 8) < EPL ? (T == kElemF32 ? 4 : 8) : EPL;

// Whether rows of `ld` elements of type T from `p` take vector accesses.
template <int T, int EPL>
__device__ __forceinline__ bool vectors(const void *p, int64_t ld) {
  constexpr int BYTES = kVec<T, EPL> * (T == kElemF32 ? 4 : 2);
  return reinterpret_cast<uintptr_t>(p) % BYTES == 0 && ld % kVec<T, EPL> == 0;
}

// The token's logits over its 16 lanes: v[j] is expert EPL (lane % 16) + j, -inf
// past the last expert and for NaN; true if the token has a NaN.
template <int T, int EPL>
__device__ __forceinline__ bool load_logits(const RouteParams &p, int token, float (&v)[EPL]) {
  constexpr int V = kVec<T, EPL>;
  const int e0 = (threadIdx.x & 15) * EPL;
  const int64_t row = (int64_t)token * p.ld;
  const bool vec = vectors<T, EPL>(p.logits, p.ld);
#pragma unroll
  for (int q = 0; q < EPL; q += V) {
    if (vec && token < p.tokens && e0 + q + V <= p.experts) {
      typedef typename RouteElem<T>::type E;
      typedef E VE __attribute__((ext_vector_type(V)));
      const VE x = *reinterpret_cast<const VE *>(static_cast<const E *>(p.logits) + row + e0 + q);
#pragma unroll
      for (int j = 0; j < V; ++j)
        v[q + j] = (float)x[j];
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int e = e0 + q + j;
        v[q + j] = token < p.tokens && e < p.experts ? load1<T>(p.logits, row + e) : -INFINITY;
      }
    }
  }
  bool nan = false;
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    nan |= v[j] != v[j];
    v[j] = v[j] != v[j] ? -INFINITY : v[j];
  }
  const uint64_t any = __ballot(nan);
  return (any >> ((threadIdx.x & 63) & ~15)) & 0xffffu;
}

// Chooses for the token of this lane's 16-lane row. Lane j (and j + 16 for
// top_k > 16) ends with choice j: cid (-1: none) and its weight.
template <int T, int EPL>
__device__ __forceinline__ void choose(const RouteParams &p, int token, int (&cid)[2],
                                       float (&cw)[2]) {
  const int l16 = threadIdx.x & 15;
  float v[EPL];
  const bool nan = load_logits<T, EPL>(p, token, v);
  float all = 0.f, m = 0.f;
  float cv[2] = {-INFINITY, -INFINITY};
  cid[0] = cid[1] = -1;
  for (int r = 0; r < p.top_k; ++r) {
    float best = v[0];
    int at = 0;
#pragma unroll
    for (int j = 1; j < EPL; ++j)
      if (v[j] > best) {
        best = v[j];
        at = j;
      }
    at += l16 * EPL;
    static_for<4>([&](auto d) {
      const float ov = other_lane<decltype(d)::value>(best);
      const int oa = other_lane<decltype(d)::value>(at);
      const bool take = ov > best || (ov == best && oa < at);
      best = take ? ov : best;
      at = take ? oa : at;
    });
    if (r == 0) {
      m = best > -INFINITY ? best : 0.f;
      if (!p.renormalize) {
#pragma unroll
        for (int j = 0; j < EPL; ++j)
          all += exp_below(v[j] - m);
      }
    }
    const bool ok = best > -INFINITY;
    if (l16 == (r & 15)) {
      cv[r >> 4] = best;
      cid[r >> 4] = ok ? at : -1;
    }
#pragma unroll
    for (int j = 0; j < EPL; ++j)
      v[j] = at == l16 * EPL + j ? -INFINITY : v[j];
  }
  const float e0 = exp_below(cv[0] - m), e1 = exp_below(cv[1] - m);
  float total = row_sum(p.renormalize ? e0 + e1 : all);
  total = total > 0.f || total != total ? total : 1.f;
  total = nan || m == INFINITY ? NAN : total;
  cw[0] = cid[0] >= 0 ? e0 / total : 0.f;
  cw[1] = cid[1] >= 0 ? e1 / total : 0.f;
}

// One workgroup's tokens [t0, t0 + 64 words): choices, weights, and the masks
// of the experts they name (LDS, words per expert).
template <int T, int EPL>
__device__ __forceinline__ void choose_block(const RouteParams &p, int t0, int words,
                                             unsigned long long *mask) {
  const int l16 = threadIdx.x & 15, group = threadIdx.x >> 4, groups = blockDim.x >> 4;
  for (int i = threadIdx.x; i < p.experts * words; i += blockDim.x)
    mask[i] = 0;
  __syncthreads();
  const int end = min(p.tokens - t0, 64 * words);
  for (int b0 = 0; b0 < end; b0 += groups) {
    const int b = b0 + group; // the same trip count in every wave's lanes
    const int token = b < end ? t0 + b : p.tokens;
    int cid[2];
    float cw[2];
    choose<T, EPL>(p, token, cid, cw);
    if (token >= p.tokens)
      continue;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int j = 16 * h + l16;
      if (j < p.top_k) {
        const int64_t at = (int64_t)token * p.top_k + j;
        p.ids[at] = cid[h];
        p.weights[at] = cw[h];
        if (cid[h] >= 0)
          atomicOr(mask + cid[h] * words + (b >> 6), 1ull << (b & 63));
      }
    }
  }
  __threadfence_block();
  __syncthreads();
}

// exclusive sums of first[0 .. n) in place (n <= 512), by the first wave
__device__ __forceinline__ void exclusive_scan(int *first, int n) {
  if (threadIdx.x < 64) {
    int carry = 0;
    for (int e0 = 0; e0 < n; e0 += 64) {
      const int e = e0 + (int)threadIdx.x;
      const int c = e < n ? first[e] : 0;
      const int upto = wave_scan(c);
      if (e < n)
        first[e] = carry + upto - c;
      carry += last_lane(upto);
    }
    if (threadIdx.x == 0)
      first[n] = carry;
  }
  __syncthreads();
}

// Few tokens: one workgroup does it all.
template <int T, int EPL>
__global__ __launch_bounds__(1024) void route_small(RouteParams p) {
  __shared__ unsigned long long mask[kRouteMaxExperts * (kSmallTokens / 64)];
  __shared__ int first[kRouteMaxExperts + 1];
  const int words = (p.tokens + 63) / 64;
  choose_block<T, EPL>(p, 0, words, mask);
  for (int e = threadIdx.x; e < p.experts; e += blockDim.x) {
    int c = 0;
    for (int w = 0; w < words; ++w)
      c += __popcll(mask[e * words + w]);
    first[e] = c;
  }
  __syncthreads();
  exclusive_scan(first, p.experts);
  for (int e = threadIdx.x; e <= p.experts; e += blockDim.x)
    p.offsets[e] = first[e];
  const int pairs = p.tokens * p.top_k;
  for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
    const int t = i / p.top_k, e = p.ids[i];
    int slot = -1;
    if (e >= 0) {
      slot = first[e];
      for (int w = 0; w < (t >> 6); ++w)
        slot += __popcll(mask[e * words + w]);
      slot += __popcll(mask[e * words + (t >> 6)] & ((1ull << (t & 63)) - 1));
      p.rows[slot] = t;
    }
    p.slots[i] = slot;
  }
  for (int i = first[p.experts] + threadIdx.x; i < pairs; i += blockDim.x)
    p.rows[i] = -1;
}

// Many tokens, step 1: a workgroup's 64 tokens; ranks within them to `slots`,
// its counts per expert to ws[block][expert].
template <int T, int EPL>
__global__ __launch_bounds__(1024) void route_blocks(RouteParams p) {
  __shared__ unsigned long long mask[kRouteMaxExperts];
  const int t0 = blockIdx.x * kTokenBlock;
  choose_block<T, EPL>(p, t0, 1, mask);
  for (int e = threadIdx.x; e < p.experts; e += blockDim.x)
    p.ws[(int64_t)blockIdx.x * p.experts + e] = __popcll(mask[e]);
  const int here = min(p.tokens - t0, kTokenBlock);
  for (int i = threadIdx.x; i < here * p.top_k; i += blockDim.x) {
    const int64_t at = (int64_t)t0 * p.top_k + i;
    const int e = p.ids[at];
    p.slots[at] =
        e < 0 ? -1 : (int)__popcll(mask[e] & ((1ull << (i / p.top_k)) - 1));
  }
}

// Step 2: per expert the exclusive sums of its counts over the blocks, in
// place, and its total. A workgroup takes 64 experts (its lanes) and its 16
// waves a sixteenth of the blocks each.
__global__ __launch_bounds__(1024) void route_scan(RouteParams p, int blocks) {
  __shared__ int part[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int e = blockIdx.x * 64 + lane;
  const int per = (blocks + 15) / 16;
  const int b0 = min(blocks, w * per), b1 = min(blocks, b0 + per);
  int *c = p.ws + (e < p.experts ? e : 0);
  int sum = 0;
#pragma unroll 8
  for (int b = b0; b < b1; ++b)
    sum += c[(int64_t)b * p.experts];
  part[w][lane] = sum;
  __syncthreads();
  int at = 0;
  for (int i = 0; i < w; ++i)
    at += part[i][lane];
  if (e >= p.experts)
    return;
  if (w == 15)
    p.ws[(int64_t)blocks * p.experts + e] = at + sum;
  int b = b0;
  for (; b + 8 <= b1; b += 8) {
    int v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = c[(int64_t)(b + i) * p.experts];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      c[(int64_t)(b + i) * p.experts] = at;
      at += v[i];
    }
  }
  for (; b < b1; ++b) {
    const int v = c[(int64_t)b * p.experts];
    c[(int64_t)b * p.experts] = at;
    at += v;
  }
}

// Step 3: the pairs' slots from the experts' first slots, the blocks' sums and
// the ranks. SUMS: step 2 was left out, and each workgroup sums the counts of all
// blocks itself, and of those before it, its threads a share of the blocks each.
template <bool SUMS>
__global__ __launch_bounds__(1024) void route_place(RouteParams p, int blocks) {
  __shared__ int first[kRouteMaxExperts + 1], before[kRouteMaxExperts];
  __shared__ int part[SUMS ? 2 : 1][SUMS ? 1024 : 1];
  if constexpr (SUMS) {
    const int wide = (p.experts + 63) / 64 * 64, shares = 1024 / wide;
    const int e = threadIdx.x % wide, share = threadIdx.x / wide;
    const int me = blockIdx.x, per = (blocks + shares - 1) / shares;
    int all = 0, mine = 0;
    if (e < p.experts && share < shares) {
      const int *c = p.ws + e;
      const int b1 = min(blocks, (share + 1) * per);
#pragma unroll 8
      for (int b = share * per; b < b1; ++b) {
        const int v = c[(int64_t)b * p.experts];
        all += v;
        mine += b < me ? v : 0;
      }
    }
    part[0][threadIdx.x] = all;
    part[1][threadIdx.x] = mine;
    __syncthreads();
    if (threadIdx.x < p.experts) {
      for (int i = 1; i < shares; ++i) {
        all += part[0][i * wide + threadIdx.x];
        mine += part[1][i * wide + threadIdx.x];
      }
      first[threadIdx.x] = all;
      before[threadIdx.x] = mine;
    }
  } else {
    for (int e = threadIdx.x; e < p.experts; e += blockDim.x) {
      first[e] = p.ws[(int64_t)blocks * p.experts + e];
      before[e] = p.ws[(int64_t)blockIdx.x * p.experts + e];
    }
  }
  __syncthreads();
  exclusive_scan(first, p.experts);
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e <= p.experts; e += blockDim.x)
      p.offsets[e] = first[e];
  const int t0 = blockIdx.x * kTokenBlock;
  const int here = min(p.tokens - t0, kTokenBlock);
  const int used = first[p.experts];
  for (int i = threadIdx.x; i < here * p.top_k; i += blockDim.x) {
    const int64_t at = (int64_t)t0 * p.top_k + i;
    const int e = p.ids[at];
    if (e >= 0) {
      const int slot = p.slots[at] + first[e] + before[e];
      p.slots[at] = slot;
      p.rows[slot] = t0 + i / p.top_k;
    }
    if (at >= used) // places no pair takes
      p.rows[at] = -1;
  }
}

template <int T, int EPL>
__global__ __launch_bounds__(256) void route_backward_kernel(RouteParams p) {
  const int l16 = threadIdx.x & 15;
  const int token = blockIdx.x * 16 + (threadIdx.x >> 4);
  float v[EPL], g[EPL];
  const bool nan = load_logits<T, EPL>(p, token, v);
  const bool live = token < p.tokens;
  // choice j of the token: lane j % 16, register j / 16
  int cid[2];
  float cg[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int j = 16 * h + l16;
    const bool has = live && j < p.top_k;
    const int64_t at = (int64_t)(live ? token : 0) * p.top_k + (has ? j : 0);
    cid[h] = has ? p.ids[at] : -1;
    cg[h] = has ? p.dweights[at] : 0.f;
  }
  uint32_t shown = 0; // bit j: the lane's expert j is chosen
#pragma unroll
  for (int j = 0; j < EPL; ++j)
    g[j] = 0.f;
  // each choice to the token's 16 lanes (lane moves: row_newbcast)
  static_for<32>([&](auto r_c) {
    constexpr int R = decltype(r_c)::value, H = R / 16, CTRL = 0x150 + R % 16;
    if (R < p.top_k) {
      const int id = __builtin_amdgcn_update_dpp(cid[H], cid[H], CTRL, 0xf, 0xf, false);
      const float d = __builtin_bit_cast(
          float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, cg[H]),
                                             __builtin_bit_cast(int, cg[H]), CTRL, 0xf, 0xf,
                                             false));
      const int mine = id >= 0 && id / EPL == l16 ? id % EPL : -1;
#pragma unroll
      for (int j = 0; j < EPL; ++j)
        g[j] = mine == j ? d : g[j];
      shown |= mine >= 0 ? 1u << mine : 0u;
    }
  });
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    if (p.renormalize && !((shown >> j) & 1))
      v[j] = -INFINITY;
    m = fmaxf(m, v[j]);
  }
  m = row_max(m);
  m = m > -INFINITY ? m : 0.f;
  float total = 0.f, gw = 0.f;
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    v[j] = exp_below(v[j] - m);
    total += v[j];
    gw += g[j] * v[j];
  }
  total = row_sum(total);
  total = total > 0.f || total != total ? total : 1.f;
  total = nan || m == INFINITY ? NAN : total;
  const float inv = 1.f / total;
  gw = row_sum(gw) * inv;
  if (!live)
    return;
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    // an expert outside the softmax gets 0, whatever the token's others are
    const bool in = !p.renormalize || ((shown >> j) & 1);
    v[j] = in ? v[j] * inv * (g[j] - gw) : 0.f;
  }
  constexpr int V = kVec<T, EPL>;
  typedef typename RouteElem<T>::type E;
  typedef E VE __attribute__((ext_vector_type(V)));
  const int e0 = l16 * EPL;
  E *row = static_cast<E *>(p.dlogits) + (int64_t)token * p.ldd + e0;
  const bool vec = vectors<T, EPL>(p.dlogits, p.ldd);
#pragma unroll
  for (int q = 0; q < EPL; q += V) {
    if (vec && e0 + q + V <= p.experts) {
      VE x;
#pragma unroll
      for (int j = 0; j < V; ++j)
        x[j] = (E)v[q + j];
      *reinterpret_cast<VE *>(row + q) = x;
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (e0 + q + j < p.experts)
          row[q + j] = (E)v[q + j];
    }
  }
}

template <int T, int EPL>
hipError_t route_t(const RouteParams &p, hipStream_t s) {
  if (p.tokens <= kSmallTokens) {
    // 16 lanes a token, whole waves
    const int threads = min(1024, (p.tokens * 16 + 63) / 64 * 64);
    hipLaunchKernelGGL((route_small<T, EPL>), dim3(1), dim3(max(256, threads)), 0, s, p);
    return hipGetLastError();
  }
  const int blocks = (p.tokens + kTokenBlock - 1) / kTokenBlock;
  hipLaunchKernelGGL((route_blocks<T, EPL>), dim3(blocks), dim3(1024), 0, s, p);
  // up to 512 blocks the last step sums them itself (its reads are at most 1 MB a
  // workgroup): one launch less
  if (blocks <= kSumBlocks) {
    hipLaunchKernelGGL(route_place<true>, dim3(blocks), dim3(1024), 0, s, p, blocks);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(route_scan, dim3((p.experts + 63) / 64), dim3(1024), 0, s, p, blocks);
  hipLaunchKernelGGL(route_place<false>, dim3(blocks), dim3(256), 0, s, p, blocks);
  return hipGetLastError();
}

template <int T, int EPL>
hipError_t backward_t(const RouteParams &p, hipStream_t s) {
  hipLaunchKernelGGL((route_backward_kernel<T, EPL>), dim3((p.tokens + 15) / 16), dim3(256), 0,
                     s, p);
  return hipGetLastError();
}

template <int T>
hipError_t route_e(const RouteParams &p, bool backward, hipStream_t s) {
  // experts a lane holds: the smallest build that has room
  if (p.experts <= 64)
    return backward ? backward_t<T, 4>(p, s) : route_t<T, 4>(p, s);
  if (p.experts <= 128)
    return backward ? backward_t<T, 8>(p, s) : route_t<T, 8>(p, s);
  if (p.experts <= 256)
    return backward ? backward_t<T, 16>(p, s) : route_t<T, 16>(p, s);
  return backward ? backward_t<T, 32>(p, s) : route_t<T, 32>(p, s);
}

hipError_t route_any(const RouteParams &p, bool backward, hipStream_t s) {
  switch (p.dtype) {
  case kElemF32: return route_e<kElemF32>(p, backward, s);
  case kElemF16: return route_e<kElemF16>(p, backward, s);
  default: return route_e<kElemBF16>(p, backward, s);
  }
}

} // namespace

// the blocks' counts and the experts' totals
size_t route_workspace_bytes(int tokens, int experts, int) {
  if (tokens <= kSmallTokens)
    return 0;
  const size_t blocks = ((size_t)tokens + kTokenBlock - 1) / kTokenBlock;
  return (blocks + 1) * (size_t)experts * sizeof(int);
}

hipError_t launch_route(const RouteParams &p, hipStream_t s) { return route_any(p, false, s); }
hipError_t launch_route_backward(const RouteParams &p, hipStream_t s) {
  return route_any(p, true, s);
}

} // namespace tbk
