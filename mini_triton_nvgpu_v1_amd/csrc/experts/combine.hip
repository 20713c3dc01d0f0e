// The weighted sum of each token's expert rows, and its gradients:
//   out[t] = sum_j w[t,j] y[slot[t,j]]
//   dy[slot[t,j]] = w[t,j] dout[t],  dw[t,j] = <dout[t], y[slot[t,j]]>
// Sums are f32; out and dy are rounded once. A slot outside [0, y_rows) (-1:
// the pair was not routed) adds nothing, and its dw is 0.
//
// Bound by memory: every row of y is read once (and of dy written once), in
// whole 16-byte pieces, 64 lanes on consecutive columns; a wave's slots and
// weights are the same for all its lanes. The rows on their way are held as
// they lie in memory and become f32 when they are added: half the registers,
// six waves on a SIMD unit rather than four in the gradient.
// 8192 tokens of 8 bf16 rows of 4096: the sum takes 101-104 us (5.8-6.0 TB/s),
// its gradients 229-232 us (4.9 TB/s read and written; 269 us with rows held as f32).
#include "experts_device.h"

namespace tbk {

namespace {

constexpr int kChunk = 512;  // columns a wave takes at a time: 8 a lane
constexpr int kTogether = 8; // rows loaded before the first is added

__device__ __forceinline__ int uniform_slot(const CombineParams &p, int64_t at) {
  const int s = __builtin_amdgcn_readfirstlane(p.slots[at]);
  return s >= 0 && s < p.y_rows ? s : -1;
}

// a wave: one token, 512 columns
template <int T, bool ONCE>
__global__ __launch_bounds__(256) void combine_kernel(CombineParams p, int chunks) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t item = (int64_t)blockIdx.x * 4 + wave;
  const int64_t token = item / chunks;
  const int col = (int)(item % chunks) * kChunk + lane * 8;
  if (token >= p.tokens)
    return;
  const bool in = col < p.width;
  f32x8 sum = {};
  for (int j0 = 0; j0 < p.top_k; j0 += kTogether) {
    typename Raw8<T>::type v[kTogether];
    float w[kTogether];
#pragma unroll
    for (int j = 0; j < kTogether; ++j) {
      w[j] = 0.f;
      v[j] = (typename Raw8<T>::type){};
      if (j0 + j < p.top_k) {
        const int64_t at = token * p.top_k + j0 + j;
        const int s = uniform_slot(p, at);
        if (s >= 0) {
          w[j] = p.weights ? p.weights[at] : 1.f;
          if (in)
            v[j] = load_raw8<T, ONCE>(p.y, (int64_t)s * p.ldy + col);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kTogether; ++j)
      sum += w[j] * to_f32(v[j]);
  }
  if (in)
    store8<T, ONCE>(p.out, token * p.ldo + col, sum);
}

// a wave: one token, all columns
template <int T, bool ONCE>
__global__ __launch_bounds__(256) void combine_backward_kernel(CombineParams p) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t token = (int64_t)blockIdx.x * 4 + wave;
  if (token >= p.tokens)
    return;
  for (int j0 = 0; j0 < p.top_k; j0 += kTogether) {
    int slot[kTogether];
    float w[kTogether], dot[kTogether];
#pragma unroll
    for (int j = 0; j < kTogether; ++j) {
      const int64_t at = token * p.top_k + j0 + j;
      slot[j] = j0 + j < p.top_k ? uniform_slot(p, at) : -1;
      w[j] = slot[j] >= 0 ? (p.weights ? p.weights[at] : 1.f) : 0.f;
      dot[j] = 0.f;
    }
    for (int col = lane * 8; col < p.width; col += kChunk) {
      const f32x8 d = load8<T>(p.dout, token * p.ldo + col);
      typename Raw8<T>::type v[kTogether];
#pragma unroll
      for (int j = 0; j < kTogether; ++j)
        if (slot[j] >= 0)
          v[j] = load_raw8<T, ONCE>(p.y, (int64_t)slot[j] * p.ldy + col);
#pragma unroll
      for (int j = 0; j < kTogether; ++j)
        if (slot[j] >= 0) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            dot[j] += (float)v[j][i] * d[i];
          store8<T, ONCE>(p.dy, (int64_t)slot[j] * p.lddy + col, w[j] * d);
        }
    }
#pragma unroll
    for (int j = 0; j < kTogether; ++j) {
      float x = dot[j];
#pragma unroll
      for (int o = 1; o < 64; o *= 2)
        x += __shfl_xor(x, o);
      if (p.dweights && lane == 0 && j0 + j < p.top_k)
        p.dweights[token * p.top_k + j0 + j] = x;
    }
  }
}

constexpr int sizeof_elem(int t) { return t == kElemF32 ? 4 : 2; }

// Rows that do not fit the L2 caches (32 MB) are read and written past them
// (8192 tokens, 8 rows of 4096 bf16, sum and gradients: 394 us through them, 368 past
// them, then with rows held as f32); smaller ones stay there for the kernels around.
bool large(const CombineParams &p, int size) {
  return (int64_t)p.tokens * p.top_k * p.width * size >= (int64_t)64 << 20;
}

template <int T>
hipError_t combine_t(const CombineParams &p, hipStream_t s) {
  const int chunks = (p.width + kChunk - 1) / kChunk;
  const int64_t waves = (int64_t)p.tokens * chunks;
  const dim3 grid((unsigned)((waves + 3) / 4)), block(256);
  if (large(p, sizeof_elem(T)))
    hipLaunchKernelGGL((combine_kernel<T, true>), grid, block, 0, s, p, chunks);
  else
    hipLaunchKernelGGL((combine_kernel<T, false>), grid, block, 0, s, p, chunks);
  return hipGetLastError();
}

template <int T>
hipError_t backward_t(const CombineParams &p, hipStream_t s) {
  const dim3 grid((unsigned)((p.tokens + 3) / 4)), block(256);
  if (large(p, sizeof_elem(T)))
    hipLaunchKernelGGL((combine_backward_kernel<T, true>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((combine_backward_kernel<T, false>), grid, block, 0, s, p);
  return hipGetLastError();
}

} // namespace

hipError_t launch_combine(const CombineParams &p, hipStream_t s) {
  switch (p.dtype) {
  case kElemF32: return combine_t<kElemF32>(p, s);
  case kElemF16: return combine_t<kElemF16>(p, s);
  default: return combine_t<kElemBF16>(p, s);
  }
}

hipError_t launch_combine_backward(const CombineParams &p, hipStream_t s) {
  switch (p.dtype) {
  case kElemF32: return backward_t<kElemF32>(p, s);
  case kElemF16: return backward_t<kElemF16>(p, s);
  default: return backward_t<kElemBF16>(p, s);
  }
}

} // namespace tbk
