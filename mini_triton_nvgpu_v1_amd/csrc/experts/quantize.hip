// Values to e4m3 with an f32 scale for each 1 x 128 block (activations) or
// 128 x 128 block (weights):
//   a = max(2^-100, largest finite-comparable |x| of the block)
//   scale = a / 448,  q = round to nearest even (x * (448 / a))
// 448 is e4m3's largest value. The floor 2^-100 keeps both quotients normal
// f32 numbers, and a block of zeros gives zeros. A NaN does not enter a and is
// NaN in q; an infinity makes the block's scale infinite, so that the block
// stands for NaN and infinities, never for finite values.
//
// Bound by memory: x is read once and q written once. A 1 x 128 block lies
// over 16 lanes, 8 values each; a 128 x 128 block over a workgroup, 64 each,
// which stay in registers between the two steps. 8192 x 4096 bf16 in 1 x 128
// blocks: 24-27 us, 3.7-4.2 TB/s.
#include "experts_device.h"

namespace tbk {

namespace {

constexpr float kF8Max = 448.f;
constexpr float kTiny = 0x1p-100f;

__device__ __forceinline__ uint64_t to_f8(f32x8 x, float inv) {
  x *= inv;
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[4], x[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[6], x[7], hi, true);
  return (uint32_t)lo | ((uint64_t)(uint32_t)hi << 32);
}

__device__ __forceinline__ float amax8(f32x8 x) {
  float m = kTiny;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    m = fmaxf(m, fabsf(x[i]));
  return m;
}

template <int T>
__global__ __launch_bounds__(256) void quantize_rows(QuantizeParams p, int kb) {
  const int l16 = threadIdx.x & 15;
  const int64_t items = p.batch * p.rows * kb;
  const int64_t item = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  if (item >= items)
    return;
  const int64_t row = item / kb;
  const int b = (int)(item % kb), col = b * 128 + l16 * 8;
  const bool in = col < p.cols;
  f32x8 x = {};
  if (in)
    x = load8<T>(p.x, (row / p.rows) * p.x_stride + (row % p.rows) * p.ldx + col);
  float m = amax8(x);
#pragma unroll
  for (int d = 1; d < 16; d *= 2)
    m = fmaxf(m, __shfl_xor(m, d, 16));
  if (in)
    *reinterpret_cast<uint64_t *>(static_cast<char *>(p.q) + row * p.cols + col) =
        to_f8(x, kF8Max / m);
  if (l16 == 0)
    p.scale[row * kb + b] = m / kF8Max;
}

template <int T>
__global__ __launch_bounds__(256) void quantize_tiles(QuantizeParams p, int rb, int kb) {
  __shared__ float part[4];
  const int64_t item = blockIdx.x;
  const int b = (int)(item % kb);
  const int64_t r = item / kb % rb, batch = item / kb / rb;
  const int l16 = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const int col = b * 128 + l16 * 8;
  f32x8 x[8];
  float m = kTiny;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = r * 128 + r0 + 16 * i;
    x[i] = (f32x8){};
    if (col < p.cols && row < p.rows)
      x[i] = load8<T>(p.x, batch * p.x_stride + row * p.ldx + col);
    m = fmaxf(m, amax8(x[i]));
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2)
    m = fmaxf(m, __shfl_xor(m, d));
  if ((threadIdx.x & 63) == 0)
    part[threadIdx.x >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  const float inv = kF8Max / m;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = r * 128 + r0 + 16 * i;
    if (col < p.cols && row < p.rows)
      *reinterpret_cast<uint64_t *>(static_cast<char *>(p.q) +
                                    (batch * p.rows + row) * p.cols + col) = to_f8(x[i], inv);
  }
  if (threadIdx.x == 0)
    p.scale[item] = m / kF8Max;
}

template <int T>
hipError_t quantize_t(const QuantizeParams &p, hipStream_t s) {
  const int kb = (p.cols + 127) / 128;
  if (p.block_rows == 1) {
    const int64_t items = p.batch * p.rows * kb;
    hipLaunchKernelGGL(quantize_rows<T>, dim3((unsigned)((items + 15) / 16)), dim3(256), 0, s, p,
                       kb);
  } else {
    const int rb = (int)((p.rows + 127) / 128);
    hipLaunchKernelGGL(quantize_tiles<T>, dim3((unsigned)(p.batch * rb * kb)), dim3(256), 0, s,
                       p, rb, kb);
  }
  return hipGetLastError();
}

} // namespace

hipError_t launch_quantize(const QuantizeParams &p, hipStream_t s) {
  switch (p.dtype) {
  case kElemF32: return quantize_t<kElemF32>(p, s);
  case kElemF16: return quantize_t<kElemF16>(p, s);
  default: return quantize_t<kElemBF16>(p, s);
  }
}

} // namespace tbk
