// Int8 kernels for gfx950 (device code only; the checks and the launches are in sh_int8.cpp):
// quantisation of tokens and the product with a SquareQ weight.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "sh_int8_args.h"
#include "stagehand_native.h"

namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float load_value(const void* p, uint64_t i, uint32_t dtype) {
  if (dtype == SH_DTYPE_BF16) return (float)static_cast<const __bf16*>(p)[i];
  if (dtype == SH_DTYPE_F16) return (float)static_cast<const _Float16*>(p)[i];
  return static_cast<const float*>(p)[i];
}

__device__ __forceinline__ void store_value(void* p, uint64_t i, float v, uint32_t dtype) {
  if (dtype == SH_DTYPE_BF16) static_cast<__bf16*>(p)[i] = (__bf16)v;
  else if (dtype == SH_DTYPE_F16) static_cast<_Float16*>(p)[i] = (_Float16)v;
  else static_cast<float*>(p)[i] = v;
}

// A token's factor 127 / a and scale a / 127 from the bits of a = max |x|. The bits order as the
// values do, with infinities and NaNs last, so their maximum finds a NaN too.
__device__ __forceinline__ void token_scale(uint32_t amax_bits, float* inv, float* scale) {
  const float amax = __builtin_bit_cast(float, amax_bits);
  if (amax_bits >= 0x7F800000u) {
    *inv = 0.0f;
    *scale = __builtin_nanf("");
  } else if (amax < 0x1p-120f) {  // 127 / a would overflow
    *inv = 0.0f;
    *scale = 0.0f;
  } else {
    *inv = 127.0f / amax;
    *scale = amax * (1.0f / 127.0f);
  }
}

// |x * inv| is at most 127 (1 + 2^-23), which rounds to 127. inv = 0 stands for a token without values:
// a NaN or an infinity times 0 must give 0, not a NaN.
__device__ __forceinline__ int32_t quantize(float x, float inv) {
  return inv == 0.0f ? 0 : (int32_t)__builtin_rintf(x * inv);
}

}  // namespace

// One workgroup of 256 per token.
extern "C" __global__ __launch_bounds__(256) void sh_quantize_tokens_kernel(sh::QuantizeArgs a) {
  __shared__ uint32_t part[4];
  __shared__ int32_t part_sum[4];
  const uint64_t t = blockIdx.x;
  const uint64_t at = t * a.x_ld;
  uint32_t amax = 0;
  for (uint32_t i = threadIdx.x; i < a.cols; i += 256)
    amax = max(amax, __builtin_bit_cast(uint32_t, load_value(a.x, at + i, a.dtype)) & 0x7FFFFFFFu);
  for (int m = 32; m >= 1; m >>= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, m));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x / 64] = amax;
  __syncthreads();
  amax = max(max(part[0], part[1]), max(part[2], part[3]));
  float inv, scale;
  token_scale(amax, &inv, &scale);
  int8_t* q = static_cast<int8_t*>(a.q) + t * a.q_ld;
  int32_t sum = 0;
  for (uint32_t i = threadIdx.x; i < a.q_ld; i += 256) {
    const int32_t v = i < a.cols ? quantize(load_value(a.x, at + i, a.dtype), inv) : 0;
    q[i] = (int8_t)v;
    sum += v;
  }
  for (int m = 32; m >= 1; m >>= 1) sum += __shfl_xor(sum, m);
  if ((threadIdx.x & 63) == 0) part_sum[threadIdx.x / 64] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    a.scale[t] = scale;
    if (a.sums != nullptr) a.sums[t] = part_sum[0] + part_sum[1] + part_sum[2] + part_sum[3];
  }
}

// Each wavefront: 16 tokens x 64 rows, operands straight from global memory. In a 16x16x64 MFMA lane
// l gives row l % 16 of each operand, bytes (l / 16) * 16 .. + 15, and holds elements (l / 16) * 4 + r
// of the first operand's rows for column l % 16 of the second's.
extern "C" __global__ __launch_bounds__(256) void sh_matmul_i8_kernel(sh::MatmulI8Args a) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64;
  const uint32_t row_tiles = (a.rows + 63) / 64;
  const uint64_t tile = (uint64_t)blockIdx.x * 4 + wave;
  const uint32_t t0 = (uint32_t)(tile / row_tiles) * 16, n0 = (uint32_t)(tile % row_tiles) * 64;
  if (t0 >= a.tokens) return;
  const uint32_t l16 = lane & 15, part = lane / 16;
  const uint32_t t = min(t0 + l16, a.tokens - 1);
  const int8_t* tp = static_cast<const int8_t*>(a.tq) + (uint64_t)t * a.t_ld + part * 16;
  const int8_t* wp[4];
  for (uint32_t f = 0; f < 4; ++f)
    wp[f] = static_cast<const int8_t*>(a.wq) + (uint64_t)min(n0 + f * 16 + l16, a.rows - 1) * a.w_ld + part * 16;
  i32x4 acc[4] = {};
  for (uint32_t k = 0; k < a.cols; k += 64) {
    // the tokens' rows are zero-filled to a multiple of 128; the weight's end at a multiple of 16
    const i32x4 tv = *reinterpret_cast<const i32x4*>(tp + k);
#pragma unroll
    for (uint32_t f = 0; f < 4; ++f) {
      i32x4 wv = {};
      if (k + part * 16 < a.cols) wv = *reinterpret_cast<const i32x4*>(wp[f] + k);
      acc[f] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv, tv, acc[f], 0, 0, 0);
    }
  }
  if (t0 + l16 >= a.tokens) return;
  const float ts = a.t_scale[t];
  const float sum = a.w_zp != nullptr ? (float)a.t_sums[t] : 0.0f;
#pragma unroll
  for (uint32_t f = 0; f < 4; ++f) {
#pragma unroll
    for (uint32_t r = 0; r < 4; ++r) {
      const uint32_t n = n0 + f * 16 + part * 4 + r;
      if (n >= a.rows) continue;
      float v = (float)acc[f][r];
      if (a.w_zp != nullptr) v = __builtin_fmaf(-a.w_zp[n], sum, v);
      v *= ts * a.w_scale[n];
      if (a.bias != nullptr) v += a.bias[n];
      store_value(a.out, (uint64_t)t * a.out_ld + n, v, a.out_dtype);
    }
  }
}
