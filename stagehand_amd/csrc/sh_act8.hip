// Activations in 8 bits and back for gfx950 (device code only; the checks and the launches are in sh_act8.cpp,
// the format in sh_act8_device.h).
//
// Both ways are bound by HBM: each value is read once and written once, 3.03 bytes for bf16. A work-item takes one chunk of
// 8 values, whole vectors both ways; four neighbours share a group, whose maximum takes two data-parallel moves.
//
// Measured: 16384 x 4096 bf16 written 37 us (5.5 TB/s), read 34 us (6.0); four chunks a work-item 40 and 34 us.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "sh_act8_args.h"
#include "sh_act8_device.h"
#include "sh_internal.h"
#include "stagehand_native.h"

namespace {

struct Place {
  uint32_t row, col;
};
__device__ __forceinline__ Place place_of(const sh::Act8Args& a, uint32_t chunk) {
  const uint32_t row = sh::udiv(chunk, a.magic);
  return {row, (chunk - row * a.row_chunks) * 8};
}

template <typename T>
__device__ __forceinline__ void quantize_body(const sh::Act8Args& a) {
  const uint32_t c = blockIdx.x * sh::kAct8Threads + threadIdx.x;
  if (c >= a.chunks) return;  // whole groups of four work-items
  const Place p = place_of(a, c);
  auto v = Values8<T>::zero();
  if (p.col < a.cols) v = Values8<T>::load(static_cast<const T*>(a.x) + p.row * a.x_ld + p.col, a.cols - p.col);
  float f[8];
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i) f[i] = (float)v[i];
  const uint32_t e = group_exponent(f);
  static_cast<uint2*>(a.q)[c] = quantize8<T>(f, e);
  if (c % 4 == 0) static_cast<uint8_t*>(a.exponent)[c / 4] = (uint8_t)e;
}

template <typename T>
__device__ __forceinline__ void dequantize_body(const sh::Act8Args& a) {
  const uint32_t c = blockIdx.x * sh::kAct8Threads + threadIdx.x;
  if (c >= a.chunks) return;
  const Place p = place_of(a, c);
  if (p.col >= a.cols) return;
  float f[8];
  dequantize8(static_cast<const uint2*>(a.q)[c], group_scale(static_cast<const uint8_t*>(a.exponent)[c / 4]), f);
  Values8<T>::store(static_cast<T*>(a.x) + p.row * a.x_ld + p.col, f, a.cols - p.col);
}

}  // namespace

#define SH_ACT8(name, T)                                                                                        \
  extern "C" __global__ __launch_bounds__(sh::kAct8Threads) void sh_act8_quantize_##name##_kernel(sh::Act8Args a) { \
    quantize_body<T>(a);                                                                                        \
  }                                                                                                             \
  extern "C" __global__ __launch_bounds__(sh::kAct8Threads) void sh_act8_dequantize_##name##_kernel(sh::Act8Args a) { \
    dequantize_body<T>(a);                                                                                      \
  }
SH_ACT8(bf16, __bf16)
SH_ACT8(f16, _Float16)
SH_ACT8(f32, float)
