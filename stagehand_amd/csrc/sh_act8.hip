// Activations in 8 bits and back for gfx950 (device code only; the checks and the launches are in sh_act8.cpp,
// the format in sh_act8_device.h).
//
// Both ways are bound by HBM: each value is read once and written once, 3.03 bytes for bf16. A work-item takes chunks of
// 8 values, whole vectors both ways; four neighbours share a group, whose maximum takes two data-parallel moves.

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
  typename Values8<T>::Vec v[sh::kAct8Chunks];
  const uint32_t first = blockIdx.x * (sh::kAct8Threads * sh::kAct8Chunks) + threadIdx.x;
#pragma unroll
  for (uint32_t j = 0; j < sh::kAct8Chunks; ++j) {
    const uint32_t c = first + j * sh::kAct8Threads;
    v[j] = Values8<T>::zero();
    if (c >= a.chunks) continue;
    const Place p = place_of(a, c);
    if (p.col < a.cols) v[j] = Values8<T>::load(static_cast<const T*>(a.x) + p.row * a.x_ld + p.col, a.cols - p.col);
  }
#pragma unroll
  for (uint32_t j = 0; j < sh::kAct8Chunks; ++j) {
    const uint32_t c = first + j * sh::kAct8Threads;
    if (c >= a.chunks) continue;  // whole groups of four work-items
    float f[8];
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) f[i] = (float)v[j][i];
    const uint32_t e = group_exponent(f);
    static_cast<uint2*>(a.q)[c] = quantize8<T>(f, e);
    if (c % 4 == 0) static_cast<uint8_t*>(a.exponent)[c / 4] = (uint8_t)e;
  }
}

template <typename T>
__device__ __forceinline__ void dequantize_body(const sh::Act8Args& a) {
  uint2 q[sh::kAct8Chunks];
  uint32_t e[sh::kAct8Chunks];
  const uint32_t first = blockIdx.x * (sh::kAct8Threads * sh::kAct8Chunks) + threadIdx.x;
#pragma unroll
  for (uint32_t j = 0; j < sh::kAct8Chunks; ++j) {
    const uint32_t c = first + j * sh::kAct8Threads;
    if (c >= a.chunks) continue;
    q[j] = static_cast<const uint2*>(a.q)[c];
    e[j] = static_cast<const uint8_t*>(a.exponent)[c / 4];
  }
#pragma unroll
  for (uint32_t j = 0; j < sh::kAct8Chunks; ++j) {
    const uint32_t c = first + j * sh::kAct8Threads;
    if (c >= a.chunks) continue;
    const Place p = place_of(a, c);
    if (p.col >= a.cols) continue;
    float f[8];
    dequantize8(q[j], group_scale(e[j]), f);
    Values8<T>::store(static_cast<T*>(a.x) + p.row * a.x_ld + p.col, f, a.cols - p.col);
  }
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
