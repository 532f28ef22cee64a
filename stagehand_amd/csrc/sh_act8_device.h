// Device code of the 8-bit format of activations, for the kernels that write and read it.
//
// 32 neighbouring values share a power of two 2^k, the smallest with max |x| <= 127 * 2^k (k = -126 at least), and are
// kept as q = rint(x * 2^-k). The product by a power of two is exact, so the rounding to q is the only one, and
// q * 2^k has 7 significant bits: exact in bf16, fp16 (for what came from fp16) and fp32. The exponent is kept as
// the biased byte k + 127; 255 marks a group with an infinity or a NaN, which is read back as NaNs.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "stagehand_native.h"

namespace {

template <typename T>
struct Values8 {
  typedef T Vec __attribute__((ext_vector_type(8)));
  typedef Vec Any __attribute__((aligned(2)));  // gfx950 loads and stores whole vectors at any address

  static __device__ __forceinline__ Vec zero() {
    Vec v;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) v[i] = (T)0.0f;
    return v;
  }
  // Values p[0 .. count - 1], zeros behind them.
  static __device__ __forceinline__ Vec load(const T* p, uint32_t count) {
    if (count >= 8) return *reinterpret_cast<const Any*>(p);
    Vec v = zero();
#pragma unroll
    for (uint32_t i = 0; i < 7; ++i)
      if (i < count) v[i] = p[i];
    return v;
  }
  static __device__ __forceinline__ void store(T* p, const float (&in)[8], uint32_t count) {
    if (count >= 8) {
      Vec v;
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) v[i] = (T)in[i];
      *reinterpret_cast<Any*>(p) = v;
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 7; ++i)
        if (i < count) p[i] = (T)in[i];
    }
  }
};

// The larger of v and the value that another work-item of the four holds.
template <int CTRL>
__device__ __forceinline__ uint32_t max_moved(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false));
}

// The exponent byte of a group whose values four neighbouring work-items hold, 8 each. The bits of |x| order as the
// values do, with infinities and NaNs last.
__device__ __forceinline__ uint32_t group_exponent(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i) m = max(m, __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu);
  m = max_moved<0xB1>(m);  // quad_perm 1,0,3,2
  m = max_moved<0x4E>(m);  // quad_perm 2,3,0,1
  if (m >= 0x7F800000u) return 255;
  // max |x| = 1.f * 2^E; 127 * 2^k = 1.984375 * 2^(k + 6): k = E - 6, and one more where 1.f is more than 1.984375,
  // which the sum carries into the exponent
  const uint32_t biased = (m + 0x1FFFFu) >> 23;
  return max(biased, 7u) - 6;
}

// q of 8 values of a group with exponent byte e. Values that came from T: where 64 * 2^k is not a number of T any
// more (fp16 k = 10, others k = 122), multiples end with 63.
template <typename T>
__device__ __forceinline__ uint2 quantize8(const float (&v)[8], uint32_t e) {
  constexpr uint32_t kTop = __is_same(T, _Float16) ? 137 : 249;
  const float inverse = __builtin_bit_cast(float, (254u - e) << 23);  // 2^-k
  const float most = e == kTop ? 63.0f : 127.0f;
  uint32_t b[8];
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i) {
    const float r = __builtin_amdgcn_fmed3f(__builtin_rintf(v[i] * inverse), -most, most);
    b[i] = (uint32_t)(int32_t)r;
  }
  auto pack = [&](uint32_t i) {
    const uint32_t lo = __builtin_amdgcn_perm(b[i + 1], b[i], 0x0C0C0400u), hi = __builtin_amdgcn_perm(b[i + 3], b[i + 2], 0x0C0C0400u);
    return lo | hi << 16;
  };
  return e == 255 ? make_uint2(0, 0) : make_uint2(pack(0), pack(4));
}

// 2^k, or NaN.
__device__ __forceinline__ float group_scale(uint32_t e) {
  return __builtin_bit_cast(float, e == 255 ? 0x7FC00000u : e << 23);
}

// Byte I of q, as a signed number. Written as assembly: the compiler takes two instructions for three of the bytes.
template <uint32_t I>
__device__ __forceinline__ float signed_byte(uint32_t q) {
  float v;
  if constexpr (I == 0) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(v) : "v"(q));
  else if constexpr (I == 1) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(v) : "v"(q));
  else if constexpr (I == 2) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(v) : "v"(q));
  else asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(v) : "v"(q));
  return v;
}

__device__ __forceinline__ void dequantize4(uint32_t q, float scale, float* v) {
  v[0] = signed_byte<0>(q) * scale;
  v[1] = signed_byte<1>(q) * scale;
  v[2] = signed_byte<2>(q) * scale;
  v[3] = signed_byte<3>(q) * scale;
}

__device__ __forceinline__ void dequantize8(uint2 q, float scale, float (&v)[8]) {
  dequantize4(q.x, scale, v);
  dequantize4(q.y, scale, v + 4);
}

}  // namespace
