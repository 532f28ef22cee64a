// The gradient of a Linear's weight from its kept input, for gfx950 (device code only; the checks and the launches
// are in sh_act8.cpp, the format of the input in sh_act8_device.h).
//
//   dW[o][i] = sum over the tokens t of dy[t][o] x^[t][i],  db[o] = sum over t of dy[t][o]
//
// x^ is exact in the 16-bit types (7 significant bits), so the matrix cores multiply the very numbers that were kept, and
// sum in fp32. A gradient in fp32 goes in as three bf16 parts that add up to its 24 bits, each multiplied by itself.
//
// Both operands lie with the tokens, over which is summed, in their slow direction. Tiles go through LDS as they lie, x^
// in 16 bits, and the transposing LDS reads give the lanes what a fragment needs.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "sh_act8_args.h"
#include "sh_act8_device.h"
#include "stagehand_native.h"

namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));

// What the matrix cores multiply for a gradient in T, and in how many parts.
template <typename T>
struct Multiplied {
  typedef __bf16 Type;
  static constexpr uint32_t kParts = 1;
};
template <>
struct Multiplied<_Float16> {
  typedef _Float16 Type;
  static constexpr uint32_t kParts = 1;
};
template <>
struct Multiplied<float> {
  typedef __bf16 Type;
  static constexpr uint32_t kParts = 3;
};

template <typename E>
__device__ __forceinline__ f32x4_t mfma(s16x8_t a, s16x8_t b, f32x4_t c) {
  typedef E Vec __attribute__((ext_vector_type(8)));
  const Vec va = __builtin_bit_cast(Vec, a), vb = __builtin_bit_cast(Vec, b);
  if constexpr (__is_same(E, _Float16)) return __builtin_amdgcn_mfma_f32_16x16x32_f16(va, vb, c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, vb, c, 0, 0, 0);
}

// A stage holds kGradStep tokens' rows of N 16-bit values. The 16 values of unit u lie in unit u ^ swizzle(t): the
// rows that a transposing read takes together, 4 of every 8, then lie in different LDS banks.
template <uint32_t N>
__device__ __forceinline__ constexpr uint32_t swizzle(uint32_t t) {
  if (N >= 128) return (t & 3) | (t >> 1 & 4);
  if (N == 64) return (t >> 1 & 1) | (t >> 2 & 2);
  return t >> 3 & 1;
}

typedef __attribute__((address_space(3))) s16x4_t* LdsRead;

// The fragment of unit u: lane l gets values of column l % 16, tokens 8 (l / 16) .. + 7.
template <uint32_t N>
__device__ __forceinline__ s16x8_t read_fragment(const short* stage, uint32_t u) {
  const uint32_t lane = threadIdx.x & 63, t = lane / 16 * 8 + lane % 16 / 4;
  const short* p = stage + t * N + (u ^ swizzle<N>(t)) * 16 + lane % 4 * 4;
  const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsRead)p);
  const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsRead)(p + 4 * N));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

template <typename T, uint32_t TO, uint32_t TI, uint32_t WO, uint32_t WI>
__device__ __forceinline__ void weight_grad(const sh::WeightGradArgs& a, short* lds) {
  using E = typename Multiplied<T>::Type;
  constexpr uint32_t kParts = Multiplied<T>::kParts, kStep = sh::kGradStep;
  constexpr uint32_t kThreads = WO * WI * 64, FO = TO / WO / 16, FI = TI / WI / 16;
  static_assert(FI == 4, "a wavefront's inputs are one group of 64 permuted ones");
  constexpr uint32_t kDy = kStep * TO, kStage = kParts * kDy + kStep * TI;
  constexpr uint32_t ND = (kDy / 8 + kThreads - 1) / kThreads, NX = (kStep * TI / 16 + kThreads - 1) / kThreads;
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t wo = wave / WI, wi = wave % WI;

  // XCDs take consecutive runs of tiles, an XCD's L2 then serves neighbouring ones
  const uint32_t tiles_o = (a.out + TO - 1) / TO, tiles_i = (a.cols + TI - 1) / TI, tiles = tiles_o * tiles_i;
  const uint32_t all = tiles * a.splits, xcd = blockIdx.x % 8;
  const uint32_t p = xcd * (all / 8) + min(xcd, all % 8) + blockIdx.x / 8;
  const uint32_t split = p / tiles, tile = p % tiles;
  const uint32_t o0 = tile % tiles_o * TO, i0 = tile / tiles_o * TI;
  const uint32_t t_begin = split * a.split_tokens, t_end = min(a.tokens, t_begin + a.split_tokens);
  const uint32_t groups = (a.cols + SH_ACT8_GROUP - 1) / SH_ACT8_GROUP;

  typename Values8<T>::Vec dy[ND];
  uint4 q[NX];
  uint32_t e[NX];
  auto load = [&](uint32_t t0) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t j = 0; j < ND; ++j) {
      const uint32_t c = j * kThreads + threadIdx.x, t = t0 + c / (TO / 8), o = o0 + c % (TO / 8) * 8;
      dy[j] = Values8<T>::zero();
      if (c < kDy / 8 && t < t_end && o < a.out) dy[j] = Values8<T>::load(static_cast<const T*>(a.dy) + t * a.dy_ld + o, a.out - o);
    }
#pragma unroll
    for (uint32_t j = 0; j < NX; ++j) {
      const uint32_t c = j * kThreads + threadIdx.x, t = t0 + c / (TI / 16), i = i0 + c % (TI / 16) * 16;
      q[j] = make_uint4(0, 0, 0, 0);
      e[j] = 1;
      if (c < kStep * TI / 16 && t < t_end && i < groups * SH_ACT8_GROUP) {
        const uint64_t at = (uint64_t)t * groups * SH_ACT8_GROUP + i;
        q[j] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.q) + at);
        e[j] = static_cast<const uint8_t*>(a.exponent)[at / SH_ACT8_GROUP];
      }
    }
  };
  typedef E Out4 __attribute__((ext_vector_type(4)));
  typedef E Out8 __attribute__((ext_vector_type(8)));
  auto put = [&](short* stage) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t j = 0; j < ND; ++j) {
      const uint32_t c = j * kThreads + threadIdx.x, t = c / (TO / 8), c8 = c % (TO / 8);
      if (c >= kDy / 8) continue;
      short* at = stage + t * TO + ((c8 / 2) ^ swizzle<TO>(t)) * 16 + c8 % 2 * 8;
      if constexpr (kParts == 1) {
        *reinterpret_cast<typename Values8<T>::Vec*>(at) = dy[j];
      } else {
        float rest[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) rest[i] = dy[j][i];
#pragma unroll
        for (uint32_t part = 0; part < kParts; ++part) {
          Out8 v;
#pragma unroll
          for (uint32_t i = 0; i < 8; ++i) {  // the next 8 significant bits; all of an infinity
            const float head = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, rest[i]) & 0xFFFF0000u);
            v[i] = (E)head;
            rest[i] = rest[i] == head ? 0.0f : rest[i] - head;
          }
          *reinterpret_cast<Out8*>(at + part * kDy) = v;
        }
      }
    }
#pragma unroll
    for (uint32_t j = 0; j < NX; ++j) {
      const uint32_t c = j * kThreads + threadIdx.x, t = c / (TI / 16), c16 = c % (TI / 16);
      if (c >= kStep * TI / 16) continue;
      const float scale = group_scale(e[j]);
      const uint32_t words[4] = {q[j].x, q[j].y, q[j].z, q[j].w};
#pragma unroll
      for (uint32_t f = 0; f < 4; ++f) {  // column c16 * 16 + f * 4 + m is column c16 % 4 * 4 + m of fragment f
        float v[4];
        dequantize4(words[f], scale, v);
        Out4 out;
#pragma unroll
        for (uint32_t m = 0; m < 4; ++m) out[m] = (E)v[m];
        *reinterpret_cast<Out4*>(stage + kParts * kDy + t * TI + ((c16 / 4 * 4 + f) ^ swizzle<TI>(t)) * 16 + c16 % 4 * 4) = out;
      }
    }
  };

  f32x4_t acc[FO][FI] = {}, bias[FO] = {};
  const bool with_bias = a.dbias != nullptr && i0 == 0 && wi == 0;
  s16x8_t ones;
  {
    Out8 v;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) v[i] = (E)1.0f;
    ones = __builtin_bit_cast(s16x8_t, v);
  }
  load(t_begin);
  put(lds);
  uint32_t s = 0;
  for (uint32_t t0 = t_begin; t0 < t_end; t0 += kStep) {
    __syncthreads();  // stage s is written, and read the one that is written next
    const bool more = t0 + kStep < t_end;
    if (more) load(t0 + kStep);
    const short* stage = lds + s * kStage;
    s16x8_t x[FI];
#pragma unroll
    for (uint32_t j = 0; j < FI; ++j) x[j] = read_fragment<TI>(stage + kParts * kDy, wi * FI + j);
#pragma unroll
    for (uint32_t part = 0; part < kParts; ++part) {
#pragma unroll
      for (uint32_t i = 0; i < FO; ++i) {
        const s16x8_t d = read_fragment<TO>(stage + part * kDy, wo * FO + i);
#pragma unroll
        for (uint32_t j = 0; j < FI; ++j) acc[i][j] = mfma<E>(x[j], d, acc[i][j]);
        if (with_bias) bias[i] = mfma<E>(ones, d, bias[i]);
      }
    }
    s ^= 1;
    if (more) put(lds + s * kStage);
  }

  // lane: output l % 16 of each fragment of outputs, 16 consecutive inputs
  const uint32_t i = i0 + wi * (TI / WI) + lane / 16 * 16;
  const uint32_t count = i < a.cols ? a.cols - i : 0;
  float* sums = a.partials;
  if (sums != nullptr) sums += split * ((uint64_t)a.out * a.cols + (a.dbias != nullptr ? a.out : 0));
#pragma unroll
  for (uint32_t f = 0; f < FO; ++f) {
    const uint32_t o = o0 + wo * (TO / WO) + f * 16 + lane % 16;
    if (o >= a.out) continue;
    float v[2][8];
#pragma unroll
    for (uint32_t j = 0; j < 16; ++j) v[j / 8][j % 8] = acc[f][j / 4][j % 4];
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t n = count > h * 8 ? count - h * 8 : 0;
      if (sums != nullptr) {
        Values8<float>::store(sums + (uint64_t)o * a.cols + i + h * 8, v[h], n);
      } else {
        const uint64_t at = o * a.dw_ld + i + h * 8;
        if (a.out_dtype == SH_DTYPE_BF16) Values8<__bf16>::store(static_cast<__bf16*>(a.dweight) + at, v[h], n);
        else if (a.out_dtype == SH_DTYPE_F16) Values8<_Float16>::store(static_cast<_Float16*>(a.dweight) + at, v[h], n);
        else Values8<float>::store(static_cast<float*>(a.dweight) + at, v[h], n);
      }
    }
    if (with_bias && lane < 16) {  // every row of the product with ones
      if (sums != nullptr) sums[(uint64_t)a.out * a.cols + o] = bias[f][0];
      else if (a.out_dtype == SH_DTYPE_BF16) static_cast<__bf16*>(a.dbias)[o] = (__bf16)bias[f][0];
      else if (a.out_dtype == SH_DTYPE_F16) static_cast<_Float16*>(a.dbias)[o] = (_Float16)bias[f][0];
      else static_cast<float*>(a.dbias)[o] = bias[f][0];
    }
  }
}

}  // namespace

// The tiles of sh_act8_args.h.
#define SH_WEIGHT_GRAD(name, T, TO, TI, WO, WI)                                                                   \
  extern "C" __global__ __launch_bounds__(WO * WI * 64) void sh_weight_grad_##name##_##TO##x##TI##_kernel(sh::WeightGradArgs a) { \
    __shared__ alignas(16) short lds[2 * sh::kGradStep * (Multiplied<T>::kParts * TO + TI)];                      \
    weight_grad<T, TO, TI, WO, WI>(a, lds);                                                                       \
  }
#define SH_WEIGHT_GRAD_TILES(name, T)       \
  SH_WEIGHT_GRAD(name, T, 32, 128, 2, 2)    \
  SH_WEIGHT_GRAD(name, T, 128, 128, 2, 2)   \
  SH_WEIGHT_GRAD(name, T, 256, 256, 2, 4)
SH_WEIGHT_GRAD_TILES(bf16, __bf16)
SH_WEIGHT_GRAD_TILES(f16, _Float16)
SH_WEIGHT_GRAD_TILES(f32, float)

// dweight and dbias from the sums of the splits, in their order: four values a work-item, then the biases.
extern "C" __global__ __launch_bounds__(sh::kGradJoinThreads) void sh_weight_grad_join_kernel(sh::WeightGradArgs a) {
  const uint64_t n = (uint64_t)blockIdx.x * sh::kGradJoinThreads + threadIdx.x;
  const uint32_t quads = (a.cols + 3) / 4;
  const uint64_t weights = (uint64_t)a.out * quads, set = (uint64_t)a.out * a.cols + (a.dbias != nullptr ? a.out : 0);
  void* out = a.dweight;
  uint64_t from, to;
  uint32_t count;
  if (n < weights) {
    const uint32_t o = (uint32_t)(n / quads), i = (uint32_t)(n - (uint64_t)o * quads) * 4;
    from = (uint64_t)o * a.cols + i;
    to = o * a.dw_ld + i;
    count = min(a.cols - i, 4u);
  } else {
    to = n - weights;
    if (a.dbias == nullptr || to >= a.out) return;
    out = a.dbias;
    from = (uint64_t)a.out * a.cols + to;
    count = 1;
  }
  typedef float Vec __attribute__((ext_vector_type(4)));
  typedef Vec Any __attribute__((aligned(4)));
  float v[4] = {};
  const float* p = a.partials + from;
  if (count == 4) {
#pragma unroll 8
    for (uint32_t s = 0; s < a.splits; ++s) {
      const Vec x = *reinterpret_cast<const Any*>(p + s * set);
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) v[j] += x[j];
    }
  } else {
    for (uint32_t s = 0; s < a.splits; ++s)
#pragma unroll
      for (uint32_t j = 0; j < 3; ++j)
        if (j < count) v[j] += p[s * set + j];
  }
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    if (j >= count) continue;
    if (a.out_dtype == SH_DTYPE_BF16) static_cast<__bf16*>(out)[to + j] = (__bf16)v[j];
    else if (a.out_dtype == SH_DTYPE_F16) static_cast<_Float16*>(out)[to + j] = (_Float16)v[j];
    else static_cast<float*>(out)[to + j] = v[j];
  }
}
