// The gradient of a Linear's weight from its kept input, for gfx950 (device code only; the checks and the launches
// are in sh_act8.cpp, the format of the input in sh_act8_device.h).
//
//   dW[o][i] = sum over the tokens t of dy[t][o] x^[t][i],  db[o] = sum over t of dy[t][o]
//
// x^ is exact in the 16-bit types (7 significant bits), so the matrix cores multiply the very numbers that were kept, and
// sum in fp32. A gradient in fp32 goes in as three bf16 parts that add up to its 24 bits, each multiplied by itself; below
// 2^-110 they lose what lies under 2^-133, the least number of bf16.
//
// Both operands lie with the tokens, over which is summed, in their slow direction. Tiles go through LDS as they lie, x^
// in 16 bits, and the transposing LDS reads give the lanes what a fragment needs.
//
// Large products are bound by what stands around the matrix cores, which are busy 48% of the cycles: the issue of the
// instructions that turn bytes into 16-bit values, which every tile of outputs does again, LDS and the barriers, at the clock
// that their power allows. 16384 x 16384 x 4096 (tokens x outputs x inputs) takes 1.86 to 2.04 ms, 1080 to 1180 TFLOP/s, 4608 x
// 4096 x 4096 133 to 146 us; reading the input back in 16 bits and a product of the installed library 1.87 ms and 144 us on a
// card where these took 1.98 ms and 142 us: what is gained at that size is the input's memory. Small ones are bound by the
// latency of their first loads and steps (1024^3 12.8 us), adapters of rank 32 by both and the joining of parts (4096 x 32 x 4096
// 13.9 us for 17 MB; 4096 x 4096 x 32, of whose tiles three quarters hold no inputs, 15). fp32 gradients have four wavefronts a
// workgroup, one or two a SIMD: 4608 x 4096 x 4096 669 us, 231 TFLOP/s. What it took, at 16384 x 16384 x 4096:
// - Three stages in LDS and fragments that are read ahead, over a barrier in the middle of a stage (2493 -> 2131 us).
// - One conversion instruction a byte, and instructions spread between the products (2131 -> 2010 us): an MFMA of 16 cycles
//   hides three others of its SIMD, no more.
// - Conversion in one half of a stage and the writes to LDS in the other (2010 -> 1874 us): in one half they took 1310 of its
//   2040 cycles.
// - Eight wavefronts for the 128 x 128 tile: four, one a SIMD, wait for every LDS read (16384 x 1024 x 1024 253 -> 190 us).
// Not kept: fragments read three ahead, loads started earlier, raised wave priority (no difference); inputs laid out for
// stores of 32-bit sums in the 16-bit kernels (1930 us); acc in 4 wavefronts of 128 x 128 (the compiler spills).

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

// A stage holds the rows of N 16-bit values of some tokens. The 16 values of unit u lie in unit u ^ swizzle(t): the
// rows that a transposing read takes together, 4 of every 8, then lie in different LDS banks.
template <uint32_t N>
__device__ __forceinline__ constexpr uint32_t swizzle(uint32_t t) {
  if (N >= 128) return (t & 3) | (t >> 1 & 4);
  if (N == 64) return (t >> 1 & 1) | (t >> 2 & 2);
  return t >> 3 & 1;
}

typedef __attribute__((address_space(3))) s16x4_t* LdsRead;

// Where a lane's reads of unit 0 start. Unit u lies at this ^ 16 u: the other parts of the place have no bits there.
template <uint32_t N>
__device__ __forceinline__ uint32_t read_place() {
  const uint32_t lane = threadIdx.x & 63, t = lane / 16 * 8 + lane % 16 / 4;
  return t * N + swizzle<N>(t) * 16 + lane % 4 * 4;
}

// The fragment of unit u: lane l gets values of column l % 16, tokens 8 (l / 16) .. + 7.
template <uint32_t N>
__device__ __forceinline__ s16x8_t read_fragment(const short* stage, uint32_t place, uint32_t u) {
  const short* p = stage + (place ^ u * 16);
  const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsRead)p);
  const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsRead)(p + 4 * N));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Buffer resource of `rows` rows from p on, `ld` bytes apart, of which the last ends after `width` bytes: reads past that give 0.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_resource(const void* p, uint32_t ld, uint32_t rows, uint32_t width) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, rows > 0 ? (rows - 1) * ld + width : 0, 0x00020000);
}

// Stores N neighbouring values, or the first `count` of them.
template <typename T, uint32_t N>
__device__ __forceinline__ void store_run(T* out, const float (&v)[N], uint32_t count) {
  typedef T Run __attribute__((ext_vector_type(N)));
  typedef Run Any __attribute__((aligned(2)));
  if (count >= N) {
    Run x;
#pragma unroll
    for (uint32_t j = 0; j < N; ++j) x[j] = (T)v[j];
    *reinterpret_cast<Any*>(out) = x;
  } else {
#pragma unroll
    for (uint32_t j = 0; j < N; ++j)
      if (j < count) out[j] = (T)v[j];
  }
}

// f(0), f(1) .. f(N - 1) with constants for the compiler.
template <uint32_t I>
struct Constant {
  static constexpr uint32_t value = I;
};
template <uint32_t N, uint32_t I = 0, typename F>
__device__ __forceinline__ void each(const F& f) {
  if constexpr (I < N) {
    f(Constant<I>{});
    each<N, I + 1>(f);
  }
}

template <typename T, uint32_t TO, uint32_t TI, uint32_t WO, uint32_t WI, uint32_t kStep>
__device__ __forceinline__ void weight_grad(const sh::WeightGradArgs& a, short* lds) {
  using E = typename Multiplied<T>::Type;
  constexpr uint32_t kParts = Multiplied<T>::kParts;
  constexpr uint32_t kThreads = WO * WI * 64, FO = TO / WO / 16, FI = TI / WI / 16;
  static_assert(FI == 4, "a wavefront's inputs are one group of 64 permuted ones");
  constexpr uint32_t kDy = kStep * TO, kStage = kParts * kDy + kStep * TI, kGroups64 = TI / 64;
  constexpr uint32_t ND = kDy / 8 / kThreads, NX = kStep * TI / 16 / kThreads;
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t wo = wave / WI, wi = wave % WI;

  // XCDs take consecutive runs of tiles, which run down groups of kGroup tiles of outputs: an XCD's L2 then serves a block of
  // 4 x 8 tiles.
  constexpr uint32_t kGroup = 4;
  const uint32_t tiles_o = (a.out + TO - 1) / TO, tiles_i = (a.cols + TI - 1) / TI, tiles = tiles_o * tiles_i;
  const uint32_t all = tiles * a.splits, xcd = blockIdx.x % 8;
  const uint32_t p = xcd * (all / 8) + min(xcd, all % 8) + blockIdx.x / 8;
  const uint32_t split = p / tiles, tile = p % tiles;
  const uint32_t group = tile / (kGroup * tiles_i), in_group = tile % (kGroup * tiles_i), g_rows = min(tiles_o - group * kGroup, kGroup);
  const uint32_t o0 = (group * kGroup + in_group % g_rows) * TO, i0 = in_group / g_rows * TI;
  const uint32_t t_begin = split * a.split_tokens, t_end = min(a.tokens, t_begin + a.split_tokens);
  const uint32_t groups = (a.cols + SH_ACT8_GROUP - 1) / SH_ACT8_GROUP;

  // A stage on its way to LDS. The next one that is loaded starts at dy_at, q_at and e_at and has `left` tokens at most.
  struct Staged {
    typename Values8<T>::Vec dy[ND];
    uint4 q[NX];
    uint32_t e[NX];
  };
  const T* dy_at = static_cast<const T*>(a.dy) + t_begin * a.dy_ld + o0;
  const uint8_t* q_at = static_cast<const uint8_t*>(a.q) + (uint64_t)t_begin * groups * SH_ACT8_GROUP + i0;
  const uint8_t* e_at = static_cast<const uint8_t*>(a.exponent) + (uint64_t)t_begin * groups + i0 / SH_ACT8_GROUP;
  uint32_t left = t_begin < t_end ? t_end - t_begin : 0;
  const uint32_t dy_ld = (uint32_t)a.dy_ld * sizeof(T), q_ld = groups * SH_ACT8_GROUP;
  const uint32_t dy_t = threadIdx.x / (TO / 8), dy_o = threadIdx.x % (TO / 8) * 8;
  const uint32_t q_t = threadIdx.x / (TI / 16), q_i = threadIdx.x % (TI / 16) * 16;
  const uint32_t dy_off = dy_t * dy_ld + dy_o * sizeof(T), q_off = q_t * q_ld + q_i, e_off = q_t * groups + q_i / SH_ACT8_GROUP;
  const bool dy_odd = sizeof(T) == 2 && a.out % 2 != 0;
  constexpr uint32_t kDyRows = kThreads / (TO / 8), kQRows = kThreads / (TI / 16);
  auto load = [&](Staged& v) __attribute__((always_inline)) {
    const uint32_t rows = min(left, kStep);
    const auto qr = rows_resource(q_at, q_ld, rows, q_ld - i0), er = rows_resource(e_at, groups, rows, groups - i0 / SH_ACT8_GROUP);
#pragma unroll
    for (uint32_t j = 0; j < NX; ++j) {
      v.q[j] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(qr, q_off + j * kQRows * q_ld, 0, 0));
      v.e[j] = __builtin_amdgcn_raw_buffer_load_b8(er, e_off + j * kQRows * groups, 0, 0);
    }
    // An odd number of 16-bit values ends within a word, which is not read past the resource's end: where another row
    // follows, the resource ends after that word.
    const auto dr = rows_resource(dy_at, dy_ld, rows, (a.out - o0) * (uint32_t)sizeof(T) + (dy_odd && left > kStep ? 2 : 0));
#pragma unroll
    for (uint32_t j = 0; j < ND; ++j) {
      typedef uint32_t Words __attribute__((ext_vector_type(4 * sizeof(T) / 2)));
      Words w;
#pragma unroll
      for (uint32_t k = 0; k < sizeof(T) / 2; ++k) {
        const auto part = __builtin_amdgcn_raw_buffer_load_b128(dr, dy_off + j * kDyRows * dy_ld + k * 16, 0, 0);
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) w[k * 4 + i] = part[i];
      }
      v.dy[j] = __builtin_bit_cast(typename Values8<T>::Vec, w);
    }
    if (dy_odd && left <= kStep) {  // the last value of all is read by itself
#pragma unroll
      for (uint32_t j = 0; j < ND; ++j) {
        const uint32_t t = dy_t + j * kDyRows, last = a.out - 1 - o0 - dy_o;
        if (t + 1 != rows || last >= 8) continue;
        const T value = dy_at[t * a.dy_ld + dy_o + last];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
          if (i == last) v.dy[j][i] = value;
      }
    }
    dy_at += kStep * a.dy_ld;
    q_at += kStep * q_ld;
    e_at += kStep * groups;
    left -= rows;
  };
  typedef E Out4 __attribute__((ext_vector_type(4)));
  typedef E Out8 __attribute__((ext_vector_type(8)));
  // Sums over the tokens that a work-item stages: always of the same 8 outputs.
  const bool with_bias = a.dbias != nullptr && i0 == 0;
  float bias[8] = {};
  const uint32_t dy_place = dy_t * TO + ((dy_o / 16) ^ swizzle<TO>(dy_t)) * 16 + dy_o % 16;
  static_assert(kDyRows % 16 == 0 || ND == 1, "a work-item's rows have one swizzle");
  auto add_bias = [&](const Staged& v) __attribute__((always_inline)) {
    if (!with_bias) return;
#pragma unroll
    for (uint32_t j = 0; j < ND; ++j)
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) bias[i] += (float)v.dy[j][i];
  };
  auto put_dy = [&](const Staged& v, short* stage, uint32_t j) __attribute__((always_inline)) {
    short* at = stage + dy_place + j * kDyRows * TO;
    if constexpr (kParts == 1) {
      *reinterpret_cast<typename Values8<T>::Vec*>(at) = v.dy[j];
    } else {
      float rest[8];
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) rest[i] = v.dy[j][i];
#pragma unroll
      for (uint32_t part = 0; part < kParts; ++part) {
        Out8 out;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {  // the next 8 significant bits, as far as bf16 has them; all of an infinity
          const float head = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, rest[i]) & 0xFFFF0000u);
          out[i] = (E)head;
          rest[i] = rest[i] == head ? 0.0f : rest[i] - head;
        }
        *reinterpret_cast<Out8*>(at + part * kDy) = out;
      }
    }
  };
  // Unit j * kGroups64 + g is fragment j of the group g of 64 columns. It holds columns 16 p + 4 j + m of the group, at 4 p + m:
  // a lane of the product then has 16 consecutive inputs for 16-byte stores of 16-bit values. Or, for gradients in fp32, which
  // are stored as such, columns 16 j + 4 p + m: the lanes' 4 consecutive inputs of a fragment lie side by side (4608 x 4096 x
  // 4096 683 -> 665 us).
  static_assert(kQRows % 16 == 0 || NX == 1, "a work-item's rows have one swizzle");
  constexpr bool kSpread = sizeof(T) == 2;
  constexpr uint32_t kXStep = kSpread ? kGroups64 * 16 : 4;
  const uint32_t q_c = q_i / 16;
  const uint32_t x_place = q_t * TI + ((kSpread ? q_c / 4 : q_c % 4 * kGroups64 + q_c / 4) ^ swizzle<TI>(q_t)) * 16 + (kSpread ? q_c % 4 * 4 : 0);
  // In two steps, as their instructions hide behind products of different halves of a stage.
  Out4 packed[NX][4];
  auto convert_x = [&](const Staged& v, uint32_t j, uint32_t f) __attribute__((always_inline)) {
    const uint32_t words[4] = {v.q[j].x, v.q[j].y, v.q[j].z, v.q[j].w};
    float x[4];
    dequantize4(words[f], group_scale(v.e[j]), x);
#pragma unroll
    for (uint32_t m = 0; m < 4; ++m) packed[j][f][m] = (E)x[m];
  };
  auto put_x = [&](short* stage, uint32_t j, uint32_t f) __attribute__((always_inline)) {
    *reinterpret_cast<Out4*>(stage + kParts * kDy + (x_place ^ f * kXStep) + j * kQRows * TI) = packed[j][f];
  };
  static_assert(kStep * TI / 16 % kThreads == 0 && kDy / 8 % kThreads == 0, "every work-item stages inputs and gradients");
  const uint32_t x_read = read_place<TI>() ^ wi * 16, dy_read = read_place<TO>() ^ wo * FO * 16;
  // Fragment j of x^, of the stage's tokens 32 k .. 32 k + 31.
  auto read_x = [&](const short* stage, uint32_t k, uint32_t j) __attribute__((always_inline)) {
    return read_fragment<TI>(stage + kParts * kDy + k * 32 * TI, x_read, j * kGroups64);
  };
  // Fragment b of dy: of tokens 32 (b / kOf32) on, of part b % kOf32 / FO.
  constexpr uint32_t kOf32 = kParts * FO;
  auto read_dy = [&](const short* stage, uint32_t b) __attribute__((always_inline)) {
    return read_fragment<TO>(stage + b % kOf32 / FO * kDy + b / kOf32 * 32 * TO, dy_read, b % FO);
  };

  f32x4_t acc[FO][FI] = {};
  // A stage's products go in NB blocks, one for each fragment of dy, which is read kAhead blocks before. The blocks before
  // block kBarrier also write the next stage to LDS and start the loads of the one after the next two. After the barrier the
  // next stage's first fragments are read and the inputs of the one after it converted. A third stage of LDS is written
  // while the other two are read. The instructions of a block are spread between its products: all at once they would
  // hold up the products of both wavefronts of a SIMD.
  constexpr uint32_t K32 = kStep / 32, NB = K32 * kOf32, kBarrier = K32 == 1 ? NB / 2 : NB - kOf32;
  constexpr uint32_t kAhead = NB - kBarrier < 2 ? NB - kBarrier : 2, kFirstHalf = kBarrier > 0 ? kBarrier : 1, kWrites = NX * 4 + ND;
  static_assert(K32 == 1 || K32 % 2 == 0, "stages start with the same half of x");
  Staged staged[2];
  s16x8_t x[2][FI], d[NB + kAhead];
  auto multiply = [&](auto turn, uint32_t s) __attribute__((always_inline)) {
    constexpr uint32_t V = decltype(turn)::value;
    const short* stage = lds + s * kStage;
    short* next = lds + (s == 2 ? 0 : s + 1) * kStage;
    each<NB>([&](auto block) __attribute__((always_inline)) {
      constexpr uint32_t B = decltype(block)::value, K = B / kOf32, X = K32 == 1 ? V : K % 2;
      if constexpr (B == 0) add_bias(staged[V ^ 1]);
      if constexpr (B < kFirstHalf) {
        each<(B + 1) * kWrites / kFirstHalf, B * kWrites / kFirstHalf>([&](auto w) __attribute__((always_inline)) {
          constexpr uint32_t I = decltype(w)::value;
          if constexpr (I < NX * 4) put_x(next, I / 4, I % 4);
          else put_dy(staged[V ^ 1], next, I - NX * 4);
        });
        if constexpr (B == kFirstHalf - 1) load(staged[V ^ 1]);
      }
      if constexpr (B + kAhead < NB) d[B + kAhead] = read_dy(stage, B + kAhead);
      if constexpr (B == kBarrier) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      }
      // the other half of x: of the next 32 tokens, or of the next stage
      constexpr uint32_t kLead = K + 1 < K32 ? K * kOf32 : kBarrier, kOf = (K + 1 < K32 ? kLead + kOf32 : NB) - kLead;
      if constexpr (B >= kLead) {
        each<(B - kLead + 1) * FI / kOf, (B - kLead) * FI / kOf>([&](auto j) __attribute__((always_inline)) {
          constexpr uint32_t J = decltype(j)::value;
          x[X ^ 1][J] = K + 1 < K32 ? read_x(stage, K + 1, J) : read_x(next, 0, J);
        });
      }
      if constexpr (B >= kBarrier) {
        constexpr uint32_t kFirst = (B - kBarrier) * NX * 4 / (NB - kBarrier), kLast = (B - kBarrier + 1) * NX * 4 / (NB - kBarrier);
        each<kLast, kFirst>([&](auto c) __attribute__((always_inline)) { convert_x(staged[V], decltype(c)::value / 4, decltype(c)::value % 4); });
      }
      if constexpr (B + kAhead >= NB) d[B + kAhead] = read_dy(next, B + kAhead - NB);
      each<FI>([&](auto j) __attribute__((always_inline)) {
        constexpr uint32_t J = decltype(j)::value;
        acc[B % FO][J] = mfma<E>(x[X][J], d[B], acc[B % FO][J]);
      });
      each<FI>([&](auto) __attribute__((always_inline)) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // an LDS read
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a product
        __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);  // VALU
        __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);  // an LDS write
        __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // a load
      });
      __builtin_amdgcn_sched_barrier(0);
    });
#pragma unroll
    for (uint32_t b = 0; b < kAhead; ++b) d[b] = d[NB + b];
  };
  load(staged[0]);
  add_bias(staged[0]);
  auto convert_all = [&](const Staged& v) __attribute__((always_inline)) {
    each<NX * 4>([&](auto i) __attribute__((always_inline)) { convert_x(v, decltype(i)::value / 4, decltype(i)::value % 4); });
  };
  convert_all(staged[0]);
  each<NX * 4>([&](auto i) __attribute__((always_inline)) { put_x(lds, decltype(i)::value / 4, decltype(i)::value % 4); });
  each<ND>([&](auto j) __attribute__((always_inline)) { put_dy(staged[0], lds, decltype(j)::value); });
  load(staged[1]);
  load(staged[0]);
  convert_all(staged[1]);
  __syncthreads();
#pragma unroll
  for (uint32_t j = 0; j < FI; ++j) x[0][j] = read_x(lds, 0, j);
#pragma unroll
  for (uint32_t b = 0; b < kAhead; ++b) d[b] = read_dy(lds, b);
  uint32_t s = 0;
  for (uint32_t t0 = t_begin; t0 < t_end; t0 += 2 * kStep) {
    multiply(Constant<0>{}, s);
    s = s == 2 ? 0 : s + 1;
    multiply(Constant<1>{}, s);
    s = s == 2 ? 0 : s + 1;
  }

  // lane: output l % 16 of each fragment of outputs
  float* sums = a.partials;
  if (sums != nullptr) sums += split * ((uint64_t)a.out * a.cols + (a.dbias != nullptr ? a.out : 0));
  const uint32_t part = lane / 16, first = i0 + wi * (TI / WI);
#pragma unroll
  for (uint32_t f = 0; f < FO; ++f) {
    const uint32_t o = o0 + wo * (TO / WO) + f * 16 + lane % 16;
    if (o >= a.out) continue;
    // neighbouring sums, of inputs i on
    auto store = [&](const auto& v, uint32_t i) __attribute__((always_inline)) {
      constexpr uint32_t N = sizeof(v) / 4;
      const uint32_t n = i < a.cols ? a.cols - i : 0;
      if (sums != nullptr) return store_run<float, N>(sums + (uint64_t)o * a.cols + i, v, n);
      const uint64_t at = o * a.dw_ld + i;
      if (a.out_dtype == SH_DTYPE_BF16) store_run<__bf16, N>(static_cast<__bf16*>(a.dweight) + at, v, n);
      else if (a.out_dtype == SH_DTYPE_F16) store_run<_Float16, N>(static_cast<_Float16*>(a.dweight) + at, v, n);
      else store_run<float, N>(static_cast<float*>(a.dweight) + at, v, n);
    };
    if constexpr (kSpread) {
#pragma unroll
      for (uint32_t h = 0; h < 2; ++h) {
        float v[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) v[j] = acc[f][h * 2 + j / 4][j % 4];
        store(v, first + part * 16 + h * 8);
      }
    } else {
#pragma unroll
      for (uint32_t j = 0; j < FI; ++j) {
        const float v[4] = {acc[f][j][0], acc[f][j][1], acc[f][j][2], acc[f][j][3]};
        store(v, first + j * 16 + part * 4);
      }
    }
  }
  if (!with_bias) return;
  // an output's sums, in their order
  __syncthreads();  // the stages are not read any more
  float* sum = reinterpret_cast<float*>(lds);
#pragma unroll
  for (uint32_t k = 0; k < 8; ++k) sum[dy_t * TO + dy_o + k] = bias[k];
  __syncthreads();
  for (uint32_t k = threadIdx.x; k < TO; k += kThreads) {
    const uint32_t o = o0 + k;
    if (o >= a.out) continue;
    float v = 0.0f;
#pragma unroll
    for (uint32_t r = 0; r < kDyRows; ++r) v += sum[r * TO + k];
    if (sums != nullptr) sums[(uint64_t)a.out * a.cols + o] = v;
    else if (a.out_dtype == SH_DTYPE_BF16) static_cast<__bf16*>(a.dbias)[o] = (__bf16)v;
    else if (a.out_dtype == SH_DTYPE_F16) static_cast<_Float16*>(a.dbias)[o] = (_Float16)v;
    else static_cast<float*>(a.dbias)[o] = v;
  }
}

}  // namespace

// The tiles of sh_act8_args.h.
#define SH_WEIGHT_GRAD(name, T, TO, TI, WO, WI, STEP)                                                             \
  extern "C" __global__ __launch_bounds__(WO * WI * 64, 2) void sh_weight_grad_##name##_##TO##x##TI##_kernel(sh::WeightGradArgs a) { \
    __shared__ alignas(16) short lds[3 * STEP * (Multiplied<T>::kParts * TO + TI)];                               \
    weight_grad<T, TO, TI, WO, WI, STEP>(a, lds);                                                                 \
  }
SH_WEIGHT_GRAD(bf16, __bf16, 32, 128, 2, 2, 128)
SH_WEIGHT_GRAD(bf16, __bf16, 64, 128, 4, 2, 64)
SH_WEIGHT_GRAD(bf16, __bf16, 128, 128, 4, 2, 64)
SH_WEIGHT_GRAD(bf16, __bf16, 256, 256, 2, 4, 32)
SH_WEIGHT_GRAD(f16, _Float16, 32, 128, 2, 2, 128)
SH_WEIGHT_GRAD(f16, _Float16, 64, 128, 4, 2, 64)
SH_WEIGHT_GRAD(f16, _Float16, 128, 128, 4, 2, 64)
SH_WEIGHT_GRAD(f16, _Float16, 256, 256, 2, 4, 32)
SH_WEIGHT_GRAD(f32, float, 32, 128, 2, 2, 64)
SH_WEIGHT_GRAD(f32, float, 64, 128, 2, 2, 32)
SH_WEIGHT_GRAD(f32, float, 128, 128, 2, 2, 32)

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
