// Int8 kernels for gfx950 (device code only; the checks and the launches are in sh_int8.cpp):
// quantisation of tokens and the product with a SquareQ weight.
//
//   tokens:   a_t = max_k |x_tk|,  q_tk = rint(x_tk (127 / a_t)),  s_t = a_t / 127,  sum_t = sum_k q_tk
//   product:  y_tn = s_t w_n (sum_k q_tk Q_nk - z_n sum_t) + b_n   for W_nk = (Q_nk - z_n) w_n
//
// The sums are exact, in 32-bit integers, so they may be taken in any order and split in any way; scales, zero
// points and bias come once at the end, in fp32, and one rounding to the output's type.
//
// Three regimes. Quantisation reads 2 (4) bytes a value and writes 1: HBM. Few tokens: the weight's bytes from
// HBM. Many tokens: the matrix cores, which on random int8 values reach 3.9 P operations a second on this chip
// without any memory traffic (4.9 P on zeros: the clock falls with the power that the operands take).

#include <hip/hip_runtime.h>

#include <cstdint>

#include "sh_int8_args.h"
#include "stagehand_native.h"

namespace {

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

// A token's scale as a factor for the rows' scales, within 2^-64 and 2^65, and what is left, a power of two, for the
// token's sums (1 for all ordinary scales): the outputs are (sum on_sum) (w on_row) + bias. scale * w by itself
// would overflow, or lose its bits below 2^-126, where the output is an ordinary number: scales go from 2^-127 to
// 2^121. These products do so only for rows' scales under 2^-62 or over 2^62.
struct TokenFactors {
  float on_sum, on_row;
};
__device__ __forceinline__ bool ordinary(float scale) { return scale >= 0x1p-64f && scale < 0x1p65f; }
__device__ __forceinline__ TokenFactors token_factors(float scale) {
  if (ordinary(scale)) return {1.0f, scale};
  const uint32_t e = __builtin_bit_cast(uint32_t, scale) >> 23 & 0xFF, near = min(max(e, 127u - 64), 127u + 64);
  const uint32_t rest = 127 + max(e, 1u) - near;  // subnormal scales have the exponent 1, too
  return {__builtin_bit_cast(float, rest << 23), scale * __builtin_bit_cast(float, (254 - rest) << 23)};
}

// ── quantisation ──────────────────────────────────────────────────────────

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));

// Eight consecutive values of a token as they lie in memory. gfx950 loads 16 bytes from any address.
template <typename T>
struct Chunk {
  static constexpr uint32_t kWords = sizeof(T) * 2;
  uint32_t w[kWords];

  // The first `count` of them; the rest are 0. `beyond`: memory goes on for eight values past the end.
  __device__ __forceinline__ void load(const T* p, uint32_t count, bool beyond) {
    if (count >= 8 || (beyond && count > 0)) {
#pragma unroll
      for (uint32_t i = 0; i < kWords / 4; ++i) {
        const u32x4 v = *(reinterpret_cast<const u32x4_a2*>(p) + i);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) w[i * 4 + j] = v[j];
      }
      if (count < 8) {
#pragma unroll
        for (uint32_t i = 0; i < kWords; ++i) {
          if constexpr (sizeof(T) == 4) w[i] = i < count ? w[i] : 0;
          else w[i] &= 2 * i + 1 < count ? 0xFFFFFFFFu : 2 * i < count ? 0xFFFFu : 0;
        }
      }
    } else {
#pragma unroll
      for (uint32_t i = 0; i < kWords; ++i) w[i] = 0;
      if (count == 0) return;
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
          if (i < count) w[i] = __builtin_bit_cast(uint32_t, p[i]);
      } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
          if (i < count) w[i / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, p[i]) << (i % 2 * 16);
      }
    }
  }

  // The largest of m and the magnitudes' bits (16-bit types: two maxima side by side). Bits order as
  // magnitudes do, with infinities and NaNs last: a maximum of floats would pass over a NaN.
  __device__ __forceinline__ uint32_t amax(uint32_t m) const {
#pragma unroll
    for (uint32_t i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4) {
        m = max(m, w[i] & 0x7FFFFFFFu);
      } else {
        const u16x2 v = __builtin_bit_cast(u16x2, w[i] & 0x7FFF7FFFu);
        m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m), v));
      }
    }
    return m;
  }

  __device__ __forceinline__ float value(uint32_t i) const {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, w[i]);
    else if constexpr (__is_same(T, __bf16))
      return __builtin_bit_cast(float, i % 2 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    else return (float)__builtin_bit_cast(T, (uint16_t)(w[i / 2] >> (i % 2 * 16)));
  }

  // rint(x * inv) of the eight values as bytes. |x * inv| is at most 127 (1 + 2^-23): added to 1.5 * 2^23 it is
  // rounded to an integer, ties to even, that the sum's low byte holds. `mask` is 0 for a token of zeros or
  // with a NaN or an infinity, else all ones.
  __device__ __forceinline__ uint2 quantize(float inv, uint32_t mask) const {
#pragma clang fp contract(off)  // the product is rounded before the sum
    uint32_t b[8];
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const float p = value(i) * inv;
      b[i] = __builtin_bit_cast(uint32_t, p + 12582912.0f);
    }
    uint2 q;
    q.x = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0C0C0400u), __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400u), 0x05040100u) & mask;
    q.y = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[7], b[6], 0x0C0C0400u), __builtin_amdgcn_perm(b[5], b[4], 0x0C0C0400u), 0x05040100u) & mask;
    return q;
  }
};

// The bits of the larger float magnitude from amax()'s word.
template <typename T>
__device__ __forceinline__ uint32_t amax_bits(uint32_t m) {
  if constexpr (sizeof(T) == 4) return m;
  const uint32_t h = max(m & 0xFFFFu, m >> 16);
  if constexpr (__is_same(T, __bf16)) return h << 16;
  return __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(_Float16, (uint16_t)h));
}

// The maximum and the sum over a wavefront, by data-parallel primitives: within rows of 16 lanes every step adds
// a half that already agrees, then rows 0 and 2 are carried into 1 and 3 and the lower half into the upper.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t otherwise, uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)otherwise, (int)v, CTRL, ROWS, 0xF, false);
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = max(v, moved<0xB1, 0xF>(v, v));   // quad_perm 1,0,3,2
  v = max(v, moved<0x4E, 0xF>(v, v));   // quad_perm 2,3,0,1
  v = max(v, moved<0x141, 0xF>(v, v));  // row_half_mirror
  v = max(v, moved<0x140, 0xF>(v, v));  // row_mirror
  v = max(v, moved<0x142, 0xA>(v, v));  // row_bcast:15
  v = max(v, moved<0x143, 0xC>(v, v));  // row_bcast:31
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

__device__ __forceinline__ int32_t wave_sum(int32_t s) {
  uint32_t v = (uint32_t)s;
  v += moved<0xB1, 0xF>(0, v);
  v += moved<0x4E, 0xF>(0, v);
  v += moved<0x141, 0xF>(0, v);
  v += moved<0x140, 0xF>(0, v);
  v += moved<0x142, 0xA>(0, v);
  v += moved<0x143, 0xC>(0, v);
  return (int32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// Whether a token's end may be read eight values too far: another token of at least as many lies behind it.
__device__ __forceinline__ bool goes_on(uint32_t t, uint32_t tokens, uint64_t ld, uint32_t cols) {
  return t + 1 < tokens && ld >= cols && cols >= 8;
}

// WAVES wavefronts per token, C chunks of each work-item in registers between the maximum and the rounding:
// the token is read once if its cols are at most WAVES * 512 * C, else its end is read twice (the second time
// out of a cache). Bound by HBM: 16384 x 16384 bf16 145 us (5.6 TB/s), 8192 x 8192 31 us (6.5 TB/s, part of it
// from the memory-side cache). A workgroup of 256 for every token, with two passes over it: 590 and 116 us.
template <typename T, uint32_t WAVES, uint32_t C>
__device__ __forceinline__ void quantize_body(const sh::QuantizeArgs& a) {
  constexpr uint32_t kWide = WAVES * 64;  // chunks side by side
  const uint32_t wave = threadIdx.x / 64;
  const uint32_t t = WAVES == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
  const uint32_t me = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
  if (WAVES == 1 && t >= a.tokens) return;
  const T* x = static_cast<const T*>(a.x) + (uint64_t)t * a.x_ld;
  const uint32_t chunks = (uint32_t)(a.q_ld / 8);  // past cols they are zeros
  auto left = [&](uint32_t c) { return c * 8 < a.cols ? a.cols - c * 8 : 0; };
  const bool beyond = goes_on(t, a.tokens, a.x_ld, a.cols);
  Chunk<T> held[C];
  uint32_t m = 0;
#pragma unroll
  for (uint32_t j = 0; j < C; ++j) held[j].load(x + (uint64_t)(j * kWide + me) * 8, left(j * kWide + me), beyond);
#pragma unroll
  for (uint32_t j = 0; j < C; ++j) m = held[j].amax(m);
  for (uint32_t c = C * kWide + me; c < chunks; c += kWide) {
    Chunk<T> v;
    v.load(x + (uint64_t)c * 8, left(c), beyond);
    m = v.amax(m);
  }
  m = wave_max(amax_bits<T>(m));
  __shared__ uint32_t part[4];
  __shared__ int32_t part_sum[4];
  if constexpr (WAVES > 1) {
    if ((threadIdx.x & 63) == 0) part[wave] = m;
    __syncthreads();
    m = max(max(part[0], part[1]), max(part[2], part[3]));
  }
  float inv, scale;
  token_scale(m, &inv, &scale);
  const uint32_t mask = inv == 0.0f ? 0u : ~0u;
  uint2* q = reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.q) + (uint64_t)t * a.q_ld);
  int32_t sum = 0;
  auto put = [&](const Chunk<T>& v, uint32_t c) {
    const uint2 b = v.quantize(inv, mask);
    sum = __builtin_amdgcn_sdot4((int)b.x, 0x01010101, sum, false);
    sum = __builtin_amdgcn_sdot4((int)b.y, 0x01010101, sum, false);
    q[c] = b;
  };
#pragma unroll
  for (uint32_t j = 0; j < C; ++j)
    if (j * kWide + me < chunks) put(held[j], j * kWide + me);
  for (uint32_t c = C * kWide + me; c < chunks; c += kWide) {
    Chunk<T> v;
    v.load(x + (uint64_t)c * 8, left(c), beyond);
    put(v, c);
  }
  sum = wave_sum(sum);
  if constexpr (WAVES > 1) {
    if ((threadIdx.x & 63) == 0) part_sum[wave] = sum;
    __syncthreads();
    sum = part_sum[0] + part_sum[1] + part_sum[2] + part_sum[3];
  }
  if (me == 0) {
    a.scale[t] = scale;
    if (a.sums != nullptr) a.sums[t] = sum;
  }
}

}  // namespace

#define SH_QUANTIZE(name, T)                                                                              \
  extern "C" __global__ __launch_bounds__(256) void sh_quantize_##name##_512_kernel(sh::QuantizeArgs a) {  \
    quantize_body<T, 1, 1>(a);                                                                            \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(256) void sh_quantize_##name##_2048_kernel(sh::QuantizeArgs a) { \
    quantize_body<T, 1, 4>(a);                                                                            \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(256) void sh_quantize_##name##_4096_kernel(sh::QuantizeArgs a) { \
    quantize_body<T, 1, 8>(a);                                                                            \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(256) void sh_quantize_##name##_16384_kernel(sh::QuantizeArgs a) { \
    quantize_body<T, 4, 8>(a);                                                                            \
  }
SH_QUANTIZE(bf16, __bf16)
SH_QUANTIZE(f16, _Float16)
SH_QUANTIZE(f32, float)

// ── the tiled product ─────────────────────────────────────────────────────

namespace {

typedef int32_t i32x4_t __attribute__((ext_vector_type(4)));

constexpr uint32_t kPastEnd = 0x80000000u;  // an offset outside every resource
constexpr uint32_t kStep = 128;  // bytes of a row that one stage holds: a cache line, two MFMAs'

// Bytes of a quantised token that are multiplied: whole steps, zeros past cols. How far apart the tokens lie has no
// part in it.
__device__ __forceinline__ constexpr uint32_t token_bytes(uint32_t cols) { return (cols + kStep - 1) / kStep * kStep; }

// The 16-byte chunk c of a stage's row lies in slot c ^ swizzle(row): the 16 rows of a fragment then lie in
// different LDS banks.
__device__ __forceinline__ constexpr uint32_t swizzle(uint32_t row) { return (row >> 1) & 7; }

// Buffer resource of up to `tile` rows from row `first` on, each `width` of the `ld` bytes to the next: reads past
// the last row's width give 0.
__device__ __forceinline__ i32x4_t rows_resource(const void* base, uint64_t ld, uint64_t width, uint32_t first,
                                                 uint32_t count, uint32_t tile) {
  const uint64_t p = (uint64_t)base + (uint64_t)first * ld;
  i32x4_t r;
  r[0] = __builtin_amdgcn_readfirstlane((int32_t)(uint32_t)p);
  r[1] = __builtin_amdgcn_readfirstlane((int32_t)(uint32_t)(p >> 32) & 0xFFFF);  // stride 0
  r[2] = __builtin_amdgcn_readfirstlane((int32_t)(uint32_t)((min(count - first, tile) - 1) * ld + width));
  r[3] = 0x00020000;
  return r;
}

// Brings 16 bytes per lane from the resource into LDS, at lds (in M0) + 16 * lane. Written as assembly: the compiler
// would wait for the load before the next LDS read, whatever stage that reads. It has no output register;
// whoever reads the stage waits for it (vmcnt) and for the barrier after that. The whole offset is in the register
// that the resource's range check covers.
__device__ __forceinline__ void load_to_lds(i32x4_t r, uint32_t lds, uint32_t offset) {
  asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"{m0}"(lds), "v"(offset), "s"(r));
}

// Stores N consecutive values, or the first `count` of them. Whole runs are stored as vectors whatever their
// address (gfx950 stores vectors anywhere).
template <typename T, uint32_t N>
__device__ __forceinline__ void store_run(T* out, const float (&v)[N], uint32_t count) {
  constexpr uint32_t kPer = N * sizeof(T) < 16 ? N : 16 / sizeof(T);
  typedef T Run __attribute__((ext_vector_type(kPer)));
  typedef Run RunAny __attribute__((aligned(2)));
  if (count >= N) {
#pragma unroll
    for (uint32_t i = 0; i < N / kPer; ++i) {
      Run x;
#pragma unroll
      for (uint32_t j = 0; j < kPer; ++j) x[j] = (T)v[i * kPer + j];
      *reinterpret_cast<RunAny*>(out + i * kPer) = x;
    }
  } else {
#pragma unroll
    for (uint32_t j = 0; j < N; ++j)
      if (j < count) out[j] = (T)v[j];
  }
}

// f(0), f(1) .. f(N - 1) with constants for the compiler: registers are not indexed at run time whatever it unrolls.
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

// TT tokens x TN rows by WT x WN wavefronts, each with FT x FN MFMA tiles; D stages. XCDs take consecutive runs of
// tiles, which run down groups of GROUP tiles in the tokens: an XCD's L2 then serves a block of 4 x 8 tiles (16384 x
// 4096 x 16384: 780 us in groups of 4, 850 of 8).
//
// Bound by the matrix cores and their clock. 16384 x 4096 x 16384: 773 us, 2840 TOPS, the MFMA pipes busy 77% of
// the cycles at 1.76 GHz, no LDS bank conflicts, 81% of the L2 reads hits. What it took, at that size or at 4608 x
// 21504 x 3072:
// - Loads of whole 128-byte lines per row. Rows of 64 bytes reach half the L2's rate (16.5 against 30 to 35
//   TB/s), and a ring of five such stages 2050 TOPS.
// - Loads straight to LDS, fragments double-buffered in registers: an LDS read is waited for a half stage later.
// - Reads and loads spread between the MFMAs (863 -> 773 us).
// - A permutation of the weight's rows that leaves every lane 16 consecutive outputs, 16-byte stores: 2-byte
//   stores took 34 us a tile.
// - 16x16x64 MFMAs: with 32x32x32 ones the cores alone reach 2.6 P operations a second, with these 3.9.
// A workgroup that goes on to its next tile with that tile's first stages on their way was no faster (274 us
// against 268), nor a third stage of tokens, nor raised wave priority around the MFMAs.
template <uint32_t TT, uint32_t TN, uint32_t WT, uint32_t WN, uint32_t D, uint32_t GROUP>
__device__ __forceinline__ void matmul_tile(const sh::MatmulI8Args& a, uint8_t* lds) {
  constexpr uint32_t kStage = (TT + TN) * kStep;
  constexpr uint32_t kWaves = WT * WN;
  constexpr uint32_t FT = TT / WT / 16, FN = TN / WN / 16;
  constexpr uint32_t LT = TT / 8 / kWaves, LN = TN / 8 / kWaves, kLoads = LT + LN;  // of 8 rows per wavefront
  static_assert(FN == 4, "a wavefront's rows are one group of 64 permuted ones");
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t tiles_t = (a.tokens + TT - 1) / TT, tiles_n = (a.rows + TN - 1) / TN, tiles = tiles_t * tiles_n;
  const uint32_t xcd = blockIdx.x % 8;
  const uint32_t p = xcd * (tiles / 8) + min(xcd, tiles % 8) + blockIdx.x / 8;
  const uint32_t group = p / (GROUP * tiles_n), in_group = p % (GROUP * tiles_n);
  const uint32_t g_rows = min(tiles_t - group * GROUP, GROUP);
  const uint32_t t0 = (group * GROUP + in_group % g_rows) * TT, n0 = in_group / g_rows * TN;
  const uint32_t end = token_bytes(a.cols);
  const i32x4_t tr = rows_resource(a.tq, a.t_ld, end, t0, a.tokens, TT);
  const i32x4_t wr = rows_resource(a.wq, a.w_ld, a.w_ld, n0, a.rows, TN);

  // Lane l of a load brings slot l % 8 of row l / 8. The rows of the weight lie permuted in LDS, so that the
  // MFMA results of one lane are 16 consecutive ones: fragment f, row i holds row (i / 4) * 16 + f * 4 + i % 4
  // of the wavefront's 64.
  uint32_t t_off[LT], n_off[LN];
  each<LT>([&](auto j) __attribute__((always_inline)) {
    const uint32_t row = (decltype(j)::value * kWaves + wave) * 8 + lane / 8;
    t_off[decltype(j)::value] = row * (uint32_t)a.t_ld + ((lane % 8) ^ swizzle(row)) * 16;
  });
  each<LN>([&](auto j) __attribute__((always_inline)) {
    const uint32_t row = (decltype(j)::value * kWaves + wave) * 8 + lane / 8;
    const uint32_t src = row / 64 * 64 + row % 16 / 4 * 16 + row / 16 % 4 * 4 + row % 4;
    n_off[decltype(j)::value] = src * (uint32_t)a.w_ld + ((lane % 8) ^ swizzle(row)) * 16;
  });
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + wave * 1024;
  // Load i of a stage: first the tokens', then the rows'. Past the end the offset is outside the resource: such
  // a load reads nothing and keeps the count of loads in flight the same.
  auto load = [&](auto i, uint32_t stage, uint32_t k) __attribute__((always_inline)) {
    constexpr uint32_t I = decltype(i)::value;
    k = k < end ? k : kPastEnd;
    if constexpr (I < LT) load_to_lds(tr, lds0 + stage * kStage + I * kWaves * 1024, t_off[I] + k);
    else load_to_lds(wr, lds0 + stage * kStage + TT * kStep + (I - LT) * kWaves * 1024, n_off[I - LT] + k);
  };
  const uint32_t l16 = lane & 15, part = lane / 16;
  const uint32_t wt = wave / WN, wn = wave % WN;
  i32x4_t acc[FT][FN] = {};
  const uint8_t* t_at = lds + (wt * (TT / WT) + l16) * kStep;
  const uint8_t* n_at = lds + (TT + wn * (TN / WN) + l16) * kStep;
  struct Fragments {
    i32x4_t t[FT], n[FN];
  };
  uint32_t s = 0;  // the stage that is multiplied
  // Read i of a half stage: first the rows' fragments, then the tokens'.
  auto read = [&](Fragments& f, auto i, uint32_t half) __attribute__((always_inline)) {
    constexpr uint32_t I = decltype(i)::value;
    const uint32_t slot = ((half * 4 + part) ^ swizzle(l16)) * 16 + s * kStage;
    if constexpr (I < FN) f.n[I] = *reinterpret_cast<const i32x4_t*>(n_at + slot + I * 16 * kStep);
    else f.t[I - FN] = *reinterpret_cast<const i32x4_t*>(t_at + slot + (I - FN) * 16 * kStep);
  };
  // The products of one half stage, in FT parts. Each part starts the LDS reads (READS) and the loads (LOADS)
  // that its products hide: all at once they would hold up the products of both wavefronts of a SIMD.
  auto multiply = [&](auto reads, auto loads, const Fragments& f, Fragments& next, uint32_t half, uint32_t stage,
                      uint32_t k) __attribute__((always_inline)) {
    each<FT>([&](auto part_of) __attribute__((always_inline)) {
      constexpr uint32_t I = decltype(part_of)::value;
      if constexpr (decltype(reads)::value) {
        constexpr uint32_t kFrom = I * (FT + FN) / FT, kTo = (I + 1) * (FT + FN) / FT;
        each<kTo, kFrom>([&](auto r) __attribute__((always_inline)) { read(next, r, half); });
      }
      if constexpr (decltype(loads)::value) {
        constexpr uint32_t kFrom = I * kLoads / FT, kTo = (I + 1) * kLoads / FT;
        each<kTo, kFrom>([&](auto l) __attribute__((always_inline)) { load(l, stage, k); });
      }
      each<FN>([&](auto j) __attribute__((always_inline)) {
        constexpr uint32_t J = decltype(j)::value;
        acc[I][J] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f.n[J], f.t[I], acc[I][J], 0, 0, 0);
      });
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  constexpr Constant<0> kNo;
  constexpr Constant<1> kYes;
  // A ring of D stages. The fragments of a half stage are read into registers while the half before is
  // multiplied, so a stage is read to its end when the first half of its products is done: the loads that take
  // its place start there and have the products of D - 1 stages to land in.
  // Each wavefront waits for its own loads of the next stage, then the barrier says that everyone's have landed
  // and that everyone has read the stage whose place the next loads take.
  Fragments f0, f1;
  each<D>([&](auto d) __attribute__((always_inline)) {
    each<kLoads>([&](auto i) __attribute__((always_inline)) { load(i, decltype(d)::value, decltype(d)::value * kStep); });
  });
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 1) * kLoads) : "memory");
  __syncthreads();
  each<FT + FN>([&](auto i) __attribute__((always_inline)) { read(f0, i, 0); });
  for (uint32_t k = 0; k + kStep < end; k += kStep) {
    multiply(kYes, kNo, f0, f1, 1, 0, 0);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 2) * kLoads) : "memory");
    __syncthreads();
    const uint32_t free = s;
    s = s == D - 1 ? 0 : s + 1;
    multiply(kYes, kYes, f1, f0, 0, free, k + D * kStep);
  }
  multiply(kYes, kNo, f0, f1, 1, 0, 0);
  multiply(kNo, kNo, f1, f0, 0, 0, 0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load may outlive the workgroup

  // lane: token t0 + .. + l16 of each token fragment, 16 consecutive rows
  const uint32_t n = n0 + wn * (TN / WN) + part * 16;
  if (n >= a.rows) return;
  const uint32_t count = min(a.rows - n, 16u);
  float ws[16], wz[16], wb[16];
#pragma unroll
  for (uint32_t j = 0; j < 16; ++j) {
    ws[j] = j < count ? a.w_scale[n + j] : 0.0f;
    wz[j] = j < count && a.w_zp != nullptr ? a.w_zp[n + j] : 0.0f;
    wb[j] = j < count && a.bias != nullptr ? a.bias[n + j] : 0.0f;
  }
  each<FT>([&](auto i) __attribute__((always_inline)) {
    constexpr uint32_t I = decltype(i)::value;
    const uint32_t t = t0 + wt * (TT / WT) + I * 16 + l16;
    if (t >= a.tokens) return;
    const float scale = a.t_scale[t];
    const float sum = a.w_zp != nullptr ? (float)a.t_sums[t] : 0.0f;
    float v[16];
    auto finish = [&](TokenFactors f) __attribute__((always_inline)) {
      each<16>([&](auto j) __attribute__((always_inline)) {
        constexpr uint32_t J = decltype(j)::value;
        // wz is 0 without zero points: the same value
        const float acc_z = __builtin_fmaf(-wz[J], sum, (float)acc[I][J / 4][J % 4]);
        v[J] = __builtin_fmaf(acc_z * f.on_sum, ws[J] * f.on_row, wb[J]);
      });
    };
    if (ordinary(scale)) finish({1.0f, scale});  // two paths: one product less for each output
    else finish(token_factors(scale));
    const uint64_t at = (uint64_t)t * a.out_ld + n;
    if (a.out_dtype == SH_DTYPE_BF16) store_run(static_cast<__bf16*>(a.out) + at, v, count);
    else if (a.out_dtype == SH_DTYPE_F16) store_run(static_cast<_Float16*>(a.out) + at, v, count);
    else store_run(static_cast<float*>(a.out) + at, v, count);
  });
}

}  // namespace

// ── the product for few tokens ────────────────────────────────────────────

namespace {

// Joins the W wavefronts' sums of rows n .. n + 3 for token t (64 entries apart) and stores the outputs.
template <uint32_t W>
__device__ __forceinline__ void store_joined(const sh::MatmulI8Args& a, const i32x4_t* sums, uint32_t t, uint32_t n,
                                             float scale, int32_t t_sum) {
  if (n >= a.rows) return;
  i32x4_t v = sums[0];
#pragma unroll
  for (uint32_t w = 1; w < W; ++w) v += sums[w * 64];
  const uint32_t count = min(a.rows - n, 4u);
  const TokenFactors f = token_factors(scale);
  float y[4];
#pragma unroll
  for (uint32_t r = 0; r < 4; ++r) {
    const bool in = r < count;
    const float ws = in ? a.w_scale[n + r] : 0.0f;
    const float wz = in && a.w_zp != nullptr ? a.w_zp[n + r] : 0.0f;
    const float wb = in && a.bias != nullptr ? a.bias[n + r] : 0.0f;
    y[r] = __builtin_fmaf(__builtin_fmaf(-wz, (float)t_sum, (float)v[r]) * f.on_sum, ws * f.on_row, wb);
  }
  const uint64_t at = (uint64_t)t * a.out_ld + n;
  if (a.out_dtype == SH_DTYPE_BF16) store_run(static_cast<__bf16*>(a.out) + at, y, count);
  else if (a.out_dtype == SH_DTYPE_F16) store_run(static_cast<_Float16*>(a.out) + at, y, count);
  else store_run(static_cast<float*>(a.out) + at, y, count);
}

// 16 FT tokens x 16 FN rows by W wavefronts, each with every W-th 128 columns. A wavefront keeps a ring of D
// stages of its own in LDS (tokens, then rows), so nothing waits for another wavefront until the sums are
// joined at the end. Bound by the weight's bytes: 8 x 18432 x 3072 12 us (4.7 TB/s), 1 x 16384 x 4096 15 us (4.5
// TB/s); a launch of less than 16 MB takes 3 to 7 us whatever it reads. The loads go through LDS because a
// fragment's lanes take 16 rows at a time: read straight to registers, a row's lines come 16 bytes a request
// (1 x 4096 x 4096 82 us).
template <uint32_t FT, uint32_t FN, uint32_t W, uint32_t D>
__device__ __forceinline__ void matmul_skinny(const sh::MatmulI8Args& a, uint8_t* lds) {
  constexpr uint32_t kStage = (FT + FN) * 16 * kStep;
  constexpr uint32_t kLoads = 2 * (FT + FN);  // of 8 rows each
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t tiles_n = (a.rows + 16 * FN - 1) / (16 * FN);
  const uint32_t t0 = blockIdx.x / tiles_n * (16 * FT), n0 = blockIdx.x % tiles_n * (16 * FN);
  const uint32_t end = token_bytes(a.cols);
  const i32x4_t tr = rows_resource(a.tq, a.t_ld, end, t0, a.tokens, 16 * FT);
  const i32x4_t wr = rows_resource(a.wq, a.w_ld, a.w_ld, n0, a.rows, 16 * FN);
  // row + 8 has the swizzle of row with bit 2 changed: two offsets cover every load
  const uint32_t row = lane / 8, slot = lane % 8;
  const uint32_t s0 = (slot ^ swizzle(row)) * 16, s1 = (slot ^ swizzle(row + 8)) * 16;
  const uint32_t t_ld = (uint32_t)a.t_ld, w_ld = (uint32_t)a.w_ld;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + wave * D * kStage;
  auto load = [&](uint32_t stage, uint32_t k) {
#pragma unroll
    for (uint32_t j = 0; j < 2 * FN; ++j)
      load_to_lds(wr, lds0 + stage * kStage + (2 * FT + j) * 1024, (row + j * 8) * w_ld + (j % 2 ? s1 : s0) + k);
#pragma unroll
    for (uint32_t j = 0; j < 2 * FT; ++j)
      load_to_lds(tr, lds0 + stage * kStage + j * 1024, (row + j * 8) * t_ld + (j % 2 ? s1 : s0) + k);
  };
  const uint32_t l16 = lane & 15, part = lane / 16;
  const uint8_t* mine = lds + wave * D * kStage + l16 * kStep;
  i32x4_t acc[FT][FN] = {};
#pragma unroll
  for (uint32_t i = 0; i < D; ++i) {
    const uint32_t k = (i * W + wave) * kStep;
    load(i, k < end ? k : kPastEnd);
  }
  uint32_t s = 0;
  for (uint32_t k = wave * kStep; k < end; k += W * kStep) {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 1) * kLoads) : "memory");
    i32x4_t tf[2][FT], nf[2][FN];
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint8_t* at = mine + s * kStage + ((h * 4 + part) ^ swizzle(l16)) * 16;
#pragma unroll
      for (uint32_t i = 0; i < FT; ++i) tf[h][i] = *reinterpret_cast<const i32x4_t*>(at + i * 16 * kStep);
#pragma unroll
      for (uint32_t j = 0; j < FN; ++j) nf[h][j] = *reinterpret_cast<const i32x4_t*>(at + (FT + j) * 16 * kStep);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the place is loaded again
    const uint32_t next = k + D * W * kStep;
    load(s, next < end ? next : kPastEnd);
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
      for (uint32_t i = 0; i < FT; ++i)
#pragma unroll
        for (uint32_t j = 0; j < FN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(nf[h][j], tf[h][i], acc[i][j], 0, 0, 0);
    s = s == D - 1 ? 0 : s + 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing may land on the sums below
  __syncthreads();
  i32x4_t* sums = reinterpret_cast<i32x4_t*>(lds);
#pragma unroll
  for (uint32_t i = 0; i < FT; ++i)
#pragma unroll
    for (uint32_t j = 0; j < FN; ++j) sums[((i * FN + j) * W + wave) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (uint32_t f = wave; f < FT * FN; f += W) {
    const uint32_t t = t0 + f / FN * 16 + l16, n = n0 + f % FN * 16 + part * 4;
    if (t >= a.tokens) continue;
    store_joined<W>(a, sums + f * W * 64 + lane, t, n, a.t_scale[t], a.w_zp != nullptr ? a.t_sums[t] : 0);
  }
}

}  // namespace

// ── a few tokens, quantised where they are multiplied ─────────────────────

namespace {

// As matmul_skinny for up to 16 tokens, which every workgroup quantises for itself into LDS: one launch. The weight's
// first loads start when the tokens have arrived and their maxima are known, and are on their way while the tokens are
// rounded: the memory's latency comes twice, one after the other, before the first product. A wavefront's piece of a token is 512 values; all of them, PIECES / W a
// wavefront, stay in registers between maximum and rounding. In `a`, tq is the tokens as they are, t_ld their
// distance in elements; t_scale and t_sums are not used.
template <typename T, uint32_t FN, uint32_t W, uint32_t D, uint32_t PIECES>
__device__ __forceinline__ void linear_few(const sh::MatmulI8Args& a, uint8_t* ring, uint8_t* tq, uint32_t* amax,
                                           int32_t* sum) {
  constexpr uint32_t kStage = FN * 16 * kStep;
  constexpr uint32_t kLoads = 2 * FN;
  constexpr uint32_t kMine = PIECES / W;
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t n0 = blockIdx.x * (16 * FN);
  const uint32_t end = token_bytes(a.cols);
  const uint32_t q_ld = end + 16;  // 16 bytes more: the rows of a fragment in different LDS banks
  const uint32_t pieces = (a.cols + 511) / 512;

  Chunk<T> held[kMine];
  uint32_t token_of[kMine], at_of[kMine];
#pragma unroll
  for (uint32_t j = 0; j < kMine; ++j) {
    const uint32_t item = j * W + wave;
    // item / pieces: exact for item < 64, pieces <= 64 (the quotient's error is under 64 / 2^16)
    const uint32_t t = item * ((65536 + pieces - 1) / pieces) >> 16, at = ((item - t * pieces) * 64 + lane) * 8;
    token_of[j] = t;
    at_of[j] = at;
    if (t < a.tokens)
      held[j].load(static_cast<const T*>(a.tq) + (uint64_t)t * a.t_ld + at, at < a.cols ? a.cols - at : 0,
                   goes_on(t, a.tokens, a.t_ld, a.cols));
  }
  if (threadIdx.x < 16) {
    amax[threadIdx.x] = 0;
    sum[threadIdx.x] = 0;
  }
  __syncthreads();
#pragma unroll
  for (uint32_t j = 0; j < kMine; ++j) {
    const uint32_t t = token_of[j];
    if (t >= a.tokens) continue;
    const uint32_t m = wave_max(amax_bits<T>(held[j].amax(0)));
    if (lane == 0) atomicMax(amax + t, m);
  }

  const i32x4_t wr = rows_resource(a.wq, a.w_ld, a.w_ld, n0, a.rows, 16 * FN);
  const uint32_t row = lane / 8, slot = lane % 8;
  const uint32_t s0 = (slot ^ swizzle(row)) * 16, s1 = (slot ^ swizzle(row + 8)) * 16;
  const uint32_t w_ld = (uint32_t)a.w_ld;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)ring + wave * D * kStage;
  auto load = [&](uint32_t stage, uint32_t k) {
#pragma unroll
    for (uint32_t j = 0; j < 2 * FN; ++j)
      load_to_lds(wr, lds0 + stage * kStage + j * 1024, (row + j * 8) * w_ld + (j % 2 ? s1 : s0) + k);
  };
#pragma unroll
  for (uint32_t i = 0; i < D; ++i) {
    const uint32_t k = (i * W + wave) * kStep;
    load(i, k < end ? k : kPastEnd);
  }

  __syncthreads();
#pragma unroll
  for (uint32_t j = 0; j < kMine; ++j) {
    const uint32_t t = token_of[j], at = at_of[j];
    if (t >= a.tokens) continue;
    float inv, scale;
    token_scale(amax[t], &inv, &scale);
    const uint2 b = held[j].quantize(inv, inv == 0.0f ? 0u : ~0u);
    if (at < end) *reinterpret_cast<uint2*>(tq + t * q_ld + at) = b;
    if (a.w_zp != nullptr) {
      const int32_t v = wave_sum(__builtin_amdgcn_sdot4((int)b.y, 0x01010101, __builtin_amdgcn_sdot4((int)b.x, 0x01010101, 0, false), false));
      if (lane == 0) atomicAdd(sum + t, v);
    }
  }
  __syncthreads();

  const uint32_t l16 = lane & 15, part = lane / 16;
  const uint8_t* mine = ring + wave * D * kStage + l16 * kStep;
  const uint8_t* token = tq + min(l16, a.tokens - 1) * q_ld + part * 16;
  i32x4_t acc[FN] = {};
  uint32_t s = 0;
  for (uint32_t k = wave * kStep; k < end; k += W * kStep) {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 1) * kLoads) : "memory");
    i32x4_t tf[2], nf[2][FN];
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint8_t* at = mine + s * kStage + ((h * 4 + part) ^ swizzle(l16)) * 16;
      tf[h] = *reinterpret_cast<const i32x4_t*>(token + k + h * 64);
#pragma unroll
      for (uint32_t j = 0; j < FN; ++j) nf[h][j] = *reinterpret_cast<const i32x4_t*>(at + j * 16 * kStep);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the place is loaded again
    const uint32_t next = k + D * W * kStep;
    load(s, next < end ? next : kPastEnd);
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
      for (uint32_t j = 0; j < FN; ++j)
        acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(nf[h][j], tf[h], acc[j], 0, 0, 0);
    s = s == D - 1 ? 0 : s + 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing may land on the sums below
  __syncthreads();
  i32x4_t* sums = reinterpret_cast<i32x4_t*>(ring);
#pragma unroll
  for (uint32_t j = 0; j < FN; ++j) sums[(j * W + wave) * 64 + lane] = acc[j];
  __syncthreads();
  if (wave >= FN || l16 >= a.tokens) return;
  float inv, scale;
  token_scale(amax[l16], &inv, &scale);
  store_joined<W>(a, sums + wave * W * 64 + lane, l16, n0 + wave * 16 + part * 4, scale, sum[l16]);
}

}  // namespace

#define SH_LINEAR_FEW(name, T, tile, FN, W, D, PIECES)                                                        \
  extern "C" __global__ __launch_bounds__(W * 64) void sh_linear_i8_##name##_##tile##_kernel(sh::MatmulI8Args a) { \
    __shared__ alignas(16) uint8_t ring[W * D * FN * 16 * kStep];                                             \
    __shared__ alignas(16) uint8_t tq[PIECES * 512 + 16 * 16];                                                \
    __shared__ uint32_t amax[16];                                                                             \
    __shared__ int32_t sum[16];                                                                               \
    linear_few<T, FN, W, D, PIECES>(a, ring, tq, amax, sum);                                                  \
  }
SH_LINEAR_FEW(bf16, __bf16, 16x16, 1, 8, 3, sh::kFewPiecesNarrow)
SH_LINEAR_FEW(bf16, __bf16, 16x32, 2, 4, 2, sh::kFewPiecesWide)
SH_LINEAR_FEW(f16, _Float16, 16x16, 1, 8, 3, sh::kFewPiecesNarrow)
SH_LINEAR_FEW(f16, _Float16, 16x32, 2, 4, 2, sh::kFewPiecesWide)
SH_LINEAR_FEW(f32, float, 16x16, 1, 8, 3, sh::kFewPiecesNarrow)
SH_LINEAR_FEW(f32, float, 16x32, 2, 4, 2, sh::kFewPiecesWide)

// The tiles of sh_int8_args.h.
#define SH_MATMUL_FEW(name, FT, FN, W, D)                                                                     \
  extern "C" __global__ __launch_bounds__(W * 64) void sh_matmul_i8_##name##_kernel(sh::MatmulI8Args a) {      \
    __shared__ alignas(16) uint8_t lds[W * D * (FT + FN) * 16 * kStep];                                       \
    matmul_skinny<FT, FN, W, D>(a, lds);                                                                      \
  }
#define SH_MATMUL_TILE(name, TT, TN, WT, WN, D, GROUP)                                                        \
  extern "C" __global__ __launch_bounds__(WT * WN * 64) void sh_matmul_i8_##name##_kernel(sh::MatmulI8Args a) { \
    __shared__ alignas(16) uint8_t lds[D * (TT + TN) * kStep];                                                \
    matmul_tile<TT, TN, WT, WN, D, GROUP>(a, lds);                                                            \
  }
SH_MATMUL_FEW(16x16, 1, 1, 8, 3)
SH_MATMUL_FEW(16x32, 1, 2, 4, 3)
SH_MATMUL_FEW(32x32, 2, 2, 4, 2)
SH_MATMUL_TILE(64x64, 64, 64, 4, 1, 4, 8)
SH_MATMUL_TILE(128x128, 128, 128, 4, 2, 3, 4)
SH_MATMUL_TILE(128x256, 128, 256, 4, 4, 3, 4)
SH_MATMUL_TILE(256x256, 256, 256, 2, 4, 2, 4)
