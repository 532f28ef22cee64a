// Layer norm, forward and backward, for gfx950 (device code only; the checks and the launches are in
// sh_layer_norm.cpp).
//
// With n = (x - mean) r, r = (var + eps)^(-1/2), and a gain w (1 + w when modulated): y = n w + b. For a gradient dy,
// with g = dy w: dx = r (g - mean(g) - n mean(g n)), dw = sum of dy n and db = sum of dy over the tokens that share w, b.
//
// Bound by HBM: each value is read once and written once (backward: x and dy read, dx written). A team holds a row in
// registers, so mean and variance take two passes over registers and one over memory: differences from a first mean, whose
// own mean corrects both. A first mean alone is off by the roundings of the sum and of the division, which r, up to eps^(-1/2),
// multiplies: rows of 1155 times 1000 had norms of 0.03 in the place of 0. The next row is on its way while one is worked on.
// The forward leaves mean and r of each token for the backward pass. The gradients of w and b are summed in registers over a
// workgroup's tokens and joined by a second kernel, always in the same order; every workgroup's sums are written and read once
// more, so there are few workgroups.
//
// Measured: forward 2 x 8192 tokens x 4096 bf16 46 us (5.9 TB/s), keeping the input as well 66-70 us (4.9), fp32 100 us (5.4),
// 4608 x 4096 15 us (5.0; 0.5 us of it the correction of the mean), 65536 x 256 14.5 us (4.6), 8192 x 16384 102 us (5.3);
// backward with the joining kernel, 2 x 8192 x 4096 86-89 us (4.6 TB/s), from the kept input 72-74 (4.6), fp32 157-164 (5.0) and
// 124-127; 8192 x 16384, whose rows load nothing ahead, 169-175 (4.7) and 142-153, 8 of them the joining; a large copy 5.2 TB/s
// by torch, 6.6 by this library's kernel. Two chunks a work-item against one: 46 and 54 us; 1024 work-items a compute unit against
// 2048 and 512: 46, 49 and 53 us. Not kept: one or two rows for each of many short workgroups, which stream copies faster (73 us:
// their start, weights and barriers come with every row), two teams with joined sums in a workgroup of the backward pass (87
// against 84 us; 3 x 1013 x 1155 20 against 21), shuffles through LDS for a wavefront's sums.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "sh_act8_device.h"
#include "sh_layer_norm_args.h"

namespace {

template <int CTRL>
__device__ __forceinline__ float add_moved(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}
// The sum over groups of `lanes` (a power of two from 4 on) neighbouring work-items, in all of them: halves of 2, 4, 8 and
// 16 by data-parallel moves (each adds a half that already agrees), 32 and 64 by exchanges: two copies of v exchange rows
// of 16 (then halves), so that each has one half of the sum everywhere. These are assembly: the compiler takes both
// results of its builtin to be one where both arguments are.
__device__ __forceinline__ float group_sum(float v, uint32_t lanes) {
  v = add_moved<0xB1>(v);                    // quad_perm 1,0,3,2
  v = add_moved<0x4E>(v);                    // quad_perm 2,3,0,1
  if (lanes >= 8) v = add_moved<0x141>(v);   // row_half_mirror
  if (lanes >= 16) v = add_moved<0x140>(v);  // row_mirror
  if (lanes >= 32) {
    float other = v;
    asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(v), "+v"(other));
    v += other;
  }
  if (lanes >= 64) {
    float other = v;
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(v), "+v"(other));
    v += other;
  }
  return v;
}

constexpr uint32_t kMostWaves = sh::kNormMostWaves;

// Sums over a team, in all of it: the workgroup if TEAM, else groups of `lanes` work-items. Two sets of slots in turn: a
// set is written again only after the barrier of the other, which everyone reaches after reading it. Slots that no
// wavefront has hold zeros.
template <bool TEAM, uint32_t N>
struct TeamSum {
  float (*slots)[N][kMostWaves];  // [2][N][kMostWaves] of LDS
  uint32_t lanes, turn = 0;

  __device__ __forceinline__ TeamSum(float (*slots)[N][kMostWaves], uint32_t lanes) : slots(slots), lanes(lanes) {
    if constexpr (TEAM) {  // by the wavefront that is before the first barrier with the others
      if (threadIdx.x < 2 * N * kMostWaves && threadIdx.x % kMostWaves >= blockDim.x / 64) (&slots[0][0][0])[threadIdx.x] = 0.0f;
    }
  }
  template <uint32_t M>
  __device__ __forceinline__ void operator()(float (&v)[M]) {
    static_assert(M <= N, "a slot for each sum");
#pragma unroll
    for (uint32_t i = 0; i < M; ++i) v[i] = group_sum(v[i], TEAM ? 64 : lanes);
    if constexpr (TEAM) {
      if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (uint32_t i = 0; i < M; ++i) slots[turn][i][threadIdx.x / 64] = v[i];
      }
      __syncthreads();
#pragma unroll
      for (uint32_t i = 0; i < M; ++i) {
        v[i] = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kMostWaves; ++w) v[i] += slots[turn][i][w];
      }
      turn ^= 1;
    }
  }
};

// 8 values of a weight or bias at p; 0 behind `count` and without one.
__device__ __forceinline__ void load_params(const void* p, uint32_t dtype, uint64_t at, uint32_t count, float (&v)[8]) {
  auto values = [&](auto zero) {
    using T = decltype(zero);
    const auto raw = Values8<T>::load(static_cast<const T*>(p) + at, p != nullptr ? count : 0);
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) v[i] = (float)raw[i];
  };
  if (dtype == SH_DTYPE_BF16) values(__bf16{});
  else if (dtype == SH_DTYPE_F16) values(_Float16{});
  else values(float{});
}

// A weight as a gain: 1 without one.
__device__ __forceinline__ void as_gain(const sh_layer_norm_args& a, float (&w)[8]) {
  if (!a.modulate && a.weight != nullptr) return;
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i) w[i] += 1.0f;
}

__device__ __forceinline__ void store_params(void* p, uint32_t dtype, uint64_t at, uint32_t count, const float (&v)[8]) {
  if (dtype == SH_DTYPE_BF16) Values8<__bf16>::store(static_cast<__bf16*>(p) + at, v, count);
  else if (dtype == SH_DTYPE_F16) Values8<_Float16>::store(static_cast<_Float16*>(p) + at, v, count);
  else Values8<float>::store(static_cast<float*>(p) + at, v, count);
}

// A work-item's share of the rows: chunks of 8 values, and the tokens of a group that its team takes.
template <bool TEAM, uint32_t C>
struct Mine {
  uint32_t item, items;  // in the team
  uint32_t group, team, teams;  // of the group
  uint32_t cols;

  __device__ __forceinline__ Mine(const sh::LayerNormKernelArgs& ka) : cols(ka.a.cols) {
    items = ka.lanes;
    item = TEAM ? threadIdx.x : threadIdx.x & (items - 1);
    group = blockIdx.x / ka.per_group;
    const uint32_t block = blockIdx.x - group * ka.per_group, of_block = TEAM ? 1 : sh::kNormThreads / items;
    team = block * of_block + (TEAM ? 0 : threadIdx.x / items);
    teams = ka.per_group * of_block;
  }
  __device__ __forceinline__ uint32_t chunk(uint32_t j) const { return j * items + item; }
  __device__ __forceinline__ uint32_t col(uint32_t j) const { return chunk(j) * 8; }
  __device__ __forceinline__ uint32_t count(uint32_t j) const { return col(j) < cols ? min(cols - col(j), 8u) : 0; }
};

struct Token {
  uint64_t b, s, row;

  __device__ __forceinline__ Token(const sh_layer_norm_args& a, uint32_t group, uint32_t t) {
    if (a.per_batch || a.batch == 1) b = group, s = t;
    else b = t / a.seq, s = t - (uint32_t)b * a.seq;
    row = b * a.seq + s;
  }
  __device__ __forceinline__ uint64_t at(const sh_rows& r) const { return b * r.batch_stride + s * r.seq_stride; }
};

template <typename T, bool TEAM, uint32_t C>
__device__ __forceinline__ void forward(const sh::LayerNormKernelArgs& ka) {
  const sh_layer_norm_args& a = ka.a;
  const Mine<TEAM, C> m(ka);
  __shared__ alignas(16) float slots[2][2][kMostWaves];
  TeamSum<TEAM, 2> team_sum(slots, ka.lanes);
  const float rcols = 1.0f / (float)a.cols;
  const uint32_t row_chunks = (a.cols + SH_ACT8_GROUP - 1) / SH_ACT8_GROUP * (SH_ACT8_GROUP / 8);
  typename Values8<T>::Vec next[C];
  auto load = [&](uint32_t t) __attribute__((always_inline)) {
    const T* x = static_cast<const T*>(a.x.data) + Token(a, m.group, t).at(a.x);
#pragma unroll
    for (uint32_t j = 0; j < C; ++j) next[j] = Values8<T>::load(x + m.col(j), m.count(j));
  };
  if (m.team < ka.tokens) load(m.team);
  float w[C][8], b[C][8];
#pragma unroll
  for (uint32_t j = 0; j < C; ++j) {
    load_params(a.weight, a.weight_dtype, m.group * a.weight_batch_stride + m.col(j), m.count(j), w[j]);
    load_params(a.bias, a.weight_dtype, m.group * a.bias_batch_stride + m.col(j), m.count(j), b[j]);
    as_gain(a, w[j]);
  }
  for (uint32_t t = m.team; t < ka.tokens; t += m.teams) {
    const Token token(a, m.group, t);
    float v[C][8], sum[1] = {0.0f};
#pragma unroll
    for (uint32_t j = 0; j < C; ++j)
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) v[j][i] = (float)next[j][i];
    if (t + m.teams < ka.tokens) load(t + m.teams);  // on its way while this row is worked on
    if (a.q != nullptr) {
#pragma unroll
      for (uint32_t j = 0; j < C; ++j) {
        if (m.chunk(j) >= row_chunks) continue;  // whole groups of four work-items
        const uint32_t e = group_exponent(v[j]);
        const uint64_t at = token.row * row_chunks + m.chunk(j);
        static_cast<uint2*>(a.q)[at] = quantize8<T>(v[j], e);
        if (m.item % 4 == 0) static_cast<uint8_t*>(a.exponent)[at / 4] = (uint8_t)e;
      }
    }
#pragma unroll
    for (uint32_t j = 0; j < C; ++j)
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) sum[0] += v[j][i];
    team_sum(sum);
    // Differences from the product sum * rcols as it is, which the mean below starts from too: neither rounds it.
    float sums[2] = {0.0f, 0.0f};
#pragma unroll
    for (uint32_t j = 0; j < C; ++j) {
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) {
        v[j][i] = i < m.count(j) ? __builtin_fmaf(sum[0], -rcols, v[j][i]) : 0.0f;
        sums[0] += v[j][i];
        sums[1] = __builtin_fmaf(v[j][i], v[j][i], sums[1]);
      }
    }
    team_sum(sums);
    const float off = sums[0] * rcols, mean = __builtin_fmaf(sum[0], rcols, off);
    float var = __builtin_fmaf(off, -off, sums[1] * rcols);
    if (var < 0.0f) var = 0.0f;  // and a NaN stays one
    const float r = 1.0f / __builtin_sqrtf(var + a.eps), shift = -off * r;
    T* y = static_cast<T*>(a.y.data) + token.at(a.y);
#pragma unroll
    for (uint32_t j = 0; j < C; ++j) {
      float out[8];
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) out[i] = __builtin_fmaf(__builtin_fmaf(v[j][i], r, shift), w[j][i], b[j][i]);
      Values8<T>::store(y + m.col(j), out, m.count(j));
    }
    if (a.stats != nullptr && m.item == 0) {
      a.stats[2 * token.row] = mean;
      a.stats[2 * token.row + 1] = r;
    }
  }
}

// A row of the input as it lies in memory, or as it was kept.
template <typename T, bool TEAM, uint32_t C, bool KEPT>
struct InputRow {
  typename Values8<T>::Vec raw[C];

  __device__ __forceinline__ void load(const sh_layer_norm_args& a, const Mine<TEAM, C>& m, const Token& token) {
    const T* x = static_cast<const T*>(a.x.data) + token.at(a.x);
#pragma unroll
    for (uint32_t j = 0; j < C; ++j) raw[j] = Values8<T>::load(x + m.col(j), m.count(j));
  }
  __device__ __forceinline__ void values(uint32_t j, float (&v)[8]) const {
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) v[i] = (float)raw[j][i];
  }
};
template <typename T, bool TEAM, uint32_t C>
struct InputRow<T, TEAM, C, true> {
  uint2 q[C];
  uint32_t e[C];

  __device__ __forceinline__ void load(const sh_layer_norm_args& a, const Mine<TEAM, C>& m, const Token& token) {
    const uint32_t row_chunks = (a.cols + SH_ACT8_GROUP - 1) / SH_ACT8_GROUP * (SH_ACT8_GROUP / 8);
#pragma unroll
    for (uint32_t j = 0; j < C; ++j) {
      q[j] = make_uint2(0, 0);
      e[j] = 1;
      if (m.chunk(j) >= row_chunks) continue;
      const uint64_t at = token.row * row_chunks + m.chunk(j);
      q[j] = static_cast<const uint2*>(a.q)[at];
      e[j] = static_cast<const uint8_t*>(a.exponent)[at / 4];
    }
  }
  __device__ __forceinline__ void values(uint32_t j, float (&v)[8]) const { dequantize8(q[j], group_scale(e[j]), v); }
};

template <typename T, bool TEAM, uint32_t C, bool KEPT>
__device__ __forceinline__ void backward(const sh::LayerNormKernelArgs& ka) {
  const sh_layer_norm_args& a = ka.a;
  const Mine<TEAM, C> m(ka);
  __shared__ alignas(16) float slots[2][2][kMostWaves];
  TeamSum<TEAM, 2> team_sum(slots, ka.lanes);
  const float rcols = 1.0f / (float)a.cols;
  InputRow<T, TEAM, C, KEPT> next_x;
  typename Values8<T>::Vec next_dy[C];
  float next_mean = 0.0f, next_r = 0.0f;
  auto load = [&](uint32_t t) __attribute__((always_inline)) {
    const Token token(a, m.group, t);
    next_x.load(a, m, token);
    const T* dy = static_cast<const T*>(a.dy.data) + token.at(a.dy);
#pragma unroll
    for (uint32_t j = 0; j < C; ++j) next_dy[j] = Values8<T>::load(dy + m.col(j), m.count(j));  // zeros past the row add nothing below
    next_mean = a.stats[2 * token.row];
    next_r = a.stats[2 * token.row + 1];
  };
  constexpr bool kAhead = C < 4;  // longer rows' registers do not hold another row
  if (kAhead && m.team < ka.tokens) load(m.team);
  float w[C][8], dw[C][8] = {}, db[C][8] = {};
#pragma unroll
  for (uint32_t j = 0; j < C; ++j) {
    load_params(a.weight, a.weight_dtype, m.group * a.weight_batch_stride + m.col(j), m.count(j), w[j]);
    as_gain(a, w[j]);
  }
  for (uint32_t t = m.team; t < ka.tokens; t += m.teams) {
    if (!kAhead) load(t);
    const float mean = next_mean, r = next_r;
    float n[C][8], g[C][8], sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (uint32_t j = 0; j < C; ++j) {
      next_x.values(j, n[j]);
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) g[j][i] = (float)next_dy[j][i];
    }
    if (kAhead && t + m.teams < ka.tokens) load(t + m.teams);  // on its way while this row is worked on
#pragma unroll
    for (uint32_t j = 0; j < C; ++j) {
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) {
        n[j][i] = (n[j][i] - mean) * r;
        dw[j][i] = __builtin_fmaf(g[j][i], n[j][i], dw[j][i]);
        db[j][i] += g[j][i];
        g[j][i] *= w[j][i];
        sum[0] += g[j][i];
        sum[1] = __builtin_fmaf(g[j][i], n[j][i], sum[1]);
      }
    }
    if (a.dx.data == nullptr) continue;
    team_sum(sum);
    const float mean_g = sum[0] * rcols, mean_gn = sum[1] * rcols;
    T* dx = static_cast<T*>(a.dx.data) + Token(a, m.group, t).at(a.dx);
#pragma unroll
    for (uint32_t j = 0; j < C; ++j) {
      float out[8];
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) out[i] = r * (g[j][i] - mean_g - n[j][i] * mean_gn);
      Values8<T>::store(dx + m.col(j), out, m.count(j));
    }
  }
  if (a.dweight == nullptr && a.dbias == nullptr) return;
  if constexpr (!TEAM) {  // the teams' sums, in their order
    constexpr uint32_t kThreads = sh::kNormThreads;
    __shared__ float part[2][C][8][kThreads];
#pragma unroll
    for (uint32_t j = 0; j < C; ++j)
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) part[0][j][i][threadIdx.x] = dw[j][i], part[1][j][i][threadIdx.x] = db[j][i];
    __syncthreads();
    if (threadIdx.x >= m.items) return;
    for (uint32_t k = threadIdx.x + m.items; k < kThreads; k += m.items) {
#pragma unroll
      for (uint32_t j = 0; j < C; ++j)
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) dw[j][i] += part[0][j][i][k], db[j][i] += part[1][j][i][k];
    }
  }
#pragma unroll
  for (uint32_t j = 0; j < C; ++j) {
    if (ka.partials == nullptr) {  // the workgroup has all of the group's tokens
      const uint64_t at = (uint64_t)m.group * a.cols + m.col(j);
      if (a.dweight != nullptr) store_params(a.dweight, a.weight_dtype, at, m.count(j), dw[j]);
      if (a.dbias != nullptr) store_params(a.dbias, a.weight_dtype, at, m.count(j), db[j]);
    } else {
      float* p = ka.partials + (uint64_t)blockIdx.x * 2 * a.cols + m.col(j);
      Values8<float>::store(p, dw[j], m.count(j));
      Values8<float>::store(p + a.cols, db[j], m.count(j));
    }
  }
}

}  // namespace

// The shapes of sh_layer_norm_args.h.
#define SH_NORM(name, T, shape, TEAM, C)                                                                                      \
  extern "C" __global__ __launch_bounds__(sh::norm_most_threads(TEAM)) void sh_layer_norm_##name##_##shape##_kernel(          \
      sh::LayerNormKernelArgs ka) {                                                                                           \
    forward<T, TEAM, C>(ka);                                                                                                  \
  }                                                                                                                           \
  extern "C" __global__ __launch_bounds__(sh::norm_most_threads(TEAM)) void sh_layer_norm_backward_##name##_##shape##_kernel( \
      sh::LayerNormKernelArgs ka) {                                                                                           \
    backward<T, TEAM, C, false>(ka);                                                                                          \
  }                                                                                                                           \
  extern "C" __global__ __launch_bounds__(sh::norm_most_threads(TEAM)) void sh_layer_norm_backward_kept_##name##_##shape##_kernel( \
      sh::LayerNormKernelArgs ka) {                                                                                           \
    backward<T, TEAM, C, true>(ka);                                                                                           \
  }
#define SH_NORM_SHAPES(name, T)          \
  SH_NORM(name, T, wave1, false, 1)      \
  SH_NORM(name, T, wave2, false, 2)      \
  SH_NORM(name, T, team2, true, 2)       \
  SH_NORM(name, T, team4, true, 4)
SH_NORM_SHAPES(bf16, __bf16)
SH_NORM_SHAPES(f16, _Float16)
SH_NORM_SHAPES(f32, float)

// The gradients of a group's weight and bias from its workgroups' sums: 32 values a workgroup, each added up by 32
// work-items, every 32nd sum each, that are joined in order.
extern "C" __global__ __launch_bounds__(sh::kNormJoinThreads) void sh_layer_norm_join_kernel(sh::LayerNormKernelArgs ka) {
  constexpr uint32_t kCols = sh::kNormJoinCols, kRows = sh::kNormJoinThreads / kCols;
  const sh_layer_norm_args& a = ka.a;
  const uint32_t blocks = (a.cols + kCols - 1) / kCols;
  const uint32_t which = blockIdx.x / blocks % 2, group = blockIdx.x / blocks / 2;
  const uint32_t col = blockIdx.x % blocks * kCols + threadIdx.x % kCols;
  void* out = which == 0 ? a.dweight : a.dbias;
  if (out == nullptr) return;
  __shared__ float part[kRows][kCols];
  float v = 0.0f;
  if (col < a.cols) {
    const float* p = ka.partials + ((uint64_t)group * ka.per_group * 2 + which) * a.cols + col;
#pragma unroll 8
    for (uint32_t k = threadIdx.x / kCols; k < ka.per_group; k += kRows) v += p[(uint64_t)k * 2 * a.cols];
  }
  part[threadIdx.x / kCols][threadIdx.x % kCols] = v;
  __syncthreads();
  if (threadIdx.x >= kCols || col >= a.cols) return;
  v = 0.0f;
  for (uint32_t k = 0; k < kRows; ++k) v += part[k][threadIdx.x];
  const uint64_t at = (uint64_t)group * a.cols + col;
  if (a.weight_dtype == SH_DTYPE_BF16) static_cast<__bf16*>(out)[at] = (__bf16)v;
  else if (a.weight_dtype == SH_DTYPE_F16) static_cast<_Float16*>(out)[at] = (_Float16)v;
  else static_cast<float*>(out)[at] = v;
}
