// Query/key norms with the position rotation for gfx950 (device code only; the checks and the
// launches are in sh_qk_norm.cpp).
//
// A head's values are taken as dim / 2 pairs. Pairs p < rot / 2 are rotated: (p, p + rot / 2), or
// (2p, 2p + 1) when interleaved. The values past rot form pairs the same way with the angle 0, so
// every pair is handled alike.
//
// With n = x r w, r = (mean(x^2) + eps)^(-1/2), and R the rotation by the token's angles: y = R n. For a gradient
// dy, with g = R^-1 dy and x^ = x r: dw = sum over all heads and tokens of g x^, and dx = r (g w - x^ mean(g w x^)).
// Both means come from one pass over a head's values: mean(g w x^) = r mean(g w x).
//
// The work is bound by HBM: each value is read once and written once (backward: two reads, one write). A
// group of `lanes` work-items holds a head, kQkSlots pairs each, in registers: the statistics, the rotation and
// the gradient need no second read and no shared memory, and the backward pass takes the statistics again
// instead of reading them. A group keeps its token's cosines and sines while it takes the token's heads one
// after another, and the weights for its life. The weights' gradients are summed in registers, over a
// workgroup, and over the workgroups by a second small kernel, always in the same order.
//
// Measured: 4608 tokens x 48 heads of 128 bf16 20 us (5.7 TB/s; 24.5 us, 4.7 TB/s, where the caches do not help),
// 2 x 8192 x 64 heads forward 100 us (5.4 TB/s) and backward 140 to 166 us (4.9 to 5.8 TB/s); a large copy 5.1 TB/s
// by torch, 6.6 by this library's kernel. Heads of 64 4.4 TB/s: pieces of 128 bytes at the outputs' stride.
// Scalar loads of single values took 5 times as long (115 us). Not kept: the next head's values loaded
// ahead (113 against 108 us), consecutive tokens for one XCD (33 against 24.5 us at 4608 tokens), non-temporal
// loads (10% slower backward) and stores (what the backward gained the next forward lost).

#include <hip/hip_runtime.h>

#include <cstdint>

#include "sh_qk_norm_args.h"

namespace {

constexpr uint32_t kSlots = sh::kQkSlots;

// V values at any address of memory (gfx950 loads and stores whole vectors there), or at a multiple of ALIGN
// bytes of LDS.
template <typename T, uint32_t V, uint32_t ALIGN = 2>
struct Run {
  typedef T Vec __attribute__((ext_vector_type(V)));
  typedef Vec VecAny __attribute__((aligned(ALIGN)));

  static __device__ __forceinline__ Vec load(const T* p) {
    if constexpr (V == 1) return Vec{*p};
    else return *reinterpret_cast<const VecAny*>(p);
  }
  static __device__ __forceinline__ void store(T* p, const float (&in)[V]) {
    if constexpr (V == 1) {
      *p = (T)in[0];
    } else {
      Vec v;
#pragma unroll
      for (uint32_t i = 0; i < V; ++i) v[i] = (T)in[i];
      *reinterpret_cast<VecAny*>(p) = v;
    }
  }
};

// A weight of `dim` values in fp32 (ones without one).
__device__ __forceinline__ void share_weight(float* shared, const void* w, uint32_t dtype, uint32_t dim) {
  for (uint32_t i = threadIdx.x; i < dim; i += sh::kQkThreads) {
    float v = 1.0f;
    if (w != nullptr) {
      if (dtype == SH_DTYPE_BF16) v = (float)static_cast<const __bf16*>(w)[i];
      else if (dtype == SH_DTYPE_F16) v = (float)static_cast<const _Float16*>(w)[i];
      else v = static_cast<const float*>(w)[i];
    }
    shared[i] = v;
  }
}

// The sum over the `lanes` (a power of two) neighbouring work-items of a group, in all of them: halves of
// 2, 4, 8 and 16 by data-parallel primitives (each adds a half that already agrees), 32 and 64 by shuffles.
template <int CTRL>
__device__ __forceinline__ float add_moved(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ float group_sum(float v, uint32_t lanes) {
  if (lanes >= 2) v = add_moved<0xB1>(v);   // quad_perm 1,0,3,2
  if (lanes >= 4) v = add_moved<0x4E>(v);   // quad_perm 2,3,0,1
  if (lanes >= 8) v = add_moved<0x141>(v);  // row_half_mirror
  if (lanes >= 16) v = add_moved<0x140>(v);  // row_mirror
  if (lanes >= 32) v += __shfl_xor(v, 16);
  if (lanes >= 64) v += __shfl_xor(v, 32);
  return v;
}

// v^(-1/2). The instruction is good to an ulp and takes no subnormal numbers.
__device__ __forceinline__ float inv_sqrt(float v) {
  return v >= 0x1p-100f ? __builtin_amdgcn_rsqf(v) : 1.0f / __builtin_sqrtf(v);
}

// What a work-item knows of its pairs: chunk j is V pairs from p[j] on.
template <typename T, uint32_t V, bool INTERLEAVED>
struct Pairs {
  static constexpr uint32_t kChunks = kSlots / V;
  uint32_t lane, lanes, half, rot_half;

  __device__ __forceinline__ Pairs(const sh_qk_norm_rope_args& a, uint32_t lane, uint32_t lanes)
      : lane(lane), lanes(lanes), half(a.dim / 2), rot_half(a.rot / 2) {}
  __device__ __forceinline__ uint32_t first(uint32_t j) const { return (j * lanes + lane) * V; }
  __device__ __forceinline__ bool in(uint32_t j) const { return first(j) < half; }
  __device__ __forceinline__ bool rotated(uint32_t j) const { return first(j) < rot_half; }
  // places of the chunk's first pair: with rot / 2 and dim / 2 pairs, the second half of the rotated values
  // starts at rot / 2, the others at rot and at rot + (dim - rot) / 2
  __device__ __forceinline__ uint32_t i0(uint32_t j) const {
    return INTERLEAVED ? 2 * first(j) : first(j) + (rotated(j) ? 0 : rot_half);
  }
  __device__ __forceinline__ uint32_t i1(uint32_t j) const {
    return INTERLEAVED ? 2 * first(j) + 1 : first(j) + (rotated(j) ? rot_half : half);
  }

  // A head's values as they lie in memory: a load in flight until they are looked at.
  template <typename U>
  struct Raw {
    typename Run<U, V>::Vec a[kChunks], b[kChunks];

    __device__ __forceinline__ void values(float (&v0)[kSlots], float (&v1)[kSlots]) const {
#pragma unroll
      for (uint32_t j = 0; j < kChunks; ++j) {
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) {
          if constexpr (INTERLEAVED) {
            // pair i is values 2 i and 2 i + 1 of the 2 V that a and b hold
            v0[j * V + i] = 2 * i < V ? (float)a[j][2 * i % V] : (float)b[j][2 * i % V];
            v1[j * V + i] = 2 * i + 1 < V ? (float)a[j][(2 * i + 1) % V] : (float)b[j][(2 * i + 1) % V];
          } else {
            v0[j * V + i] = (float)a[j][i];
            v1[j * V + i] = (float)b[j][i];
          }
        }
      }
    }
  };

  template <uint32_t ALIGN = 2, typename U>
  __device__ __forceinline__ Raw<U> load(const U* base) const {
    Raw<U> r;
#pragma unroll
    for (uint32_t j = 0; j < kChunks; ++j) {
      r.a[j] = r.b[j] = (U)0.0f;
      if (in(j)) {
        r.a[j] = Run<U, V, ALIGN>::load(base + i0(j));
        r.b[j] = Run<U, V, ALIGN>::load(base + (INTERLEAVED ? i0(j) + V : i1(j)));
      }
    }
    return r;
  }

  template <uint32_t ALIGN = 2, typename U>
  __device__ __forceinline__ void store(U* base, const float (&v0)[kSlots], const float (&v1)[kSlots]) const {
#pragma unroll
    for (uint32_t j = 0; j < kChunks; ++j) {
      if (!in(j)) continue;
      float a[V], b[V];
#pragma unroll
      for (uint32_t i = 0; i < V; ++i) {
        if constexpr (INTERLEAVED) {
          // values 0 .. V - 1 and V .. 2 V - 1 of the 2 V that lie together
          a[i] = i % 2 ? v1[j * V + i / 2] : v0[j * V + i / 2];
          b[i] = (V + i) % 2 ? v1[j * V + (V + i) / 2] : v0[j * V + (V + i) / 2];
        } else {
          a[i] = v0[j * V + i];
          b[i] = v1[j * V + i];
        }
      }
      Run<U, V, ALIGN>::store(base + i0(j), a);
      Run<U, V, ALIGN>::store(base + (INTERLEAVED ? i0(j) + V : i1(j)), b);
    }
  }

  // A weight that share_weight() has put into LDS.
  __device__ __forceinline__ void load_weight(const float* shared, float (&v0)[kSlots], float (&v1)[kSlots]) const {
    load<(V >= 4 ? 16 : 4 * V)>(shared).values(v0, v1);
  }

  // Cosines and sines of the token at (b, s). Where its position has no row, NaN, also for the values past rot.
  __device__ __forceinline__ void load_angles(const sh_qk_norm_rope_args& a, uint64_t b, uint64_t s, float (&c)[kSlots],
                                              float (&n)[kSlots]) const {
    int64_t row = 0;
    bool known = true;
    if (a.rot > 0) {
      if (a.positions == nullptr) row = a.start + (int64_t)s;
      else if (a.position_bytes == 8) row = static_cast<const int64_t*>(a.positions)[b * a.position_batch_stride + s];
      else row = static_cast<const int32_t*>(a.positions)[b * a.position_batch_stride + s];
      known = row >= 0 && row < (int64_t)a.table_rows;
    }
#pragma unroll
    for (uint32_t j = 0; j < kChunks; ++j) {
      float x[V], y[V];
#pragma unroll
      for (uint32_t i = 0; i < V; ++i) {
        x[i] = known ? 1.0f : __builtin_nanf("");
        y[i] = known ? 0.0f : __builtin_nanf("");
      }
      if (rotated(j) && known) {
        const uint64_t at = (uint64_t)row * a.table_ld + first(j);
        const typename Run<float, V>::Vec cv = Run<float, V>::load(a.cos + at), sv = Run<float, V>::load(a.sin + at);
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) x[i] = cv[i], y[i] = sv[i];
      }
#pragma unroll
      for (uint32_t i = 0; i < V; ++i) c[j * V + i] = x[i], n[j * V + i] = y[i];
    }
  }
};

// What a workgroup has to do: the first q_grid take the queries, the others the keys. The groups of a
// wavefront lie side by side: `abreast` of them share a token and take every abreast-th of its heads, segment by
// segment; a wavefront's unit is one segment of 64 / lanes / abreast tokens.
struct Share {
  const sh_heads& in;
  const sh_heads& out;
  const sh_heads& din;
  uint32_t heads, block, grid, segments, abreast, phase, token_of, per_wave;
  uint64_t units;

  __device__ __forceinline__ Share(const sh::QkNormKernelArgs& ka, bool is_k)
      : in(is_k ? ka.a.k : ka.a.q), out(is_k ? ka.a.k_out : ka.a.q_out), din(is_k ? ka.a.dk : ka.a.dq) {
    const sh::QkNormPart& part = ka.part[is_k];
    heads = is_k ? ka.a.k_heads : ka.a.q_heads;
    block = blockIdx.x - (is_k ? ka.part[0].grid : 0);
    grid = part.grid;
    segments = part.segments;
    abreast = part.abreast;
    units = part.units;
    const uint32_t group = (threadIdx.x & 63) / ka.lanes;
    phase = group & (abreast - 1);
    token_of = group / abreast;
    per_wave = 64 / ka.lanes / abreast;
  }
};

template <typename T, uint32_t V, bool INTERLEAVED>
__device__ __forceinline__ void forward(const sh::QkNormKernelArgs& ka) {
  const sh_qk_norm_rope_args& a = ka.a;
  const bool is_k = blockIdx.x >= ka.part[0].grid;
  const Share m(ka, is_k);
  const uint32_t lanes = ka.lanes;
  const Pairs<T, V, INTERLEAVED> pairs(a, threadIdx.x & (lanes - 1), lanes);
  const float rdim = 1.0f / (float)a.dim;
  const uint64_t tokens = (uint64_t)a.batch * a.seq;
  __shared__ alignas(16) float shared[SH_QK_MAX_DIM];
  share_weight(shared, is_k ? a.k_weight : a.q_weight, a.weight_dtype, a.dim);
  __syncthreads();
  float w0[kSlots], w1[kSlots];
  pairs.load_weight(shared, w0, w1);
  constexpr uint32_t kWaves = sh::kQkThreads / 64;
  for (uint64_t unit = (uint64_t)m.block * kWaves + threadIdx.x / 64; unit < m.units; unit += (uint64_t)m.grid * kWaves) {
    const uint64_t t = unit / m.segments * m.per_wave + m.token_of;
    const uint32_t seg = (uint32_t)(unit % m.segments);
    if (t >= tokens) continue;
    const uint64_t b = t / a.seq, s = t % a.seq;
    const T* x = static_cast<const T*>(m.in.data) + b * m.in.batch_stride + s * m.in.seq_stride;
    T* y = static_cast<T*>(m.out.data) + b * m.out.batch_stride + s * m.out.seq_stride;
    float c[kSlots], n[kSlots];
    pairs.load_angles(a, b, s, c, n);
    for (uint32_t h = seg * m.abreast + m.phase; h < m.heads; h += m.segments * m.abreast) {
      float x0[kSlots], x1[kSlots], sq = 0.0f;
      pairs.load(x + h * m.in.head_stride).values(x0, x1);
#pragma unroll
      for (uint32_t i = 0; i < kSlots; ++i) sq = __builtin_fmaf(x0[i], x0[i], __builtin_fmaf(x1[i], x1[i], sq));
      const float r = inv_sqrt(group_sum(sq, lanes) * rdim + a.eps);
#pragma unroll
      for (uint32_t i = 0; i < kSlots; ++i) {
        const float n0 = x0[i] * r * w0[i], n1 = x1[i] * r * w1[i];
        x0[i] = n0 * c[i] - n1 * n[i];
        x1[i] = n1 * c[i] + n0 * n[i];
      }
      pairs.store(y + h * m.out.head_stride, x0, x1);
    }
  }
}

template <typename T, uint32_t V, bool INTERLEAVED>
__device__ __forceinline__ void backward(const sh::QkNormKernelArgs& ka) {
  const sh_qk_norm_rope_args& a = ka.a;
  const bool is_k = blockIdx.x >= ka.part[0].grid;
  const Share m(ka, is_k);
  const uint32_t lanes = ka.lanes, wave = threadIdx.x / 64;
  const Pairs<T, V, INTERLEAVED> pairs(a, threadIdx.x & (lanes - 1), lanes);
  const float rdim = 1.0f / (float)a.dim;
  const uint64_t tokens = (uint64_t)a.batch * a.seq;
  constexpr uint32_t kWaves = sh::kQkThreads / 64;
  __shared__ alignas(16) float shared[kWaves][SH_QK_MAX_DIM];
  share_weight(shared[0], is_k ? a.k_weight : a.q_weight, a.weight_dtype, a.dim);
  __syncthreads();
  float w0[kSlots], w1[kSlots], dw0[kSlots] = {}, dw1[kSlots] = {};
  pairs.load_weight(shared[0], w0, w1);
  for (uint64_t unit = (uint64_t)m.block * kWaves + wave; unit < m.units; unit += (uint64_t)m.grid * kWaves) {
    const uint64_t t = unit / m.segments * m.per_wave + m.token_of;
    const uint32_t seg = (uint32_t)(unit % m.segments);
    if (t >= tokens) continue;
    const uint64_t b = t / a.seq, s = t % a.seq;
    const T* x = static_cast<const T*>(m.in.data) + b * m.in.batch_stride + s * m.in.seq_stride;
    const T* dy = static_cast<const T*>(m.out.data) + b * m.out.batch_stride + s * m.out.seq_stride;
    T* dx = static_cast<T*>(m.din.data) + b * m.din.batch_stride + s * m.din.seq_stride;
    float c[kSlots], n[kSlots];
    pairs.load_angles(a, b, s, c, n);
    for (uint32_t h = seg * m.abreast + m.phase; h < m.heads; h += m.segments * m.abreast) {
      float x0[kSlots], x1[kSlots], y0[kSlots], y1[kSlots], sq = 0.0f, dot = 0.0f;
      const auto xr = pairs.load(x + h * m.in.head_stride);
      const auto yr = pairs.load(dy + h * m.out.head_stride);
      xr.values(x0, x1);
      yr.values(y0, y1);
#pragma unroll
      for (uint32_t i = 0; i < kSlots; ++i) {
        const float g0 = y0[i] * c[i] + y1[i] * n[i], g1 = y1[i] * c[i] - y0[i] * n[i];
        y0[i] = g0;
        y1[i] = g1;
        sq = __builtin_fmaf(x0[i], x0[i], __builtin_fmaf(x1[i], x1[i], sq));
        dot = __builtin_fmaf(g0 * w0[i], x0[i], __builtin_fmaf(g1 * w1[i], x1[i], dot));
      }
      const float r = inv_sqrt(group_sum(sq, lanes) * rdim + a.eps);
      const float mean = group_sum(dot, lanes) * r * rdim;  // of h x^
#pragma unroll
      for (uint32_t i = 0; i < kSlots; ++i) {
        x0[i] *= r;
        x1[i] *= r;
        dw0[i] = __builtin_fmaf(y0[i], x0[i], dw0[i]);
        dw1[i] = __builtin_fmaf(y1[i], x1[i], dw1[i]);
        x0[i] = r * (y0[i] * w0[i] - x0[i] * mean);
        x1[i] = r * (y1[i] * w1[i] - x1[i] * mean);
      }
      if (m.din.data != nullptr) pairs.store(dx + h * m.din.head_stride, x0, x1);
    }
  }
  if (ka.partials == nullptr) return;
  // The workgroup's sums: over a wavefront's groups, then over the wavefronts, always in the same order.
#pragma unroll
  for (uint32_t i = 0; i < kSlots; ++i) {
    for (uint32_t d = lanes; d < 64; d *= 2) {
      dw0[i] += __shfl_xor(dw0[i], (int)d);
      dw1[i] += __shfl_xor(dw1[i], (int)d);
    }
  }
  __syncthreads();
  if ((threadIdx.x & 63) < lanes) pairs.template store<(V >= 4 ? 16 : 4 * V)>(shared[wave], dw0, dw1);
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < a.dim; i += sh::kQkThreads) {
    float v = 0.0f;
    for (uint32_t w = 0; w < kWaves; ++w) v += shared[w][i];
    ka.partials[(uint64_t)blockIdx.x * a.dim + i] = v;
  }
}

}  // namespace

#define SH_QK(name, T, V)                                                                                           \
  extern "C" __global__ __launch_bounds__(sh::kQkThreads) void sh_qk_norm_##name##_##V##_kernel(                    \
      sh::QkNormKernelArgs ka) {                                                                                    \
    forward<T, V, false>(ka);                                                                                       \
  }                                                                                                                 \
  extern "C" __global__ __launch_bounds__(sh::kQkThreads) void sh_qk_norm_##name##_##V##_interleaved_kernel(        \
      sh::QkNormKernelArgs ka) {                                                                                    \
    forward<T, V, true>(ka);                                                                                        \
  }                                                                                                                 \
  extern "C" __global__ __launch_bounds__(sh::kQkThreads) void sh_qk_norm_backward_##name##_##V##_kernel(           \
      sh::QkNormKernelArgs ka) {                                                                                    \
    backward<T, V, false>(ka);                                                                                      \
  }                                                                                                                 \
  extern "C" __global__ __launch_bounds__(sh::kQkThreads) void sh_qk_norm_backward_##name##_##V##_interleaved_kernel( \
      sh::QkNormKernelArgs ka) {                                                                                    \
    backward<T, V, true>(ka);                                                                                       \
  }
SH_QK(bf16, __bf16, 8)
SH_QK(bf16, __bf16, 4)
SH_QK(bf16, __bf16, 2)
SH_QK(bf16, __bf16, 1)
SH_QK(f16, _Float16, 8)
SH_QK(f16, _Float16, 4)
SH_QK(f16, _Float16, 2)
SH_QK(f16, _Float16, 1)
SH_QK(f32, float, 8)
SH_QK(f32, float, 4)
SH_QK(f32, float, 2)
SH_QK(f32, float, 1)

// dweight[i] = sum of the workgroups' partial sums. A workgroup takes 32 values i of the queries' or the keys'
// weight; 8 work-items add up each, every 8th partial, and are joined in order.
extern "C" __global__ __launch_bounds__(sh::kQkThreads) void sh_qk_norm_dweight_kernel(sh::QkNormKernelArgs ka) {
  const sh_qk_norm_rope_args& a = ka.a;
  const uint32_t blocks = (a.dim + 31) / 32;
  const uint32_t which = blockIdx.x / blocks, i = blockIdx.x % blocks * 32 + threadIdx.x % 32;
  void* out = which == 0 ? a.dq_weight : a.dk_weight;
  if (out == nullptr) return;
  __shared__ float part[8][32];
  float v = 0.0f;
  if (i < a.dim) {
    const float* p = ka.partials + (which == 0 ? 0 : (uint64_t)ka.part[0].grid * a.dim) + i;
#pragma unroll 8
    for (uint32_t b = threadIdx.x / 32; b < ka.part[which].grid; b += 8) v += p[(uint64_t)b * a.dim];
  }
  part[threadIdx.x / 32][threadIdx.x % 32] = v;
  __syncthreads();
  if (threadIdx.x >= 32 || i >= a.dim) return;
  v = 0.0f;
  for (uint32_t w = 0; w < 8; ++w) v += part[w][threadIdx.x];
  if (a.weight_dtype == SH_DTYPE_BF16) static_cast<__bf16*>(out)[i] = (__bf16)v;
  else if (a.weight_dtype == SH_DTYPE_F16) static_cast<_Float16*>(out)[i] = (_Float16)v;
  else static_cast<float*>(out)[i] = v;
}
