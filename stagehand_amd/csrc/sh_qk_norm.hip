// Query/key norms with the position rotation for gfx950 (device code only; the checks and the
// launches are in sh_qk_norm.cpp).
//
// A head's values are taken as dim / 2 pairs. Pairs p < rot / 2 are rotated: (p, p + rot / 2), or
// (2p, 2p + 1) when interleaved. The values past rot form pairs the same way with the angle 0, so
// every pair is handled alike. `lanes` work-items share a head, each holds kQkSlots pairs in registers.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "sh_qk_norm_args.h"

namespace {

constexpr uint32_t kSlots = sh::kQkSlots;

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

// The places of pair p's two values in a head.
__device__ __forceinline__ void pair_places(uint32_t p, uint32_t dim, uint32_t rot, bool interleaved, uint32_t* i0,
                                            uint32_t* i1) {
  if (interleaved) {
    *i0 = 2 * p;
    *i1 = 2 * p + 1;
  } else if (p < rot / 2) {
    *i0 = p;
    *i1 = p + rot / 2;
  } else {
    *i0 = rot / 2 + p;
    *i1 = *i0 + (dim - rot) / 2;
  }
}

struct Row {
  uint64_t b, h, s;
};

__device__ __forceinline__ uint64_t at(const sh_heads& v, const Row& r) {
  return r.b * v.batch_stride + r.h * v.head_stride + r.s * v.seq_stride;
}

// A token's row of the tables, or -1 where it has none.
__device__ __forceinline__ int64_t table_row(const sh_qk_norm_rope_args& a, const Row& r) {
  int64_t p;
  if (a.positions == nullptr) p = a.start + (int64_t)r.s;
  else if (a.position_bytes == 8) p = static_cast<const int64_t*>(a.positions)[r.b * a.position_batch_stride + r.s];
  else p = static_cast<const int32_t*>(a.positions)[r.b * a.position_batch_stride + r.s];
  return p >= 0 && p < (int64_t)a.table_rows ? p : -1;
}

template <bool BACKWARD>
__device__ __forceinline__ void qk_norm_body(const sh::QkNormKernelArgs& ka) {
  const sh_qk_norm_rope_args& a = ka.a;
  const bool is_k = blockIdx.x >= ka.q_grid;
  const uint32_t block = is_k ? blockIdx.x - ka.q_grid : blockIdx.x;
  const uint32_t grid = is_k ? ka.k_grid : ka.q_grid;
  const uint32_t heads = is_k ? a.k_heads : a.q_heads;
  const sh_heads& in = is_k ? a.k : a.q;
  const sh_heads& out = is_k ? a.k_out : a.q_out;
  const sh_heads& din = is_k ? a.dk : a.dq;
  const void* weight = is_k ? a.k_weight : a.q_weight;
  const uint32_t lanes = ka.lanes, groups = sh::kQkThreads / lanes;
  const uint32_t lane = threadIdx.x % lanes, group = threadIdx.x / lanes;
  const bool interleaved = a.interleaved != 0;
  const float rdim = 1.0f / (float)a.dim;
  float dw0[kSlots] = {}, dw1[kSlots] = {};

  const uint64_t rows = (uint64_t)a.batch * a.seq * heads;
  for (uint64_t row = (uint64_t)block * groups + group; row < rows; row += (uint64_t)grid * groups) {
    const Row r{row / heads / a.seq, row % heads, row / heads % a.seq};
    const int64_t tr = a.rot > 0 ? table_row(a, r) : 0;
    float x0[kSlots], x1[kSlots], sq = 0.0f;
#pragma unroll
    for (uint32_t j = 0; j < kSlots; ++j) {
      const uint32_t p = j * lanes + lane;
      x0[j] = x1[j] = 0.0f;
      if (p < a.dim / 2) {
        uint32_t i0, i1;
        pair_places(p, a.dim, a.rot, interleaved, &i0, &i1);
        x0[j] = load_value(in.data, at(in, r) + i0, a.dtype);
        x1[j] = load_value(in.data, at(in, r) + i1, a.dtype);
      }
      sq += x0[j] * x0[j] + x1[j] * x1[j];
    }
    for (uint32_t m = lanes / 2; m >= 1; m >>= 1) sq += __shfl_xor(sq, (int)m);
    const float rstd = 1.0f / __builtin_sqrtf(sq * rdim + a.eps);
    float g0[kSlots], g1[kSlots], dot = 0.0f;
#pragma unroll
    for (uint32_t j = 0; j < kSlots; ++j) {
      const uint32_t p = j * lanes + lane;
      if (p >= a.dim / 2) continue;
      uint32_t i0, i1;
      pair_places(p, a.dim, a.rot, interleaved, &i0, &i1);
      float c = 1.0f, s = 0.0f;
      if (p < a.rot / 2) {
        c = tr < 0 ? __builtin_nanf("") : a.cos[(uint64_t)tr * a.table_ld + p];
        s = tr < 0 ? __builtin_nanf("") : a.sin[(uint64_t)tr * a.table_ld + p];
      }
      const float w0 = weight != nullptr ? load_value(weight, i0, a.weight_dtype) : 1.0f;
      const float w1 = weight != nullptr ? load_value(weight, i1, a.weight_dtype) : 1.0f;
      x0[j] *= rstd;
      x1[j] *= rstd;
      if (!BACKWARD) {
        const float n0 = x0[j] * w0, n1 = x1[j] * w1;
        store_value(out.data, at(out, r) + i0, n0 * c - n1 * s, a.dtype);
        store_value(out.data, at(out, r) + i1, n1 * c + n0 * s, a.dtype);
      } else {
        const float y0 = load_value(out.data, at(out, r) + i0, a.dtype);
        const float y1 = load_value(out.data, at(out, r) + i1, a.dtype);
        g0[j] = y0 * c + y1 * s;
        g1[j] = y1 * c - y0 * s;
        dw0[j] += g0[j] * x0[j];
        dw1[j] += g1[j] * x1[j];
        g0[j] *= w0;
        g1[j] *= w1;
        dot += g0[j] * x0[j] + g1[j] * x1[j];
      }
    }
    if (BACKWARD && din.data != nullptr) {
      for (uint32_t m = lanes / 2; m >= 1; m >>= 1) dot += __shfl_xor(dot, (int)m);
      const float mean = dot * rdim;
#pragma unroll
      for (uint32_t j = 0; j < kSlots; ++j) {
        const uint32_t p = j * lanes + lane;
        if (p >= a.dim / 2) continue;
        uint32_t i0, i1;
        pair_places(p, a.dim, a.rot, interleaved, &i0, &i1);
        store_value(din.data, at(din, r) + i0, rstd * (g0[j] - x0[j] * mean), a.dtype);
        store_value(din.data, at(din, r) + i1, rstd * (g1[j] - x1[j] * mean), a.dtype);
      }
    }
  }
  if (BACKWARD && ka.partials != nullptr) {
    // the workgroup's sums, group after group
    __shared__ float sums[SH_QK_MAX_DIM];
    for (uint32_t i = threadIdx.x; i < a.dim; i += sh::kQkThreads) sums[i] = 0.0f;
    __syncthreads();
    for (uint32_t g = 0; g < groups; ++g) {
      if (g == group) {
#pragma unroll
        for (uint32_t j = 0; j < kSlots; ++j) {
          const uint32_t p = j * lanes + lane;
          if (p >= a.dim / 2) continue;
          uint32_t i0, i1;
          pair_places(p, a.dim, a.rot, interleaved, &i0, &i1);
          sums[i0] += dw0[j];
          sums[i1] += dw1[j];
        }
      }
      __syncthreads();
    }
    for (uint32_t i = threadIdx.x; i < a.dim; i += sh::kQkThreads)
      ka.partials[(uint64_t)blockIdx.x * a.dim + i] = sums[i];
  }
}

}  // namespace

extern "C" __global__ __launch_bounds__(sh::kQkThreads) void sh_qk_norm_rope_kernel(sh::QkNormKernelArgs ka) {
  qk_norm_body<false>(ka);
}

extern "C" __global__ __launch_bounds__(sh::kQkThreads) void sh_qk_norm_rope_backward_kernel(sh::QkNormKernelArgs ka) {
  qk_norm_body<true>(ka);
}

// dweight[i] = sum of the workgroups' partial sums: workgroup 0 the queries', workgroup 1 the keys'.
extern "C" __global__ __launch_bounds__(sh::kQkThreads) void sh_qk_norm_dweight_kernel(sh::QkNormKernelArgs ka) {
  const sh_qk_norm_rope_args& a = ka.a;
  const uint32_t first = blockIdx.x == 0 ? 0 : ka.q_grid;
  const uint32_t count = blockIdx.x == 0 ? ka.q_grid : ka.k_grid;
  void* out = blockIdx.x == 0 ? a.dq_weight : a.dk_weight;
  if (out == nullptr) return;
  for (uint32_t i = threadIdx.x; i < a.dim; i += sh::kQkThreads) {
    float v = 0.0f;
    for (uint32_t b = 0; b < count; ++b) v += ka.partials[(uint64_t)(first + b) * a.dim + i];
    store_value(out, i, v, a.weight_dtype);
  }
}
