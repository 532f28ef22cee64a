// RMS norms of queries and keys with the position rotation, forward and backward (no reference
// counterpart: the reference runs the models' own torch modules).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "sh_internal.h"
#include "sh_qk_norm_args.h"
#include "stagehand_native.h"

namespace {

using sh::dtype_bytes;
using sh::known_dtype;
using sh::misaligned;

int check_heads(const sh_heads& v, const char* name, uint32_t heads, uint32_t dtype, const char* who) {
  if (heads == 0) return SH_OK;
  if (v.data == nullptr) return sh::fail(SH_ERR_INVALID, "%s: %s is NULL", who, name);
  if (misaligned(v.data, dtype_bytes(dtype)))
    return sh::fail(SH_ERR_INVALID, "%s: %s is not aligned to its type", who, name);
  return SH_OK;
}

int check(const sh_qk_norm_rope_args* a, bool backward, const char* who) {
  if (a == nullptr) return sh::fail(SH_ERR_INVALID, "%s: args is NULL", who);
  if (!known_dtype(a->dtype)) return sh::fail(SH_ERR_INVALID, "%s: unknown dtype %u", who, a->dtype);
  if (!known_dtype(a->weight_dtype))
    return sh::fail(SH_ERR_INVALID, "%s: unknown weight_dtype %u", who, a->weight_dtype);
  if (a->dim < 2 || a->dim % 2 != 0 || a->dim > SH_QK_MAX_DIM)
    return sh::fail(SH_ERR_INVALID, "%s: dim %u is not an even number in 2 .. %u", who, a->dim, SH_QK_MAX_DIM);
  if (a->rot % 2 != 0 || a->rot > a->dim)
    return sh::fail(SH_ERR_INVALID, "%s: rot %u is not an even number in 0 .. %u", who, a->rot, a->dim);
  if (!(a->eps >= 0.0f) || std::isinf(a->eps)) return sh::fail(SH_ERR_INVALID, "%s: eps is negative or not finite", who);
  if ((double)a->batch * a->seq * std::max(a->q_heads, a->k_heads) > 4294967295.0)
    return sh::fail(SH_ERR_INVALID, "%s: %u x %u tokens of %u and %u heads are too many for one launch", who, a->batch,
                    a->seq, a->q_heads, a->k_heads);
  if (a->batch == 0 || a->seq == 0) return SH_OK;
  if (a->rot > 0) {
    if (a->cos == nullptr || a->sin == nullptr) return sh::fail(SH_ERR_INVALID, "%s: cos or sin is NULL", who);
    if (misaligned(a->cos, 4) || misaligned(a->sin, 4))
      return sh::fail(SH_ERR_INVALID, "%s: cos or sin is not 4-byte aligned", who);
    if (a->table_rows > 1 && a->table_ld < a->rot / 2)
      return sh::fail(SH_ERR_INVALID, "%s: table_ld %llu is less than rot / 2 = %u", who,
                      (unsigned long long)a->table_ld, a->rot / 2);
    if (a->positions != nullptr) {
      if (a->position_bytes != 4 && a->position_bytes != 8)
        return sh::fail(SH_ERR_INVALID, "%s: position_bytes %u is not 4 or 8", who, a->position_bytes);
      if (misaligned(a->positions, a->position_bytes))
        return sh::fail(SH_ERR_INVALID, "%s: positions is not aligned to its type", who);
    } else if (a->start < 0 || a->start > (int64_t)a->table_rows || a->seq > a->table_rows - (uint64_t)a->start) {
      return sh::fail(SH_ERR_INVALID, "%s: positions %lld .. %lld are not all in the tables' %u rows", who,
                      (long long)a->start, (long long)a->start + a->seq - 1, a->table_rows);
    }
  }
  if (int st = check_heads(a->q, "q", a->q_heads, a->dtype, who)) return st;
  if (int st = check_heads(a->k, "k", a->k_heads, a->dtype, who)) return st;
  if (int st = check_heads(a->q_out, "q_out", a->q_heads, a->dtype, who)) return st;
  if (int st = check_heads(a->k_out, "k_out", a->k_heads, a->dtype, who)) return st;
  if (misaligned(a->q_weight, dtype_bytes(a->weight_dtype)) || misaligned(a->k_weight, dtype_bytes(a->weight_dtype)))
    return sh::fail(SH_ERR_INVALID, "%s: a weight is not aligned to its type", who);
  if (backward) {
    if (misaligned(a->dq.data, dtype_bytes(a->dtype)) || misaligned(a->dk.data, dtype_bytes(a->dtype)))
      return sh::fail(SH_ERR_INVALID, "%s: dq or dk is not aligned to its type", who);
    if (misaligned(a->dq_weight, dtype_bytes(a->weight_dtype)) ||
        misaligned(a->dk_weight, dtype_bytes(a->weight_dtype)))
      return sh::fail(SH_ERR_INVALID, "%s: a weight's gradient is not aligned to its type", who);
  }
  return SH_OK;
}

// Work-items that share a head: the power of two that holds dim / 2 pairs, kQkSlots each.
uint32_t lanes_of(uint32_t dim) {
  uint32_t lanes = 1;
  while (lanes * sh::kQkSlots < dim / 2) lanes *= 2;
  return lanes;
}

// log2 of the pairs that are loaded and stored together, 8 at most: a head's rotated pairs and all its pairs
// come in whole runs.
uint32_t log_run(const sh_qk_norm_rope_args* a) {
  uint32_t n = 3;
  while ((a->rot / 2 | a->dim / 2) & ((1u << n) - 1)) --n;
  return n;
}

constexpr uint32_t kComputeUnits = 256;
constexpr uint32_t kWaves = sh::kQkThreads / 64;
// Workgroups at most: what runs at a time, so that each loads the weights once and takes many tokens.
constexpr uint32_t kForwardGrid = 8 * kComputeUnits, kBackwardGrid = 3 * kComputeUnits;

sh::QkNormKernelArgs kernel_args(const sh_qk_norm_rope_args* a, bool backward) {
  sh::QkNormKernelArgs ka{};
  ka.a = *a;
  ka.lanes = lanes_of(a->dim);
  const uint64_t tokens = (uint64_t)a->batch * a->seq, all = (uint64_t)a->q_heads + a->k_heads;
  for (int i = 0; i < 2; ++i) {
    sh::QkNormPart& p = ka.part[i];
    const uint32_t heads = i == 0 ? a->q_heads : a->k_heads;
    p.abreast = p.segments = 1;
    if (heads == 0 || tokens == 0) continue;
    while (p.abreast < heads && p.abreast < 64 / ka.lanes) p.abreast *= 2;
    const uint64_t per_wave = 64 / ka.lanes / p.abreast, groups = (tokens + per_wave - 1) / per_wave;
    // Few tokens: their heads are spread over more wavefronts, to eight a compute unit.
    const uint64_t most = ((uint64_t)heads + p.abreast - 1) / p.abreast;
    p.segments = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(most, 8 * kComputeUnits / groups));
    p.units = groups * p.segments;
    const uint64_t grid = std::max<uint64_t>(1, (backward ? kBackwardGrid : kForwardGrid) * heads / all);
    p.grid = (uint32_t)std::min<uint64_t>((p.units + kWaves - 1) / kWaves, grid);
  }
  return ka;
}

uint32_t grid_of(const sh::QkNormKernelArgs& ka) { return ka.part[0].grid + ka.part[1].grid; }

bool wants_dweight(const sh_qk_norm_rope_args* a) { return a->dq_weight != nullptr || a->dk_weight != nullptr; }

uint64_t partial_bytes(const sh::QkNormKernelArgs& ka) {
  return wants_dweight(&ka.a) ? 4ull * ka.a.dim * grid_of(ka) : 0;
}

// Four kernels for each type and run: forward, forward interleaved, backward, backward interleaved.
sh::KernelId kernel_of(const sh_qk_norm_rope_args* a, bool backward) {
  static_assert(sh::kKernQkNormBackwardF321Interleaved - sh::kKernQkNormBf168 == 3 * 4 * 4 - 1, "one kernel per variant");
  return (sh::KernelId)(sh::kKernQkNormBf168 + ((a->dtype - SH_DTYPE_BF16) * 4 + 3 - log_run(a)) * 4 + (backward ? 2 : 0) +
                        (a->interleaved ? 1 : 0));
}

}  // namespace

extern "C" int sh_qk_norm_rope(const sh_qk_norm_rope_args* args, void* stream) {
  const char* who = "sh_qk_norm_rope";
  sh::clear_error();
  if (int st = check(args, false, who)) return st;
  const sh::QkNormKernelArgs ka = kernel_args(args, false);
  if (grid_of(ka) == 0) return SH_OK;
  void* list[] = {(void*)&ka};
  return sh::launch_kernel(kernel_of(args, false), grid_of(ka), sh::kQkThreads, (hipStream_t)stream, list, who);
}

extern "C" int sh_qk_norm_rope_workspace(const sh_qk_norm_rope_args* args, uint64_t* bytes) {
  const char* who = "sh_qk_norm_rope_workspace";
  sh::clear_error();
  if (bytes == nullptr) return sh::fail(SH_ERR_INVALID, "%s: bytes is NULL", who);
  if (args == nullptr) return sh::fail(SH_ERR_INVALID, "%s: args is NULL", who);
  if (args->dim > SH_QK_MAX_DIM)
    return sh::fail(SH_ERR_INVALID, "%s: dim %u is more than %u", who, args->dim, SH_QK_MAX_DIM);
  *bytes = partial_bytes(kernel_args(args, true));
  return SH_OK;
}

extern "C" int sh_qk_norm_rope_backward(const sh_qk_norm_rope_args* args, void* workspace, uint64_t workspace_bytes,
                                        void* stream) {
  const char* who = "sh_qk_norm_rope_backward";
  sh::clear_error();
  if (int st = check(args, true, who)) return st;
  sh::QkNormKernelArgs ka = kernel_args(args, true);
  const uint64_t need = partial_bytes(ka);
  if (workspace_bytes < need || (need > 0 && workspace == nullptr))
    return sh::fail(SH_ERR_INVALID, "%s: the workspace holds %llu bytes, %llu are needed", who,
                    (unsigned long long)workspace_bytes, (unsigned long long)need);
  if (misaligned(workspace, 16)) return sh::fail(SH_ERR_INVALID, "%s: workspace is not 16-byte aligned", who);
  ka.partials = wants_dweight(args) ? static_cast<float*>(workspace) : nullptr;
  void* list[] = {(void*)&ka};
  if (grid_of(ka) > 0)
    if (int st = sh::launch_kernel(kernel_of(args, true), grid_of(ka), sh::kQkThreads, (hipStream_t)stream, list, who))
      return st;
  if (!wants_dweight(args)) return SH_OK;
  // without tokens the sums are over nothing: zeros
  return sh::launch_kernel(sh::kKernQkNormDweight, 2 * ((args->dim + 31) / 32), sh::kQkThreads, (hipStream_t)stream, list, who);
}
