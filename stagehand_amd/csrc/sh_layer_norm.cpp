// Layer norm, forward and backward (no reference counterpart: the reference runs the models' own torch modules).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "sh_internal.h"
#include "sh_layer_norm_args.h"
#include "stagehand_native.h"

namespace {

// Sequences with a weight of their own, a workgroup each at least, in one launch of under 2^32 work-items.
constexpr uint32_t kMostGroups = 0xFFFFFFFFu / sh::norm_most_threads(true);

using sh::dtype_bytes;
using sh::known_dtype;
using sh::misaligned;

int check_rows(const sh_rows& r, const char* name, uint32_t dtype, const char* who) {
  if (r.data == nullptr) return sh::fail(SH_ERR_INVALID, "%s: %s is NULL", who, name);
  if (misaligned(r.data, dtype_bytes(dtype))) return sh::fail(SH_ERR_INVALID, "%s: %s is not aligned to its type", who, name);
  return SH_OK;
}

int check(const sh_layer_norm_args* a, bool backward, const char* who) {
  if (a == nullptr) return sh::fail(SH_ERR_INVALID, "%s: args is NULL", who);
  if (!known_dtype(a->dtype)) return sh::fail(SH_ERR_INVALID, "%s: unknown dtype %u", who, a->dtype);
  if (!known_dtype(a->weight_dtype)) return sh::fail(SH_ERR_INVALID, "%s: unknown weight_dtype %u", who, a->weight_dtype);
  if (a->cols == 0 || a->cols > SH_LAYER_NORM_MAX_COLS)
    return sh::fail(SH_ERR_INVALID, "%s: cols %u is not in 1 .. %u", who, a->cols, SH_LAYER_NORM_MAX_COLS);
  if (!(a->eps >= 0.0f) || std::isinf(a->eps)) return sh::fail(SH_ERR_INVALID, "%s: eps is negative or not finite", who);
  if ((uint64_t)a->batch * a->seq > 0x7FFFFFFFu || (a->per_batch && a->batch > kMostGroups))
    return sh::fail(SH_ERR_INVALID, "%s: %u x %u tokens are too many for one launch", who, a->batch, a->seq);
  const uint32_t wb = dtype_bytes(a->weight_dtype);
  if (misaligned(a->weight, wb) || misaligned(a->bias, wb) || misaligned(a->dweight, wb) || misaligned(a->dbias, wb))
    return sh::fail(SH_ERR_INVALID, "%s: weight, bias or a gradient of them is not aligned to its type", who);
  if (a->batch == 0 || a->seq == 0) return SH_OK;
  if (misaligned(a->stats, 4)) return sh::fail(SH_ERR_INVALID, "%s: stats is not 4-byte aligned", who);
  if ((a->q == nullptr) != (a->exponent == nullptr))
    return sh::fail(SH_ERR_INVALID, "%s: q and exponent are given together or not at all", who);
  if (misaligned(a->q, 16)) return sh::fail(SH_ERR_INVALID, "%s: q is not 16-byte aligned", who);
  if (!backward) {
    if (int st = check_rows(a->x, "x", a->dtype, who)) return st;
    return check_rows(a->y, "y", a->dtype, who);
  }
  if (a->stats == nullptr) return sh::fail(SH_ERR_INVALID, "%s: stats is NULL", who);
  if (a->q == nullptr)
    if (int st = check_rows(a->x, "x", a->dtype, who)) return st;
  if (misaligned(a->dx.data, dtype_bytes(a->dtype))) return sh::fail(SH_ERR_INVALID, "%s: dx is not aligned to its type", who);
  return check_rows(a->dy, "dy", a->dtype, who);
}

constexpr uint32_t kComputeUnits = 256;

int shape_of(uint32_t cols) {
  int i = 0;
  while (sh::norm_capacity(sh::kNormShapes[i]) < cols) ++i;
  return i;
}

sh::LayerNormKernelArgs kernel_args(const sh_layer_norm_args* a, bool backward) {
  sh::LayerNormKernelArgs ka{};
  ka.a = *a;
  ka.groups = a->per_batch ? a->batch : 1;
  ka.tokens = a->per_batch ? a->seq : a->batch * a->seq;
  const sh::NormShape shape = sh::kNormShapes[shape_of(a->cols)];
  const uint32_t chunks = (a->cols + 7) / 8;
  uint32_t teams = 1;  // of a workgroup
  if (shape.team) {
    ka.lanes = (chunks + 64 * shape.chunks - 1) / (64 * shape.chunks) * 64;
  } else {
    for (ka.lanes = 4; ka.lanes < 64 && ka.lanes < chunks;) ka.lanes *= 2;
    teams = sh::kNormThreads / ka.lanes;
  }
  const uint32_t threads = shape.team ? ka.lanes : sh::kNormThreads, groups = std::max(1u, ka.groups);
  const uint32_t useful = (ka.tokens + teams - 1) / teams;
  uint32_t per_group;
  if (!backward) {
    // Work-items a compute unit, times in us. 65536 x 256: 1024 15.1, 1536 14.5, 2048 14.9; x 512 26.2, 24.6, 25.9. Longer rows, 2 x
    // 8192 x 4096: 512 53, 1024 46, 2048 49.
    per_group = kComputeUnits * ((shape.chunks == 1 ? 1536 : 1024) / threads) / groups;
  } else {
    // Every workgroup leaves a set of sums, that is written and read once more: 16 MB of them at most, and no team has fewer
    // than three tokens.
    const uint32_t fit = (16u << 20) / (8 * a->cols) / kComputeUnits;
    per_group = std::min(kComputeUnits * (shape.team ? std::min(std::max(fit, 1u), 4u) : 3) / groups, (useful + 2) / 3);
  }
  ka.per_group = std::max(1u, std::min(per_group, useful));
  return ka;
}

bool wants_params(const sh_layer_norm_args* a) { return a->dweight != nullptr || a->dbias != nullptr; }

uint64_t partial_bytes(const sh::LayerNormKernelArgs& ka) {
  if (!wants_params(&ka.a) || ka.per_group == 1) return 0;
  return 8ull * ka.a.cols * ka.groups * ka.per_group;
}

// Three kernels for each type and shape: forward, backward, backward from what was kept.
sh::KernelId kernel_of(const sh_layer_norm_args* a, int pass) {
  static_assert(sh::kKernLayerNormJoin - sh::kKernLayerNormBf16Wave1 == 3 * sh::kNormShapeCount * 3, "one kernel per variant");
  return (sh::KernelId)(sh::kKernLayerNormBf16Wave1 + ((a->dtype - SH_DTYPE_BF16) * sh::kNormShapeCount + shape_of(a->cols)) * 3 + pass);
}

int launch(const sh::LayerNormKernelArgs& ka, int pass, hipStream_t stream, const char* who) {
  void* list[] = {(void*)&ka};
  return sh::launch_kernel(kernel_of(&ka.a, pass), ka.groups * ka.per_group,
                           sh::kNormShapes[shape_of(ka.a.cols)].team ? ka.lanes : sh::kNormThreads, stream, list, who);
}

}  // namespace

extern "C" int sh_layer_norm(const sh_layer_norm_args* args, void* stream) {
  const char* who = "sh_layer_norm";
  sh::clear_error();
  if (int st = check(args, false, who)) return st;
  if (args->batch == 0 || args->seq == 0) return SH_OK;
  return launch(kernel_args(args, false), 0, (hipStream_t)stream, who);
}

extern "C" int sh_layer_norm_workspace(const sh_layer_norm_args* args, uint64_t* bytes) {
  const char* who = "sh_layer_norm_workspace";
  sh::clear_error();
  if (bytes == nullptr) return sh::fail(SH_ERR_INVALID, "%s: bytes is NULL", who);
  if (args == nullptr) return sh::fail(SH_ERR_INVALID, "%s: args is NULL", who);
  if (args->cols == 0 || args->cols > SH_LAYER_NORM_MAX_COLS)
    return sh::fail(SH_ERR_INVALID, "%s: cols %u is not in 1 .. %u", who, args->cols, SH_LAYER_NORM_MAX_COLS);
  *bytes = partial_bytes(kernel_args(args, true));
  return SH_OK;
}

extern "C" int sh_layer_norm_backward(const sh_layer_norm_args* args, void* workspace, uint64_t workspace_bytes, void* stream) {
  const char* who = "sh_layer_norm_backward";
  sh::clear_error();
  if (int st = check(args, true, who)) return st;
  sh::LayerNormKernelArgs ka = kernel_args(args, true);
  const uint64_t need = partial_bytes(ka);
  if (workspace_bytes < need || (need > 0 && workspace == nullptr))
    return sh::fail(SH_ERR_INVALID, "%s: the workspace holds %llu bytes, %llu are needed", who,
                    (unsigned long long)workspace_bytes, (unsigned long long)need);
  if (misaligned(workspace, 16)) return sh::fail(SH_ERR_INVALID, "%s: workspace is not 16-byte aligned", who);
  if (ka.groups == 0 || (ka.tokens == 0 && !wants_params(args))) return SH_OK;
  ka.partials = need > 0 ? static_cast<float*>(workspace) : nullptr;
  // without tokens the sums are over nothing: zeros
  if (int st = launch(ka, args->q != nullptr ? 2 : 1, (hipStream_t)stream, who)) return st;
  if (need == 0) return SH_OK;
  void* list[] = {(void*)&ka};
  const uint32_t blocks = (args->cols + sh::kNormJoinCols - 1) / sh::kNormJoinCols;
  return sh::launch_kernel(sh::kKernLayerNormJoin, ka.groups * 2 * blocks, sh::kNormJoinThreads, (hipStream_t)stream, list, who);
}
