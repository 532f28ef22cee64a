// Activations kept in 8 bits, and the weight gradients that read them (no reference counterpart: the reference
// leaves activations to torch).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "sh_act8_args.h"
#include "sh_internal.h"
#include "stagehand_native.h"

namespace {

using sh::dtype_bytes;
using sh::known_dtype;
using sh::misaligned;

uint32_t groups_of(uint32_t cols) { return cols / SH_ACT8_GROUP + (cols % SH_ACT8_GROUP != 0); }

int check_kept(const sh_act8* k, const char* who) {
  if (k == nullptr) return sh::fail(SH_ERR_INVALID, "%s: kept is NULL", who);
  if (k->cols == 0 || k->cols > SH_ACT8_MAX_COLS)
    return sh::fail(SH_ERR_INVALID, "%s: cols %u is not in 1 .. %u", who, k->cols, SH_ACT8_MAX_COLS);
  if ((uint64_t)k->tokens * groups_of(k->cols) * (SH_ACT8_GROUP / 8) > 0xFFFFFFFFull - sh::kAct8Threads)
    return sh::fail(SH_ERR_INVALID, "%s: %u tokens of %u values are too many for one launch", who, k->tokens, k->cols);
  if (k->tokens > 0 && (k->q == nullptr || k->exponent == nullptr))
    return sh::fail(SH_ERR_INVALID, "%s: q or exponent is NULL", who);
  if (misaligned(k->q, 16)) return sh::fail(SH_ERR_INVALID, "%s: q is not 16-byte aligned", who);
  return SH_OK;
}

int check_values(const void* x, const char* name, uint32_t dtype, uint32_t tokens, const char* who) {
  if (!known_dtype(dtype)) return sh::fail(SH_ERR_INVALID, "%s: unknown dtype %u", who, dtype);
  if (tokens == 0) return SH_OK;
  if (x == nullptr) return sh::fail(SH_ERR_INVALID, "%s: %s is NULL", who, name);
  if (misaligned(x, dtype_bytes(dtype))) return sh::fail(SH_ERR_INVALID, "%s: %s is not aligned to its type", who, name);
  return SH_OK;
}

// Rows of more than one do not overlap.
int check_apart(uint64_t ld, uint32_t rows, uint32_t cols, const char* name, const char* who) {
  if (rows > 1 && ld < cols)
    return sh::fail(SH_ERR_INVALID, "%s: %s %llu is less than the %u values of a row", who, name, (unsigned long long)ld, cols);
  return SH_OK;
}

int launch_act8(const sh_act8* k, void* x, uint64_t x_ld, uint32_t dtype, bool back, hipStream_t stream, const char* who) {
  static_assert(sh::kKernAct8QuantizeF16 == sh::kKernAct8QuantizeBf16 + 2 && sh::kKernAct8QuantizeF32 == sh::kKernAct8QuantizeBf16 + 4,
                "two kernels for each type, in the order of enum sh_dtype");
  if (k->tokens == 0) return SH_OK;
  sh::Act8Args a{};
  a.x = x;
  a.q = k->q;
  a.exponent = k->exponent;
  a.x_ld = x_ld;
  a.row_chunks = groups_of(k->cols) * (SH_ACT8_GROUP / 8);
  a.chunks = k->tokens * a.row_chunks;
  a.magic = sh::udiv_magic(a.row_chunks);
  a.tokens = k->tokens;
  a.cols = k->cols;
  constexpr uint32_t per = sh::kAct8Threads;
  void* args[] = {(void*)&a};
  return sh::launch_kernel((sh::KernelId)(sh::kKernAct8QuantizeBf16 + (dtype - SH_DTYPE_BF16) * 2 + back), (a.chunks + per - 1) / per,
                           sh::kAct8Threads, stream, args, who);
}

struct GradPlan {
  int tile;
  uint64_t tiles;
  uint32_t splits, split_tokens;
  uint64_t bytes;
};

constexpr uint32_t kComputeUnits = 256;

// The tile, and into how many parts the tokens are split, of the least estimated time: rounds of workgroups over the
// compute units, one on each, times the steps of a part; and the parts' sums, written and read once at 3.5 TB/s, with a launch of
// 3 us. Around the switches, times in us (tile, parts), * where the estimate leads:
//   1013 x 1000 x 1155    *64x128 1: 16  2: 23   128x128 1: 18  2: 21   256x256 1: 40
//   1013 x 2000 x 1155    64x128 1: 22   *128x128 1: 18  2: 34   256x256 1: 41
//   4096 x 1024 x 2048    *64x128 1: 46  2: 44   128x128 1: 51  2: 39   256x256 4: 53
//   4096 x 2048 x 2048    64x128 1: 66   *128x128 1: 52  2: 72   256x256 1: 115  4: 64
//   16384 x 1024 x 1024   128x128 1: 190  *4: 61   256x256 4: 124
//   4608 x 4096 x 4096    *256x256 1: 145   128x128 1: 297     fp32: 64x128 1: 578   *128x128 1: 669
//   16384 x 64 x 4096     32x128 4: 44  8: 47   64x128 4: 50  *8: 31   128x128 8: 33
//   4096 x 32 x 4096      32x128 4: 17  *8: 13   64x128 8: 14
//   512 x 1024 x 1024     *32x128 1: 9  2: 20   64x128 1: 9   128x128 1: 10
// The estimates are off by up to a sixth, and two workgroups of 64 x 128 fit a compute unit, which the rounds do not count: 4096 x
// 1024 x 2048 and the fp32 row go past the shortest time.
GradPlan plan_of(const sh_act8* k, uint32_t out, uint32_t dtype, bool bias) {
  const bool wide = dtype == SH_DTYPE_F32;
  const uint64_t sums = (uint64_t)out * k->cols + (bias ? out : 0);
  GradPlan best{};
  double best_cost = 0;
  for (int i = 0; i < sh::kGradTileCount; ++i) {
    const sh::GradTile& t = sh::kGradTiles[i];
    const uint32_t step = t.of[wide].step;
    if (step == 0) continue;
    const uint64_t tiles = ((uint64_t)out + t.out - 1) / t.out * (((uint64_t)k->cols + t.in - 1) / t.in);
    const uint32_t steps = std::max(1u, (k->tokens + step - 1) / step);
    for (uint32_t parts = 1; parts <= steps && (parts == 1 || tiles * parts <= 2 * kComputeUnits); parts += parts < 16 ? 1 : parts) {
      const uint32_t part_steps = (steps + parts - 1) / parts, splits = (steps + part_steps - 1) / part_steps;
      const double rounds = (double)((tiles * splits + kComputeUnits - 1) / kComputeUnits);
      const double join = splits > 1 ? 300 + (double)sums * 8 * splits / 35e3 : 0;
      const double cost = rounds * part_steps * t.of[wide].cost + join;
      if (best.tiles != 0 && cost >= best_cost) continue;
      best_cost = cost;
      best = {i, tiles, splits, part_steps * step, splits > 1 ? 4 * sums * splits : 0};
    }
  }
  return best;
}

}  // namespace

extern "C" int sh_act8_quantize(const void* x, uint32_t dtype, uint64_t x_ld, const sh_act8* kept, void* stream) {
  const char* who = "sh_act8_quantize";
  sh::clear_error();
  if (int st = check_kept(kept, who)) return st;
  if (int st = check_values(x, "x", dtype, kept->tokens, who)) return st;
  return launch_act8(kept, const_cast<void*>(x), x_ld, dtype, false, (hipStream_t)stream, who);
}

extern "C" int sh_act8_dequantize(const sh_act8* kept, void* out, uint32_t dtype, uint64_t out_ld, void* stream) {
  const char* who = "sh_act8_dequantize";
  sh::clear_error();
  if (int st = check_kept(kept, who)) return st;
  if (int st = check_values(out, "out", dtype, kept->tokens, who)) return st;
  if (int st = check_apart(out_ld, kept->tokens, kept->cols, "out_ld", who)) return st;
  return launch_act8(kept, out, out_ld, dtype, true, (hipStream_t)stream, who);
}

extern "C" int sh_weight_grad_act8_workspace(const sh_act8* kept, uint32_t dtype, uint32_t out_features, uint32_t bias, uint64_t* bytes) {
  const char* who = "sh_weight_grad_act8_workspace";
  sh::clear_error();
  if (bytes == nullptr) return sh::fail(SH_ERR_INVALID, "%s: bytes is NULL", who);
  if (int st = check_kept(kept, who)) return st;
  if (!known_dtype(dtype)) return sh::fail(SH_ERR_INVALID, "%s: unknown dtype %u", who, dtype);
  *bytes = plan_of(kept, out_features, dtype, bias != 0).bytes;
  return SH_OK;
}

extern "C" int sh_weight_grad_act8(const void* dy, uint32_t dtype, uint64_t dy_ld, uint32_t out_features, const sh_act8* kept,
                                   void* dweight, uint32_t out_dtype, uint64_t dw_ld, void* dbias, void* workspace,
                                   uint64_t workspace_bytes, void* stream) {
  const char* who = "sh_weight_grad_act8";
  sh::clear_error();
  if (int st = check_kept(kept, who)) return st;
  if (int st = check_values(dy, "dy", dtype, out_features == 0 ? 0 : kept->tokens, who)) return st;
  if (out_features > SH_WEIGHT_GRAD_MAX_OUT || dy_ld > SH_WEIGHT_GRAD_MAX_OUT)
    return sh::fail(SH_ERR_INVALID, "%s: out_features %u or dy_ld %llu is more than %u", who, out_features, (unsigned long long)dy_ld,
                    SH_WEIGHT_GRAD_MAX_OUT);
  // the kernels read up to a word past the end of a row that another one follows
  if (int st = check_apart(dy_ld, kept->tokens, out_features, "dy_ld", who)) return st;
  if (int st = check_values(dweight, "dweight", out_dtype, out_features, who)) return st;
  if (int st = check_apart(dw_ld, out_features, kept->cols, "dw_ld", who)) return st;
  if (misaligned(dbias, dtype_bytes(out_dtype))) return sh::fail(SH_ERR_INVALID, "%s: dbias is not aligned to its type", who);
  if (out_features == 0) return SH_OK;
  const GradPlan p = plan_of(kept, out_features, dtype, dbias != nullptr);
  if (workspace_bytes < p.bytes || (p.bytes > 0 && workspace == nullptr))
    return sh::fail(SH_ERR_INVALID, "%s: the workspace holds %llu bytes, %llu are needed", who,
                    (unsigned long long)workspace_bytes, (unsigned long long)p.bytes);
  if (misaligned(workspace, 16)) return sh::fail(SH_ERR_INVALID, "%s: workspace is not 16-byte aligned", who);
  const uint32_t threads = sh::kGradTiles[p.tile].of[dtype == SH_DTYPE_F32].threads;
  if (p.tiles * p.splits > 0xFFFFFFFFull / threads)
    return sh::fail(SH_ERR_INVALID, "%s: %u x %u gradients are too many for one launch", who, out_features, kept->cols);
  sh::WeightGradArgs a{};
  a.dy = dy;
  a.q = kept->q;
  a.exponent = kept->exponent;
  a.dweight = dweight;
  a.dbias = dbias;
  a.partials = p.splits > 1 ? static_cast<float*>(workspace) : nullptr;
  // rows past the last of a part lie behind its end only at a distance of a row's values, also where there is one row
  a.dy_ld = kept->tokens > 1 ? dy_ld : out_features;
  a.dw_ld = dw_ld;
  a.tokens = kept->tokens;
  a.out = out_features;
  a.cols = kept->cols;
  a.splits = p.splits;
  a.split_tokens = p.split_tokens;
  a.out_dtype = out_dtype;
  static_assert(sh::kKernWeightGradJoin - sh::kKernWeightGradBf1632x128 == 3 * sh::kGradTileCount - 1, "one kernel per type and tile");
  void* args[] = {(void*)&a};
  if (int st = sh::launch_kernel((sh::KernelId)(sh::kKernWeightGradBf1632x128 + (dtype - SH_DTYPE_BF16) * sh::kGradTileCount + p.tile),
                                 (uint32_t)(p.tiles * p.splits), threads, (hipStream_t)stream, args, who))
    return st;
  if (p.splits == 1) return SH_OK;
  const uint64_t values = (uint64_t)out_features * ((kept->cols + 3) / 4) + (dbias != nullptr ? out_features : 0);
  const uint64_t blocks = (values + sh::kGradJoinThreads - 1) / sh::kGradJoinThreads;
  return sh::launch_kernel(sh::kKernWeightGradJoin, (uint32_t)blocks, sh::kGradJoinThreads, (hipStream_t)stream, args, who);
}
