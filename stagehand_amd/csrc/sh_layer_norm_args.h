// Arguments of the layer norm kernels, shared by the launches (sh_layer_norm.cpp) and the device code
// (sh_layer_norm.hip).
#pragma once

#include <cstdint>

#include "stagehand_native.h"

namespace sh {

struct LayerNormKernelArgs {
  sh_layer_norm_args a;
  float* partials;    // backward: sums of each workgroup, cols of dweight's, then cols of dbias'; nullptr: not wanted
  uint32_t groups;    // of tokens that share weight and bias
  uint32_t tokens;    // of a group
  uint32_t per_group;  // workgroups
};

// Rows are held by teams of wavefronts, 8 values a work-item and chunk.
struct NormShape {
  uint32_t waves, chunks;
};
constexpr NormShape kNormShapes[] = {{1, 1}, {1, 2}, {4, 1}, {4, 2}, {8, 2}, {16, 2}};
constexpr int kNormShapeCount = sizeof(kNormShapes) / sizeof(kNormShapes[0]);
constexpr uint32_t norm_capacity(NormShape s) { return s.waves * 64 * 8 * s.chunks; }
constexpr uint32_t norm_teams(uint32_t waves) { return waves == 1 ? 4 : 1; }  // of a workgroup
constexpr uint32_t norm_threads(uint32_t waves) { return waves * norm_teams(waves) * 64; }
static_assert(norm_capacity(kNormShapes[kNormShapeCount - 1]) == SH_LAYER_NORM_MAX_COLS, "the last shape holds the longest rows");

constexpr uint32_t kNormJoinThreads = 1024, kNormJoinCols = 32;

}  // namespace sh
