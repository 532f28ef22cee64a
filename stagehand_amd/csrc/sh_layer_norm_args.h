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
  uint32_t lanes;      // work-items that share a row: the workgroup's, or a power of two of them from 4 to 64
};

// A row is held by up to 64 work-items of a workgroup of kNormThreads, or by a `team`: a workgroup of up to kNormMostWaves
// wavefronts; `chunks` times 8 values a work-item.
struct NormShape {
  bool team;
  uint32_t chunks;
};
constexpr NormShape kNormShapes[] = {{false, 1}, {false, 2}, {true, 2}, {true, 4}};
constexpr int kNormShapeCount = sizeof(kNormShapes) / sizeof(kNormShapes[0]);
constexpr uint32_t kNormThreads = 256, kNormMostWaves = 8;
constexpr uint32_t norm_capacity(NormShape s) { return (s.team ? kNormMostWaves : 1) * 64 * 8 * s.chunks; }
constexpr uint32_t norm_most_threads(bool team) { return team ? 64 * kNormMostWaves : kNormThreads; }
static_assert(norm_capacity(kNormShapes[kNormShapeCount - 1]) == SH_LAYER_NORM_MAX_COLS, "the last shape holds the longest rows");

constexpr uint32_t kNormJoinThreads = 1024, kNormJoinCols = 32;

}  // namespace sh
