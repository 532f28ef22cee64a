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
  uint32_t threads;    // of a workgroup
};

// A row is held by a wavefront, kNormTeams of them in a workgroup, or by a workgroup of up to kNormMostWaves; `chunks` times
// 8 values a work-item.
struct NormShape {
  bool team;
  uint32_t chunks;
};
constexpr NormShape kNormShapes[] = {{false, 1}, {false, 2}, {true, 1}, {true, 2}, {true, 4}};
constexpr int kNormShapeCount = sizeof(kNormShapes) / sizeof(kNormShapes[0]);
constexpr uint32_t kNormTeams = 4, kNormMostWaves = 8;
constexpr uint32_t norm_capacity(NormShape s) { return (s.team ? kNormMostWaves : 1) * 64 * 8 * s.chunks; }
constexpr uint32_t norm_most_threads(bool team) { return 64 * (team ? kNormMostWaves : kNormTeams); }
static_assert(norm_capacity(kNormShapes[kNormShapeCount - 1]) == SH_LAYER_NORM_MAX_COLS, "the last shape holds the longest rows");

constexpr uint32_t kNormJoinThreads = 1024, kNormJoinCols = 32;

}  // namespace sh
