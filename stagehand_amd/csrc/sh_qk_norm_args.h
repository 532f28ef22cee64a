// Arguments of the query/key norm kernels, shared by the launches (sh_qk_norm.cpp) and the device
// code (sh_qk_norm.hip).
#pragma once

#include <cstdint>

#include "stagehand_native.h"

namespace sh {

// The queries' or the keys' share of a launch.
struct QkNormPart {
  uint64_t units;     // of a wavefront: a segment of the heads of 64 / lanes / abreast tokens
  uint32_t grid;      // workgroups
  uint32_t abreast;   // heads of a token side by side, a power of two
  uint32_t segments;  // parts of a token's heads, each taken by a wavefront of its own
};

struct QkNormKernelArgs {
  sh_qk_norm_rope_args a;
  float* partials;     // backward: a row of dim sums for each workgroup, or nullptr
  QkNormPart part[2];  // queries, keys
  uint32_t lanes;      // work-items that share a head, a power of two
};

constexpr uint32_t kQkThreads = 256;
constexpr uint32_t kQkSlots = 8;  // pairs of values that a work-item holds

}  // namespace sh
