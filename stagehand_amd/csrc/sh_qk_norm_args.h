// Arguments of the query/key norm kernels, shared by the launches (sh_qk_norm.cpp) and the device
// code (sh_qk_norm.hip).
#pragma once

#include <cstdint>

#include "stagehand_native.h"

namespace sh {

struct QkNormKernelArgs {
  sh_qk_norm_rope_args a;
  float* partials;   // backward: one row of dim sums for each workgroup, or nullptr
  uint32_t q_grid;   // workgroups of the queries; the rest take the keys
  uint32_t k_grid;
  uint32_t lanes;    // work-items that share a head, a power of two
};

constexpr uint32_t kQkThreads = 256;
constexpr uint32_t kQkSlots = 8;  // pairs of values that a work-item holds

}  // namespace sh
