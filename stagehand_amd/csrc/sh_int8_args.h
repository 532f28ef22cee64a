// Arguments of the int8 kernels, shared by the launches (sh_int8.cpp) and the device code
// (sh_int8.hip).
#pragma once

#include <cstdint>

namespace sh {

struct QuantizeArgs {
  const void* x;
  void* q;
  float* scale;
  int32_t* sums;  // nullptr: not wanted
  uint64_t x_ld;  // elements
  uint64_t q_ld;  // bytes
  uint32_t tokens;
  uint32_t cols;
  uint32_t dtype;
};

struct MatmulI8Args {
  const void* tq;  // quantised tokens
  const float* t_scale;
  const int32_t* t_sums;
  const void* wq;
  const float* w_scale;
  const float* w_zp;
  const float* bias;
  void* out;
  uint64_t t_ld;    // bytes
  uint64_t w_ld;    // bytes
  uint64_t out_ld;  // elements
  uint32_t tokens;
  uint32_t rows;
  uint32_t cols;
  uint32_t out_dtype;
};

}  // namespace sh
