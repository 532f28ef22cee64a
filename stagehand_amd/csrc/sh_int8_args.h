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

// Pieces of 512 values that one launch quantises and multiplies (at most 16 tokens), for weights of up to
// kNarrowRows rows, which 16 rows a workgroup spread over the whole chip, and for wider ones, with 32 rows a
// workgroup and more than one workgroup on a compute unit.
constexpr uint32_t kNarrowRows = 32 * 255;
constexpr uint32_t kFewPiecesNarrow = 64, kFewPiecesWide = 32;

// The product's kernels, smallest tile first.
struct MatmulTile {
  uint32_t tokens, rows, threads;
  uint32_t cost;    // of 128 columns on a full chip, in 10 ns
  bool fractional;  // several workgroups share a compute unit: a last round that is not full costs its share
};
constexpr MatmulTile kMatmulTiles[] = {
    {16, 16, 512, 11, true},    {16, 32, 256, 15, true},     {32, 32, 256, 19, true},     {64, 64, 256, 30, true},
    {128, 128, 512, 62, false}, {128, 256, 1024, 100, false}, {256, 256, 512, 175, false},
};
constexpr int kMatmulTileCount = sizeof(kMatmulTiles) / sizeof(kMatmulTiles[0]);

}  // namespace sh
