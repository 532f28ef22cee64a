// Arguments of the kernels of activations kept in 8 bits, shared by the launches (sh_act8.cpp) and the device
// code (sh_act8.hip, sh_weight_grad.hip).
#pragma once

#include <cstdint>

namespace sh {

// Rows of groups of SH_ACT8_GROUP values, and one exponent byte a group.
struct Act8Args {
  void* x;  // read by the quantisation, written by the other way
  void* q;
  void* exponent;
  uint64_t x_ld;    // elements
  uint64_t magic;   // of a division by the chunks of a row
  uint32_t chunks;  // of 8 values, in all rows; a row has whole groups of them
  uint32_t row_chunks;
  uint32_t tokens, cols;
};

constexpr uint32_t kAct8Threads = 256;

struct WeightGradArgs {
  const void* dy;
  const void* q;
  const void* exponent;
  void* dweight;
  void* dbias;  // nullptr: not wanted
  // With splits > 1: sums of each split, dweight's then dbias', and the kernel that joins them writes dweight and dbias.
  float* partials;
  uint64_t dy_ld, dw_ld;  // elements
  uint32_t tokens, out, cols;
  uint32_t splits;        // parts of the tokens, each summed by workgroups of its own
  uint32_t split_tokens;  // tokens of a part, a multiple of the tile's step
  uint32_t out_dtype;
};

// Tiles of outputs x inputs of dweight. For gradients of 16 and of 32 bits: the work-items, the tokens that are staged at a
// time (0: there is no such kernel), and how long that takes, in 10 ns (MI355X).
struct GradTile {
  uint32_t out, in;
  struct {
    uint32_t threads, step, cost;
  } of[2];
};
constexpr GradTile kGradTiles[] = {
    {32, 128, {{256, 128, 120}, {256, 64, 100}}},
    {64, 128, {{512, 64, 60}, {256, 32, 70}}},
    {128, 128, {{512, 64, 85}, {256, 32, 118}}},
    {256, 256, {{512, 32, 93}, {0, 0, 0}}},
};
constexpr int kGradTileCount = sizeof(kGradTiles) / sizeof(kGradTiles[0]);
constexpr uint32_t kGradJoinThreads = 256;

}  // namespace sh
