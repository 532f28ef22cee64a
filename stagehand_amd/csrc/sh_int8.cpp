// Linear layers on SquareQ weights that stay in int8 (no reference counterpart: the reference
// dequantises them, src/stagehand/scheduler.py:285-308, and multiplies in bf16).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "sh_int8_args.h"
#include "sh_internal.h"
#include "stagehand_native.h"

namespace {

using sh::dtype_bytes;
using sh::known_dtype;
using sh::misaligned;

uint64_t token_ld(uint32_t cols) {
  return ((uint64_t)cols + SH_I8_TOKEN_ALIGN - 1) / SH_I8_TOKEN_ALIGN * SH_I8_TOKEN_ALIGN;
}

int check_weight(const sh_i8_weight* w, const char* who) {
  if (w == nullptr) return sh::fail(SH_ERR_INVALID, "%s: w is NULL", who);
  if (w->cols == 0 || w->cols > SH_I8_MAX_COLS)
    return sh::fail(SH_ERR_INVALID, "%s: cols %u is not in 1 .. %u", who, w->cols, SH_I8_MAX_COLS);
  if (w->ld % 16 != 0 || w->ld < w->cols || w->ld > (1u << 20))
    return sh::fail(SH_ERR_INVALID, "%s: ld %llu of the weight is not a multiple of 16 in %u .. %u", who,
                    (unsigned long long)w->ld, w->cols, 1u << 20);
  if (w->rows > 0 && (w->q == nullptr || w->scale == nullptr))
    return sh::fail(SH_ERR_INVALID, "%s: the weight's q or scale is NULL", who);
  if (misaligned(w->q, 16)) return sh::fail(SH_ERR_INVALID, "%s: the weight's q is not 16-byte aligned", who);
  if (misaligned(w->scale, 4) || misaligned(w->zero_point, 4) || misaligned(w->bias, 4))
    return sh::fail(SH_ERR_INVALID, "%s: the weight's scale, zero_point or bias is not 4-byte aligned", who);
  return SH_OK;
}

int check_x(const void* x, uint32_t dtype, uint64_t x_ld, uint32_t tokens, uint32_t cols, const char* who) {
  if (!known_dtype(dtype)) return sh::fail(SH_ERR_INVALID, "%s: unknown dtype %u", who, dtype);
  if (cols == 0 || cols > SH_I8_MAX_COLS)
    return sh::fail(SH_ERR_INVALID, "%s: cols %u is not in 1 .. %u", who, cols, SH_I8_MAX_COLS);
  if (tokens == 0) return SH_OK;
  if (x == nullptr) return sh::fail(SH_ERR_INVALID, "%s: x is NULL", who);
  if (misaligned(x, dtype_bytes(dtype))) return sh::fail(SH_ERR_INVALID, "%s: x is not aligned to its type", who);
  (void)x_ld;  // any stride: rows of x may overlap, they are only read
  return SH_OK;
}

int check_out(const void* out, uint32_t dtype, uint64_t out_ld, uint32_t tokens, uint32_t rows, const char* who) {
  if (!known_dtype(dtype)) return sh::fail(SH_ERR_INVALID, "%s: unknown out dtype %u", who, dtype);
  if (tokens == 0 || rows == 0) return SH_OK;
  if (out == nullptr) return sh::fail(SH_ERR_INVALID, "%s: out is NULL", who);
  if (misaligned(out, dtype_bytes(dtype))) return sh::fail(SH_ERR_INVALID, "%s: out is not aligned to its type", who);
  if (tokens > 1 && out_ld < rows)
    return sh::fail(SH_ERR_INVALID, "%s: out_ld %llu is less than the weight's %u rows", who,
                    (unsigned long long)out_ld, rows);
  return SH_OK;
}

int check_tokens(const void* q, uint64_t q_ld, const float* scale, const int32_t* sums, uint32_t tokens, uint32_t cols,
                 const char* who) {
  if (q_ld % SH_I8_TOKEN_ALIGN != 0 || q_ld < cols || q_ld > (1u << 20))
    return sh::fail(SH_ERR_INVALID, "%s: q_ld %llu is not a multiple of %u in %u .. %u", who, (unsigned long long)q_ld,
                    SH_I8_TOKEN_ALIGN, cols, 1u << 20);
  if (tokens > 0 && (q == nullptr || scale == nullptr)) return sh::fail(SH_ERR_INVALID, "%s: q or scale is NULL", who);
  if (misaligned(q, 16)) return sh::fail(SH_ERR_INVALID, "%s: q is not 16-byte aligned", who);
  if (misaligned(scale, 4) || misaligned(sums, 4))
    return sh::fail(SH_ERR_INVALID, "%s: scale or sums is not 4-byte aligned", who);
  return SH_OK;
}

int launch_quantize(const sh::QuantizeArgs& a, hipStream_t stream, const char* who) {
  static_assert(sh::kKernQuantizeF16512 == sh::kKernQuantizeBf16512 + 4 &&
                    sh::kKernQuantizeF32512 == sh::kKernQuantizeBf16512 + 8,
                "four kernels for each type, in the order of enum sh_dtype");
  const uint32_t width = a.cols <= 512 ? 0 : a.cols <= 2048 ? 1 : a.cols <= 4096 ? 2 : 3;
  const uint32_t grid = width < 3 ? (a.tokens + 3) / 4 : a.tokens;
  void* args[] = {(void*)&a};
  return sh::launch_kernel((sh::KernelId)(sh::kKernQuantizeBf16512 + (a.dtype - SH_DTYPE_BF16) * 4 + width), grid, 256,
                           stream, args, who);
}

// The tile of the least estimated time: rounds of tiles over the 256 compute units, times what 128 columns of
// one round take (MI355X, measured over 64 to 1500 tiles of 3072 and 4096 columns). The number of columns has no
// part in it: what a tile's start and its stores take is not in the cost, and products of a few hundred columns,
// where that counts, were not measured tile by tile (9953 x 949 x 590 takes 20 us, its bytes and operations 5).
// Larger tiles read LDS and the caches less for each product (8192^3: 256 x 256 415 us, 128 x 256 475, 128 x 128
// 580, 64 x 64 880), smaller ones leave fewer compute units idle. Around the switches, times in us:
//   64 x 4096 x 4096     32x32 8.6   64x64 11          1024 x 4096 x 4096   128x128 20   128x256 25   256x256 42
//   128 x 9216 x 3072    64x64 13.4  32x32 21          2048 x 4096 x 4096   128x256 33   128x128 37   256x256 44
//   256 x 9216 x 3072    128x128 16  64x64 18          1024 x 12288 x 3072  256x256 41   128x256 45
//   512 x 9216 x 3072    128x256 22  128x128 28        4608 x 3072 x 3072   256x256 40   128x256 44
int choose_tile(uint32_t tokens, uint32_t rows) {
  int best = 0;
  double best_cost = 0;
  for (int i = 0; i < sh::kMatmulTileCount; ++i) {
    const sh::MatmulTile& m = sh::kMatmulTiles[i];
    const double tiles = (double)((tokens + (uint64_t)m.tokens - 1) / m.tokens) * ((rows + (uint64_t)m.rows - 1) / m.rows);
    const double rounds = m.fractional ? std::max(1.0, tiles / 256) : std::ceil(tiles / 256);
    const double cost = rounds * m.cost;
    if (i == 0 || cost < best_cost) best = i, best_cost = cost;
  }
  return best;
}

int launch_matmul(const sh::MatmulI8Args& a, hipStream_t stream, const char* who) {
  const int i = choose_tile(a.tokens, a.rows);
  const sh::MatmulTile& m = sh::kMatmulTiles[i];
  const uint64_t grid = ((uint64_t)a.tokens + m.tokens - 1) / m.tokens * (((uint64_t)a.rows + m.rows - 1) / m.rows);
  if (grid > 0xFFFFFFFFull / m.threads)
    return sh::fail(SH_ERR_INVALID, "%s: %u tokens x %u rows are too many for one launch", who, a.tokens, a.rows);
  void* args[] = {(void*)&a};
  static_assert(sh::kKernMatmulI8256x256 - sh::kKernMatmulI816x16 == sh::kMatmulTileCount - 1, "one kernel per tile");
  return sh::launch_kernel((sh::KernelId)(sh::kKernMatmulI816x16 + i), (uint32_t)grid, m.threads, stream, args, who);
}

// Whether the tokens are few enough for every workgroup to quantise them for itself: one launch less, about 4
// us of a call, for work that is done once by each of the weight's rows / 16 or rows / 32 workgroups. Measured
// (one launch against two): 1 x 4096 x 4096 7.5 and 11 us, 1 x 18432 x 3072 12.4 and 16, 4 x 18432 x 3072 14.2
// and 15.9, 8 x 4096 x 3072 7.4 and 11.3; past the limits 8 x 18432 x 3072 24 and 16.
bool in_one_launch(uint32_t tokens, const sh_i8_weight* w) {
  const uint64_t pieces = (uint64_t)tokens * ((w->cols + 511) / 512);
  return tokens <= 16 && pieces <= (w->rows > sh::kNarrowRows ? sh::kFewPiecesWide : sh::kFewPiecesNarrow);
}

struct Workspace {
  uint64_t q_ld, sums, scale, bytes;
};

// q, then the scales, then the sums.
Workspace workspace_of(uint32_t tokens, const sh_i8_weight* w) {
  Workspace s{};
  if (in_one_launch(tokens, w)) return s;
  s.q_ld = token_ld(w->cols);
  s.scale = s.q_ld * tokens;
  s.sums = s.scale + 4ull * tokens;
  s.bytes = s.sums + 4ull * tokens;
  return s;
}

}  // namespace

extern "C" int sh_quantize_tokens(const void* x, uint32_t dtype, uint64_t x_ld, uint32_t tokens, uint32_t cols, void* q,
                                  uint64_t q_ld, float* scale, int32_t* sums, void* stream) {
  const char* who = "sh_quantize_tokens";
  sh::clear_error();
  if (int st = check_x(x, dtype, x_ld, tokens, cols, who)) return st;
  if (int st = check_tokens(q, q_ld, scale, sums, tokens, cols, who)) return st;
  if (tokens == 0) return SH_OK;
  if (tokens > 0xFFFFFFFFu / 256)
    return sh::fail(SH_ERR_INVALID, "%s: %u tokens are too many for one launch", who, tokens);
  const sh::QuantizeArgs a{x, q, scale, sums, x_ld, q_ld, tokens, cols, dtype};
  return launch_quantize(a, (hipStream_t)stream, who);
}

extern "C" int sh_matmul_i8(const void* q, uint64_t q_ld, const float* scale, const int32_t* sums, uint32_t tokens,
                            const sh_i8_weight* w, void* out, uint32_t out_dtype, uint64_t out_ld, void* stream) {
  const char* who = "sh_matmul_i8";
  sh::clear_error();
  if (int st = check_weight(w, who)) return st;
  if (int st = check_tokens(q, q_ld, scale, sums, tokens, w->cols, who)) return st;
  if (int st = check_out(out, out_dtype, out_ld, tokens, w->rows, who)) return st;
  if (tokens == 0 || w->rows == 0) return SH_OK;
  if (w->zero_point != nullptr && sums == nullptr)
    return sh::fail(SH_ERR_INVALID, "%s: sums is NULL, but the weight has zero points", who);
  const sh::MatmulI8Args a{q,   scale, sums, w->q,   w->scale, w->zero_point, w->bias, out,
                           q_ld, w->ld, out_ld, tokens, w->rows, w->cols,       out_dtype};
  return launch_matmul(a, (hipStream_t)stream, who);
}

extern "C" int sh_linear_i8_workspace(uint32_t tokens, const sh_i8_weight* w, uint64_t* bytes) {
  sh::clear_error();
  if (bytes == nullptr) return sh::fail(SH_ERR_INVALID, "sh_linear_i8_workspace: bytes is NULL");
  if (int st = check_weight(w, "sh_linear_i8_workspace")) return st;
  *bytes = workspace_of(tokens, w).bytes;
  return SH_OK;
}

extern "C" int sh_linear_i8(const void* x, uint32_t dtype, uint64_t x_ld, uint32_t tokens, const sh_i8_weight* w,
                            void* out, uint64_t out_ld, void* workspace, uint64_t workspace_bytes, void* stream) {
  const char* who = "sh_linear_i8";
  sh::clear_error();
  if (int st = check_weight(w, who)) return st;
  if (int st = check_x(x, dtype, x_ld, tokens, w->cols, who)) return st;
  if (int st = check_out(out, dtype, out_ld, tokens, w->rows, who)) return st;
  if (tokens == 0 || w->rows == 0) return SH_OK;
  const Workspace s = workspace_of(tokens, w);
  if (workspace_bytes < s.bytes || (s.bytes > 0 && workspace == nullptr))
    return sh::fail(SH_ERR_INVALID, "%s: the workspace holds %llu bytes, %llu are needed", who,
                    (unsigned long long)workspace_bytes, (unsigned long long)s.bytes);
  if (misaligned(workspace, 16)) return sh::fail(SH_ERR_INVALID, "%s: workspace is not 16-byte aligned", who);
  if (in_one_launch(tokens, w)) {
    const bool wide = w->rows > sh::kNarrowRows;
    const uint32_t grid = wide ? (w->rows + 31) / 32 : (w->rows + 15) / 16;
    if (grid > 0xFFFFFFFFu / 512) return sh::fail(SH_ERR_INVALID, "%s: %u rows are too many for one launch", who, w->rows);
    const sh::MatmulI8Args a{x,    nullptr, nullptr, w->q,   w->scale, w->zero_point, w->bias, out,
                             x_ld, w->ld,   out_ld,  tokens, w->rows,  w->cols,       dtype};
    void* args[] = {(void*)&a};
    static_assert(sh::kKernLinearI8F1616x16 == sh::kKernLinearI8Bf1616x16 + 2 &&
                      sh::kKernLinearI8F3216x16 == sh::kKernLinearI8Bf1616x16 + 4,
                  "two kernels for each type, in the order of enum sh_dtype");
    return sh::launch_kernel((sh::KernelId)(sh::kKernLinearI8Bf1616x16 + (dtype - SH_DTYPE_BF16) * 2 + wide), grid,
                             wide ? 256 : 512, (hipStream_t)stream, args, who);
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  float* scale = reinterpret_cast<float*>(ws + s.scale);
  int32_t* sums = reinterpret_cast<int32_t*>(ws + s.sums);
  if (int st = sh_quantize_tokens(x, dtype, x_ld, tokens, w->cols, ws, s.q_ld, scale, sums, stream)) return st;
  return sh_matmul_i8(ws, s.q_ld, scale, sums, tokens, w, out, dtype, out_ld, stream);
}
