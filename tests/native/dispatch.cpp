// Which kernels the operators' C entry points launch: the host sources that choose them (sh_int8.cpp,
// sh_qk_norm.cpp), linked with a launch that prints the kernel's id instead (tests/test_operator_dispatch.py
// builds and runs it). Reads one call a line:
//   quantize TOKENS COLS DTYPE
//   linear TOKENS ROWS COLS DTYPE
//   norm BATCH Q_HEADS K_HEADS SEQ DIM ROT DTYPE INTERLEAVED BACKWARD
// and prints a line of ids, relative to the first operator's kernel, for each.

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <iostream>
#include <sstream>
#include <string>

#include "sh_internal.h"
#include "stagehand_native.h"

namespace sh {

void clear_error() {}
int fail(int status, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  std::vfprintf(stderr, fmt, ap);
  va_end(ap);
  std::fputc('\n', stderr);
  return status;
}
int launch_kernel(KernelId id, uint32_t grid, uint32_t block, hipStream_t, void**, const char* who) {
  if (grid == 0 || (uint64_t)grid * block > 0xFFFFFFFFull) return fail(SH_ERR_INVALID, "%s: grid %u of %u", who, grid, block);
  std::printf("%d ", id - kKernQuantizeBf16512);
  return SH_OK;
}

}  // namespace sh

int main() {
  void* const p = reinterpret_cast<void*>(uintptr_t{1} << 20);  // aligned, never read
  float* const f = static_cast<float*>(p);
  std::string line, what;
  while (std::getline(std::cin, line)) {
    std::istringstream in(line);
    in >> what;
    int st = SH_ERR_INVALID;
    if (what == "quantize") {
      uint32_t tokens, cols, dtype;
      in >> tokens >> cols >> dtype;
      st = sh_quantize_tokens(p, dtype, cols, tokens, cols, p, (cols + 127ull) / 128 * 128, f, static_cast<int32_t*>(p), nullptr);
    } else if (what == "linear") {
      uint32_t tokens, dtype;
      sh_i8_weight w{};
      in >> tokens >> w.rows >> w.cols >> dtype;
      w.q = p;
      w.ld = (w.cols + 127ull) / 128 * 128;
      w.scale = f;
      uint64_t need = 0;
      st = sh_linear_i8_workspace(tokens, &w, &need);
      if (st == SH_OK) st = sh_linear_i8(p, dtype, w.cols, tokens, &w, p, w.rows, p, need, nullptr);
    } else if (what == "norm") {
      sh_qk_norm_rope_args a{};
      bool backward;
      in >> a.batch >> a.q_heads >> a.k_heads >> a.seq >> a.dim >> a.rot >> a.dtype >> a.interleaved >> backward;
      for (sh_heads* h : {&a.q, &a.k, &a.q_out, &a.k_out, &a.dq, &a.dk}) h->data = p;
      a.cos = a.sin = f;
      a.table_ld = a.rot / 2;
      a.table_rows = a.seq;
      a.weight_dtype = a.dtype;
      a.eps = 1e-6f;
      if (backward) {
        a.dq_weight = a.dk_weight = p;
        uint64_t need = 0;
        st = sh_qk_norm_rope_workspace(&a, &need);
        if (st == SH_OK) st = sh_qk_norm_rope_backward(&a, p, need, nullptr);
      } else {
        st = sh_qk_norm_rope(&a, nullptr);
      }
    }
    if (!in || st != SH_OK) {
      std::fprintf(stderr, "status %d for: %s\n", st, line.c_str());
      return 1;
    }
    std::printf("\n");
  }
  return 0;
}
