// Which kernels the training operators' C entry points launch: the host sources that choose them (sh_layer_norm.cpp,
// sh_act8.cpp), linked with a launch that prints the kernel's id instead (tests/test_training_dispatch.py builds and
// runs it). Reads one call a line:
//   norm BATCH SEQ COLS DTYPE PER_BATCH PASS        (0 forward, 1 backward, 2 backward from what was kept)
//   keep TOKENS COLS DTYPE BACK
//   grad TOKENS OUT COLS DTYPE BIAS
// and prints a line of ids, relative to the first of these operators' kernels, for each.

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
  if (grid == 0 || block == 0 || block > 1024 || (uint64_t)grid * block > 0xFFFFFFFFull)
    return fail(SH_ERR_INVALID, "%s: grid %u of %u", who, grid, block);
  std::printf("%d ", id - kKernLayerNormBf16Wave1);
  return SH_OK;
}

}  // namespace sh

int main() {
  void* const p = reinterpret_cast<void*>(uintptr_t{1} << 20);  // aligned, never read
  std::string line, what;
  while (std::getline(std::cin, line)) {
    std::istringstream in(line);
    in >> what;
    int st = SH_ERR_INVALID;
    uint64_t need = 0;
    if (what == "norm") {
      sh_layer_norm_args a{};
      int pass;
      in >> a.batch >> a.seq >> a.cols >> a.dtype >> a.per_batch >> pass;
      a.weight_dtype = a.dtype;
      a.eps = 1e-6f;
      a.x.data = a.y.data = a.dy.data = a.dx.data = p;
      a.stats = static_cast<float*>(p);
      if (pass == 2) a.q = a.exponent = p;
      if (pass == 0) {
        st = sh_layer_norm(&a, nullptr);
      } else {
        a.dweight = a.dbias = p;
        st = sh_layer_norm_workspace(&a, &need);
        if (st == SH_OK) st = sh_layer_norm_backward(&a, p, need, nullptr);
      }
    } else {
      sh_act8 k{p, p, 0, 0};
      uint32_t dtype;
      if (what == "keep") {
        bool back;
        in >> k.tokens >> k.cols >> dtype >> back;
        st = back ? sh_act8_dequantize(&k, p, dtype, k.cols, nullptr) : sh_act8_quantize(p, dtype, k.cols, &k, nullptr);
      } else if (what == "grad") {
        uint32_t out;
        bool bias;
        in >> k.tokens >> out >> k.cols >> dtype >> bias;
        st = sh_weight_grad_act8_workspace(&k, dtype, out, bias, &need);
        if (st == SH_OK) st = sh_weight_grad_act8(p, dtype, out, out, &k, p, dtype, k.cols, bias ? p : nullptr, p, need, nullptr);
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
