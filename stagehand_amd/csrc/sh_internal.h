// Internal helpers shared by the native sources: error reporting and the
// division-by-invariant used to map a flat element index to its row.
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <functional>
#include <string>
#include <vector>

#include "stagehand_native.h"

namespace sh {

// Records the failure text for sh_last_error() on the calling thread and
// returns `status` so call sites can `return fail(...)`.
int fail(int status, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
void clear_error();

// HIP call wrapper: converts a hipError_t into SH_ERR_HIP with the call text.
#define SH_HIP(call)                                                              \
  do {                                                                            \
    hipError_t sh_e_ = (call);                                                    \
    if (sh_e_ != hipSuccess)                                                      \
      return ::sh::fail(SH_ERR_HIP, "HIP error %d (%s) in %s", (int)sh_e_,       \
                        hipGetErrorString(sh_e_), #call);                         \
  } while (0)

// Of the operators' arguments: enum sh_dtype, and an address that is not a multiple of n (a power of two).
inline bool known_dtype(uint32_t d) { return d == SH_DTYPE_BF16 || d == SH_DTYPE_F16 || d == SH_DTYPE_F32; }
inline uint32_t dtype_bytes(uint32_t d) { return d == SH_DTYPE_F32 ? 4 : 2; }
inline bool misaligned(const void* p, uint32_t n) { return ((uintptr_t)p & (n - 1)) != 0; }

// Live native objects by kind, for sh_shutdown's report. Each object struct holds a
// Live<kind> member, so construction and destruction keep the count.
enum LiveKind : int { kLivePool = 0, kLiveLoader, kLiveSaveback, kLiveTurbo, kLiveVmm, kLiveFile, kLiveKinds };
extern std::atomic<int64_t> g_live[kLiveKinds];
template <int K>
struct Live {
  Live() { g_live[K].fetch_add(1, std::memory_order_relaxed); }
  ~Live() { g_live[K].fetch_sub(1, std::memory_order_relaxed); }
  Live(const Live&) = delete;
  Live& operator=(const Live&) = delete;
};

// Names the calling thread (at most 15 characters shown): every thread the library starts
// is called "sh-<role>", so a process can tell them from the runtime's own threads.
void name_thread(const char* name);

// Runs fn(i) for every i in [0, n) on up to `threads` of the shared host copy
// threads (the calling thread included); returns when all calls are done.
void parallel_for(size_t n, unsigned threads, const std::function<void(size_t)>& fn);

// One unit of host staging work: a memcpy (file == nullptr) or a read of
// `bytes` at `file_off` of `file` into dst.
struct IoPiece {
  uint8_t* dst;
  const uint8_t* src;
  sh_file* file;
  uint64_t file_off;
  uint64_t bytes;
};
// Appends a memcpy cut into pieces of at most 8 MiB.
void append_copy(std::vector<IoPiece>& out, void* dst, const void* src, uint64_t bytes);
// Appends a file read cut at 8 MiB file offsets (pieces stay aligned for O_DIRECT).
void append_read(std::vector<IoPiece>& out, sh_file* f, uint64_t file_off, uint64_t bytes, void* dst);
// Checks that [file_off, file_off + bytes) lies inside the file (SH_ERR_INVALID otherwise).
int check_range(const sh_file* f, uint64_t file_off, uint64_t bytes, const char* who);
// Executes the pieces on up to `threads` copy threads; SH_ERR_IO (with the
// failing file, offset and errno in the last error) when a read fails.
int run_io(const std::vector<IoPiece>& pieces, int threads);
// The buffered descriptor of a file that has no O_DIRECT descriptor, else -1:
// the descriptor on which read-ahead advice is worth giving.
int advice_fd(const sh_file* f);

// The library's kernels (sh_kernels.cpp): loaded per device from the embedded code objects on
// first use, unloaded by sh_shutdown.
enum KernelId : int {
  kKernDequantBf16 = 0,
  kKernDequantBf16Zp,
  kKernCastBf16,
  kKernMixed,
  kKernMixedZp,
  kKernMixedPaced,
  kKernMixedPacedZp,
  kKernUnpackArgs,
  kKernUnpackArgsZp,
  kKernPutDescs,
  kKernFillTileMap,
  kKernDigest,
  kKernDigestWide,
  kKernDigestCompare,
  kKernDigestCompareWide,
  // int8: one quantisation per type and columns held in registers, in this order
  kKernQuantizeBf16512,
  kKernQuantizeBf162048,
  kKernQuantizeBf164096,
  kKernQuantizeBf1616384,
  kKernQuantizeF16512,
  kKernQuantizeF162048,
  kKernQuantizeF164096,
  kKernQuantizeF1616384,
  kKernQuantizeF32512,
  kKernQuantizeF322048,
  kKernQuantizeF324096,
  kKernQuantizeF3216384,
  // one product per tile of sh_int8_args.h, in this order
  kKernMatmulI816x16,
  kKernMatmulI816x32,
  kKernMatmulI832x32,
  kKernMatmulI864x64,
  kKernMatmulI8128x128,
  kKernMatmulI8128x256,
  kKernMatmulI8256x256,
  // quantisation and product in one, per type and tile
  kKernLinearI8Bf1616x16,
  kKernLinearI8Bf1616x32,
  kKernLinearI8F1616x16,
  kKernLinearI8F1616x32,
  kKernLinearI8F3216x16,
  kKernLinearI8F3216x32,
  // query/key norms: per type and run of pairs, forward and backward, halves and interleaved
  kKernQkNormBf168,
  kKernQkNormBf168Interleaved,
  kKernQkNormBackwardBf168,
  kKernQkNormBackwardBf168Interleaved,
  kKernQkNormBf164,
  kKernQkNormBf164Interleaved,
  kKernQkNormBackwardBf164,
  kKernQkNormBackwardBf164Interleaved,
  kKernQkNormBf162,
  kKernQkNormBf162Interleaved,
  kKernQkNormBackwardBf162,
  kKernQkNormBackwardBf162Interleaved,
  kKernQkNormBf161,
  kKernQkNormBf161Interleaved,
  kKernQkNormBackwardBf161,
  kKernQkNormBackwardBf161Interleaved,
  kKernQkNormF168,
  kKernQkNormF168Interleaved,
  kKernQkNormBackwardF168,
  kKernQkNormBackwardF168Interleaved,
  kKernQkNormF164,
  kKernQkNormF164Interleaved,
  kKernQkNormBackwardF164,
  kKernQkNormBackwardF164Interleaved,
  kKernQkNormF162,
  kKernQkNormF162Interleaved,
  kKernQkNormBackwardF162,
  kKernQkNormBackwardF162Interleaved,
  kKernQkNormF161,
  kKernQkNormF161Interleaved,
  kKernQkNormBackwardF161,
  kKernQkNormBackwardF161Interleaved,
  kKernQkNormF328,
  kKernQkNormF328Interleaved,
  kKernQkNormBackwardF328,
  kKernQkNormBackwardF328Interleaved,
  kKernQkNormF324,
  kKernQkNormF324Interleaved,
  kKernQkNormBackwardF324,
  kKernQkNormBackwardF324Interleaved,
  kKernQkNormF322,
  kKernQkNormF322Interleaved,
  kKernQkNormBackwardF322,
  kKernQkNormBackwardF322Interleaved,
  kKernQkNormF321,
  kKernQkNormF321Interleaved,
  kKernQkNormBackwardF321,
  kKernQkNormBackwardF321Interleaved,
  kKernQkNormDweight,
  // layer norms: per type and shape of sh_layer_norm_args.h: forward, backward, backward from what was kept
  kKernLayerNormBf16Wave1,
  kKernLayerNormBackwardBf16Wave1,
  kKernLayerNormBackwardKeptBf16Wave1,
  kKernLayerNormBf16Wave2,
  kKernLayerNormBackwardBf16Wave2,
  kKernLayerNormBackwardKeptBf16Wave2,
  kKernLayerNormBf16Team2,
  kKernLayerNormBackwardBf16Team2,
  kKernLayerNormBackwardKeptBf16Team2,
  kKernLayerNormBf16Team4,
  kKernLayerNormBackwardBf16Team4,
  kKernLayerNormBackwardKeptBf16Team4,
  kKernLayerNormF16Wave1,
  kKernLayerNormBackwardF16Wave1,
  kKernLayerNormBackwardKeptF16Wave1,
  kKernLayerNormF16Wave2,
  kKernLayerNormBackwardF16Wave2,
  kKernLayerNormBackwardKeptF16Wave2,
  kKernLayerNormF16Team2,
  kKernLayerNormBackwardF16Team2,
  kKernLayerNormBackwardKeptF16Team2,
  kKernLayerNormF16Team4,
  kKernLayerNormBackwardF16Team4,
  kKernLayerNormBackwardKeptF16Team4,
  kKernLayerNormF32Wave1,
  kKernLayerNormBackwardF32Wave1,
  kKernLayerNormBackwardKeptF32Wave1,
  kKernLayerNormF32Wave2,
  kKernLayerNormBackwardF32Wave2,
  kKernLayerNormBackwardKeptF32Wave2,
  kKernLayerNormF32Team2,
  kKernLayerNormBackwardF32Team2,
  kKernLayerNormBackwardKeptF32Team2,
  kKernLayerNormF32Team4,
  kKernLayerNormBackwardF32Team4,
  kKernLayerNormBackwardKeptF32Team4,
  kKernLayerNormJoin,
  // activations in 8 bits and back, per type
  kKernAct8QuantizeBf16,
  kKernAct8DequantizeBf16,
  kKernAct8QuantizeF16,
  kKernAct8DequantizeF16,
  kKernAct8QuantizeF32,
  kKernAct8DequantizeF32,
  // weight gradients: per type and tile of sh_act8_args.h, without the largest for fp32
  kKernWeightGradBf1632x128,
  kKernWeightGradBf1664x128,
  kKernWeightGradBf16128x128,
  kKernWeightGradBf16256x256,
  kKernWeightGradF1632x128,
  kKernWeightGradF1664x128,
  kKernWeightGradF16128x128,
  kKernWeightGradF16256x256,
  kKernWeightGradF3232x128,
  kKernWeightGradF3264x128,
  kKernWeightGradF32128x128,
  kKernWeightGradJoin,
  kKernelCount
};
// Launches kernel `id` of the current device: a 1-D grid of `grid` workgroups of `block`
// work-items on `stream`; args[i] points to the i-th kernel argument.
int launch_kernel(KernelId id, uint32_t grid, uint32_t block, hipStream_t stream, void** args, const char* who);
// Device address of the unpack code object's `scratch` array on the current device.
int noalloc_scratch(void** ptr, const char* who);
// Waits for each device that has the kernels loaded, then unloads them (sh_shutdown).
int unload_kernels();
// Number of devices with the kernels loaded.
int kernels_loaded();
// Ends sh_unpack_noalloc's per-device ordering state (sh_shutdown, before unload_kernels).
void noalloc_release();

// Most chunks one digest launch may cover: one 256-work-item workgroup per chunk, in a 1-D
// grid that stays under 2^32 work-items.
constexpr uint64_t kMaxDigestChunks = 0xFFFFFFFFull / 256u;

// Chunk digests (sh_digest.cpp): the launches behind sh_block_digest / sh_block_changed, for
// the loader and the save-back engine.
int launch_block_digest(const void* buf, uint64_t bytes, uint32_t chunk_bytes, uint64_t* digests, hipStream_t stream);
int launch_block_changed(const void* buf, uint64_t bytes, uint32_t chunk_bytes, const uint64_t* digests,
                         uint8_t* changed, hipStream_t stream);

// floor(n / d) for every 32-bit n, with magic = ceil(2^64 / d) for d >= 2 and
// magic = 0 for d == 1. The quotient is floor(n * magic / 2^64): with
// magic = 2^64/d + eps (0 <= eps < 1), the error term n*eps/2^64 < 2^-32 <= 1/d
// never carries the fractional part of n/d past the next integer.
__host__ __device__ inline uint64_t udiv_magic(uint32_t d) {
  return d <= 1 ? 0ull : (UINT64_MAX / d) + 1ull;
}

__host__ __device__ inline uint32_t udiv(uint32_t n, uint64_t magic) {
  if (magic == 0) return n;
  const uint64_t lo = (uint64_t)n * (uint32_t)magic;
  const uint64_t hi = (uint64_t)n * (uint32_t)(magic >> 32);
  return (uint32_t)((hi + (lo >> 32)) >> 32);
}

}  // namespace sh
