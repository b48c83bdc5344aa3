// Checks of arguments that the C entry points over paged caches share.
#pragma once

#include <cuda_runtime.h>

#include <algorithm>
#include <cstddef>
#include <cstdint>

#include "common.hpp"
#include "jal.h"

namespace jal {

constexpr uint64_t kMaxPositions = 0x7fffffffull - 65536;  // tiles run past the last position by less than 65536
constexpr uint64_t kMaxInt = 0x7fffffffull;

inline bool float_type(int t) { return t == JAL_F32 || t == JAL_F16 || t == JAL_BF16; }
inline size_t type_bytes(int t) { return t == JAL_F32 ? 4 : 2; }

// `p` is memory of the current device: a tensor of another device, or of the
// host, would fault in the kernel.
inline void on_device(const void *p, const char *what, int device) {
  cudaPointerAttributes a = {};
  JAL_CUDA(cudaPointerGetAttributes(&a, p));
  if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged)
    fail(JAL_ERR_INVALID_ARGUMENT, "%s is not device memory", what);
  if (a.type == cudaMemoryTypeDevice && a.device != device)
    fail(JAL_ERR_INVALID_ARGUMENT, "%s is on device %d, the current device is %d", what, a.device, device);
}
inline int current_device() {
  int d = 0;
  JAL_CUDA(cudaGetDevice(&d));
  return d;
}
inline void aligned16(const void *p, const char *what) {
  if ((uintptr_t)p % 16) fail(JAL_ERR_TENSOR_BOUNDS, "%s is not 16-byte aligned", what);
}
// Arrays that kernels read and write as 4-byte values: an address between two of
// them would fault.
inline void aligned4(const void *p, const char *what) {
  if ((uintptr_t)p % 4) fail(JAL_ERR_TENSOR_BOUNDS, "%s is not 4-byte aligned", what);
}

// A batch over caches of n_seqs table rows with that many positions each.
inline jal_ragged_batch checked_batch(const jal_ragged_batch *in, uint64_t n_seqs, uint64_t positions) {
  NEED(in);
  jal_ragged_batch b = *in;
  NEED(b.q_start);
  NEED(b.kv_len);
  aligned4(b.q_start, "q_start");
  aligned4(b.kv_len, "kv_len");
  if (b.n_seqs > n_seqs)
    fail(JAL_ERR_TENSOR_BOUNDS, "batch of %llu sequences over a table of %llu", (unsigned long long)b.n_seqs,
         (unsigned long long)n_seqs);
  if (b.n_rows > kMaxPositions) fail(JAL_ERR_TENSOR_BOUNDS, "batch of 2^31 rows or more");
  if (b.max_q_len > b.n_rows) b.max_q_len = b.n_rows;
  b.max_kv_len = std::min<uint64_t>(std::max<uint64_t>(b.max_kv_len, 1), positions);
  return b;
}

inline int64_t row_stride(size_t stride, size_t width, const char *what) {
  if (stride == 0) stride = width;
  if (stride < width || stride % 8 || stride > (1ull << 40))
    fail(JAL_ERR_TENSOR_BOUNDS, "%s stride %zu: a multiple of 8, at least %zu", what, stride, width);
  return (int64_t)stride;
}

}  // namespace jal
