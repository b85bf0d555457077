// Helpers of the operators of a served batch.
#pragma once

#include <atomic>

#include "common.cuh"

namespace fa {

// Raises a kernel's limit of dynamic shared memory, once per device.
template <auto Kernel>
inline int allow_smem(int bytes, const char* what) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && dev < 64 && ((done.load(std::memory_order_relaxed) >> dev) & 1)) return FA_OK;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return cuda_fail(e, what);
  if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return FA_OK;
}

// (cols x rows x heads x pages) tiled tensor map of a 16-bit cache of pages, 128-byte swizzle, out-of-range elements read
// as 0.  box_cols * 2 bytes must not exceed 128.  Strides in elements.
int make_tensor_map_4d(CUtensorMap* m, const void* base, int dtype, int cols, int rows, int64_t row_stride, int heads,
                       int64_t head_stride, int pages, int64_t page_stride, int box_cols, int box_rows);

}  // namespace fa
