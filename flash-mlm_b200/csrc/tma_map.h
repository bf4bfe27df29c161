// TMA tensor maps over the C ABI's [batch][heads][rows][head_dim] views.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>

#include "common.h"
#include "ptx.cuh"

namespace fmlm {

inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// Encodes a 4-D tiled map {D, rows, heads, batch} over `v` with a box of
// {swizzle_bytes / 2, box_rows, 1, 1} and the matching shared-memory swizzle.
// Empty views get a 1-row map over `fallback` that the kernel never loads.  The
// row stride of one row is not looked at.
inline int encode_view(CUtensorMap* m, const fmlm_view4& v, int D, int box_rows, int dtype, const void* fallback,
                const char* name) {
  auto enc = encode_fn();
  if (!enc) return set_error(FMLM_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const int swb = std::min(128, D * 2);
  const bool empty = v.data == nullptr || v.rows <= 0 || v.heads <= 0 || v.batch <= 0;
  const void* base = empty ? fallback : v.data;
  if (!aligned16(base)) return set_error(FMLM_ERR_INVALID, "%s: base address must be 16-byte aligned", name);
  cuuint64_t dims[4], strides[3];
  dims[0] = static_cast<cuuint64_t>(D);
  dims[1] = empty ? 1 : static_cast<cuuint64_t>(v.rows);
  dims[2] = empty ? 1 : static_cast<cuuint64_t>(v.heads);
  dims[3] = empty ? 1 : static_cast<cuuint64_t>(v.batch);
  const int64_t rs = empty || v.rows == 1 ? D : v.row_stride;
  int64_t hs = empty ? D : v.head_stride;
  int64_t bs = empty ? D : v.batch_stride;
  if (!empty) {
    if (rs < D || (rs * 2) % 16 != 0) return set_error(FMLM_ERR_INVALID, "%s: row stride must be >= head_dim and a multiple of 8 elements", name);
    if (v.heads == 1 && (hs <= 0 || (hs * 2) % 16 != 0)) hs = rs * v.rows;
    if (v.batch == 1 && (bs <= 0 || (bs * 2) % 16 != 0)) bs = hs * v.heads;
    if ((hs * 2) % 16 != 0 || hs <= 0 || (bs * 2) % 16 != 0 || bs <= 0)
      return set_error(FMLM_ERR_INVALID, "%s: head/batch strides must be positive multiples of 8 elements", name);
  }
  strides[0] = static_cast<cuuint64_t>(rs) * 2;
  strides[1] = static_cast<cuuint64_t>(hs) * 2;
  strides[2] = static_cast<cuuint64_t>(bs) * 2;
  cuuint32_t box[4] = {static_cast<cuuint32_t>(swb / 2), static_cast<cuuint32_t>(box_rows), 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUtensorMapSwizzle sw = swb == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                : swb == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                            : CU_TENSOR_MAP_SWIZZLE_32B;
  const CUtensorMapDataType dt =
      dtype == FMLM_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  auto encode = [&] {
    return enc(m, dt, 4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  if (r == CUDA_ERROR_INVALID_CONTEXT) {
    // A thread that has made no runtime call yet (an autograd worker, say) has
    // no current context; the runtime would bind one at its first launch.
    int dev = 0;
    cudaGetDevice(&dev);
    cudaSetDevice(dev);
    r = encode();
  }
  if (r != CUDA_SUCCESS) return set_error(FMLM_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed (%d)", name, (int)r);
  return FMLM_OK;
}

}  // namespace fmlm
