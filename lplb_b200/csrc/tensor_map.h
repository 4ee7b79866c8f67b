// Tensor maps of the kernels that load their operands by TMA.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace lplb {

// The driver entry point is fetched at run time so that the library has no link-time
// dependency on libcuda (it is imported on GPU-less build hosts too).
inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }
  return fn;
}

// A map with rows of 128 bytes in shared memory, 128-byte swizzle, zeros outside the tensor.  Returns 0 on
// success, -1 without the driver's entry point, -2 for a base or stride off a 16-byte boundary.
inline int encode_tensor_map(CUtensorMap* out, CUtensorMapDataType type, const void* base, uint32_t rank, const cuuint64_t* dims,
                             const cuuint64_t* strides, const cuuint32_t* box) {
  auto fn = tensor_map_encoder();
  if (!fn) return -1;
  if ((reinterpret_cast<uintptr_t>(base) & 15) || strides[0] % 16) return -2;
  const cuuint32_t elem_strides[5] = {1, 1, 1, 1, 1};
  auto encode = [&] {
    return fn(out, type, rank, const_cast<void*>(base), dims, strides, box, elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult rc = encode();
  // The driver's call wants a current context, which a thread that has not called the runtime yet (a backward pass's, whose first
  // kernel this is) does not have: the runtime makes one current when the device is set.
  int device = 0;
  if (rc == CUDA_ERROR_INVALID_CONTEXT && cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess) rc = encode();
  return rc == CUDA_SUCCESS ? 0 : (int)rc;
}

}  // namespace lplb
