// Tensor maps for the kernels outside gemm_sm100.cu, from the same cache.
#pragma once
#include <cstdint>
#include <cuda.h>

namespace gonn {

// `strides`: rank - 1 of them, in bytes.  Elements outside `dims` read as zero.
bool encode_tensor_map(CUtensorMap* map, CUtensorMapDataType dtype, uint32_t rank, const void* base,
                       const uint64_t* dims, const uint64_t* strides, const uint32_t* box,
                       CUtensorMapSwizzle swizzle);

}  // namespace gonn
