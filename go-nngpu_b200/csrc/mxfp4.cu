// Microscaled 4-bit operands (MXFP4: e2m1 codes, one power-of-two scale for 32 of them):
// quantisation and back.  The next precision below the fp16 path, no counterpart in the
// reference; the product is in mxfp4_gemm.cu.
#include "kernels.h"
#include "launch.cuh"
#include "mxfp4.cuh"
#include "ptx.cuh"

namespace gonn {

namespace {

using namespace mxfp4;

__host__ __device__ __forceinline__ uint64_t scale_at(uint64_t row, uint64_t block, uint64_t groups) {
  return ((row >> 7) * groups + (block >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

// One thread per block of 32, the padding of the scales included.
__global__ void __launch_bounds__(128) quantize_kernel(const float* __restrict__ src, Mxfp4Layout l,
                                                       uint64_t row_step, uint64_t col_step,
                                                       uint8_t* __restrict__ packed) {
  ptx::grid_dependency_release();  // programmatic dependent launch: see launch.cuh
  ptx::grid_dependency_wait();
  const uint64_t all_rows = (l.rows + 127) / 128 * 128, all_blocks = l.groups * 4;
  for (uint64_t i = blockIdx.x * uint64_t(blockDim.x) + threadIdx.x; i < all_rows * all_blocks;
       i += uint64_t(gridDim.x) * blockDim.x) {
    const uint64_t row = i / all_blocks, block = i % all_blocks;
    uint32_t byte = 0;
    if (row < l.rows && block < l.blocks) {
      float v[32];
      uint32_t amax = 0;
      for (int j = 0; j < 32; ++j) {
        const uint64_t col = block * 32 + j;
        v[j] = col < l.cols ? src[row * row_step + col * col_step] : 0.f;
        amax = max(amax, __float_as_uint(v[j]) & 0x7fffffffu);
      }
      byte = scale_byte(amax);
      const float f = inverse_scale(byte);
      for (int j = 0; j < 16; ++j)
        packed[row * l.row_bytes + block * 16 + j] =
            byte == kScaleNan ? 0 : uint8_t(encode2(v[2 * j] * f, v[2 * j + 1] * f));
    }
    packed[l.scale_offset + scale_at(row, block, l.groups)] = uint8_t(byte);
  }
}

__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* __restrict__ packed, Mxfp4Layout l,
                                                         float* __restrict__ dst) {
  ptx::grid_dependency_release();  // programmatic dependent launch: see launch.cuh
  ptx::grid_dependency_wait();
  for (uint64_t i = blockIdx.x * uint64_t(blockDim.x) + threadIdx.x; i < l.rows * l.cols;
       i += uint64_t(gridDim.x) * blockDim.x) {
    const uint64_t row = i / l.cols, col = i % l.cols;
    const uint32_t two = packed[row * l.row_bytes + col / 2];
    const float s = scale_value(packed[l.scale_offset + scale_at(row, col / 32, l.groups)]);
    dst[i] = decode((col & 1) ? two >> 4 : two & 15u) * s;
  }
}

uint32_t grid_for(uint64_t items, uint32_t per_block, uint32_t most) {
  const uint64_t n = (items + per_block - 1) / per_block;
  return uint32_t(n < most ? n : most);
}

}  // namespace

cudaError_t launch_mxfp4_quantize(const float* src, uint64_t rows, uint64_t cols, bool transposed,
                                  void* packed, cudaStream_t stream) {
  const Mxfp4Layout l(transposed ? cols : rows, transposed ? rows : cols);
  const uint64_t items = (l.rows + 127) / 128 * 128 * l.groups * 4;
  return launch_kernel(quantize_kernel, dim3(grid_for(items, 128, 148 * 16)), dim3(128), 0, stream, src, l,
                       transposed ? uint64_t(1) : cols, transposed ? cols : uint64_t(1),
                       static_cast<uint8_t*>(packed));
}

cudaError_t launch_mxfp4_dequantize(const void* packed, uint64_t rows, uint64_t cols, float* dst,
                                    cudaStream_t stream) {
  const Mxfp4Layout l(rows, cols);
  return launch_kernel(dequantize_kernel, dim3(grid_for(rows * cols, 256, 148 * 16)), dim3(256), 0, stream,
                       static_cast<const uint8_t*>(packed), l, dst);
}

}  // namespace gonn
