// Microscaled 4-bit operands (MXFP4: e2m1 codes, one power-of-two scale for 32 of them):
// quantisation and back.  The next precision below the fp16 path, no counterpart in the
// reference; the product is in mxfp4_gemm.cu.
//
// All three kernels are bound by HBM: 4 bytes of float32 an element on one side, 17/32 byte on the
// other.  Every word of four scales (four blocks of a row, which lie side by side in the scales'
// tile order) has one writer, which also writes the zeros of the padding.
#include <algorithm>

#include "kernels.h"
#include "launch.cuh"
#include "mxfp4.cuh"
#include "ptx.cuh"

namespace gonn {

namespace {

using namespace mxfp4;

constexpr uint32_t SEGMENT = 256;  // elements of a row that a warp takes at once: 8 a lane

// The 8 warps of a block take the rows i, i + 1 of each of the four 32-row groups of a tile of 128
// rows: their scale words fill 32 neighbouring bytes of a tile.
__device__ __forceinline__ uint64_t row_of_warp(uint32_t block, uint32_t warp) {
  return uint64_t(block >> 4) * 128 + (warp & 3u) * 32 + (block & 15u) * 2 + (warp >> 2);
}
__device__ __forceinline__ uint64_t scale_word(uint64_t row, uint64_t group, uint64_t groups) {
  return ((row >> 7) * groups + group) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// Blocks along the rows of src.  A lane holds 8 neighbouring elements, four lanes a block of 32.
// Rows that do not start on 16 bytes are read a float a lane and change hands in shared memory.
template <bool VEC>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const float* __restrict__ src, Mxfp4Layout l,
                                                            uint8_t* __restrict__ packed) {
  ptx::grid_dependency_release();  // programmatic dependent launch: see launch.cuh
  ptx::grid_dependency_wait();
  __shared__ float4 staged[VEC ? 1 : 8][VEC ? 1 : SEGMENT / 4];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t row = row_of_warp(blockIdx.x, warp);
  const bool live = row < l.rows;
  const float* x = src + (live ? row : 0) * l.cols;
  const uint32_t segments = uint32_t((l.groups + 1) / 2);
  for (uint32_t seg = blockIdx.y; seg < segments; seg += gridDim.y) {
    const uint64_t col = uint64_t(seg) * SEGMENT + lane * 8;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    if (VEC) {  // cols is a multiple of 4
      if (live && col < l.cols) a = __ldcs(reinterpret_cast<const float4*>(x + col));
      if (live && col + 4 < l.cols) b = __ldcs(reinterpret_cast<const float4*>(x + col) + 1);
    } else {
      float* mine = reinterpret_cast<float*>(staged[warp]);
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        const uint64_t at = uint64_t(seg) * SEGMENT + j * 32 + lane;
        mine[j * 32 + lane] = live && at < l.cols ? __ldcs(x + at) : 0.f;
      }
      __syncwarp();
      a = staged[warp][lane * 2];
      b = staged[warp][lane * 2 + 1];
      __syncwarp();
    }
    const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    uint32_t amax = 0;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(v[j]) & 0x7fffffffu);
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const bool in = live && col / 32 < l.blocks;
    const uint32_t byte = in ? scale_byte(amax) : 0u;
    const float f = inverse_scale(byte);
    uint32_t codes = 0;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) codes |= encode2(v[2 * j] * f, v[2 * j + 1] * f) << (8 * j);
    if (byte == kScaleNan) codes = 0;
    if (in) *reinterpret_cast<uint32_t*>(packed + row * l.row_bytes + col / 2) = codes;
    // the bytes of four blocks, from lanes 0, 4, 8, 12 of each half warp
    const uint32_t from = lane & 16u;
    uint32_t word = 0;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) word |= __shfl_sync(0xffffffffu, byte, from + j * 4) << (8 * j);
    const uint64_t group = uint64_t(seg) * 2 + (lane >> 4);
    if ((lane & 15u) == 0 && group < l.groups)
      *reinterpret_cast<uint32_t*>(packed + l.scale_offset + scale_word(row, group, l.groups)) = word;
  }
}

// Blocks down the columns of src [l.cols, l.rows]: a thread takes one column, four blocks of it,
// so that a warp's loads cover 128 contiguous bytes and a thread's codes 64.
__global__ void __launch_bounds__(128) quantize_columns_kernel(const float* __restrict__ src, Mxfp4Layout l,
                                                               uint8_t* __restrict__ packed) {
  ptx::grid_dependency_release();  // programmatic dependent launch: see launch.cuh
  ptx::grid_dependency_wait();
  const uint64_t row = uint64_t(blockIdx.x) * 128 + threadIdx.x;
  const bool live = row < l.rows;
  for (uint64_t group = blockIdx.y; group < l.groups; group += gridDim.y) {
    uint32_t word = 0;
#pragma unroll 1
    for (uint32_t q = 0; q < 4; ++q) {
      const uint64_t block = group * 4 + q;
      if (!live || block >= l.blocks) break;
      const float* x = src + block * 32 * l.rows + row;
      float v[32];
      uint32_t amax = 0;
      if (block * 32 + 32 <= l.cols) {
#pragma unroll
        for (uint32_t j = 0; j < 32; ++j) v[j] = __ldcs(x + j * l.rows);
      } else {
#pragma unroll
        for (uint32_t j = 0; j < 32; ++j) v[j] = block * 32 + j < l.cols ? x[j * l.rows] : 0.f;
      }
#pragma unroll
      for (uint32_t j = 0; j < 32; ++j) amax = max(amax, __float_as_uint(v[j]) & 0x7fffffffu);
      const uint32_t byte = scale_byte(amax);
      const float f = inverse_scale(byte);
      uint32_t codes[4] = {0, 0, 0, 0};
      if (byte != kScaleNan) {
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j) codes[j / 4] |= encode2(v[2 * j] * f, v[2 * j + 1] * f) << (8 * (j % 4));
      }
      *reinterpret_cast<uint4*>(packed + row * l.row_bytes + block * 16) =
          make_uint4(codes[0], codes[1], codes[2], codes[3]);
      word |= byte << (8 * q);
    }
    *reinterpret_cast<uint32_t*>(packed + l.scale_offset + scale_word(row, group, l.groups)) = word;
  }
}

// Two 16-byte stores a lane, each covering 512 contiguous bytes a warp (VEC: rows start on 16
// bytes), or eight of 4 bytes; a lane takes the codes for them from the lane that loaded them.
template <bool VEC>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* __restrict__ packed, Mxfp4Layout l,
                                                         float* __restrict__ dst) {
  ptx::grid_dependency_release();  // programmatic dependent launch: see launch.cuh
  ptx::grid_dependency_wait();
  constexpr uint32_t PIECE = VEC ? 4 : 1, PIECES = SEGMENT / 32 / PIECE;
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t row = row_of_warp(blockIdx.x, threadIdx.x >> 5);
  if (row >= l.rows) return;
  const uint8_t* scales = packed + l.scale_offset;
  const uint32_t segments = uint32_t((l.groups + 1) / 2);
  for (uint32_t seg = blockIdx.y; seg < segments; seg += gridDim.y) {
    const uint64_t first = uint64_t(seg) * SEGMENT;
    // eight codes a lane; the scale of lane's block (the first 8 lanes hold the segment's)
    const bool here = first / 32 + lane / 4 < l.blocks;
    const uint32_t codes =
        here ? __ldcs(reinterpret_cast<const uint32_t*>(packed + row * l.row_bytes + first / 2) + lane) : 0u;
    const uint64_t block = first / 32 + (lane & 7u);
    const float scale = block < l.blocks
                            ? scale_value(scales[scale_word(row, block >> 2, l.groups) + (block & 3)]) : 0.f;
#pragma unroll
    for (uint32_t i = 0; i < PIECES; ++i) {
      const uint32_t at = (i * 32 + lane) * PIECE;  // element of the segment
      const uint32_t mine = __shfl_sync(0xffffffffu, codes, at / 8) >> (at % 8 * 4);
      const float s = __shfl_sync(0xffffffffu, scale, at / 32);
      float* out = dst + row * l.cols + first + at;
      if (first + at < l.cols) {
        if (VEC)
          __stcs(reinterpret_cast<float4*>(out), make_float4(decode(mine) * s, decode(mine >> 4) * s,
                                                             decode(mine >> 8) * s, decode(mine >> 12) * s));
        else
          *out = decode(mine) * s;
      }
    }
  }
}

// Grid over the row tiles and, as far as those do not fill the GPU, over the segments of a row.
dim3 row_grid(const Mxfp4Layout& l) {
  const uint64_t x = (l.rows + 127) / 128 * 16, segments = (l.groups + 1) / 2;
  const uint64_t y = std::min({std::max<uint64_t>(1, 148 * 16 / x), segments, uint64_t(65535)});
  return dim3(uint32_t(x), uint32_t(y));
}

bool vector_rows(const float* p, uint64_t cols) {
  return (cols & 3) == 0 && (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}

}  // namespace

cudaError_t launch_mxfp4_quantize(const float* src, uint64_t rows, uint64_t cols, bool transposed,
                                  void* packed, cudaStream_t stream) {
  uint8_t* out = static_cast<uint8_t*>(packed);
  if (transposed) {
    const Mxfp4Layout l(cols, rows);
    const dim3 grid(uint32_t((l.rows + 127) / 128), uint32_t(std::min<uint64_t>(l.groups, 65535)));
    return launch_kernel(quantize_columns_kernel, grid, dim3(128), 0, stream, src, l, out);
  }
  const Mxfp4Layout l(rows, cols);
  return launch_kernel(vector_rows(src, cols) ? quantize_rows_kernel<true> : quantize_rows_kernel<false>, row_grid(l),
                       dim3(256), 0, stream, src, l, out);
}

cudaError_t launch_mxfp4_dequantize(const void* packed, uint64_t rows, uint64_t cols, float* dst,
                                    cudaStream_t stream) {
  const Mxfp4Layout l(rows, cols);
  return launch_kernel(vector_rows(dst, cols) ? dequantize_kernel<true> : dequantize_kernel<false>, row_grid(l),
                       dim3(256), 0, stream, static_cast<const uint8_t*>(packed), l, dst);
}

}  // namespace gonn
