// Kernels of the 4-bit microscaled format (mxfp4.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace moe {

// rows x (32 * blocks) values, `pitch` bytes between rows, to codes and tiled
// exponents. Exponents of rows up to pad_rows and of blocks up to
// 4 * k_tiles are written as zero.
template <int kType>
__global__ void mxfp4_quantize_kernel(const uint8_t* x, int64_t pitch, int rows, int blocks, int k_tiles, int pad_rows,
                                      int vec32, uint8_t* q, uint8_t* scale);
__global__ void mxfp4_gate_kernel(const float* sums, int rows, int blocks, int k_tiles, int act, uint8_t* q,
                                  uint8_t* scale);
template <int kType>
__global__ void mxfp4_dequantize_kernel(const uint8_t* q, const uint8_t* scale, int64_t total, int blocks, int k_tiles,
                                        int vec32, uint8_t* out);

}  // namespace moe
