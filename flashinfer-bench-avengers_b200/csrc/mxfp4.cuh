// 4-bit microscaled blocks: what a thread does with one block, and the
// kernels (mxfp4.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "dense_ptx.cuh"
#include "ffn_math.cuh"

namespace moe {

// kWords 32-bit words at `src` (16-byte aligned; whole sectors if vec32).
template <int kWords>
__device__ __forceinline__ void load_words(const void* src, bool vec32, uint32_t* r) {
  if (vec32) {
#pragma unroll
    for (int j = 0; j < kWords; j += 8) ld_global_32(r + j, static_cast<const uint32_t*>(src) + j);
  } else {
#pragma unroll
    for (int j = 0; j < kWords; j += 4) {
      const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const uint32_t*>(src) + j);
      r[j] = q.x, r[j + 1] = q.y, r[j + 2] = q.z, r[j + 3] = q.w;
    }
  }
}

// The 32 values of a block.
template <int kType>
__device__ __forceinline__ void unpack_words(const uint32_t* r, float* v) {
#pragma unroll
  for (int j = 0; j < (kType == kTypeFp32 ? 32 : 16); ++j) {
    if (kType == kTypeFp32) {
      v[j] = __uint_as_float(r[j]);
    } else {
      const float2 f = unpack_16(r[j], kType);
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  }
}

// The exponent byte and the 16 bytes of codes of 32 values.
__device__ __forceinline__ uint32_t mx_block(const float* v, uint4* codes) {
  uint32_t amax = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j) amax = max(amax, __float_as_uint(v[j]) & 0x7fffffffu);
  const uint32_t byte = mx_exponent(amax);
  *codes = make_uint4(0, 0, 0, 0);
  if (byte != 255u) {
    const float inv = mx_inverse(byte);
    *codes = make_uint4(mx_pack8(v, inv), mx_pack8(v + 8, inv), mx_pack8(v + 16, inv), mx_pack8(v + 24, inv));
  }
  return byte;
}

// rows x (32 * blocks) values, `pitch` bytes between rows, to codes and tiled
// exponents (whole tiles: zero where no block is). Grid: (k_tiles, ceil(rows /
// 128)).
template <int kType>
__global__ void mxfp4_quantize_kernel(const uint8_t* x, int64_t pitch, int rows, int blocks, int k_tiles, int vec32,
                                      uint8_t* q, uint8_t* scale);
__global__ void mxfp4_gate_kernel(const float* sums, int rows, int blocks, int k_tiles, int act, uint8_t* q,
                                  uint8_t* scale);
template <int kType>
__global__ void mxfp4_dequantize_kernel(const uint8_t* q, const uint8_t* scale, int64_t total, int blocks, int k_tiles,
                                        int vec32, uint8_t* out);

}  // namespace moe
