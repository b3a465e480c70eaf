// 4-bit microscaled blocks (OCP MX, e2m1 elements): quantiser, dequantiser,
// and the quantiser of gated sums.
//
// A block is 32 consecutive columns of a row. Its exponent is floor(log2 of
// the largest magnitude) - 2, its elements the nearest e2m1 numbers (ties to
// even, beyond 6 to 6) to x / 2^exponent; scaling by a power of two is exact,
// so the only rounding is the 4-bit one. All three kernels give one thread
// whole blocks: it reads whole 32-byte sectors and holds the block in
// registers, so the block maximum needs no exchange between threads. Bound by
// HBM: 2 (or 4) bytes in and 17/32 byte out per element; 16384 x 7168 bf16 at
// 6.6 TB/s (quantiser) and 6.2 TB/s (dequantiser).
#include <cuda_runtime.h>

#include <cstdint>

#include "dense_ptx.cuh"
#include "ffn_math.cuh"
#include "mxfp4.cuh"

namespace moe {

namespace {

// Codes of a block, and its exponent byte into the row's word of the tiled
// array. Called by whole warps: the four threads of a word are neighbours,
// of the same row. `live`: the block exists; `padded`: its exponent byte does
// (zero where the block does not).
__device__ __forceinline__ void store_block(const float* v, bool live, bool padded, int64_t row, int block,
                                            int k_tiles, uint8_t* q_row, uint8_t* scale) {
  uint32_t byte = 0;
  if (live) {
    uint4 c;
    byte = mx_block(v, &c);
    *reinterpret_cast<uint4*>(q_row + 16 * static_cast<int64_t>(block)) = c;
  }
  uint32_t word = byte << (8 * (block & 3));
  word |= __shfl_xor_sync(0xffffffffu, word, 1);
  word |= __shfl_xor_sync(0xffffffffu, word, 2);
  if (padded && (block & 3) == 0)
    *reinterpret_cast<uint32_t*>(scale + mx_scale_offset(row, block, k_tiles)) = word;
}

}  // namespace

// One CTA takes 128 rows x one exponent tile (four blocks). Its exponent
// bytes meet in shared memory and leave as a whole 512-byte tile; written word
// by word from CTAs of one row each they cost a tenth more transactions
// (16384 x 7168 bf16 53.9 -> 45.0 us, all of the measured copy rate; with two
// tiles a CTA 49 us). A thread's two blocks are loaded together.
template <int kType>
__global__ void __launch_bounds__(256, kType == kTypeFp32 ? 2 : 4)
    mxfp4_quantize_kernel(const uint8_t* x, int64_t pitch, int rows, int blocks, int k_tiles, int vec32, uint8_t* q,
                          uint8_t* scale) {
  __shared__ __align__(16) uint8_t s_scale[512];
  pdl_wait();
  pdl_launch_next();
  constexpr int kBytes = kType == kTypeFp32 ? 128 : 64;
  constexpr int kWords = kBytes / 4;
  const int tid = static_cast<int>(threadIdx.x);
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * 128 + tid / 4;   // and 64 rows further
  const int block = static_cast<int>(blockIdx.x) * 4 + (tid & 3);
  uint32_t raw[2][kWords];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t row = row0 + 64 * j;
    if (row < rows && block < blocks)
      load_words<kWords>(x + row * pitch + static_cast<int64_t>(block) * kBytes, vec32 != 0, raw[j]);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t row = row0 + 64 * j;
    uint32_t byte = 0;
    if (row < rows && block < blocks) {
      float v[32];
      unpack_words<kType>(raw[j], v);
      uint4 codes;
      byte = mx_block(v, &codes);
      *reinterpret_cast<uint4*>(q + (row * blocks + block) * 16) = codes;
    }
    const int r = tid / 4 + 64 * j;
    s_scale[(r & 31) * 16 + (r >> 5) * 4 + (tid & 3)] = static_cast<uint8_t>(byte);
  }
  __syncthreads();
  if (tid < 32)
    *reinterpret_cast<uint4*>(scale + (static_cast<int64_t>(blockIdx.y) * k_tiles + blockIdx.x) * 512 + tid * 16) =
        *reinterpret_cast<const uint4*>(s_scale + tid * 16);
}

// h = act(gate) * up of fp32 sums [rows, 2 n] (up, then gate), in 4 bits. (Lets
// the next kernel start after its own wait, as every kernel here: 4-bit block
// of H = 7168, I = 2048 at 16 tokens 15.45 -> 15.19 us against before it, at
// 64 the same.)
__global__ void __launch_bounds__(256)
    mxfp4_gate_kernel(const float* sums, int rows, int blocks, int k_tiles, int act, uint8_t* q, uint8_t* scale) {
  pdl_wait();
  pdl_launch_next();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int per_row = 4 * k_tiles;
  const int row = static_cast<int>(i / per_row);
  const int block = static_cast<int>(i - static_cast<int64_t>(row) * per_row);
  const bool live = row < rows && block < blocks;
  float v[32];
  if (live) {
    const float* up = sums + static_cast<int64_t>(row) * 64 * blocks + 32 * block;
    uint32_t u[32], g[32];
    load_words<32>(up, true, u);
    load_words<32>(up + 32 * blocks, true, g);
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(u[j]) * act_value(__uint_as_float(g[j]), act);
  }
  store_block(v, live, row < rows, row, block, k_tiles, q + static_cast<int64_t>(row) * blocks * 16, scale);
}

template <int kType>
__global__ void __launch_bounds__(256)
    mxfp4_dequantize_kernel(const uint8_t* q, const uint8_t* scale, int64_t total, int blocks, int k_tiles, int vec32,
                            uint8_t* out) {
  pdl_wait();
  pdl_launch_next();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= total) return;
  const int64_t row = i / blocks;
  const int block = static_cast<int>(i - row * blocks);
  const uint32_t byte = scale[mx_scale_offset(row, block, k_tiles)];
  // 2^(byte - 127); byte 0 is a subnormal, 255 is NaN
  const float f = __uint_as_float(byte == 0u ? 0x00400000u : byte == 255u ? 0x7fc00000u : byte << 23);
  const uint4 c = *reinterpret_cast<const uint4*>(q + 16 * i);
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  float v[32];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 t0, t1, t2, t3;\n\t"
        "mov.b32 {t0, t1, t2, t3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, t0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, t1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, t2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, t3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w[j]));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 p = unpack_16(h[e], kTypeFp16);
      v[8 * j + 2 * e] = p.x * f;
      v[8 * j + 2 * e + 1] = p.y * f;
    }
  }
  constexpr int kWords = kType == kTypeFp32 ? 32 : 16;
  uint32_t r[kWords];
#pragma unroll
  for (int j = 0; j < kWords; ++j)
    r[j] = kType == kTypeFp32 ? __float_as_uint(v[j]) : pack_16(v[(2 * j) & 31], v[(2 * j + 1) & 31], kType);
  uint32_t* dst = reinterpret_cast<uint32_t*>(out) + i * kWords;
  if (vec32) {
#pragma unroll
    for (int j = 0; j < kWords; j += 8) st_global_32(dst + j, r + j);
  } else {
#pragma unroll
    for (int j = 0; j < kWords; j += 4)
      *reinterpret_cast<uint4*>(dst + j) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
  }
}

template __global__ void mxfp4_quantize_kernel<kTypeBf16>(const uint8_t*, int64_t, int, int, int, int, uint8_t*, uint8_t*);
template __global__ void mxfp4_quantize_kernel<kTypeFp16>(const uint8_t*, int64_t, int, int, int, int, uint8_t*, uint8_t*);
template __global__ void mxfp4_quantize_kernel<kTypeFp32>(const uint8_t*, int64_t, int, int, int, int, uint8_t*, uint8_t*);
template __global__ void mxfp4_dequantize_kernel<kTypeBf16>(const uint8_t*, const uint8_t*, int64_t, int, int, int,
                                                            uint8_t*);
template __global__ void mxfp4_dequantize_kernel<kTypeFp16>(const uint8_t*, const uint8_t*, int64_t, int, int, int,
                                                            uint8_t*);
template __global__ void mxfp4_dequantize_kernel<kTypeFp32>(const uint8_t*, const uint8_t*, int64_t, int, int, int,
                                                            uint8_t*);

}  // namespace moe
