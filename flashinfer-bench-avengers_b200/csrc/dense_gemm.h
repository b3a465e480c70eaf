// Launch interface of the dense GEMM kernels (dense_gemm.cu: CTA pairs for
// large batches; dense_skinny.cu: few tokens).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace moe {

// What a GEMM does with its fp32 sums.
enum DenseEpi : int {
  kEpiStore = 0,       // out[r, c] = sum, rounded to out_type
  kEpiGated = 1,       // h = act(gate) * up from the up and gate sums; optionally the sums in fp32
  kEpiGatedQuant = 2,  // the same h, in 4 bits with block exponents
  kEpiDact = 3,        // sums are dh: [du | dg] from the saved up and gate sums
};

// Where the streaming form's token operand comes from.
enum TokenSource : int {
  kFromMatrix = 0,     // A, a 16-bit or 4-bit matrix
  kFromRows = 1,       // 4-bit: unquantised rows (DenseParams x, of type `type`)
  kFromSums = 2,       // 4-bit: act(gate) * up of fp32 sums [m, 2 k] (DenseParams x)
};

// Operands of the 16-bit GEMMs: K-contiguous ("K-major") or contiguous along
// the output dimension ("MN-major").
struct DenseOperand {
  const void* base;
  int64_t rows;      // rows of the stored matrix
  int64_t cols;      // elements per row
  int64_t pitch;     // bytes between rows
};

struct DenseParams {
  int64_t m;           // output rows
  int n;               // output columns (gated: features)
  int k;               // contraction length
  int act;             // activation code
  int type;            // operand type code (bf16 / fp16)
  int out_type;        // type code of `out`
  void* out;           // [m, n], row pitch ldo elements; kEpiDact: [m, 2 n]
  int64_t ldo;
  float* preact;       // fp32 [m, 2 n]: written by kEpiGated when set, read by kEpiDact
  uint8_t* q;          // kEpiGatedQuant: codes [m, n / 2]
  uint8_t* q_scale;    //   and tiled exponents
  uint32_t* status;    // sticky device status word
  int x_source;        // TokenSource (4-bit streaming form)
  const void* x;       // its rows, x_pitch bytes apart
  int64_t x_pitch;
  // derived by the launcher
  int bn, n_step, b_half, m_tiles, n_tiles, k_iters, vec32, stages, stage_bytes;
};

struct MxOperand {
  const void* q;       // [rows, K / 2] codes
  const void* scale;   // tiled exponents
  int64_t rows;
};

// B of every GEMM must be complete before the call's first kernel starts: it
// is read before the previous kernel has finished. A may be its result.
//
// D = A B^T over CTA pairs; a_mn / b_mn: the operand is stored K x M (K x N).
// kEpiGated: B has 2 n rows, up then gate. Returns a MOE_B200 status code.
int launch_dense_pair(DenseEpi epi, const DenseOperand& a, bool a_mn, const DenseOperand& b, bool b_mn, DenseParams p,
                      int sm_count, bool dependent, cudaStream_t s);

// The same for 4-bit operands (kEpiStore, kEpiGatedQuant).
int launch_mx_pair(DenseEpi epi, const MxOperand& a, const MxOperand& b, DenseParams p, int sm_count, bool dependent,
                   cudaStream_t s);

// Few rows of A: out = A B^T streaming B, K split over a cluster
// (kEpiStore and kEpiGated; 4-bit: kEpiStore).
int launch_dense_skinny(DenseEpi epi, const DenseOperand& a, const DenseOperand& b, DenseParams p, int sm_count,
                        bool dependent, cudaStream_t s);
int launch_mx_skinny(const MxOperand& a, const MxOperand& b, DenseParams p, int sm_count, bool dependent,
                     cudaStream_t s);

// Whether launch_mx_skinny takes sources other than kFromMatrix at this size.
bool mx_skinny_quantizes(int64_t m, int64_t n, int64_t k, int sm_count);

// The current device's sticky status word of the dense kernels (a library
// global), or null when its address cannot be had.
uint32_t* dense_status_word();

}  // namespace moe
