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
  kEpiBackward = 3,    // preact set: the sums are dh, out = [du | dg] with the saved up and gate sums;
                       // otherwise out[r, c] = sum
};

// Where the streaming form's token operand comes from.
enum TokenSource : int {
  kFromMatrix = 0,     // A, a 16-bit or 4-bit matrix
  kFromRows = 1,       // 4-bit: unquantised rows (DenseParams x, of type `type`)
  kFromSums = 2,       // 4-bit: act(gate) * up of fp32 sums [m, 2 k] (DenseParams x)
};

// A stored matrix of 16-bit elements.
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
  void* out;           // [m, n], row pitch ldo elements; [du | dg]: [m, 2 n]
  int64_t ldo;
  void* out_lo;        // streaming form: what the rounding of h (when set) or [du | dg] left, rounded again
  float* preact;       // fp32 [m, 2 n]: written by kEpiGated when set, read by kEpiBackward
  uint8_t* q;          // kEpiGatedQuant: codes [m, n / 2]
  uint8_t* q_scale;    //   and tiled exponents
  uint32_t* status;    // sticky device status word
  int x_source;        // TokenSource (4-bit streaming form)
  const void* x;       // its rows, x_pitch bytes apart
  int64_t x_pitch;
  // derived by the launcher
  int bn, n_step, b_half, m_tiles, n_tiles, k_iters, vec32, vec16, a_mn, copy_bytes;
  int early;           // B may be read before the kernel before has finished
};

// D = A B^T with B stored K x N, and A stored M x K or (a_mn) K x M.
struct DenseProduct {
  DenseOperand a, b;
  bool a_mn;
  DenseParams p;
};

struct MxOperand {
  const void* q;       // [rows, K / 2] codes
  const void* scale;   // tiled exponents
  int64_t rows;
};

// Every kernel starts under the end of the one before it, whatever that was
// (programmatic dependent launch), and waits for it before it touches memory:
// block at one token 21.2 -> 20.3 us, 4-bit linear 8.1 -> 6.9, training step
// 333 x 1032 x 520 36 -> 34 against ordinary launches of a call's first
// kernel. With `dependent` the kernel follows another of the same call; then
// it reads B, an input of the whole call, before it waits. That is sound
// because each kernel waits before it lets the next one start: when a call's
// second kernel starts, all work before the call is complete.
//
// D = A B^T over CTA pairs, both operands stored along K (kEpiStore,
// kEpiGated: B has 2 n rows, up then gate). Returns a MOE_B200 status code.
int launch_dense_pair(DenseEpi epi, const DenseOperand& a, const DenseOperand& b, const DenseParams& p, int sm_count,
                      bool dependent, cudaStream_t s);

// How a launch cuts its products into tiles.
struct DensePlan {
  int bn[2];           // columns per tile of the first product, of the others
  int splits;          // K parts (a single product)
  int lead;
  int64_t cost;        // expected, in cycles
};

// Up to three products of the backward pass that do not depend on each other,
// in one launch; all but the first have the same K.
DensePlan plan_dense_backward(const DenseProduct* products, int count, int sm_count);
int launch_dense_backward(const DenseProduct* products, int count, const DensePlan& plan, int sm_count, bool dependent,
                          cudaStream_t s);

// 4-bit operands over CTA pairs (kEpiStore, kEpiGatedQuant).
int launch_mx_pair(DenseEpi epi, const MxOperand& a, const MxOperand& b, const DenseParams& p, int sm_count,
                   bool dependent, cudaStream_t s);

// Few rows of A (16 bits: up to 64; 4 bits: up to 128): out = A B^T streaming
// B, K split over a cluster (kEpiStore and kEpiGated; kEpiBackward with B
// stored K x N; 4-bit: kEpiStore). With a_lo set the operand is a and what its
// rounding left, a_lo / rest_scale.
int launch_dense_skinny(DenseEpi epi, const DenseOperand& a, const void* a_lo, const DenseOperand& b, DenseParams p,
                        int sm_count, bool dependent, cudaStream_t s);
int launch_mx_skinny(const MxOperand& a, const MxOperand& b, DenseParams p, int sm_count, bool dependent,
                     cudaStream_t s);

// Whether launch_mx_skinny takes sources other than kFromMatrix at this size.
bool mx_skinny_quantizes(int64_t m, int64_t n, int64_t k, int sm_count);

// The current device's sticky status word of the dense kernels (a library
// global), or null when its address cannot be had.
uint32_t* dense_status_word();

}  // namespace moe
