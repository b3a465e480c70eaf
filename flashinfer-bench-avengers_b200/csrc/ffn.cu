// C ABI of the dense feed-forward block and of 4-bit microscaled matrices
// (declared in include/moe_b200.h): argument checks, workspaces, the choice
// of kernel, launches. The reference has no counterpart: it implements the
// routed experts of a layer only.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "../../include/moe_b200.h"
#include "dense_gemm.h"
#include "ffn_math.cuh"
#include "host_common.h"
#include "moe_kernels.cuh"
#include "mxfp4.cuh"

namespace moe {
namespace {

constexpr int64_t kMaxDim = 65536;
// Up to this many tokens the GEMMs stream the weights through
// dense_skinny.cu; above (and for the weights' gradients), they run over CTA
// pairs. 16 bits, block over pairs / streaming at 64, 96 and 128 tokens: H =
// 2048, I = 1024 15.2 / 13.9, 16.3 / 21.2 and 17.3 / 24.3 us; 7168, 512 17.9 /
// 16.5, 19.2 / 17.9 and 19.1 / 19.9; 7168, 2048 30.5 / 25.3, 31.1 / 28.3 and
// 31.7 / 31.2. 4 bits, the same block: at 80 tokens 14.1 / 15.7, 18.8 / 17.3
// and 21.5 / 20.1, at 128 14.9 / 18.2, 19.3 / 21.0 and 22.3 / 24.1. A 4-bit
// product alone, whose sums take no further kernel, streams for longer (4096 x
// 7168 at 128 tokens 15.4 / 12.2, 1024 x 2048 9.1 / 7.8). One limit for weights
// of any size, because the block's rounding hangs on it too: the largest lose up
// to 10 % at 65 to 96 tokens by it, where small ones would lose 30 %.
constexpr int64_t kStreamTokens = MOE_B200_FFN_TWO_PART_TOKENS;
constexpr int64_t kMxStreamTokens = 128;

size_t round256(size_t x) { return (x + 255) / 256 * 256; }

bool type16(int t) { return t == MOE_B200_TYPE_BF16 || t == MOE_B200_TYPE_FP16; }
bool any_type(int t) { return type16(t) || t == MOE_B200_TYPE_FP32; }
bool valid_act(int a) { return a == MOE_B200_ACT_SILU || a == MOE_B200_ACT_GELU_TANH; }
bool tokens_ok(int64_t t) { return t >= 0 && t <= MOE_B200_MAX_TOKENS; }
bool dim_ok(int64_t d, int64_t multiple) { return d >= multiple && d <= kMaxDim && d % multiple == 0; }
// Pitch of a row-major operand in elements.
bool pitch_ok(int64_t pitch, int64_t cols) { return pitch >= cols && pitch <= (int64_t(1) << 32); }
bool pitch_aligned(int64_t pitch, int bytes) { return pitch * bytes % 16 == 0; }

struct Device {
  int sm_count;
  uint32_t* status;
};

int open_device(Device* d) {
  DeviceInfo di;
  const int st = current_device_info(&di);
  if (st != MOE_B200_OK) return st;
  d->sm_count = di.sm_count;
  d->status = dense_status_word();
  return d->status != nullptr ? MOE_B200_OK : MOE_B200_ERR_CUDA;
}

DenseOperand rows_of(const void* base, int64_t rows, int64_t cols, int64_t pitch_elems) {
  return DenseOperand{base, rows, cols, pitch_elems * 2};
}

// ---- the forward GEMMs: out = x w^T, gated or plain ------------------------
int forward_gemm(DenseEpi epi, const DenseOperand& x, const void* x_lo, const DenseOperand& w, const DenseParams& p,
                 const Device& d, bool dependent, cudaStream_t s) {
  if (p.m <= kStreamTokens) return launch_dense_skinny(epi, x, x_lo, w, p, d.sm_count, dependent, s);
  return launch_dense_pair(epi, x, w, p, d.sm_count, dependent, s);
}

// ---- 4-bit matrices ---------------------------------------------------------
size_t mx_scale_bytes(int64_t rows, int64_t cols) {
  return static_cast<size_t>(div_up(rows, 128)) * static_cast<size_t>(div_up(cols, 128)) * 512;
}

struct MxBuffers {
  uint8_t* q;
  uint8_t* scale;
};

size_t mx_bytes(int64_t rows, int64_t cols) {
  return round256(static_cast<size_t>(rows) * cols / 2) + round256(mx_scale_bytes(rows, cols));
}

MxBuffers mx_place(uint8_t* at, int64_t rows, int64_t cols) {
  return MxBuffers{at, at + round256(static_cast<size_t>(rows) * cols / 2)};
}

int quantize(const void* x, int type, int64_t rows, int64_t cols, int64_t pitch, uint8_t* q, uint8_t* scale,
             bool early, cudaStream_t s) {
  const int64_t pitch_bytes = pitch * (type == MOE_B200_TYPE_FP32 ? 4 : 2);
  const int vec32 = aligned(x, 32) && pitch_bytes % 32 == 0;
  const int k_tiles = static_cast<int>(div_up(cols, 128));
  const dim3 grid(static_cast<unsigned>(k_tiles), static_cast<unsigned>(div_up(rows, 128)));
  auto kern = type == MOE_B200_TYPE_BF16   ? mxfp4_quantize_kernel<kTypeBf16>
              : type == MOE_B200_TYPE_FP16 ? mxfp4_quantize_kernel<kTypeFp16>
                                           : mxfp4_quantize_kernel<kTypeFp32>;
  return launch_kernel(kern, grid, 256, 0, s, early, static_cast<const uint8_t*>(x), pitch_bytes,
                       static_cast<int>(rows), static_cast<int>(cols / 32), k_tiles, vec32, q, scale) == cudaSuccess
             ? MOE_B200_OK
             : MOE_B200_ERR_CUDA;
}

// Before a GEMM the quantiser starts under the end of the kernel before it
// while it has at most one CTA per SM. A larger grid would crowd the SMs that
// a GEMM before it leaves first, and end later for it (4-bit linear 4096 x
// 7168 started early: at 256 tokens 16.4 -> 15.7 us, at 1024 19.6 -> 20.3, at
// 8192 106.7 -> 111.7).
bool quantize_early(int64_t rows, int64_t cols, const Device& d) {
  return div_up(rows, 128) * div_up(cols, 128) <= d.sm_count;
}

// x [p->m, p->k] to 4 bits, in `to` or (`inside`) by the GEMM itself.
int rows_to_4_bits(const void* x, int type, int64_t pitch, const MxBuffers& to, bool inside, DenseParams* p,
                   const Device& d, cudaStream_t s) {
  if (!inside) return quantize(x, type, p->m, p->k, pitch, to.q, to.scale, quantize_early(p->m, p->k, d), s);
  p->x_source = kFromRows;
  p->x = x;
  p->x_pitch = pitch * (type == MOE_B200_TYPE_FP32 ? 4 : 2);
  return MOE_B200_OK;
}

int mx_gemm(const MxOperand& a, const MxOperand& b, const DenseParams& p, const Device& d, int64_t stream_tokens,
            bool dependent, cudaStream_t s) {
  if (p.m <= stream_tokens) return launch_mx_skinny(a, b, p, d.sm_count, dependent, s);
  return launch_mx_pair(kEpiStore, a, b, p, d.sm_count, dependent, s);
}

DenseParams params(const Device& d, int64_t m, int64_t n, int64_t k, int type, int act, void* out, int64_t ldo,
                   int out_type) {
  DenseParams p;
  std::memset(&p, 0, sizeof(p));
  p.m = m;
  p.n = static_cast<int>(n);
  p.k = static_cast<int>(k);
  p.act = act;
  p.type = type;
  p.out = out;
  p.ldo = ldo;
  p.out_type = out_type;
  p.status = d.status;
  return p;
}

// The 4-bit block over CTA pairs quantises the hidden in the first GEMM's
// epilogue, where the gate rows start on an exponent tile. Otherwise the sums
// go through memory in fp32. (The streaming form with its up and gate tiles
// in one cluster was slower than that: 32 against 24 us at 128 tokens.)
bool fused_gate_quant(int64_t T, int64_t I) { return T > kStreamTokens && I % 128 == 0; }

size_t mx_ffn_bytes(int64_t T, int64_t H, int64_t I) {
  return mx_bytes(T, H) + mx_bytes(T, I) + (fused_gate_quant(T, I) ? 0 : round256(static_cast<size_t>(T) * I * 8));
}

// Only the bits that this read reports: kernels on other streams set bits at
// any time, and one set after the copy is the next read's.
__global__ void clear_status_kernel(uint32_t* word, uint32_t reported) { atomicAnd(word, ~reported); }

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

size_t moe_b200_gated_ffn_workspace_bytes(int64_t num_tokens, int64_t hidden_size, int64_t inter_size) {
  if (!tokens_ok(num_tokens) || !dim_ok(hidden_size, 8) || !dim_ok(inter_size, 8)) return 0;
  // the hidden, and what its rounding left
  const size_t hidden = round256(static_cast<size_t>(num_tokens) * inter_size * 2);
  return (num_tokens <= kStreamTokens ? 2 : 1) * hidden + 256;
}

int moe_b200_gated_ffn(const void* x, int64_t x_pitch, const void* w13, const void* w2, int dtype, int activation,
                       int64_t num_tokens, int64_t hidden_size, int64_t inter_size, void* output, float* preact,
                       void* hidden, void* workspace, size_t workspace_bytes, void* stream) {
  const int64_t T = num_tokens, H = hidden_size, I = inter_size;
  if (!tokens_ok(T) || !dim_ok(H, 8) || !dim_ok(I, 8) || !type16(dtype) || !valid_act(activation) ||
      !pitch_ok(x_pitch, H))
    return MOE_B200_ERR_INVALID_ARGUMENT;
  if (T == 0) return MOE_B200_OK;
  const bool two_part = T <= kStreamTokens;
  const bool need_workspace = !hidden || two_part;
  if (!x || !w13 || !w2 || !output || (need_workspace && !workspace)) return MOE_B200_ERR_INVALID_ARGUMENT;
  if (!aligned(x, 16) || !pitch_aligned(x_pitch, 2) || !aligned(w13, 16) || !aligned(w2, 16) || !aligned(output, 16) ||
      !aligned(preact, 32) || !aligned(hidden, 16) || !aligned(workspace, 256))
    return MOE_B200_ERR_MISALIGNED;
  if (need_workspace && workspace_bytes < moe_b200_gated_ffn_workspace_bytes(T, H, I))
    return MOE_B200_ERR_WORKSPACE_TOO_SMALL;
  Device d;
  int st = open_device(&d);
  if (st != MOE_B200_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  void* h = hidden ? hidden : ws;
  void* h_lo = two_part ? ws + round256(static_cast<size_t>(T) * I * 2) : nullptr;
  DenseParams p = params(d, T, I, H, dtype, activation, h, I, dtype);
  p.preact = preact;
  p.out_lo = h_lo;
  st = forward_gemm(kEpiGated, rows_of(x, T, H, x_pitch), nullptr, rows_of(w13, 2 * I, H, H), p, d, false, s);
  if (st != MOE_B200_OK) return st;
  return forward_gemm(kEpiStore, rows_of(h, T, I, I), h_lo, rows_of(w2, H, I, I),
                      params(d, T, H, I, dtype, activation, output, H, dtype), d, true, s);
}

size_t moe_b200_gated_ffn_backward_workspace_bytes(int64_t num_tokens, int64_t hidden_size, int64_t inter_size) {
  if (!tokens_ok(num_tokens) || !dim_ok(hidden_size, 8) || !dim_ok(inter_size, 8)) return 0;
  // [du | dg], and what its rounding left
  return round256(static_cast<size_t>(num_tokens) * inter_size * 4 * (num_tokens <= kStreamTokens ? 2 : 1)) + 256;
}

int moe_b200_gated_ffn_backward(const void* grad_output, int64_t grad_pitch, const void* x, int64_t x_pitch,
                                const void* w13, const void* w2, const float* preact, const void* hidden, int dtype,
                                int activation, int64_t num_tokens, int64_t hidden_size, int64_t inter_size,
                                void* grad_x, void* grad_w13, void* grad_w2, void* workspace, size_t workspace_bytes,
                                void* stream) {
  const int64_t T = num_tokens, H = hidden_size, I = inter_size;
  if (!tokens_ok(T) || !dim_ok(H, 8) || !dim_ok(I, 8) || !type16(dtype) || !valid_act(activation) ||
      !pitch_ok(x_pitch, H) || !pitch_ok(grad_pitch, H))
    return MOE_B200_ERR_INVALID_ARGUMENT;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (T == 0) {
    // sums over no tokens
    if ((grad_w13 && cudaMemsetAsync(grad_w13, 0, static_cast<size_t>(4 * I * H), s) != cudaSuccess) ||
        (grad_w2 && cudaMemsetAsync(grad_w2, 0, static_cast<size_t>(2 * I * H), s) != cudaSuccess))
      return MOE_B200_ERR_CUDA;
    return MOE_B200_OK;
  }
  const bool need_dact = grad_x || grad_w13;
  if (!grad_output || (need_dact && (!w2 || !preact || !workspace)) || (grad_x && !w13) || (grad_w13 && !x) ||
      (grad_w2 && !hidden))
    return MOE_B200_ERR_INVALID_ARGUMENT;
  if (!aligned(grad_output, 16) || !pitch_aligned(grad_pitch, 2) || !aligned(x, 16) || !pitch_aligned(x_pitch, 2) ||
      !aligned(w13, 16) || !aligned(w2, 16) || !aligned(preact, 32) || !aligned(hidden, 16) || !aligned(grad_x, 16) ||
      !aligned(grad_w13, 16) || !aligned(grad_w2, 16) || !aligned(workspace, 256))
    return MOE_B200_ERR_MISALIGNED;
  if (need_dact && workspace_bytes < moe_b200_gated_ffn_backward_workspace_bytes(T, H, I))
    return MOE_B200_ERR_WORKSPACE_TOO_SMALL;
  Device d;
  int st = open_device(&d);
  if (st != MOE_B200_OK) return st;
  const DenseOperand dy = rows_of(grad_output, T, H, grad_pitch);
  const DenseOperand dact = rows_of(workspace, T, 2 * I, 2 * I);
  // dh = dy W2 gives [du | dg]; then dx = [du | dg] W13, dW13 = [du | dg]^T x
  // and dW2 = dy^T h.
  DenseParams p_dh = params(d, T, I, H, dtype, activation, workspace, 2 * I, dtype);
  p_dh.preact = const_cast<float*>(preact);
  const DenseProduct dh = {dy, rows_of(w2, H, I, I), false, p_dh};
  const DenseProduct dx = {dact, rows_of(w13, 2 * I, H, H), false,
                           params(d, T, H, 2 * I, dtype, activation, grad_x, H, dtype)};
  const DenseProduct dw13 = {dact, rows_of(x, T, H, x_pitch), true,
                             params(d, 2 * I, H, T, dtype, activation, grad_w13, H, dtype)};
  const DenseProduct dw2 = {dy, rows_of(hidden, T, I, I), true,
                            params(d, H, I, T, dtype, activation, grad_w2, I, dtype)};
  if (T <= kStreamTokens) {
    // the weights are streamed as in the forward pass, then written
    void* lo = need_dact ? static_cast<uint8_t*>(workspace) + static_cast<size_t>(T) * I * 4 : nullptr;
    p_dh.out_lo = lo;
    if (need_dact) st = launch_dense_skinny(kEpiBackward, dh.a, nullptr, dh.b, p_dh, d.sm_count, false, s);
    if (st == MOE_B200_OK && grad_x)
      st = launch_dense_skinny(kEpiBackward, dx.a, lo, dx.b, dx.p, d.sm_count, true, s);
    DenseProduct dw[2];
    int n = 0;
    if (grad_w13) dw[n++] = dw13;
    if (grad_w2) dw[n++] = dw2;
    if (st != MOE_B200_OK || n == 0) return st;
    return launch_dense_backward(dw, n, plan_dense_backward(dw, n, d.sm_count), d.sm_count, need_dact, s);
  }
  DenseProduct first[2], second[3];
  int n1 = 0, n2 = 0;
  if (need_dact) first[n1++] = dh;
  if (grad_x) second[n2++] = dx;
  if (grad_w13) second[n2++] = dw13;
  DensePlan plan1 = {}, plan2 = {};
  if (n1 > 0) plan1 = plan_dense_backward(first, n1, d.sm_count);
  if (n2 > 0) plan2 = plan_dense_backward(second, n2, d.sm_count);
  if (grad_w2) {
    // beside dh, or beside the others while dh has its K range split
    first[n1] = second[n2] = dw2;
    const DensePlan with1 = plan_dense_backward(first, n1 + 1, d.sm_count);
    const DensePlan with2 = n2 > 0 ? plan_dense_backward(second, n2 + 1, d.sm_count) : DensePlan{};
    if (n2 == 0 || with1.cost + plan2.cost <= plan1.cost + with2.cost) {
      plan1 = with1;
      ++n1;
    } else {
      plan2 = with2;
      ++n2;
    }
  }
  if (n1 > 0) st = launch_dense_backward(first, n1, plan1, d.sm_count, false, s);
  if (st != MOE_B200_OK || n2 == 0) return st;
  return launch_dense_backward(second, n2, plan2, d.sm_count, n1 > 0, s);
}

size_t moe_b200_mxfp4_scale_bytes(int64_t rows, int64_t cols) {
  if (!tokens_ok(rows) || !dim_ok(cols, 32)) return 0;
  return mx_scale_bytes(rows, cols);
}

int moe_b200_mxfp4_quantize(const void* x, int64_t x_pitch, int dtype, int64_t rows, int64_t cols, void* q, void* scale,
                            void* stream) {
  if (!tokens_ok(rows) || !dim_ok(cols, 32) || !any_type(dtype) || !pitch_ok(x_pitch, cols))
    return MOE_B200_ERR_INVALID_ARGUMENT;
  if (rows == 0) return MOE_B200_OK;
  if (!x || !q || !scale) return MOE_B200_ERR_INVALID_ARGUMENT;
  if (!aligned(x, 16) || !pitch_aligned(x_pitch, dtype == MOE_B200_TYPE_FP32 ? 4 : 2) || !aligned(q, 16) ||
      !aligned(scale, 16))
    return MOE_B200_ERR_MISALIGNED;
  Device d;
  const int st = open_device(&d);
  if (st != MOE_B200_OK) return st;
  return quantize(x, dtype, rows, cols, x_pitch, static_cast<uint8_t*>(q), static_cast<uint8_t*>(scale),
                  true, static_cast<cudaStream_t>(stream));
}

int moe_b200_mxfp4_dequantize(const void* q, const void* scale, int64_t rows, int64_t cols, int dtype, void* out,
                              void* stream) {
  if (!tokens_ok(rows) || !dim_ok(cols, 32) || !any_type(dtype)) return MOE_B200_ERR_INVALID_ARGUMENT;
  if (rows == 0) return MOE_B200_OK;
  if (!q || !scale || !out) return MOE_B200_ERR_INVALID_ARGUMENT;
  if (!aligned(q, 16) || !aligned(scale, 16) || !aligned(out, 16)) return MOE_B200_ERR_MISALIGNED;
  Device d;
  const int st = open_device(&d);
  if (st != MOE_B200_OK) return st;
  const int blocks = static_cast<int>(cols / 32);
  const int64_t total = rows * blocks;
  auto kern = dtype == MOE_B200_TYPE_BF16   ? mxfp4_dequantize_kernel<kTypeBf16>
              : dtype == MOE_B200_TYPE_FP16 ? mxfp4_dequantize_kernel<kTypeFp16>
                                            : mxfp4_dequantize_kernel<kTypeFp32>;
  const int vec32 = aligned(out, 32);
  return launch_kernel(kern, static_cast<unsigned>(div_up(total, 256)), 256, 0, static_cast<cudaStream_t>(stream), true,
                       static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(scale), total, blocks,
                       static_cast<int>(div_up(cols, 128)), vec32, static_cast<uint8_t*>(out)) == cudaSuccess
             ? MOE_B200_OK
             : MOE_B200_ERR_CUDA;
}

int moe_b200_mxfp4_matmul(const void* a_q, const void* a_scale, const void* b_q, const void* b_scale, int64_t m,
                          int64_t n, int64_t k, int dtype, void* out, void* stream) {
  if (!tokens_ok(m) || n < 1 || n > MOE_B200_MAX_TOKENS || !dim_ok(k, 32) || !any_type(dtype))
    return MOE_B200_ERR_INVALID_ARGUMENT;
  if (m == 0) return MOE_B200_OK;
  if (!a_q || !a_scale || !b_q || !b_scale || !out) return MOE_B200_ERR_INVALID_ARGUMENT;
  if (!aligned(a_q, 16) || !aligned(a_scale, 16) || !aligned(b_q, 16) || !aligned(b_scale, 16) || !aligned(out, 16))
    return MOE_B200_ERR_MISALIGNED;
  Device d;
  const int st = open_device(&d);
  if (st != MOE_B200_OK) return st;
  return mx_gemm(MxOperand{a_q, a_scale, m}, MxOperand{b_q, b_scale, n},
                 params(d, m, n, k, MOE_B200_TYPE_BF16, 0, out, n, dtype), d, kMxStreamTokens, false,
                 static_cast<cudaStream_t>(stream));
}

size_t moe_b200_mxfp4_linear_workspace_bytes(int64_t num_tokens, int64_t k) {
  if (!tokens_ok(num_tokens) || !dim_ok(k, 32)) return 0;
  return mx_bytes(num_tokens, k) + 256;
}

int moe_b200_mxfp4_linear(const void* x, int64_t x_pitch, int dtype, const void* w_q, const void* w_scale,
                          int64_t num_tokens, int64_t n, int64_t k, void* out, void* workspace, size_t workspace_bytes,
                          void* stream) {
  const int64_t T = num_tokens;
  if (!tokens_ok(T) || n < 1 || n > MOE_B200_MAX_TOKENS || !dim_ok(k, 32) || !any_type(dtype) || !pitch_ok(x_pitch, k))
    return MOE_B200_ERR_INVALID_ARGUMENT;
  if (T == 0) return MOE_B200_OK;
  if (!x || !w_q || !w_scale || !out || !workspace) return MOE_B200_ERR_INVALID_ARGUMENT;
  if (!aligned(x, 16) || !pitch_aligned(x_pitch, dtype == MOE_B200_TYPE_FP32 ? 4 : 2) || !aligned(w_q, 16) ||
      !aligned(w_scale, 16) || !aligned(out, 16) || !aligned(workspace, 256))
    return MOE_B200_ERR_MISALIGNED;
  if (workspace_bytes < moe_b200_mxfp4_linear_workspace_bytes(T, k)) return MOE_B200_ERR_WORKSPACE_TOO_SMALL;
  Device d;
  int st = open_device(&d);
  if (st != MOE_B200_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const MxBuffers xq = mx_place(static_cast<uint8_t*>(workspace), T, k);
  DenseParams p = params(d, T, n, k, dtype, 0, out, n, dtype);
  const bool inside = mx_skinny_quantizes(T, n, k, d.sm_count);
  st = rows_to_4_bits(x, dtype, x_pitch, xq, inside, &p, d, s);
  if (st != MOE_B200_OK) return st;
  return mx_gemm(MxOperand{xq.q, xq.scale, T}, MxOperand{w_q, w_scale, n}, p, d, kMxStreamTokens, !inside, s);
}

size_t moe_b200_mxfp4_gated_ffn_workspace_bytes(int64_t num_tokens, int64_t hidden_size, int64_t inter_size) {
  if (!tokens_ok(num_tokens) || !dim_ok(hidden_size, 32) || !dim_ok(inter_size, 32)) return 0;
  return mx_ffn_bytes(num_tokens, hidden_size, inter_size) + 256;
}

int moe_b200_mxfp4_gated_ffn(const void* x, int64_t x_pitch, int dtype, const void* w13_q, const void* w13_scale,
                             const void* w2_q, const void* w2_scale, int activation, int64_t num_tokens,
                             int64_t hidden_size, int64_t inter_size, void* output, void* workspace,
                             size_t workspace_bytes, void* stream) {
  const int64_t T = num_tokens, H = hidden_size, I = inter_size;
  if (!tokens_ok(T) || !dim_ok(H, 32) || !dim_ok(I, 32) || !any_type(dtype) || !valid_act(activation) ||
      !pitch_ok(x_pitch, H))
    return MOE_B200_ERR_INVALID_ARGUMENT;
  if (T == 0) return MOE_B200_OK;
  if (!x || !w13_q || !w13_scale || !w2_q || !w2_scale || !output || !workspace) return MOE_B200_ERR_INVALID_ARGUMENT;
  if (!aligned(x, 16) || !pitch_aligned(x_pitch, dtype == MOE_B200_TYPE_FP32 ? 4 : 2) || !aligned(w13_q, 16) ||
      !aligned(w13_scale, 16) || !aligned(w2_q, 16) || !aligned(w2_scale, 16) || !aligned(output, 16) ||
      !aligned(workspace, 256))
    return MOE_B200_ERR_MISALIGNED;
  if (workspace_bytes < moe_b200_mxfp4_gated_ffn_workspace_bytes(T, H, I)) return MOE_B200_ERR_WORKSPACE_TOO_SMALL;
  Device d;
  int st = open_device(&d);
  if (st != MOE_B200_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const MxBuffers xq = mx_place(ws, T, H);
  const MxBuffers hq = mx_place(ws + mx_bytes(T, H), T, I);
  const MxOperand xo{xq.q, xq.scale, T}, ho{hq.q, hq.scale, T};
  const MxOperand w13{w13_q, w13_scale, 2 * I}, w2{w2_q, w2_scale, H};
  if (fused_gate_quant(T, I)) {
    DenseParams p = params(d, T, I, H, dtype, activation, nullptr, 0, dtype);
    p.q = hq.q;
    p.q_scale = hq.scale;
    st = quantize(x, dtype, T, H, x_pitch, xq.q, xq.scale, quantize_early(T, H, d), s);
    if (st != MOE_B200_OK) return st;
    st = launch_mx_pair(kEpiGatedQuant, xo, w13, p, d.sm_count, true, s);
    if (st != MOE_B200_OK) return st;
    return mx_gemm(ho, w2, params(d, T, H, I, dtype, activation, output, H, dtype), d, kStreamTokens, true, s);
  }
  float* sums = reinterpret_cast<float*>(ws + mx_bytes(T, H) + mx_bytes(T, I));
  DenseParams p = params(d, T, 2 * I, H, dtype, activation, sums, 2 * I, MOE_B200_TYPE_FP32);
  const bool x_inside = mx_skinny_quantizes(T, 2 * I, H, d.sm_count);
  st = rows_to_4_bits(x, dtype, x_pitch, xq, x_inside, &p, d, s);
  if (st != MOE_B200_OK) return st;
  st = mx_gemm(xo, w13, p, d, kStreamTokens, !x_inside, s);
  if (st != MOE_B200_OK) return st;
  DenseParams p2 = params(d, T, H, I, dtype, activation, output, H, dtype);
  if (mx_skinny_quantizes(T, H, I, d.sm_count)) {
    p2.x_source = kFromSums;
    p2.x = sums;
    p2.x_pitch = 8 * I;
  } else {
    const int k_tiles = static_cast<int>(div_up(I, 128));
    if (launch_kernel(mxfp4_gate_kernel, static_cast<unsigned>(div_up(T * 4 * k_tiles, 256)), 256, 0, s, true,
                      static_cast<const float*>(sums), static_cast<int>(T), static_cast<int>(I / 32), k_tiles,
                      activation, hq.q, hq.scale) != cudaSuccess)
      return MOE_B200_ERR_CUDA;
  }
  return mx_gemm(ho, w2, p2, d, kStreamTokens, true, s);
}

int moe_b200_dense_status_address(void** address) {
  if (address == nullptr) return MOE_B200_ERR_INVALID_ARGUMENT;
  Device d;
  const int st = open_device(&d);
  if (st == MOE_B200_OK) *address = d.status;
  return st;
}

int moe_b200_dense_read_status(uint32_t* status, void* stream) {
  if (status == nullptr) return MOE_B200_ERR_INVALID_ARGUMENT;
  Device d;
  const int st = open_device(&d);
  if (st != MOE_B200_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint32_t v = 0;
  if (cudaMemcpyAsync(&v, d.status, sizeof(v), cudaMemcpyDeviceToHost, s) != cudaSuccess ||
      cudaStreamSynchronize(s) != cudaSuccess)
    return MOE_B200_ERR_CUDA;
  if (v != 0) {
    clear_status_kernel<<<1, 1, 0, s>>>(d.status, v);
    if (cudaGetLastError() != cudaSuccess || cudaStreamSynchronize(s) != cudaSuccess) return MOE_B200_ERR_CUDA;
  }
  *status = v;
  return v == 0 ? MOE_B200_OK : MOE_B200_ERR_DEVICE_TIMEOUT;
}

}  // extern "C"
