// Dense GEMMs with few rows (sm_100a): out[t, n] = sum_k x[t, k] w[n, k] for
// up to 64 tokens (a 4-bit product alone: 128), where streaming the weights is
// the whole cost.
//
// The weights take the MMA's M side (128 rows per tile) and the tokens its N
// side (16 to 128), so a handful of tokens wastes no tensor time and every
// shared-memory stage is almost all weights. K is split over a cluster of S
// CTAs (1 to 8, as many as fill the SMs), each streaming its K range through
// a ring of stages; the partial sums then meet through distributed shared
// memory, the CTAs sharing out the output and adding the S parts in a fixed
// order. Nothing is accumulated with atomics, so results do not depend on
// timing.
//
// Gated form (16-bit): the tile's 128 rows are 64 up rows and the 64 gate
// rows of the same features, and the adding threads apply the activation.
//
// Backward form (16-bit): the weights are stored K x N, as dh = dy W2 and dx =
// [du | dg] W13 read them; the descriptor takes them so, and the adding
// threads of dh compute du and dg, in two parts like the hidden (gradients at
// 16 tokens, H = 7168, I = 2048, against CTA pairs: 53 -> 50 us, of x alone 34
// -> 22; H = 2048, I = 1024 21 -> 17; at 64 tokens 55 -> 57, 38 -> 29 and 22
// -> 22).
//
// The 16-bit block keeps its hidden (and [du | dg] for dx) in two 16-bit
// numbers, h rounded and what that left, rounded again (times a factor that
// keeps it in range, rest_scale): the second product takes both as
// neighbouring token tiles of one MMA (N = 2 x 16 to 2 x 64) and their sums
// are added with the parts. The result then carries one rounding instead of
// two. Up to 32 tokens this is free, the tokens being next to nothing beside
// the weights; at 64 it costs 3 % (25.6 -> 26.4 us).
//
// 4-bit, up to four tokens: the kernel brings its token operand to 4 bits
// itself, from x or from the fp32 up and gate sums of the GEMM before. Each
// CTA needs only its K range, a few KB, so that every cluster repeats the same
// quantisation costs less than a kernel of its own in between (one token, 4096
// x 7168: 9.2 -> 8.7 us, the block 16.0 -> 14.9 us and one and two launches
// less; equal at four tokens, slower from eight: 10.1 against 11.8 us).
//
// Two GEMMs of a call overlap (programmatic dependent launch): weights are
// inputs of the whole call, so the second kernel requests its first ring of
// weight tiles before it waits for the first; only the token operand comes
// from that. It is let go when its predecessor requests its own
// last ring, so HBM does not idle under the first one's tail. (Asking for the
// rest of the K range into L2 as well was no faster.)
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "../../include/moe_b200.h"
#include "dense_gemm.h"
#include "dense_ptx.cuh"
#include "ffn_math.cuh"
#include "host_common.h"
#include "moe_kernels.cuh"
#include "mxfp4.cuh"

namespace moe {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxStages = 12;
constexpr int kWeightTile = 16384;             // 128 rows of 128 bytes
constexpr int kHeader = 1024;                  // barriers
constexpr int kSmemSmall = 110 * 1024;         // stages and staged tokens: two CTAs per SM
constexpr int kSmemLarge = 224 * 1024;
constexpr int kExtra = kHeader + 1024;         // + alignment
static_assert(kSmemLarge + kExtra <= 227 * 1024, "shared memory");
static_assert(2 * (kSmemSmall + kExtra + 1024) <= 228 * 1024, "two CTAs per SM");
constexpr int kQuantWarps = 6;                 // warps 2..7 bring x to 4 bits
constexpr int kQuantMaxRows = 4;
constexpr int kQuantMaxBytes = 48 * 1024;

struct SkinnyShape {
  int bn;            // the tokens, rounded up to a multiple of 16 (at most 128)
  int x_rows;        // rows of a staged token tile: bn, or 2 bn of a two-part operand
  int splits;        // CTAs per cluster
  int stages;
  int stage_bytes;
  int xq_off;        // staged 4-bit tokens, after the ring
  int xq_iters;      // most K steps of a CTA
  int tmem_cols;
  int smem_bytes;
};

// Brings blocks of 32 columns of the CTA's K range to 4 bits, into shared
// memory in the layout of the token operand. Four threads hold a block, eight
// columns each; the loads of a batch of blocks are issued together.
template <int kSrc, int kType>
__device__ __forceinline__ void stage_tokens(const DenseParams& p, const SkinnyShape& sh, uint8_t* codes,
                                             uint8_t* exponents, int live, int kb0, int iters, int tid) {
  constexpr int kBatch = kType == kTypeFp32 ? 2 : 4;
  const int chunks = iters * 32;               // of eight columns per row; past K: zero codes and exponents
  const int k_chunks = p.k >> 3;
  const int total = live * chunks;             // a multiple of 32: whole warps
  for (int e0 = tid; e0 < total; e0 += kBatch * kQuantWarps * 32) {
    float v[kBatch][8];
    int row[kBatch], at[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int e = e0 + i * kQuantWarps * 32;
      row[i] = e / chunks;
      at[i] = e - row[i] * chunks;
      const int c = kb0 * 32 + at[i];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
      if (e < total && c < k_chunks) {
        const uint8_t* src = static_cast<const uint8_t*>(p.x) + row[i] * p.x_pitch;
        if constexpr (kType == kTypeFp32) {
          const float4* f = reinterpret_cast<const float4*>(src + static_cast<int64_t>(c) * 32);
          const float4 lo = f[0], hi = f[1];
          v[i][0] = lo.x, v[i][1] = lo.y, v[i][2] = lo.z, v[i][3] = lo.w;
          v[i][4] = hi.x, v[i][5] = hi.y, v[i][6] = hi.z, v[i][7] = hi.w;
          if constexpr (kSrc == kFromSums) {
            const float4* g = reinterpret_cast<const float4*>(src + static_cast<int64_t>(p.k) * 4 +
                                                              static_cast<int64_t>(c) * 32);
            const float4 gl = g[0], gh = g[1];
            v[i][0] *= act_value(gl.x, p.act), v[i][1] *= act_value(gl.y, p.act);
            v[i][2] *= act_value(gl.z, p.act), v[i][3] *= act_value(gl.w, p.act);
            v[i][4] *= act_value(gh.x, p.act), v[i][5] *= act_value(gh.y, p.act);
            v[i][6] *= act_value(gh.z, p.act), v[i][7] *= act_value(gh.w, p.act);
          }
        } else {
          const uint4 q = *reinterpret_cast<const uint4*>(src + static_cast<int64_t>(c) * 16);
          const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = unpack_16(w[j], kType);
            v[i][2 * j] = f.x;
            v[i][2 * j + 1] = f.y;
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (e0 + i * kQuantWarps * 32 >= total) break;   // the same for a whole warp
      uint32_t amax = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(v[i][j]) & 0x7fffffffu);
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const uint32_t byte = mx_exponent(amax);
      const int b = at[i] >> 2;                        // block of the CTA's range
      const int r = row[i];
      // the 128-byte swizzle: 16-byte piece c of row r lies at c ^ (r % 8)
      uint8_t* dst = codes + (b >> 3) * (sh.bn * 128) + r * 128 + (((b & 7) ^ (r & 7)) << 4) + (at[i] & 3) * 4;
      *reinterpret_cast<uint32_t*>(dst) = byte == 255u ? 0u : mx_pack8(v[i], mx_inverse(byte));
      if ((at[i] & 3) == 0) exponents[(b >> 2) * 512 + r * 16 + (b & 3)] = static_cast<uint8_t>(byte);
    }
  }
}

// [du | dg] of four columns and a token, in two parts, from dh and the saved
// u and g (`pre`).
__device__ __forceinline__ void store_dact(const DenseParams& p, const float* pre, int64_t at, const float4& dh) {
  const float4 u = *reinterpret_cast<const float4*>(pre);
  const float4 g = *reinterpret_cast<const float4*>(pre + p.n);
  const float d[4] = {dh.x, dh.y, dh.z, dh.w}, up[4] = {u.x, u.y, u.z, u.w}, gate[4] = {g.x, g.y, g.z, g.w};
  float v[2][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float value, slope;
    act_value_slope(gate[j], p.act, value, slope);
    v[0][j] = d[j] * value;
    v[1][j] = d[j] * up[j] * slope;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint2 hi = make_uint2(pack_16(v[i][0], v[i][1], p.type), pack_16(v[i][2], v[i][3], p.type));
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at + i * p.n) = hi;
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out_lo) + at + i * p.n) =
        make_uint2(pack_rest_16(v[i][0], v[i][1], hi.x, p.type), pack_rest_16(v[i][2], v[i][3], hi.y, p.type));
  }
}

}  // namespace

template <bool kMx, int kEpi, int kSrc>
__global__ void __launch_bounds__(kThreads)
    dense_skinny_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                        const __grid_constant__ CUtensorMap tm_sfw, const __grid_constant__ CUtensorMap tm_sfx,
                        const DenseParams p, const SkinnyShape sh) {
  constexpr bool kGate = kEpi == kEpiGated;
  constexpr bool kWMn = kEpi == kEpiBackward;  // weights stored K x N
  constexpr bool kQuantX = kSrc != kFromMatrix;
  constexpr int kUnit = kGate ? 64 : 128;      // features per cluster
  static_assert(!(kMx && kGate) && (kMx || !kQuantX), "");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* header = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~static_cast<uintptr_t>(1023));
  uint8_t* smem = header + kHeader;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(header);
  uint64_t* empty_bar = full_bar + kMaxStages;
  uint64_t* done_bar = empty_bar + kMaxStages;
  uint64_t* xq_bar = done_bar + 1;             // the staged 4-bit tokens are there
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(xq_bar + 1);
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_cta_rank());
  const int n0 = static_cast<int>(blockIdx.x) / sh.splits * kUnit;   // first feature of the tile
  const int kb0 = static_cast<int>(static_cast<int64_t>(p.k_iters) * rank / sh.splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(p.k_iters) * (rank + 1) / sh.splits);
  const int iters = kb1 - kb0;
  const int live = static_cast<int>(p.m);      // tokens, at most sh.bn
  const int x_bytes = kQuantX ? 0 : sh.x_rows * 128;                        // of a stage

  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_x);
    for (int s = 0; s < sh.stages; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 1);
      mbar_init(smem_u32(&empty_bar[s]), 1);
    }
    mbar_init(smem_u32(done_bar), 1);
    mbar_init(smem_u32(xq_bar), kQuantWarps);
    *s_abort = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 2) {
    tmem_alloc(smem_u32(s_tmem), static_cast<uint32_t>(sh.tmem_cols));
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  if (warp != 0) pdl_wait();   // no bounded wait starts before the predecessor is done

  if (warp == 0) {
    // ---------------------------------------------------------- producer
    const bool issue = elect_lane();
    const uint32_t bytes = kWeightTile + x_bytes + (kMx ? (kQuantX ? 1024 : 2048) : 0);
    const int kt = kMx ? (p.k + 127) >> 7 : 0;
    const uint32_t base = smem_u32(smem);
    const uint32_t full0 = smem_u32(full_bar);
    // A stage: weights, tokens, then exponents of both.
    auto load_w = [&](int i, int stage) {
      const uint32_t bar = full0 + 8u * stage;
      const uint32_t sw = base + stage * sh.stage_bytes;
      const int x = (kb0 + i) * (kMx ? 128 : 64);
      mbar_arrive_expect_tx(bar, bytes);
      if constexpr (kMx) {
        tma_load_2d(sw, &tm_w, bar, x, n0);
        tma_load_2d(sw + kWeightTile + x_bytes, &tm_sfw, bar, 0, (n0 >> 7) * kt + 2 * (kb0 + i));
      } else if constexpr (kWMn) {
        tma_load_2d(sw, &tm_w, bar, n0, x);
        tma_load_2d(sw + kWeightTile / 2, &tm_w, bar, n0 + 64, x);
      } else {
        tma_load_2d(sw, &tm_w, bar, x, n0);
        tma_load_2d(sw + kWeightTile / 2, &tm_w, bar, x, n0 + (kGate ? p.n : 64));
      }
    };
    auto load_x = [&](int i, int stage) {
      if (kQuantX) return;
      const uint32_t bar = full0 + 8u * stage;
      const uint32_t sx = base + stage * sh.stage_bytes + kWeightTile;
      tma_load_2d(sx, &tm_x, bar, (kb0 + i) * (kMx ? 128 : 64), 0);
      if (!kMx && sh.x_rows != sh.bn) tma_load_2d(sx + sh.bn * 128, &tm_sfx, bar, (kb0 + i) * 64, 0);
      if (kMx) tma_load_2d(sx + x_bytes + 1024, &tm_sfx, bar, 0, 2 * (kb0 + i));
    };
    const int first = min(sh.stages, iters);
    // The next kernel of the call may start once this CTA requests its last
    // ring (25.5 us for the block at one token; 26.3 released at the start).
    const int release = max(iters - sh.stages, 0);
    if (issue && p.early)
      for (int i = 0; i < first; ++i) load_w(i, i);
    __syncwarp();
    pdl_wait();
    if (release < first) pdl_launch_next();
    if (issue)
      for (int i = 0; i < first; ++i) {
        if (!p.early) load_w(i, i);
        load_x(i, i);
      }
    __syncwarp();
    int stage = first == sh.stages ? 0 : first;
    uint32_t ph = 0;
    bool ok = true;
    for (int i = first; i < iters; ++i) {
      ok = warp_wait(smem_u32(empty_bar) + 8u * stage, ph, s_abort, p.status, kStatusTimeoutProducer);
      if (!ok) break;
      if (issue) {
        load_w(i, stage);
        load_x(i, stage);
      }
      if (i == release) pdl_launch_next();
      __syncwarp();
      if (++stage == sh.stages) {
        stage = 0;
        ph ^= 1u;
      }
    }
    // The last ring's stages are handed back too: no arrival may still be on
    // its way to this CTA's shared memory when it leaves.
    for (int i = iters - first; ok && i < iters; ++i)
      ok = warp_wait(smem_u32(empty_bar) + 8u * (i % sh.stages), (i / sh.stages) & 1, s_abort, p.status,
                     kStatusTimeoutProducer);
    if (!ok) drain_copies();
  } else if (warp == 1) {
    // --------------------------------------------------------------- MMA
    const bool issue = elect_lane();
    const uint32_t idesc0 = kMx ? idesc_mxf4(128, sh.bn, 0) : idesc_f16(128, sh.x_rows, p.type == kTypeFp16, kWMn, false);
    const uint32_t idesc1 = kMx ? idesc_mxf4(128, sh.bn, 2) : idesc0;
    const uint32_t base = smem_u32(smem);
    const uint32_t lo_w0 = kWMn ? desc_lo_mnmajor(base) : desc_lo_kmajor(base);
    const uint32_t lo_s0 = desc_lo_scale(base + kWeightTile + x_bytes);
    const uint32_t lo_x0 = desc_lo_kmajor(base + (kQuantX ? sh.xq_off : kWeightTile));
    const uint32_t lo_sx0 = kQuantX ? desc_lo_scale(base + sh.xq_off + sh.xq_iters * sh.bn * 128)
                                    : lo_s0 + 64;
    int stage = 0;
    uint32_t ph = 0;
    bool ok = !kQuantX || warp_wait(smem_u32(xq_bar), 0, s_abort, p.status, kStatusTimeoutMma);
    for (int i = 0; ok && i < iters; ++i) {
      if (!warp_wait(smem_u32(full_bar) + 8u * stage, ph, s_abort, p.status, kStatusTimeoutMma)) break;
      const uint32_t off = static_cast<uint32_t>(stage * (sh.stage_bytes >> 4));
      const uint32_t lo_w = lo_w0 + off;
      const uint32_t lo_x = lo_x0 + (kQuantX ? static_cast<uint32_t>(i * sh.bn * 8) : off);
      tc_fence_after();
      if (issue) {
        if constexpr (kMx) {
          const uint32_t lo_s = lo_s0 + off;
          const uint32_t lo_sx = lo_sx0 + (kQuantX ? static_cast<uint32_t>(i * 64) : off);
          // each stage has its own exponent columns: a stage that is full
          // again has been read
          const uint32_t sfw = tmem + sh.bn + 16 * stage;
          const uint32_t sfx = sfw + 8;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            tmem_copy_scales<1>(sfw + 4 * j, desc_of(kDescHiPlain, lo_s + 32 * j));
            tmem_copy_scales<1>(sfx + 4 * j, desc_of(kDescHiPlain, lo_sx + 32 * j));
          }
          const int left = p.k - (kb0 + i) * 256;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (k == 0 || left > 64 * k)
              umma_mxf4<1>(tmem, desc_of(kDescHiSw128, lo_w + 2 * k), desc_of(kDescHiSw128, lo_x + 2 * k),
                           k & 1 ? idesc1 : idesc0, sfw + 4 * (k >> 1), sfx + 4 * (k >> 1), i | k);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16<1>(tmem, desc_of(kDescHiSw128, lo_w + (kWMn ? 128 : 2) * k), desc_of(kDescHiSw128, lo_x + 2 * k), idesc0, i | k);
        }
        umma_commit(smem_u32(empty_bar) + 8u * stage);
        if (i == iters - 1) umma_commit(smem_u32(done_bar));
      }
      __syncwarp();
      if (++stage == sh.stages) {
        stage = 0;
        ph ^= 1u;
      }
    }
  } else if constexpr (kQuantX) {
    uint8_t* codes = smem + sh.xq_off;
    uint8_t* exponents = codes + sh.xq_iters * sh.bn * 128;
    const int tid = static_cast<int>(threadIdx.x) - 64;
    if (kSrc == kFromSums || p.type == kTypeFp32)
      stage_tokens<kSrc, kTypeFp32>(p, sh, codes, exponents, live, kb0, iters, tid);
    else if (p.type == kTypeBf16)
      stage_tokens<kSrc, kTypeBf16>(p, sh, codes, exponents, live, kb0, iters, tid);
    else
      stage_tokens<kSrc, kTypeFp16>(p, sh, codes, exponents, live, kb0, iters, tid);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(xq_bar));
  }

  // ------------------------------------- partial sums into shared memory
  const bool ready = mbar_wait(smem_u32(done_bar), 0, s_abort, p.status, kStatusTimeoutEpilogue);
  const bool all_ready = __syncthreads_and(ready);
  float* red = reinterpret_cast<float*>(smem);   // [row / 4][token][4], over the drained stages
  const int pitch = 4 * (sh.bn + 1);             // odd in 16 bytes: neighbouring rows in different banks
  if (all_ready) {
    tc_fence_after();
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const int row = (warp & 3) * 32 + lane;
    const float unscale = rest_unscale(p.type);
    for (int c = 16 * (warp >> 2); c < sh.bn; c += 32) {   // every other 16 tokens
      uint32_t r[16];
      tmem_ld16(lanes + c, r);
      tmem_wait_ld();
      if (!kMx && sh.x_rows != sh.bn) {   // a two-part operand: both parts' sums
        uint32_t lo[16];
        tmem_ld16(lanes + sh.bn + c, lo);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(fmaf(__uint_as_float(lo[j]), unscale, __uint_as_float(r[j])));
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) red[(row >> 2) * pitch + 4 * (c + j) + (row & 3)] = __uint_as_float(r[j]);
    }
  }
  cluster_sync();

  // --------------------------- this CTA's share of the output, all parts
  if (all_ready) {
    const uint32_t red_addr = smem_u32(red);
    uint32_t part[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) part[q] = q < sh.splits ? map_to_cta(red_addr, (rank + q) & (sh.splits - 1)) : 0u;
    // Sums of four neighbouring rows of token t, parts in a fixed order: this
    // CTA's first, so that the CTAs do not all read from one at a time.
    auto sums = [&](int t, int row) {
      float4 a[8];
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q < sh.splits) a[q] = ld_cluster_f32x4(part[q] + ((row >> 2) * pitch + 4 * t) * 4);
      float4 v = a[0];
#pragma unroll
      for (int q = 1; q < 8; ++q)
        if (q < sh.splits) v.x += a[q].x, v.y += a[q].y, v.z += a[q].z, v.w += a[q].w;
      return v;
    };
    const int share = kUnit / sh.splits;
    // A thread adds four columns of a token; the threads of a warp take
    // neighbouring tokens, whose parts lie side by side (with a token's columns
    // side by side instead, 64 tokens took 27.4 against 25.7 us; at 128 that
    // order was 1 % faster).
    for (int i = static_cast<int>(threadIdx.x); i < share / 4 * sh.bn; i += kThreads) {
      const int t = i % sh.bn;
      const int f = rank * share + i / sh.bn * 4;   // first of the four features in the tile
      if (t < live && n0 + f < p.n) {
        float4 sum = sums(t, f);
        const int64_t row = t;
        if (kGate) {
          const float4 gate = sums(t, 64 + f);
          if (p.preact != nullptr) {
            float* pre = p.preact + row * (2 * static_cast<int64_t>(p.n)) + n0 + f;
            *reinterpret_cast<float4*>(pre) = sum;
            *reinterpret_cast<float4*>(pre + p.n) = gate;
          }
          sum.x *= act_value(gate.x, p.act), sum.y *= act_value(gate.y, p.act);
          sum.z *= act_value(gate.z, p.act), sum.w *= act_value(gate.w, p.act);
        }
        const int64_t at = row * p.ldo + n0 + f;
        if (kWMn && p.preact != nullptr) {
          store_dact(p, p.preact + row * (2 * static_cast<int64_t>(p.n)) + n0 + f, at, sum);
        } else if (p.out_type == kTypeFp32) {
          float* out = static_cast<float*>(p.out) + at;
          if (p.vec32) {
            *reinterpret_cast<float4*>(out) = sum;
          } else {
            out[0] = sum.x;
            if (n0 + f + 1 < p.n) out[1] = sum.y;
            if (n0 + f + 2 < p.n) out[2] = sum.z;
            if (n0 + f + 3 < p.n) out[3] = sum.w;
          }
        } else {
          const uint2 v = make_uint2(pack_16(sum.x, sum.y, p.out_type), pack_16(sum.z, sum.w, p.out_type));
          uint16_t* out = static_cast<uint16_t*>(p.out) + at;
          if (kGate && p.out_lo != nullptr) {
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out_lo) + at) =
                make_uint2(pack_rest_16(sum.x, sum.y, v.x, p.out_type), pack_rest_16(sum.z, sum.w, v.y, p.out_type));
          }
          if (p.vec32) {
            *reinterpret_cast<uint2*>(out) = v;
          } else {
            out[0] = static_cast<uint16_t>(v.x);
            if (n0 + f + 1 < p.n) out[1] = static_cast<uint16_t>(v.x >> 16);
            if (n0 + f + 2 < p.n) out[2] = static_cast<uint16_t>(v.y);
            if (n0 + f + 3 < p.n) out[3] = static_cast<uint16_t>(v.y >> 16);
          }
        }
      }
    }
  }
  tc_fence_before();
  cluster_sync_relaxed();   // the others have read this CTA's part
  tc_fence_after();
  if (warp == 2) tmem_dealloc(tmem, static_cast<uint32_t>(sh.tmem_cols));
}

namespace {

template <bool kMx, int kEpi, int kSrc>
int launch_skinny(const CUtensorMap& w, const CUtensorMap& x, const CUtensorMap& sfw, const CUtensorMap& sfx,
                  DenseParams p, const SkinnyShape& sh, int units, bool dependent, cudaStream_t s) {
  p.early = dependent;
  auto kern = dense_skinny_kernel<kMx, kEpi, kSrc>;
  static OncePerDevice ready;
  if (!ready([&] {
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLarge + kExtra) ==
               cudaSuccess;
      }))
    return MOE_B200_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(units * sh.splits));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sh.smem_bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(sh.splits);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, w, x, sfw, sfx, p, sh) == cudaSuccess ? MOE_B200_OK : MOE_B200_ERR_CUDA;
}


// K parts: a power of two up to 8, at most one per K step, as many as keep
// the grid within one CTA per SM; up to 64 tokens within two per SM while a
// CTA keeps eight steps (block at one token 24.3 -> 21.9 us; at 128 tokens
// the larger stages leave no room for two, and shorter K ranges spend their
// time adding: 4-bit linear at 64 tokens 11.4 -> 12.7 us).
// Shared memory: a small allocation leaves room for a second CTA, of this
// grid or of the call's next kernel, whose first weights then stream under
// this one's tail (27.5 -> 25.5 us).
SkinnyShape choose_shape(const DenseParams& p, bool mx, bool gate, bool quant_x, int sm_count, bool two_part = false) {
  SkinnyShape sh;
  sh.bn = static_cast<int>(div_up(p.m, 16) * 16);
  sh.x_rows = two_part ? 2 * sh.bn : sh.bn;
  const int64_t ctas = div_up(p.n, gate ? 64 : 128);
  sh.splits = 1;
  while (sh.splits < 8 && 2 * sh.splits <= p.k_iters) {
    const int next = 2 * sh.splits;
    const int per_sm = sh.bn <= 64 && p.k_iters >= 8 * next ? 2 : 1;
    if (next * ctas > static_cast<int64_t>(per_sm) * sm_count) break;
    sh.splits = next;
  }
  sh.xq_iters = quant_x ? static_cast<int>(div_up(p.k_iters, sh.splits)) : 0;
  const int xq_bytes = sh.xq_iters * (sh.bn * 128 + 1024);
  sh.stage_bytes = kWeightTile + (quant_x ? 0 : sh.x_rows * 128) + (mx ? (quant_x ? 1024 : 2048) : 0);
  const int room = (sh.bn <= 64 ? kSmemSmall : kSmemLarge) - xq_bytes;
  sh.stages = room / sh.stage_bytes;
  const int most = static_cast<int>(div_up(p.k_iters, sh.splits));
  if (sh.stages > most) sh.stages = most;
  if (sh.stages > kMaxStages) sh.stages = kMaxStages;
  if (sh.stages < 2) sh.stages = 2;
  sh.xq_off = sh.stages * sh.stage_bytes;
  int bytes = sh.xq_off + xq_bytes;
  const int red = (sh.bn + 1) * 512;           // the partial sums reuse the stages
  if (bytes < red) bytes = red;
  const int cols = sh.x_rows + (mx ? 16 * sh.stages : 0);   // at most 128 + 6 * 16 or 64 + 12 * 16
  sh.tmem_cols = 32;
  while (sh.tmem_cols < cols) sh.tmem_cols *= 2;
  // At least the share of the SM's shared memory that its tensor memory is of
  // the 512 columns: CTAs that fit an SM together then always find their
  // columns free. Clusters whose CTAs held columns on one SM and waited for
  // them on another could otherwise wait for each other.
  const int least = sh.tmem_cols * (228 * 1024 / 512) - 1024;
  sh.smem_bytes = bytes + kExtra < least ? least : bytes + kExtra;
  return sh;
}

}  // namespace

int launch_dense_skinny(DenseEpi epi, const DenseOperand& a, const void* a_lo, const DenseOperand& b, DenseParams p,
                        int sm_count, bool dependent, cudaStream_t s) {
  const bool gate = epi == kEpiGated;
  p.k_iters = static_cast<int>(div_up(p.k, 64));
  p.vec32 = 1;   // four columns at a time: n and ldo are multiples of 8
  const SkinnyShape sh = choose_shape(p, false, gate, false, sm_count, a_lo != nullptr);
  const int units = static_cast<int>(div_up(p.n, gate ? 64 : 128));
  CUtensorMap tw, tx, tlo;
  if (!encode_2d(&tw, b.base, 2, b.cols, b.rows, b.pitch, 64, 64) ||
      !encode_2d(&tx, a.base, 2, a.cols, a.rows, a.pitch, 64, sh.bn) ||
      !encode_2d(&tlo, a_lo != nullptr ? a_lo : a.base, 2, a.cols, a.rows, a.pitch, 64, sh.bn))
    return MOE_B200_ERR_DRIVER;
  if (epi == kEpiBackward)
    return launch_skinny<false, kEpiBackward, kFromMatrix>(tw, tx, tw, tlo, p, sh, units, dependent, s);
  return gate ? launch_skinny<false, kEpiGated, kFromMatrix>(tw, tx, tw, tlo, p, sh, units, dependent, s)
              : launch_skinny<false, kEpiStore, kFromMatrix>(tw, tx, tw, tlo, p, sh, units, dependent, s);
}

// Up to kQuantMaxRows tokens, while the staged tokens of a CTA's K range leave room
// for the stages.
bool mx_skinny_quantizes(int64_t m, int64_t n, int64_t k, int sm_count) {
  if (m > kQuantMaxRows) return false;
  DenseParams p;
  std::memset(&p, 0, sizeof(p));
  p.m = m;
  p.n = static_cast<int>(n);
  p.k = static_cast<int>(k);
  p.k_iters = static_cast<int>(div_up(k, 256));
  const SkinnyShape sh = choose_shape(p, true, false, true, sm_count);
  return sh.xq_iters * (sh.bn * 128 + 1024) <= kQuantMaxBytes;
}

int launch_mx_skinny(const MxOperand& a, const MxOperand& b, DenseParams p, int sm_count, bool dependent,
                     cudaStream_t s) {
  p.k_iters = static_cast<int>(div_up(p.k, 256));
  p.vec32 = p.n % 4 == 0 && p.ldo % 4 == 0;   // four columns at a time
  const SkinnyShape sh = choose_shape(p, true, false, p.x_source != kFromMatrix, sm_count);
  const int units = static_cast<int>(div_up(p.n, 128));
  const int64_t kt = div_up(p.k, 128);
  CUtensorMap tw, tx, tsw, tsx;
  if (!encode_2d(&tw, b.q, 1, p.k / 2, b.rows, p.k / 2, 128, 128) ||
      !encode_2d(&tsw, b.scale, 2, 256, div_up(b.rows, 128) * kt, 512, 256, 2, false))
    return MOE_B200_ERR_DRIVER;
  if (p.x_source == kFromRows)
    return launch_skinny<true, kEpiStore, kFromRows>(tw, tw, tsw, tsw, p, sh, units, dependent, s);
  if (p.x_source == kFromSums)
    return launch_skinny<true, kEpiStore, kFromSums>(tw, tw, tsw, tsw, p, sh, units, dependent, s);
  if (!encode_2d(&tx, a.q, 1, p.k / 2, a.rows, p.k / 2, 128, sh.bn) ||
      !encode_2d(&tsx, a.scale, 2, 256, div_up(a.rows, 128) * kt, 512, 256, 2, false))
    return MOE_B200_ERR_DRIVER;
  return launch_skinny<true, kEpiStore, kFromMatrix>(tw, tx, tsw, tsx, p, sh, units, dependent, s);
}

}  // namespace moe
