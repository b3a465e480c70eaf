// Dense GEMMs with few rows (sm_100a): out[t, n] = sum_k x[t, k] w[n, k] for
// up to 128 tokens per tile, where streaming the weights is the whole cost.
//
// The weights take the MMA's M side (128 rows per tile) and the tokens its N
// side (16 to 128), so a handful of tokens wastes no tensor time and every
// shared-memory stage is almost all weights. K is split over a cluster of S
// CTAs (1 to 8, as many as fill the SMs), each streaming its K range through
// a ring of about 200 KB; the partial sums then meet through distributed
// shared memory, CTA r adding the S parts of its 128 / S output columns in
// CTA order. Nothing is accumulated with atomics, so results do not depend
// on timing.
//
// Gated form: the tile's 128 rows are 64 up rows and the 64 gate rows of the
// same features, and the adding thread applies the activation.
//
// Two GEMMs of a call overlap (programmatic dependent launch): weights are
// inputs of the whole call, so a kernel requests its first ring of weight
// tiles before it waits for its predecessor; only the token operand comes
// from the kernel before. It is let go when its predecessor requests its own
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

namespace moe {

namespace {

constexpr int kSkinnyThreads = 128;
constexpr int kMaxStages = 12;
constexpr int kWeightTile = 16384;             // 128 rows of 128 bytes
constexpr int kRingSmall = 108 * 1024;          // two CTAs per SM
constexpr int kRingLarge = 212 * 1024;
constexpr int kSkinnyExtra = (2 * kMaxStages + 1) * 8 + 16 + 1024;
static_assert(kRingLarge + kSkinnyExtra <= 227 * 1024, "shared memory");
static_assert(2 * (kRingSmall + kSkinnyExtra + 1024) <= 228 * 1024, "two CTAs per SM");

struct SkinnyShape {
  int bn;            // tokens per tile (multiple of 16)
  int splits;        // CTAs per cluster
  int stages;
  int stage_bytes;
  int ring_bytes;
};

}  // namespace

template <bool kMx, bool kGate>
__global__ void __launch_bounds__(kSkinnyThreads, 1)
    dense_skinny_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                        const __grid_constant__ CUtensorMap tm_sfw, const __grid_constant__ CUtensorMap tm_sfx,
                        const DenseParams p, const SkinnyShape sh) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + sh.ring_bytes);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + kMaxStages;
  uint64_t* done_bar = bars + 2 * kMaxStages;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(done_bar + 1);
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
  constexpr uint32_t kCols = kMx ? 256 : 128;   // accumulator, then (4-bit) two exponent buffers of 16 columns

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_cta_rank());
  const int n0 = static_cast<int>(blockIdx.x) / sh.splits * (kGate ? 64 : 128);   // first feature of the tile
  const int t0 = static_cast<int>(blockIdx.y) * sh.bn;
  const int kb0 = static_cast<int>(static_cast<int64_t>(p.k_iters) * rank / sh.splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(p.k_iters) * (rank + 1) / sh.splits);
  const int iters = kb1 - kb0;

  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_x);
    for (int s = 0; s < sh.stages; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 1);
      mbar_init(smem_u32(&empty_bar[s]), 1);
    }
    mbar_init(smem_u32(done_bar), 1);
    *s_abort = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 2) {
    tmem_alloc(smem_u32(s_tmem), kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  if (warp != 0) pdl_wait();   // no bounded wait starts before the predecessor is done

  if (warp == 0) {
    const bool issue = elect_lane();
    const uint32_t bytes = kWeightTile + sh.bn * 128 + (kMx ? 2048 : 0);
    const int kt = kMx ? (p.k + 127) >> 7 : 0;
    const uint32_t base = smem_u32(smem);
    const uint32_t full0 = smem_u32(full_bar);
    // Stage i of this CTA: weights (and their exponents), and tokens.
    auto load_w = [&](int i, int stage) {
      const uint32_t bar = full0 + 8u * stage;
      const uint32_t sw = base + stage * sh.stage_bytes;
      const int x = (kb0 + i) * (kMx ? 128 : 64);
      mbar_arrive_expect_tx(bar, bytes);
      tma_load_2d(sw, &tm_w, bar, x, n0);
      tma_load_2d(sw + kWeightTile / 2, &tm_w, bar, x, n0 + (kGate ? p.n : 64));
      if (kMx) tma_load_2d(sw + kWeightTile + sh.bn * 128, &tm_sfw, bar, 0, (n0 >> 7) * kt + 2 * (kb0 + i));
    };
    auto load_x = [&](int i, int stage) {
      const uint32_t bar = full0 + 8u * stage;
      const uint32_t sx = base + stage * sh.stage_bytes + kWeightTile;
      tma_load_2d(sx, &tm_x, bar, (kb0 + i) * (kMx ? 128 : 64), t0);
      if (kMx) tma_load_2d(sx + sh.bn * 128 + 1024, &tm_sfx, bar, 0, (t0 >> 7) * kt + 2 * (kb0 + i));
    };
    const int first = min(sh.stages, iters);
    // The next kernel of the call may start once this CTA requests its last
    // ring (25.5 us for the block at one token; 26.3 released at the start).
    const int release = max(iters - sh.stages, 0);
    if (issue)
      for (int i = 0; i < first; ++i) load_w(i, i);
    if (release < first) pdl_launch_next();
    __syncwarp();
    pdl_wait();
    if (issue)
      for (int i = 0; i < first; ++i) load_x(i, i);
    __syncwarp();
    int stage = first == sh.stages ? 0 : first;
    uint32_t ph = 0;
    for (int i = first; i < iters; ++i) {
      if (!warp_wait(smem_u32(empty_bar) + 8u * stage, ph, s_abort, p.status, kStatusTimeoutProducer)) {
        drain_copies();
        break;
      }
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
  } else if (warp == 1) {
    const bool issue = elect_lane();
    const uint32_t idesc0 = kMx ? idesc_mxf4(128, sh.bn, 0) : idesc_f16(128, sh.bn, p.type == kTypeFp16, false, false);
    const uint32_t idesc1 = kMx ? idesc_mxf4(128, sh.bn, 2) : idesc0;
    const uint32_t lo_w0 = desc_lo_kmajor(smem_u32(smem));
    const uint32_t lo_x0 = lo_w0 + (kWeightTile >> 4);
    const uint32_t lo_s0 = desc_lo_scale(smem_u32(smem) + kWeightTile + sh.bn * 128);
    int stage = 0, old = sh.stages - 2;   // 4-bit: the stage before last, and its phase
    uint32_t ph = 0, old_ph = 1, sf = 0;
    for (int i = 0; i < iters; ++i) {
      if (!warp_wait(smem_u32(full_bar) + 8u * stage, ph, s_abort, p.status, kStatusTimeoutMma)) break;
      const uint32_t off = static_cast<uint32_t>(stage * (sh.stage_bytes >> 4));
      const uint32_t lo_w = lo_w0 + off, lo_x = lo_x0 + off;
      if constexpr (kMx) {
        // these exponent columns were last read two stages ago (the first
        // two waits pass at once)
        if (!warp_wait(smem_u32(empty_bar) + 8u * old, old_ph, s_abort, p.status, kStatusTimeoutMma)) break;
        if (++old == sh.stages) {
          old = 0;
          old_ph ^= 1u;
        }
      }
      tc_fence_after();
      if (issue) {
        if constexpr (kMx) {
          const uint32_t lo_s = lo_s0 + off;
          const uint32_t sfw = tmem + 128 + sf;
          const uint32_t sfx = sfw + 8;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            tmem_copy_scales<1>(sfw + 4 * j, desc_of(kDescHiPlain, lo_s + 32 * j));
            tmem_copy_scales<1>(sfx + 4 * j, desc_of(kDescHiPlain, lo_s + 64 + 32 * j));
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
            umma_f16<1>(tmem, desc_of(kDescHiSw128, lo_w + 2 * k), desc_of(kDescHiSw128, lo_x + 2 * k), idesc0, i | k);
        }
        umma_commit(smem_u32(empty_bar) + 8u * stage);
        if (i == iters - 1) umma_commit(smem_u32(done_bar));
      }
      __syncwarp();
      sf ^= 16u;
      if (++stage == sh.stages) {
        stage = 0;
        ph ^= 1u;
      }
    }
  }

  // ------------------------------------- partial sums into shared memory
  const bool ready = mbar_wait(smem_u32(done_bar), 0, s_abort, p.status, kStatusTimeoutEpilogue);
  const bool all_ready = __syncthreads_and(ready);
  float* red = reinterpret_cast<float*>(smem);   // [token][128 rows], over the drained ring
  if (all_ready) {
    tc_fence_after();
    for (int c = 0; c < sh.bn; c += 16) {
      uint32_t r[16];
      tmem_ld16(tmem + (static_cast<uint32_t>(warp * 32) << 16) + c, r);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < 16; ++j) red[(c + j) * 128 + threadIdx.x] = __uint_as_float(r[j]);
    }
  }
  cluster_sync();

  // --------------------------- this CTA's share of the columns, all parts
  if (all_ready) {
    const int share = (kGate ? 64 : 128) / sh.splits;
    const int quads = share / 4;                                          // threads per token
    const int f = rank * share + static_cast<int>(threadIdx.x) % quads * 4;   // first of four features in the tile
    const int per = kSkinnyThreads / quads;                               // tokens per pass
    const uint32_t red_addr = smem_u32(red);
    uint32_t part[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) part[q] = q < sh.splits ? map_to_cta(red_addr, q) : 0u;
    const int live = static_cast<int>(p.m - t0 < sh.bn ? p.m - t0 : sh.bn);
    if (n0 + f < p.n) {
#pragma unroll 2
      for (int t = static_cast<int>(threadIdx.x) / quads; t < live; t += per) {
        float4 a[8], b[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          if (q < sh.splits) {
            a[q] = ld_cluster_f32x4(part[q] + (t * 128 + f) * 4);
            if (kGate) b[q] = ld_cluster_f32x4(part[q] + (t * 128 + 64 + f) * 4);
          }
        }
        float4 sum = a[0], gate = b[0];
#pragma unroll
        for (int q = 1; q < 8; ++q) {
          if (q < sh.splits) {
            sum.x += a[q].x, sum.y += a[q].y, sum.z += a[q].z, sum.w += a[q].w;
            if (kGate) gate.x += b[q].x, gate.y += b[q].y, gate.z += b[q].z, gate.w += b[q].w;
          }
        }
        const int64_t row = static_cast<int64_t>(t0) + t;
        if (kGate) {
          if (p.preact != nullptr) {
            float* pre = p.preact + row * (2 * static_cast<int64_t>(p.n)) + n0 + f;
            *reinterpret_cast<float4*>(pre) = sum;
            *reinterpret_cast<float4*>(pre + p.n) = gate;
          }
          sum.x *= act_value(gate.x, p.act), sum.y *= act_value(gate.y, p.act);
          sum.z *= act_value(gate.z, p.act), sum.w *= act_value(gate.w, p.act);
        }
        const int64_t at = row * p.ldo + n0 + f;
        if (p.out_type == kTypeFp32) {
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
  if (warp == 2) tmem_dealloc(tmem, kCols);
}

namespace {

template <bool kMx, bool kGate>
int launch_skinny(const CUtensorMap& w, const CUtensorMap& x, const CUtensorMap& sfw, const CUtensorMap& sfx,
                  const DenseParams& p, SkinnyShape sh, int units, int token_tiles, bool dependent, cudaStream_t s) {
  auto kern = dense_skinny_kernel<kMx, kGate>;
  static OncePerDevice ready;
  if (!ready([&] {
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingLarge + kSkinnyExtra) ==
               cudaSuccess;
      }))
    return MOE_B200_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(units * sh.splits), static_cast<unsigned>(token_tiles));
  cfg.blockDim = dim3(kSkinnyThreads);
  cfg.dynamicSmemBytes = sh.ring_bytes + kSkinnyExtra;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(sh.splits);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, w, x, sfw, sfx, p, sh) == cudaSuccess ? MOE_B200_OK : MOE_B200_ERR_CUDA;
}

// As many K parts (a power of two up to 8, at most one per K step) as keep
// the grid within one CTA per SM.
SkinnyShape choose_shape(const DenseParams& p, int units, int token_tiles, int bn, int extra, int sm_count) {
  SkinnyShape sh;
  sh.bn = bn;
  sh.splits = 1;
  while (sh.splits < 8 && 2 * sh.splits * units * token_tiles <= sm_count && 2 * sh.splits <= p.k_iters)
    sh.splits *= 2;
  sh.stage_bytes = kWeightTile + bn * 128 + extra;
  // Up to 64 tokens a ring of 108 KB: the next GEMM of the call fits on the
  // SM beside this one and streams its first weights under this one's tail.
  sh.ring_bytes = bn <= 64 ? kRingSmall : kRingLarge;
  sh.stages = sh.ring_bytes / sh.stage_bytes;
  if (sh.stages > kMaxStages) sh.stages = kMaxStages;
  return sh;
}

int token_tile(int64_t m) { return m >= 128 ? 128 : static_cast<int>(div_up(m, 16) * 16); }

}  // namespace

int launch_dense_skinny(DenseEpi epi, const DenseOperand& a, const DenseOperand& b, DenseParams p, int sm_count,
                        bool dependent, cudaStream_t s) {
  const bool gate = epi == kEpiGated;
  p.k_iters = static_cast<int>(div_up(p.k, 64));
  p.vec32 = 1;   // four columns at a time: n and ldo are multiples of 8
  const int units = static_cast<int>(div_up(p.n, gate ? 64 : 128));
  const int bn = token_tile(p.m);
  const int token_tiles = static_cast<int>(div_up(p.m, bn));
  const SkinnyShape sh = choose_shape(p, units, token_tiles, bn, 0, sm_count);
  CUtensorMap tw, tx;
  if (!encode_2d(&tw, b.base, 2, b.cols, b.rows, b.pitch, 64, 64) ||
      !encode_2d(&tx, a.base, 2, a.cols, a.rows, a.pitch, 64, bn))
    return MOE_B200_ERR_DRIVER;
  return gate ? launch_skinny<false, true>(tw, tx, tw, tx, p, sh, units, token_tiles, dependent, s)
              : launch_skinny<false, false>(tw, tx, tw, tx, p, sh, units, token_tiles, dependent, s);
}

int launch_mx_skinny(const MxOperand& a, const MxOperand& b, DenseParams p, int sm_count, bool dependent,
                     cudaStream_t s) {
  p.k_iters = static_cast<int>(div_up(p.k, 256));
  p.vec32 = p.n % 4 == 0 && p.ldo % 4 == 0;   // four columns at a time
  const int units = static_cast<int>(div_up(p.n, 128));
  const int bn = token_tile(p.m);
  const int token_tiles = static_cast<int>(div_up(p.m, bn));
  const SkinnyShape sh = choose_shape(p, units, token_tiles, bn, 2048, sm_count);
  const int64_t kt = div_up(p.k, 128);
  CUtensorMap tw, tx, tsw, tsx;
  if (!encode_2d(&tw, b.q, 1, p.k / 2, b.rows, p.k / 2, 128, 64) ||
      !encode_2d(&tx, a.q, 1, p.k / 2, a.rows, p.k / 2, 128, bn) ||
      !encode_2d(&tsw, b.scale, 2, 256, div_up(b.rows, 128) * kt, 512, 256, 2, false) ||
      !encode_2d(&tsx, a.scale, 2, 256, div_up(a.rows, 128) * kt, 512, 256, 2, false))
    return MOE_B200_ERR_DRIVER;
  return launch_skinny<true, false>(tw, tx, tsw, tsx, p, sh, units, token_tiles, dependent, s);
}

}  // namespace moe
