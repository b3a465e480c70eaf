// Dense GEMMs over CTA pairs (sm_100a): D[m, n] = sum_k A[m, k] B[n, k] with
// 16-bit or 4-bit microscaled operands, fp32 sums in tensor memory.
//
// One tile is 256 output rows x up to 256 output columns, computed by a pair
// of CTAs with tcgen05.mma.cta_group::2: each CTA stages its 128 rows of A
// and its half of B's rows, so a 128-byte K slice costs 32 KB of shared
// memory per CTA instead of the 48 KB of a single-CTA 128 x 256 tile, and
// each B byte is fetched once per pair. Persistent: one pair per two SMs
// walks the tiles; two accumulators in tensor memory let the epilogue of one
// tile run under the MMAs of the next.
//
// Roles per CTA: warp 0 TMA producer, warp 1 MMA issuer (of the pair's first
// CTA only), warp 2 owns tensor memory, warps 4-7 epilogue, one 32-lane
// quarter of the accumulator each. The pair's loads all count on the first
// CTA's `full` barrier; its commits free the stage in both CTAs.
//
// Each epilogue thread owns an output row and writes 32-byte sectors: full
// sectors need no staging through shared memory, and L2 merges a row's
// sectors before they reach HBM.
//
// The operands may be stored along K or along the output dimension (the
// gradients need W^T and X^T): the shared-memory descriptors take both, so
// nothing is transposed in memory.
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
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

__device__ uint32_t g_dense_status;

uint32_t* dense_status_word() {
  static std::atomic<uint32_t*> words[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  uint32_t* word = words[dev].load(std::memory_order_acquire);
  if (word == nullptr) {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_dense_status) != cudaSuccess) return nullptr;
    word = static_cast<uint32_t*>(p);
    words[dev].store(word, std::memory_order_release);
  }
  return word;
}

namespace {

constexpr int kTileBytes = 16384;   // 128 rows (or 128 MN elements x 64 K) of 128 bytes

constexpr int kMaxStages = 12;
constexpr int kRingBytes = 224 * 1024;
constexpr int kNumBars = 2 * kMaxStages + 4;
constexpr int kPairSmem = kRingBytes + kNumBars * 8 + 16 + 1024;
static_assert(kPairSmem <= 227 * 1024, "shared memory");

template <bool kMx>
struct PairTraits {
  static constexpr int kScaleBytes = kMx ? 3072 : 0;   // A: 2 K tiles, B: 2 row tiles x 2 K tiles of 512 bytes
  // Tensor memory: two accumulators of up to 256 columns. With 4-bit
  // operands 48 columns hold the staged exponents (2 x 24), and the
  // accumulators overlap in 48 columns, which the epilogue drains first.
  static constexpr int kAcc1 = kMx ? 208 : 256;
};
constexpr int kScaleCol = 464;   // 4-bit: the first of those 48 columns

constexpr int kEpiWarps = 8;
constexpr int kPairThreads = (4 + kEpiWarps) * 32;

struct Tile {
  int m0, n0;   // first output row of the pair, first output column
};

// Tiles in bands of 8 row tiles, rows fastest: the pairs running at one time
// cover a near-square block of the output, so A and B slices are re-read
// from L2.
__device__ __forceinline__ Tile tile_at(int t, const DenseParams& p) {
  constexpr int kBand = 8;
  const int per_band = kBand * p.n_tiles;
  const int band = t / per_band;
  const int r = t - band * per_band;
  const int rows = min(kBand, p.m_tiles - band * kBand);
  Tile o;
  o.n0 = (r / rows) * p.n_step;
  o.m0 = (band * kBand + r % rows) * 256;
  return o;
}

// Writes 16 consecutive 16-bit outputs: columns c .. c+15 of a row, those
// below n (n and c multiples of 8).
__device__ __forceinline__ void store_row16(uint16_t* row, int c, int n, const uint32_t* v, bool vec32) {
  if (vec32 && c + 16 <= n) {
    st_global_32(row + c, v);
  } else {
    if (c + 8 <= n) *reinterpret_cast<uint4*>(row + c) = make_uint4(v[0], v[1], v[2], v[3]);
    if (c + 16 <= n) *reinterpret_cast<uint4*>(row + c + 8) = make_uint4(v[4], v[5], v[6], v[7]);
  }
}

}  // namespace

template <bool kMx, bool kAMn, bool kBMn, int kEpi>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    dense_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                      const __grid_constant__ CUtensorMap tm_sfa, const __grid_constant__ CUtensorMap tm_sfb,
                      const DenseParams p) {
  using Tr = PairTraits<kMx>;
  constexpr bool kGate = kEpi == kEpiGated || kEpi == kEpiGatedQuant;
  const int kS = p.stages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kRingBytes);
  uint64_t* full_bar = bars;                 // first CTA: both CTAs' copies of a stage have landed
  uint64_t* empty_bar = bars + kMaxStages;   // the stage's MMAs are done
  uint64_t* accf_bar = bars + 2 * kMaxStages;   // accumulator complete
  uint64_t* acce_bar = accf_bar + 2;     // first CTA: both CTAs' epilogues are through with an accumulator
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(bars + kNumBars);
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_cta_rank();
  const int pair = blockIdx.x >> 1;
  const int pairs = gridDim.x >> 1;
  const int tiles = p.m_tiles * p.n_tiles;

  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tm_a);
    prefetch_tmap(&tm_b);
    for (int s = 0; s < kS; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 1);
      mbar_init(smem_u32(&empty_bar[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&accf_bar[b]), 1);
      mbar_init(smem_u32(&acce_bar[b]), 2 * kEpiWarps);
    }
    *s_abort = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 2) {
    tmem_alloc_pair(smem_u32(s_tmem), 512);
    tmem_relinquish_pair();
  }
  pdl_launch_next();
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  // Everything above overlaps the previous kernel's tail. (The producer waits
  // for that kernel below; no bounded wait of the others starts before.)
  if (warp != 0) pdl_wait();

  if (warp == 0) {
    // ---------------------------------------------------------- producer
    const bool issue = elect_lane();
    const int b_rows = p.bn >> 1;                          // B rows this CTA stages
    const int b_atoms = kBMn ? (b_rows + 63) >> 6 : 0;
    const uint32_t bytes =
        kTileBytes + (kBMn ? static_cast<uint32_t>(b_atoms) * 8192u : static_cast<uint32_t>(b_rows) * 128u) +
        Tr::kScaleBytes;
    const int kt = kMx ? (p.k + 127) >> 7 : 0;             // exponent tiles along K
    const uint32_t base = smem_u32(smem);
    const uint32_t full0 = smem_u32(full_bar);
    const uint32_t full0_pair = map_to_cta(full0, 0);
    auto load_b = [&](int n0, int kb, int stage) {
      const uint32_t bar = full0_pair + 8u * stage;
      const uint32_t sb = base + stage * p.stage_bytes + kTileBytes;
      const int bnr = n0 + static_cast<int>(rank) * p.b_half;
      if (rank == 0) mbar_arrive_expect_tx(full0 + 8u * stage, 2u * bytes);
      if constexpr (kMx) {
        tma_load_2d_pair(sb, &tm_b, bar, kb * 128, bnr);
        tma_load_2d_pair(sb + kTileBytes + 1024, &tm_sfb, bar, 0, (n0 >> 7) * kt + 2 * kb);
        tma_load_2d_pair(sb + kTileBytes + 2048, &tm_sfb, bar, 0, ((n0 + p.b_half) >> 7) * kt + 2 * kb);
      } else if constexpr (kBMn) {
        tma_load_2d_pair(sb, &tm_b, bar, bnr, kb * 64);
        if (b_atoms > 1) tma_load_2d_pair(sb + 8192, &tm_b, bar, bnr + 64, kb * 64);
      } else {
        tma_load_2d_pair(sb, &tm_b, bar, kb * 64, bnr);
      }
    };
    auto load_a = [&](int m0, int kb, int stage) {
      const uint32_t bar = full0_pair + 8u * stage;
      const uint32_t sa = base + stage * p.stage_bytes;
      const int am = m0 + static_cast<int>(rank) * 128;
      if constexpr (kMx) {
        tma_load_2d_pair(sa, &tm_a, bar, kb * 128, am);
        tma_load_2d_pair(sa + 2 * kTileBytes, &tm_sfa, bar, 0, (am >> 7) * kt + 2 * kb);
      } else if constexpr (kAMn) {
        tma_load_2d_pair(sa, &tm_a, bar, am, kb * 64);
        tma_load_2d_pair(sa + 8192, &tm_a, bar, am + 64, kb * 64);
      } else {
        tma_load_2d_pair(sa, &tm_a, bar, kb * 64, am);
      }
    };
    // B is an input of the whole call (weights, or saved by another call):
    // its part of the first ring does not wait for the predecessor.
    const int early = min(kS, p.k_iters);
    if (issue) {
      const int n0 = tile_at(pair, p).n0;
      for (int kb = 0; kb < early; ++kb) load_b(n0, kb, kb);
    }
    __syncwarp();
    pdl_wait();
    int stage = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int t = pair; ok && t < tiles; t += pairs) {
      const Tile tl = tile_at(t, p);
      const int skip = t == pair ? early : 0;   // K steps whose B is on its way already
      for (int kb = 0; kb < p.k_iters; ++kb) {
        if (kb >= skip && !warp_wait(smem_u32(empty_bar) + 8u * stage, ph ^ 1u, s_abort, p.status,
                                     kStatusTimeoutProducer)) {
          ok = false;
          break;
        }
        if (issue) {
          if (kb >= skip) load_b(tl.n0, kb, stage);
          load_a(tl.m0, kb, stage);
        }
        __syncwarp();
        if (++stage == kS) {
          stage = 0;
          ph ^= 1u;
        }
      }
    }
    if (!ok) drain_copies();
  } else if (warp == 1) {
    // --------------------------------------------------------------- MMA
    if (rank == 0) {
      const bool issue = elect_lane();
      int stage = 0;
      uint32_t ph = 0;
      bool ok = true;
      int it = 0;                 // tiles done by this pair
      int old = kS - 2;           // 4-bit: the stage before last, and its phase
      uint32_t old_ph = 1, sf = 0;
      const uint32_t idesc0 = kMx ? idesc_mxf4(256, 256, 0) : idesc_f16(256, p.bn, p.type == kTypeFp16, kAMn, kBMn);
      const uint32_t idesc1 = kMx ? idesc_mxf4(256, 256, 2) : idesc0;
      const uint32_t base = smem_u32(smem);
      const uint32_t lo_a0 = kAMn ? desc_lo_mnmajor(base) : desc_lo_kmajor(base);
      const uint32_t lo_b0 = kBMn ? desc_lo_mnmajor(base + kTileBytes) : desc_lo_kmajor(base + kTileBytes);
      const uint32_t lo_s0 = desc_lo_scale(base + 2 * kTileBytes);
      for (int t = pair; ok && t < tiles; t += pairs, ++it) {
        const int buf = it & 1;
        const uint32_t d = tmem + (buf ? Tr::kAcc1 : 0);
        if (kMx ? it >= 1 : it >= 2) {
          const uint32_t bar = smem_u32(&acce_bar[kMx ? 0 : buf]);
          const uint32_t par = kMx ? static_cast<uint32_t>(it - 1) & 1u : (static_cast<uint32_t>(it >> 1) - 1u) & 1u;
          if (!__all_sync(0xffffffffu, mbar_wait_cluster(bar, par, s_abort, p.status, kStatusTimeoutMma))) break;
          tc_fence_after();
        }
        for (int kb = 0; kb < p.k_iters; ++kb) {
          if (!warp_wait(smem_u32(full_bar) + 8u * stage, ph, s_abort, p.status, kStatusTimeoutMma)) {
            ok = false;
            break;
          }
          const uint32_t off = static_cast<uint32_t>(stage * (p.stage_bytes >> 4));
          const uint32_t lo_a = lo_a0 + off, lo_b = lo_b0 + off;
          if constexpr (kMx) {
            // The exponent columns written now were last read two stages ago
            // (the first two waits pass at once).
            if (!warp_wait(smem_u32(empty_bar) + 8u * old, old_ph, s_abort, p.status, kStatusTimeoutMma)) {
              ok = false;
              break;
            }
            if (++old == kS) {
              old = 0;
              old_ph ^= 1u;
            }
          }
          tc_fence_after();
          if (issue) {
            if constexpr (kMx) {
              const uint32_t lo_s = lo_s0 + off;
              const uint32_t sfa = tmem + kScaleCol + sf;
              const uint32_t sfb = sfa + 8;
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                tmem_copy_scales<2>(sfa + 4 * j, desc_of(kDescHiPlain, lo_s + 32 * j));
                tmem_copy_scales<2>(sfb + 8 * j, desc_of(kDescHiPlain, lo_s + 64 + 32 * j));
                tmem_copy_scales<2>(sfb + 8 * j + 4, desc_of(kDescHiPlain, lo_s + 128 + 32 * j));
              }
              const int left = p.k - kb * 256;
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (k == 0 || left > 64 * k)
                  umma_mxf4<2>(d, desc_of(kDescHiSw128, lo_a + 2 * k), desc_of(kDescHiSw128, lo_b + 2 * k),
                               k & 1 ? idesc1 : idesc0, sfa + 4 * (k >> 1), sfb + 8 * (k >> 1), kb | k);
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_f16<2>(d, desc_of(kDescHiSw128, lo_a + (kAMn ? 128 : 2) * k),
                            desc_of(kDescHiSw128, lo_b + (kBMn ? 128 : 2) * k), idesc0, kb | k);
            }
            umma_commit_pair(smem_u32(empty_bar) + 8u * stage);
            if (kb == p.k_iters - 1) umma_commit_pair(smem_u32(&accf_bar[buf]));
          }
          __syncwarp();
          sf ^= 24u;
          if (++stage == kS) {
            stage = 0;
            ph ^= 1u;
          }
        }
      }
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------- epilogue
    const int quarter = warp & 3;
    const int half = (warp - 4) >> 2;   // two warps per quarter, taking turns at 32-column chunks
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const int width = kGate ? p.n_step : p.bn;   // output columns of a tile
    const int chunks = (width + 31) >> 5;
    const bool vec32 = p.vec32 != 0;
    int it = 0;
    for (int t = pair; t < tiles; t += pairs, ++it) {
      const Tile tl = tile_at(t, p);
      const int buf = it & 1;
      const bool ready = mbar_wait(smem_u32(&accf_bar[buf]), static_cast<uint32_t>(it >> 1) & 1u, s_abort, p.status,
                                   kStatusTimeoutEpilogue);
      if (!__all_sync(0xffffffffu, ready)) break;
      tc_fence_after();
      const uint32_t acc = lanes + (buf ? Tr::kAcc1 : 0);
      const int64_t row = static_cast<int64_t>(tl.m0) + rank * 128 + quarter * 32 + lane;
      const bool live = row < p.m;
      const int end = min(p.n, tl.n0 + width);   // first column past this tile
      for (int i = half; i < chunks; i += 2) {
        // 4-bit operands: the columns shared with the other accumulator first
        const int c = 32 * (kMx && buf == 0 ? chunks - 1 - i : i);
        uint32_t r[32];
        __syncwarp();
        if constexpr (kGate) {
          uint32_t g[32];
          tmem_ld32(acc + c, r);
          tmem_ld32(acc + p.n_step + c, g);
          tmem_wait_ld();
          if (kMx && i == half) {
            tc_fence_before();
            if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&acce_bar[0]), 0));
            __syncwarp();
          }
          if (live && tl.n0 + c < end) {
            if constexpr (kEpi == kEpiGated) {
              if (p.preact != nullptr) {
                float* pre = p.preact + row * (2 * static_cast<int64_t>(p.n)) + tl.n0 + c;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  if (tl.n0 + c + 8 * j < end) {
                    st_global_32(pre + 8 * j, r + 8 * j);
                    st_global_32(pre + p.n + 8 * j, g + 8 * j);
                  }
              }
            }
            float h[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) h[j] = act_value(__uint_as_float(g[j]), p.act) * __uint_as_float(r[j]);
            if constexpr (kEpi == kEpiGated) {
              uint16_t* out = static_cast<uint16_t*>(p.out) + row * p.ldo;
              uint32_t v[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) v[j] = pack_16(h[2 * j], h[2 * j + 1], p.type);
              store_row16(out, tl.n0 + c, end, v, vec32);
              store_row16(out, tl.n0 + c + 16, end, v + 8, vec32);
            } else {
              uint4 v;
              const uint32_t byte = mx_block(h, &v);
              *reinterpret_cast<uint4*>(p.q + (row * p.n + tl.n0 + c) / 2) = v;
              p.q_scale[mx_scale_offset(row, (tl.n0 + c) >> 5, (p.n + 127) >> 7)] = static_cast<uint8_t>(byte);
            }
          }
        } else {
          tmem_ld32(acc + c, r);
          tmem_wait_ld();
          if (kMx && i == half) {
            tc_fence_before();
            if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&acce_bar[0]), 0));
            __syncwarp();
          }
          if (live && tl.n0 + c < end) {
            if constexpr (kEpi == kEpiStore) {
              if (p.out_type == kTypeFp32) {
                float* out = static_cast<float*>(p.out) + row * p.ldo + tl.n0 + c;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  if (vec32 && tl.n0 + c + 8 * j + 8 <= end) {
                    st_global_32(out + 8 * j, r + 8 * j);
                  } else {
                    for (int e = 0; e < 8; ++e)
                      if (tl.n0 + c + 8 * j + e < end) out[8 * j + e] = __uint_as_float(r[8 * j + e]);
                  }
                }
              } else {
                uint16_t* out = static_cast<uint16_t*>(p.out) + row * p.ldo;
                uint32_t v[16];
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  v[j] = pack_16(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]), p.out_type);
                if (kMx && !vec32) {
                  // any n: column by column
                  for (int j = 0; j < 32; ++j)
                    if (tl.n0 + c + j < end) out[tl.n0 + c + j] = static_cast<uint16_t>(v[j >> 1] >> (16 * (j & 1)));
                } else {
                  store_row16(out, tl.n0 + c, end, v, vec32);
                  store_row16(out, tl.n0 + c + 16, end, v + 8, vec32);
                }
              }
            } else {   // kEpiDact
              const float* pre = p.preact + row * (2 * static_cast<int64_t>(p.n)) + tl.n0 + c;
              uint16_t* out = static_cast<uint16_t*>(p.out) + row * p.ldo;
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                uint32_t u[16] = {}, g[16] = {};
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if (tl.n0 + c + 16 * j + 8 * e < end) {
                    ld_global_32(u + 8 * e, pre + 16 * j + 8 * e);
                    ld_global_32(g + 8 * e, pre + p.n + 16 * j + 8 * e);
                  }
                uint32_t du[8], dg[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  float v[2], w[2];
#pragma unroll
                  for (int l = 0; l < 2; ++l) {
                    float value, slope;
                    act_value_slope(__uint_as_float(g[2 * e + l]), p.act, value, slope);
                    const float dh = __uint_as_float(r[16 * j + 2 * e + l]);
                    v[l] = dh * value;
                    w[l] = dh * __uint_as_float(u[2 * e + l]) * slope;
                  }
                  du[e] = pack_16(v[0], v[1], p.type);
                  dg[e] = pack_16(w[0], w[1], p.type);
                }
                store_row16(out, tl.n0 + c + 16 * j, end, du, vec32);
                store_row16(out + p.n, tl.n0 + c + 16 * j, end, dg, vec32);
              }
            }
          }
        }
      }
      if (!kMx) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&acce_bar[buf]), 0));
      }
    }
  }

  // No CTA leaves while the other may still reach its shared or tensor memory.
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync_relaxed();
  tc_fence_after();
  if (warp == 2) tmem_dealloc_pair(tmem, 512);
}

namespace {

template <bool kMx, bool kAMn, bool kBMn, int kEpi>
int launch_pair(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& sfa, const CUtensorMap& sfb,
                const DenseParams& p, int sm_count, bool dependent, cudaStream_t s) {
  auto kern = dense_pair_kernel<kMx, kAMn, kBMn, kEpi>;
  constexpr int smem = kPairSmem;
  static OncePerDevice ready;
  if (!ready([&] {
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess;
      }))
    return MOE_B200_ERR_CUDA;
  const int64_t tiles = static_cast<int64_t>(p.m_tiles) * p.n_tiles;
  const int pairs = static_cast<int>(tiles < sm_count / 2 ? tiles : sm_count / 2);
  return launch_kernel(kern, 2 * pairs, kPairThreads, smem, s, dependent, a, b, sfa, sfb, p) == cudaSuccess
             ? MOE_B200_OK
             : MOE_B200_ERR_CUDA;
}

// As many stages as the ring holds: a K step's loads take about 1.8 us to
// come back, so with six stages a step takes 300 ns however narrow the tile.
void set_ring(DenseParams* p, int stage_bytes) {
  p->stage_bytes = stage_bytes;
  p->stages = kRingBytes / stage_bytes < kMaxStages ? kRingBytes / stage_bytes : kMaxStages;
}

// Columns per tile (the MMA's N, 64 to 256): the fewest time units over all
// waves of tiles. A K step costs an MMA 2 N cycles and the loads 256 + N (A's
// 128 rows and N / 2 rows of B per CTA; at about 64 bytes a cycle from L2 the
// two meet at N = 256); a tile's start and epilogue cost about 1500 more.
// B stored along N is loaded in 64-column atoms whatever N is. Against 256
// throughout: training step at 4096 tokens 813 -> 786 us, at 333 x 1032 x 520
// 75 -> 55 us.
int choose_bn(const DenseParams& p, bool gate, bool b_mn, int pairs) {
  const int64_t m_tiles = div_up(p.m, 256), k = div_up(p.k, 64);
  int best = 256;
  int64_t best_cost = INT64_MAX;
  // the columns of a tile come in whole 32-byte stores: 16 features
  for (int bn = 256; bn >= 64; bn -= gate ? 32 : 16) {
    const int step = gate ? bn / 2 : bn;
    const int64_t waves = div_up(m_tiles * div_up(p.n, step), pairs);
    const int64_t b_cols = b_mn ? div_up(bn / 2, 64) * 128 : bn;
    const int64_t load = 256 + b_cols, mma = 2 * bn;
    const int64_t cost = waves * (k * (load > mma ? load : mma) + 1500);
    if (cost < best_cost) {
      best_cost = cost;
      best = bn;
    }
  }
  return best;
}

}  // namespace

int launch_dense_pair(DenseEpi epi, const DenseOperand& a, bool a_mn, const DenseOperand& b, bool b_mn, DenseParams p,
                      int sm_count, bool dependent, cudaStream_t s) {
  const bool gate = epi == kEpiGated;
  p.bn = choose_bn(p, gate, b_mn, sm_count / 2);
  p.n_step = gate ? p.bn / 2 : p.bn;
  p.b_half = gate ? p.n : p.bn / 2;
  p.m_tiles = static_cast<int>(div_up(p.m, 256));
  p.n_tiles = static_cast<int>(div_up(p.n, p.n_step));
  p.k_iters = static_cast<int>(div_up(p.k, 64));
  set_ring(&p, kTileBytes + (b_mn ? static_cast<int>(div_up(p.bn / 2, 64)) * 8192 : p.bn / 2 * 128));
  const int64_t dact_half = epi == kEpiDact ? static_cast<int64_t>(p.n) * 2 : 0;
  p.vec32 = aligned(p.out, 32) && (p.ldo * 2) % 32 == 0 && dact_half % 32 == 0;
  CUtensorMap ta, tb;
  if (!encode_2d(&ta, a.base, 2, a.cols, a.rows, a.pitch, 64, a_mn ? 64 : 128) ||
      !encode_2d(&tb, b.base, 2, b.cols, b.rows, b.pitch, 64, b_mn ? 64 : p.bn / 2))
    return MOE_B200_ERR_DRIVER;
  if (epi == kEpiGated && !a_mn && !b_mn)
    return launch_pair<false, false, false, kEpiGated>(ta, tb, ta, tb, p, sm_count, dependent, s);
  if (epi == kEpiDact && !a_mn && b_mn)
    return launch_pair<false, false, true, kEpiDact>(ta, tb, ta, tb, p, sm_count, dependent, s);
  if (epi == kEpiStore && !a_mn && !b_mn)
    return launch_pair<false, false, false, kEpiStore>(ta, tb, ta, tb, p, sm_count, dependent, s);
  if (epi == kEpiStore && !a_mn && b_mn)
    return launch_pair<false, false, true, kEpiStore>(ta, tb, ta, tb, p, sm_count, dependent, s);
  if (epi == kEpiStore && a_mn && b_mn)
    return launch_pair<false, true, true, kEpiStore>(ta, tb, ta, tb, p, sm_count, dependent, s);
  return MOE_B200_ERR_INVALID_ARGUMENT;
}

int launch_mx_pair(DenseEpi epi, const MxOperand& a, const MxOperand& b, DenseParams p, int sm_count, bool dependent,
                   cudaStream_t s) {
  const bool gate = epi == kEpiGatedQuant;
  p.bn = 256;
  p.n_step = gate ? 128 : 256;
  p.b_half = gate ? p.n : 128;
  p.m_tiles = static_cast<int>(div_up(p.m, 256));
  p.n_tiles = static_cast<int>(div_up(p.n, p.n_step));
  p.k_iters = static_cast<int>(div_up(p.k, 256));
  set_ring(&p, 2 * kTileBytes + PairTraits<true>::kScaleBytes);
  const int esz = p.out_type == kTypeFp32 ? 4 : 2;
  p.vec32 = aligned(p.out, 32) && (p.ldo * esz) % 32 == 0 && p.n % 8 == 0;
  const int64_t kt = div_up(p.k, 128);
  CUtensorMap ta, tb, tsa, tsb;
  if (!encode_2d(&ta, a.q, 1, p.k / 2, a.rows, p.k / 2, 128, 128) ||
      !encode_2d(&tb, b.q, 1, p.k / 2, b.rows, p.k / 2, 128, 128) ||
      !encode_2d(&tsa, a.scale, 2, 256, div_up(a.rows, 128) * kt, 512, 256, 2, false) ||
      !encode_2d(&tsb, b.scale, 2, 256, div_up(b.rows, 128) * kt, 512, 256, 2, false))
    return MOE_B200_ERR_DRIVER;
  if (gate) return launch_pair<true, false, false, kEpiGatedQuant>(ta, tb, tsa, tsb, p, sm_count, dependent, s);
  return launch_pair<true, false, false, kEpiStore>(ta, tb, tsa, tsb, p, sm_count, dependent, s);
}

}  // namespace moe
