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
// CTA only), warp 2 owns tensor memory, warps 4-11 epilogue, two to each
// 32-lane quarter of the accumulator. The pair's loads all count on the first
// CTA's `full` barrier; its commits free the stage in both CTAs.
//
// Each epilogue thread owns an output row and writes 32-byte sectors: full
// sectors need no staging through shared memory, and L2 merges a row's
// sectors before they reach HBM.
//
// What bounds it (4096 tokens, H = 7168, I = 2048): a K step of a 256 x 256
// tile takes 550 cycles, 512 of them MMA; the loads are then 60 bytes a cycle
// and SM, 14 TB/s over the GPU, which is all that L2 gave the same loads
// without MMAs. Under sustained load the power cap sets the clock (1.1 to 1.5
// GHz), and the rate is that of the vendor's library GEMM on the same
// operands. A K step of 4-bit operands has the same bytes and the same MMA
// cycles for four times the operations: 6.1 PFLOP/s at 28 steps a tile. With 8
// steps a tile takes 5,700 cycles for 4,096 of MMA, 735 of them until the
// accumulator's shared columns are free and 1,070 for loads.
//
// The operands may be stored along K or along the output dimension (the
// gradients need W^T and X^T): the shared-memory descriptors take both, so
// nothing is transposed in memory.
//
// Where the tiles of a product are few, their K range is split over 2 or 4
// pairs of one cluster: the partial tiles meet through distributed shared
// memory, each CTA adding the parts of its share of the rows in a fixed order
// (block at 256 tokens 44.5 -> 35.8 us, at 512 49.5 -> 46.4 us).
//
// One launch takes up to three products whose tiles follow one another in the
// walk. Of the backward pass's products dW2 depends on neither dh nor dx and
// dW13, and dx and dW13 not on each other: in two launches, dW2 in the one
// where it costs less, they fill their last waves and save a kernel's start
// and end each (training step at 4096 tokens 824 -> 796 us, 333 x 1032 x 520
// 48 -> 39 us). With dh split and dW2 beside dx and dW13, against dW2 always
// beside an unsplit dh: gradients at H = 7168, I = 2048 and 129 tokens 95 ->
// 68 us, at 512 103 -> 93, at 1024 156 -> 147; 1024 x 2048 x 1024 41 -> 37 (57,
// 86, 147 and 37 since).
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
  static constexpr int kScaleBytes = kMx ? 6 * 512 : 0;   // A: 2 K tiles, B: 2 row tiles x 2 K tiles of 512 bytes
  // Tensor memory: two accumulators of up to 256 columns. With 4-bit
  // operands 48 columns hold the staged exponents (2 x 24), and the
  // accumulators overlap in 48 columns, which the epilogue drains first.
  static constexpr int kAcc1 = kMx ? 208 : 256;
};
constexpr int kScaleCol = 464;   // 4-bit: the first of those 48 columns

constexpr int kEpiWarps = 8;
constexpr int kPairThreads = (4 + kEpiWarps) * 32;

// One launch: up to three products, their tiles numbered one after the other.
struct DenseGroup {
  DenseParams p[3];
  int tiles0, tiles1;   // tiles of the first, of the first two
  int tiles;            // of all
  int own, more, lead;  // tile_at
  int stages, stage_bytes;
  int splits;        // pairs of a cluster that share a tile's K range
};

// Tensor maps: A, B of the first product, then of the others; 4-bit: A, B and
// their exponents.
struct PairMaps {
  CUtensorMap m[6];
};

struct Work {
  int g;             // which product
  int m0, n0;        // first output row of the pair, first output column
};

// The j-th tile of a pair, -1 behind its last. The pairs take turns, first at
// the tiles of the first product: each has `own` of them, the first `more`
// pairs one more. The others then take `lead` tiles of the other products
// before the turns go on, for the tiles of the first may be several times as
// long.
template <bool kGrouped>
__device__ __forceinline__ int tile_at(const DenseGroup& grp, int pair, int pairs, int j) {
  int t = pair + j * pairs;
  if constexpr (kGrouped) {
    int s = j - grp.own - (pair < grp.more);
    if (s >= 0) {
      const int idle = pairs - grp.more;
      if (pair >= grp.more && s < grp.lead) {
        t = s * idle + pair - grp.more;
      } else {
        if (pair >= grp.more) s -= grp.lead;
        t = grp.lead * idle + s * pairs + pair;
      }
      t += grp.tiles0;
    }
  }
  return t < grp.tiles ? t : -1;
}

// Tiles in bands of 8 row tiles, rows fastest: the pairs running at one time
// cover a near-square block of the output, so A and B slices are re-read
// from L2.
template <bool kGrouped>
__device__ __forceinline__ Work work_at(int t, const DenseGroup& grp) {
  constexpr int kBand = 8;
  Work o;
  o.g = kGrouped ? (t >= grp.tiles0) + (t >= grp.tiles1) : 0;
  if (o.g) t -= o.g == 1 ? grp.tiles0 : grp.tiles1;
  const DenseParams& p = grp.p[o.g];
  const int per_band = kBand * p.n_tiles;
  const int band = t / per_band;
  const int r = t - band * per_band;
  const int rows = min(kBand, p.m_tiles - band * kBand);
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

// ---- epilogues: 32 (or 16) columns of one row, those below `end` -----------

// act(gate) * up, rounded to 16 bits (with the sums, where they are saved) or
// to one 4-bit block.
template <int kEpi>
__device__ __forceinline__ void store_gated(const DenseParams& p, int64_t row, int col, int end, const uint32_t* up,
                                            const uint32_t* gate) {
  if constexpr (kEpi == kEpiGated) {
    if (p.preact != nullptr) {
      float* pre = p.preact + row * (2 * static_cast<int64_t>(p.n)) + col;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col + 8 * j < end) {
          st_global_32(pre + 8 * j, up + 8 * j);
          st_global_32(pre + p.n + 8 * j, gate + 8 * j);
        }
    }
  }
  float h[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) h[j] = act_value(__uint_as_float(gate[j]), p.act) * __uint_as_float(up[j]);
  if constexpr (kEpi == kEpiGated) {
    uint16_t* out = static_cast<uint16_t*>(p.out) + row * p.ldo;
    uint32_t v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = pack_16(h[2 * j], h[2 * j + 1], p.type);
    store_row16(out, col, end, v, p.vec32);
    store_row16(out, col + 16, end, v + 8, p.vec32);
  } else {
    uint4 v;
    const uint32_t byte = mx_block(h, &v);
    *reinterpret_cast<uint4*>(p.q + (row * p.n + col) / 2) = v;
    p.q_scale[mx_scale_offset(row, col >> 5, (p.n + 127) >> 7)] = static_cast<uint8_t>(byte);
  }
}

// The sums themselves, rounded to the output's type, in the widest stores that
// the rows' starts allow. 4-bit product 4096 x 4096 x 2048 in bf16: rows on 32
// bytes 16.7 us, rows on 16 (4104 columns, or an output 16 bytes into a buffer)
// 22-25 (173 column by column), 4100 columns 172; in fp32 4100 columns 43 (123
// column by column).
template <bool kMx>
__device__ __forceinline__ void store_plain(const DenseParams& p, int64_t row, int col, int end, const uint32_t* r) {
  if (kMx && p.out_type == kTypeFp32) {
    float* out = static_cast<float*>(p.out) + row * p.ldo + col;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (p.vec32 && col + 8 * j + 8 <= end) {
        st_global_32(out + 8 * j, r + 8 * j);
      } else if (p.vec16) {
#pragma unroll
        for (int e = 8 * j; e < 8 * j + 8; e += 4)
          if (col + e < end) *reinterpret_cast<uint4*>(out + e) = make_uint4(r[e], r[e + 1], r[e + 2], r[e + 3]);
      } else {
        for (int e = 0; e < 8; ++e)
          if (col + 8 * j + e < end) out[8 * j + e] = __uint_as_float(r[8 * j + e]);
      }
    }
    return;
  }
  uint16_t* out = static_cast<uint16_t*>(p.out) + row * p.ldo;
  uint32_t v[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] = pack_16(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]), p.out_type);
  if (kMx && !p.vec16) {
    // rows that start anywhere: column by column
    for (int j = 0; j < 32; ++j)
      if (col + j < end) out[col + j] = static_cast<uint16_t>(v[j >> 1] >> (16 * (j & 1)));
  } else {
    store_row16(out, col, end, v, p.vec32);
    store_row16(out, col + 16, end, v + 8, p.vec32);
  }
}

// Saved up and gate sums of 16 columns.
struct Saved {
  uint32_t u[16], g[16];
};

__device__ __forceinline__ void load_saved(const DenseParams& p, int64_t row, int col, int end, Saved& s) {
  const float* pre = p.preact + row * (2 * static_cast<int64_t>(p.n)) + col;
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (col + 8 * e < end) {
      ld_global_32(s.u + 8 * e, pre + 8 * e);
      ld_global_32(s.g + 8 * e, pre + p.n + 8 * e);
    }
}

// [du | dg] = [dh act(g) | dh u act'(g)] of two columns, rounded to 16 bits.
__device__ __forceinline__ void dact_pair(const uint32_t* dh, const uint32_t* u, const uint32_t* g,
                                          const DenseParams& p, uint32_t& du, uint32_t& dg) {
  float v[2], w[2];
#pragma unroll
  for (int l = 0; l < 2; ++l) {
    float value, slope;
    act_value_slope(__uint_as_float(g[l]), p.act, value, slope);
    const float d = __uint_as_float(dh[l]);
    v[l] = d * value;
    w[l] = d * __uint_as_float(u[l]) * slope;
  }
  du = pack_16(v[0], v[1], p.type);
  dg = pack_16(w[0], w[1], p.type);
}

// The same of 16 columns, stored.
__device__ __forceinline__ void store_dact(const DenseParams& p, int64_t row, int col, int end, const uint32_t* dh,
                                           const Saved& s) {
  uint32_t du[8], dg[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dact_pair(dh + 2 * e, s.u + 2 * e, s.g + 2 * e, p, du[e], dg[e]);
  uint16_t* out = static_cast<uint16_t*>(p.out) + row * p.ldo;
  store_row16(out, col, end, du, p.vec32);
  store_row16(out + p.n, col, end, dg, p.vec32);
}

// K steps of split s begin here.
__device__ __forceinline__ int k_begin(int k_iters, int s, int splits) {
  return splits == 1 ? s * k_iters : k_iters * s / splits;
}

// Floats between the rows of a partial tile: 256 columns and a 16-byte shift,
// so that threads writing different rows do not meet in a bank.
constexpr int kPartPitch = 260;
static_assert(128 * kPartPitch * 4 <= kRingBytes, "partial tile");

// A CTA's share of its 128 rows of the cluster's tile: eight columns per
// thread, the parts of all pairs requested together and added in a fixed
// order (its own pair's first), then the epilogue.
template <int kEpi>
__device__ __forceinline__ void add_parts(const DenseParams& p, const Work& w, uint32_t smem, uint32_t rank, int split,
                                          int splits) {
  constexpr bool kGate = kEpi == kEpiGated;
  const int rows = 128 / splits;
  const int width = kGate ? p.n_step : p.bn;
  const int eighths = width / 8;
  uint32_t part[4];
#pragma unroll
  for (int q = 0; q < 4; ++q)
    part[q] = q < splits ? map_to_cta(smem, 2 * ((split + q) & (splits - 1)) + rank) : 0u;
  auto sums = [&](int row, int c, uint32_t* out) {
    float4 a[4][2];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (q < splits) {
        a[q][0] = ld_cluster_f32x4(part[q] + (row * kPartPitch + c) * 4);
        a[q][1] = ld_cluster_f32x4(part[q] + (row * kPartPitch + c + 4) * 4);
      }
    float4 lo = a[0][0], hi = a[0][1];
#pragma unroll
    for (int q = 1; q < 4; ++q)
      if (q < splits) {
        lo.x += a[q][0].x, lo.y += a[q][0].y, lo.z += a[q][0].z, lo.w += a[q][0].w;
        hi.x += a[q][1].x, hi.y += a[q][1].y, hi.z += a[q][1].z, hi.w += a[q][1].w;
      }
    out[0] = __float_as_uint(lo.x), out[1] = __float_as_uint(lo.y), out[2] = __float_as_uint(lo.z);
    out[3] = __float_as_uint(lo.w), out[4] = __float_as_uint(hi.x), out[5] = __float_as_uint(hi.y);
    out[6] = __float_as_uint(hi.z), out[7] = __float_as_uint(hi.w);
  };
  for (int i = static_cast<int>(threadIdx.x); i < rows * eighths; i += kPairThreads) {
    const int r = split * rows + i / eighths;
    const int c = i % eighths * 8;
    const int64_t row = static_cast<int64_t>(w.m0) + rank * 128 + r;
    const int col = w.n0 + c;
    if (row >= p.m || col >= p.n) continue;
    uint32_t v[8];
    sums(r, c, v);
    if constexpr (kGate) {
      uint32_t g[8];
      sums(r, p.n_step + c, g);
      if (p.preact != nullptr) {
        float* pre = p.preact + row * (2 * static_cast<int64_t>(p.n)) + col;
        st_global_32(pre, v);
        st_global_32(pre + p.n, g);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = __float_as_uint(act_value(__uint_as_float(g[j]), p.act) * __uint_as_float(v[j]));
    }
    uint16_t* out = static_cast<uint16_t*>(p.out) + row * p.ldo + col;
    uint32_t o[4];
    if (kEpi == kEpiBackward && p.preact != nullptr) {
      const float* pre = p.preact + row * (2 * static_cast<int64_t>(p.n)) + col;
      uint32_t u[8], g[8], dg[4];
      ld_global_32(u, pre);
      ld_global_32(g, pre + p.n);
#pragma unroll
      for (int j = 0; j < 4; ++j) dact_pair(v + 2 * j, u + 2 * j, g + 2 * j, p, o[j], dg[j]);
      *reinterpret_cast<uint4*>(out + p.n) = make_uint4(dg[0], dg[1], dg[2], dg[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = pack_16(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]), p.out_type);
    }
    *reinterpret_cast<uint4*>(out) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// 4-bit: the columns the next accumulator needs are in registers.
__device__ __forceinline__ void release_early(uint64_t* acce_bar, int lane) {
  tc_fence_before();
  if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&acce_bar[0]), 0));
  __syncwarp();
}

}  // namespace

// kSplits: clusters of several pairs take one tile each, `split` telling the
// pairs apart; otherwise clusters of one pair walk the tiles. (One kernel for
// both took 0.3 us longer per launch.)
template <bool kMx, bool kBMn, int kEpi, bool kSplits>
__global__ void __launch_bounds__(kPairThreads, 1)
    dense_pair_kernel(const __grid_constant__ PairMaps maps, const __grid_constant__ DenseGroup grp) {
  using Tr = PairTraits<kMx>;
  constexpr bool kGate = kEpi == kEpiGated || kEpi == kEpiGatedQuant;
  constexpr bool kGrouped = kEpi == kEpiBackward;   // several products, A stored either way
  const int kS = grp.stages;
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
  const int splits = kSplits ? grp.splits : 1;
  const uint32_t cta = cluster_cta_rank();
  const uint32_t rank = cta & 1u;
  const uint32_t lead = cta & ~1u;
  const int split = kSplits ? static_cast<int>(cta >> 1) : 0;
  const uint32_t pair_mask = 3u << lead;
  const int log_ctas = kSplits ? 32 - __clz(splits) : 1;   // of a cluster
  const int pair = static_cast<int>(blockIdx.x >> log_ctas);
  const int pairs = static_cast<int>(gridDim.x >> log_ctas);
  auto tile_of = [&](int j) { return tile_at<kGrouped>(grp, pair, pairs, j); };
  uint32_t* const status = grp.p[0].status;

  if (warp == 0 && lane == 0) {
    prefetch_tmap(&maps.m[0]);
    prefetch_tmap(&maps.m[1]);
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
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  // Everything above overlaps the previous kernel's tail. (The producer waits
  // for that kernel below; no bounded wait of the others starts before.)
  if (warp != 0) {
    pdl_wait();
    pdl_launch_next();
  }

  if (warp == 0) {
    // ---------------------------------------------------------- producer
    const bool issue = elect_lane();
    const uint32_t base = smem_u32(smem);
    const uint32_t full0 = smem_u32(full_bar);
    const uint32_t full0_pair = map_to_cta(full0, lead);
    // B's part of a stage, and the count of bytes both CTAs' parts bring.
    auto load_b = [&](const Work& w, int kb, int stage) {
      const DenseParams& p = grp.p[w.g];
      const uint32_t bar = full0_pair + 8u * stage;
      const uint32_t sb = base + stage * grp.stage_bytes + kTileBytes;
      const int bnr = w.n0 + static_cast<int>(rank) * p.b_half;
      if (rank == 0) mbar_arrive_expect_tx(full0 + 8u * stage, 2u * p.copy_bytes);
      if constexpr (kMx) {
        const int kt = (p.k + 127) >> 7;   // exponent tiles along K
        tma_load_2d_pair(sb, &maps.m[1], bar, kb * 128, bnr);
        tma_load_2d_pair(sb + kTileBytes + 1024, &maps.m[3], bar, 0, (w.n0 >> 7) * kt + 2 * kb);
        tma_load_2d_pair(sb + kTileBytes + 2048, &maps.m[3], bar, 0, ((w.n0 + p.b_half) >> 7) * kt + 2 * kb);
      } else if constexpr (kBMn) {
        const CUtensorMap* map = &maps.m[2 * w.g + 1];
        tma_load_2d_pair(sb, map, bar, bnr, kb * 64);
        if (p.bn > 128) tma_load_2d_pair(sb + 8192, map, bar, bnr + 64, kb * 64);
      } else {
        tma_load_2d_pair(sb, &maps.m[1], bar, kb * 64, bnr);
      }
    };
    auto load_a = [&](const Work& w, int kb, int stage) {
      const DenseParams& p = grp.p[w.g];
      const uint32_t bar = full0_pair + 8u * stage;
      const uint32_t sa = base + stage * grp.stage_bytes;
      const int am = w.m0 + static_cast<int>(rank) * 128;
      if constexpr (kMx) {
        tma_load_2d_pair(sa, &maps.m[0], bar, kb * 128, am);
        tma_load_2d_pair(sa + 2 * kTileBytes, &maps.m[2], bar, 0, (am >> 7) * ((p.k + 127) >> 7) + 2 * kb);
      } else {
        const CUtensorMap* map = &maps.m[2 * w.g];
        if (kGrouped && p.a_mn) {
          tma_load_2d_pair(sa, map, bar, am, kb * 64);
          tma_load_2d_pair(sa + 8192, map, bar, am + 64, kb * 64);
        } else {
          tma_load_2d_pair(sa, map, bar, kb * 64, am);
        }
      }
    };
    // B is an input of the whole call (weights, or saved by another call):
    // behind a kernel of the same call its part of the first ring does not
    // wait for that kernel.
    const int t0 = tile_of(0);
    const Work w0 = work_at<kGrouped>(max(t0, 0), grp);
    const int first = k_begin(grp.p[w0.g].k_iters, split, splits);
    const int early =
        grp.p[0].early && t0 >= 0 ? min(kS, k_begin(grp.p[w0.g].k_iters, split + 1, splits) - first) : 0;
    if (issue)
      for (int i = 0; i < early; ++i) load_b(w0, first + i, i);
    __syncwarp();
    pdl_wait();
    int stage = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int it = 0, t; ok && (t = tile_of(it)) >= 0; ++it) {
      const Work w = work_at<kGrouped>(t, grp);
      const int kb0 = k_begin(grp.p[w.g].k_iters, split, splits);
      const int kb1 = k_begin(grp.p[w.g].k_iters, split + 1, splits);
      const int skip = kb0 + (it == 0 ? early : 0);   // K steps whose B is on its way already
      for (int kb = kb0; kb < kb1; ++kb) {
        if (kb >= skip &&
            !warp_wait(smem_u32(empty_bar) + 8u * stage, ph ^ 1u, s_abort, status, kStatusTimeoutProducer)) {
          ok = false;
          break;
        }
        if (issue) {
          if (kb >= skip) load_b(w, kb, stage);
          load_a(w, kb, stage);
        }
        __syncwarp();
        if (++stage == kS) {
          stage = 0;
          ph ^= 1u;
        }
      }
    }
    // The MMAs hand back the last ring's stages too, by arrivals in both CTAs
    // that no load waits for: they are awaited here, so that none is still on
    // its way to a CTA that has left. (A stage never used passes at once.)
    for (int s = 0; ok && s < kS; ++s) {
      ok = warp_wait(smem_u32(empty_bar) + 8u * stage, ph ^ 1u, s_abort, status, kStatusTimeoutProducer);
      if (++stage == kS) {
        stage = 0;
        ph ^= 1u;
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
      int old = kS - 2;           // 4-bit: the stage before last, and its phase
      uint32_t old_ph = 1, sf = 0;
      const uint32_t base = smem_u32(smem);
      const uint32_t lo_b0 = kBMn ? desc_lo_mnmajor(base + kTileBytes) : desc_lo_kmajor(base + kTileBytes);
      const uint32_t lo_s0 = desc_lo_scale(base + 2 * kTileBytes);
      for (int it = 0, t; ok && (t = tile_of(it)) >= 0; ++it) {   // `it` tiles are done
        const DenseParams& p = grp.p[work_at<kGrouped>(t, grp).g];
        const bool a_mn = kGrouped && p.a_mn;
        const uint32_t idesc0 = kMx ? idesc_mxf4(256, 256, 0) : idesc_f16(256, p.bn, p.type == kTypeFp16, a_mn, kBMn);
        const uint32_t idesc1 = kMx ? idesc_mxf4(256, 256, 2) : idesc0;
        const uint32_t lo_a0 = a_mn ? desc_lo_mnmajor(base) : desc_lo_kmajor(base);
        const uint32_t a_step = a_mn ? 128 : 2;
        const int kb0 = k_begin(p.k_iters, split, splits), kb1 = k_begin(p.k_iters, split + 1, splits);
        const int buf = it & 1;
        const uint32_t d = tmem + (buf ? Tr::kAcc1 : 0);
        if (kMx ? it >= 1 : it >= 2) {
          const uint32_t bar = smem_u32(&acce_bar[kMx ? 0 : buf]);
          const uint32_t par = kMx ? static_cast<uint32_t>(it - 1) & 1u : (static_cast<uint32_t>(it >> 1) - 1u) & 1u;
          if (!__all_sync(0xffffffffu, mbar_wait_cluster(bar, par, s_abort, status, kStatusTimeoutMma))) break;
          tc_fence_after();
        }
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!warp_wait(smem_u32(full_bar) + 8u * stage, ph, s_abort, status, kStatusTimeoutMma)) {
            ok = false;
            break;
          }
          const uint32_t off = static_cast<uint32_t>(stage * (grp.stage_bytes >> 4));
          const uint32_t lo_a = lo_a0 + off, lo_b = lo_b0 + off;
          if constexpr (kMx) {
            // The exponent columns written now were last read two stages ago
            // (the first two waits pass at once).
            if (!warp_wait(smem_u32(empty_bar) + 8u * old, old_ph, s_abort, status, kStatusTimeoutMma)) {
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
                umma_f16<2>(d, desc_of(kDescHiSw128, lo_a + a_step * k),
                            desc_of(kDescHiSw128, lo_b + (kBMn ? 128 : 2) * k), idesc0, (kb - kb0) | k);
            }
            umma_commit_pair(smem_u32(empty_bar) + 8u * stage, pair_mask);
            if (kb == kb1 - 1) umma_commit_pair(smem_u32(&accf_bar[buf]), pair_mask);
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
    int next[2] = {tile_of(0), tile_of(1)};
    for (int it = 0; next[0] >= 0; ++it) {
      const Work w = work_at<kGrouped>(next[0], grp);
      next[0] = next[1];
      next[1] = next[1] >= 0 ? tile_of(it + 2) : -1;
      const DenseParams& p = grp.p[w.g];
      const int width = kGate ? p.n_step : p.bn;   // output columns of a tile
      const int chunks = (width + 31) >> 5;
      const int buf = it & 1;
      const int64_t row = static_cast<int64_t>(w.m0) + rank * 128 + quarter * 32 + lane;
      const bool live = row < p.m;
      const int end = min(p.n, w.n0 + width);      // first column past this tile
      // dh: the saved sums of the first two 16-column pieces are on their way
      // while the accumulator is still being computed.
      const bool dact = kEpi == kEpiBackward && p.preact != nullptr && !kSplits;
      Saved saved[2];
      if (dact) {
        load_saved(p, row, w.n0 + 32 * half, live ? end : 0, saved[0]);
        load_saved(p, row, w.n0 + 32 * half + 16, live ? end : 0, saved[1]);
      }
      const bool ready = mbar_wait(smem_u32(&accf_bar[buf]), static_cast<uint32_t>(it >> 1) & 1u, s_abort, status,
                                   kStatusTimeoutEpilogue);
      if (!__all_sync(0xffffffffu, ready)) break;
      tc_fence_after();
      const uint32_t acc = lanes + (buf ? Tr::kAcc1 : 0);
      // A tile to come needs these columns. Otherwise nobody waits for the
      // arrival, and it could reach the first CTA after that has left.
      const bool reused = next[kMx ? 0 : 1] >= 0;
      if constexpr (kSplits) {
        // this pair's part of the sums, one row per thread, over the drained ring
        float* part = reinterpret_cast<float*>(smem) + (quarter * 32 + lane) * kPartPitch;
        for (int c = 32 * half; c < p.bn; c += 64) {
          uint32_t r[32];
          tmem_ld32(acc + c, r);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<uint4*>(part + c + j) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
        }
        break;
      }
      for (int i = half; i < chunks; i += 2) {
        // 4-bit operands: the columns shared with the other accumulator first
        const int c = 32 * (kMx && buf == 0 ? chunks - 1 - i : i);
        const int col = w.n0 + c;
        uint32_t r[32];
        __syncwarp();
        if constexpr (kGate) {
          uint32_t g[32];
          tmem_ld32(acc + c, r);
          tmem_ld32(acc + p.n_step + c, g);
          tmem_wait_ld();
          if (kMx && i == half && reused) release_early(acce_bar, lane);
          if (live && col < end) store_gated<kEpi>(p, row, col, end, r, g);
        } else {
          tmem_ld32(acc + c, r);
          tmem_wait_ld();
          if (kMx && i == half && reused) release_early(acce_bar, lane);
          if (dact) {
            const int next = i + 2 < chunks && live ? end : 0;
            if (live && col < end) store_dact(p, row, col, end, r, saved[0]);
            load_saved(p, row, col + 64, next, saved[0]);
            if (live && col + 16 < end) store_dact(p, row, col + 16, end, r + 16, saved[1]);
            load_saved(p, row, col + 80, next, saved[1]);
          } else if (live && col < end) {
            store_plain<kMx>(p, row, col, end, r);
          }
        }
      }
      if (!kMx && reused) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&acce_bar[buf]), lead));
      }
    }
  }

  if constexpr (kSplits) {
    __syncwarp();
    cluster_sync();   // every pair's part is there
    if (*s_abort == 0) add_parts<kEpi>(grp.p[0], work_at<false>(pair, grp), smem_u32(smem), rank, split, splits);
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

// As many stages as the ring holds.
void set_ring(DenseGroup* grp, int stage_bytes) {
  grp->stage_bytes = stage_bytes;
  grp->stages = kRingBytes / stage_bytes < kMaxStages ? kRingBytes / stage_bytes : kMaxStages;
}

template <bool kMx, bool kBMn, int kEpi, bool kSplits>
int launch_kernel_pair(const PairMaps& maps, DenseGroup grp, int sm_count, bool dependent, cudaStream_t s) {
  grp.p[0].early = dependent;
  auto kern = dense_pair_kernel<kMx, kBMn, kEpi, kSplits>;
  constexpr int smem = kPairSmem;
  static OncePerDevice ready;
  if (!ready([&] {
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess;
      }))
    return MOE_B200_ERR_CUDA;
  const int pairs = grp.splits > 1 ? grp.tiles * grp.splits : grp.tiles < sm_count / 2 ? grp.tiles : sm_count / 2;
  const int walkers = pairs / grp.splits;
  grp.own = grp.tiles0 / walkers;
  grp.more = grp.tiles0 % walkers;
  if (grp.more == 0) grp.lead = 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs));
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(2 * grp.splits);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, maps, grp) == cudaSuccess ? MOE_B200_OK : MOE_B200_ERR_CUDA;
}

template <bool kMx, bool kBMn, int kEpi>
int launch_pair(const PairMaps& maps, const DenseGroup& grp, int sm_count, bool dependent, cudaStream_t s) {
  if constexpr (!kMx)
    if (grp.splits > 1) return launch_kernel_pair<kMx, kBMn, kEpi, true>(maps, grp, sm_count, dependent, s);
  return launch_kernel_pair<kMx, kBMn, kEpi, false>(maps, grp, sm_count, dependent, s);
}

// Time units of a tile of bn columns: a K step costs an MMA 2 N cycles and the
// loads 256 + N (A's 128 rows and N / 2 rows of B per CTA; at about 64 bytes a
// cycle from L2 the two meet at N = 256; B stored along N comes in 64-column
// atoms whatever N is), and about 400 to issue; a tile's start and epilogue
// cost about 700 + 4 N more.
int64_t tile_cost(const DenseParams& p, int bn, bool b_mn, int splits = 1) {
  int64_t step = 256 + (b_mn ? (bn > 128 ? 256 : 128) : bn);
  if (step < 2 * bn) step = 2 * bn;
  if (step < 400) step = 400;
  return div_up(div_up(p.k, 64), splits) * step + 700 + 4 * bn;
}

int64_t tile_count(const DenseParams& p, int step) { return div_up(p.m, 256) * div_up(p.n, step); }

// Clusters of `ctas` (4 or 8) that run at once on the current device; 0 if that
// cannot be told.
int max_clusters(int ctas) {
  static std::atomic<int> known[2][64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  std::atomic<int>& slot = known[ctas == 8][dev];
  int n = slot.load(std::memory_order_relaxed);
  if (n == 0) {
    auto kern = dense_pair_kernel<false, false, kEpiGated, true>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(kPairThreads);
    cfg.dynamicSmemBytes = kPairSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(ctas);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess)
      return 0;
    slot.store(n, std::memory_order_relaxed);
  }
  return n;
}

// Columns per tile (the MMA's N) and K splits of one product: the fewest time
// units over all waves of tiles. Choosing the columns, against 256 throughout:
// training step at 4096 tokens 813 -> 786 us, at 333 x 1032 x 520 75 -> 55 us.
// A pair's MMA takes N in multiples of 32, which also keeps the columns of a
// tile in whole 32-byte stores. A split product is one wave of clusters and
// adds its parts for 6000 units, in the backward pass for fewer with narrow
// tiles (training step at 333 x 1032 x 520 32.5 -> 30.5 us, at 512 x 7168 x
// 2048 135.5 -> 128.4; in the forward pass that chose worse: block at 129 x
// 1024 x 512 10.6 -> 11.6). (How many clusters of 4 or 8 CTAs run at once
// depends on how the GPU's SMs are grouped, 33 and 15 where this was measured;
// one more made 256 tokens take 56 us.)
DensePlan choose_shape(const DenseParams& p, bool gate, bool b_mn, int sm_count) {
  DensePlan plan = {};
  plan.cost = INT64_MAX;
  for (int splits = 1; splits <= 4; splits *= 2) {
    if (splits > 1 && div_up(p.k, 64) < 4 * splits) break;
    for (int bn = 256; bn >= 64; bn -= 32) {
      const int64_t tiles = tile_count(p, gate ? bn / 2 : bn);
      if (splits > 1 && tiles > max_clusters(2 * splits)) continue;
      const int64_t waves = splits > 1 ? 1 : div_up(tiles, sm_count / 2);
      const int64_t cost = waves * tile_cost(p, bn, b_mn, splits) + (splits > 1 ? (b_mn ? 2500 + 14 * bn : 6000) : 0);
      if (cost < plan.cost) plan = DensePlan{{bn, 0}, splits, 0, cost};
    }
  }
  return plan;
}

// The same for several products of which all but the first have one K and take
// one width. Before the last turns every pair has `own` tiles of the first
// product, some one more, the others `lead` tiles of the rest (tile_at): as
// many as fit beside it, or one.
DensePlan choose_shapes(const DenseProduct* products, int count, int sm_count) {
  constexpr int kWidths = 7;   // 256, 224, .. 64
  const int pairs = sm_count / 2;
  int tiles[2][kWidths] = {}, costs[2][kWidths] = {};
  for (int i = 0; i < count; ++i)
    for (int w = 0; w < kWidths; ++w) {
      tiles[i > 0][w] += static_cast<int>(tile_count(products[i].p, 256 - 32 * w));
      costs[i > 0][w] = static_cast<int>(tile_cost(products[i].p, 256 - 32 * w, true));
    }
  DensePlan plan = {};
  plan.cost = INT64_MAX;
  for (int w0 = 0; w0 < kWidths; ++w0) {
    const int own = tiles[0][w0] / pairs, more = tiles[0][w0] % pairs, idle = pairs - more;
    const int64_t c0 = costs[0][w0];
    for (int w1 = 0; w1 < kWidths; ++w1) {
      const int rest = tiles[1][w1], c1 = costs[1][w1];
      const int fit = static_cast<int>(c0) / c1;
      for (int lead = 1; lead <= fit + 1; lead = lead < fit ? fit : lead + 1) {
        const int ahead = more == 0 ? 0 : lead * idle < rest ? lead * idle : rest;
        const int64_t beside = static_cast<int64_t>(div_up(ahead, idle)) * c1;
        const int64_t last = more == 0 ? 0 : c0 > beside ? c0 : beside;
        const int64_t cost = own * c0 + last + div_up(rest - ahead, pairs) * c1;
        if (cost < plan.cost) plan = DensePlan{{256 - 32 * w0, 256 - 32 * w1}, 1, lead, cost};
        if (more == 0) break;
      }
    }
  }
  return plan;
}

// Derived fields of a 16-bit product with its bn chosen.
void finish(DenseParams* p, bool gate, bool b_mn) {
  p->n_step = gate ? p->bn / 2 : p->bn;
  p->b_half = gate ? p->n : p->bn / 2;
  p->m_tiles = static_cast<int>(div_up(p->m, 256));
  p->n_tiles = static_cast<int>(div_up(p->n, p->n_step));
  p->k_iters = static_cast<int>(div_up(p->k, 64));
  p->copy_bytes = kTileBytes + (b_mn ? (p->bn > 128 ? 16384 : 8192) : p->bn / 2 * 128);
}

}  // namespace

int launch_dense_pair(DenseEpi epi, const DenseOperand& a, const DenseOperand& b, const DenseParams& params,
                      int sm_count, bool dependent, cudaStream_t s) {
  const bool gate = epi == kEpiGated;
  DenseGroup grp;
  std::memset(&grp, 0, sizeof(grp));
  grp.splits = 1;
  DenseParams& p = grp.p[0];
  p = params;
  const DensePlan plan = choose_shape(p, gate, false, sm_count);
  p.bn = plan.bn[0];
  grp.splits = plan.splits;
  finish(&p, gate, false);
  p.vec32 = aligned(p.out, 32) && (p.ldo * 2) % 32 == 0;
  grp.tiles0 = grp.tiles1 = grp.tiles = p.m_tiles * p.n_tiles;
  set_ring(&grp, p.copy_bytes);
  PairMaps maps;
  if (!encode_2d(&maps.m[0], a.base, 2, a.cols, a.rows, a.pitch, 64, 128) ||
      !encode_2d(&maps.m[1], b.base, 2, b.cols, b.rows, b.pitch, 64, p.bn / 2))
    return MOE_B200_ERR_DRIVER;
  for (int i = 2; i < 6; ++i) maps.m[i] = maps.m[0];
  return gate ? launch_pair<false, false, kEpiGated>(maps, grp, sm_count, dependent, s)
              : launch_pair<false, false, kEpiStore>(maps, grp, sm_count, dependent, s);
}

DensePlan plan_dense_backward(const DenseProduct* products, int count, int sm_count) {
  return count == 1 ? choose_shape(products[0].p, false, true, sm_count) : choose_shapes(products, count, sm_count);
}

int launch_dense_backward(const DenseProduct* products, int count, const DensePlan& plan, int sm_count, bool dependent,
                          cudaStream_t s) {
  DenseGroup grp;
  std::memset(&grp, 0, sizeof(grp));
  grp.splits = plan.splits;
  grp.lead = plan.lead;
  PairMaps maps;
  int stage = 0;
  for (int i = 0; i < count; ++i) {
    const DenseOperand &a = products[i].a, &b = products[i].b;
    DenseParams& p = grp.p[i];
    p = products[i].p;
    p.bn = plan.bn[i > 0];
    p.a_mn = products[i].a_mn;
    finish(&p, false, true);
    // dh is written as du and, n columns on, dg
    p.vec32 = aligned(p.out, 32) && (p.ldo * 2) % 32 == 0 && (p.preact == nullptr || p.n % 16 == 0);
    grp.tiles += p.m_tiles * p.n_tiles;
    if (i == 0) grp.tiles0 = grp.tiles;
    if (i <= 1) grp.tiles1 = grp.tiles;
    stage = stage > p.copy_bytes ? stage : p.copy_bytes;
    if (!encode_2d(&maps.m[2 * i], a.base, 2, a.cols, a.rows, a.pitch, 64, p.a_mn ? 64 : 128) ||
        !encode_2d(&maps.m[2 * i + 1], b.base, 2, b.cols, b.rows, b.pitch, 64, 64))
      return MOE_B200_ERR_DRIVER;
  }
  for (int i = 2 * count; i < 6; ++i) maps.m[i] = maps.m[0];
  set_ring(&grp, stage);
  return launch_pair<false, true, kEpiBackward>(maps, grp, sm_count, dependent, s);
}

int launch_mx_pair(DenseEpi epi, const MxOperand& a, const MxOperand& b, const DenseParams& params, int sm_count,
                   bool dependent, cudaStream_t s) {
  const bool gate = epi == kEpiGatedQuant;
  DenseGroup grp;
  std::memset(&grp, 0, sizeof(grp));
  grp.splits = 1;
  DenseParams& p = grp.p[0];
  p = params;
  p.bn = 256;
  p.n_step = gate ? 128 : 256;
  p.b_half = gate ? p.n : 128;
  p.m_tiles = static_cast<int>(div_up(p.m, 256));
  p.n_tiles = static_cast<int>(div_up(p.n, p.n_step));
  p.k_iters = static_cast<int>(div_up(p.k, 256));
  p.copy_bytes = 2 * kTileBytes + PairTraits<true>::kScaleBytes;
  const int esz = p.out_type == kTypeFp32 ? 4 : 2;
  p.vec32 = aligned(p.out, 32) && (p.ldo * esz) % 32 == 0 && p.n % 8 == 0;
  p.vec16 = (p.ldo * esz) % 16 == 0 && p.n * esz % 16 == 0;   // the output starts on 16 bytes
  grp.tiles0 = grp.tiles1 = grp.tiles = p.m_tiles * p.n_tiles;
  set_ring(&grp, p.copy_bytes);
  const int64_t kt = div_up(p.k, 128);
  PairMaps maps;
  if (!encode_2d(&maps.m[0], a.q, 1, p.k / 2, a.rows, p.k / 2, 128, 128) ||
      !encode_2d(&maps.m[1], b.q, 1, p.k / 2, b.rows, p.k / 2, 128, 128) ||
      !encode_2d(&maps.m[2], a.scale, 2, 256, div_up(a.rows, 128) * kt, 512, 256, 2, false) ||
      !encode_2d(&maps.m[3], b.scale, 2, 256, div_up(b.rows, 128) * kt, 512, 256, 2, false))
    return MOE_B200_ERR_DRIVER;
  maps.m[4] = maps.m[5] = maps.m[0];
  return gate ? launch_pair<true, false, kEpiGatedQuant>(maps, grp, sm_count, dependent, s)
              : launch_pair<true, false, kEpiStore>(maps, grp, sm_count, dependent, s);
}

}  // namespace moe
