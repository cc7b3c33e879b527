// Microscaled 4-bit GEMM (e2m1 elements, a scale per block of K) with the 8-bit GEMMs'
// epilogues, for sm_100a (tcgen05 block-scaled tensor-core products, TMEM accumulators).
//
//   acc[m, n] = sum_b sx[m, b] sw[n, b] sum_{k in b} x[m, k] w[n, k]      (fp32 accumulation)
//   out[m, n] = cast( ((acc * xs[m]) * ws[n or 0]) + bias[n] )            (xs, ws optional)
//   gated: out[m, n] = bf16( res[m, n] + gate[g(m), n] * (the value above before its cast) )
// The gated form rounds once: keeping torch's three bf16 roundings, as the 8-bit sibling does, costs
// 1.5 times the error (2.6e-3 against 1.7e-3 of the result's norm at K = 12288).
//
//   mxfp4: blocks of 32, power-of-two scales (e8m0);  nvfp4: blocks of 16, e4m3 scales.
// Two codes a byte (even k in the low half), so a 128-byte swizzled row of shared memory holds
// 256 elements and one MMA (K = 64) reads 32 bytes of it, as the 8-bit kinds do: the operand
// side is the 8-bit GEMM's, byte for byte.  The block scales come in tiles of 128 rows x 4
// blocks (512 bytes, row r and block b at (r % 32) * 16 + (r / 32) * 4 + b), tiles of a row
// group consecutive along K: one such tile is what tcgen05.cp moves into four TMEM columns, so
// a stage's scales are one contiguous copy per row group and need no rearrangement.
#pragma once

#include "gemm.cuh"

namespace t8g {
namespace gemm4 {

using gemm::BK;
using gemm::BM;
using gemm::kOutBF16;
using gemm::kOutF16;
using gemm::kOutF32;
using gemm::kOutGated;
using gemm::NUM_THREADS;
using gemm::OutTraits;

constexpr int kStageK = 2 * BK;    // elements of K per stage (one 128-byte row)
constexpr int kMmaK = 64;          // elements of K per MMA
constexpr int kScaleTile = 512;    // bytes of a 128-row x 4-block scale tile

// Scale tiles per row group and stage: 256 elements are 8 (mxfp4) or 16 (nvfp4) blocks.
__host__ __device__ constexpr int stage_tiles(bool mx) { return mx ? 2 : 4; }

struct Args : gemm::Args {
  int kstages;      // stages along K (the last one may be partial)
  int last_steps;   // MMAs of the last stage (1..4)
  void* out;        // kernels that store directly: out and its row stride in elements
  int64_t ld_out;
};

// Shared-memory descriptors of stage 0; a stage further on adds its bytes / 16 to the address field
// (14 bits, which hold any shared-memory address / 16, so the sum never leaves it).
struct StageDescs {
  uint64_t a, b, sfa, sfb;
};

// One stage's work of the MMA warp, issued by one elected lane: its scales to TMEM, then STEPS K = 64
// products.  `sa_t` / `sb_t`: TMEM columns of A's scales (4 per tile) and B's (4 * B_GROUPS per
// tile), B's moved by `sb_off` to this output tile's rows.
template <bool MX, bool PAIR, int B_GROUPS, int STEPS>
__device__ __forceinline__ void stage_scales_n(const StageDescs& d, uint32_t sa_t, uint32_t sb_t) {
  constexpr int kTiles = stage_tiles(MX);
  constexpr int kUsed = MX ? (STEPS + 1) / 2 : STEPS;
#pragma unroll
  for (int t = 0; t < kUsed; ++t) {
    tmem_cp_scales<PAIR>(sa_t + 4u * t, d.sfa + t * (kScaleTile / 16));
#pragma unroll
    for (int g = 0; g < B_GROUPS; ++g)
      tmem_cp_scales<PAIR>(sb_t + 4u * (B_GROUPS * t + g), d.sfb + (g * kTiles + t) * (kScaleTile / 16));
  }
}
template <bool MX, bool PAIR, int B_GROUPS, int STEPS>
__device__ __forceinline__ void stage_products_n(uint32_t d_tmem, const StageDescs& d, uint32_t sa_t, uint32_t sb_t,
                                                 uint32_t sb_off, uint32_t idesc, uint32_t accumulate) {
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const uint32_t t = MX ? k >> 1 : k;
    const uint32_t id = MX ? static_cast<uint32_t>(k & 1) * ((2u << 29) | (2u << 4)) : 0u;
    mma_fp4<MX, PAIR>(d_tmem, d.a + 2 * k, d.b + 2 * k, idesc | id, sa_t + 4u * t, sb_t + 4u * B_GROUPS * t + sb_off,
                      k == 0 ? accumulate : 1u);
  }
}

template <bool MX, bool PAIR, int B_GROUPS>
__device__ __forceinline__ void stage_mmas(uint32_t d_tmem, const StageDescs& d, uint32_t sa_t, uint32_t sb_t,
                                           uint32_t sb_off, uint32_t idesc, int steps, uint32_t accumulate) {
#define T8G_STAGE(STEPS)                                                                            \
  stage_scales_n<MX, PAIR, B_GROUPS, STEPS>(d, sa_t, sb_t);                                         \
  stage_products_n<MX, PAIR, B_GROUPS, STEPS>(d_tmem, d, sa_t, sb_t, sb_off, idesc, accumulate)
  if (steps == 4) {
    T8G_STAGE(4);
  } else if (steps == 3) {
    T8G_STAGE(3);
  } else if (steps == 2) {
    T8G_STAGE(2);
  } else {
    T8G_STAGE(1);
  }
#undef T8G_STAGE
}

// ---------------------------------------------------------------- 1-SM kernel
// For outputs of few tiles: one 128 x TBN tile per cluster of S CTAs (1..8) that split K.  Each CTA
// leaves its partial tile in its shared memory; the tile's pieces of eight columns are dealt over
// the threads of all S CTAs, and a thread sums its pieces over the partial tiles in rank
// order (a fixed order, so results repeat) through distributed shared memory.
// A tile has `arows` rows of A to load (the rows of M, a multiple of 8): a box that reaches past M
// by most of its rows loads several times slower, and its slot would hold nothing.  The MMA
// still reads 128 rows, whatever the ring holds there: those rows' sums are not stored.
// About 104 KB a CTA, so that two share an SM and one's start and end overlap the other's stream.
constexpr int kSmallMaxStages = 16;
constexpr uint32_t kSmallSmem = 104 * 1024;

template <bool MX, int TBN>
struct SmallCfg {
  static constexpr uint32_t kTiles = stage_tiles(MX);
  static constexpr uint32_t kBBytes = TBN * BK;
  static constexpr uint32_t kSfBytes = kTiles * kScaleTile;   // per operand (one 128-row group)
  static constexpr uint32_t kSfCols = 2u * 4u * kTiles;       // A's and B's scale columns of a stage
  static constexpr uint32_t kTmemCols = TBN + 2 * kSfCols <= 128 ? 128 : 256;   // scales double-buffered
  static constexpr uint32_t kPitch = TBN + 4;                 // floats per row of a partial tile
  __host__ __device__ static constexpr uint32_t stage_bytes(uint32_t arows) { return arows * BK + kBBytes + 2 * kSfBytes; }
  __host__ __device__ static constexpr uint32_t partial_bytes(uint32_t rows) { return rows * kPitch * 4; }
};

// Eight output columns [n, n + 8) of row m from their sums (fewer at the right edge).
template <int OUT>
__device__ __forceinline__ void store_eight(const Args& a, int m, int n, float (&f)[8]) {
  const float xs = a.xs ? __ldg(a.xs + m) : 1.f;
  const int left = a.N - n;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int c = min(n + j, a.N - 1);
    f[j] = __fmul_rn(__fmul_rn(f[j], xs), a.ws ? __ldg(a.ws + (a.ws_stride ? c : 0)) : 1.f);
    if (a.bias != nullptr) f[j] = __fadd_rn(f[j], OutTraits<OUT>::to_f32(a.bias, c));
  }
  const int64_t at = static_cast<int64_t>(m) * a.ld_out + n;
  if constexpr (OUT == kOutF32) {
    float* o = static_cast<float*>(a.out) + at;
    if (left >= 8) {
      reinterpret_cast<float4*>(o)[0] = make_float4(f[0], f[1], f[2], f[3]);
      reinterpret_cast<float4*>(o)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < left) o[j] = f[j];
    }
  } else {
    if constexpr (OUT == kOutGated) {   // N is a multiple of 8
      const int64_t grow = a.gate_index ? static_cast<int64_t>(__ldg(a.gate_index + m)) : m / a.rows_per_gate;
      const uint4 g4 = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.gate) + grow * a.ld_gate + n));
      // res may be out itself: an ordinary load
      const uint4 r4 = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.res) + static_cast<int64_t>(m) * a.ld_res + n);
      const uint32_t gw[4] = {g4.x, g4.y, g4.z, g4.w}, rw[4] = {r4.x, r4.y, r4.z, r4.w};
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const float2 o = fma2_rn(bf2_to_f2(gw[p]), make_float2(f[2 * p], f[2 * p + 1]), bf2_to_f2(rw[p]));
        f[2 * p] = o.x;
        f[2 * p + 1] = o.y;
      }
    }
    uint32_t h[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) h[p] = OutTraits<OUT>::pack2(f[2 * p], f[2 * p + 1]);
    uint16_t* o = static_cast<uint16_t*>(a.out) + at;
    if (left >= 8) {
      *reinterpret_cast<uint4*>(o) = make_uint4(h[0], h[1], h[2], h[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < left) o[j] = static_cast<uint16_t>(h[j / 2] >> (16 * (j & 1)));
    }
  }
}

template <bool MX, int OUT, int TBN>
__global__ void __launch_bounds__(NUM_THREADS, 2)
    gemm_fp4_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                    const __grid_constant__ CUtensorMap tm_sfa, const __grid_constant__ CUtensorMap tm_sfb,
                    const Args args, const int S, const uint32_t arows, const int stages) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kSmallMaxStages], empty[kSmallMaxStages], done;
  __shared__ uint32_t tmem_slot;
  using C = SmallCfg<MX, TBN>;
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  // rings: A, B, A's scales, B's scales (every slot a multiple of 1024 bytes)
  const uint32_t a_bytes = arows * BK;
  uint8_t* ring_b = smem + stages * a_bytes;
  uint8_t* ring_sfa = ring_b + stages * C::kBBytes;
  uint8_t* ring_sfb = ring_sfa + stages * C::kSfBytes;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x) % S;
  const int tile = static_cast<int>(blockIdx.x) / S;
  const int tiles_n = (args.N + TBN - 1) / TBN;
  const int tm = tile / tiles_n;
  const int tn = tile - tm * tiles_n;
  const int kb0 = static_cast<int>(static_cast<int64_t>(args.kstages) * rank / S);
  const int kb1 = static_cast<int>(static_cast<int64_t>(args.kstages) * (rank + 1) / S);

  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(&done, 1);
    fence_mbarrier_init();
    prefetch_tensormap(&tm_a);
    prefetch_tensormap(&tm_b);
    prefetch_tensormap(&tm_sfa);
    prefetch_tensormap(&tm_sfb);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;

  bool have = false;   // epilogue warps: the accumulator is complete
  if (warp == 0) {
    if (lane == 0) {
      const uint64_t pol_a = policy_evict_normal();
      const uint64_t pol_b = policy_evict_last();
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_sleep(&empty[stage], phase ^ 1u, kStatusTimeoutProducer)) break;
        mbar_arrive_expect_tx(&full[stage], C::stage_bytes(arows));
        tma_load_2d(ring_b + stage * C::kBBytes, &tm_b, &full[stage], kb * BK, tn * TBN, pol_b);
        tma_load_2d(ring_sfb + stage * C::kSfBytes, &tm_sfb, &full[stage], kb * (static_cast<int>(C::kSfBytes) / 8),
                    tn * TBN / BM, pol_b);
        tma_load_2d(smem + stage * a_bytes, &tm_a, &full[stage], kb * BK, tm * BM, pol_a);
        tma_load_2d(ring_sfa + stage * C::kSfBytes, &tm_sfa, &full[stage], kb * (static_cast<int>(C::kSfBytes) / 8), tm,
                    pol_a);
        ++issued;
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      // every issued copy must land before the CTA may exit
      for (int i = 0; i < stages && i < issued; ++i) {
        const int n = issued - 1 - i;
        if (!mbar_wait_sleep(&full[n % stages], static_cast<uint32_t>((n / stages) & 1), kStatusTimeoutDrain)) break;
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = make_idesc_fp4(MX, BM, TBN);
    const uint32_t sb_off = static_cast<uint32_t>(tn * TBN % BM / 32);
    const StageDescs d0 = {smem_desc_k_sw128(smem_u32(smem)), smem_desc_k_sw128(smem_u32(ring_b)),
                           smem_desc_scales(smem_u32(ring_sfa)), smem_desc_scales(smem_u32(ring_sfb))};
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait_warp(&full[stage], phase, kStatusTimeoutMma)) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t sa_t = tmem_base + TBN + static_cast<uint32_t>(kb & 1) * C::kSfCols;
        const uint32_t i = static_cast<uint32_t>(stage);
        const StageDescs d = {d0.a + i * (a_bytes / 16), d0.b + i * (C::kBBytes / 16), d0.sfa + i * (C::kSfBytes / 16),
                              d0.sfb + i * (C::kSfBytes / 16)};
        stage_mmas<MX, false, 1>(tmem_base, d, sa_t, sa_t + 4u * C::kTiles, sb_off, idesc,
                                 kb == args.kstages - 1 ? args.last_steps : kStageK / kMmaK, kb != kb0);
        tc_commit(&empty[stage]);
        if (kb == kb1 - 1) tc_commit(&done);
      }
      __syncwarp();
      if (++stage == stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    // every MMA (and its shared-memory reads) completes before teardown; a wait that gave up leaves
    // `done` to the waits' own limits
    mbar_wait_warp(&done, 0, kStatusTimeoutDrain);
  } else {
    have = mbar_wait_warp(&done, 0, kStatusTimeoutEpilogue);
    tc_fence_after();
  }

  // The rings' slots are all consumed once `done` completed: the partial tile goes there.
  float* part = reinterpret_cast<float*>(smem);
  const int rows = min(BM, args.M - tm * BM);
  const int quarter = warp & 3;
  if (warp >= 2 && quarter * 32 < rows) {
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    float* prow = part + static_cast<uint32_t>(quarter * 32 + lane) * C::kPitch;
#pragma unroll
    for (int c = 0; c < TBN; c += 32) {
      uint32_t r[32];
      tmem_ld_32x32b_x32(t_row + static_cast<uint32_t>(c), r);
      tmem_ld_wait_regs(r);
      if (quarter * 32 + lane < rows) {
#pragma unroll
        for (int j = 0; j < 32; j += 4)
          *reinterpret_cast<uint4*>(prow + c + j) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
      }
    }
  }
  __syncwarp();
  if (S > 1)
    cluster_sync();
  else
    __syncthreads();
  if (warp >= 2 && have) {
    constexpr int kPieces = TBN / 8;
    for (int u = rank * 128 + static_cast<int>(threadIdx.x) - 64; u < rows * kPieces; u += S * 128) {
      const int rr = u / kPieces;
      const int cc = (u - rr * kPieces) * 8;
      const int n = tn * TBN + cc;
      if (n >= args.N) continue;
      const float* at = part + static_cast<uint32_t>(rr) * C::kPitch + cc;
      float f[8];
      if (S == 1) {
        const float4 lo = reinterpret_cast<const float4*>(at)[0], hi = reinterpret_cast<const float4*>(at)[1];
        f[0] = lo.x, f[1] = lo.y, f[2] = lo.z, f[3] = lo.w, f[4] = hi.x, f[5] = hi.y, f[6] = hi.z, f[7] = hi.w;
      } else {
        const uint32_t addr = smem_u32(at);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = 0.f;
#pragma unroll 4
        for (int q = 0; q < S; ++q) {
          const uint32_t p = mapa_shared(addr, static_cast<uint32_t>(q));
          const float4 lo = ld_cluster_f32x4(p), hi = ld_cluster_f32x4(p + 16);
          f[0] = __fadd_rn(f[0], lo.x), f[1] = __fadd_rn(f[1], lo.y), f[2] = __fadd_rn(f[2], lo.z);
          f[3] = __fadd_rn(f[3], lo.w), f[4] = __fadd_rn(f[4], hi.x), f[5] = __fadd_rn(f[5], hi.y);
          f[6] = __fadd_rn(f[6], hi.z), f[7] = __fadd_rn(f[7], hi.w);
        }
      }
      store_eight<OUT>(args, tm * BM + rr, n, f);
    }
  }
  __syncwarp();
  if (S > 1) cluster_sync();   // no CTA leaves while another reads its partial tile

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
}

// ---------------------------------------------------------------- 2-SM kernel
// The 8-bit pair kernel's scheme (gemm.cuh): a cluster of two CTAs computes 256 x 256 tiles with
// cta_group::2 MMAs, persistent over tiles.  What differs is the room in TMEM: two 256-column
// accumulators would leave no columns for the scales.  The accumulators therefore overlap by kOver
// columns,
//     [0, 256)   [256 - kOver, 512 - kOver)   scales [512 - kOver, 512)
// and a tile's epilogue reads the shared columns first and then reports them free, so that the next tile's
// MMAs wait for one chunk of the epilogue, not for all of it.  (Tiles of 192 columns would need no
// overlap, but feed the tensor cores 17 % more operand bytes per product.)
// A CTA needs its own 128 rows' scales of A but those of all 256 rows of W: both CTAs load them.
//
// Eight epilogue warps share a CTA's half of a tile: warp 2 + 4 h + i reads the 32 lanes 32 ((2 + i) % 4) .. of columns [128 h, 128 h + 128).
constexpr int kEpiWarps = 8;
constexpr int kPairThreads = 64 + 32 * kEpiWarps;
constexpr int kHalfCols = gemm::BN / 2;

// Channel parameters of a tile: weight scales and the bias in the output type.
template <int OUT>
struct PairParams {
  float ws[gemm::BN];
  uint32_t bias[gemm::BN * OutTraits<OUT>::kBytes / 4];
};

template <bool MX, int OUT>
struct PairCfg {
  static constexpr int kTiles = stage_tiles(MX);
  static constexpr int kABytes = 128 * BK;
  static constexpr int kBBytes = 128 * BK;
  static constexpr int kSfaBytes = kTiles * kScaleTile;
  static constexpr int kSfbBytes = 2 * kTiles * kScaleTile;
  static constexpr int kStageBytes = kABytes + kBBytes + kSfaBytes + kSfbBytes;
  static constexpr int kEpiBufs = OUT == kOutGated ? 2 : 1;   // 4 KB pieces per warp (gated: its whole residual slice)
  static constexpr int kStages = (OUT == kOutGated || (!MX && OUT == kOutF32)) ? 4 : 5;
  static constexpr int kOver = MX ? 32 : 64;             // >= 12 kTiles scale columns
  struct Smem {
    uint8_t a[kStages][kABytes];
    uint8_t b[kStages][kBBytes];
    alignas(1024) uint8_t epi[kEpiWarps][kEpiBufs][4096];
    uint8_t gate[kEpiWarps][OUT == kOutGated ? 2 * kHalfCols : 16];
    alignas(128) uint8_t sfa[kStages][kSfaBytes];
    alignas(128) uint8_t sfb[kStages][kSfbBytes];
    PairParams<OUT> params[2];
    uint64_t full[kStages];
    uint64_t empty[kStages];
    uint64_t tmem_full[2];
    uint64_t shared_free;
    uint64_t drain;
    uint32_t tmem_base;
  };
  static constexpr size_t kSmemBytes = sizeof(Smem) + 1024;
  static_assert(kSmemBytes <= 227 * 1024, "shared memory");
  static_assert(12 * kTiles <= kOver, "the scales fit the columns between the accumulators");
};

// ws (1 without weight scales) and bias (0 without one) of the tile's columns.
template <int OUT>
__device__ __forceinline__ void stage_params(const Args& args, int n_tile0, int e, PairParams<OUT>& tp) {
  static_assert(gemm::BN == 32 * kEpiWarps, "one column per epilogue thread");
  const int n = n_tile0 + e;
  const bool in = n < args.N;
  tp.ws[e] = args.ws == nullptr ? 1.f : in ? __ldg(args.ws + (args.ws_stride ? n : 0)) : 0.f;
  if constexpr (OUT == kOutF32)
    tp.bias[e] = (in && args.bias) ? static_cast<const uint32_t*>(args.bias)[n] : 0u;
  else
    reinterpret_cast<uint16_t*>(tp.bias)[e] = (in && args.bias) ? static_cast<const uint16_t*>(args.bias)[n] : 0;
}

// Gated form: the residual rows of a warp's 32 x 128 slice are copied into its staging pieces (the
// layout of the stores: 16-byte piece q of row r at q ^ (r & 7)) while the tile's MMAs run, each
// then replaced by the output and stored from there; a gate row that all 32 rows share is
// copied beside them.
struct GatedSlice {
  const uint16_t* gate_row;   // this lane's gate row at the slice's first column (null: row >= M)
  bool shared_gate;           // every valid row of the warp uses lane 0's gate row
};
__device__ __forceinline__ GatedSlice gated_prefetch(const Args& args, uint8_t (*rbuf)[4096], uint8_t* gbuf, int row0,
                                                     int n0, int lane) {
  GatedSlice g;
  const int m = row0 + lane;
  const int cols = args.N - n0;   // may be <= 0
  int64_t grow = -1;
  if (m < args.M) grow = args.gate_index ? static_cast<int64_t>(__ldg(args.gate_index + m)) : m / args.rows_per_gate;
  g.gate_row = m < args.M ? static_cast<const uint16_t*>(args.gate) + grow * args.ld_gate + n0 : nullptr;
  const int64_t grow0 = __shfl_sync(0xffffffffu, grow, 0);
  g.shared_gate = __all_sync(0xffffffffu, m >= args.M || grow == grow0);
  if (lane == 0) bulk_wait_group_read<0>();   // the previous tile's stores have read the pieces
  __syncwarp();
  // eight lanes copy 128 consecutive bytes of a row, four rows at a time (a lane copying its own row read every
  // sector twice: nvfp4 32768 x 3072 x 3072 175 us, 151 so; x 12288: 455, 444)
  const int q = lane & 7, r0 = lane >> 3;
  const uint16_t* src = static_cast<const uint16_t*>(args.res) + static_cast<int64_t>(row0 + r0) * args.ld_res + n0 + 8 * q;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = r0 + 4 * i;
#pragma unroll
    for (int c = 0; c < kHalfCols / 64; ++c) {
      const bool in = row0 + row < args.M && c * 64 + 8 * q < cols;
      cp_async_16(rbuf[c] + row * 128 + ((q ^ (row & 7)) * 16),
                  in ? static_cast<const void*>(src + c * 64) : gemm::rbuf_src_dummy(), in ? 16u : 0u);
    }
    src += 4 * args.ld_res;
  }
  if (g.shared_gate && lane < kHalfCols / 8) {
    const uint16_t* g0 = static_cast<const uint16_t*>(args.gate) + grow0 * args.ld_gate + n0;
    const bool in = 8 * lane < cols;
    cp_async_16(gbuf + lane * 16, in ? static_cast<const void*>(g0 + 8 * lane) : gemm::rbuf_src_dummy(), in ? 16u : 0u);
  }
  cp_async_commit();
  return g;
}

// The columns of a staged piece row past its last whole 16 bytes before N: `left` columns from n on.
template <int OUT>
__device__ __noinline__ void store_tail(const Args& args, const uint8_t* buf, int lane, int row0, int n, int left) {
  constexpr int kBytes = OutTraits<OUT>::kBytes;
  constexpr int kPer = 16 / kBytes;
  const uint8_t* last = buf + lane * 128 + ((left / kPer) ^ (lane & 7)) * 16;
  uint8_t* out = static_cast<uint8_t*>(args.out) + (static_cast<int64_t>(row0 + lane) * args.ld_out + n + left / kPer * kPer) * kBytes;
  for (int j = 0; j < left % kPer; ++j) {
    if constexpr (kBytes == 4)
      reinterpret_cast<uint32_t*>(out)[j] = reinterpret_cast<const uint32_t*>(last)[j];
    else
      reinterpret_cast<uint16_t*>(out)[j] = reinterpret_cast<const uint16_t*>(last)[j];
  }
}

// A warp's report that its reads of TMEM so far are done: what the MMAs behind `bar` (a cluster address) may
// overwrite.  Every lane's loads are complete (tcgen05.wait::ld) and ordered before the arrival by its own fence.
__device__ __forceinline__ void report_read(uint32_t bar, int lane) {
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive_cluster_relaxed(bar);
}

// Epilogue of a warp's 32 x 128 slice of a tile (columns n0 .. of the output, `half` of the tile).
// `shared`: this half holds the columns that the other accumulator uses too, its last ones if half is
// 1 and its first if it is 0; they are read first and `shared_bar` (the leader's, a cluster
// address) is then told.
// SCALED: the values are multiplied by row and weight scales.
template <bool MX, int OUT, bool SCALED>
__device__ __forceinline__ void epilogue_pair(const Args& args, const CUtensorMap* tm_out,
                                              typename PairCfg<MX, OUT>::Smem& s, int ew, int half,
                                              const GatedSlice& gs, uint32_t t_row, int row0, int n0, int lane,
                                              uint64_t pol_out, float xs_r, const PairParams<OUT>& tp, bool shared,
                                              uint32_t shared_bar) {
  // 64 columns at a time; 32 for 4-byte outputs (a 128-byte piece of a row) and in mxfp4's gated form, whose
  // accumulators share 32 columns and are told free that much earlier (16384 x 9216 x 3072: 198 us, 206 with 64;
  // nvfp4 shares 64: 222, 216)
  constexpr int kCols = (OUT == kOutF32 || (OUT == kOutGated && MX)) ? 32 : 64;
  constexpr int kPieceChunks = OUT == kOutGated ? 64 / kCols : 1;
  constexpr int kChunks = kHalfCols / kCols;
  constexpr int kFirst = (PairCfg<MX, OUT>::kOver + kCols - 1) / kCols;   // chunks that hold the shared columns
  const bool has_bias = args.bias != nullptr;
  const float2 xs2 = make_float2(xs_r, xs_r);
  const int cols = args.N - n0;
  uint32_t r[kCols / 32][32];
  auto load = [&](int i) {
    const int c = half ? kChunks - 1 - i : i;
#pragma unroll
    for (int h = 0; h < kCols / 32; ++h) tmem_ld_32x32b_x32(t_row + static_cast<uint32_t>(c * kCols + 32 * h), r[h]);
  };
  load(0);
#pragma unroll 1
  for (int i = 0; i < kChunks; ++i) {
    const int c = half ? kChunks - 1 - i : i;
#pragma unroll
    for (int h = 0; h < kCols / 32; ++h) tmem_ld_wait_regs(r[h]);
    float v[kCols];
#pragma unroll
    for (int j = 0; j < kCols; ++j) v[j] = __uint_as_float(r[j / 32][j % 32]);
    if (shared && i == kFirst - 1) report_read(shared_bar, lane);   // the next tile's MMAs wait for this
    if (i + 1 < kChunks) load(i + 1);
    if constexpr (OUT == kOutGated) {
      if (i == 0) {   // the residual is in (the next tile's MMAs do not wait for it)
        cp_async_wait_all();
        __syncwarp();
      }
    }
    if (c * kCols >= cols) continue;
    const float4* wq = reinterpret_cast<const float4*>(tp.ws + half * kHalfCols + c * kCols);
    uint8_t* buf = s.epi[ew][OUT == kOutGated ? c / kPieceChunks : 0];
    if constexpr (OUT == kOutGated) {
      const uint4* bq2 = reinterpret_cast<const uint4*>(tp.bias + (half * kHalfCols + c * kCols) / 2);
#pragma unroll
      for (int q = 0; q < kCols / 8; ++q) {
        const float4 w0 = SCALED ? wq[2 * q] : float4{}, w1 = SCALED ? wq[2 * q + 1] : float4{};
        const float2 wp[4] = {make_float2(w0.x, w0.y), make_float2(w0.z, w0.w), make_float2(w1.x, w1.y),
                              make_float2(w1.z, w1.w)};
        const uint4 b4 = has_bias ? bq2[q] : make_uint4(0, 0, 0, 0);
        const uint32_t bw[4] = {b4.x, b4.y, b4.z, b4.w};
        const int col = c * kCols + 8 * q;
        uint4* cell = reinterpret_cast<uint4*>(buf + lane * 128 + (((q + c % kPieceChunks * 4) ^ (lane & 7)) * 16));
        const uint4 r4 = *cell;
        uint4 g4 = make_uint4(0, 0, 0, 0);
        if (gs.shared_gate)
          g4 = *reinterpret_cast<const uint4*>(s.gate[ew] + (c * (kCols / 8) + q) * 16);
        else if (gs.gate_row != nullptr && col < cols)
          g4 = __ldg(reinterpret_cast<const uint4*>(gs.gate_row + col));
        const uint32_t rw[4] = {r4.x, r4.y, r4.z, r4.w};
        const uint32_t gw[4] = {g4.x, g4.y, g4.z, g4.w};
        uint32_t o[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          float2 f = make_float2(v[8 * q + 2 * p], v[8 * q + 2 * p + 1]);
          if constexpr (SCALED) f = mul2_rn(mul2_rn(f, xs2), wp[p]);
          if (has_bias) f = add_f32_bf16x2(f, bw[p]);
          o[p] = f2_to_bf2(fma2_rn(bf2_to_f2(gw[p]), f, bf2_to_f2(rw[p])));
        }
        *cell = make_uint4(o[0], o[1], o[2], o[3]);
      }
    } else {
      // eight 16-byte pieces of the row: four fp32 or eight two-byte outputs each
      const uint4* bq = reinterpret_cast<const uint4*>(tp.bias + (half * kHalfCols + c * kCols) * OutTraits<OUT>::kBytes / 4);
      uint4 o[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        if constexpr (OUT == kOutF32) {
          const uint4 b4 = bq[q];
          float2 f0 = make_float2(v[4 * q], v[4 * q + 1]), f1 = make_float2(v[4 * q + 2], v[4 * q + 3]);
          if constexpr (SCALED) {
            const float4 w4 = wq[q];
            f0 = mul2_rn(mul2_rn(f0, xs2), make_float2(w4.x, w4.y));
            f1 = mul2_rn(mul2_rn(f1, xs2), make_float2(w4.z, w4.w));
          }
          if (has_bias) {
            f0 = make_float2(__fadd_rn(f0.x, __uint_as_float(b4.x)), __fadd_rn(f0.y, __uint_as_float(b4.y)));
            f1 = make_float2(__fadd_rn(f1.x, __uint_as_float(b4.z)), __fadd_rn(f1.y, __uint_as_float(b4.w)));
          }
          o[q] = make_uint4(__float_as_uint(f0.x), __float_as_uint(f0.y), __float_as_uint(f1.x), __float_as_uint(f1.y));
        } else {
          const float4 w0 = SCALED ? wq[2 * q] : float4{}, w1 = SCALED ? wq[2 * q + 1] : float4{};
          const float2 wp[4] = {make_float2(w0.x, w0.y), make_float2(w0.z, w0.w), make_float2(w1.x, w1.y),
                                make_float2(w1.z, w1.w)};
          const uint4 b4 = has_bias ? bq[q] : make_uint4(0, 0, 0, 0);
          const uint32_t bw[4] = {b4.x, b4.y, b4.z, b4.w};
          uint32_t h[4];
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            float2 f = make_float2(v[8 * q + 2 * p], v[8 * q + 2 * p + 1]);
            if constexpr (SCALED) f = mul2_rn(mul2_rn(f, xs2), wp[p]);
            if (has_bias) f = OUT == kOutF16 ? add_f32_f16x2(f, bw[p]) : add_f32_bf16x2(f, bw[p]);
            h[p] = OutTraits<OUT>::pack2(f.x, f.y);
          }
          o[q] = make_uint4(h[0], h[1], h[2], h[3]);
        }
      }
      if (lane == 0) bulk_wait_group_read<0>();   // the warp's previous store has read the piece
      __syncwarp();
#pragma unroll
      for (int q = 0; q < 8; ++q) *reinterpret_cast<uint4*>(buf + lane * 128 + ((q ^ (lane & 7)) * 16)) = o[q];
      // TMA stores whole 16-byte pieces: the map ends at the last whole one before N, and the columns
      // after it are stored one by one (what lies past N is not this call's to write)
      constexpr int kPer = 16 / OutTraits<OUT>::kBytes;
      const int left = cols - c * kCols;
      if (left < kCols && left % kPer != 0 && row0 + lane < args.M) store_tail<OUT>(args, buf, lane, row0, n0 + c * kCols, left);
    }
    if constexpr (kPieceChunks == 2) {
      // a piece is stored with its second chunk, or with its only one before N (the skipped one is the upper,
      // which the other half's order takes first)
      if (i % 2 == 0 && (half == 1 || (c + 1) * kCols < cols)) continue;
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_2d(tm_out, buf, n0 + c / kPieceChunks * (kPieceChunks * kCols), row0, pol_out);
      bulk_commit_group();
    }
  }
}

template <bool MX, int OUT, bool SCALED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    gemm_fp4_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                         const __grid_constant__ CUtensorMap tm_sfa, const __grid_constant__ CUtensorMap tm_sfb,
                         const __grid_constant__ CUtensorMap tm_out, const Args args) {
  extern __shared__ uint8_t smem_raw[];
  using C = PairCfg<MX, OUT>;
  using gemm::BN;
  using gemm::P_BM;
  const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
  typename C::Smem& s = *reinterpret_cast<typename C::Smem*>(smem_raw + pad);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int pair = static_cast<int>(blockIdx.x >> 1);
  const int npairs = static_cast<int>(gridDim.x >> 1);
  const int tiles_n = (args.N + BN - 1) / BN;
  const int num_tiles = (args.M + P_BM - 1) / P_BM * tiles_n;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    mbar_init(&s.tmem_full[0], 1);
    mbar_init(&s.tmem_full[1], 1);
    mbar_init(&s.shared_free, 2 * kEpiWarps);
    mbar_init(&s.drain, 1);
    fence_mbarrier_init();
    prefetch_tensormap(&tm_a);
    prefetch_tensormap(&tm_b);
    prefetch_tensormap(&tm_sfa);
    prefetch_tensormap(&tm_sfb);
    prefetch_tensormap(&tm_out);
  }
  if (warp == 1) {
    tmem_alloc_pair(&s.tmem_base, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();   // both CTAs' barriers initialised before any cross-CTA signal
  tc_fence_after();
  const uint32_t tmem_base = s.tmem_base;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    if (lane == 0) {
      const uint64_t pol_a = policy_evict_normal();
      const uint64_t pol_b = policy_evict_last();
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < num_tiles; tile += npairs) {
        const int tm = tile / tiles_n;
        const int tn = tile - tm * tiles_n;
        for (int kb = 0; kb < args.kstages; ++kb) {
          if (!mbar_wait_sleep(&s.empty[stage], phase ^ 1u, kStatusTimeoutProducer)) {
            ok = false;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(&s.full[stage], 2 * C::kStageBytes);
          const uint32_t bar = mapa_shared(smem_u32(&s.full[stage]), 0);
          tma_load_2d_pair(s.a[stage], &tm_a, bar, kb * BK, tm * P_BM + rank * 128, pol_a);
          tma_load_2d_pair(s.b[stage], &tm_b, bar, kb * BK, tn * BN + rank * 128, pol_b);
          tma_load_2d_pair(s.sfa[stage], &tm_sfa, bar, kb * (C::kSfaBytes / 8), tm * 2 + rank, pol_a);
          tma_load_2d_pair(s.sfb[stage], &tm_sfb, bar, kb * (C::kSfaBytes / 8), tn * 2, pol_b);
          ++issued;
          if (++stage == C::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // the leader sees every copy of the pair land on its `full` barriers
      if (rank == 0) {
        for (int i = 0; i < C::kStages && i < issued; ++i) {
          const int n = issued - 1 - i;
          if (!mbar_wait_sleep(&s.full[n % C::kStages], static_cast<uint32_t>((n / C::kStages) & 1), kStatusTimeoutDrain)) break;
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader only)
    if (rank == 0) {
      constexpr uint32_t idesc = make_idesc_fp4(MX, P_BM, BN);
      const uint32_t sa_t = tmem_base + 512u - C::kOver;
      const uint32_t sb_t = sa_t + 4u * C::kTiles;
      const StageDescs d0 = {smem_desc_k_sw128(smem_u32(s.a[0])), smem_desc_k_sw128(smem_u32(s.b[0])),
                             smem_desc_scales(smem_u32(s.sfa[0])), smem_desc_scales(smem_u32(s.sfb[0]))};
      int stage = 0, local = 0;
      uint32_t phase = 0;
      bool ok = true, any = false;
      for (int tile = pair; ok && tile < num_tiles; tile += npairs, ++local) {
        const int acc = local & 1;
        const uint32_t d_tmem = tmem_base + (acc ? 256u - C::kOver : 0u);
        int kb = 0;
        if (local > 0 && args.kstages > 1) {
          // The first stage's scales go to TMEM while the tile before still hands over the columns its
          // accumulator shares with this one.  (Its other columns were read before that tile's
          // epilogue began: every warp reports.)
          if (!mbar_wait_warp(&s.full[stage], phase, kStatusTimeoutMma)) break;
          tc_fence_after();
          const StageDescs d = {d0.a + stage * (C::kABytes / 16), d0.b + stage * (C::kBBytes / 16),
                                d0.sfa + stage * (C::kSfaBytes / 16), d0.sfb + stage * (C::kSfbBytes / 16)};
          if (elect_one()) stage_scales_n<MX, true, 2, 4>(d, sa_t, sb_t);
          __syncwarp();
          if (!mbar_wait_warp(&s.shared_free, static_cast<uint32_t>(local - 1) & 1u, kStatusTimeoutMma)) break;
          tc_fence_after();
          if (elect_one()) {
            stage_products_n<MX, true, 2, 4>(d_tmem, d, sa_t, sb_t, 0u, idesc, 0u);
            tc_commit_both(smem_u32(&s.empty[stage]));
          }
          __syncwarp();
          if (++stage == C::kStages) {
            stage = 0;
            phase ^= 1u;
          }
          kb = 1;
        } else if (local > 0) {
          if (!mbar_wait_warp(&s.shared_free, static_cast<uint32_t>(local - 1) & 1u, kStatusTimeoutMma)) break;
          tc_fence_after();
        }
        for (; kb < args.kstages; ++kb) {
          if (!mbar_wait_warp(&s.full[stage], phase, kStatusTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (elect_one()) {
            const StageDescs d = {d0.a + stage * (C::kABytes / 16), d0.b + stage * (C::kBBytes / 16),
                                  d0.sfa + stage * (C::kSfaBytes / 16), d0.sfb + stage * (C::kSfbBytes / 16)};
            stage_mmas<MX, true, 2>(d_tmem, d, sa_t, sb_t, 0u, idesc,
                                    kb == args.kstages - 1 ? args.last_steps : kStageK / kMmaK, kb != 0);
            tc_commit_both(smem_u32(&s.empty[stage]));
            if (kb == args.kstages - 1) tc_commit_both(smem_u32(&s.tmem_full[acc]));
          }
          __syncwarp();
          any = true;
          if (++stage == C::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (any) {
        if (elect_one()) tc_commit_pair(mapa_shared(smem_u32(&s.drain), 0));
        __syncwarp();
        mbar_wait_warp(&s.drain, 0, kStatusTimeoutDrain);
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int ew = warp - 2;
    const int half = ew >> 2;
    const int quarter = warp & 3;
    const int e = threadIdx.x - 64;
    const uint64_t pol_out = policy_evict_first();
    const uint32_t shared_bar = mapa_shared(smem_u32(&s.shared_free), 0);
    int local = 0;
    bool ok = true;
    for (int tile = pair; tile < num_tiles; tile += npairs, ++local) {
      const int tm = tile / tiles_n;
      const int tn = tile - tm * tiles_n;
      const int acc = local & 1;
      const int row0 = tm * P_BM + rank * 128 + quarter * 32;
      const int n0 = tn * BN + half * kHalfCols;
      // the shared columns are the upper half's of accumulator 0 and the lower half's of 1
      const bool shared = row0 < args.M && half != acc;
      stage_params<OUT>(args, tn * BN, e, s.params[acc]);
      const float xs_r = (row0 + lane < args.M && args.xs) ? __ldg(args.xs + row0 + lane) : 1.f;
      GatedSlice gs{};
      if constexpr (OUT == kOutGated) {
        if (row0 < args.M) gs = gated_prefetch(args, s.epi[ew], s.gate[ew], row0, n0, lane);
      }
      // all warps staged the parameters; they leave together if any wait for the tile before ran out
      if (named_bar_any(1, 32 * kEpiWarps, !ok)) break;
      ok = mbar_wait_warp(&s.tmem_full[acc], static_cast<uint32_t>((local >> 1) & 1), kStatusTimeoutEpilogue);
      tc_fence_after();
      // The other half, and a warp without rows, report as well, which tells that they are done with the tile
      // before.  Only now: this tile's MMAs began when the tile before had all its reports, so no warp's
      // report for this tile can be taken for a slower warp's for that one.
      if (ok && !shared) report_read(shared_bar, lane);
      if (ok && row0 < args.M) {
        const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + (acc ? 256u - C::kOver : 0u) +
                               static_cast<uint32_t>(half * kHalfCols);
        epilogue_pair<MX, OUT, SCALED>(args, &tm_out, s, ew, half, gs, t_row, row0, n0, lane, pol_out, xs_r, s.params[acc],
                                       shared, shared_bar);
      }
    }
    if constexpr (OUT == kOutGated) cp_async_wait_all();   // a residual copy left by a wait that gave up
    if (lane == 0) bulk_wait_group_all();
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();   // the pair's MMAs, copies and cross-CTA signals are all done
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

}  // namespace gemm4
}  // namespace t8g
