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
using gemm::EPI_COLS;
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

// MMAs of one stage: copy its scales to TMEM, then `steps` K = 64 products.  `sa_t` / `sb_t`:
// TMEM columns of A's scales (4 per tile) and B's (4 * B_GROUPS per tile); `sb_off`: first
// column of this tile's rows within B's scale word columns.
template <bool MX, bool PAIR, int B_GROUPS>
__device__ __forceinline__ void stage_mmas(uint32_t d_tmem, uint32_t a0, uint32_t b0, uint32_t sfa, uint32_t sfb,
                                           uint32_t sa_t, uint32_t sb_t, uint32_t sb_off, uint32_t idesc, int steps,
                                           bool first) {
  constexpr int kTiles = stage_tiles(MX);
  const int tiles = MX ? (steps + 1) >> 1 : steps;
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    if (t < tiles) {
      tmem_cp_scales<PAIR>(sa_t + 4u * t, smem_desc_scales(sfa + t * kScaleTile));
#pragma unroll
      for (int g = 0; g < B_GROUPS; ++g)
        tmem_cp_scales<PAIR>(sb_t + 4u * (B_GROUPS * t + g), smem_desc_scales(sfb + (g * kTiles + t) * kScaleTile));
    }
  }
#pragma unroll
  for (int k = 0; k < kStageK / kMmaK; ++k) {
    if (k < steps) {
      const uint32_t t = MX ? k >> 1 : k;
      const uint32_t id = MX ? static_cast<uint32_t>(k & 1) * ((2u << 29) | (2u << 4)) : 0u;
      mma_fp4<MX, PAIR>(d_tmem, smem_desc_k_sw128(a0 + k * 32), smem_desc_k_sw128(b0 + k * 32), idesc | id,
                        sa_t + 4u * t, sb_t + 4u * B_GROUPS * t + sb_off, (first && k == 0) ? 0u : 1u);
    }
  }
}

// ---------------------------------------------------------------- epilogue arithmetic
// One output element from its accumulator, in the 8-bit GEMMs' operation order.
template <int OUT>
__device__ __forceinline__ void store_one(const Args& a, int m, int n, float acc, float xs_r, int64_t grow) {
  float f = __fmul_rn(acc, xs_r);
  f = __fmul_rn(f, a.ws ? __ldg(a.ws + (a.ws_stride ? n : 0)) : 1.f);
  if (a.bias != nullptr) f = __fadd_rn(f, OutTraits<OUT>::to_f32(a.bias, n));
  const int64_t at = static_cast<int64_t>(m) * a.ld_out + n;
  if constexpr (OUT == kOutF32) {
    static_cast<float*>(a.out)[at] = f;
  } else if constexpr (OUT == kOutF16) {
    static_cast<__half*>(a.out)[at] = __float2half_rn(f);
  } else if constexpr (OUT == kOutBF16) {
    static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(f);
  } else {
    const float g = __bfloat162float(static_cast<const __nv_bfloat16*>(a.gate)[grow * a.ld_gate + n]);
    const float r = __bfloat162float(static_cast<const __nv_bfloat16*>(a.res)[static_cast<int64_t>(m) * a.ld_res + n]);
    static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(__fmaf_rn(g, f, r));
  }
}

// ---------------------------------------------------------------- 1-SM kernel
// One 128 x TBN output tile per cluster of gridDim-given size S (1..8): the S CTAs split K, each
// leaves its partial tile in its own shared memory, and CTA r sums columns [r, r + 1) * TBN / S of
// all partials in rank order (a fixed order, so results repeat) and stores them.
template <bool MX, int TBN>
struct Cfg {
  static constexpr int kTiles = stage_tiles(MX);
  static constexpr int kABytes = BM * BK;
  static constexpr int kBBytes = TBN * BK;
  static constexpr int kSfBytes = kTiles * kScaleTile;   // per operand (one 128-row group)
  static constexpr int kStageBytes = kABytes + kBBytes + 2 * kSfBytes;
  static constexpr int kStages = (200 * 1024) / kStageBytes;
  static constexpr uint32_t kSfCols = 2u * 4u * kTiles;  // A's and B's scale columns of a stage
  static constexpr uint32_t kTmemCols = TBN + 2 * kSfCols <= 128 ? 128 : 256;   // scales double-buffered
  static constexpr int kPitch = TBN + 1;                 // floats per row of a partial tile
  struct Smem {
    uint8_t a[kStages][kABytes];
    uint8_t b[kStages][kBBytes];
    alignas(1024) uint8_t sfa[kStages][kSfBytes];
    uint8_t sfb[kStages][kSfBytes];
    uint64_t full[kStages];
    uint64_t empty[kStages];
    uint64_t done;
    uint64_t drain;
    uint32_t tmem_base;
  };
  static constexpr size_t kSmemBytes = sizeof(Smem) + 1024;
  static_assert(kSmemBytes <= 227 * 1024, "shared memory");
  static_assert(static_cast<int>(sizeof(float)) * BM * kPitch <= kStages * kABytes, "partial tile fits the A ring");
};

template <bool MX, int OUT, int TBN>
__global__ void __launch_bounds__(NUM_THREADS, 1)
    gemm_fp4_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                    const __grid_constant__ CUtensorMap tm_sfa, const __grid_constant__ CUtensorMap tm_sfb,
                    const Args args, const int S) {
  extern __shared__ uint8_t smem_raw[];
  using C = Cfg<MX, TBN>;
  const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
  typename C::Smem& s = *reinterpret_cast<typename C::Smem*>(smem_raw + pad);
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
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    mbar_init(&s.done, 1);
    fence_mbarrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&s.tmem_base, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = s.tmem_base;

  bool have = false;   // epilogue warps: the accumulator is complete
  if (warp == 0) {
    if (lane == 0) {
      const uint64_t pol_a = policy_evict_normal();
      const uint64_t pol_b = policy_evict_last();
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&s.empty[stage], phase ^ 1u, kStatusTimeoutProducer)) break;
        mbar_arrive_expect_tx(&s.full[stage], C::kStageBytes);
        tma_load_2d(s.b[stage], &tm_b, &s.full[stage], kb * BK, tn * TBN, pol_b);
        tma_load_2d(s.sfb[stage], &tm_sfb, &s.full[stage], kb * (C::kSfBytes / 8), tn * TBN / BM, pol_b);
        tma_load_2d(s.a[stage], &tm_a, &s.full[stage], kb * BK, tm * BM, pol_a);
        tma_load_2d(s.sfa[stage], &tm_sfa, &s.full[stage], kb * (C::kSfBytes / 8), tm, pol_a);
        ++issued;
        if (++stage == C::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      // every issued copy must land before the CTA may exit
      for (int i = 0; i < C::kStages && i < issued; ++i) {
        const int n = issued - 1 - i;
        if (!mbar_wait(&s.full[n % C::kStages], static_cast<uint32_t>((n / C::kStages) & 1), kStatusTimeoutDrain)) break;
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = make_idesc_fp4(MX, BM, TBN);
      const uint32_t sb_off = static_cast<uint32_t>(tn * TBN % BM / 32);
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&s.full[stage], phase, kStatusTimeoutMma)) break;
        tc_fence_after();
        const uint32_t sa_t = tmem_base + TBN + static_cast<uint32_t>(kb & 1) * C::kSfCols;
        stage_mmas<MX, false, 1>(tmem_base, smem_u32(s.a[stage]), smem_u32(s.b[stage]), smem_u32(s.sfa[stage]),
                                 smem_u32(s.sfb[stage]), sa_t, sa_t + 4u * C::kTiles, sb_off, idesc,
                                 kb == args.kstages - 1 ? args.last_steps : kStageK / kMmaK, kb == kb0);
        tc_commit(&s.empty[stage]);
        if (++stage == C::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      tc_commit(&s.done);   // also when a wait gave up: completes once the issued MMAs have
      mbar_wait(&s.done, 0, kStatusTimeoutDrain);
    }
  } else {
    have = mbar_wait(&s.done, 0, kStatusTimeoutEpilogue);
    tc_fence_after();
  }

  const int quarter = warp & 3;
  const int row = quarter * 32 + lane;
  const int m = tm * BM + row;
  const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
  if (S == 1) {
    if (warp >= 2 && have) {
      const float xs_r = (m < args.M && args.xs) ? __ldg(args.xs + m) : 1.f;
      const int64_t grow = (OUT == kOutGated && m < args.M) ? (args.gate_index ? args.gate_index[m] : m / args.rows_per_gate) : 0;
      for (int c = 0; c < TBN; c += EPI_COLS) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(t_row + static_cast<uint32_t>(c), r);
        tmem_ld_wait_regs(r);
        if (m < args.M) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (tn * TBN + c + j < args.N) store_one<OUT>(args, m, tn * TBN + c + j, __uint_as_float(r[j]), xs_r, grow);
        }
      }
    }
  } else {
    // the A ring's stages are all consumed once `done` completed: the partial tile goes there
    float* part = reinterpret_cast<float*>(s.a);
    if (warp >= 2) {
      for (int c = 0; c < TBN; c += EPI_COLS) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(t_row + static_cast<uint32_t>(c), r);
        tmem_ld_wait_regs(r);
#pragma unroll
        for (int j = 0; j < 32; ++j) part[row * C::kPitch + c + j] = __uint_as_float(r[j]);
      }
    }
    __syncwarp();
    cluster_sync();
    if (warp >= 2 && have) {
      const int e = threadIdx.x - 64;
      const int cols = TBN / S;
      const int rows = min(BM, args.M - tm * BM);
      for (int i = e; i < rows * cols; i += 128) {
        const int rr = i / cols;
        const int cc = rank * cols + (i - rr * cols);
        const int n = tn * TBN + cc;
        if (n >= args.N) continue;
        const uint32_t at = smem_u32(part + rr * C::kPitch + cc);
        float acc = 0.f;
        for (int q = 0; q < S; ++q) acc = __fadd_rn(acc, ld_cluster_f32(mapa_shared(at, static_cast<uint32_t>(q))));
        const int mm = tm * BM + rr;
        const int64_t grow = OUT == kOutGated ? (args.gate_index ? args.gate_index[mm] : mm / args.rows_per_gate) : 0;
        store_one<OUT>(args, mm, n, acc, args.xs ? __ldg(args.xs + mm) : 1.f, grow);
      }
    }
    __syncwarp();
    cluster_sync();   // no CTA leaves while another reads its partial tile
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
}


}  // namespace gemm4
}  // namespace t8g
