// Row kernels of the microscaled 4-bit formats (bound by HBM and instruction issue): quantisation of bf16 rows, RMSNorm +
// modulation + quantisation, SwiGLU + quantisation, and the inverse.
//
// e2m1 values 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign, rounded to nearest (ties to the even
// code), saturating at 6; two codes a byte, the even column in the low half.
//   mxfp4: block of 32, scale 2^(floor(log2 amax) - 2), stored as its exponent + 127 (e8m0), at
//          least 0: from the bf16 exponent field e of amax it is max(e - 2, 0);
//   nvfp4: block of 16, row scale 2^r with the least r >= -100 that has amax(row) <= 6 * 448 * 2^r,
//          block scale e4m3(amax / (6 * 2^r)).
// The values quantised are bf16 (8 significant bits), also behind a norm or a SwiGLU, so that the
// fused forms give exactly what quantising their stored bf16 result gives (where that lies next to a border between
// two bf16 values, its float32 evaluation may round the other way than float64 would, and one code with it).  Every decision is
// then exact in fp32: mxfp4's x / scale is a shift; for nvfp4 x / scale either is one of the seven
// borders between e2m1 values or at least 2^-10 away from it (x and border * scale are both
// integers of at most 8 bits on a common grid), so a quotient rounded to a multiple of 2^-14, which the fp32 adder does
// (add and subtract 1.5 * 2^9), falls on the border exactly when x does (a negative x below 2^-15 of its scale becomes
// the code of +0, where -0 would be its rounding).
// A block with a NaN or an infinity has a NaN scale; a row with one has (nvfp4) a NaN row scale,
// so every product with that row is NaN.
//
// Scales are stored in tiles of 128 rows x 4 blocks (gemm_fp4.cuh).  Blocks past a row's last one, up to a
// multiple of 4, are written as 0 (their codes are read as 0, and 0 times a NaN scale would not
// be); rows past the last one are left as they were (they reach no output that is stored).
#pragma once

#include "rows.cuh"

namespace t8g {
namespace rows {

struct Fp4Out {
  uint8_t* q;        // [S, D / 2]
  int64_t ld_q;      // bytes
  uint8_t* sf;       // scale tiles
  float* q_scale;    // [S], nvfp4 only
  int64_t S;
  int words;         // 4-block scale words of a row
};

// Address of scale word 0 of a row; word w is 512 * w bytes on.
__host__ __device__ __forceinline__ int64_t scale_row(int64_t row, int words) {
  return (row >> 7) * words * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// max(|a|, |b|, |c|), NaN if any of them is.
__device__ __forceinline__ float max3_abs_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(fabsf(c)));
  return d;
}
// Largest magnitude of eight values; NaN if one is NaN.
__device__ __forceinline__ float absmax8(const float2 (&v)[4]) {
  const float a = max3_abs_nan(v[0].x, v[0].y, v[1].x);
  const float b = max3_abs_nan(v[1].y, v[2].x, v[2].y);
  return max3_abs_nan(max3_abs_nan(a, b, v[3].x), v[3].y, 0.f);
}
__device__ __forceinline__ uint32_t warp_max_u32(uint32_t v) {
  uint32_t r;
  asm volatile("redux.sync.max.u32 %0, %1, 0xffffffff;" : "=r"(r) : "r"(v));
  return r;
}

// nvfp4: the row scale 2^r from the row's largest magnitude (bf16 bits) and its inverse (0 for a row
// with a NaN or an infinity, whose scale is NaN).
__device__ __forceinline__ float row_scale_fp4(uint32_t amax, float* inverse) {
  if (amax >= 0x7F80u) {
    *inverse = 0.f;
    return __uint_as_float(0x7FC00000u);
  }
  // 6 * 448 = 1.3125 * 2^11, and 0.3125 is 40 / 128
  const int r = max(static_cast<int>(amax >> 7) - 127 - 11 + ((amax & 0x7Fu) > 40u ? 1 : 0), -100);
  *inverse = __uint_as_float(static_cast<uint32_t>(127 - r) << 23);
  return __uint_as_float(static_cast<uint32_t>(127 + r) << 23);
}

// The row scales of S rows of zeros.
__global__ void __launch_bounds__(256) zero_row_scales_fp4_kernel(float* q_scale, int64_t S) {
  float inverse;
  const float scale = row_scale_fp4(0u, &inverse);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; row < S;
       row += static_cast<int64_t>(gridDim.x) * blockDim.x)
    q_scale[row] = scale;
}

// Eight fp32 values -> eight e2m1 codes (first value in the lowest four bits).
__device__ __forceinline__ uint32_t cvt_e2m1x8(const float2 (&v)[4]) {
  uint32_t r;
  asm("{ .reg .b8 a, b, c, d;\n"
      "  cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n"
      "  cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      "  cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n"
      "  cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
      "  mov.b32 %0, {a, b, c, d}; }"
      : "=r"(r)
      : "f"(v[0].x), "f"(v[0].y), "f"(v[1].x), "f"(v[1].y), "f"(v[2].x), "f"(v[2].y), "f"(v[3].x), "f"(v[3].y));
  return r;
}
__device__ __forceinline__ float e4m3_to_f32(uint32_t byte) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(byte)));
  return __half2float(__ushort_as_half(static_cast<uint16_t>(h & 0xFFFFu)));
}
__device__ __forceinline__ float rcp_approx(float v) {   // within 1 ulp; see the 2^-14 rounding above
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// A lane's vector c of a row (c % 32 is the lane; vectors of a warp step are consecutive; zeros past the
// row's end), unpacked: the maximum of the block it lies in (4 lanes a block for mxfp4, 2 for nvfp4;
// every lane of the warp takes part).
template <bool MX>
__device__ __forceinline__ float block_max_fp4(const float2 (&v)[4]) {
  uint32_t b = __float_as_uint(absmax8(v));   // magnitudes compare as their bits, NaN above all
  b = max(b, __shfl_xor_sync(0xFFFFFFFFu, b, 1));
  if constexpr (MX) b = max(b, __shfl_xor_sync(0xFFFFFFFFu, b, 2));
  return __uint_as_float(b);
}

// The vector's eight codes and its block's scale byte, from the block's maximum.
template <bool MX>
__device__ __forceinline__ uint32_t codes_fp4(float2 (&v)[4], float amax, float row_inverse, uint32_t& byte) {
  if constexpr (MX) {
    const uint32_t b = __float_as_uint(amax);
    const int e = max(static_cast<int>(b >> 23) - 2, 0);
    const bool finite = b < 0x7F800000u;
    byte = finite ? static_cast<uint32_t>(e) : 255u;
    const float mult = finite ? __uint_as_float(static_cast<uint32_t>(254 - e) << 23) : 0.f;
#pragma unroll
    for (int p = 0; p < 4; ++p) v[p] = mul2_rn(v[p], make_float2(mult, mult));
  } else {
    // RN(t / 6) with one correction step (quant8 of rows.cuh), then e4m3
    const float t = __fmul_rn(amax, row_inverse);
    const float sixth = 1.0f / 6.0f;
    const float q0 = __fmul_rn(t, sixth);
    const float q1 = __fmaf_rn(__fmaf_rn(-6.0f, q0, t), sixth, q0);
    byte = cvt_e4m3x2(q1, 0.f);
    const float sb = e4m3_to_f32(byte);
    const float mult = sb > 0.f ? __fmul_rn(row_inverse, rcp_approx(sb)) : 0.f;
    const float2 mult2 = make_float2(mult, mult);
    constexpr float kGrid = 768.f;   // 1.5 * 2^9: one ulp is 2^-14
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const float2 y = fma2_rn(v[p], mult2, make_float2(kGrid, kGrid));
      v[p] = add2_rn(y, make_float2(-kGrid, -kGrid));
    }
  }
  return cvt_e2m1x8(v);
}

// Where a lane's vectors go: the same for every row of a kernel, so kept from row to row.  The vectors are
// c, c + step, ...; `step` is a multiple of 32, so their scale bytes are equally far apart.
struct Fp4Lane {
  int q0, q_step;     // byte of the codes within a row of q
  int sf0, sf_step;   // byte of the block's scale from the row's first one
  int steps;          // vectors of the warp: of at least one lane
  uint32_t codes;     // bit i: vector i exists
  uint32_t scales;    // bit i: this lane writes vector i's block scale
};
template <bool MX>
__device__ __forceinline__ Fp4Lane fp4_lane(int c, int step, int nvec, int n) {
  constexpr int kLanes = MX ? 4 : 2;   // per block
  Fp4Lane l;
  l.q0 = 4 * c;
  l.q_step = 4 * step;
  l.sf0 = 512 * (c / (4 * kLanes)) + ((c / kLanes) & 3);
  l.sf_step = 512 * (step / (4 * kLanes));
  l.codes = l.scales = 0u;
  const int first = c & ~31;
  l.steps = first < nvec ? (nvec - first + step - 1) / step : 0;
  for (int i = 0; i < n; ++i, c += step) {
    if (c < nvec) l.codes |= 1u << i;
    // blocks past the row's last, up to a multiple of four, get the 0 that vectors of zeros have
    if ((c & (kLanes - 1)) == 0 && (c & ~(4 * kLanes - 1)) < nvec) l.scales |= 1u << i;
  }
  return l;
}

// Codes and scale of a lane's vector i, stored.
template <bool MX>
__device__ __forceinline__ void store_vec_fp4(uint8_t* qrow, uint8_t* sfrow, const Fp4Lane& l, int i, float2 (&v)[4],
                                              float amax, float row_inverse) {
  uint32_t byte;
  const uint32_t codes = codes_fp4<MX>(v, amax, row_inverse, byte);
  if (l.codes >> i & 1u) *reinterpret_cast<uint32_t*>(qrow + l.q0 + i * l.q_step) = codes;
  if (l.scales >> i & 1u) sfrow[l.sf0 + i * l.sf_step] = static_cast<uint8_t>(byte);
}

// ---------------------------------------------------------------- direct row kernels
// Quantisation and norm: a row group of T threads per row with its V vectors a thread in registers
// (thread t holds vectors t, t + T, ...), loaded straight from global memory (quantisation: while the row
// before is worked on); a CTA holds as many groups as make 256 threads, a group takes consecutive
// rows.  No ring and no set-up: a single row takes one round trip to memory.  (T, V) is the canonical row-group shape, which makes
// the norm's sum of squares the 8-bit kernels', bit for bit.
__device__ __forceinline__ uint4 ld_stream_v4(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// Row maximum (bf16 bits) over a row group.
__device__ __forceinline__ uint32_t group_max_u32(const RowGroup& grp, uint32_t v, float* red) {
  v = warp_max_u32(v);
  if (grp.T == 32) return v;
  const int lane = grp.t & 31;
  if (lane == 0) red[grp.t >> 5] = __uint_as_float(v);
  group_sync(grp);
  return warp_max_u32(lane < (grp.T >> 5) ? __float_as_uint(red[lane]) : 0u);
}

// Quantises the V vectors a thread of the group holds (zeros past the row's end).  The row's maximum
// comes from the block maxima, which the scales need anyway.
template <bool MX, int V>
__device__ __forceinline__ void group_quant_fp4(const RowGroup& grp, const Fp4Out& o, int64_t row, const uint4 (&u)[V],
                                                const Fp4Lane& lane, float* red) {
  uint8_t* qrow = o.q + row * o.ld_q;
  uint8_t* sfrow = o.sf + scale_row(row, o.words);
  float top[V];
  float inverse = 0.f;
  if constexpr (!MX) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (i >= lane.steps) break;
      float2 v[4];
      unpack_pairs(u[i], v);
      top[i] = block_max_fp4<MX>(v);
      m = max(m, __float_as_uint(top[i]));
    }
    const float scale = row_scale_fp4(group_max_u32(grp, m, red) >> 16, &inverse);   // bf16 values: low half 0, or NaN
    if (grp.t == 0) o.q_scale[row] = scale;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (i >= lane.steps) break;
    float2 v[4];
    unpack_pairs(u[i], v);
    if constexpr (MX) top[i] = block_max_fp4<MX>(v);
    store_vec_fp4<MX>(qrow, sfrow, lane, i, v, top[i], inverse);
  }
}

template <int V>
__device__ __forceinline__ void load_row_fp4(uint4 (&v)[V], const __nv_bfloat16* x, int t, int T, int nvec) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = t + T * i;
    v[i] = c < nvec ? ld_stream_v4(x + 8 * c) : make_uint4(0, 0, 0, 0);
  }
}

enum Fp4Source : int { kFp4Plain = 0, kFp4Norm = 1, kFp4NormWeight = 2 };

// rows_per_group rows for each group; a holds x (and, for the norm, its operands).
// Three vectors a thread keep to 64 registers, so that two of the widest CTAs share an SM: with the next row
// and the modulation held in registers the norm had one, and 8192 x 8192 mxfp4 took 96 us (now 74, nvfp4 87).  What is
// left of the norm's distance from HBM (26 us) is that a row is loaded only when the one before is done, and that its
// modulation is read again for every row.
template <bool MX, int V, int SRC>
__global__ void __launch_bounds__(512, V == 3 ? 2 : 1) rows_fp4_kernel(const RmsArgs a, const Fp4Out o, const int T,
                                                       const int64_t rows_per_group) {
  // two of each, used by rows in turn: a warp may write the next row's partials while another still
  // reads this row's, and the next row's barrier lies between this row's reads and the one after's writes
  __shared__ float red_sum[2][16], red_max[2][16];
  const RowGroup grp = row_group(T);
  int turn = 0;
  const int nvec = a.D >> 3;
  const float fD = static_cast<float>(a.D);
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * grp.count + grp.index) * rows_per_group;
  const int64_t end = min(first + rows_per_group, a.S);
  if (first >= end) return;   // a whole group leaves: its barriers are its own
  const Fp4Lane where = fp4_lane<MX>(grp.t, T, nvec, V);
  uint4 v[V];
  [[maybe_unused]] uint4 next[SRC == kFp4Plain ? V : 1];
  load_row_fp4<V>(v, a.x + first * a.ld_x, grp.t, T, nvec);
  for (int64_t row = first; row < end; ++row) {
    if constexpr (SRC == kFp4Plain) {
      if (row + 1 < end) load_row_fp4<V>(next, a.x + (row + 1) * a.ld_x, grp.t, T, nvec);
    } else {
      const int64_t m = a.mod_index ? static_cast<int64_t>(__ldg(a.mod_index + row)) : row / a.rows_per_mod;
      // vectors past the row's end are zeros and leave the sums as they are
      float2 acc = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        acc = sumsq_bf16x2(acc, v[i].x);
        acc = sumsq_bf16x2(acc, v[i].y);
        acc = sumsq_bf16x2(acc, v[i].z);
        acc = sumsq_bf16x2(acc, v[i].w);
      }
      const float ss = block_sum(grp, __fadd_rn(acc.x, acc.y), red_sum[turn] + grp.index * (T >> 5));
      const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, fD), a.eps)));
      const float2 inv2 = make_float2(inv, inv);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c = grp.t + T * i;
        if (c >= nvec) continue;   // stays zero
        uint4 su = ld_v4(a.scale + m * a.ld_mod + 8 * c);
        if (!a.scale_is_multiplier)
          su = make_uint4(one_plus_bf16x2(su.x), one_plus_bf16x2(su.y), one_plus_bf16x2(su.z), one_plus_bf16x2(su.w));
        const uint4 bu = ld_v4(a.shift + m * a.ld_mod + 8 * c);
        uint4 wu = make_uint4(0, 0, 0, 0);
        if constexpr (SRC == kFp4NormWeight) wu = ld_v4(a.w + 8 * c);
        const uint32_t xw[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        const uint32_t sw[4] = {su.x, su.y, su.z, su.w};
        const uint32_t bw[4] = {bu.x, bu.y, bu.z, bu.w};
        const uint32_t ww[4] = {wu.x, wu.y, wu.z, wu.w};
        uint32_t h[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          float2 t = mul2_rn(bf2_to_f2(xw[p]), inv2);
          if constexpr (SRC == kFp4NormWeight) t = mul2_rn(t, bf2_to_f2(ww[p]));
          h[p] = f2_to_bf2(add_f32_bf16x2(mul2_rn(t, bf2_to_f2(sw[p])), bw[p]));
        }
        v[i] = make_uint4(h[0], h[1], h[2], h[3]);
      }
    }
    group_quant_fp4<MX, V>(grp, o, row, v, where, red_max[turn] + grp.index * (T >> 5));
    turn ^= 1;
    if constexpr (SRC == kFp4Plain) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = next[i];
    } else {
      if (row + 1 < end) load_row_fp4<V>(v, a.x + (row + 1) * a.ld_x, grp.t, T, nvec);
    }
  }
}

// ---------------------------------------------------------------- register-resident warp rows
// The norm of many rows of 256 NV elements: one row per warp on the warp ring of rows.cuh (lane l holds
// vectors 32 k + l), so that the per-row work (sums, reciprocal square root, scale) is shared by NV
// vectors a lane instead of three, and no warp waits for another; the modulation of the CTA's middle row
// and the norm weight are cached in shared memory (fill_mod_cache).  The sum of squares is the same
// canonical tree.  Bound by instruction issue and latency (70 % of issue slots): 16 warps (128 registers) take 53 us at
// 32768 x 3072 mxfp4 and 55 us nvfp4, 20 warps 55 and 63, 24 (which spill) 64 and 72, with one slot each
// (it refills as soon as the row is in registers).

// bf16(h) of one vector, and max |h| (float32, NaN above all) folded into amax.
template <bool HAS_W>
__device__ __forceinline__ uint4 rms_h_fp4(const uint4& xu, float2 inv2, const uint4& wu, const float2 (&s)[4],
                                           const uint4& bu, float& amax) {
  const uint32_t xw[4] = {xu.x, xu.y, xu.z, xu.w};
  const uint32_t ww[4] = {wu.x, wu.y, wu.z, wu.w};
  const uint32_t bw[4] = {bu.x, bu.y, bu.z, bu.w};
  uint32_t hw[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    float2 t = mul2_rn(bf2_to_f2(xw[p]), inv2);
    if constexpr (HAS_W) t = mul2_rn(t, bf2_to_f2(ww[p]));
    const float2 h = add_f32_bf16x2(mul2_rn(t, s[p]), bw[p]);
    amax = max3_abs_nan(amax, h.x, h.y);
    hw[p] = f2_to_bf2(h);
  }
  return make_uint4(hw[0], hw[1], hw[2], hw[3]);
}

// The same with the modulation read from global memory, out of line: a row whose modulation row is not the
// CTA's cached one.
template <bool HAS_W>
__device__ __noinline__ uint4 rms_h_fp4_global(const __nv_bfloat16* srow, const __nv_bfloat16* brow, int multiplier, int c,
                                               uint4 xu, float inv, uint4 wu, float* amax) {
  uint4 su = ld_v4(srow + 8 * c);
  if (!multiplier)
    su = make_uint4(one_plus_bf16x2(su.x), one_plus_bf16x2(su.y), one_plus_bf16x2(su.z), one_plus_bf16x2(su.w));
  float2 s[4];
  unpack_pairs(su, s);
  float m = *amax;
  const uint4 hu = rms_h_fp4<HAS_W>(xu, make_float2(inv, inv), wu, s, ld_v4(brow + 8 * c), m);
  *amax = m;
  return hu;
}

constexpr int kFp4NormWarps = 16;

template <bool MX, int NV, bool HAS_W>
__global__ void __launch_bounds__(32 * kFp4NormWarps, 1)
    rms_mod_fp4_reg_kernel(const RmsArgs a, const WarpRingGeom g, const Fp4Out o) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const int lane = threadIdx.x & 31;
  float4* cache = mod_cache_of<NV>(smem, g);
  const int64_t cm = fill_mod_cache<NV, HAS_W>(a, g, cache);
  __syncthreads();
  constexpr uint32_t kAll = (1u << NV) - 1u;   // every vector of the row exists
  Fp4Lane where = fp4_lane<MX>(lane, 32, 32 * NV, 0);
  where.codes = kAll;
  where.scales = (lane & (MX ? 3 : 1)) == 0 ? kAll : 0u;
  int64_t cur_m = -1, seg_end = -1;
  auto src = [&](int64_t r) -> const void* { return a.x + r * a.ld_x; };
  warp_row_loop_reg(
      smem, g, a.S, src, [&](const uint8_t* slot, int64_t) { return load_row_regs<NV>(slot, lane); },
      [&](int64_t row, RowRegs<NV>& r) {
        const int64_t m = mod_row_of(a, row, cur_m, seg_end);
        const float inv = row_inv_reg<NV>(r, a.eps);
        float amax = 0.f;
        if (m == cm) {
          const float2 inv2 = make_float2(inv, inv);
#pragma unroll
          for (int k = 0; k < NV; ++k) {
            const int c = 32 * k + lane;
            float2 s[4];
            uint4 bu, wu = make_uint4(0, 0, 0, 0);
            mod_of<NV>(a, cache, true, m, c, s, bu);
            if constexpr (HAS_W) wu = weight_of<NV>(cache, c);
            r.v[k] = rms_h_fp4<HAS_W>(r.v[k], inv2, wu, s, bu, amax);
          }
        } else {
#pragma unroll
          for (int k = 0; k < NV; ++k) {
            const int c = 32 * k + lane;
            uint4 wu = make_uint4(0, 0, 0, 0);
            if constexpr (HAS_W) wu = weight_of<NV>(cache, c);
            r.v[k] = rms_h_fp4_global<HAS_W>(a.scale + m * a.ld_mod, a.shift + m * a.ld_mod, a.scale_is_multiplier, c,
                                             r.v[k], inv, wu, &amax);
          }
        }
        float inverse = 0.f;
        if constexpr (!MX) {
          // max |bf16(h)| = bf16(max |h|): rounding is monotone and symmetric (a NaN stays one)
          const float top = __uint_as_float(warp_max_u32(__float_as_uint(amax)));
          const float scale = row_scale_fp4(__bfloat16_as_ushort(__float2bfloat16_rn(top)), &inverse);
          if (lane == 0) o.q_scale[row] = scale;
        }
        uint8_t* qrow = o.q + row * o.ld_q;
        uint8_t* sfrow = o.sf + scale_row(row, o.words);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          float2 v[4];
          unpack_pairs(r.v[k], v);
          store_vec_fp4<MX>(qrow, sfrow, where, k, v, block_max_fp4<MX>(v), inverse);
        }
      });
}

// ---------------------------------------------------------------- SwiGLU
// act = bf16((gate * sigmoid(gate)) * up) as swiglu_kernel computes it, on its ring (the sigmoid table
// is worth loading only once per CTA), quantised from registers.
template <bool MX, int V>
__global__ void __launch_bounds__(1024) swiglu_fp4_kernel(const SwigluArgs a, const RingGeom g, const Fp4Out o,
                                                          const int T) {
  extern __shared__ __align__(1024) uint8_t smem[];
  load_sigmoid_table(reinterpret_cast<uint32_t*>(smem), threadIdx.x, blockDim.x);
  const uint32_t sig = smem_u32(smem);
  __syncthreads();
  const RowGroup grp = row_group(T);
  uint8_t* ring = smem + kSigmoidBytes + static_cast<size_t>(grp.index) * ring_bytes(g);
  const int nvec = a.F >> 3;
  const Fp4Lane where = fp4_lane<MX>(grp.t, T, nvec, V);
  auto src = [&](int64_t r, int part) -> const void* { return (part ? a.up : a.gate) + r * a.ld_in; };
  row_loop(ring, g, grp, a.M, src, [&](int64_t row, uint8_t* slot, const RingState& rs) {
    const uint8_t* up = slot + g.part_bytes;
    float unused = 0.f;
    uint4 v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = grp.t + T * i;
      v[i] = c < nvec ? swiglu8(slot, up, c, sig, unused, false) : make_uint4(0, 0, 0, 0);
    }
    group_quant_fp4<MX, V>(grp, o, row, v, where, rs.red_max);
  });
}

// ---------------------------------------------------------------- inverse
// out[m, k] = cast((code * block scale) * row scale), one vector of eight values per thread.
// OUT: 0 bf16, 1 fp16, 2 fp32.
// Eight codes -> their e2m1 values.
__device__ __forceinline__ void decode_e2m1x8(uint32_t codes, float2 (&v)[4]) {
  uint32_t h[4];
  asm("{ .reg .b8 a, b, c, d;\n"
      "  mov.b32 {a, b, c, d}, %4;\n"
      "  cvt.rn.f16x2.e2m1x2 %0, a;\n"
      "  cvt.rn.f16x2.e2m1x2 %1, b;\n"
      "  cvt.rn.f16x2.e2m1x2 %2, c;\n"
      "  cvt.rn.f16x2.e2m1x2 %3, d; }"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
#pragma unroll
  for (int p = 0; p < 4; ++p) v[p] = __half22float2(*reinterpret_cast<const __half2*>(&h[p]));
}

struct DequantFp4Args {
  const uint8_t* q;
  int64_t ld_q;
  const uint8_t* sf;
  const float* q_scale;   // or null (1)
  void* out;
  int64_t ld_out;
  int64_t S;
  int D;
  int words;
};

// Thread = one vector of eight columns in the four rows r, r + 32, r + 64, r + 96 of a scale tile, whose scale
// words are 16 consecutive bytes; the grid's y strides over such groups of rows.
template <bool MX, int OUT>
__global__ void __launch_bounds__(256) dequant_rows_fp4_kernel(const DequantFp4Args a) {
  const int nvec = a.D >> 3;
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= nvec) return;
  const int block = MX ? c >> 2 : c >> 1;
  const int64_t groups = (a.S + 127) / 128 * 32;
  constexpr int kRows = 4;
  for (int64_t grp = blockIdx.y; grp < groups; grp += gridDim.y) {
    const int64_t row0 = (grp >> 5) * 128 + (grp & 31);
    if (row0 >= a.S) continue;
    uint32_t codes[kRows], byte[kRows];
    float rs[kRows];
    const uint4 words = __ldg(reinterpret_cast<const uint4*>(a.sf + scale_row(row0, a.words) + 512 * static_cast<int64_t>(block >> 2)));
    const uint32_t w4[kRows] = {words.x, words.y, words.z, words.w};
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int64_t row = min(row0 + 32 * r, a.S - 1);
      codes[r] = __ldg(reinterpret_cast<const uint32_t*>(a.q + row * a.ld_q + 4 * static_cast<int64_t>(c)));
      byte[r] = (w4[r] >> (8 * (block & 3))) & 0xFFu;
      rs[r] = a.q_scale ? __ldg(a.q_scale + row) : 1.f;
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int64_t row = row0 + 32 * r;
      if (row >= a.S) break;
      const float sb = MX ? __uint_as_float(byte[r] == 255u ? 0x7FC00000u : byte[r] == 0u ? 0x00400000u : byte[r] << 23)
                          : e4m3_to_f32(byte[r]);
      float2 v[4];
      decode_e2m1x8(codes[r], v);
#pragma unroll
      for (int p = 0; p < 4; ++p) v[p] = mul2_rn(mul2_rn(v[p], make_float2(sb, sb)), make_float2(rs[r], rs[r]));
      const int64_t at = row * a.ld_out + 8 * static_cast<int64_t>(c);
      if constexpr (OUT == 2) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(a.out) + at);
        p[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        p[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
      } else {
        uint32_t w[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          if constexpr (OUT == 0) {
            w[p] = f2_to_bf2(v[p]);
          } else {
            const __half2 h = __floats2half2_rn(v[p].x, v[p].y);
            w[p] = *reinterpret_cast<const uint32_t*>(&h);
          }
        }
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}

}  // namespace rows
}  // namespace t8g
