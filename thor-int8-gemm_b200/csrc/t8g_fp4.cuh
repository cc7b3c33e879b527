// C ABI of the microscaled 4-bit entry points (host side; part of t8g.cu's translation unit).
#pragma once

namespace {

bool fp4_kind(int kind) { return kind == T8G_QUANT_MXFP4 || kind == T8G_QUANT_NVFP4; }

// 4-block scale words of a row of `K` elements.
int64_t fp4_words(int64_t K, int kind) { return kind == T8G_QUANT_MXFP4 ? (K + 127) / 128 : (K + 63) / 64; }

int check_fp4_rows(const char* what, int64_t S, int64_t D, int kind, int64_t dmax) {
  g_last_error[0] = '\0';
  if (S < 0 || D < 0) return fail(T8G_ERR_INVALID_ARGUMENT, "%s: negative size", what);
  if (!fp4_kind(kind)) return fail(T8G_ERR_INVALID_ARGUMENT, "%s: quant_kind %d is not a 4-bit format", what, kind);
  if (D % 8) return fail(T8G_ERR_INVALID_ARGUMENT, "%s: row length %lld is not a multiple of 8", what, (long long)D);
  if (D > dmax) return fail(T8G_ERR_UNSUPPORTED, "%s: row length %lld exceeds %lld", what, (long long)D, (long long)dmax);
  if (S >= (int64_t(1) << 40)) return fail(T8G_ERR_UNSUPPORTED, "%s: too many rows", what);
  return T8G_OK;
}

// The operand of a 4-bit matrix [rows, K]: q (row pitch in bytes), scale tiles, row scale.
int check_fp4_operand(const char* what, const void* q, int64_t ld_q, const void* sf, const float* scale, int64_t K,
                      int kind, bool need_scale) {
  if (!q || !sf) return fail(T8G_ERR_INVALID_ARGUMENT, "%s: codes or block scales are null", what);
  if (!aligned(q, 16) || !aligned(sf, 16))
    return fail(T8G_ERR_INVALID_ARGUMENT, "%s: codes and block scales must be 16-byte aligned", what);
  if (ld_q < K / 2 || ld_q % 16)
    return fail(T8G_ERR_INVALID_ARGUMENT, "%s: row stride %lld must hold %lld bytes and be a multiple of 16", what,
                (long long)ld_q, (long long)(K / 2));
  if (need_scale && kind == T8G_QUANT_NVFP4 && !scale) return fail(T8G_ERR_INVALID_ARGUMENT, "%s: q_scale is null", what);
  if (!aligned(scale, 4)) return fail(T8G_ERR_INVALID_ARGUMENT, "%s: row scales must be 4-byte aligned", what);
  return T8G_OK;
}

t8g::rows::Fp4Out fp4_out(void* q, int64_t ld_q, void* sf, float* q_scale, int64_t S, int64_t D, int kind) {
  t8g::rows::Fp4Out o;
  o.q = static_cast<uint8_t*>(q);
  o.ld_q = ld_q;
  o.sf = static_cast<uint8_t*>(sf);
  o.q_scale = q_scale;
  o.S = S;
  o.words = static_cast<int>(fp4_words(D, kind));
  return o;
}

// Rows without elements: no codes and no block scales, but nvfp4's row scales, which are those of rows of zeros.
int empty_rows_fp4(const char* what, float* q_scale, int64_t S, int kind, void* stream) {
  if (kind != T8G_QUANT_NVFP4 || !q_scale) return T8G_OK;
  if (!aligned(q_scale, 4)) return fail(T8G_ERR_INVALID_ARGUMENT, "%s: row scales must be 4-byte aligned", what);
  int dev;
  DeviceInfo info;
  const int rc = current_device(&dev, &info);
  if (rc) return rc;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>((S + 255) / 256, 8 * info.sms));
  t8g::rows::zero_row_scales_fp4_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(q_scale, S);
  return launch_checked(what);
}

// Vectors per thread of a direct row kernel: the canonical shape's, rounded up to a compiled one.
#define T8G_DISPATCH_FP4_V(v, ...)                     \
  if ((v) <= 3) {                                      \
    constexpr int V = 3;                               \
    __VA_ARGS__;                                       \
  } else if ((v) <= 6) {                               \
    constexpr int V = 6;                               \
    __VA_ARGS__;                                       \
  } else {                                             \
    constexpr int V = 12;                              \
    __VA_ARGS__;                                       \
  }

// Rows from which the register-resident warp kernels run (rows of 256 NV elements).
constexpr int64_t kFp4RegRows = 2048;

// Launch a direct row kernel: T threads a row, as many rows a CTA as make 256 threads, and no more CTAs
// than the device holds at a time (each group then takes several consecutive rows).
template <bool MX, int V, int SRC>
int launch_rows_fp4(const t8g::rows::RmsArgs& a, const t8g::rows::Fp4Out& o, int T, int dev, int sms, cudaStream_t st,
                    const char* what) {
  auto kern = t8g::rows::rows_fp4_kernel<MX, V, SRC>;
  const int groups = T <= 128 ? 256 / T : 1;
  const int threads = groups * T;
  // resident CTAs per SM, looked up once per device and block size (a multiple of 32)
  static std::atomic<int> occ_of[kMaxDevices][17] = {};
  std::atomic<int>& known = occ_of[dev][threads / 32];
  int occ = known.load(std::memory_order_relaxed);
  if (occ == 0) {
    T8G_CHECK_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kern, threads, 0), "occupancy query");
    occ = occ < 1 ? 1 : occ;
    known.store(occ, std::memory_order_relaxed);
  }
  const int64_t held = static_cast<int64_t>(occ) * sms * groups;   // rows in work at a time
  const int64_t per_group = (a.S + held - 1) / held;
  const int64_t grid = (a.S + per_group * groups - 1) / (per_group * groups);
  kern<<<static_cast<unsigned>(grid), threads, 0, st>>>(a, o, T, per_group);
  T8G_CHECK_CUDA(cudaGetLastError(), what);
  return T8G_OK;
}

template <int SRC>
int dispatch_rows_fp4(const t8g::rows::RmsArgs& a, const t8g::rows::Fp4Out& o, int quant_kind, int dev, int sms,
                      cudaStream_t st, const char* what) {
  using namespace t8g::rows;
  const bool mx = quant_kind == T8G_QUANT_MXFP4;
  if constexpr (SRC != kFp4Plain) {
    const int nv = reg_nv(a.D);
    if (nv && a.S >= kFp4RegRows) {
      constexpr bool W = SRC == kFp4NormWeight;
      WarpLaunch l;
      l.max_warps = kFp4NormWarps;
      l.stages = 1;
      l.contiguous = true;
      l.tail_bytes = static_cast<size_t>((W ? 8 : 6) * a.D);   // fp32 multiplier + bf16 shift (+ bf16 weight)
      l.smem_budget = kRowSmemLimit;
      const uint32_t row_bytes = static_cast<uint32_t>(2 * a.D);
      int rc = T8G_OK;
      if (mx) {
        T8G_DISPATCH_NV(nv, rc = launch_warp_rows(rms_mod_fp4_reg_kernel<true, NV, W>, a, row_bytes, a.S, dev, sms, st, l, what, o));
      } else {
        T8G_DISPATCH_NV(nv, rc = launch_warp_rows(rms_mod_fp4_reg_kernel<false, NV, W>, a, row_bytes, a.S, dev, sms, st, l, what, o));
      }
      return rc;
    }
  }
  const int T = row_shape(a.D).T;
  const int v = (a.D / 8 + T - 1) / T;
  if (mx) {
    T8G_DISPATCH_FP4_V(v, return (launch_rows_fp4<true, V, SRC>(a, o, T, dev, sms, st, what)))
  } else {
    T8G_DISPATCH_FP4_V(v, return (launch_rows_fp4<false, V, SRC>(a, o, T, dev, sms, st, what)))
  }
}

// ----------------------------------------------------------------- GEMM
struct Fp4Gemm {
  const void *x, *x_sf, *w, *w_sf;
  int64_t ld_x, ld_w, M, N, K;
  int kind;
};

template <bool MX, int OUT, int TBN>
int launch_gemm_fp4_small(const Fp4Gemm& p, const t8g::gemm4::Args& args, int split, int dev, cudaStream_t st) {
  using namespace t8g::gemm4;
  using C = SmallCfg<MX, TBN>;
  static std::atomic<bool> attr_done[kMaxDevices] = {};
  auto kern = gemm_fp4_kernel<MX, OUT, TBN>;
  int rc = ensure_smem_attr(kern, dev, kSmallSmem, attr_done);
  if (rc) return rc;
  const int64_t words = fp4_words(p.K, p.kind);
  const uint32_t sf_box = C::kSfBytes / 8;   // a stage's scale tiles of a row group, as 8-byte elements
  const uint32_t arows = static_cast<uint32_t>(std::min<int64_t>((p.M + 7) / 8 * 8, BM));
  CUtensorMap ta, tb, tsa, tsb;
  if ((rc = encode_2d(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.x, p.K / 2, p.M, p.ld_x, BK, arows, CU_TENSOR_MAP_SWIZZLE_128B)))
    return rc;
  if ((rc = encode_2d(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.w, p.K / 2, p.N, p.ld_w, BK, TBN, CU_TENSOR_MAP_SWIZZLE_128B)))
    return rc;
  if ((rc = encode_2d(&tsa, CU_TENSOR_MAP_DATA_TYPE_INT64, p.x_sf, words * 64, (p.M + 127) / 128, words * 512, sf_box, 1,
                      CU_TENSOR_MAP_SWIZZLE_NONE)))
    return rc;
  if ((rc = encode_2d(&tsb, CU_TENSOR_MAP_DATA_TYPE_INT64, p.w_sf, words * 64, (p.N + 127) / 128, words * 512, sf_box, 1,
                      CU_TENSOR_MAP_SWIZZLE_NONE)))
    return rc;
  const int64_t tiles = ((p.M + BM - 1) / BM) * ((p.N + TBN - 1) / TBN);
  if (tiles * split >= (int64_t(1) << 31)) return fail(T8G_ERR_UNSUPPORTED, "gemm_fp4: too many tiles");
  // as many stages as fit, at least two (the MMA reads 16 KB from the start of any A slot: the B ring
  // behind the A ring holds that much)
  const int stages = static_cast<int>(std::min<uint32_t>((kSmallSmem - 1024) / C::stage_bytes(arows), kSmallMaxStages));
  static_assert(2 * C::stage_bytes(BM) + 1024 <= kSmallSmem && 2 * C::kBBytes >= 128 * BK, "two stages fit");
  static_assert(C::partial_bytes(BM) + 1024 <= kSmallSmem, "a partial tile fits");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * split), 1, 1);
  cfg.blockDim = dim3(NUM_THREADS, 1, 1);
  cfg.dynamicSmemBytes = kSmallSmem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = static_cast<unsigned>(split);
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  T8G_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, ta, tb, tsa, tsb, args, split, arows, stages), "gemm_fp4 launch");
  return T8G_OK;
}

template <bool MX, int OUT, bool SCALED>
int launch_gemm_fp4_pair(const Fp4Gemm& p, const t8g::gemm4::Args& args, int dev, int sms, cudaStream_t st) {
  using namespace t8g::gemm4;
  using C = PairCfg<MX, OUT>;
  static std::atomic<bool> attr_done[kMaxDevices] = {};
  auto kern = gemm_fp4_pair_kernel<MX, OUT, SCALED>;
  int rc = ensure_smem_attr(kern, dev, C::kSmemBytes, attr_done);
  if (rc) return rc;
  const int64_t words = fp4_words(p.K, p.kind);
  const uint32_t sf_box = C::kSfaBytes / 8;
  constexpr int esz = OutTraits<OUT>::kBytes;
  CUtensorMap ta, tb, tsa, tsb, to;
  if ((rc = encode_2d(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.x, p.K / 2, p.M, p.ld_x, BK, 128, CU_TENSOR_MAP_SWIZZLE_128B)))
    return rc;
  if ((rc = encode_2d(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.w, p.K / 2, p.N, p.ld_w, BK, 128, CU_TENSOR_MAP_SWIZZLE_128B)))
    return rc;
  if ((rc = encode_2d(&tsa, CU_TENSOR_MAP_DATA_TYPE_INT64, p.x_sf, words * 64, (p.M + 127) / 128, words * 512, sf_box, 1,
                      CU_TENSOR_MAP_SWIZZLE_NONE)))
    return rc;
  if ((rc = encode_2d(&tsb, CU_TENSOR_MAP_DATA_TYPE_INT64, p.w_sf, words * 64, (p.N + 127) / 128, words * 512, sf_box, 2,
                      CU_TENSOR_MAP_SWIZZLE_NONE)))
    return rc;
  const CUtensorMapDataType out_dt = OUT == kOutF32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : OUT == kOutF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                      : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  // 32 rows of 128 bytes: 64 two-byte or 32 four-byte columns, up to N's last whole 16-byte piece
  if ((rc = encode_2d(&to, out_dt, args.out, p.N / (16 / esz) * (16 / esz), p.M, args.ld_out * esz, 128 / esz, 32, CU_TENSOR_MAP_SWIZZLE_128B)))
    return rc;
  const int64_t tiles = ((p.M + 255) / 256) * ((p.N + 255) / 256);
  if (tiles >= (int64_t(1) << 31)) return fail(T8G_ERR_UNSUPPORTED, "gemm_fp4: too many tiles");
  const int64_t pairs = std::min<int64_t>(tiles, sms / 2);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs), 1, 1);
  cfg.blockDim = dim3(kPairThreads, 1, 1);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = st;
  cfg.attrs = nullptr;   // the kernel declares its cluster shape (2, 1, 1)
  cfg.numAttrs = 0;
  T8G_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, ta, tb, tsa, tsb, to, args), "gemm_fp4 pair launch");
  return T8G_OK;
}

// Which kernel, tile width and split (device times of one call, nvfp4, on a B200 with 148 SMs):
//   the pair kernel has a floor of 7 to 10 us and then the full rate; it runs above 64 rows when its
//   256 x 256 tiles occupy more than a quarter of the SMs (128 x 9216 x 3072: 10.2 us, 11.9 with the small
//   kernel), and above 128 rows also when K is too short to be worth splitting (at most 8 stages:
//   256 x 1024 x 1024 7.5 us against 8.3, but 256 x 3072 x 12288 20.5 against 18.3); its stores want a whole
//   16-byte piece of columns;
//   the small kernel takes the tile width and the power-of-two split that bring the CTAs nearest to
//   one an SM (1 x 9216 x 3072: 72 tiles x 2 7.3 us, x 1 8.5, x 4 10.5; 1 x 3072 x 3072: 24 x 4 5.8,
//   x 8 6.6), 128 columns where both widths come equally near (1 x 9216 x 3072: 144 x 1 of 64 columns
//   9.5), 64 above 64 rows, where the partial tiles' sums weigh more (128 x 3072 x 3072: 9.6, 10.0).
struct SmallPlan {
  int64_t ctas;
  int split;
};
SmallPlan small_plan(int64_t M, int64_t N, int tbn, int kstages, int sms) {
  const int64_t tiles = (M + 127) / 128 * ((N + tbn - 1) / tbn);
  int split = 1;
  while (split < 8 && tiles * split * 2 <= sms && split * 2 <= kstages) split *= 2;
  return {std::min<int64_t>(tiles * split, sms), split};
}

template <bool MX, int OUT>
int launch_gemm_fp4(const Fp4Gemm& p, const t8g::gemm4::Args& args, int dev, int sms, cudaStream_t st) {
  const bool many = (p.M + 255) / 256 * ((p.N + 255) / 256) * 8 > sms;
  if (((p.M > 64 && many) || (p.M > 128 && args.kstages <= 8)) && p.N >= 8) {   // a whole 16-byte piece to store
    // mxfp4 without row or weight scales, as the row operators give it, skips the two products by 1 (9472 x
    // 8192 x 512: 36 us, 45 with them; x 1024: 43, 48); the gated epilogue spills in that form and keeps them
    if constexpr (MX && OUT != t8g::gemm4::kOutGated) {
      if (!args.xs && !args.ws) return launch_gemm_fp4_pair<MX, OUT, false>(p, args, dev, sms, st);
    }
    return launch_gemm_fp4_pair<MX, OUT, true>(p, args, dev, sms, st);
  }
  const SmallPlan w = small_plan(p.M, p.N, 128, args.kstages, sms), n = small_plan(p.M, p.N, 64, args.kstages, sms);
  if (n.ctas > w.ctas || (n.ctas == w.ctas && p.M > 64))
    return launch_gemm_fp4_small<MX, OUT, 64>(p, args, n.split, dev, st);
  return launch_gemm_fp4_small<MX, OUT, 128>(p, args, w.split, dev, st);
}

// Argument checks shared by the two products, and the kernel arguments.
int gemm_fp4_args(const Fp4Gemm& p, const float* x_scale, const float* w_scale, int64_t w_scale_numel, const void* bias,
                  int64_t bias_numel, void* out, int esz, int64_t ld_out, t8g::gemm4::Args* a) {
  if (!out) return fail(T8G_ERR_INVALID_ARGUMENT, "out is null");
  int rc = check_fp4_operand("x", p.x, p.ld_x, p.x_sf, x_scale, p.K, p.kind, false);
  if (rc) return rc;
  if ((rc = check_fp4_operand("w", p.w, p.ld_w, p.w_sf, w_scale, p.K, p.kind, false))) return rc;
  if (w_scale && w_scale_numel != 1 && w_scale_numel != p.N)
    return fail(T8G_ERR_INVALID_ARGUMENT, "w_scale numel %lld is neither 1 nor N=%lld", (long long)w_scale_numel, (long long)p.N);
  if (bias_numel != 0 && bias_numel != p.N)
    return fail(T8G_ERR_INVALID_ARGUMENT, "bias numel %lld is neither 0 nor N=%lld", (long long)bias_numel, (long long)p.N);
  if (bias_numel && (!bias || !aligned(bias, esz))) return fail(T8G_ERR_INVALID_ARGUMENT, "bias is null or not aligned");
  if (ld_out < p.N) return fail(T8G_ERR_INVALID_ARGUMENT, "out's row stride is smaller than the row");
  if ((ld_out * esz) % 16 || !aligned(out, 16))
    return fail(T8G_ERR_INVALID_ARGUMENT, "out must be 16-byte aligned, with a row stride that is a multiple of 16 bytes");
  a->xs = x_scale;
  a->ws = w_scale;
  a->ws_stride = w_scale_numel == 1 ? 0 : 1;
  a->bias = bias_numel ? bias : nullptr;
  a->M = static_cast<int>(p.M);
  a->N = static_cast<int>(p.N);
  a->K = static_cast<int>(p.K);
  a->out = out;
  a->ld_out = ld_out;
  a->kstages = static_cast<int>((p.K + t8g::gemm4::kStageK - 1) / t8g::gemm4::kStageK);
  a->last_steps = static_cast<int>((p.K - static_cast<int64_t>(a->kstages - 1) * t8g::gemm4::kStageK + t8g::gemm4::kMmaK - 1) /
                                   t8g::gemm4::kMmaK);
  return T8G_OK;
}

int check_gemm_fp4_sizes(int64_t M, int64_t N, int64_t K, int kind) {
  g_last_error[0] = '\0';
  if (!fp4_kind(kind)) return fail(T8G_ERR_INVALID_ARGUMENT, "quant_kind %d is not a 4-bit format", kind);
  if (M < 0 || N < 0 || K < 8 || K % 8)
    return fail(T8G_ERR_INVALID_ARGUMENT, "bad sizes M=%lld N=%lld K=%lld (K a multiple of 8, at least 8)", (long long)M,
                (long long)N, (long long)K);
  if (M >= (int64_t(1) << 31) - 256 || N >= (int64_t(1) << 31) - 256 || K >= (int64_t(1) << 31))
    return fail(T8G_ERR_UNSUPPORTED, "M, N and K must each be below 2^31 - 256");
  return T8G_OK;
}

}  // namespace

extern "C" {

int64_t t8g_fp4_scale_bytes(int64_t rows, int64_t K, int quant_kind) {
  if (rows < 0 || K < 0 || !fp4_kind(quant_kind)) return -1;
  return (rows + 127) / 128 * fp4_words(K, quant_kind) * 512;
}

int t8g_quant_rows_fp4(const void* x, int64_t ld_x, void* q, int64_t ld_q, void* sf, float* q_scale, int64_t S, int64_t D,
                       int quant_kind, void* stream) {
  using namespace t8g::rows;
  int rc = check_fp4_rows("quant_rows_fp4", S, D, quant_kind, 49152);
  if (rc || S == 0) return rc;
  if (D == 0) return empty_rows_fp4("quant_rows_fp4", q_scale, S, quant_kind, stream);
  if ((rc = check_bf16_matrix("x", x, ld_x, D, true))) return rc;
  if ((rc = check_fp4_operand("q", q, ld_q, sf, q_scale, D, quant_kind, true))) return rc;
  int dev;
  DeviceInfo info;
  if ((rc = current_device(&dev, &info))) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  RmsArgs a = {};
  a.x = static_cast<const __nv_bfloat16*>(x);
  a.ld_x = ld_x;
  a.S = S;
  a.D = static_cast<int>(D);
  return dispatch_rows_fp4<kFp4Plain>(a, fp4_out(q, ld_q, sf, q_scale, S, D, quant_kind), quant_kind, dev, info.sms, st,
                                      "quant_rows_fp4");
}

int t8g_rms_mod_quant_fp4(const void* x, int64_t ld_x, const void* w, const void* shift, const void* scale,
                          int64_t ld_mod, const int32_t* mod_index, int64_t rows_per_mod, int scale_is_multiplier,
                          float eps, void* q, int64_t ld_q, void* sf, float* q_scale, int64_t S, int64_t D,
                          int quant_kind, void* stream) {
  using namespace t8g::rows;
  int rc = check_fp4_rows("rms_mod_quant_fp4", S, D, quant_kind, 49152);
  if (rc || S == 0) return rc;
  if (D == 0) return empty_rows_fp4("rms_mod_quant_fp4", q_scale, S, quant_kind, stream);
  if ((rc = check_bf16_matrix("x", x, ld_x, D, true))) return rc;
  if ((rc = check_bf16_matrix("shift", shift, ld_mod, D, true))) return rc;
  if ((rc = check_bf16_matrix("scale", scale, ld_mod, D, true))) return rc;
  if (w && !aligned(w, 16)) return fail(T8G_ERR_INVALID_ARGUMENT, "w must be 16-byte aligned");
  if (mod_index && !aligned(mod_index, 4)) return fail(T8G_ERR_INVALID_ARGUMENT, "mod_index must be 4-byte aligned");
  if (!mod_index && rows_per_mod < 1) return fail(T8G_ERR_INVALID_ARGUMENT, "rows_per_mod must be >= 1 without mod_index");
  if ((rc = check_fp4_operand("q", q, ld_q, sf, q_scale, D, quant_kind, true))) return rc;
  int dev;
  DeviceInfo info;
  if ((rc = current_device(&dev, &info))) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  RmsArgs a = {};
  a.x = static_cast<const __nv_bfloat16*>(x);
  a.ld_x = ld_x;
  a.w = static_cast<const __nv_bfloat16*>(w);
  a.shift = static_cast<const __nv_bfloat16*>(shift);
  a.scale = static_cast<const __nv_bfloat16*>(scale);
  a.ld_mod = ld_mod;
  a.mod_index = mod_index;
  a.rows_per_mod = rows_per_mod < 1 ? 1 : rows_per_mod;
  a.scale_is_multiplier = scale_is_multiplier;
  a.eps = eps;
  a.S = S;
  a.D = static_cast<int>(D);
  const Fp4Out o = fp4_out(q, ld_q, sf, q_scale, S, D, quant_kind);
  return w ? dispatch_rows_fp4<kFp4NormWeight>(a, o, quant_kind, dev, info.sms, st, "rms_mod_quant_fp4")
           : dispatch_rows_fp4<kFp4Norm>(a, o, quant_kind, dev, info.sms, st, "rms_mod_quant_fp4");
}

int t8g_swiglu_quant_fp4(const void* gate, const void* up, int64_t ld_in, void* q, int64_t ld_q, void* sf, float* q_scale,
                         int64_t M, int64_t F, int quant_kind, void* stream) {
  using namespace t8g::rows;
  int rc = check_fp4_rows("swiglu_quant_fp4", M, F, quant_kind, 24576);
  if (rc || M == 0) return rc;
  if (F == 0) return empty_rows_fp4("swiglu_quant_fp4", q_scale, M, quant_kind, stream);
  if ((rc = check_bf16_matrix("gate", gate, ld_in, F, true))) return rc;
  if ((rc = check_bf16_matrix("up", up, ld_in, F, true))) return rc;
  if ((rc = check_fp4_operand("q", q, ld_q, sf, q_scale, F, quant_kind, true))) return rc;
  int dev;
  DeviceInfo info;
  if ((rc = current_device(&dev, &info))) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  SwigluArgs a = {};
  a.gate = static_cast<const __nv_bfloat16*>(gate);
  a.up = static_cast<const __nv_bfloat16*>(up);
  a.ld_in = ld_in;
  a.M = M;
  a.F = static_cast<int>(F);
  const Fp4Out o = fp4_out(q, ld_q, sf, q_scale, M, F, quant_kind);
  const int T = swiglu_shape(F).T;   // at most three vectors a thread
  const RingGeom g = ring_geom(F, 2);
  return quant_kind == T8G_QUANT_MXFP4
             ? launch_swiglu(swiglu_fp4_kernel<true, kSwigluVecs>, T, a, g, M, dev, info.sms, st, "swiglu_quant_fp4", o)
             : launch_swiglu(swiglu_fp4_kernel<false, kSwigluVecs>, T, a, g, M, dev, info.sms, st, "swiglu_quant_fp4", o);
}

int t8g_dequant_rows_fp4(const void* q, int64_t ld_q, const void* sf, const float* q_scale, void* out, int out_dtype,
                         int64_t ld_out, int64_t S, int64_t D, int quant_kind, void* stream) {
  using namespace t8g::rows;
  int rc = check_fp4_rows("dequant_rows_fp4", S, D, quant_kind, (int64_t(1) << 31) - 8);
  if (rc) return rc;
  if (out_dtype < T8G_OUT_BF16 || out_dtype > T8G_OUT_F32) return fail(T8G_ERR_INVALID_ARGUMENT, "unknown out_dtype %d", out_dtype);
  if (S == 0 || D == 0) return T8G_OK;
  if ((rc = check_fp4_operand("q", q, ld_q, sf, q_scale, D, quant_kind, false))) return rc;
  if (!out || !aligned(out, 16)) return fail(T8G_ERR_INVALID_ARGUMENT, "out must be 16-byte aligned");
  if (ld_out < D || ld_out % 8) return fail(T8G_ERR_INVALID_ARGUMENT, "out row stride must be >= D and a multiple of 8");
  int dev;
  DeviceInfo info;
  if ((rc = current_device(&dev, &info))) return rc;
  DequantFp4Args a;
  a.q = static_cast<const uint8_t*>(q);
  a.ld_q = ld_q;
  a.sf = static_cast<const uint8_t*>(sf);
  a.q_scale = q_scale;
  a.out = out;
  a.ld_out = ld_out;
  a.S = S;
  a.D = static_cast<int>(D);
  a.words = static_cast<int>(fp4_words(D, quant_kind));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // 256 vectors of four rows a CTA and step; groups of rows are strided over when the grid holds fewer
  const unsigned gx = static_cast<unsigned>((D / 8 + 255) / 256);
  const dim3 grid(gx, static_cast<unsigned>(std::min<int64_t>((S + 127) / 128 * std::min<int64_t>(S, 32), 65535)));
#define T8G_DEQUANT(MX)                                                                               \
  switch (out_dtype) {                                                                                \
    case T8G_OUT_BF16: dequant_rows_fp4_kernel<MX, 0><<<grid, 256, 0, st>>>(a); break;                \
    case T8G_OUT_F16: dequant_rows_fp4_kernel<MX, 1><<<grid, 256, 0, st>>>(a); break;                 \
    default: dequant_rows_fp4_kernel<MX, 2><<<grid, 256, 0, st>>>(a); break;                          \
  }
  if (quant_kind == T8G_QUANT_MXFP4) {
    T8G_DEQUANT(true)
  } else {
    T8G_DEQUANT(false)
  }
#undef T8G_DEQUANT
  return launch_checked("dequant_rows_fp4 launch");
}

int t8g_gemm_fp4(const void* x, const void* x_sf, const float* x_scale, const void* w, const void* w_sf,
                 const float* w_scale, int64_t w_scale_numel, const void* bias, int64_t bias_numel, void* out,
                 int out_dtype, int64_t M, int64_t N, int64_t K, int64_t ld_x, int64_t ld_w, int64_t ld_out,
                 int quant_kind, void* stream) {
  using namespace t8g::gemm4;
  int rc = check_gemm_fp4_sizes(M, N, K, quant_kind);
  if (rc) return rc;
  if (out_dtype < T8G_OUT_BF16 || out_dtype > T8G_OUT_F32) return fail(T8G_ERR_INVALID_ARGUMENT, "unknown out_dtype %d", out_dtype);
  if (M == 0 || N == 0) return T8G_OK;
  const Fp4Gemm p = {x, x_sf, w, w_sf, ld_x, ld_w, M, N, K, quant_kind};
  Args a = {};
  if ((rc = gemm_fp4_args(p, x_scale, w_scale, w_scale_numel, bias, bias_numel, out, out_dtype == T8G_OUT_F32 ? 4 : 2, ld_out, &a)))
    return rc;
  int dev;
  DeviceInfo info;
  if ((rc = current_device(&dev, &info))) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (quant_kind == T8G_QUANT_MXFP4) {
    switch (out_dtype) {
      case T8G_OUT_BF16: return launch_gemm_fp4<true, kOutBF16>(p, a, dev, info.sms, st);
      case T8G_OUT_F16: return launch_gemm_fp4<true, kOutF16>(p, a, dev, info.sms, st);
      default: return launch_gemm_fp4<true, kOutF32>(p, a, dev, info.sms, st);
    }
  }
  switch (out_dtype) {
    case T8G_OUT_BF16: return launch_gemm_fp4<false, kOutBF16>(p, a, dev, info.sms, st);
    case T8G_OUT_F16: return launch_gemm_fp4<false, kOutF16>(p, a, dev, info.sms, st);
    default: return launch_gemm_fp4<false, kOutF32>(p, a, dev, info.sms, st);
  }
}

int t8g_gemm_fp4_gated(const void* x, const void* x_sf, const float* x_scale, const void* w, const void* w_sf,
                       const float* w_scale, int64_t w_scale_numel, const void* bias, int64_t bias_numel, const void* res,
                       int64_t ld_res, const void* gate, int64_t ld_gate, const int32_t* gate_index,
                       int64_t rows_per_gate, void* out, int64_t M, int64_t N, int64_t K, int64_t ld_x, int64_t ld_w,
                       int64_t ld_out, int quant_kind, void* stream) {
  using namespace t8g::gemm4;
  int rc = check_gemm_fp4_sizes(M, N, K, quant_kind);
  if (rc) return rc;
  if (N % 8) return fail(T8G_ERR_INVALID_ARGUMENT, "N=%lld must be a multiple of 8", (long long)N);
  if (M == 0 || N == 0) return T8G_OK;
  const Fp4Gemm p = {x, x_sf, w, w_sf, ld_x, ld_w, M, N, K, quant_kind};
  Args a = {};
  if ((rc = gemm_fp4_args(p, x_scale, w_scale, w_scale_numel, bias, bias_numel, out, 2, ld_out, &a))) return rc;
  if (!res || !gate) return fail(T8G_ERR_INVALID_ARGUMENT, "res or gate is null");
  if (!gate_index && rows_per_gate < 1)
    return fail(T8G_ERR_INVALID_ARGUMENT, "rows_per_gate must be positive when gate_index is null");
  if (ld_res < N || ld_gate < N || ld_res % 8 || ld_gate % 8 || !aligned(res, 16) || !aligned(gate, 16) || !aligned(gate_index, 4))
    return fail(T8G_ERR_INVALID_ARGUMENT, "res and gate must be 16-byte aligned, with row strides >= N that are multiples of 8");
  if (out != res) {
    // out and res are either the same matrix or disjoint
    const uintptr_t o0 = reinterpret_cast<uintptr_t>(out), r0 = reinterpret_cast<uintptr_t>(res);
    const uintptr_t o1 = o0 + static_cast<uintptr_t>(((M - 1) * ld_out + N) * 2);
    const uintptr_t r1 = r0 + static_cast<uintptr_t>(((M - 1) * ld_res + N) * 2);
    if (o0 < r1 && r0 < o1) return fail(T8G_ERR_INVALID_ARGUMENT, "out overlaps res without being res");
  } else if (ld_out != ld_res) {
    return fail(T8G_ERR_INVALID_ARGUMENT, "out is res but ld_out != ld_res");
  }
  a.res = res;
  a.gate = gate;
  a.gate_index = gate_index;
  a.ld_res = ld_res;
  a.ld_gate = ld_gate;
  a.rows_per_gate = gate_index ? 1 : rows_per_gate;
  int dev;
  DeviceInfo info;
  if ((rc = current_device(&dev, &info))) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return quant_kind == T8G_QUANT_MXFP4 ? launch_gemm_fp4<true, kOutGated>(p, a, dev, info.sms, st)
                                       : launch_gemm_fp4<false, kOutGated>(p, a, dev, info.sms, st);
}

}  // extern "C"
