// Plain GEMMs on sm_100a tensor cores and the implicit-GEMM convolution:
// launchers and C entries over the kernels of gemm_impl.cuh.
#include "gemm_impl.cuh"

namespace rb200 {

std::atomic<unsigned long long *> g_clock_stamps{nullptr};
std::atomic<int> g_clock_ctas{0};
std::atomic<int> g_clock_dev{-1};
std::atomic<int> g_tile_mode{ROUGE_B200_TILES_AUTO};

namespace {

template <MmaKind KIND, int BN, bool PAIR, int OUT>
int launch_conv_bn(const CUtensorMap &ta, const void *Wt, GemmArgs g, cudaStream_t st) {
  using C = Cfg<KIND, BN, false>;
  auto make_b = [&](int box_rows, CUtensorMap *tb) {
    return make_tmap_2d(tb, Wt,
                        C::ESIZE == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                      : CU_TENSOR_MAP_DATA_TYPE_UINT16,
                        g.K, g.N, static_cast<uint64_t>(g.K) * C::ESIZE, C::BK, box_rows);
  };
  return launch_tiles<KIND, BN, false, OUT, true, PAIR>(ta, make_b, g, st);
}

}  // namespace

// Implicit-GEMM convolution, NHWC in, f32 NHWC out (+ bias): f16/bf16
// inputs (kind::f16, 64 channels per k-block) or f32 inputs read as tf32
// (kind::tf32, 32 channels per k-block).
// GEMM view: M = N*OH*OW output pixels, N = Cout, K = KH*KW*Cin in
// (kr, kc, c) order, so the weights [Cout][KH][KW][Cin] are the K-major B
// operand as stored. The A tile of k-block (tap, c0) is one im2col TMA load:
// 128 consecutive output pixels (crossing rows and images) x BK channels of
// filter tap (kr, kc), zeros in the padding. Y has row pitch ldy >= Cout
// and element type out_type: f32, or 16-bit (kind::f16 only) holding bf16
// or, with f16out, IEEE half. blas != 0: Y = alpha * acc + beta * Y (no
// bias), the old Y read only when beta != 0.
template <MmaKind KIND>
int launch_conv(int N, int H, int W, int Cin, int Cout, int KH, int KW, int stride, int pad,
                const void *X, const void *Wt, const float *bias, void *Y, long long ldy,
                int is_bf16, int out_type, int f16out, int blas, float alpha, float beta,
                cudaStream_t st) {
  using C0 = Cfg<KIND, 128, false>;
  const int OH = (H + 2 * pad - KH) / stride + 1, OW = (W + 2 * pad - KW) / stride + 1;
  GemmArgs g{};
  g.M = N * OH * OW;
  g.N = Cout;
  g.K = KH * KW * Cin;
  g.C = Y;
  g.ldc = ldy;
  g.bf16 = is_bf16 ? 1 : 0;
  g.bias = bias;
  g.vec16 = (reinterpret_cast<uintptr_t>(bias) & 15u) == 0;
  g.use_tma_store = vec_ok(Y, ldy, out_type);
  g.f16out = f16out;
  g.blas = blas;
  g.alpha = alpha;
  g.beta = beta;
  g.err = device_error_word();
  g.conv_cblocks = Cin / C0::BK;
  g.conv_kw = KW;
  g.conv_oh = OH;
  g.conv_ow = OW;
  g.conv_stride = stride;
  g.conv_pad = pad;
  g.conv_cin = Cin;
  CUtensorMap ta;
  int s = make_tmap_im2col_nhwc(&ta, X,
                                C0::ESIZE == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                               : CU_TENSOR_MAP_DATA_TYPE_UINT16,
                                C0::ESIZE, N, H, W, Cin, -pad, -pad, pad - (KW - 1), pad - (KH - 1),
                                C0::BK, kBM, stride, stride);
  if (s != ROUGE_B200_OK) return s;
  const int sms = current_sm_count();
  const long long tiles256 = static_cast<long long>((g.M + kBM - 1) / kBM) * ((Cout + 255) / 256);
  const bool pair = g_tile_mode.load() == ROUGE_B200_TILES_AUTO
                        ? (Cout > 128 && tiles256 >= sms)
                        : g_tile_mode.load() == ROUGE_B200_TILES_PAIR;
  const int bn = (pair || (Cout > 128 && tiles256 >= sms)) ? 256 : 128;
  const int bm = pair ? 2 * kBM : kBM;
  g.num_m = (g.M + bm - 1) / bm;
  g.num_n = (Cout + bn - 1) / bn;
  g.num_k = KH * KW * g.conv_cblocks;
  g.num_tiles = g.num_m * g.num_n;
  if constexpr (KIND == MmaKind::F16) {
    if (out_type == ROUGE_B200_OUT_BF16) {
      if (pair) return launch_conv_bn<KIND, 256, true, ROUGE_B200_OUT_BF16>(ta, Wt, g, st);
      return bn == 256 ? launch_conv_bn<KIND, 256, false, ROUGE_B200_OUT_BF16>(ta, Wt, g, st)
                       : launch_conv_bn<KIND, 128, false, ROUGE_B200_OUT_BF16>(ta, Wt, g, st);
    }
  }
  if (out_type != ROUGE_B200_OUT_F32) return set_status(ROUGE_B200_EUNSUPPORTED);
  if (pair) return launch_conv_bn<KIND, 256, true, ROUGE_B200_OUT_F32>(ta, Wt, g, st);
  return bn == 256 ? launch_conv_bn<KIND, 256, false, ROUGE_B200_OUT_F32>(ta, Wt, g, st)
                   : launch_conv_bn<KIND, 128, false, ROUGE_B200_OUT_F32>(ta, Wt, g, st);
}

int launch_conv_f16(int N, int H, int W, int Cin, int Cout, int KH, int KW, int stride, int pad,
                    const uint16_t *X, const uint16_t *Wt, const float *bias, float *Y,
                    int is_bf16, cudaStream_t st) {
  return launch_conv<MmaKind::F16>(N, H, W, Cin, Cout, KH, KW, stride, pad, X, Wt, bias, Y, Cout,
                                   is_bf16, ROUGE_B200_OUT_F32, 0, 0, 1.0f, 0.0f, st);
}

// f32 NHWC convolution with tf32 operands (Cin a multiple of 32, inputs of
// at least 128 KB, 16-byte aligned X and Wt).
int launch_conv_tf32(int N, int H, int W, int Cin, int Cout, int KH, int KW, int stride, int pad,
                     const float *X, const float *Wt, const float *bias, float *Y, long long ldy,
                     cudaStream_t st) {
  return launch_conv<MmaKind::TF32>(N, H, W, Cin, Cout, KH, KW, stride, pad, X, Wt, bias, Y, ldy,
                                    0, ROUGE_B200_OUT_F32, 0, 0, 1.0f, 0.0f, st);
}

// The cuDNN-forward form: Y (row pitch ldy, element type y_type: T_F32,
// T_F16 or T_BF16) = alpha * conv(X, Wt) + beta * Y. ab_type T_F16 / T_BF16
// (kind::f16, Cin % 64 == 0) or T_F32 (kind::tf32, Cin % 32 == 0; the
// caller splits operands for f32 accuracy). Checked by the caller.
int launch_conv_blas(int ab_type, int N, int H, int W, int Cin, int Cout, int KH, int KW,
                     int stride, int pad, const void *X, const void *Wt, float alpha, float beta,
                     void *Y, long long ldy, int y_type, cudaStream_t st) {
  const int out = y_type == ROUGE_B200_T_F32 ? ROUGE_B200_OUT_F32 : ROUGE_B200_OUT_BF16;
  const int f16out = y_type == ROUGE_B200_T_F16 ? 1 : 0;
  if (ab_type == ROUGE_B200_T_F32)
    return launch_conv<MmaKind::TF32>(N, H, W, Cin, Cout, KH, KW, stride, pad, X, Wt, nullptr, Y,
                                      ldy, 0, out, f16out, 1, alpha, beta, st);
  return launch_conv<MmaKind::F16>(N, H, W, Cin, Cout, KH, KW, stride, pad, X, Wt, nullptr, Y, ldy,
                                   ab_type == ROUGE_B200_T_BF16 ? 1 : 0, out, f16out, 1, alpha, beta,
                                   st);
}

int launch_gemm_i8(int M, int N, int K, const int8_t *A, long long lda, const int8_t *B,
                   long long ldb, int b_layout, const float *sa, int a_rows, const float *sb,
                   int b_cols, void *Cp, long long ldc, int out_type, cudaStream_t st) {
  GemmArgs g{};
  g.M = M; g.N = N; g.K = K;
  g.C = Cp; g.ldc = ldc;
  g.scales_a = sa; g.scales_b = sb; g.a_rows = a_rows; g.b_cols = b_cols;
  g.use_tma_store = vec_ok(Cp, ldc, out_type);
  g.vec16 = (reinterpret_cast<uintptr_t>(sb) & 15u) == 0;
  g.err = device_error_word();
  return launch_kind<MmaKind::I8>(A, lda, B, ldb, b_layout, g, out_type, st);
}

int launch_quant_i8_rows(const float *x, int rows, int cols, float *scales, int8_t *out,
                         cudaStream_t st);

// The W8A8 linear step: per-row quantization of X (codes Aq, scales sa)
// and C = dequant(Aq . Wq^T). One launch of the CTA-pair int8 kernel with
// the quantizer fused (see GemmArgs::fq_x) when K <= 4096 (a row fits a
// 16 KB slot) and the problem takes CTA-pair tiles; otherwise the row
// quantizer, then the GEMM.
int launch_w8a8_linear(int M, int N, int K, const float *X, const int8_t *Wq, const float *sw,
                       int8_t *Aq, float *sa, void *Cp, long long ldc, int out_type, unsigned *ws,
                       cudaStream_t st) {
  const bool fuse = K <= 4096 && (reinterpret_cast<uintptr_t>(X) & 15u) == 0 && use_pair_tiles(M, N);
  if (!fuse) {
    int s = launch_quant_i8_rows(X, M, K, sa, Aq, st);
    if (s != ROUGE_B200_OK) return s;
    return launch_gemm_i8(M, N, K, Aq, K, Wq, K, ROUGE_B200_B_NK, sa, 1, sw, 1, Cp, ldc, out_type,
                          st);
  }
  GemmArgs g{};
  g.M = M; g.N = N; g.K = K;
  g.C = Cp; g.ldc = ldc;
  g.scales_a = sa; g.scales_b = sw; g.a_rows = 1; g.b_cols = 1;
  g.use_tma_store = vec_ok(Cp, ldc, out_type);
  g.vec16 = (reinterpret_cast<uintptr_t>(sw) & 15u) == 0;
  g.err = device_error_word();
  g.fq_x = X;
  g.fq_codes = Aq;
  g.fq_scales = sa;
  g.fq_cnt = ws;
  g.n_fast = 1;
  g.num_m = (M + 2 * kBM - 1) / (2 * kBM);
  g.num_n = (N + 255) / 256;
  g.num_k = (K + kBKBytes - 1) / kBKBytes;
  g.num_tiles = g.num_m * g.num_n;
  CUtensorMap ta;
  int s = make_tmap_2d(&ta, Aq, CU_TENSOR_MAP_DATA_TYPE_UINT8, K, M, static_cast<uint64_t>(K),
                       kBKBytes, kBM);
  if (s != ROUGE_B200_OK) return s;
  auto make_b = [&](int box_rows, CUtensorMap *tb) {
    return make_tmap_2d(tb, Wq, CU_TENSOR_MAP_DATA_TYPE_UINT8, K, N, static_cast<uint64_t>(K),
                        kBKBytes, box_rows);
  };
  switch (out_type) {
    case ROUGE_B200_OUT_F32:
      return launch_tiles<MmaKind::I8, 256, false, ROUGE_B200_OUT_F32, false, true, true>(ta, make_b, g, st);
    case ROUGE_B200_OUT_BF16:
      return launch_tiles<MmaKind::I8, 256, false, ROUGE_B200_OUT_BF16, false, true, true>(ta, make_b, g, st);
    default:
      return launch_tiles<MmaKind::I8, 256, false, ROUGE_B200_OUT_I32, false, true, true>(ta, make_b, g, st);
  }
}

// As launch_gemm_i8, with the device word that receives a timeout status
// supplied by the caller.
int launch_gemm_i8_with_err(int M, int N, int K, const int8_t *A, long long lda, const int8_t *B,
                            long long ldb, int b_layout, const float *sa, int a_rows,
                            const float *sb, int b_cols, void *Cp, long long ldc, int out_type,
                            int *err, cudaStream_t st) {
  GemmArgs g{};
  g.M = M; g.N = N; g.K = K;
  g.C = Cp; g.ldc = ldc;
  g.scales_a = sa; g.scales_b = sb; g.a_rows = a_rows; g.b_cols = b_cols;
  g.use_tma_store = vec_ok(Cp, ldc, out_type);
  g.vec16 = (reinterpret_cast<uintptr_t>(sb) & 15u) == 0;
  g.err = err;
  return launch_kind<MmaKind::I8>(A, lda, B, ldb, b_layout, g, out_type, st);
}

// The int8 GEMM with its output broadcast to every rank's C (see
// GemmArgs::bcast): the sharded W8A8 GEMM's all-gather fused into the
// epilogue.
int launch_gemm_i8_bcast(int M, int N, int K, const int8_t *A, long long lda, const int8_t *B,
                         long long ldb, int b_layout, const float *sa, int a_rows,
                         const float *sb, int b_cols, void *mc, void *const *peers, int npeers,
                         long long ldc, int col_off, int out_type, cudaStream_t st) {
  GemmArgs g{};
  g.M = M; g.N = N; g.K = K;
  g.scales_a = sa; g.scales_b = sb; g.a_rows = a_rows; g.b_cols = b_cols;
  g.use_tma_store = 0;
  g.vec16 = (reinterpret_cast<uintptr_t>(sb) & 15u) == 0;
  g.err = device_error_word();
  g.bcast = mc;
  g.npeers = mc ? 0 : npeers;
  for (int r = 0; r < g.npeers; ++r) g.peers[r] = peers[r];
  g.col_off = col_off;
  g.bld = ldc;
  return launch_kind<MmaKind::I8>(A, lda, B, ldb, b_layout, g, out_type, st);
}

int launch_gemm_e4m3(int M, int N, int K, const uint8_t *A, long long lda, const uint8_t *B,
                     long long ldb, int b_layout, const float *scale_a, const float *scale_b,
                     void *Cp, long long ldc, int out_type, cudaStream_t st) {
  GemmArgs g{};
  g.M = M; g.N = N; g.K = K;
  g.C = Cp; g.ldc = ldc;
  g.scale_a = scale_a; g.scale_b = scale_b;
  g.use_tma_store = vec_ok(Cp, ldc, out_type);
  g.err = device_error_word();
  return launch_kind<MmaKind::F8F6F4>(A, lda, B, ldb, b_layout, g, out_type, st);
}

int launch_gemm_f16(int M, int N, int K, const uint16_t *A, long long lda, const uint16_t *B,
                    long long ldb, int b_layout, int is_bf16, void *Cp, long long ldc,
                    int out_type, cudaStream_t st) {
  GemmArgs g{};
  g.M = M; g.N = N; g.K = K;
  g.C = Cp; g.ldc = ldc;
  g.bf16 = is_bf16 ? 1 : 0;
  g.use_tma_store = vec_ok(Cp, ldc, out_type);
  g.err = device_error_word();
  return launch_kind<MmaKind::F16>(A, lda, B, ldb, b_layout, g, out_type, st);
}

// BLAS-form GEMM on the f16 / bf16 / tf32 / e4m3 kinds:
// C[M][N] (f32, row pitch ldc) = alpha * A[M][K] . B^T + beta * C, A K-major
// (row pitch lda), B per b_layout (tf32 needs ROUGE_B200_B_NK).
// kind: 0 e4m3, 1 f16, 2 bf16, 3 tf32. tile_hint (kTileHint*) fixes the
// tile shape of this call; kTileHintAuto keeps the process-wide choice.
int launch_gemm_blas_tiles(int kind, int M, int N, int K, const void *A, long long lda,
                           const void *B, long long ldb, int b_layout, float alpha, float beta,
                           float *Cp, long long ldc, int tile_hint, cudaStream_t st) {
  if (tile_hint < kTileHintAuto || tile_hint > kTileHintPair) return set_status(ROUGE_B200_EINVAL);
  GemmArgs g{};
  g.tile_hint = tile_hint;
  g.M = M; g.N = N; g.K = K;
  g.C = Cp; g.ldc = ldc;
  g.blas = 1;
  g.alpha = alpha;
  g.beta = beta;
  g.bf16 = kind == 2 ? 1 : 0;
  g.use_tma_store = vec_ok(Cp, ldc, ROUGE_B200_OUT_F32);
  g.err = device_error_word();
  switch (kind) {
    case 0:
      return launch_kind<MmaKind::F8F6F4>(A, lda, B, ldb, b_layout, g, ROUGE_B200_OUT_F32, st);
    case 1:
    case 2:
      return launch_kind<MmaKind::F16>(A, lda, B, ldb, b_layout, g, ROUGE_B200_OUT_F32, st);
    case 3:
      if (b_layout != ROUGE_B200_B_NK) return set_status(ROUGE_B200_EUNSUPPORTED);
      return launch_kind<MmaKind::TF32>(A, lda, B, ldb, b_layout, g, ROUGE_B200_OUT_F32, st);
    default:
      return set_status(ROUGE_B200_EINVAL);
  }
}

int launch_gemm_blas(int kind, int M, int N, int K, const void *A, long long lda, const void *B,
                     long long ldb, int b_layout, float alpha, float beta, float *Cp,
                     long long ldc, cudaStream_t st) {
  return launch_gemm_blas_tiles(kind, M, N, K, A, lda, B, ldb, b_layout, alpha, beta, Cp, ldc,
                                kTileHintAuto, st);
}

// launch_gemm_blas over `batch` items stacked by rows (K-major B only):
// item i computes C[i*M + m][n] = alpha * sum_k A[i*M + m][k] B[i*N + n][k]
// (+ beta * C). M must be a multiple of 256 when batch > 1.
int launch_gemm_blas_batched(int kind, int M, int N, int K, const void *A, long long lda,
                             const void *B, long long ldb, float alpha, float beta, float *Cp,
                             long long ldc, int batch, cudaStream_t st) {
  if (batch <= 1)
    return launch_gemm_blas(kind, M, N, K, A, lda, B, ldb, ROUGE_B200_B_NK, alpha, beta, Cp, ldc,
                            st);
  if (M % 256 != 0 || kind != 3) return set_status(ROUGE_B200_EUNSUPPORTED);
  GemmArgs g{};
  g.M = M * batch; g.N = N; g.K = K;
  g.item_m = M;
  g.C = Cp; g.ldc = ldc;
  g.blas = 1;
  g.alpha = alpha;
  g.beta = beta;
  g.use_tma_store = vec_ok(Cp, ldc, ROUGE_B200_OUT_F32);
  g.err = device_error_word();
  return launch_kind<MmaKind::TF32>(A, lda, B, ldb, ROUGE_B200_B_NK, g, ROUGE_B200_OUT_F32, st);
}

// Block-scaled (MXFP8) GEMM on CTA pairs with 256 x 256 tiles:
// C[M][N] = sum_k (a[m][k] * 2^(sfa - 127)) (b[n][k] * 2^(sfb - 127)),
// f32 accumulation; A [M][K], B [N][K] e4m3 / e5m2 codes (row pitches lda,
// ldb bytes), scales in the tcgen05 atom layout (rouge_b200_mx_scale_atoms).
int launch_gemm_mx(int M, int N, int K, const uint8_t *A, long long lda, int fmt_a,
                   const uint8_t *sfa, const uint8_t *B, long long ldb, int fmt_b,
                   const uint8_t *sfb, void *Cp, long long ldc, int out_type, cudaStream_t st) {
  GemmArgs g{};
  g.M = M; g.N = N; g.K = K;
  g.C = Cp; g.ldc = ldc;
  g.scales_a = reinterpret_cast<const float *>(sfa);
  g.scales_b = reinterpret_cast<const float *>(sfb);
  g.mx_fmt_a = fmt_a;
  g.mx_fmt_b = fmt_b;
  g.sf_kblocks = (K + 127) / 128;
  g.use_tma_store = vec_ok(Cp, ldc, out_type);
  g.err = device_error_word();
  g.num_m = (M + 2 * kBM - 1) / (2 * kBM);
  g.num_n = (N + 255) / 256;
  g.num_k = (K + 127) / 128;
  g.num_tiles = g.num_m * g.num_n;
  if (out_type == ROUGE_B200_OUT_BF16)
    return launch_gemm_impl<MmaKind::MXF8, 256, false, ROUGE_B200_OUT_BF16, true>(A, lda, B, ldb, g,
                                                                                  st);
  return launch_gemm_impl<MmaKind::MXF8, 256, false, ROUGE_B200_OUT_F32, true>(A, lda, B, ldb, g,
                                                                               st);
}

// Block-scaled NVFP4 GEMM on CTA pairs, 256 x 256 tiles:
// C[M][N] = gs_a gs_b sum_k (a[m][k] * sa) (b[n][k] * sb), a / b packed
// e2m1 (two per byte, the lower-index element in the low nibble; row
// pitches K / 2 bytes), UE4M3 block scales per 16 K in the tcgen05 atom
// layout (rouge_b200_nvfp4_scale_atoms), gs_a / gs_b device floats or null.
template <MmaKind KIND>
int launch_gemm_fp4(int M, int N, int K, const uint8_t *A, const uint8_t *sfa, const float *gs_a,
                    const uint8_t *B, const uint8_t *sfb, const float *gs_b, void *Cp,
                    long long ldc, int out_type, cudaStream_t st) {
  GemmArgs g{};
  g.M = M; g.N = N; g.K = K;
  g.C = Cp; g.ldc = ldc;
  g.scales_a = reinterpret_cast<const float *>(sfa);
  g.scales_b = reinterpret_cast<const float *>(sfb);
  g.scale_a = gs_a && gs_b ? gs_a : nullptr;
  g.scale_b = gs_a && gs_b ? gs_b : nullptr;
  g.mx_fmt_a = 1;  // E2M1 of kind::mxf4nvf4 / kind::mxf4
  g.mx_fmt_b = 1;
  g.sf_kblocks = (K + 255) / 256;
  g.use_tma_store = vec_ok(Cp, ldc, out_type);
  g.err = device_error_word();
  g.num_m = (M + 2 * kBM - 1) / (2 * kBM);
  g.num_n = (N + 255) / 256;
  g.num_k = (K + 255) / 256;
  g.num_tiles = g.num_m * g.num_n;
  const uint64_t kbytes = static_cast<uint64_t>(K) / 2;
  CUtensorMap ta;
  int s = make_tmap_2d(&ta, A, CU_TENSOR_MAP_DATA_TYPE_UINT8, kbytes, M, kbytes, kBKBytes, kBM);
  if (s != ROUGE_B200_OK) return s;
  auto make_b = [&](int box_rows, CUtensorMap *tb) {
    return make_tmap_2d(tb, B, CU_TENSOR_MAP_DATA_TYPE_UINT8, kbytes, N, kbytes, kBKBytes, box_rows);
  };
  if (out_type == ROUGE_B200_OUT_BF16)
    return launch_tiles<KIND, 256, false, ROUGE_B200_OUT_BF16, false, true>(ta, make_b, g, st);
  return launch_tiles<KIND, 256, false, ROUGE_B200_OUT_F32, false, true>(ta, make_b, g, st);
}

}  // namespace rb200

using namespace rb200;

extern "C" {

int rouge_b200_gemm_nvfp4(int M, int N, int K, const uint8_t *A, const uint8_t *sfa,
                          const float *gs_a, const uint8_t *B, const uint8_t *sfb,
                          const float *gs_b, void *C, int ldc, int out_type, void *stream) {
  if (M <= 0 || N <= 0 || K <= 0 || !A || !B || !sfa || !sfb || !C || ldc < N ||
      (out_type != ROUGE_B200_OUT_F32 && out_type != ROUGE_B200_OUT_BF16))
    return set_status(ROUGE_B200_EINVAL);
  if (K % 32 || (reinterpret_cast<uintptr_t>(A) & 15u) || (reinterpret_cast<uintptr_t>(B) & 15u) ||
      (reinterpret_cast<uintptr_t>(sfa) & 15u) || (reinterpret_cast<uintptr_t>(sfb) & 15u))
    return set_status(ROUGE_B200_EUNSUPPORTED);
  const int s = device_ready();
  if (s != ROUGE_B200_OK) return s;
  return launch_gemm_fp4<MmaKind::NVF4>(M, N, K, A, sfa, gs_a, B, sfb, gs_b, C, ldc, out_type,
                                       as_stream(stream));
}

int rouge_b200_gemm_mxfp4(int M, int N, int K, const uint8_t *A, const uint8_t *sfa,
                          const uint8_t *B, const uint8_t *sfb, void *C, int ldc, int out_type,
                          void *stream) {
  if (M <= 0 || N <= 0 || K <= 0 || !A || !B || !sfa || !sfb || !C || ldc < N ||
      (out_type != ROUGE_B200_OUT_F32 && out_type != ROUGE_B200_OUT_BF16))
    return set_status(ROUGE_B200_EINVAL);
  if (K % 32 || (reinterpret_cast<uintptr_t>(A) & 15u) || (reinterpret_cast<uintptr_t>(B) & 15u) ||
      (reinterpret_cast<uintptr_t>(sfa) & 15u) || (reinterpret_cast<uintptr_t>(sfb) & 15u))
    return set_status(ROUGE_B200_EUNSUPPORTED);
  const int s = device_ready();
  if (s != ROUGE_B200_OK) return s;
  return launch_gemm_fp4<MmaKind::MXF4>(M, N, K, A, sfa, nullptr, B, sfb, nullptr, C, ldc, out_type,
                                        as_stream(stream));
}

int rouge_b200_gemm_mx(int M, int N, int K, const uint8_t *A, int fmt_a, const uint8_t *sfa,
                       const uint8_t *B, int fmt_b, const uint8_t *sfb, void *C, int ldc,
                       int out_type, void *stream) {
  if (M <= 0 || N <= 0 || K <= 0 || !A || !B || !sfa || !sfb || !C || ldc < N)
    return set_status(ROUGE_B200_EINVAL);
  if ((fmt_a != 0 && fmt_a != 1) || (fmt_b != 0 && fmt_b != 1) ||
      (out_type != ROUGE_B200_OUT_F32 && out_type != ROUGE_B200_OUT_BF16))
    return set_status(ROUGE_B200_EINVAL);
  if (K % 32 || (reinterpret_cast<uintptr_t>(A) & 15u) || (reinterpret_cast<uintptr_t>(B) & 15u) ||
      (reinterpret_cast<uintptr_t>(sfa) & 15u) || (reinterpret_cast<uintptr_t>(sfb) & 15u))
    return set_status(ROUGE_B200_EUNSUPPORTED);
  const int s = device_ready();
  if (s != ROUGE_B200_OK) return s;
  return launch_gemm_mx(M, N, K, A, K, fmt_a, sfa, B, K, fmt_b, sfb, C, ldc, out_type,
                        as_stream(stream));
}

int rouge_b200_set_clock_probe(unsigned long long *stamps, int ctas) {
  if (ctas < 0) return set_status(ROUGE_B200_EINVAL);
  if (!stamps || ctas == 0) {
    g_clock_stamps.store(nullptr);
    return ROUGE_B200_OK;
  }
  g_clock_dev.store(current_device());
  g_clock_ctas.store(ctas);
  g_clock_stamps.store(stamps);
  return ROUGE_B200_OK;
}

int rouge_b200_set_tile_mode(int mode) {
  if (mode != ROUGE_B200_TILES_AUTO && mode != ROUGE_B200_TILES_SINGLE &&
      mode != ROUGE_B200_TILES_PAIR)
    return set_status(ROUGE_B200_EINVAL);
  return g_tile_mode.exchange(mode);
}

int rouge_b200_gemm_i8(int M, int N, int K, const int8_t *A, const int8_t *B, int b_layout,
                       const float *scales_a, int a_rows, const float *scales_b, int b_cols,
                       void *C, int ldc, int out_type, void *stream) {
  int s = check_common(M, N, K, A, B, C, ldc, b_layout, out_type, 1);
  if (s != ROUGE_B200_OK) return set_status(s);
  if (out_type != ROUGE_B200_OUT_I32 && (!scales_a || !scales_b)) return set_status(ROUGE_B200_EINVAL);
  s = device_ready();
  if (s != ROUGE_B200_OK) return s;
  const long long ldb = b_layout == ROUGE_B200_B_KN ? N : K;
  return launch_gemm_i8(M, N, K, A, K, B, ldb, b_layout, scales_a, a_rows, scales_b, b_cols, C,
                        ldc, out_type, as_stream(stream));
}

size_t rouge_b200_w8a8_workspace_bytes(int M) {
  return M > 0 ? (static_cast<size_t>(M + 127) / 128 + 2) * sizeof(unsigned) : 0;
}

int rouge_b200_w8a8_linear(int M, int N, int K, const float *X, const int8_t *Wq, const float *sw,
                           int8_t *Aq, float *sa, void *C, int ldc, int out_type, void *workspace,
                           void *stream) {
  if (!X || !sw || !sa || !workspace) return set_status(ROUGE_B200_EINVAL);
  int s = check_common(M, N, K, Aq, Wq, C, ldc, ROUGE_B200_B_NK, out_type, 1);
  if (s != ROUGE_B200_OK) return set_status(s);
  if ((K & 3) || (reinterpret_cast<uintptr_t>(X) & 15u) || (reinterpret_cast<uintptr_t>(workspace) & 3u))
    return set_status(ROUGE_B200_EUNSUPPORTED);
  s = device_ready();
  if (s != ROUGE_B200_OK) return s;
  return launch_w8a8_linear(M, N, K, X, Wq, sw, Aq, sa, C, ldc, out_type,
                            static_cast<unsigned *>(workspace), as_stream(stream));
}

int rouge_b200_gemm_i8_bcast(int M, int N, int K, const int8_t *A, const int8_t *B, int b_layout,
                             const float *scales_a, int a_rows, const float *scales_b, int b_cols,
                             void *C_mc, void *const *C_peers, int npeers, long long ldc,
                             int col_off, int out_type, void *stream) {
  if (M <= 0 || N <= 0 || K <= 0 || !A || !B || col_off < 0 || ldc < static_cast<long long>(col_off) + N)
    return set_status(ROUGE_B200_EINVAL);
  if (b_layout != ROUGE_B200_B_KN && b_layout != ROUGE_B200_B_NK) return set_status(ROUGE_B200_EINVAL);
  if (out_type != ROUGE_B200_OUT_F32 && out_type != ROUGE_B200_OUT_BF16 &&
      out_type != ROUGE_B200_OUT_I32)
    return set_status(ROUGE_B200_EINVAL);
  if (out_type != ROUGE_B200_OUT_I32 && (!scales_a || !scales_b)) return set_status(ROUGE_B200_EINVAL);
  if (!C_mc && (!C_peers || npeers < 1 || npeers > 8)) return set_status(ROUGE_B200_EINVAL);
  const long long esz = out_type == ROUGE_B200_OUT_BF16 ? 2 : 4;
  // 16-byte vectors: row pitch, column offset and width in whole vectors.
  if ((ldc * esz) % 16 || (col_off * esz) % 16 || N % 8 || K % 16 ||
      (b_layout == ROUGE_B200_B_KN && N % 16) ||
      (reinterpret_cast<uintptr_t>(A) & 15u) || (reinterpret_cast<uintptr_t>(B) & 15u) ||
      (reinterpret_cast<uintptr_t>(C_mc) & 15u))
    return set_status(ROUGE_B200_EUNSUPPORTED);
  if (!C_mc)
    for (int r = 0; r < npeers; ++r)
      if (!C_peers[r] || (reinterpret_cast<uintptr_t>(C_peers[r]) & 15u))
        return set_status(ROUGE_B200_EINVAL);
  int s = device_ready();
  if (s != ROUGE_B200_OK) return s;
  const long long ldb = b_layout == ROUGE_B200_B_KN ? N : K;
  return launch_gemm_i8_bcast(M, N, K, A, K, B, ldb, b_layout, scales_a, a_rows, scales_b, b_cols,
                              C_mc, C_peers, npeers, ldc, col_off, out_type, as_stream(stream));
}

int rouge_b200_gemm_e4m3(int M, int N, int K, const uint8_t *A, const uint8_t *B, int b_layout,
                         const float *scale_a, const float *scale_b, void *C, int ldc,
                         int out_type, void *stream) {
  int s = check_common(M, N, K, A, B, C, ldc, b_layout, out_type, 1);
  if (s != ROUGE_B200_OK) return set_status(s);
  if (out_type == ROUGE_B200_OUT_I32 || (!scale_a) != (!scale_b)) return set_status(ROUGE_B200_EINVAL);
  s = device_ready();
  if (s != ROUGE_B200_OK) return s;
  const long long ldb = b_layout == ROUGE_B200_B_KN ? N : K;
  return launch_gemm_e4m3(M, N, K, A, K, B, ldb, b_layout, scale_a, scale_b, C, ldc, out_type,
                          as_stream(stream));
}

int rouge_b200_conv2d_nhwc_f16(int N, int H, int W, int Cin, int Cout, int KH, int KW, int stride,
                               int pad, const uint16_t *X, const uint16_t *Wt, const float *bias,
                               float *Y, int is_bf16, void *stream) {
  if (!X || !Wt || !Y || N <= 0 || H <= 0 || W <= 0 || Cin <= 0 || Cout <= 0 || KH <= 0 ||
      KW <= 0 || stride <= 0 || pad < 0)
    return set_status(ROUGE_B200_EINVAL);
  const long long OH = (static_cast<long long>(H) + 2 * pad - KH) / stride + 1;
  const long long OW = (static_cast<long long>(W) + 2 * pad - KW) / stride + 1;
  if (OH <= 0 || OW <= 0) return set_status(ROUGE_B200_EINVAL);  // conv.cpp:249
  // im2col TMA limits: 64-channel boxes, corners in [-128, 127], filter
  // offsets below 256, traversal stride up to 8; inputs of at least 128 KB.
  const long long xbytes = static_cast<long long>(N) * H * W * Cin * 2;
  if (Cin % 64 || Cout % 4 || pad > 128 || pad - (KW - 1) < -128 || pad - (KH - 1) < -128 ||
      KH > 256 || KW > 256 || stride > 8 || xbytes < 131072 ||
      static_cast<long long>(N) * OH * OW > 0x7fffffffLL ||
      (reinterpret_cast<uintptr_t>(X) & 15u) || (reinterpret_cast<uintptr_t>(Wt) & 15u))
    return set_status(ROUGE_B200_EUNSUPPORTED);
  int s = device_ready();
  if (s != ROUGE_B200_OK) return s;
  return launch_conv_f16(N, H, W, Cin, Cout, KH, KW, stride, pad, X, Wt, bias, Y, is_bf16,
                         as_stream(stream));
}

int rouge_b200_gemm_f16(int M, int N, int K, const uint16_t *A, const uint16_t *B, int b_layout,
                        int is_bf16, void *C, int ldc, int out_type, void *stream) {
  int s = check_common(M, N, K, A, B, C, ldc, b_layout, out_type, 2);
  if (s != ROUGE_B200_OK) return set_status(s);
  if (out_type == ROUGE_B200_OUT_I32) return set_status(ROUGE_B200_EINVAL);
  s = device_ready();
  if (s != ROUGE_B200_OK) return s;
  const long long ldb = b_layout == ROUGE_B200_B_KN ? N : K;
  return launch_gemm_f16(M, N, K, A, K, B, ldb, b_layout, is_bf16, C, ldc, out_type,
                         as_stream(stream));
}

}  // extern "C"
