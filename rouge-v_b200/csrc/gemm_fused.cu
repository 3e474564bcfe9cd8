// GEMMs with bias, activation and residual in the epilogue: the kernels of
// gemm_impl.cuh instantiated with EP, for the int8, e4m3 and f16 / bf16
// kinds.
//
// The epilogue warps hold 32 f32 sums of one row per lane, so bias and
// activation cost registers only, and overlap the next tile's MMAs
// (double-buffered accumulator). The residual is read once, by the lanes
// that round and store the same elements. Measured: int8 16 x 8192 x 8192 with
// bias and residual 20.1 us (3376 GB/s); int8 4096^3 with the same 60.8 (2262
// TOP/s; 60.4 without epilogue); bf16 1000 x 14336 x 4096 with gelu, f32 out, 107
// (1095 TFLOP/s; without gelu 99.7: the last tiles' epilogue is not under any
// MMA); e4m3 8192^3 with silu and residual 425 to 430 (2555 and more).
#include "gemm_impl.cuh"

namespace rb200 {
namespace {

// The fused epilogue's fields (checked by check_epilogue).
void set_epilogue(GemmArgs &g, const RougeB200Epilogue &ep) {
  g.ep_bias = ep.bias;
  g.ep_res = ep.residual;
  g.ep_ldr = ep.ldr;
  g.ep_rtype = ep.residual_type;
  g.ep_act = ep.act;
  g.ep_bias16 = (reinterpret_cast<uintptr_t>(ep.bias) & 15u) == 0;
  const int es = ep.residual_type == ROUGE_B200_T_F32 ? 4 : 2;
  g.ep_res16 = (reinterpret_cast<uintptr_t>(ep.residual) & 15u) == 0 && (ep.ldr * es) % 16 == 0;
}

int check_epilogue(const RougeB200Epilogue *ep, int N, int out_type) {
  if (!ep || out_type == ROUGE_B200_OUT_I32) return ROUGE_B200_EINVAL;
  if (ep->act < ROUGE_B200_ACT_NONE || ep->act > ROUGE_B200_ACT_SILU) return ROUGE_B200_EINVAL;
  if (reinterpret_cast<uintptr_t>(ep->bias) & 3u) return ROUGE_B200_EINVAL;
  if (ep->residual) {
    const int t = ep->residual_type;
    if (t != ROUGE_B200_T_F32 && t != ROUGE_B200_T_F16 && t != ROUGE_B200_T_BF16)
      return ROUGE_B200_EINVAL;
    if (ep->ldr < N ||
        (reinterpret_cast<uintptr_t>(ep->residual) & (t == ROUGE_B200_T_F32 ? 3u : 1u)))
      return ROUGE_B200_EINVAL;
  }
  return ROUGE_B200_OK;
}

}  // namespace
}  // namespace rb200

using namespace rb200;

extern "C" {

int rouge_b200_gemm_i8_fused(int M, int N, int K, const int8_t *A, const int8_t *B, int b_layout,
                             const float *scales_a, int a_rows, const float *scales_b, int b_cols,
                             const RougeB200Epilogue *ep, void *C, int ldc, int out_type,
                             void *stream) {
  int s = check_common(M, N, K, A, B, C, ldc, b_layout, out_type, 1);
  if (s == ROUGE_B200_OK) s = check_epilogue(ep, N, out_type);
  if (s == ROUGE_B200_OK && (!scales_a || !scales_b)) s = ROUGE_B200_EINVAL;
  if (s != ROUGE_B200_OK) return set_status(s);
  s = device_ready();
  if (s != ROUGE_B200_OK) return s;
  GemmArgs g{};
  g.M = M; g.N = N; g.K = K;
  g.C = C; g.ldc = ldc;
  g.scales_a = scales_a; g.scales_b = scales_b; g.a_rows = a_rows; g.b_cols = b_cols;
  g.use_tma_store = vec_ok(C, ldc, out_type);
  g.vec16 = (reinterpret_cast<uintptr_t>(scales_b) & 15u) == 0;
  g.err = device_error_word();
  set_epilogue(g, *ep);
  return launch_kind<MmaKind::I8, true>(A, K, B, b_layout == ROUGE_B200_B_KN ? N : K, b_layout, g,
                                        out_type, as_stream(stream));
}

int rouge_b200_gemm_e4m3_fused(int M, int N, int K, const uint8_t *A, const uint8_t *B,
                               int b_layout, const float *scale_a, const float *scale_b,
                               const RougeB200Epilogue *ep, void *C, int ldc, int out_type,
                               void *stream) {
  int s = check_common(M, N, K, A, B, C, ldc, b_layout, out_type, 1);
  if (s == ROUGE_B200_OK) s = check_epilogue(ep, N, out_type);
  if (s == ROUGE_B200_OK && (!scale_a) != (!scale_b)) s = ROUGE_B200_EINVAL;
  if (s != ROUGE_B200_OK) return set_status(s);
  s = device_ready();
  if (s != ROUGE_B200_OK) return s;
  GemmArgs g{};
  g.M = M; g.N = N; g.K = K;
  g.C = C; g.ldc = ldc;
  g.scale_a = scale_a; g.scale_b = scale_b;
  g.use_tma_store = vec_ok(C, ldc, out_type);
  g.err = device_error_word();
  set_epilogue(g, *ep);
  return launch_kind<MmaKind::F8F6F4, true>(A, K, B, b_layout == ROUGE_B200_B_KN ? N : K, b_layout,
                                            g, out_type, as_stream(stream));
}

int rouge_b200_gemm_f16_fused(int M, int N, int K, const uint16_t *A, const uint16_t *B,
                              int b_layout, int is_bf16, const RougeB200Epilogue *ep, void *C,
                              int ldc, int out_type, void *stream) {
  int s = check_common(M, N, K, A, B, C, ldc, b_layout, out_type, 2);
  if (s == ROUGE_B200_OK) s = check_epilogue(ep, N, out_type);
  if (s != ROUGE_B200_OK) return set_status(s);
  s = device_ready();
  if (s != ROUGE_B200_OK) return s;
  GemmArgs g{};
  g.M = M; g.N = N; g.K = K;
  g.C = C; g.ldc = ldc;
  g.bf16 = is_bf16 ? 1 : 0;
  g.use_tma_store = vec_ok(C, ldc, out_type);
  g.err = device_error_word();
  set_epilogue(g, *ep);
  return launch_kind<MmaKind::F16, true>(A, K, B, b_layout == ROUGE_B200_B_KN ? N : K, b_layout, g,
                                         out_type, as_stream(stream));
}

}  // extern "C"
