// Residual addition, RMS norm and 8-bit output in one kernel:
//   h = round_T(x + r)               written to h_out (the residual stream)
//   y = (float)(h / sqrt(sum h^2 / n + eps)) * w      (transformer.cpp:33-40)
//   codes, scales = per-row int8 (quant_int8.cpp:72-90) or MXFP8 e4m3
//                   blocks of 32 (narrow.cpp:200-265) of y
// with the same arithmetic as those steps apart: sum of squares, inverse
// root and the scaled product in double, so the codes are those of
// rouge_rmsnorm followed by the quantizer.
//
// Memory-bound: a row is read once and stays in registers (16 values per
// thread) over both reductions -- the sum of squares, then the row maximum
// of y -- and the codes. One to 32 warps share a row, so that 512 to 16384
// columns fit; longer rows take the looping kernel, which reads h again.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "i8code.cuh"
#include "narrow.cuh"
#include "runtime.cuh"

namespace rb200 {
namespace {

constexpr int kPerThread = 16;  // row values a thread holds

struct NormArgs {
  const void *x, *r;
  long long ldx, ldr, ldh;
  const float *w;
  float eps;
  int rows, cols;
  void *h;
  void *codes, *scales;
};

template <int T>
struct Elem {
  using type = uint16_t;
};
template <>
struct Elem<ROUGE_B200_T_F32> {
  using type = float;
};

// V consecutive elements (V * sizeof(element) bytes, aligned) as f32.
template <int T, int V>
__device__ __forceinline__ void load_vec(const void *base, long long at, float (&v)[V]) {
  if constexpr (T == ROUGE_B200_T_F32) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      const float4 t = *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + at + 4 * q);
      v[4 * q] = t.x; v[4 * q + 1] = t.y; v[4 * q + 2] = t.z; v[4 * q + 3] = t.w;
    }
  } else {
    uint32_t u[V / 2];
    const uint16_t *p = static_cast<const uint16_t *>(base) + at;
    if constexpr (V == 8) {
      const uint4 t = *reinterpret_cast<const uint4 *>(p);
      u[0] = t.x; u[1] = t.y; u[2] = t.z; u[3] = t.w;
    } else {
      const uint2 t = *reinterpret_cast<const uint2 *>(p);
      u[0] = t.x; u[1] = t.y;
    }
#pragma unroll
    for (int q = 0; q < V / 2; ++q) {
      if constexpr (T == ROUGE_B200_T_F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[q]));
        v[2 * q] = f.x; v[2 * q + 1] = f.y;
      } else {
        v[2 * q] = __uint_as_float(u[q] << 16);
        v[2 * q + 1] = __uint_as_float(u[q] & 0xFFFF0000u);
      }
    }
  }
}

// Rounds v to the element type (v then holds the rounded values) and stores.
template <int T, int V>
__device__ __forceinline__ void round_store(void *base, long long at, float (&v)[V]) {
  if constexpr (T == ROUGE_B200_T_F32) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q)
      *reinterpret_cast<float4 *>(static_cast<float *>(base) + at + 4 * q) =
          make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
  } else {
    uint32_t u[V / 2];
#pragma unroll
    for (int q = 0; q < V / 2; ++q) {
      if constexpr (T == ROUGE_B200_T_F16) {
        u[q] = f16x2_rn(v[2 * q], v[2 * q + 1]);
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[q]));
        v[2 * q] = f.x; v[2 * q + 1] = f.y;
      } else {
        u[q] = bf16x2_rn(v[2 * q], v[2 * q + 1]);
        v[2 * q] = __uint_as_float(u[q] << 16);
        v[2 * q + 1] = __uint_as_float(u[q] & 0xFFFF0000u);
      }
    }
    uint16_t *p = static_cast<uint16_t *>(base) + at;
    if constexpr (V == 8)
      *reinterpret_cast<uint4 *>(p) = make_uint4(u[0], u[1], u[2], u[3]);
    else
      *reinterpret_cast<uint2 *>(p) = make_uint2(u[0], u[1]);
  }
}

__device__ __forceinline__ void group_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(threads) : "memory");
}

// Reductions over the WPR warps of a row group; `slot` holds 2 x WPR values
// of this group, used in turn so that one barrier per reduction is enough
// (a slot is written again only after the other reduction's barrier).
template <int WPR, class V, class Op>
__device__ __forceinline__ V group_reduce(V v, V *slot, int group, int wig, int lane, Op op) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if constexpr (WPR > 1) {
    if (lane == 0) slot[wig] = v;
    group_sync(group, WPR * 32);
    v = slot[0];
#pragma unroll
    for (int i = 1; i < WPR; ++i) v = op(v, slot[i]);
  }
  return v;
}

// y of one value: (float)(h * inv), then * w, both rounded (rouge_rmsnorm).
__device__ __forceinline__ float norm_value(float h, double inv, float w) {
  return __fmul_rn(__double2float_rn(__dmul_rn(static_cast<double>(h), inv)), w);
}

__device__ __forceinline__ double norm_inverse(double ss, int n, float eps) {
  return __ddiv_rn(1.0, __dsqrt_rn(__dadd_rn(__ddiv_rn(ss, static_cast<double>(n)),
                                             static_cast<double>(eps))));
}

// Codes of V consecutive values of one row starting at column c. I8: from
// the row's scale; MX: each block of 32 is V-value lanes next to each other.
template <int FMT, int V>
__device__ __forceinline__ void store_codes(const NormArgs &a, int row, int c, const float (&y)[V],
                                            bool live, double inv, float inv_f, bool exact_row) {
  uint32_t w[V / 4];
  if constexpr (FMT == ROUGE_B200_Q_I8_ROWS) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q)
      w[q] = encode4_i8_x2(make_float4(y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]), inv,
                           inv_f, exact_row);
  } else {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) m = fmaxf(m, fabsf(y[j]));
#pragma unroll
    for (int o = 1; o < 32 / V; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint32_t sc = mx_scale_code(block_pow(m, 448.0f));
    const float si = e8m0_inverse(sc);
#pragma unroll
    for (int q = 0; q < V / 4; ++q)
      w[q] = mx_encode4_f8<kE4M3>(make_float4(y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]), si);
    if (live && c % 32 == 0)
      static_cast<uint8_t *>(a.scales)[static_cast<size_t>(row) * (a.cols / 32) + c / 32] =
          static_cast<uint8_t>(sc);
  }
  if (!live) return;
  uint8_t *out = static_cast<uint8_t *>(a.codes) + static_cast<size_t>(row) * a.cols + c;
  if constexpr (V == 8)
    *reinterpret_cast<uint2 *>(out) = make_uint2(w[0], w[1]);
  else
    *reinterpret_cast<uint32_t *>(out) = w[0];
}

// Scale of an int8 row from the maximum of |y| (quant_int8.cpp:82-84).
__device__ __forceinline__ float row_scale(float amax) {
  const double m = static_cast<double>(amax);
  return m > 0.0 ? __double2float_rn(__ddiv_rn(m, 127.0)) : 1.0f;
}

template <int T, int V, int FMT, int WPR>
__global__ void __launch_bounds__(WPR > 8 ? WPR * 32 : 256)
    norm_quant_kernel(const NormArgs a) {
  constexpr int kWarps = WPR > 8 ? WPR : 8, kGroups = kWarps / WPR, kNv = kPerThread / V;
  __shared__ double sum_slot[kWarps];
  __shared__ float max_slot[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = warp / WPR, wig = warp % WPR;
  const int tig = wig * 32 + lane;  // thread within the row group
  for (int row = blockIdx.x * kGroups + group; row < a.rows; row += gridDim.x * kGroups) {
    float h[kNv][V];
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < kNv; ++i) {
      const int c = (i * WPR * 32 + tig) * V;
      if (c < a.cols) {
        load_vec<T, V>(a.x, row * a.ldx + c, h[i]);
        if (a.r) {
          float t[V];
          load_vec<T, V>(a.r, row * a.ldr + c, t);
#pragma unroll
          for (int j = 0; j < V; ++j) h[i][j] = __fadd_rn(h[i][j], t[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) h[i][j] = 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < kNv; ++i) {
      const int c = (i * WPR * 32 + tig) * V;
      if (a.r && c < a.cols) round_store<T, V>(a.h, row * a.ldh + c, h[i]);
#pragma unroll
      for (int j = 0; j < V; ++j) ss = __fma_rn(static_cast<double>(h[i][j]), h[i][j], ss);
    }
    ss = group_reduce<WPR>(ss, sum_slot + group * WPR, group, wig, lane,
                           [](double p, double q) { return __dadd_rn(p, q); });
    const double inv_rms = norm_inverse(ss, a.cols, a.eps);
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < kNv; ++i) {
      const int c = (i * WPR * 32 + tig) * V;
      float wv[V];
      if (c < a.cols) {
        load_vec<ROUGE_B200_T_F32, V>(a.w, c, wv);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) wv[j] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        h[i][j] = c < a.cols ? norm_value(h[i][j], inv_rms, wv[j]) : 0.0f;
        amax = fmaxf(amax, fabsf(h[i][j]));
      }
    }
    double inv = 0.0;
    float inv_f = 0.0f;
    bool exact_row = false;
    if constexpr (FMT == ROUGE_B200_Q_I8_ROWS) {
      amax = group_reduce<WPR>(amax, max_slot + group * WPR, group, wig, lane,
                               [](float p, float q) { return fmaxf(p, q); });
      const float s = row_scale(amax);
      inv = __ddiv_rn(1.0, static_cast<double>(s));
      inv_f = __double2float_rn(inv);
      exact_row = isinf(inv_f);
      if (tig == 0) static_cast<float *>(a.scales)[row] = s;
    } else if constexpr (WPR > 1) {
      group_sync(group, WPR * 32);  // (the sum's slots are read before the next row writes them)
    }
#pragma unroll
    for (int i = 0; i < kNv; ++i) {
      const int c = (i * WPR * 32 + tig) * V;
      store_codes<FMT, V>(a, row, c, h[i], c < a.cols, inv, inv_f, exact_row);
    }
  }
}

// Rows past 32 warps' registers: 32 warps loop over the row three times,
// reading h again (from h_out, written by the same threads, or x).
template <int T, int V, int FMT>
__global__ void __launch_bounds__(1024) norm_quant_long_kernel(const NormArgs a) {
  __shared__ double sum_slot[32];
  __shared__ float max_slot[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const void *src = a.r ? a.h : a.x;
  const long long lds = a.r ? a.ldh : a.ldx;
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    double ss = 0.0;
    for (int c = threadIdx.x * V; c < a.cols; c += 1024 * V) {
      float h[V];
      load_vec<T, V>(a.x, row * a.ldx + c, h);
      if (a.r) {
        float t[V];
        load_vec<T, V>(a.r, row * a.ldr + c, t);
#pragma unroll
        for (int j = 0; j < V; ++j) h[j] = __fadd_rn(h[j], t[j]);
        round_store<T, V>(a.h, row * a.ldh + c, h);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) ss = __fma_rn(static_cast<double>(h[j]), h[j], ss);
    }
    ss = group_reduce<32>(ss, sum_slot, 0, warp, lane,
                          [](double p, double q) { return __dadd_rn(p, q); });
    const double inv_rms = norm_inverse(ss, a.cols, a.eps);
    auto values = [&](int c, float (&y)[V]) {
      float wv[V];
      load_vec<T, V>(src, row * lds + c, y);
      load_vec<ROUGE_B200_T_F32, V>(a.w, c, wv);
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = norm_value(y[j], inv_rms, wv[j]);
    };
    double inv = 0.0;
    float inv_f = 0.0f;
    bool exact_row = false;
    if constexpr (FMT == ROUGE_B200_Q_I8_ROWS) {
      float amax = 0.0f;
      for (int c = threadIdx.x * V; c < a.cols; c += 1024 * V) {
        float y[V];
        values(c, y);
#pragma unroll
        for (int j = 0; j < V; ++j) amax = fmaxf(amax, fabsf(y[j]));
      }
      amax = group_reduce<32>(amax, max_slot, 0, warp, lane,
                              [](float p, float q) { return fmaxf(p, q); });
      const float s = row_scale(amax);
      inv = __ddiv_rn(1.0, static_cast<double>(s));
      inv_f = __double2float_rn(inv);
      exact_row = isinf(inv_f);
      if (threadIdx.x == 0) static_cast<float *>(a.scales)[row] = s;
    } else {
      __syncthreads();
    }
    // (whole warps: a block's lanes take part in its shuffles)
    for (int c0 = 0; c0 < a.cols; c0 += 1024 * V) {
      const int c = c0 + threadIdx.x * V;
      float y[V];
      if (c < a.cols) {
        values(c, y);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) y[j] = 0.0f;
      }
      store_codes<FMT, V>(a, row, c, y, c < a.cols, inv, inv_f, exact_row);
    }
  }
}

template <int T, int V, int FMT, int WPR>
int launch_wpr(const NormArgs &a, cudaStream_t st) {
  constexpr int kThreads = WPR > 8 ? WPR * 32 : 256, kGroups = kThreads / 32 / WPR;
  const long long want = (static_cast<long long>(a.rows) + kGroups - 1) / kGroups;
  const long long cap = static_cast<long long>(current_sm_count()) * (2048 / kThreads);
  norm_quant_kernel<T, V, FMT, WPR>
      <<<static_cast<unsigned>(want < cap ? want : cap), kThreads, 0, st>>>(a);
  return cuda_status(cudaGetLastError());
}

// Warps per row: the fewest whose registers hold it.
template <int T, int V, int FMT>
int launch_vec(const NormArgs &a, cudaStream_t st) {
  const int per_warp = 32 * kPerThread;
  if (a.cols <= per_warp) return launch_wpr<T, V, FMT, 1>(a, st);
  if (a.cols <= 2 * per_warp) return launch_wpr<T, V, FMT, 2>(a, st);
  if (a.cols <= 4 * per_warp) return launch_wpr<T, V, FMT, 4>(a, st);
  if (a.cols <= 8 * per_warp) return launch_wpr<T, V, FMT, 8>(a, st);
  if (a.cols <= 16 * per_warp) return launch_wpr<T, V, FMT, 16>(a, st);
  if (a.cols <= 32 * per_warp) return launch_wpr<T, V, FMT, 32>(a, st);
  const int cap = current_sm_count() * 2;
  norm_quant_long_kernel<T, V, FMT><<<a.rows < cap ? a.rows : cap, 1024, 0, st>>>(a);
  return cuda_status(cudaGetLastError());
}

template <int T, int V>
int launch_fmt(const NormArgs &a, int fmt, cudaStream_t st) {
  return fmt == ROUGE_B200_Q_I8_ROWS ? launch_vec<T, V, ROUGE_B200_Q_I8_ROWS>(a, st)
                                     : launch_vec<T, V, ROUGE_B200_Q_MX_E4M3>(a, st);
}

}  // namespace
}  // namespace rb200

using namespace rb200;

extern "C" int rouge_b200_add_rmsnorm_quant(const void *x, long long ldx, const void *residual,
                                            long long ldr, const float *w, float eps, int rows,
                                            int cols, int type, void *h_out, long long ldh,
                                            int out_fmt, void *codes, void *scales, void *stream) {
  if (rows < 0 || cols <= 0 || ldx < cols) return set_status(ROUGE_B200_EINVAL);
  if (rows > 0 && (!x || !w || !codes || !scales || (residual == nullptr) != (h_out == nullptr)))
    return set_status(ROUGE_B200_EINVAL);
  if (residual && (ldr < cols || ldh < cols)) return set_status(ROUGE_B200_EINVAL);
  if (type != ROUGE_B200_T_F32 && type != ROUGE_B200_T_F16 && type != ROUGE_B200_T_BF16)
    return set_status(ROUGE_B200_EINVAL);
  if (out_fmt != ROUGE_B200_Q_I8_ROWS && out_fmt != ROUGE_B200_Q_MX_E4M3)
    return set_status(ROUGE_B200_EINVAL);
  // vectors of 16 bytes (8 for 16-bit rows that are only 8-byte aligned)
  const int es = type == ROUGE_B200_T_F32 ? 4 : 2;
  auto aligned = [&](const void *p, long long ld, int bytes) {
    return !p || ((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(ld * es)) &
                  static_cast<uintptr_t>(bytes - 1)) == 0;
  };
  auto all = [&](int bytes) {
    return aligned(x, ldx, bytes) && aligned(residual, ldr, bytes) && aligned(h_out, ldh, bytes);
  };
  const int unit = out_fmt == ROUGE_B200_Q_I8_ROWS ? 4 : 32;
  if (cols % unit || !all(4 * es) || (reinterpret_cast<uintptr_t>(w) & 15u) ||
      (reinterpret_cast<uintptr_t>(codes) & 3u) ||
      (out_fmt == ROUGE_B200_Q_I8_ROWS && (reinterpret_cast<uintptr_t>(scales) & 3u)))
    return set_status(ROUGE_B200_EUNSUPPORTED);
  const int s = device_ready();
  if (s != ROUGE_B200_OK) return s;
  if (rows == 0) return ROUGE_B200_OK;
  NormArgs a{x, residual, ldx, ldr, ldh, w, eps, rows, cols, h_out, codes, scales};
  cudaStream_t st = as_stream(stream);
  const bool wide = type != ROUGE_B200_T_F32 && cols % 8 == 0 && all(16) &&
                    (reinterpret_cast<uintptr_t>(codes) & 7u) == 0;
  switch (type) {
    case ROUGE_B200_T_F32: return launch_fmt<ROUGE_B200_T_F32, 4>(a, out_fmt, st);
    case ROUGE_B200_T_F16:
      return wide ? launch_fmt<ROUGE_B200_T_F16, 8>(a, out_fmt, st)
                  : launch_fmt<ROUGE_B200_T_F16, 4>(a, out_fmt, st);
    default:
      return wide ? launch_fmt<ROUGE_B200_T_BF16, 8>(a, out_fmt, st)
                  : launch_fmt<ROUGE_B200_T_BF16, 4>(a, out_fmt, st);
  }
}
