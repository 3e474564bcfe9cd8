// Residual addition, RMS norm and 8-bit output in one kernel:
//   h = round_T(x + r)               written to h_out (the residual stream)
//   y = (float)(h / sqrt(sum h^2 / n + eps)) * w      (transformer.cpp:33-40)
//   codes, scales = per-row int8 (quant_int8.cpp:72-90) or MXFP8 e4m3
//                   blocks of 32 (narrow.cpp:200-265) of y
// with the arithmetic of those steps apart: sum of squares and inverse root
// in double, the scaled product rounded once (norm_value), so the codes are
// those of rouge_rmsnorm followed by the quantizer.
//
// Memory-bound: a row is read once and stays in registers (16 values per
// thread) over both reductions -- the sum of squares, then the row maximum
// of y -- and the codes, while the block's next row is on its way into other
// registers. One to 32 warps share a row, so that 512 to 16384 columns fit;
// longer rows take the looping kernel, which reads h again.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
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

// V consecutive elements of type T as they lie in memory (8 or 16 bytes).
template <int T, int V>
struct Raw {
  static constexpr int WORDS = T == ROUGE_B200_T_F32 ? V : V / 2;
  uint32_t w[WORDS];
  __device__ __forceinline__ void load(const void *base, long long at) {
    const char *p = static_cast<const char *>(base) + at * (T == ROUGE_B200_T_F32 ? 4 : 2);
    if constexpr (WORDS == 2) {
      const uint2 t = *reinterpret_cast<const uint2 *>(p);
      w[0] = t.x; w[1] = t.y;
    } else {
      const uint4 t = *reinterpret_cast<const uint4 *>(p);
      w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w;
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void unpack(float (&v)[V]) const {
#pragma unroll
    for (int q = 0; q < WORDS; ++q) {
      if constexpr (T == ROUGE_B200_T_F32) {
        v[q] = __uint_as_float(w[q]);
      } else if constexpr (T == ROUGE_B200_T_F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[q]));
        v[2 * q] = f.x; v[2 * q + 1] = f.y;
      } else {
        v[2 * q] = __uint_as_float(w[q] << 16);
        v[2 * q + 1] = __uint_as_float(w[q] & 0xFFFF0000u);
      }
    }
  }
};

template <int T, int V>
__device__ __forceinline__ void load_vec(const void *base, long long at, float (&v)[V]) {
  Raw<T, V> r;
  r.load(base, at);
  r.unpack(v);
}

// The weights of V columns.
template <int V>
__device__ __forceinline__ void load_weights(const float *w, int c, float (&v)[V]) {
#pragma unroll
  for (int q = 0; q < V / 4; ++q) {
    const float4 t = __ldg(reinterpret_cast<const float4 *>(w + c) + q);
    v[4 * q] = t.x; v[4 * q + 1] = t.y; v[4 * q + 2] = t.z; v[4 * q + 3] = t.w;
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

__device__ __forceinline__ double norm_inverse(double ss, int n, float eps) {
  return __ddiv_rn(1.0, __dsqrt_rn(__dadd_rn(__ddiv_rn(ss, static_cast<double>(n)),
                                             static_cast<double>(eps))));
}

// The row's inverse root mean square in two floats, hi + lo = the double to
// 2^-48.
struct InvRms {
  float hi, lo;
};
__device__ __forceinline__ InvRms split_inverse(double inv) {
  const float hi = __double2float_rn(inv);
  // (an infinite or NaN inverse has no low part)
  const float lo = isinf(hi) || isnan(hi) ? 0.0f : __double2float_rn(__dsub_rn(inv, hi));
  return InvRms{hi, lo};
}

// y of one value: h times the inverse rounded once to f32, then times w,
// rounded (rouge_rmsnorm's arithmetic, whose product is in double). The
// product is taken in two floats -- p + t with t good to 2^-24 of itself --
// instead of double, whose conversions run at an eighth of the rate; the
// rounded sum is the double's but where that lies within 2^-47 of the middle
// of two floats.
__device__ __forceinline__ float norm_value(float h, InvRms inv, float w) {
  const float p = __fmul_rn(h, inv.hi);
  const float t = __fmaf_rn(h, inv.lo, __fmaf_rn(h, inv.hi, -p));
  // (an infinite p has a NaN remainder; a remainder below the subnormals is 0)
  const float y = fabsf(p) < INFINITY ? __fadd_rn(p, t) : p;
  return __fmul_rn(y, w);
}

// Scale of an int8 row from the maximum of |y| (quant_int8.cpp:82-84).
struct RowScale {
  double inv;
  float scale, inv_f;
};
__device__ __forceinline__ RowScale row_scale(float amax) {
  const double m = static_cast<double>(amax);
  RowScale r;
  r.scale = m > 0.0 ? __double2float_rn(__ddiv_rn(m, 127.0)) : 1.0f;
  r.inv = __ddiv_rn(1.0, static_cast<double>(r.scale));
  r.inv_f = __double2float_rn(r.inv);
  return r;
}

// A value reduced over the WPR warps of a row group, and what `finish` makes
// of it, known to all of them: the warps' parts meet in `slot`, the group's
// first warp finishes (the double divisions are done once) and leaves the
// result in `out`. Two barriers; slot and out are written again only after
// every thread has passed another pair.
template <int WPR, class V, class R, class Op, class Finish>
__device__ __forceinline__ R group_reduce(V v, V *slot, R *out, int group, int wig, int lane, Op op,
                                          Finish finish) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if constexpr (WPR == 1) {
    return finish(v);
  } else {
    if (lane == 0) slot[wig] = v;
    group_sync(group, WPR * 32);
    if (wig == 0) {
      v = slot[lane % WPR];
#pragma unroll
      for (int o = WPR / 2; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
      const R r = finish(v);
      if (lane == 0) *out = r;
    }
    group_sync(group, WPR * 32);
    return *out;
  }
}

// Codes of V consecutive values of one row starting at column c. I8: from
// the row's scale; MX: each block of 32 is V-value lanes next to each other.
template <int FMT, int V>
__device__ __forceinline__ void store_codes(const NormArgs &a, int row, int c, const float (&y)[V],
                                            bool live, const RowScale &rs) {
  uint32_t w[V / 4];
  if constexpr (FMT == ROUGE_B200_Q_I8_ROWS) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q)
      w[q] = encode4_i8_x2(make_float4(y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]), rs.inv,
                           rs.inv_f, isinf(rs.inv_f));
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

template <int T, int V, int FMT, int WPR, bool RES>
__global__ void __launch_bounds__(WPR > 8 ? WPR * 32 : 256)
    norm_quant_kernel(const NormArgs a) {
  constexpr int kWarps = WPR > 8 ? WPR : 8, kGroups = kWarps / WPR, kNv = kPerThread / V;
  __shared__ double sum_slot[kWarps];
  __shared__ float max_slot[kWarps];
  __shared__ InvRms rms_out[kGroups];
  __shared__ RowScale scale_out[kGroups];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = warp / WPR, wig = warp % WPR;
  const int c0 = (wig * 32 + lane) * V;  // first column; the next kNv - 1 are WPR * 32 * V apart
  constexpr int kStep = WPR * 32 * V;
  Raw<T, V> xr[kNv], rr[RES ? kNv : 1];
  auto fetch = [&](int row) {
#pragma unroll
    for (int i = 0; i < kNv; ++i) {
      const int c = c0 + i * kStep;
      if (c < a.cols) {
        xr[i].load(a.x, row * a.ldx + c);
        if constexpr (RES) rr[i].load(a.r, row * a.ldr + c);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kNv; ++i) {  // (columns past the row stay zeros)
    xr[i].zero();
    if constexpr (RES) rr[i].zero();
  }
  int row = blockIdx.x * kGroups + group;
  if (row < a.rows) fetch(row);
  for (; row < a.rows; row += gridDim.x * kGroups) {
    float h[kNv][V];
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < kNv; ++i) {
      const int c = c0 + i * kStep;
      xr[i].unpack(h[i]);
      if constexpr (RES) {
        float t[V];
        rr[i].unpack(t);
#pragma unroll
        for (int j = 0; j < V; ++j) h[i][j] = __fadd_rn(h[i][j], t[j]);
        if (c < a.cols) round_store<T, V>(a.h, row * a.ldh + c, h[i]);
      }
    }
    // the next row's loads run under this row's reductions and codes
    const int next = row + gridDim.x * kGroups;
    if (next < a.rows) fetch(next);
#pragma unroll
    for (int i = 0; i < kNv; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) ss = __fma_rn(static_cast<double>(h[i][j]), h[i][j], ss);
    const InvRms inv = group_reduce<WPR>(
        ss, sum_slot + group * WPR, rms_out + group, group, wig, lane,
        [](double p, double q) { return __dadd_rn(p, q); },
        [&](double v) { return split_inverse(norm_inverse(v, a.cols, a.eps)); });
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < kNv; ++i) {
      const int c = c0 + i * kStep;
      if (c < a.cols) {
        float wv[V];
        load_weights<V>(a.w, c, wv);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          h[i][j] = norm_value(h[i][j], inv, wv[j]);
          amax = fmaxf(amax, fabsf(h[i][j]));
        }
      }
    }
    RowScale rs{};
    if constexpr (FMT == ROUGE_B200_Q_I8_ROWS) {
      rs = group_reduce<WPR>(amax, max_slot + group * WPR, scale_out + group, group, wig, lane,
                             [](float p, float q) { return fmaxf(p, q); },
                             [](float v) { return row_scale(v); });
      if (wig == 0 && lane == 0) static_cast<float *>(a.scales)[row] = rs.scale;
    }
#pragma unroll
    for (int i = 0; i < kNv; ++i) {
      const int c = c0 + i * kStep;
      store_codes<FMT, V>(a, row, c, h[i], c < a.cols, rs);
    }
  }
}

// Rows past 32 warps' registers: 32 warps loop over the row three times,
// reading h again (from h_out, written by the same threads, or x).
template <int T, int V, int FMT>
__global__ void __launch_bounds__(1024) norm_quant_long_kernel(const NormArgs a) {
  __shared__ double sum_slot[32];
  __shared__ float max_slot[32];
  __shared__ InvRms rms_out;
  __shared__ RowScale scale_out;
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
    const InvRms inv = group_reduce<32>(
        ss, sum_slot, &rms_out, 0, warp, lane, [](double p, double q) { return __dadd_rn(p, q); },
        [&](double v) { return split_inverse(norm_inverse(v, a.cols, a.eps)); });
    auto values = [&](int c, float (&y)[V]) {
      float wv[V];
      load_vec<T, V>(src, row * lds + c, y);
      load_weights<V>(a.w, c, wv);
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = norm_value(y[j], inv, wv[j]);
    };
    RowScale rs{};
    if constexpr (FMT == ROUGE_B200_Q_I8_ROWS) {
      float amax = 0.0f;
      for (int c = threadIdx.x * V; c < a.cols; c += 1024 * V) {
        float y[V];
        values(c, y);
#pragma unroll
        for (int j = 0; j < V; ++j) amax = fmaxf(amax, fabsf(y[j]));
      }
      rs = group_reduce<32>(amax, max_slot, &scale_out, 0, warp, lane,
                            [](float p, float q) { return fmaxf(p, q); },
                            [](float v) { return row_scale(v); });
      if (threadIdx.x == 0) static_cast<float *>(a.scales)[row] = rs.scale;
    }
    // (whole warps: a block's lanes take part in its shuffles)
    for (int c1 = 0; c1 < a.cols; c1 += 1024 * V) {
      const int c = c1 + threadIdx.x * V;
      float y[V];
      if (c < a.cols) {
        values(c, y);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) y[j] = 0.0f;
      }
      store_codes<FMT, V>(a, row, c, y, c < a.cols, rs);
    }
  }
}

template <class Kernel>
int launch_rows(Kernel kernel, const NormArgs &a, int threads, int groups, std::atomic<int> &per_sm,
                cudaStream_t st) {
  int n = per_sm.load();
  if (n == 0) {  // resident blocks per SM: a block takes row after row
    const int s = cuda_status(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0));
    if (s != ROUGE_B200_OK) return s;
    per_sm.store(n = n < 1 ? 1 : n);
  }
  const long long want = (static_cast<long long>(a.rows) + groups - 1) / groups;
  const long long cap = static_cast<long long>(current_sm_count()) * n;
  kernel<<<static_cast<unsigned>(want < cap ? want : cap), threads, 0, st>>>(a);
  return cuda_status(cudaGetLastError());
}

template <int T, int V, int FMT, int WPR>
int launch_wpr(const NormArgs &a, cudaStream_t st) {
  constexpr int kThreads = WPR > 8 ? WPR * 32 : 256, kGroups = kThreads / 32 / WPR;
  static std::atomic<int> with{0}, without{0};
  return a.r ? launch_rows(norm_quant_kernel<T, V, FMT, WPR, true>, a, kThreads, kGroups, with, st)
             : launch_rows(norm_quant_kernel<T, V, FMT, WPR, false>, a, kThreads, kGroups, without, st);
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
