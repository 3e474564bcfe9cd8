// Residual addition, RMS norm and 8-bit output in one kernel:
//   h = round_T(x + r)               written to h_out (the residual stream)
//   y = (float)(h / sqrt(sum h^2 / n + eps)) * w      (transformer.cpp:33-40)
//   codes, scales = per-row int8 (quant_int8.cpp:72-90) or MXFP8 e4m3
//                   blocks of 32 (narrow.cpp:200-265) of y
// with the arithmetic of those steps apart: sum of squares and inverse root
// in double, the scaled product rounded once (norm_values), so the codes are
// those of rouge_rmsnorm followed by the quantizer, unless the scaled product
// lies within about 2^-47 of itself of the middle of two floats (the sum of
// squares is added up in another order). The sign of a NaN is not kept.
//
// Memory-bound: a row is read once and stays in registers (16 values per
// thread) over both reductions -- the sum of squares, then the row maximum
// of y -- and the codes, while the block's next row is on its way into other
// registers. One to 32 warps share a row, so that 512 to 16384 columns fit;
// longer rows take the looping kernel, which reads h again. With residual: 4096
// x 4096 f32 to int8 42 us, 8191 x 8192 bf16 to MXFP8 86 (79 and 84 % of the
// copy rate); the latter uses 67 % of the issue slots. Wider f32 rows are
// slower, 4096 x 8192 98 us (68 %): 16 warps a row leave a thread 64 registers,
// of which the row, the next row and its residual are 48, and 180 bytes spill.
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

// Row values a thread holds. (32 of a 16-bit row halve the share of the
// reductions, about 90 instructions a row, but leave half the threads: 8191 x
// 8192 bf16 to MXFP8 took 104 us with 32, 86 with 16.)
constexpr int kPerThread = 16;

struct NormArgs {
  const void *x, *r;
  long long ldx, ldr, ldh;
  const float *w;
  float eps;
  int rows, cols;
  double by_cols;  // 1 / cols
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
  // this += o, rounded to the type (the 16-bit types' packed additions round
  // the exact sum once; so does the f32 sum rounded to 16 bits, since a sum
  // too long for f32 is far from the middle of two 16-bit values)
  __device__ __forceinline__ void add(const Raw &o) {
#pragma unroll
    for (int q = 0; q < WORDS; ++q) {
      if constexpr (T == ROUGE_B200_T_F32) {
        w[q] = __float_as_uint(__fadd_rn(__uint_as_float(w[q]), __uint_as_float(o.w[q])));
      } else if constexpr (T == ROUGE_B200_T_F16) {
        asm("add.rn.f16x2 %0, %0, %1;" : "+r"(w[q]) : "r"(o.w[q]));
      } else {
        asm("add.rn.bf16x2 %0, %0, %1;" : "+r"(w[q]) : "r"(o.w[q]));
      }
    }
  }
  __device__ __forceinline__ void store(void *base, long long at) const {
    char *p = static_cast<char *>(base) + at * (T == ROUGE_B200_T_F32 ? 4 : 2);
    if constexpr (WORDS == 2)
      *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
    else
      *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
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

__device__ __forceinline__ void group_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(threads) : "memory");
}

// The row's inverse root mean square: the double, and its two leading floats
// (hi + lo = the double to 2^-48). hi is infinite where two floats do not
// serve: where the double or its lower part leaves f32's normal range, and
// where the row is so small that its outputs or their remainders may.
struct InvRms {
  double full;
  float hi, lo;
};

// 1 / sqrt(ss / n + eps) to double accuracy: two Newton steps from the f32
// approximation (2^-22, 2^-43, 2^-53), in a chain a third as long as double
// division, root and division; those serve for values out of f32's range.
__device__ __forceinline__ InvRms inverse_rms(double ss, double by_n, float eps) {
  const double mean = __dmul_rn(ss, by_n);
  const double v = __dadd_rn(mean, static_cast<double>(eps));
  InvRms r;
  // 0 < mean < 2^-180 by its high word (a row of zeros is zeros either way)
  bool two_floats = static_cast<unsigned>(__double2hiint(mean) - 1) >= ((1023u - 180u) << 20) - 1u;
  if (v > 1e-30 && v < 1e30) {
    double y = static_cast<double>(rsqrtf(__double2float_rn(v)));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const double e = __fma_rn(-__dmul_rn(v, y), y, 1.0);  // 1 - v y^2
      y = __fma_rn(__dmul_rn(0.5, y), e, y);
    }
    r.full = y;
  } else {
    r.full = __ddiv_rn(1.0, __dsqrt_rn(v));
    two_floats = two_floats && !(r.full < 7.9e-31);  // 2^-100
  }
  r.hi = __double2float_rn(r.full);
  r.lo = __double2float_rn(__dsub_rn(r.full, static_cast<double>(r.hi)));
  if (!two_floats) r.hi = INFINITY;
  return r;
}

// y of V values in place: h times the inverse rounded once to f32, then
// times w, rounded (rouge_rmsnorm's arithmetic, whose product is in double).
// The product is taken in two floats -- p + t with t good to 2^-24 of itself
// -- instead of double, whose conversions run at an eighth of the rate; the
// rounded sum is the double's but where that lies within 2^-47 of the middle
// of two floats.
template <int V>
__device__ __forceinline__ void norm_values(float (&h)[V], const InvRms &inv, const float (&w)[V]) {
  if (isinf(inv.hi)) {  // (for rows of zeros without eps: NaN)
#pragma unroll
    for (int j = 0; j < V; ++j)
      h[j] = __fmul_rn(__double2float_rn(__dmul_rn(static_cast<double>(h[j]), inv.full)), w[j]);
    return;
  }
#pragma unroll
  for (int j = 0; j < V; j += 2) {
    float p0, p1, t0, t1;
    mul2(p0, p1, h[j], h[j + 1], inv.hi);
    t0 = __fmaf_rn(h[j], inv.hi, -p0);  // (paired sums have no free negation)
    t1 = __fmaf_rn(h[j + 1], inv.hi, -p1);
    fma2(t0, t1, h[j], h[j + 1], inv.lo, t0, t1);
    add2(p0, p1, p0, p1, t0, t1);
    mul2(h[j], h[j + 1], p0, p1, w[j], w[j + 1]);
  }
}

// Scale of an int8 row from the maximum of |y| (quant_int8.cpp:82-84, where
// both quotients are taken in double and rounded to f32: 127 m and s m, m the
// middle of two floats, are never within 2^-49 of a float a or of 1, so the
// f32 quotients are the same).
struct RowScale {
  float scale, inv_f;
};
__device__ __forceinline__ RowScale row_scale(float amax) {
  RowScale r;
  r.scale = amax > 0.0f ? __fdiv_rn(amax, 127.0f) : 1.0f;
  r.inv_f = __fdiv_rn(1.0f, r.scale);
  return r;
}

// A value reduced over the WPR warps of a row group, known to all of them:
// the warps' parts meet in `slot` behind one barrier and every warp adds
// them up. The slots of a reduction are written again two barriers later.
template <int WPR, class V, class Op>
__device__ __forceinline__ V group_reduce(V v, V *slot, int group, int wig, int lane, Op op) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if constexpr (WPR > 1) {
    if (lane == 0) slot[wig] = v;
    group_sync(group, WPR * 32);
    v = slot[lane % WPR];
#pragma unroll
    for (int o = WPR / 2; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  }
  return v;
}

// (not inlined: one word in a few hundred gets here, and the division's
// registers would be taken from the rows under way)
__device__ __noinline__ uint32_t encode4_i8_by(float4 t, float scale) {
  return encode4_i8_exact(t, __ddiv_rn(1.0, static_cast<double>(scale)));
}

// Codes of V consecutive values of one row starting at column c. I8: from
// the row's scale; MX: each block of 32 is V-value lanes next to each other.
template <int FMT, int V>
__device__ __forceinline__ void store_codes(const NormArgs &a, int row, int c, const float (&y)[V],
                                            bool live, const RowScale &rs) {
  uint32_t w[V / 4];
  if constexpr (FMT == ROUGE_B200_Q_I8_ROWS) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      const float4 t = make_float4(y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]);
      bool tie;
      w[q] = encode4_i8_fast(t, rs.inv_f, tie);
      if (tie || isinf(rs.inv_f)) w[q] = encode4_i8_by(t, rs.scale);
    }
  } else {
    float m = 0.0f;  // (a NaN stays: the block then takes the exact encoder)
#pragma unroll
    for (int j = 0; j < V; ++j) m = max_nan(m, fabsf(y[j]));
#pragma unroll
    for (int o = 1; o < 32 / V; o <<= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    uint32_t sc = mx_scale_code(m > 448.0f ? block_pow(m, 448.0f) : 0);
    if (__any_sync(0xffffffffu, m != m)) {
      float top = 0.0f;  // the maximum of the others
#pragma unroll
      for (int j = 0; j < V; ++j) top = fmaxf(top, fabsf(y[j]));
#pragma unroll
      for (int o = 1; o < 32 / V; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      sc = mx_scale_code(block_pow(top, 448.0f));
    }
    const float si = e8m0_inverse(sc);
#pragma unroll
    for (int q = 0; q < V / 4; ++q)
      w[q] = mx_encode4_f8<kE4M3>(make_float4(y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]),
                                  si, m != m);
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
__global__ void __launch_bounds__(WPR > 8 ? WPR * 32 : 256, WPR > 16 ? 1 : WPR > 8 ? 2 : 3)
    norm_quant_kernel(const NormArgs a) {
  constexpr int kWarps = WPR > 8 ? WPR : 8, kGroups = kWarps / WPR, kNv = kPerThread / V;
  __shared__ double sum_slot[2][kWarps];
  __shared__ float max_slot[kWarps];
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
  for (int odd = 0; row < a.rows; row += gridDim.x * kGroups, odd ^= 1) {
    float h[kNv][V];
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < kNv; ++i) {
      const int c = c0 + i * kStep;
      if constexpr (RES) {
        xr[i].add(rr[i]);
        if (c < a.cols) xr[i].store(a.h, row * a.ldh + c);
      }
      xr[i].unpack(h[i]);
    }
    // the next row's loads run under this row's reductions and codes
    const int next = row + gridDim.x * kGroups;
    if (next < a.rows) fetch(next);
#pragma unroll
    for (int i = 0; i < kNv; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) ss = __fma_rn(static_cast<double>(h[i][j]), h[i][j], ss);
    ss = group_reduce<WPR>(ss, sum_slot[odd] + group * WPR, group, wig, lane,
                           [](double p, double q) { return __dadd_rn(p, q); });
    const InvRms inv = inverse_rms(ss, a.by_cols, a.eps);
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < kNv; ++i) {
      const int c = c0 + i * kStep;
      if (c < a.cols) {
        float wv[V];
        load_weights<V>(a.w, c, wv);
        norm_values<V>(h[i], inv, wv);
#pragma unroll
        for (int j = 0; j < V; ++j) amax = fmaxf(amax, fabsf(h[i][j]));
      }
    }
    RowScale rs{};
    if constexpr (FMT == ROUGE_B200_Q_I8_ROWS) {
      rs = row_scale(group_reduce<WPR>(amax, max_slot + group * WPR, group, wig, lane,
                                       [](float p, float q) { return fmaxf(p, q); }));
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
  __shared__ double sum_slot[2][32];
  __shared__ float max_slot[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const void *src = a.r ? a.h : a.x;
  const long long lds = a.r ? a.ldh : a.ldx;
  for (int row = blockIdx.x, odd = 0; row < a.rows; row += gridDim.x, odd ^= 1) {
    double ss = 0.0;
    for (int c = threadIdx.x * V; c < a.cols; c += 1024 * V) {
      Raw<T, V> x;
      x.load(a.x, row * a.ldx + c);
      if (a.r) {
        Raw<T, V> r;
        r.load(a.r, row * a.ldr + c);
        x.add(r);
        x.store(a.h, row * a.ldh + c);
      }
      float h[V];
      x.unpack(h);
#pragma unroll
      for (int j = 0; j < V; ++j) ss = __fma_rn(static_cast<double>(h[j]), h[j], ss);
    }
    ss = group_reduce<32>(ss, sum_slot[odd], 0, warp, lane,
                          [](double p, double q) { return __dadd_rn(p, q); });
    const InvRms inv = inverse_rms(ss, a.by_cols, a.eps);
    auto values = [&](int c, float (&y)[V]) {
      float wv[V];
      load_vec<T, V>(src, row * lds + c, y);
      load_weights<V>(a.w, c, wv);
      norm_values<V>(y, inv, wv);
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
      rs = row_scale(group_reduce<32>(amax, max_slot, 0, warp, lane,
                                      [](float p, float q) { return fmaxf(p, q); }));
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
  constexpr int per_warp = 32 * kPerThread;
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
  if (rows > (1 << 30) || cols > (1 << 30)) return set_status(ROUGE_B200_EUNSUPPORTED);
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
  NormArgs a{x, residual, ldx, ldr, ldh, w, eps, rows, cols, 1.0 / cols, h_out, codes, scales};
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
