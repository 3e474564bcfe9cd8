// Writing to and reading from the paged 4-bit key / value cache.
//
// One thread per block of 16 values of one token and head: 16 elements in
// registers, so the block's maximum needs no shuffle, and 8 bytes of codes
// plus one scale byte out (or the reverse). Neighbouring threads hold
// neighbouring blocks, so a warp reads whole lines of K or V and writes
// whole sectors of the page. The floor is memory: 2 or 4 bytes in and 0.5625
// bytes out per value. 32768 bf16 tokens of 8 x 128: 39 to 41 us to write (64 to
// 67 % of the copy rate; no pipe is full: 64 % of the issue slots, 58 % of the
// integer pipe, about 200 instructions per thread), 31 to read (84 %). Two
// blocks per thread in flight gained nothing in either.
#include <cuda_runtime.h>

#include <cstdint>

#include "kv4.cuh"
#include "narrow.cuh"
#include "ptx.cuh"
#include "x86fp.cuh"

namespace rb200 {
namespace {

constexpr int kThreads = 256;

struct KvArgs {
  uint8_t *codes[2], *scales[2];
  const float *gs[2];
  const void *src[2];
  void *dst[2];
  long long ld[2];
  int page, Hkv, nblk;  // nblk = Dh / 16
  Divisor by_nblk, by_heads, by_page;
  int wide[2];  // source (or destination) and pitch are multiples of 32 bytes
  int total_slots;
  unsigned items;       // tokens * Hkv * nblk of this launch
  const int *slots;
  int *err;
};

// 32 bytes in one access (a thread's block is 32 or 64 bytes: two accesses of
// 16 would touch each of the warp's lines twice: 41.0 us instead of 30.8 to read
// 32768 bf16 tokens of 8 x 128; writing them gains 0.2).
__device__ __forceinline__ void ld32(const void *p, bool wide, uint32_t (&u)[8]) {
  if (wide) {
    asm("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7])
        : "l"(p));
    return;
  }
  const uint4 *q = static_cast<const uint4 *>(p);
  const uint4 t0 = __ldg(q), t1 = __ldg(q + 1);
  u[0] = t0.x; u[1] = t0.y; u[2] = t0.z; u[3] = t0.w;
  u[4] = t1.x; u[5] = t1.y; u[6] = t1.z; u[7] = t1.w;
}

__device__ __forceinline__ void st32(void *p, bool wide, const uint32_t (&u)[8]) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(u[0]), "r"(u[1]),
                 "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
                 : "memory");
    return;
  }
  uint4 *q = static_cast<uint4 *>(p);
  q[0] = make_uint4(u[0], u[1], u[2], u[3]);
  q[1] = make_uint4(u[4], u[5], u[6], u[7]);
}

template <int T>
__device__ __forceinline__ void load16(const void *p, long long at, bool wide, float (&v)[16]) {
  uint32_t u[8];
  if constexpr (T == ROUGE_B200_T_F32) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      ld32(static_cast<const float *>(p) + at + 8 * k, wide, u);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[8 * k + i] = __uint_as_float(u[i]);
    }
  } else {
    ld32(static_cast<const uint16_t *>(p) + at, wide, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (T == ROUGE_B200_T_F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
      } else {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
      }
    }
  }
}

template <int T>
__device__ __forceinline__ void store16(void *p, long long at, bool wide, const float (&v)[16]) {
  uint32_t u[8];
  if constexpr (T == ROUGE_B200_T_F32) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = __float_as_uint(v[8 * k + i]);
      st32(static_cast<float *>(p) + at + 8 * k, wide, u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      u[i] = T == ROUGE_B200_T_F16 ? f16x2_rn(v[2 * i], v[2 * i + 1]) : bf16x2_rn(v[2 * i], v[2 * i + 1]);
    st32(static_cast<uint16_t *>(p) + at, wide, u);
  }
}

// Where item i (token, head, block) lies: false for a skipped token.
__device__ __forceinline__ bool locate(const KvArgs &a, unsigned i, int &head, long long &el,
                                       int which, size_t &blk_at) {
  const unsigned th = a.by_nblk.div(i), blk = i - th * a.nblk;
  const unsigned t = a.by_heads.div(th);
  head = static_cast<int>(th - t * a.Hkv);
  const int slot = __ldg(a.slots + t);
  if (slot < 0) return false;
  if (slot >= a.total_slots) {
    atomicCAS(a.err, 0, ROUGE_B200_EINVAL);
    return false;
  }
  el = t * a.ld[which] + static_cast<long long>(head * a.nblk + static_cast<int>(blk)) * 16;
  const int p = a.by_page.div(slot), at = slot - p * a.page;
  blk_at = ((static_cast<size_t>(p) * a.Hkv + head) * a.page + at) * a.nblk + blk;
  return true;
}

// Quotients x / step for the codes' border tests, correctly rounded: one
// Newton step on the product with the reciprocal, whose residual is exact
// while nothing under- or overflows (quotients up to 2^24 here); a quotient
// that is exactly a border between two codes is then met exactly.
__device__ __forceinline__ void quotients(float &x, float &y, float step, float inv) {
  float q0, q1, r0, r1;
  mul2(q0, q1, x, y, inv);
  fma2(r0, r1, q0, q1, -step, x, y);
  fma2(x, y, r0, r1, inv, q0, q1);
}

// The same for one value of a block that holds an infinity or a NaN, or whose
// step or largest quotient (where the scale has saturated) is extreme:
// infinities divide to infinities, as do quotients too large, NaN stays.
__device__ __forceinline__ float quotient_any(float x, float step) { return __fdiv_rn(x, step); }

// Clears the sign of zero codes (the hardware keeps it; eight nibbles).
__device__ __forceinline__ uint32_t unsigned_zeros(uint32_t w) {
  const uint32_t mag = w & 0x77777777u;
  return mag | (w & (mag + 0x77777777u) & 0x88888888u);
}

template <int T>
__global__ void __launch_bounds__(kThreads) kv4_write_kernel(const KvArgs a) {
  const int which = blockIdx.y;
  for (unsigned i = blockIdx.x * kThreads + threadIdx.x; i < a.items; i += gridDim.x * kThreads) {
    int head;
    long long el;
    size_t at;
    if (!locate(a, i, head, el, which, at)) continue;
    float v[16];
    load16<T>(a.src[which], el, a.wide[which], v);
    const float g = a.gs[which] ? __ldg(a.gs[which] + head) : 1.0f;
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; ++j) m = max_nan(m, fabsf(v[j]));
    const bool odd = !(m < INFINITY);
    if (m != m) {  // the maximum of the others
      m = 0.0f;
#pragma unroll
      for (int j = 0; j < 16; ++j) m = fmaxf(m, fabsf(v[j]));
    }
    const uint32_t sc = cvt_pair_e4m3(__fdiv_rn(m, __fmul_rn(6.0f, g)), 0.0f) & 0xFFu;
    const uint32_t sh = e4m3x2_f16x2(sc);
    const float step = __fmul_rn(__half2float(__ushort_as_half(static_cast<unsigned short>(sh))), g);
    uint2 w = make_uint2(0u, 0u);
    if (step > 0.0f) {
      if (odd || !(step > 7.9e-31f && step < 1.2e30f) || m > 16777216.0f * step) {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = quotient_any(v[j], step);
      } else {
        const float inv = __fdiv_rn(1.0f, step);
#pragma unroll
        for (int j = 0; j < 16; j += 2) quotients(v[j], v[j + 1], step, inv);
      }
      w.x = unsigned_zeros(cvt4_e2m1(v[0], v[1], v[2], v[3]) | (cvt4_e2m1(v[4], v[5], v[6], v[7]) << 16));
      w.y = unsigned_zeros(cvt4_e2m1(v[8], v[9], v[10], v[11]) |
                           (cvt4_e2m1(v[12], v[13], v[14], v[15]) << 16));
    }
    reinterpret_cast<uint2 *>(a.codes[which])[at] = w;
    a.scales[which][at] = static_cast<uint8_t>(sc);
  }
}

template <int T>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(const KvArgs a) {
  const int which = blockIdx.y;
  for (unsigned i = blockIdx.x * kThreads + threadIdx.x; i < a.items; i += gridDim.x * kThreads) {
    int head;
    long long el;
    size_t at;
    if (!locate(a, i, head, el, which, at)) continue;
    const uint2 w = __ldg(reinterpret_cast<const uint2 *>(a.codes[which]) + at);
    const uint32_t sh = e4m3x2_f16x2(__ldg(a.scales[which] + at));
    const float s = __half2float(__ushort_as_half(static_cast<unsigned short>(sh)));
    const float g = a.gs[which] ? __ldg(a.gs[which] + head) : 1.0f;
    float v[16];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t h[4];
      e2m1x8_f16x2(k ? w.y : w.x, h);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[j]));
        v[8 * k + 2 * j] = __fmul_rn(__fmul_rn(f.x, s), g);  // (code * scale is exact)
        v[8 * k + 2 * j + 1] = __fmul_rn(__fmul_rn(f.y, s), g);
      }
    }
    store16<T>(a.dst[which], el, a.wide[which], v);
  }
}

int prepare(const RougeB200KV4 *c, const void *K, long long ldk, const void *V, long long ldv,
            int type, int T, const int *slots, KvArgs &a) {
  int s = check_kv4(c);
  if (s != ROUGE_B200_OK) return s;
  if (T < 0 || !valid_float_type(type)) return ROUGE_B200_EINVAL;
  if (T == 0) return ROUGE_B200_OK;
  const long long row = static_cast<long long>(c->Hkv) * c->Dh;
  if (!K || !V || !slots || ldk < row || ldv < row) return ROUGE_B200_EINVAL;
  const int es = type == ROUGE_B200_T_F32 ? 4 : 2;
  if (((reinterpret_cast<uintptr_t>(K) | reinterpret_cast<uintptr_t>(V)) & 15u) ||
      (ldk * es) % 16 || (ldv * es) % 16 || (reinterpret_cast<uintptr_t>(slots) & 3u))
    return ROUGE_B200_EUNSUPPORTED;
  a.codes[0] = c->k_codes; a.codes[1] = c->v_codes;
  a.scales[0] = c->k_scales; a.scales[1] = c->v_scales;
  a.gs[0] = c->gs_k; a.gs[1] = c->gs_v;
  a.ld[0] = ldk; a.ld[1] = ldv;
  a.wide[0] = (reinterpret_cast<uintptr_t>(K) & 31u) == 0 && (ldk * es) % 32 == 0;
  a.wide[1] = (reinterpret_cast<uintptr_t>(V) & 31u) == 0 && (ldv * es) % 32 == 0;
  a.page = c->page;
  a.Hkv = c->Hkv;
  a.nblk = c->Dh / 16;
  a.by_nblk = Divisor(a.nblk);
  a.by_heads = Divisor(a.Hkv);
  a.by_page = Divisor(a.page);
  a.total_slots = c->pages * c->page;
  a.slots = slots;
  return ROUGE_B200_OK;
}

// Launches `kernel` over the tokens, at most 2^30 items at a time.
template <class Kernel>
int launch_tokens(Kernel kernel, KvArgs a, int T, int esize, cudaStream_t st) {
  const int per_token = a.Hkv * a.nblk;
  const int step = per_token < (1 << 30) ? (1 << 30) / per_token : 1;
  const long long cap = static_cast<long long>(current_sm_count()) * 8;
  for (int t0 = 0; t0 < T; t0 += step) {
    const int n = T - t0 < step ? T - t0 : step;
    a.items = static_cast<unsigned>(n) * per_token;
    const long long want = (static_cast<long long>(a.items) + kThreads - 1) / kThreads;
    kernel<<<dim3(static_cast<unsigned>(want < cap ? want : cap), 2), kThreads, 0, st>>>(a);
    const int s = cuda_status(cudaGetLastError());
    if (s != ROUGE_B200_OK || T - t0 <= step) return s;
    a.slots += n;
    for (int w = 0; w < 2; ++w) {
      const long long bytes = n * a.ld[w] * esize;
      if (a.src[w]) a.src[w] = static_cast<const uint8_t *>(a.src[w]) + bytes;
      if (a.dst[w]) a.dst[w] = static_cast<uint8_t *>(a.dst[w]) + bytes;
    }
  }
  return ROUGE_B200_OK;
}

}  // namespace
}  // namespace rb200

using namespace rb200;

extern "C" {

int rouge_b200_kv4_write(const RougeB200KV4 *cache, const void *K, long long ldk, const void *V,
                         long long ldv, int type, int T, const int *slots, void *stream) {
  KvArgs a{};
  int s = prepare(cache, K, ldk, V, ldv, type, T, slots, a);
  if (s != ROUGE_B200_OK) return set_status(s);
  s = device_ready();
  if (s != ROUGE_B200_OK || T == 0) return s;
  a.src[0] = K;
  a.src[1] = V;
  a.err = device_error_word();
  if (!a.err) return set_status(ROUGE_B200_ENOMEM);
  cudaStream_t st = as_stream(stream);
  switch (type) {
    case ROUGE_B200_T_F32: return launch_tokens(kv4_write_kernel<ROUGE_B200_T_F32>, a, T, 4, st);
    case ROUGE_B200_T_F16: return launch_tokens(kv4_write_kernel<ROUGE_B200_T_F16>, a, T, 2, st);
    default: return launch_tokens(kv4_write_kernel<ROUGE_B200_T_BF16>, a, T, 2, st);
  }
}

int rouge_b200_kv4_read(const RougeB200KV4 *cache, void *K, long long ldk, void *V, long long ldv,
                        int type, int T, const int *slots, void *stream) {
  KvArgs a{};
  int s = prepare(cache, K, ldk, V, ldv, type, T, slots, a);
  if (s != ROUGE_B200_OK) return set_status(s);
  s = device_ready();
  if (s != ROUGE_B200_OK || T == 0) return s;
  a.dst[0] = K;
  a.dst[1] = V;
  a.err = device_error_word();
  if (!a.err) return set_status(ROUGE_B200_ENOMEM);
  cudaStream_t st = as_stream(stream);
  switch (type) {
    case ROUGE_B200_T_F32: return launch_tokens(kv4_read_kernel<ROUGE_B200_T_F32>, a, T, 4, st);
    case ROUGE_B200_T_F16: return launch_tokens(kv4_read_kernel<ROUGE_B200_T_F16>, a, T, 2, st);
    default: return launch_tokens(kv4_read_kernel<ROUGE_B200_T_BF16>, a, T, 2, st);
  }
}

}  // extern "C"
