// The paged 4-bit key / value cache (RougeB200KV4): argument checks and the
// conversions its kernels share.
#pragma once

#include <cuda_fp16.h>

#include <cstdint>

#include "runtime.cuh"

namespace rb200 {

// A cache the kernels can read: sizes, alignment, 31-bit slots.
inline int check_kv4(const RougeB200KV4 *c) {
  if (!c || !c->k_codes || !c->k_scales || !c->v_codes || !c->v_scales || c->pages <= 0 ||
      c->page <= 0 || c->Hkv <= 0 || c->Dh <= 0)
    return ROUGE_B200_EINVAL;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(c->k_codes) | reinterpret_cast<uintptr_t>(c->k_scales) |
                         reinterpret_cast<uintptr_t>(c->v_codes) | reinterpret_cast<uintptr_t>(c->v_scales);
  const uintptr_t gbits = reinterpret_cast<uintptr_t>(c->gs_k) | reinterpret_cast<uintptr_t>(c->gs_v);
  if (c->page % 16 || c->Dh % 16 || c->Dh > 256 || (bits & 15u) || (gbits & 3u) ||
      static_cast<long long>(c->pages) * c->page > 0x7fffffffLL)
    return ROUGE_B200_EUNSUPPORTED;
  return ROUGE_B200_OK;
}

inline bool valid_float_type(int type) {
  return type == ROUGE_B200_T_F32 || type == ROUGE_B200_T_F16 || type == ROUGE_B200_T_BF16;
}

// Division of n < 2^31 by a value fixed on the host (32-bit sizes): one
// high product and a shift, with the rounded-up reciprocal
// mul = ceil(2^(32 + shift) / d), shift = ceil(log2 d) - 1, whose error
// n (mul d - 2^(32 + shift)) / (d 2^(32 + shift)) stays below 1 / d.
struct Divisor {
  unsigned d, mul, shift;
  Divisor(unsigned v = 1) : d(v), mul(0), shift(0) {
    if (v == 1) return;
    while ((2u << shift) < v) ++shift;
    mul = static_cast<unsigned>(((1ull << (32 + shift)) + v - 1) / v);
  }
  __device__ __forceinline__ unsigned div(unsigned n) const {
    return d == 1 ? n : __umulhi(n, mul) >> shift;
  }
};

// Two e4m3 codes (low byte first) as f16, exact.
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint32_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(codes)));
  return r;
}

// Four bytes of two e2m1 codes each (low nibble first) as f16, exact.
__device__ __forceinline__ void e2m1x8_f16x2(uint32_t w, uint32_t (&o)[4]) {
  asm("{\n\t.reg .b8 t0, t1, t2, t3;\n\t"
      "mov.b32 {t0, t1, t2, t3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, t0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, t1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, t2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, t3;\n\t}"
      : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3])
      : "r"(w));
}

__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

}  // namespace rb200
