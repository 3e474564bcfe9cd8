// What the kernels of the attention over the 4-bit cache share: their
// arguments, query loads, output stores.
#pragma once

#include <cuda_fp16.h>

#include <cstdint>

#include "kv4.cuh"
#include "x86fp.cuh"

namespace rb200 {

struct AttnArgs {
  const uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
  const float *gs_k, *gs_v;
  int pages, page, Hkv, Dh;
  const void *Q;
  void *O;
  int B, Hq, group;
  const int *cu_q;
  int max_q;
  const int *kv_len;
  const int *page_table;
  int max_pages, max_kv;  // max_kv = max_pages * page
  float scale;
  int causal, window;
  Divisor by_group, by_page, by_heads, by_tiles;  // (by_tiles: row tiles per sequence at most)
  int warps;      // warps of the grid
  int sms;
  float *part;    // [2 * warps][rows * (Dh + 4)]: weighted sums, then maximum and sum per row
  int4 *joins;    // units that several warps share (see attention_kv4.cu)
  int by_unit;    // joins is indexed by unit, not by warp
  int row_tiles;  // row tiles of a sequence of max_q queries
  int *err;
};

// Long prompt chunks on the tensor cores (attention_kv4_tiles.cu): whether
// that kernel takes the call, and its launch.
bool kv4_tiles_apply(const AttnArgs &a, int type);
int launch_attention_kv4_tiles(const AttnArgs &a, int type, cudaStream_t st);

namespace {

// The queries of sequence b: first row, their number (all of them, and those
// that are computed). More than max_q, or offsets that fall or start below
// zero, are reported.
struct SeqQueries {
  int q0, all, n;
};
__device__ __forceinline__ SeqQueries seq_queries(const AttnArgs &a, int b) {
  SeqQueries q{b, 1, 1};
  if (a.cu_q) {
    q.q0 = __ldg(a.cu_q + b);
    const int end = __ldg(a.cu_q + b + 1);
    const bool falls = q.q0 < 0 || end < q.q0;
    q.all = falls ? 0 : end - q.q0;
    q.n = min(q.all, a.max_q);
    if (falls || q.all > a.max_q) atomicCAS(a.err, 0, ROUGE_B200_EINVAL);
  }
  return q;
}

// First key a query at position p may see through the window.
__device__ __forceinline__ int window_start(int p, int window) {
  return p < window ? 0 : p - window + 1;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// The power of two that takes a row of queries, whose largest magnitude is m,
// to the top of f16's range before it is rounded, 2^(kTop - 1) <= largest <
// 2^kTop, and its factors; the scores are multiplied by 2^e afterwards. 16-bit
// rows have kTop = 16: f16 values are held exactly, bf16 ones down to 2^-32 of
// the row's largest, below which they are off by at most 2^-40 of it. f32 rows
// have kTop = 15 (their high part is rounded, maybe up) and two parts, high and
// the rest times 2^11, which hold a value to 2^-23 of itself down to 2^-27 of
// the row's largest, and to 2^-50 of the largest below that.
struct RowExponent {
  int e;
  float down, down2;
};
constexpr float kSplitScale = 2048.0f;
template <int T>
__device__ __forceinline__ RowExponent row_exponent(float m) {
  constexpr int kTop = T == ROUGE_B200_T_F32 ? 15 : 16;
  RowExponent r;
  r.e = static_cast<int>(__float_as_uint(m) >> 23) - 127;
  if (r.e == 128) r.e = kTop - 1;   // (infinity or NaN: as it is)
  r.e = r.e < -100 ? -100 : r.e;    // (tiny rows stay tiny)
  r.e -= kTop - 1;
  r.down = pow2(-(r.e / 2));
  r.down2 = pow2(-(r.e - r.e / 2));
  return r;
}
// Factor of a row's raw scores to base-2 logits; kept positive, since a
// masked score is -inf before it is scaled.
__device__ __forceinline__ float row_factor(const RowExponent &r, float scale, float gk) {
  return fmaxf(scale * 1.44269504f * gk * pow2(r.e / 2) * pow2(r.e - r.e / 2), 1e-37f);
}

// 16 consecutive query values (16-byte aligned) as they lie in memory.
template <int T>
struct RawQ {
  static constexpr int VECS = T == ROUGE_B200_T_F32 ? 4 : 2;
  uint4 q[VECS];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < VECS; ++i) q[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void load(const void *p, long long at) {
    const uint4 *s = reinterpret_cast<const uint4 *>(static_cast<const char *>(p) +
                                                     at * (T == ROUGE_B200_T_F32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < VECS; ++i) q[i] = __ldg(s + i);
  }
  __device__ __forceinline__ void unpack(float *v) const {
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const uint32_t u[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (T == ROUGE_B200_T_F32) {
          v[4 * i + j] = __uint_as_float(u[j]);
        } else if constexpr (T == ROUGE_B200_T_F16) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[j]));
          v[8 * i + 2 * j] = f.x; v[8 * i + 2 * j + 1] = f.y;
        } else {
          v[8 * i + 2 * j] = __uint_as_float(u[j] << 16);
          v[8 * i + 2 * j + 1] = __uint_as_float(u[j] & 0xFFFF0000u);
        }
      }
    }
  }
};
template <int T>
__device__ __forceinline__ void load_q16(const void *p, long long at, float *v) {
  RawQ<T> r;
  r.load(p, at);
  r.unpack(v);
}

// Four consecutive output values (aligned to four).
template <int T>
__device__ __forceinline__ void store_o4(void *o, long long at, float x, float y, float z, float w) {
  if constexpr (T == ROUGE_B200_T_F32)
    *reinterpret_cast<float4 *>(static_cast<float *>(o) + at) = make_float4(x, y, z, w);
  else if constexpr (T == ROUGE_B200_T_F16)
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(o) + at) =
        make_uint2(f16x2_rn(x, y), f16x2_rn(z, w));
  else
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(o) + at) =
        make_uint2(bf16x2_rn(x, y), bf16x2_rn(z, w));
}

}  // namespace
}  // namespace rb200
