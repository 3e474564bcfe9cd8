// Attention over the paged 4-bit cache for long prompt chunks: 256 query
// rows (two tiles of 128; the group's heads times the queries) per block on
// the tcgen05 tensor cores, 128 keys at a time.
//
//   warps 0-3, 4-7  softmax of row tile 0 and 1: one thread per row. Scores
//                   of 64 keys from TMEM, running maximum and sum, weights
//                   as f16 back to TMEM (over the scores), O rescaled when
//                   the maximum has grown by more than 2^8
//   warps 8-11      one thread per key: codes from the pages to f16 K and V
//                   rows in shared memory (128-byte swizzle), one block ahead
//   warps 12, 13    issue tile 0's and 1's S = Q K^T (operands in shared
//                   memory) and O += P V (P in TMEM, V as it lies: keys x d,
//                   the N-major operand)
//
// A tile's scores are two halves of 64 keys (TMEM holds two tiles' scores and
// two O of 128 columns each): while one half is in the softmax, the tensor
// cores multiply the other half's weights by V and form its next scores. A
// half's columns hold its weights afterwards, so its next scores are issued
// when its O += P V has completed; two issuing threads, because each such
// group of MMAs takes 340 cycles to start and to be seen done, which the
// other tile's fill. (One half of 128 keys and one issuer took about 4900
// cycles per block of 128 keys; two halves take 4450.)
//
// What bounds it: 64 keys of both tiles take 2226 cycles at Dh 128, of which
// the MMAs would be 1330 by the rates of single ones (51.7 cycles at N = 64,
// 64 at N = 128) and the 16384 exponentials 1024 on 16 lanes a cycle; the rest
// are the groups' starts. 2 x 512 queries of 32 heads over up to 4096 keys: 93
// us, 553 TFLOP/s. code * scale is exact in f16; 16-bit queries are
// held as row_exponent says; weights are rounded to f16.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdint>

#include "attention_kv4.cuh"
#include "ptx.cuh"

namespace rb200 {
namespace {

constexpr int kThreads = 14 * 32;
constexpr int kKeys = 128;           // per block of K and V
constexpr int kHalf = 64;            // per step of the softmax
constexpr int kRows = 256;           // per CTA
constexpr uint32_t kChunk = 16384;   // 128 rows x 128 bytes (64 f16)
constexpr float kGrow = 8.0f;        // log2 of the growth that rescales O
constexpr float kTop = 7.0f;         // weights are held times 2^7: at most 2^15

template <int DH>
struct TileCfg {
  static constexpr int CH = DH / 64;                       // 64-value chunks of a row
  static constexpr uint32_t TILE = CH * kChunk;            // one tile of Q, K or V
  static constexpr uint32_t SMEM = 1024 + 6 * TILE + 256;  // Q x 2, K x 2, V x 2, barriers
  static constexpr uint32_t O_COL = 256;                   // TMEM: S0 0, S1 128, O0 256, O1
  static constexpr uint32_t COLS = 512;
};

// 8 codes (one 32-bit word) times a scale pair as one 16-byte unit of f16.
__device__ __forceinline__ uint4 decode8(uint32_t w, uint32_t scale2) {
  uint32_t h[4];
  e2m1x8_f16x2(w, h);
  return make_uint4(mul_f16x2(h[0], scale2), mul_f16x2(h[1], scale2), mul_f16x2(h[2], scale2),
                    mul_f16x2(h[3], scale2));
}

// Byte offset of 16-byte unit u (8 values) of row r in a swizzled tile.
__device__ __forceinline__ uint32_t unit_at(int r, int u) {
  return (u >> 3) * kChunk + r * 128 + (((u & 7) ^ (r & 7)) << 4);
}

template <int DH>
struct KeyRow {  // one key's codes and scales of K or V
  uint4 c[DH / 32];
  uint32_t s[DH / 64];  // four scales each
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < DH / 32; ++i) c[i] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int i = 0; i < DH / 64; ++i) s[i] = 0u;
  }
  __device__ __forceinline__ void load(const uint8_t *codes, const uint8_t *scales, size_t row) {
    const uint4 *p = reinterpret_cast<const uint4 *>(codes + row * (DH / 2));
#pragma unroll
    for (int i = 0; i < DH / 32; ++i) c[i] = __ldg(p + i);
    const uint32_t *q = reinterpret_cast<const uint32_t *>(scales + row * (DH / 16));
#pragma unroll
    for (int i = 0; i < DH / 64; ++i) s[i] = __ldg(q + i);
  }
  __device__ __forceinline__ void write(uint32_t tile, int r) const {
#pragma unroll
    for (int b = 0; b < DH / 16; ++b) {
      const uint32_t h = e4m3x2_f16x2((s[b / 4] >> (8 * (b & 3))) & 0xFFu);
      const uint32_t s2 = __byte_perm(h, h, 0x1010);
      const uint4 v = c[b / 2];
      const uint32_t w0 = (b & 1) ? v.z : v.x, w1 = (b & 1) ? v.w : v.y;
      const uint4 x = decode8(w0, s2), y = decode8(w1, s2);
      st_shared_v4(tile + unit_at(r, 2 * b), x.x, x.y, x.z, x.w);
      st_shared_v4(tile + unit_at(r, 2 * b + 1), y.x, y.y, y.z, y.w);
    }
  }
};

template <int DH, int T>
__global__ void __launch_bounds__(kThreads, 1) attention_kv4_tiles_kernel(const AttnArgs a, int pairs) {
  using C = TileCfg<DH>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~static_cast<uintptr_t>(1023));
  const uint32_t q_s = smem_u32(smem), k_s = q_s + 2 * C::TILE, v_s = k_s + 2 * C::TILE;
  uint64_t *bar = reinterpret_cast<uint64_t *>(smem + 6 * C::TILE);
  // [tile]; [stage]; [tile][half]
  uint64_t *q_full = bar, *k_full = bar + 2, *v_full = bar + 4, *k_empty = bar + 6, *v_empty = bar + 8,
           *s_full = bar + 10, *p_full = bar + 14, *pv_done = bar + 18, *drain = bar + 22;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bar + 24);
  volatile int *abort = reinterpret_cast<volatile int *>(bar + 25);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // unit: the last row tiles, which see the most keys, first
  const int per_seq = pairs * a.Hkv;
  const int b = blockIdx.x / per_seq, rem = blockIdx.x - b * per_seq;
  const int pair = pairs - 1 - rem / a.Hkv, hk = rem % a.Hkv;
  const SeqQueries sq = seq_queries(a, b);
  const int q0 = sq.q0, n_all = sq.all, nrows = sq.n * a.group;
  const int r0 = pair * kRows;
  if (r0 >= nrows) return;
  const int len_all = max(0, __ldg(a.kv_len + b)), p0 = len_all - n_all, len = min(len_all, a.max_kv);
  if (len_all > a.max_kv && threadIdx.x == 0) atomicCAS(a.err, 0, ROUGE_B200_EINVAL);
  const int r1 = min(r0 + kRows, nrows) - 1;
  const int hi_max = a.causal ? max(0, min(len, p0 + r1 / a.group + 1)) : len;
  const int lo_min = a.window > 0 ? window_start(p0 + r0 / a.group, a.window) : 0;
  const int first = lo_min / kKeys * kKeys;
  const int steps = hi_max > first ? (hi_max - first + kHalf - 1) / kHalf : 0;
  const int blocks = (steps + 1) / 2;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 128);
      mbar_init(&k_full[i], 128);
      mbar_init(&v_full[i], 128);
      mbar_init(&k_empty[i], 2);  // (one commit of each tile's issuer)
      mbar_init(&v_empty[i], 2);
      mbar_init(&drain[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&pv_done[i], 1);
    }
    *abort = 0;
    mbar_init_fence();
  }
  if (warp == 12) {
    tmem_alloc(tmem_slot, C::COLS);
    tmem_relinquish();
  }
  // whether the table names a page outside the cache among those with keys
  // some row sees (their keys are masked; an error, so the masks are only
  // worked out where there is one)
  const int *table = a.page_table + static_cast<size_t>(b) * a.max_pages;
  auto page_ok = [&](int pi) {
    const int id = __ldg(table + pi);
    return id >= 0 && id < a.pages;
  };
  int bad = 0;
  if (steps > 0)  // (hi_max <= max_kv: every such page is in the table)
    for (int pi = lo_min / a.page + threadIdx.x; pi <= (hi_max - 1) / a.page; pi += kThreads)
      bad |= !page_ok(pi);
  tc_fence_before_sync();
  const bool holes = __syncthreads_or(bad);
  tc_fence_after_sync();
  if (holes && threadIdx.x == 0) atomicCAS(a.err, 0, ROUGE_B200_EINVAL);
  const uint32_t tmem = *tmem_slot;
  auto fail = [&]() {
    *abort = 1;
    atomicCAS(a.err, 0, ROUGE_B200_ETIMEOUT);
  };

  if (warp < 8) {
    // ------------------------------------------------------------ softmax
    const int w = warp >> 2, tr = threadIdx.x & 127;  // tile, row in it
    const int r = r0 + w * 128 + tr;
    const bool live = r < nrows;
    const int qi = q0 + (live ? r / a.group : 0), head = hk * a.group + (live ? r % a.group : 0);
    const long long at = (static_cast<long long>(qi) * a.Hq + head) * DH;
    const int pos = p0 + r / a.group;
    const int col_hi = live ? (a.causal ? min(len, pos + 1) : len) : 0x7fffffff;
    const int col_lo = live && a.window > 0 ? window_start(pos, a.window) : 0;
    float mult;
    {  // the query row, scaled by a power of two, as f16 into the tile
      float m = 0.0f, v[16];
      if (live) {
#pragma unroll
        for (int k = 0; k < DH / 16; ++k) {
          load_q16<T>(a.Q, at + 16 * k, v);
#pragma unroll
          for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(v[i]));
        }
      }
      const RowExponent re = row_exponent<T>(m);
      mult = row_factor(re, a.scale, a.gs_k ? __ldg(a.gs_k + hk) : 1.0f);
#pragma unroll
      for (int k = 0; k < DH / 16; ++k) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = 0.0f;
        if (live) load_q16<T>(a.Q, at + 16 * k, v);
        uint32_t h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          h[i] = f16x2_rn(v[2 * i] * re.down * re.down2, v[2 * i + 1] * re.down * re.down2);
        st_shared_v4(q_s + w * C::TILE + unit_at(tr, 2 * k), h[0], h[1], h[2], h[3]);
        st_shared_v4(q_s + w * C::TILE + unit_at(tr, 2 * k + 1), h[4], h[5], h[6], h[7]);
      }
      fence_async_smem();
      mbar_arrive(&q_full[w]);
    }
    const uint32_t row_lane = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_t = tmem + w * 128 + row_lane, o_t = tmem + C::O_COL + w * DH + row_lane;
    float top = -INFINITY, sum = 0.0f;
    bool ok = true;
    for (int i = 0; i < steps; ++i) {
      const int h = i & 1, j = i >> 1;
      const uint32_t s_h = s_t + kHalf * h;
      ok = __all_sync(0xffffffffu, mbar_wait(&s_full[2 * w + h], j & 1, abort));
      if (!ok) break;
      tc_fence_after_sync();
      uint32_t x[2][32];  // the row's scores
      tmem_ld_32x32b_x32(s_h, x[0]);
      tmem_ld_32x32b_x32(s_h + 32, x[1]);
      const int key0 = first + i * kHalf;
      const bool whole = __all_sync(0xffffffffu, key0 >= col_lo && key0 + kHalf <= col_hi);
      tmem_ld_wait_regs(x[0]);
      tmem_ld_wait_regs(x[1]);
      if (!whole) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            const int key = key0 + 32 * c + k;
            if (key < col_lo || key >= col_hi) x[c][k] = 0xFF800000u;  // -inf
          }
      }
      if (holes) {  // (a page holds whole groups of 16 keys)
        const int key = key0 + 16 * (lane & 3);
        const unsigned there =
            __ballot_sync(0xffffffffu, key >= hi_max || key + 16 <= lo_min || page_ok(key / a.page));
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (!((there >> (2 * c + k / 16)) & 1u)) x[c][k] = 0xFF800000u;
      }
      float mm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int k = 0; k < 32; k += 2)
          mm[(k >> 1) & 3] = max3(mm[(k >> 1) & 3], __uint_as_float(x[c][k]), __uint_as_float(x[c][k + 1]));
      const float logit = fmaxf(fmaxf(mm[0], mm[1]), fmaxf(mm[2], mm[3])) * mult;
      const bool grow = logit > top + kGrow;  // (the first keys of a row always)
      if (__any_sync(0xffffffffu, grow)) {
        const float f = grow ? ex2(top - logit) : 1.0f;
        if (grow) top = logit;
        sum *= f;
        if (i > 0) {  // the last O += P V done, then O times f
          ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[2 * w + (h ^ 1)], ((i - 1) >> 1) & 1, abort));
          if (!ok) break;
          tc_fence_after_sync();
#pragma unroll 1
          for (int c = 0; c < DH / 16; ++c) {
            uint32_t y[16];
            tmem_ld_32x32b_x16(o_t + 16 * c, y);
            tmem_ld_wait_regs16(y);
#pragma unroll
            for (int k = 0; k < 16; ++k) y[k] = __float_as_uint(__uint_as_float(y[k]) * f);
            tmem_st_32x32b_x16(o_t + 16 * c, y);
          }
        }
      }
      const float off = top == -INFINITY ? 0.0f : kTop - top;
      float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t p[16];
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          float u0, u1;
          fma2(u0, u1, __uint_as_float(x[c][k]), __uint_as_float(x[c][k + 1]), mult, off, off);
          u0 = ex2(u0);
          u1 = ex2(u1);
          part[(k >> 1) & 3] += u0 + u1;
          p[k / 2] = f16x2_rn(u0, u1);
        }
        tmem_st_32x32b_x16(s_h + 16 * c, p);  // (over the scores, which are in registers)
      }
      sum += (part[0] + part[1]) + (part[2] + part[3]);
      tmem_st_wait();
      tc_fence_before_sync();
      mbar_arrive(&p_full[2 * w + h]);
    }
    if (ok && steps > 0) {
      ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[2 * w + ((steps - 1) & 1)],
                                             ((steps - 1) >> 1) & 1, abort));
      tc_fence_after_sync();
    }
    if (!ok && lane == 0) fail();
    if (ok) {
      const float gv = a.gs_v ? __ldg(a.gs_v + hk) : 1.0f;
      const float f = sum > 0.0f || sum != sum ? gv / sum : 0.0f;
#pragma unroll 1
      for (int c = 0; c < DH / 32; ++c) {
        uint32_t y[32];
        if (steps > 0) {
          tmem_ld_32x32b_x32(o_t + 32 * c, y);
          tmem_ld_wait_regs(y);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) y[i] = 0u;
        }
        if (live) {  // (the whole warp loads TMEM in the next round)
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)  // (a row without keys: O may hold anything times zero)
              v[k] = f == 0.0f ? 0.0f : __uint_as_float(y[i + k]) * f;
            store_o4<T>(a.O, at + 32 * c + i, v[0], v[1], v[2], v[3]);
          }
        }
        __syncwarp();
      }
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------ K and V rows
    const int kr = threadIdx.x - 256;
    KeyRow<DH> k, v;
    auto fetch = [&](int j) {
      k.zero();
      v.zero();
      const int key = first + j * kKeys + kr;
      if (j >= blocks || key >= hi_max || key < lo_min) return;  // (a key of no row: zeros)
      const int pi = key / a.page;
      const int id = __ldg(table + pi);
      if (id < 0 || id >= a.pages) return;  // (masked)
      const size_t row = (static_cast<size_t>(id) * a.Hkv + hk) * a.page + (key - pi * a.page);
      k.load(a.k_codes, a.k_scales, row);
      v.load(a.v_codes, a.v_scales, row);
    };
    fetch(0);
    for (int j = 0; j < blocks; ++j) {
      const int s = j & 1;
      const uint32_t free = ((j >> 1) & 1) ^ 1u;
      if (!__all_sync(0xffffffffu, mbar_wait(&k_empty[s], free, abort))) {
        if (lane == 0) fail();
        break;
      }
      k.write(k_s + s * C::TILE, kr);
      fence_async_smem();
      mbar_arrive(&k_full[s]);
      if (!__all_sync(0xffffffffu, mbar_wait(&v_empty[s], free, abort))) {
        if (lane == 0) fail();
        break;
      }
      v.write(v_s + s * C::TILE, kr);
      fence_async_smem();
      mbar_arrive(&v_full[s]);
      fetch(j + 1);
    }
  } else if (lane == 0 && steps > 0) {
    // ------------------------------------------------------------ MMA issuers
    const int w = warp - 12;
    const uint32_t id_s = make_idesc(1u, 0u, 0u, 0u, 0u, 128, kHalf);
    const uint32_t id_o = make_idesc(1u, 0u, 0u, 0u, 1u, 128, DH);
    bool issued = false;
    auto scores = [&](int i) {  // S of step i: Q_w K^T for its 64 keys
      const int h = i & 1, s = (i >> 1) & 1;
#pragma unroll
      for (int k = 0; k < DH / 16; ++k) {
        const uint32_t step = (k >> 2) * kChunk + (k & 3) * 32;
        umma<MmaKind::F16>(tmem + w * 128 + kHalf * h, smem_desc_sw128(q_s + w * C::TILE + step, 16, 1024),
                           smem_desc_sw128(k_s + s * C::TILE + step + h * kHalf * 128, 16, 1024), id_s,
                           k != 0);
      }
      tc_commit(&s_full[2 * w + h]);
      if (h == 1 || i == steps - 1) tc_commit(&k_empty[s]);  // the block's last scores
      issued = true;
    };
    auto run = [&]() {
      if (!mbar_wait(&q_full[w], 0, abort) || !mbar_wait(&k_full[0], 0, abort)) return false;
      tc_fence_after_sync();
      scores(0);
      if (steps > 1) scores(1);
      for (int i = 0; i < steps; ++i) {
        const int h = i & 1, j = i >> 1, s = j & 1;
        if (!mbar_wait(&p_full[2 * w + h], j & 1, abort)) return false;
        if (h == 0 && !mbar_wait(&v_full[s], (j >> 1) & 1, abort)) return false;
        tc_fence_after_sync();
#pragma unroll
        for (int k = 0; k < kHalf / 16; ++k)
          umma_f16_ta(tmem + C::O_COL + w * DH, tmem + w * 128 + kHalf * h + 8 * k,
                      smem_desc_sw128(v_s + s * C::TILE + (h * kHalf + k * 16) * 128, kChunk, 1024), id_o,
                      (i | k) != 0);
        tc_commit(&pv_done[2 * w + h]);
        if (h == 1 || i == steps - 1) tc_commit(&v_empty[s]);  // the block's last use
        if (i + 2 < steps) {
          if (h == 0 && !mbar_wait(&k_full[(j + 1) & 1], ((j + 1) >> 1) & 1, abort)) return false;
          if (!mbar_wait(&pv_done[2 * w + h], j & 1, abort)) return false;
          tc_fence_after_sync();
          scores(i + 2);
        }
      }
      return true;
    };
    if (!run()) {
      fail();
      if (issued) {  // the MMAs already issued complete before TMEM is released
        const volatile int never = 0;
        tc_commit(&drain[w]);
        mbar_wait(&drain[w], 0, &never);
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, C::COLS);
  }
}

template <int DH, int T>
int launch_tiles(const AttnArgs &a, int pairs, cudaStream_t st) {
  using C = TileCfg<DH>;
  static_assert(C::SMEM <= 232448, "exceeds the 227 KB per-CTA shared memory limit");
  auto kern = attention_kv4_tiles_kernel<DH, T>;
  static std::atomic<unsigned long long> attr_done{0};
  const unsigned long long bit = 1ull << (current_device() & 63);
  if (!(attr_done.load() & bit)) {
    const int s = cuda_status(
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    if (s != ROUGE_B200_OK) return s;
    attr_done.fetch_or(bit);
  }
  kern<<<static_cast<unsigned>(pairs) * a.Hkv * a.B, kThreads, C::SMEM, st>>>(a, pairs);
  return cuda_status(cudaGetLastError());
}

}  // namespace

// From 24 tiles of 256 rows on the tensor cores win. Tiles against warps, Dh
// 128, Hq 32, Hkv 8, 2000 keys: 6400 rows (200 queries) 54.5 and 52.7 us, 8192
// rows 54 and 62, 25600 rows 55 and 125. 16 sequences of 16 queries: 46.3 and
// 50.6. Fewer than 64 rows per unit would leave most of a tile empty. The
// choice is made for the whole call, from max_q: a block walks all keys of its
// rows, so sequences with few queries and long pasts in one call with a long
// chunk are slow here (one query over 131072 keys 2.4 ms, 62 us by the warps;
// 63 decoding sequences of 4096 keys beside a chunk of 512 364 us, 81 and 93 in
// two calls), as is a chunk over so long a past (512 queries, 131072 keys 2.4 ms).
bool kv4_tiles_apply(const AttnArgs &a, int type) {
  const double rows = static_cast<double>(a.max_q) * a.group;
  const double ctas = std::ceil(rows / kRows) * a.Hkv * a.B;
  return type != ROUGE_B200_T_F32 && (a.Dh == 64 || a.Dh == 128) && rows >= 64 &&
         rows * a.Hkv * a.B >= 24.0 * kRows && ctas < 2147483648.0;
}

int launch_attention_kv4_tiles(const AttnArgs &a, int type, cudaStream_t st) {
  const int pairs = (a.max_q * a.group + kRows - 1) / kRows;
  if (a.Dh == 64)
    return type == ROUGE_B200_T_F16 ? launch_tiles<64, ROUGE_B200_T_F16>(a, pairs, st)
                                    : launch_tiles<64, ROUGE_B200_T_BF16>(a, pairs, st);
  return type == ROUGE_B200_T_F16 ? launch_tiles<128, ROUGE_B200_T_F16>(a, pairs, st)
                                  : launch_tiles<128, ROUGE_B200_T_BF16>(a, pairs, st);
}

}  // namespace rb200
