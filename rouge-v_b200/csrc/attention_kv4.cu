// Attention of new tokens over the paged 4-bit cache (kv4.cuh):
//   O[i] = sum_t softmax_t(scale q_i . k_t) v_t
//
// A unit is one sequence, one K/V head and one tile of query rows (the
// group's heads times the queries, query-major). All units' keys, in tiles
// of 32, form one line of work that is cut evenly over the warps of the
// grid; a unit that several warps share is joined by a second kernel from
// their running maxima, sums and weighted sums. Sequences of any mix of
// lengths so load every SM alike, without knowing the lengths on the host.
//
// Each warp works by itself: its lane 0 copies the next key tiles' codes and
// scales into the warp's ring in shared memory (bulk copies; a tile is
// contiguous within its pages), and its lanes turn the codes straight into
// the fragments of mma.m16n8k16 -- no shared-memory pass over f16 data:
//   S^T = K Q^T   A = 16 keys x 16 d, B = 16 d x 8 rows
//   O^T = V^T P^T A = 16 d x 16 keys, B = 16 keys x 8 rows
// With the keys (or d) as M, 8 query rows fill the instruction's N, so one
// decoding step of a group of 8 heads wastes nothing, and P^T comes from
// S^T's accumulators by two 8 x 8 transposes. The order of d within K's
// fragments and of d among V's rows is free (Q and O follow it): a lane
// takes a run of Dh / 4 values of its key rows, and of Dh / 8 columns of its
// value rows, read with 8- or 16-byte loads.
//
// code * scale has 2 + 4 significand bits: exact in f16, as are 16-bit
// queries (scaled to [1, 2) by a power of two per row). f32 queries are split
// into two f16 parts held in two row tiles, whose scores add up; the weights
// are split the same way. Accumulation is f32.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdint>

#include "kv4.cuh"
#include "ptx.cuh"
#include "x86fp.cuh"

namespace rb200 {
namespace {

constexpr int kTile = 32;   // keys per tile
constexpr int kWarps = 8;   // per CTA
constexpr int kMinTiles = 2;  // tiles per warp before another warp joins

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
  int max_pages;
  float scale;
  int causal, window;
  int warps;      // warps of the grid
  float *part;    // [2 * warps][rows][Dh + 2]: weighted sums, then maximum and sum per row
  int4 *desc;     // [2 * warps]: sequence, head, row tile, valid
  int *err;
};

struct SeqInfo {
  int nq, len, q0;     // queries (at most max_q), keys, first query
  int p0;              // key position of query 0
  int tiles, rts;      // key tiles per unit, row tiles
  int lo_tile;         // first tile
  long long work;      // tiles of all units
};

// Work of sequence b for row tiles of `rows` rows.
__device__ __forceinline__ SeqInfo seq_info(const AttnArgs &a, int b, int rows) {
  SeqInfo s;
  s.q0 = a.cu_q ? __ldg(a.cu_q + b) : b;
  s.nq = a.cu_q ? __ldg(a.cu_q + b + 1) - s.q0 : 1;
  s.len = max(0, __ldg(a.kv_len + b));
  s.p0 = s.len - s.nq;
  s.nq = max(0, min(s.nq, a.max_q));
  int lo = 0;
  if (a.window > 0) lo = max(0, min(s.len, s.p0 - a.window + 1));
  s.lo_tile = lo / kTile;
  s.tiles = max(1, (s.len + kTile - 1) / kTile - s.lo_tile);
  s.rts = (s.nq * a.group + rows - 1) / rows;
  s.work = static_cast<long long>(s.tiles) * s.rts * a.Hkv;
  return s;
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

template <int T>
__device__ __forceinline__ float load_q(const void *q, long long at) {
  if constexpr (T == ROUGE_B200_T_F32) return static_cast<const float *>(q)[at];
  const uint16_t h = static_cast<const uint16_t *>(q)[at];
  if constexpr (T == ROUGE_B200_T_F16) return __half2float(__ushort_as_half(h));
  return __uint_as_float(static_cast<uint32_t>(h) << 16);
}

template <int T>
__device__ __forceinline__ void store_o(void *o, long long at, float v) {
  if constexpr (T == ROUGE_B200_T_F32)
    static_cast<float *>(o)[at] = v;
  else if constexpr (T == ROUGE_B200_T_F16)
    static_cast<uint16_t *>(o)[at] = static_cast<uint16_t>(f16x2_rn(v, 0.0f));
  else
    static_cast<uint16_t *>(o)[at] = static_cast<uint16_t>(bf16x2_rn(v, 0.0f));
}

// DT: Dh rounded up to 64, 128 or 256. NT: tiles of 8 mma columns. f32
// queries: columns 8.. hold the low parts of rows 0.., so 4 * NT rows.
template <int DT, int NT, int T>
struct Shape {
  static constexpr bool SPLIT = T == ROUGE_B200_T_F32;
  static constexpr int NR = SPLIT ? NT / 2 : NT;  // column tiles of distinct rows
  static constexpr int ROWS = 8 * NR;
  static constexpr int STAGES = DT == 256 ? 2 : 3;
  static_assert(!SPLIT || NT % 2 == 0, "two parts");
};

// Bytes of one stage: codes and scales of K and V of one tile.
__host__ __device__ __forceinline__ int stage_bytes(int Dh) { return kTile * Dh * 9 / 8; }

template <int DT, int NT, int T>
__global__ void __launch_bounds__(kWarps * 32, DT == 256 || NT > 2 ? 1 : 2)
    attention_kv4_kernel(const AttnArgs a) {
  using S = Shape<DT, NT, T>;
  constexpr int kBlk = DT / 64;      // K scale blocks per lane (a run of DT / 4 values)
  constexpr int kSteps = DT / 16;    // mma steps over d
  constexpr int kMt = DT / 16;       // O^T row tiles
  constexpr int kVw = DT / 64;       // words of V codes per lane and key (DT / 8 values)
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[kWarps][S::STAGES];
  __shared__ long long total_slot[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int gw = blockIdx.x * kWarps + warp;
  grid_launch_dependents();

  // total work
  {
    long long w = 0;
    for (int b = threadIdx.x; b < a.B; b += kWarps * 32) w += seq_info(a, b, S::ROWS).work;
#pragma unroll
    for (int o = 16; o; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    if (lane == 0) total_slot[warp] = w;
    if (lane == 0)
      for (int s = 0; s < S::STAGES; ++s) mbar_init(&full[warp][s], 1);
    mbar_init_fence();
  }
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) total += total_slot[i];
  // active warps, and this warp's range of tiles
  long long active = total / kMinTiles;
  active = active < 1 ? 1 : (active > a.warps ? a.warps : active);
  long long pos = gw < active ? total * gw / active : 0;
  const long long pos_end = gw < active ? total * (gw + 1) / active : 0;
  if (lane < 2) a.desc[2 * gw + lane] = make_int4(0, 0, 0, 0);
  __syncwarp();
  if (pos >= pos_end) return;

  // sequence that holds `pos`: warp scans of 32 sequences
  int b = 0;
  long long before = 0;  // work before sequence b
  for (int b0 = 0;; b0 += 32) {
    const long long w = b0 + lane < a.B ? seq_info(a, b0 + lane, S::ROWS).work : 0;
    long long inc = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    const unsigned past = __ballot_sync(0xffffffffu, before + inc > pos);
    if (past) {
      const int l = __ffs(past) - 1;
      b = b0 + l;
      before += __shfl_sync(0xffffffffu, inc - w, l);
      break;
    }
    before += __shfl_sync(0xffffffffu, inc, 31);
  }

  const int cb = a.Dh / 2, sbk = a.Dh / 16;  // bytes per key: codes, scales
  const int nblk = a.Dh / 16;
  const int stage_sz = stage_bytes(a.Dh);
  uint8_t *ring = smem + static_cast<size_t>(warp) * S::STAGES * stage_sz;
  const uint32_t ring_u = smem_u32(ring);
  const volatile int never = 0;
  uint32_t it = 0;  // tiles taken from the ring so far
  bool alive = true;

  SeqInfo si = seq_info(a, b, S::ROWS);
  while (alive && pos < pos_end) {
    while (pos >= before + si.work) {  // next sequence
      before += si.work;
      si = seq_info(a, ++b, S::ROWS);
    }
    // unit and its tiles [u_lo, u_hi) in this warp's range
    const long long in_seq = pos - before;
    const int unit = static_cast<int>(in_seq / si.tiles);
    const int first = static_cast<int>(in_seq - static_cast<long long>(unit) * si.tiles);
    const int hk = unit % a.Hkv, rt = unit / a.Hkv;
    const long long left = pos_end - pos;
    const int last = left < si.tiles - first ? first + static_cast<int>(left) : si.tiles;
    pos += last - first;
    const bool whole = first == 0 && last == si.tiles;

    // key range of the row tile, and of each column's row
    const int r0 = rt * S::ROWS, nrows = si.nq * a.group;
    const int r1 = min(r0 + S::ROWS, nrows) - 1;
    const int p0 = si.p0;
    const int hi_max = a.causal ? max(0, min(si.len, p0 + r1 / a.group + 1)) : si.len;
    const int lo_min = a.window > 0 ? max(0, p0 + r0 / a.group - a.window + 1) : 0;
    int col_lo[S::NR][2], col_hi[S::NR][2];
    int hi_min = 0x7fffffff, lo_max = 0;
#pragma unroll
    for (int j = 0; j < S::NR; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = r0 + j * 8 + 2 * t + e;
        const int p = p0 + r / a.group;
        col_hi[j][e] = r < nrows ? (a.causal ? min(si.len, p + 1) : si.len) : si.len;
        col_lo[j][e] = a.window > 0 && r < nrows ? max(0, p - a.window + 1) : 0;
      }
    hi_min = a.causal ? min(si.len, p0 + r0 / a.group + 1) : si.len;
    lo_max = a.window > 0 ? max(0, p0 + r1 / a.group - a.window + 1) : 0;
    const int t_lo = max(si.lo_tile + first, lo_min / kTile);
    const int t_hi = min(si.lo_tile + last, (hi_max + kTile - 1) / kTile);

    // ---- copies: half tiles of 16 keys, each within one page
    const int *table = a.page_table + static_cast<size_t>(b) * a.max_pages;
    auto half_page = [&](int half) {  // page of keys [16 * half, +16), -1 if none
      const int key = half * 16;
      if (key >= hi_max || key + 16 <= lo_min) return -1;  // (no row's keys)
      const int pi = key / a.page;
      const int id = pi < a.max_pages ? __ldg(table + pi) : -1;
      if (id < 0 || id >= a.pages) {
        atomicCAS(a.err, 0, ROUGE_B200_EINVAL);
        return -1;
      }
      return id;
    };
    int ids = -1, ids_base = -1;  // lane l: page of half tile ids_base + l
    unsigned ok_bits = 0;          // two bits per stage: the halves copied
    auto issue = [&](int tile, uint32_t n) {  // tile into ring slot n % STAGES
      const int h0 = 2 * tile;
      if (ids_base < 0 || h0 >= ids_base + 32) {
        ids_base = h0;
        ids = half_page(h0 + lane);
      }
      const int id0 = __shfl_sync(0xffffffffu, ids, h0 - ids_base);
      const int id1 = __shfl_sync(0xffffffffu, ids, h0 - ids_base + 1);
      const int s = n % S::STAGES;
      const unsigned bits = (id0 >= 0 ? 1u : 0u) | (id1 >= 0 ? 2u : 0u);
      ok_bits = (ok_bits & ~(3u << (2 * s))) | (bits << (2 * s));
      if (lane == 0) {
        uint8_t *dst = ring + s * stage_sz;
        const int hb = 16 * (cb + sbk) * 2;  // bytes of one half
        mbar_arrive_expect_tx(&full[warp][s], static_cast<uint32_t>(hb * ((bits & 1) + (bits >> 1))));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int id = h ? id1 : id0;
          if (id < 0) continue;
          const int key = tile * kTile + h * 16;
          const size_t row = (static_cast<size_t>(id) * a.Hkv + hk) * a.page + key % a.page;
          bulk_load(dst + h * 16 * cb, a.k_codes + row * cb, 16 * cb, &full[warp][s]);
          bulk_load(dst + kTile * cb + h * 16 * cb, a.v_codes + row * cb, 16 * cb, &full[warp][s]);
          bulk_load(dst + 2 * kTile * cb + h * 16 * sbk, a.k_scales + row * sbk, 16 * sbk,
                    &full[warp][s]);
          bulk_load(dst + 2 * kTile * cb + kTile * sbk + h * 16 * sbk, a.v_scales + row * sbk,
                    16 * sbk, &full[warp][s]);
        }
      }
    };
    int ahead = t_lo;
    uint32_t n_issued = it;
    for (; ahead < t_hi && ahead < t_lo + S::STAGES - 1; ++ahead) issue(ahead, n_issued++);

    // ---- queries as B fragments, scaled to [1, 2) per row
    uint32_t qf[NT][kSteps][2];
    float mult[S::NR][2];
    {
      const float gk = a.gs_k ? __ldg(a.gs_k + hk) : 1.0f;
#pragma unroll
      for (int j = 0; j < S::NR; ++j) {
        const int r = r0 + j * 8 + g;
        const bool live = r < nrows;
        const int qi = si.q0 + (live ? r / a.group : 0), h = hk * a.group + (live ? r % a.group : 0);
        const long long at = (static_cast<long long>(qi) * a.Hq + h) * a.Dh;
        float v[DT / 4];
        float m = 0.0f;
#pragma unroll
        for (int k = 0; k < DT / 4; ++k) {
          const int d = t * (DT / 4) + k;
          v[k] = live && d < a.Dh ? load_q<T>(a.Q, at + d) : 0.0f;
          m = fmaxf(m, fabsf(v[k]));
        }
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        // exponent of the row maximum (0 for an empty or unbounded row)
        const int e = (m > 0.0f && m < INFINITY) ? ilogbf(m) : 0;
#pragma unroll
        for (int k = 0; k < DT / 4; ++k) v[k] = scalbnf(v[k], -e);
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const float x0 = v[4 * s + 2 * p], x1 = v[4 * s + 2 * p + 1];
            const uint32_t hi = f16x2_rn(x0, x1);
            qf[j][s][p] = hi;
            if constexpr (S::SPLIT) {
              const float2 b2 = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
              qf[S::NR + j][s][p] = f16x2_rn(x0 - b2.x, x1 - b2.y);
            }
          }
        const float mine = scalbnf(a.scale * 1.44269504f * gk, e);
        mult[j][0] = __shfl_sync(0xffffffffu, mine, 8 * t);
        mult[j][1] = __shfl_sync(0xffffffffu, mine, 8 * t + 4);
      }
    }

    float o[NT][kMt][4];
    float mx[S::NR][2], sum[S::NR][2];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int m = 0; m < kMt; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][m][e] = 0.0f;
#pragma unroll
    for (int j = 0; j < S::NR; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[j][e] = -INFINITY;
        sum[j][e] = 0.0f;
      }

    for (int tile = t_lo; tile < t_hi; ++tile, ++it) {
      if (ahead < t_hi) {
        issue(ahead, n_issued++);
        ++ahead;
      }
      const int s = it % S::STAGES;
      const unsigned ok = (ok_bits >> (2 * s)) & 3u;
      if (!__all_sync(0xffffffffu, mbar_wait(&full[warp][s], (it / S::STAGES) & 1u, &never))) {
        if (lane == 0) atomicCAS(a.err, 0, ROUGE_B200_ETIMEOUT);
        alive = false;
        break;
      }
      const uint32_t kc = ring_u + s * stage_sz, vc = kc + kTile * cb;
      const uint32_t ks = kc + 2 * kTile * cb, vs = ks + kTile * sbk;
      const int key0 = tile * kTile;
      const bool masked = ok != 3u || key0 + kTile > hi_min || key0 < lo_max;

      // ---- scores of 32 keys
      float sc[2][NT][4];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[kb][j][e] = 0.0f;
        const uint32_t row0 = kb * 16 + g;
#pragma unroll
        for (int blk = 0; blk < kBlk; ++blk) {
          const int gb = t * kBlk + blk;  // block of 16 values
          uint2 w0 = make_uint2(0u, 0u), w1 = w0;
          uint32_t s0 = 0, s1 = 0;
          if (gb < nblk) {
            w0 = lds64(kc + row0 * cb + gb * 8);
            w1 = lds64(kc + (row0 + 8) * cb + gb * 8);
            s0 = lds8(ks + row0 * sbk + gb);
            s1 = lds8(ks + (row0 + 8) * sbk + gb);
          }
          const uint32_t sh = e4m3x2_f16x2(s0 | (s1 << 8));
          const uint32_t sa = __byte_perm(sh, sh, 0x1010), sb = __byte_perm(sh, sh, 0x3232);
#pragma unroll
          for (int hw = 0; hw < 2; ++hw) {
            uint32_t x[4], y[4];
            e2m1x8_f16x2(hw ? w0.y : w0.x, x);
            e2m1x8_f16x2(hw ? w1.y : w1.x, y);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              x[q] = mul_f16x2(x[q], sa);
              y[q] = mul_f16x2(y[q], sb);
            }
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) {
              const int step = blk * 4 + hw * 2 + k2;
#pragma unroll
              for (int j = 0; j < NT; ++j)
                mma16816(sc[kb][j], x[2 * k2], y[2 * k2], x[2 * k2 + 1], y[2 * k2 + 1],
                         qf[j][step][0], qf[j][step][1]);
            }
          }
        }
      }

      // ---- softmax step: lane columns 2t, 2t + 1, keys g and g + 8 of each 16
      uint32_t pf[2][NT][2];
      bool grow = false;
      float nm[S::NR][2];
#pragma unroll
      for (int j = 0; j < S::NR; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float m = mx[j][e];
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              float v = sc[kb][j][2 * u + e];
              if constexpr (S::SPLIT) v += sc[kb][S::NR + j][2 * u + e];
              v *= mult[j][e];
              if (masked) {
                const int key = key0 + kb * 16 + u * 8 + g;
                if (!((ok >> kb) & 1u) || key >= col_hi[j][e] || key < col_lo[j][e]) v = -INFINITY;
              }
              sc[kb][j][2 * u + e] = v;
              m = fmaxf(m, v);
            }
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
          nm[j][e] = m;
          grow |= m > mx[j][e];
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int j = 0; j < S::NR; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float f = nm[j][e] > mx[j][e] ? ex2(mx[j][e] - nm[j][e]) : 1.0f;
            mx[j][e] = nm[j][e];
            sum[j][e] *= f;
#pragma unroll
            for (int m = 0; m < kMt; ++m) {
              o[j][m][e] *= f;
              o[j][m][2 + e] *= f;
              if constexpr (S::SPLIT) {
                o[S::NR + j][m][e] *= f;
                o[S::NR + j][m][2 + e] *= f;
              }
            }
          }
      }
#pragma unroll
      for (int j = 0; j < S::NR; ++j) {
        float p[2][4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // (weights carry a factor 2^15, which the division by their sum
          // takes out: f16 then keeps 11 bits of weights down to 2^-29)
          const float m = mx[j][e] == -INFINITY ? 0.0f : mx[j][e] - 15.0f;
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              p[kb][2 * u + e] = ex2(sc[kb][j][2 * u + e] - m);
              sum[j][e] += p[kb][2 * u + e];
            }
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t hi = f16x2_rn(p[kb][2 * u], p[kb][2 * u + 1]);
            pf[kb][j][u] = transpose8x8(hi);
            if constexpr (S::SPLIT) {
              const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
              pf[kb][S::NR + j][u] =
                  transpose8x8(f16x2_rn(p[kb][2 * u] - f.x, p[kb][2 * u + 1] - f.y));
            }
          }
      }

      // ---- weighted sums: lane keys 2t, 2t + 1, 2t + 8, 2t + 9, values d = g * DT / 8 + ...
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const uint32_t rows[4] = {kb * 16 + 2u * t, kb * 16 + 2u * t + 1, kb * 16 + 2u * t + 8,
                                  kb * 16 + 2u * t + 9};
#pragma unroll
        for (int w = 0; w < kVw; ++w) {
          const int e0 = g * (DT / 8) + 8 * w;  // first value of this word
          uint32_t c[4] = {0, 0, 0, 0}, sv[4] = {0, 0, 0, 0};
          if (e0 < a.Dh) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              c[q] = lds32(vc + rows[q] * cb + e0 / 2);
              sv[q] = lds8(vs + rows[q] * sbk + e0 / 16);
            }
            if (masked) {  // keys of no row: a zero scale, whatever the page holds
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const int key = key0 + static_cast<int>(rows[q]);
                if (!((ok >> kb) & 1u) || key >= hi_max || key < lo_min) sv[q] = 0;
              }
            }
          }
          const uint32_t s01 = e4m3x2_f16x2(sv[0] | (sv[1] << 8));
          const uint32_t s23 = e4m3x2_f16x2(sv[2] | (sv[3] << 8));
          constexpr uint32_t kLo = 0x0F0F0F0Fu;
          uint32_t ev01[4], od01[4], ev23[4], od23[4];
          e2m1x8_f16x2((c[0] & kLo) | ((c[1] << 4) & ~kLo), ev01);
          e2m1x8_f16x2(((c[0] >> 4) & kLo) | (c[1] & ~kLo), od01);
          e2m1x8_f16x2((c[2] & kLo) | ((c[3] << 4) & ~kLo), ev23);
          e2m1x8_f16x2(((c[2] >> 4) & kLo) | (c[3] & ~kLo), od23);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t a0 = mul_f16x2(ev01[q], s01), a1 = mul_f16x2(od01[q], s01);
            const uint32_t a2 = mul_f16x2(ev23[q], s23), a3 = mul_f16x2(od23[q], s23);
#pragma unroll
            for (int j = 0; j < NT; ++j)
              mma16816(o[j][4 * w + q], a0, a1, a2, a3, pf[kb][j][0], pf[kb][j][1]);
          }
        }
      }
      __syncwarp();  // every lane has read the stage before it is filled again
    }
    if (!alive) {  // the copies still under way land before the block's memory is released
      for (uint32_t n = it; n < n_issued; ++n)
        mbar_wait(&full[warp][n % S::STAGES], (n / S::STAGES) & 1u, &never);
      break;
    }

    // ---- sums over the lanes of a column, then the unit's result or its part
    const float gv = a.gs_v ? __ldg(a.gs_v + hk) : 1.0f;
    const int slot = 2 * gw + (first == 0 ? 1 : 0);
    float *part = a.part + static_cast<size_t>(slot) * S::ROWS * (a.Dh + 2);
    if (!whole && lane == 0) a.desc[slot] = make_int4(b, hk, rt, 1);
#pragma unroll
    for (int j = 0; j < S::NR; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = sum[j][e];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        const int rr = j * 8 + 2 * t + e, r = r0 + rr;
        if (r >= nrows) continue;
        const float f = whole ? (l > 0.0f || l != l ? gv / l : 0.0f) : 1.0f;
        const int qi = si.q0 + r / a.group, h = hk * a.group + r % a.group;
        const long long at = (static_cast<long long>(qi) * a.Hq + h) * a.Dh;
#pragma unroll
        for (int m = 0; m < kMt; ++m)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int d = g * (DT / 8) + 2 * m + u;
            if (d >= a.Dh) continue;
            float v = o[j][m][2 * u + e];
            if constexpr (S::SPLIT) v += o[S::NR + j][m][2 * u + e];
            if (whole)
              store_o<T>(a.O, at + d, v * f);
            else
              part[rr * a.Dh + d] = v;
          }
        if (!whole && g == 0) {
          part[S::ROWS * a.Dh + rr] = mx[j][e];
          part[S::ROWS * (a.Dh + 1) + rr] = l;
        }
      }
  }
}

// Joins the parts of a unit that several warps computed: block (w, row)
// handles the unit whose first part is slot 2w + 1; the others are the
// first slots of the warps after it. Order and so rounding are fixed.
constexpr int kJoinThreads = 256;

template <int T>
__global__ void __launch_bounds__(kJoinThreads) attention_kv4_join_kernel(const AttnArgs a, int rows) {
  __shared__ float red[kJoinThreads];
  __shared__ float acc[kJoinThreads];
  grid_dependency_wait();
  const int w0 = blockIdx.x, rr = blockIdx.y;
  const int4 u = a.desc[2 * w0 + 1];
  if (!u.w) return;
  const int q0 = a.cu_q ? a.cu_q[u.x] : u.x;
  int nq = a.cu_q ? a.cu_q[u.x + 1] - q0 : 1;
  nq = max(0, min(nq, a.max_q));
  const int r = u.z * rows + rr;
  if (r >= nq * a.group) return;
  // parts of the unit: the first slots of w0 + 1 .. that carry it
  int n = 1;
  for (;;) {
    const int i = w0 + n + static_cast<int>(threadIdx.x);
    bool same = false;
    if (i < a.warps) {
      const int4 d = a.desc[2 * i];
      same = d.w && d.x == u.x && d.y == u.y && d.z == u.z;
    }
    const int c = __syncthreads_count(same);
    n += c;
    if (c < kJoinThreads) break;
  }
  const size_t stride = static_cast<size_t>(rows) * (a.Dh + 2);
  auto part = [&](int i) { return a.part + (i == 0 ? 2 * w0 + 1 : 2 * (w0 + i)) * stride; };
  float m = -INFINITY;
  for (int i = threadIdx.x; i < n; i += kJoinThreads) m = fmaxf(m, part(i)[rows * a.Dh + rr]);
  red[threadIdx.x] = m;
  __syncthreads();
  for (int o = kJoinThreads / 2; o; o >>= 1) {
    if (threadIdx.x < o) red[threadIdx.x] = fmaxf(red[threadIdx.x], red[threadIdx.x + o]);
    __syncthreads();
  }
  m = red[0] == -INFINITY ? 0.0f : red[0];
  // kJoinThreads / lanes groups of parts, each lane of a group 4 values of d
  const int lanes = (a.Dh + 3) / 4, groups = kJoinThreads / lanes;
  const int grp = threadIdx.x / lanes, d = (threadIdx.x % lanes) * 4;
  const float gv = a.gs_v ? a.gs_v[u.y] : 1.0f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.0f;
  if (grp < groups) {
    for (int i = grp; i < n; i += groups) {
      const float *p = part(i);
      const float f = ex2(p[rows * a.Dh + rr] - m);
      const float2 x = *reinterpret_cast<const float2 *>(p + rr * a.Dh + d);
      const float2 y = *reinterpret_cast<const float2 *>(p + rr * a.Dh + d + 2);
      l += f * p[rows * (a.Dh + 1) + rr];
      v.x += f * x.x; v.y += f * x.y; v.z += f * y.x; v.w += f * y.y;
    }
  }
  const int h = u.y * a.group + r % a.group;
  const long long at = (static_cast<long long>(q0 + r / a.group) * a.Hq + h) * a.Dh;
  const float *vals[4] = {&v.x, &v.y, &v.z, &v.w};
  __syncthreads();
  red[threadIdx.x] = l;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    acc[threadIdx.x] = *vals[k];
    __syncthreads();
    if (threadIdx.x < lanes) {
      float s = 0.0f, tl = 0.0f;
      for (int q = 0; q < groups; ++q) {
        s += acc[q * lanes + threadIdx.x];
        tl += red[q * lanes + threadIdx.x];
      }
      if (d + k < a.Dh) store_o<T>(a.O, at + d + k, (tl > 0.0f || tl != tl) ? s * (gv / tl) : 0.0f);
    }
    __syncthreads();
  }
}

int rows_of(int group, int max_q, int type) {
  const long long rows = static_cast<long long>(group) * max_q;
  if (type == ROUGE_B200_T_F32) return 8;
  return rows <= 8 ? 8 : 16;
}

// Warps of the grid: two CTAs per SM (one for heads above 128), fewer where
// even the longest sequences would leave warps without kMinTiles tiles.
int grid_warps(int B, int Hkv, int group, int Dh, int max_q, long long max_kv, int type) {
  const long long rts = (static_cast<long long>(group) * max_q + rows_of(group, max_q, type) - 1) /
                        rows_of(group, max_q, type);
  const long long tiles = max_kv < kTile ? 1 : (max_kv + kTile - 1) / kTile;
  const long long cap = static_cast<long long>(current_sm_count()) * (Dh > 128 ? 1 : 2);
  // (products kept below 2^63: each factor is below 2^31)
  long long want = cap;
  const long long units = static_cast<long long>(B) * Hkv;
  if (units < cap * kWarps * kMinTiles && rts < cap * kWarps * kMinTiles) {
    const double all = static_cast<double>(units) * rts * tiles / kMinTiles / kWarps;
    if (all < static_cast<double>(cap)) want = static_cast<long long>(std::ceil(all));
  }
  return static_cast<int>(want < 1 ? 1 : want) * kWarps;
}

size_t part_bytes(int warps, int rows, int Dh) {
  return round_up(static_cast<size_t>(2) * warps * rows * (Dh + 2) * 4, 256);
}

template <int DT, int NT, int T>
int launch_shape(const AttnArgs &a, cudaStream_t st) {
  using S = Shape<DT, NT, T>;
  auto kern = attention_kv4_kernel<DT, NT, T>;
  const int smem = kWarps * S::STAGES * stage_bytes(a.Dh);
  static std::atomic<unsigned long long> attr_done{0};
  const unsigned long long bit = 1ull << (current_device() & 63);
  if (!(attr_done.load() & bit)) {
    const int s = cuda_status(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   kWarps * S::STAGES * stage_bytes(DT)));
    if (s != ROUGE_B200_OK) return s;
    attr_done.fetch_or(bit);
  }
  kern<<<a.warps / kWarps, kWarps * 32, smem, st>>>(a);
  int s = cuda_status(cudaGetLastError());
  if (s != ROUGE_B200_OK) return s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.warps, S::ROWS, 1);
  cfg.blockDim = dim3(kJoinThreads, 1, 1);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, attention_kv4_join_kernel<T>, a, static_cast<int>(S::ROWS)));
}

template <int DT>
int launch_dt(const AttnArgs &a, int type, int rows, cudaStream_t st) {
  switch (type) {
    case ROUGE_B200_T_F32: return launch_shape<DT, 2, ROUGE_B200_T_F32>(a, st);
    case ROUGE_B200_T_F16:
      return rows == 8 ? launch_shape<DT, 1, ROUGE_B200_T_F16>(a, st)
                       : launch_shape<DT, 2, ROUGE_B200_T_F16>(a, st);
    default:
      return rows == 8 ? launch_shape<DT, 1, ROUGE_B200_T_BF16>(a, st)
                       : launch_shape<DT, 2, ROUGE_B200_T_BF16>(a, st);
  }
}

}  // namespace
}  // namespace rb200

using namespace rb200;

extern "C" {

size_t rouge_b200_attention_kv4_workspace(int B, int Hq, int Hkv, int Dh, int max_q, int max_kv,
                                          int type) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || Dh <= 0 || Dh > 256 || max_q <= 0 ||
      max_kv <= 0 || !valid_float_type(type) || device_ready() != ROUGE_B200_OK)
    return 0;
  const int warps = grid_warps(B, Hkv, Hq / Hkv, Dh, max_q, max_kv, type);
  return part_bytes(warps, rows_of(Hq / Hkv, max_q, type), Dh) + static_cast<size_t>(2) * warps * 16;
}

int rouge_b200_attention_kv4(const RougeB200KV4 *cache, const void *Q, int type, int B, int Hq,
                             const int *cu_q, int max_q, const int *kv_len, const int *page_table,
                             int max_pages, void *O, float scale, int causal, int window,
                             void *workspace, size_t workspace_bytes, void *stream) {
  int s = check_kv4(cache);
  if (s != ROUGE_B200_OK) return set_status(s);
  if (!Q || !O || !kv_len || !page_table || B <= 0 || Hq <= 0 || Hq % cache->Hkv || max_q <= 0 ||
      max_pages <= 0 || window < 0 || (!cu_q && max_q != 1) || !valid_float_type(type))
    return set_status(ROUGE_B200_EINVAL);
  const long long max_kv = static_cast<long long>(max_pages) * cache->page;
  const long long rows = static_cast<long long>(Hq / cache->Hkv) * max_q;
  if (max_kv > 0x7fffffffLL || rows > 0x7fffffffLL ||
      ((reinterpret_cast<uintptr_t>(Q) | reinterpret_cast<uintptr_t>(O)) & 15u) ||
      (reinterpret_cast<uintptr_t>(workspace) & 255u))
    return set_status(ROUGE_B200_EUNSUPPORTED);
  s = device_ready();
  if (s != ROUGE_B200_OK) return s;
  AttnArgs a{};
  a.k_codes = cache->k_codes; a.k_scales = cache->k_scales;
  a.v_codes = cache->v_codes; a.v_scales = cache->v_scales;
  a.gs_k = cache->gs_k; a.gs_v = cache->gs_v;
  a.pages = cache->pages; a.page = cache->page; a.Hkv = cache->Hkv; a.Dh = cache->Dh;
  a.Q = Q; a.O = O;
  a.B = B; a.Hq = Hq; a.group = Hq / cache->Hkv;
  a.cu_q = cu_q; a.max_q = max_q;
  a.kv_len = kv_len; a.page_table = page_table; a.max_pages = max_pages;
  a.scale = scale > 0.0f ? scale : 1.0f / std::sqrt(static_cast<float>(cache->Dh));
  a.causal = causal; a.window = window;
  const int rt_rows = rows_of(a.group, max_q, type);
  a.warps = grid_warps(B, a.Hkv, a.group, a.Dh, max_q, max_kv, type);
  const size_t pb = part_bytes(a.warps, rt_rows, a.Dh);
  if (!workspace || workspace_bytes < pb + static_cast<size_t>(2) * a.warps * 16)
    return set_status(ROUGE_B200_ETOOBIG);
  a.part = static_cast<float *>(workspace);
  a.desc = reinterpret_cast<int4 *>(static_cast<uint8_t *>(workspace) + pb);
  a.err = device_error_word();
  if (!a.err) return set_status(ROUGE_B200_ENOMEM);
  cudaStream_t st = as_stream(stream);
  if (a.Dh <= 64) return launch_dt<64>(a, type, rt_rows, st);
  if (a.Dh <= 128) return launch_dt<128>(a, type, rt_rows, st);
  return launch_dt<256>(a, type, rt_rows, st);
}

}  // extern "C"
