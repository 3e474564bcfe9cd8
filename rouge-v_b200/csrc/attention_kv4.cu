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
// code * scale has 2 + 4 significand bits: exact in f16. Queries are scaled by
// a power of two per row to the top of f16's range (row_exponent says what of
// them is held). f32 queries are split into two f16 parts held in two row
// tiles, whose scores are added; the weights, times 2^15, are split the same
// way. Accumulation is f32.
//
// 64 sequences of up to 8192 keys, Hq 64, Hkv 8, Dh 128 take 98.5 us, 59 % of the
// copy rate, with about 740 instructions per 32-key tile, 16 warps per SM, 63 %
// of the issue slots and 60 % of the integer pipe used: neither memory nor issue
// is full, four warps a scheduler do not cover one another's dependent chains.
// Rows past 8 (groups of 16 heads, several queries) take NT = 2, whose 168
// registers spill at Dh 80 to 128 (164 to 296 bytes): Hq 128 139 us.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdint>

#include "attention_kv4.cuh"
#include "ptx.cuh"

namespace rb200 {
namespace {

constexpr int kTile = 32;   // keys per tile
// Warps at work: one per tile up to four per SM, then four tiles each, up to
// the whole grid. A warp's plan, queries and result cost it about as much as
// three tiles, so more of them on few tiles lose what they hide: 16384 keys of
// 8 heads take 20 us with four tiles each, 25 with two, 36 with one; 1025
// keys 10.6 us with one, 12.5 with two, 15.9 with four.
__host__ __device__ __forceinline__ long long warps_at_work(long long tiles, int sms, int warps) {
  long long w = tiles >> 2;
  if (w < 4 * sms) w = tiles < 4 * sms ? tiles : 4 * sms;
  return w < 1 ? 1 : (w > warps ? warps : w);
}

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
  const SeqQueries q = seq_queries(a, b);
  s.q0 = q.q0;
  s.nq = q.n;
  s.len = max(0, __ldg(a.kv_len + b));
  s.p0 = s.len - q.all;
  if (s.len > a.max_kv) {  // (more keys than the table has pages for)
    atomicCAS(a.err, 0, ROUGE_B200_EINVAL);
    s.len = a.max_kv;
  }
  int lo = 0;
  if (a.window > 0) lo = min(s.len, window_start(s.p0, a.window));
  s.lo_tile = lo / kTile;
  s.tiles = max(1, (s.len + kTile - 1) / kTile - s.lo_tile);
  s.rts = (s.nq * a.group + rows - 1) / rows;  // (rows is 8 or 16)
  s.work = static_cast<long long>(s.tiles) * s.rts * a.Hkv;
  return s;
}

// a / b for a >= 0, b > 0: the 32-bit division where it fits.
__device__ __forceinline__ long long divide(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<unsigned>(a) / static_cast<unsigned>(b);
  return a / b;
}

// The sequence that lane l of the warp holds.
__device__ __forceinline__ SeqInfo seq_of_lane(const SeqInfo &m, int l) {
  SeqInfo s;
  s.nq = __shfl_sync(0xffffffffu, m.nq, l);
  s.len = __shfl_sync(0xffffffffu, m.len, l);
  s.q0 = __shfl_sync(0xffffffffu, m.q0, l);
  s.p0 = __shfl_sync(0xffffffffu, m.p0, l);
  s.tiles = __shfl_sync(0xffffffffu, m.tiles, l);
  s.rts = __shfl_sync(0xffffffffu, m.rts, l);
  s.lo_tile = __shfl_sync(0xffffffffu, m.lo_tile, l);
  s.work = __shfl_sync(0xffffffffu, m.work, l);
  return s;
}

__device__ __forceinline__ long long inclusive_scan(long long v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Key (of 16) in row r of the score products' A fragments. Lane t's rows 2t,
// 2t + 1, 2t + 8 and 2t + 9 of the weights hold the keys t, 4 + (t ^ 1), and
// 8 more: the four value rows a load reads then lie in two bank halves, and
// so do the two key rows that eight lanes read together.
__device__ __forceinline__ int key_of_row(int r) {
  const int q = (r & 7) >> 1;
  return (r & 8) + ((r & 1) ? 4 + (q ^ 1) : q);
}

// Warps per block and blocks per SM: 16 warps an SM where a warp's O^T
// accumulators and queries leave it 128 registers, 12 with 168, 8 with 255.
constexpr int warps_of(int Dh, int nt) { return Dh > 128 || nt == 1 ? 8 : 12; }
constexpr int ctas_of(int Dh, int nt) { return Dh > 128 || nt == 2 ? 1 : 2; }

// DT: Dh rounded up to 64, 128 or 256. NT: tiles of 8 mma columns. f32
// queries: columns 8.. hold the low parts (times 2^11) of rows 0.., so 4 * NT rows.
template <int DT, int NT, int T>
struct Shape {
  static constexpr bool SPLIT = T == ROUGE_B200_T_F32;
  static constexpr int NR = SPLIT ? NT / 2 : NT;  // column tiles of distinct rows
  static constexpr int ROWS = 8 * NR;
  static constexpr int STAGES = DT == 256 ? 2 : 3;
  static constexpr int WARPS = warps_of(DT, NT);
  static constexpr int CTAS = ctas_of(DT, NT);
  static_assert(!SPLIT || NT % 2 == 0, "two parts");
};

// Bytes of one stage: codes and scales of K and V of one tile.
__host__ __device__ __forceinline__ int stage_bytes(int Dh) { return kTile * Dh * 9 / 8; }

// FULL: Dh == DT, every size a constant.
template <int DT, int NT, int T, bool FULL>
__global__ void __launch_bounds__(warps_of(DT, NT) * 32, ctas_of(DT, NT))
    attention_kv4_kernel(const AttnArgs a) {
  using S = Shape<DT, NT, T>;
  constexpr int kWarps = S::WARPS;
  constexpr int kBlk = DT / 64;      // K scale blocks per lane (a run of DT / 4 values)
  constexpr int kSteps = DT / 16;    // mma steps over d
  constexpr int kMt = DT / 16;       // O^T row tiles
  constexpr int kVw = DT / 64;       // words of V codes per lane and key (DT / 8 values)
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[kWarps][S::STAGES];
  __shared__ long long total_slot[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int gw = warp * gridDim.x + blockIdx.x;  // (few warps: one per SM)
  grid_launch_dependents();

  if (lane == 0) {
    for (int s = 0; s < S::STAGES; ++s) mbar_init(&full[warp][s], 1);
    mbar_init_fence();
  }
  // sequences b0 .. b0 + 31, one per lane; total work
  int b0 = 0;
  SeqInfo mine{};
  auto hold = [&](int base) {
    b0 = base;
    mine = SeqInfo{};
    if (base + lane < a.B) mine = seq_info(a, base + lane, S::ROWS);
  };
  hold(0);
  long long inc = inclusive_scan(mine.work, lane);
  long long total = __shfl_sync(0xffffffffu, inc, 31);
  if (a.B > 32) {  // (the block adds up the others)
    long long w = 0;
    for (int b = 32 + threadIdx.x; b < a.B; b += kWarps * 32) w += seq_info(a, b, S::ROWS).work;
#pragma unroll
    for (int o = 16; o; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    if (lane == 0) total_slot[warp] = w;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) total += total_slot[i];
  }
  // active warps, and this warp's range of tiles
  const long long active = warps_at_work(total, a.sms, a.warps);
  const long long share = divide(total, active), rest = total - share * active;
  long long pos = gw * share + (gw < rest ? gw : rest);
  const long long pos_end = gw < active ? pos + share + (gw < rest ? 1 : 0) : pos;
  if (!a.by_unit && lane == 0) a.joins[gw] = make_int4(0, 0, 0, 0);
  if (pos >= pos_end) return;
  __syncwarp();

  // sequence that holds `pos`
  int b = 0;
  long long before = 0;  // work before sequence b
  for (;;) {
    const unsigned past = __ballot_sync(0xffffffffu, before + inc > pos);
    if (past) {
      const int l = __ffs(past) - 1;
      b = b0 + l;
      before += __shfl_sync(0xffffffffu, inc - mine.work, l);
      break;
    }
    before += __shfl_sync(0xffffffffu, inc, 31);
    hold(b0 + 32);
    inc = inclusive_scan(mine.work, lane);
  }

  const int Dh = FULL ? DT : a.Dh;
  const int cb = Dh / 2, sbk = Dh / 16;  // bytes per key: codes, scales
  const int nblk = Dh / 16;
  const int stage_sz = stage_bytes(Dh);
  uint8_t *ring = smem + static_cast<size_t>(warp) * S::STAGES * stage_sz;
  const volatile int never = 0;
  // this lane's copies (see issue)
  const uint8_t *copy_src = (lane & 6) == 0 ? a.k_codes : (lane & 6) == 2 ? a.v_codes
                            : (lane & 6) == 4 ? a.k_scales : a.v_scales;
  const unsigned copy_bytes = 16u * ((lane & 4) ? sbk : cb);
  const int copy_dst = ((lane & 4) ? 2 * kTile * cb : 0) + ((lane & 2) ? 2 : 0) * copy_bytes +
                       (lane & 1) * copy_bytes;
  const int k_row = key_of_row(g);                                  // + 8: the lane's other row
  const int v_row[2] = {key_of_row(2 * t), key_of_row(2 * t + 1)};  // + 8: two more
  int s_in = 0, s_out = 0;   // ring slots of the next copy and the next tile
  uint32_t parity = 0;       // of s_out's barrier
  bool alive = true;

  SeqInfo si = seq_of_lane(mine, b - b0);
  while (alive && pos < pos_end) {
    while (pos >= before + si.work) {  // next sequence
      before += si.work;
      si = seq_info(a, ++b, S::ROWS);
    }
    // unit and its tiles [u_lo, u_hi) in this warp's range
    const long long in_seq = pos - before;
    const int unit = static_cast<int>(divide(in_seq, si.tiles));
    const int first = static_cast<int>(in_seq - static_cast<long long>(unit) * si.tiles);
    const int rt = a.by_heads.div(unit), hk = unit - rt * a.Hkv;
    const long long left = pos_end - pos;
    const int last = left < si.tiles - first ? first + static_cast<int>(left) : si.tiles;
    const long long unit_end = pos + (si.tiles - first);
    pos += last - first;
    const bool whole = first == 0 && last == si.tiles;

    // key range of the row tile, and of each column's row
    const int r0 = rt * S::ROWS, nrows = si.nq * a.group;
    const int r1 = min(r0 + S::ROWS, nrows) - 1;
    const int p0 = si.p0;
    auto q_of = [&](int r) { return static_cast<int>(a.by_group.div(r)); };  // query of a row
    const int hi_max = a.causal ? max(0, min(si.len, p0 + q_of(r1) + 1)) : si.len;
    const int lo_min = a.window > 0 ? window_start(p0 + q_of(r0), a.window) : 0;
    int col_lo[S::NR][2], col_hi[S::NR][2];
    int hi_min = 0x7fffffff, lo_max = 0;
#pragma unroll
    for (int j = 0; j < S::NR; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = r0 + j * 8 + 2 * t + e;
        const int p = p0 + q_of(r);
        col_hi[j][e] = r < nrows ? (a.causal ? min(si.len, p + 1) : si.len) : si.len;
        col_lo[j][e] = a.window > 0 && r < nrows ? window_start(p, a.window) : 0;
      }
    hi_min = a.causal ? min(si.len, p0 + q_of(r0) + 1) : si.len;
    lo_max = a.window > 0 ? window_start(p0 + q_of(r1), a.window) : 0;
    const int t_lo = max(si.lo_tile + first, lo_min / kTile);
    const int t_hi = min(si.lo_tile + last, (hi_max + kTile - 1) / kTile);

    // ---- this lane's part of its query rows, on its way while the copies start
    RawQ<T> raw[S::NR][kBlk];
#pragma unroll
    for (int j = 0; j < S::NR; ++j) {
      const int r = r0 + j * 8 + g, i = q_of(r);
      const long long at =
          (static_cast<long long>(si.q0 + i) * a.Hq + hk * a.group + (r - i * a.group)) * Dh;
#pragma unroll
      for (int k = 0; k < kBlk; ++k) {
        const int d = t * (DT / 4) + 16 * k;
        raw[j][k].zero();
        if (r < nrows && (FULL || d < Dh)) raw[j][k].load(a.Q, at + d);
      }
    }

    // ---- copies: half tiles of 16 keys, each within one page. Lane l of the
    // first eight copies array l / 2 (K codes, V codes, K scales, V scales),
    // half l % 2.
    const int *table = a.page_table + static_cast<size_t>(b) * a.max_pages;
    // first row / 16 of keys [16 * half, +16) in the cache's arrays (below
    // 2^32: 16 rows take at least 128 bytes of codes), or none
    constexpr unsigned kNone = 0xFFFFFFFFu;
    auto half_row = [&](int half) {
      const int key = half * 16;
      if (key >= hi_max || key + 16 <= lo_min) return kNone;  // (no row's keys)
      const int pi = a.by_page.div(key);
      const int id = pi < a.max_pages ? __ldg(table + pi) : -1;
      if (id < 0 || id >= a.pages) {
        atomicCAS(a.err, 0, ROUGE_B200_EINVAL);
        return kNone;
      }
      return (static_cast<unsigned>(id) * a.Hkv + hk) * (a.page / 16) + (key - pi * a.page) / 16;
    };
    unsigned rows16 = kNone;       // lane l: half_row(rows_base + l)
    int rows_base = -1;
    unsigned ok_bits = 0;          // two bits per stage: the halves copied
    auto issue = [&](int tile) {  // tile into ring slot s_in
      const int h0 = 2 * tile;
      if (rows_base < 0 || h0 >= rows_base + 32) {
        rows_base = h0;
        rows16 = half_row(h0 + lane);
      }
      const unsigned row = __shfl_sync(0xffffffffu, rows16, h0 - rows_base + (lane & 1));
      const unsigned bits = __ballot_sync(0xffffffffu, row != kNone) & 3u;
      const int s = s_in;
      s_in = s == S::STAGES - 1 ? 0 : s + 1;
      ok_bits = (ok_bits & ~(3u << (2 * s))) | (bits << (2 * s));
      if (lane == 0)
        mbar_arrive_expect_tx(&full[warp][s],
                              static_cast<uint32_t>(32 * (cb + sbk) * ((bits & 1) + (bits >> 1))));
      __syncwarp();
      if (lane < 8 && row != kNone)
        bulk_load(ring + s * stage_sz + copy_dst, copy_src + static_cast<size_t>(row) * copy_bytes,
                  copy_bytes, &full[warp][s]);
    };
    int ahead = t_lo;
    for (; ahead < t_hi && ahead < t_lo + S::STAGES - 1; ++ahead) issue(ahead);

    // ---- queries as B fragments, scaled per row
    uint32_t qf[NT][kSteps][2];
    float mult[S::NR][2];
    {
      const float gk = a.gs_k ? __ldg(a.gs_k + hk) : 1.0f;
#pragma unroll
      for (int j = 0; j < S::NR; ++j) {
        float v[DT / 4];
        float m = 0.0f;
#pragma unroll
        for (int k = 0; k < kBlk; ++k) raw[j][k].unpack(v + 16 * k);
#pragma unroll
        for (int k = 0; k < DT / 4; ++k) m = fmaxf(m, fabsf(v[k]));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const RowExponent re = row_exponent<T>(m);
#pragma unroll
        for (int k = 0; k < DT / 4; ++k) v[k] = v[k] * re.down * re.down2;
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const float x0 = v[4 * s + 2 * p], x1 = v[4 * s + 2 * p + 1];
            const uint32_t hi = f16x2_rn(x0, x1);
            qf[j][s][p] = hi;
            if constexpr (S::SPLIT) {
              const float2 b2 = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
              qf[S::NR + j][s][p] = f16x2_rn((x0 - b2.x) * kSplitScale, (x1 - b2.y) * kSplitScale);
            }
          }
        const float mine = row_factor(re, a.scale, gk);
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

    int tile = t_lo;
    for (; tile < t_hi; ++tile) {
      if (ahead < t_hi) issue(ahead++);
      const int s = s_out;
      const unsigned ok = (ok_bits >> (2 * s)) & 3u;
      if (!__all_sync(0xffffffffu, mbar_wait(&full[warp][s], parity, &never))) {
        if (lane == 0) atomicCAS(a.err, 0, ROUGE_B200_ETIMEOUT);
        alive = false;
        break;
      }
      s_out = s == S::STAGES - 1 ? 0 : s + 1;
      parity ^= s_out == 0 ? 1u : 0u;
      const uint8_t *kc = ring + s * stage_sz, *vc = kc + kTile * cb;
      const uint8_t *ks = kc + 2 * kTile * cb, *vs = ks + kTile * sbk;
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
        uint32_t w[2][2 * kBlk], sx[2][kBlk];  // codes and scales (f16 pairs) of rows g, g + 8
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int row = kb * 16 + u * 8 + k_row;
          const uint8_t *pc = kc + row * cb + t * (DT / 8), *ps = ks + row * sbk + t * kBlk;
          if constexpr (FULL && kBlk >= 2) {
#pragma unroll
            for (int q = 0; q < kBlk / 2; ++q) {
              const uint4 v = *reinterpret_cast<const uint4 *>(pc + 16 * q);
              w[u][4 * q] = v.x; w[u][4 * q + 1] = v.y; w[u][4 * q + 2] = v.z; w[u][4 * q + 3] = v.w;
              const uint32_t h = e4m3x2_f16x2(*reinterpret_cast<const uint16_t *>(ps + 2 * q));
              sx[u][2 * q] = __byte_perm(h, h, 0x1010);
              sx[u][2 * q + 1] = __byte_perm(h, h, 0x3232);
            }
          } else {
#pragma unroll
            for (int q = 0; q < kBlk; ++q) {
              uint2 v = make_uint2(0u, 0u);
              uint32_t h = 0;
              if (FULL || t * kBlk + q < nblk) {
                v = *reinterpret_cast<const uint2 *>(pc + 8 * q);
                h = e4m3x2_f16x2(ps[q]);
              }
              w[u][2 * q] = v.x; w[u][2 * q + 1] = v.y;
              sx[u][q] = __byte_perm(h, h, 0x1010);
            }
          }
        }
#pragma unroll
        for (int q = 0; q < 2 * kBlk; ++q) {
          uint32_t x[4], y[4];
          e2m1x8_f16x2(w[0][q], x);
          e2m1x8_f16x2(w[1][q], y);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[i] = mul_f16x2(x[i], sx[0][q / 2]);
            y[i] = mul_f16x2(y[i], sx[1][q / 2]);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
              mma16816(sc[kb][j], x[2 * i], y[2 * i], x[2 * i + 1], y[2 * i + 1],
                       qf[j][2 * q + i][0], qf[j][2 * q + i][1]);
        }
      }

      // ---- softmax step: lane columns 2t, 2t + 1, key rows g and g + 8 of each 16
      if constexpr (S::SPLIT) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int j = 0; j < S::NR; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              sc[kb][j][e] = __fmaf_rn(sc[kb][S::NR + j][e], 1.0f / kSplitScale, sc[kb][j][e]);
      }
      if (masked) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int key = key0 + kb * 16 + u * 8 + k_row;
#pragma unroll
            for (int j = 0; j < S::NR; ++j)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (!((ok >> kb) & 1u) || key >= col_hi[j][e] || key < col_lo[j][e])
                  sc[kb][j][2 * u + e] = -INFINITY;
          }
      }
      uint32_t pf[2][NT][2];
      bool grow = false;
      float nm[S::NR][2];
#pragma unroll
      for (int j = 0; j < S::NR; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float m = fmaxf(fmaxf(sc[0][j][e], sc[0][j][2 + e]), fmaxf(sc[1][j][e], sc[1][j][2 + e]));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
          nm[j][e] = m * mult[j][e];
          grow |= nm[j][e] > mx[j][e];
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int j = 0; j < S::NR; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float f = nm[j][e] > mx[j][e] ? ex2(mx[j][e] - nm[j][e]) : 1.0f;
            mx[j][e] = fmaxf(mx[j][e], nm[j][e]);
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
          const float m = mx[j][e] == -INFINITY ? 0.0f : 15.0f - mx[j][e];
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              p[kb][2 * u + e] = ex2(__fmaf_rn(sc[kb][j][2 * u + e], mult[j][e], m));
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

      // ---- weighted sums: the lane's keys of weight rows 2t, 2t + 1, 2t + 8,
      // 2t + 9, values d = g * DT / 8 + ...
      constexpr int kSb = DT == 256 ? 2 : 1;  // scale blocks of the lane's values
      uint32_t sv[2][4][kSb];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int w = 0; w < kSb; ++w)
            sv[kb][q][w] = FULL || g * (DT / 8) + 16 * w < Dh
                               ? vs[(kb * 16 + v_row[q & 1] + (q & 2) * 4) * sbk +
                                    (DT == 64 ? g / 2 : g * kSb) + w]
                               : 0u;
      if (masked) {  // keys of no row: a zero scale, whatever the page holds
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int key = key0 + kb * 16 + v_row[q & 1] + (q & 2) * 4;
            if (!((ok >> kb) & 1u) || key >= hi_max || key < lo_min) {
#pragma unroll
              for (int w = 0; w < kSb; ++w) sv[kb][q][w] = 0u;
            }
          }
      }
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        uint32_t c[4][kVw], s01 = 0, s23 = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int row = kb * 16 + v_row[q & 1] + (q & 2) * 4;
          const uint8_t *pc = vc + row * cb + g * (DT / 16);
          if constexpr (FULL && kVw == 2) {
            const uint2 v = *reinterpret_cast<const uint2 *>(pc);
            c[q][0] = v.x; c[q][1] = v.y;
          } else if constexpr (FULL && kVw == 4) {
            const uint4 v = *reinterpret_cast<const uint4 *>(pc);
            c[q][0] = v.x; c[q][1] = v.y; c[q][2] = v.z; c[q][3] = v.w;
          } else {
#pragma unroll
            for (int w = 0; w < kVw; ++w)
              c[q][w] = FULL || g * (DT / 8) + 8 * w < Dh
                            ? *reinterpret_cast<const uint32_t *>(pc + 4 * w) : 0u;
          }
        }
#pragma unroll
        for (int w = 0; w < kVw; ++w) {
          constexpr int kPer = kVw / kSb;  // words of one scale block
          if (w % kPer == 0) {
            s01 = e4m3x2_f16x2(sv[kb][0][w / kPer] | (sv[kb][1][w / kPer] << 8));
            s23 = e4m3x2_f16x2(sv[kb][2][w / kPer] | (sv[kb][3][w / kPer] << 8));
          }
          constexpr uint32_t kLo = 0x0F0F0F0Fu;
          uint32_t ev01[4], od01[4], ev23[4], od23[4];
          e2m1x8_f16x2((c[0][w] & kLo) | ((c[1][w] << 4) & ~kLo), ev01);
          e2m1x8_f16x2(((c[0][w] >> 4) & kLo) | (c[1][w] & ~kLo), od01);
          e2m1x8_f16x2((c[2][w] & kLo) | ((c[3][w] << 4) & ~kLo), ev23);
          e2m1x8_f16x2(((c[2][w] >> 4) & kLo) | (c[3][w] & ~kLo), od23);
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
      for (; tile < ahead; ++tile) {
        mbar_wait(&full[warp][s_out], parity, &never);
        s_out = s_out == S::STAGES - 1 ? 0 : s_out + 1;
        parity ^= s_out == 0 ? 1u : 0u;
      }
      break;
    }

    // ---- sums over the lanes of a column, then the unit's result or its part
    const float gv = a.gs_v ? __ldg(a.gs_v + hk) : 1.0f;
    const int slot = 2 * gw + (first == 0 ? 1 : 0);
    float *part = a.part + static_cast<size_t>(slot) * S::ROWS * (Dh + 4);
    if (first == 0 && lane == 0) {
      // how many warps share the unit: the one that holds its last tile
      const long long e = unit_end - 1, long_end = rest * (share + 1);
      const long long w1 = e < long_end ? divide(e, share + 1) : rest + divide(e - long_end, share);
      const int n = static_cast<int>(w1) - gw + 1;
      if (a.by_unit)
        a.joins[(b * a.row_tiles + rt) * a.Hkv + hk] = make_int4(b, unit, gw, n);
      else if (n > 1)
        a.joins[gw] = make_int4(b, unit, gw, n);
    }
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
        const int i = q_of(r);
        const long long at =
            (static_cast<long long>(si.q0 + i) * a.Hq + hk * a.group + (r - i * a.group)) * Dh + g * (DT / 8);
#pragma unroll
        for (int m = 0; m < kMt; m += 2) {  // values g * DT / 8 + 2m .. + 3
          if (!FULL && g * (DT / 8) + 2 * m >= Dh) continue;
          float v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            v[k] = o[j][m + k / 2][2 * (k & 1) + e];
            if constexpr (S::SPLIT) v[k] += o[S::NR + j][m + k / 2][2 * (k & 1) + e];
          }
          if (whole)
            store_o4<T>(a.O, at + 2 * m, v[0] * f, v[1] * f, v[2] * f, v[3] * f);
          else
            *reinterpret_cast<float4 *>(part + rr * Dh + g * (DT / 8) + 2 * m) =
                make_float4(v[0], v[1], v[2], v[3]);
        }
        if (!whole && g == 0) {
          part[S::ROWS * Dh + rr] = mx[j][e];
          part[S::ROWS * (Dh + 1) + rr] = l;
        }
      }
  }
}

// Joins the parts of the units that several warps computed. joins holds, per
// unit that n warps from w0 on share, {sequence, row tile and head, w0, n}:
// by unit where there are fewer units than warps (an entry is valid if the
// unit has rows), else by w0 (n = 0: none). The first part is slot 2 w0 + 1,
// the others the first slots of the warps after it. A block joins a unit's
// rows, or the y-th of gridDim.y shares of them. Order and so rounding are
// fixed.
constexpr int kJoinThreads = 256;

template <int T>
__global__ void __launch_bounds__(kJoinThreads) attention_kv4_join_kernel(const AttnArgs a, int rows) {
  __shared__ float4 acc[kJoinThreads];
  __shared__ float weight_sum[kJoinThreads];
  __shared__ float row_max[16];
  const int tid = threadIdx.x;
  int b = 0, rt = 0, hk = 0;
  if (a.by_unit) {
    const int seq_tile = a.by_heads.div(blockIdx.x);
    hk = blockIdx.x - seq_tile * a.Hkv;
    b = a.by_tiles.div(seq_tile);
    rt = seq_tile - b * a.row_tiles;
  }
  grid_dependency_wait();
  const int4 u = __ldcg(a.joins + blockIdx.x);
  // (an entry by unit may not have been written: for a unit without rows, or
  // when a wait of the first kernel ran out. No part outside the workspace is
  // read, whatever it holds.)
  if (u.z < 0 || u.w > a.warps - u.z) return;
  if (!a.by_unit) {
    if (u.w < 2) return;
    b = u.x;
    rt = a.by_heads.div(u.y);
    hk = u.y - rt * a.Hkv;
  }
  const int q0 = a.cu_q ? a.cu_q[b] : b;
  int nq = a.cu_q ? a.cu_q[b + 1] : b + 1;
  nq = q0 < 0 ? 0 : max(0, min(nq - q0, a.max_q));  // (as seq_queries)
  const int share = rows / gridDim.y, first = blockIdx.y * share;
  const int live = min(share, nq * a.group - rt * rows - first);  // this block's rows
  if (live <= 0 || u.w < 2) return;
  const int w0 = u.z, n = u.w;
  const size_t stride = static_cast<size_t>(rows) * (a.Dh + 4);
  auto part = [&](int i) { return a.part + (i == 0 ? 2 * w0 + 1 : 2 * (w0 + i)) * stride; };
  for (int r = tid >> 5; r < live; r += kJoinThreads / 32) {
    float m = -INFINITY;
    for (int i = tid & 31; i < n; i += 32) m = fmaxf(m, part(i)[rows * a.Dh + first + r]);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((tid & 31) == 0) row_max[r] = m == -INFINITY ? 0.0f : m;
  }
  __syncthreads();
  // a thread holds 4 values of d of one row, over every groups-th part
  const int lanes = a.Dh / 4, per_row = kJoinThreads / lanes;
  const int rows_at_once = live < per_row ? live : per_row, groups = per_row / rows_at_once;
  const int d = (tid % lanes) * 4, slot = tid / lanes;
  const float gv = a.gs_v ? a.gs_v[hk] : 1.0f;
  for (int r0 = 0; r0 < live; r0 += rows_at_once) {
    const int r = r0 + slot % rows_at_once, grp = slot / rows_at_once;
    const bool on = grp < groups && r < live && slot < per_row;
    const int rr = first + r;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.0f;
    if (on) {
      const float m = row_max[r];
#pragma unroll 4
      for (int i = grp; i < n; i += groups) {
        const float *p = part(i);
        const float f = ex2(p[rows * a.Dh + rr] - m);
        const float4 x = *reinterpret_cast<const float4 *>(p + rr * a.Dh + d);
        l += f * p[rows * (a.Dh + 1) + rr];
        v.x += f * x.x; v.y += f * x.y; v.z += f * x.z; v.w += f * x.w;
      }
    }
    __syncthreads();
    acc[tid] = v;
    weight_sum[tid] = l;
    __syncthreads();
    if (on && grp == 0) {
      for (int q = 1; q < groups; ++q) {
        const int o = tid + q * rows_at_once * lanes;
        v.x += acc[o].x; v.y += acc[o].y; v.z += acc[o].z; v.w += acc[o].w;
        l += weight_sum[o];
      }
      const float f = (l > 0.0f || l != l) ? gv / l : 0.0f;
      const int row = rt * rows + rr, q = a.by_group.div(row);
      const long long at =
          (static_cast<long long>(q0 + q) * a.Hq + hk * a.group + (row - q * a.group)) * a.Dh + d;
      store_o4<T>(a.O, at, v.x * f, v.y * f, v.z * f, v.w * f);
    }
  }
}

int rows_of(int group, int max_q, int type) {
  const long long rows = static_cast<long long>(group) * max_q;
  if (type == ROUGE_B200_T_F32) return 8;
  return rows <= 8 ? 8 : 16;
}

// mma column tiles per warp (see Shape).
int nt_of(int rows, int type) { return type == ROUGE_B200_T_F32 || rows == 16 ? 2 : 1; }

// Warps of the grid on `sms` SMs: all they hold, fewer where even the longest
// sequences would leave warps idle. Not fewer on more SMs.
int grid_warps(int B, int Hkv, int group, int Dh, int max_q, long long max_kv, int type, int sms) {
  const int rows = rows_of(group, max_q, type), nt = nt_of(rows, type), warps = warps_of(Dh, nt);
  const int cap = sms * ctas_of(Dh, nt) * warps;
  const double rts = std::ceil(static_cast<double>(group) * max_q / rows);
  const double tiles = max_kv < kTile ? 1.0 : std::ceil(static_cast<double>(max_kv) / kTile);
  const double all = static_cast<double>(B) * Hkv * rts * tiles;
  const long long w = all < 1e15 ? warps_at_work(static_cast<long long>(all), sms, cap) : cap;
  // (few warps go one to an SM: a block for each, as far as they reach)
  const long long ctas = w < sms ? w : (w + warps - 1) / warps < sms ? sms : (w + warps - 1) / warps;
  return static_cast<int>(ctas) * warps;
}

size_t part_bytes(int warps, int rows, int Dh) {
  return round_up(static_cast<size_t>(2) * warps * rows * (Dh + 4) * 4, 256);
}

// Workspace of a call on all of the device's SMs: a budget of fewer
// (rouge_b200_set_sm_budget) may be set or lifted between sizing and call.
size_t workspace_bytes_of(int B, int Hkv, int group, int Dh, int max_q, long long max_kv, int type) {
  const int warps = grid_warps(B, Hkv, group, Dh, max_q, max_kv, type, device_sm_count());
  return part_bytes(warps, rows_of(group, max_q, type), Dh) + static_cast<size_t>(warps) * 16;
}

template <int DT, int NT, int T, bool FULL>
int launch_kernels(const AttnArgs &a, int join_y, cudaStream_t st) {
  using S = Shape<DT, NT, T>;
  auto kern = attention_kv4_kernel<DT, NT, T, FULL>;
  const int smem = S::WARPS * S::STAGES * stage_bytes(a.Dh);
  static std::atomic<unsigned long long> attr_done{0};
  const unsigned long long bit = 1ull << (current_device() & 63);
  if (!(attr_done.load() & bit)) {
    const int s = cuda_status(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   S::WARPS * S::STAGES * stage_bytes(DT)));
    if (s != ROUGE_B200_OK) return s;
    attr_done.fetch_or(bit);
  }
  kern<<<a.warps / S::WARPS, S::WARPS * 32, smem, st>>>(a);
  int s = cuda_status(cudaGetLastError());
  if (s != ROUGE_B200_OK) return s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.by_unit ? a.B * a.Hkv * a.row_tiles : a.warps, join_y, 1);
  cfg.blockDim = dim3(kJoinThreads, 1, 1);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, attention_kv4_join_kernel<T>, a, static_cast<int>(S::ROWS)));
}

template <int DT, int NT, int T>
int launch_shape(const AttnArgs &a, cudaStream_t st) {
  // A block joins all rows of a unit, or, where a unit may be cut into more
  // than 16 parts (few units), one row.
  const double units = static_cast<double>(a.B) * a.Hkv * a.row_tiles;
  const int join_y = a.warps > 16 * units ? Shape<DT, NT, T>::ROWS : 1;
  return a.Dh == DT ? launch_kernels<DT, NT, T, true>(a, join_y, st)
                    : launch_kernels<DT, NT, T, false>(a, join_y, st);
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
  return workspace_bytes_of(B, Hkv, Hq / Hkv, Dh, max_q, max_kv, type);
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
  if (max_kv > 0x7ffffc00LL || rows > 0x7ffffc00LL ||
      ((reinterpret_cast<uintptr_t>(Q) | reinterpret_cast<uintptr_t>(O)) & 15u) ||
      ((reinterpret_cast<uintptr_t>(cu_q) | reinterpret_cast<uintptr_t>(kv_len) |
        reinterpret_cast<uintptr_t>(page_table)) & 3u) ||
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
  a.max_kv = static_cast<int>(max_kv);
  a.scale = scale > 0.0f ? scale : 1.0f / std::sqrt(static_cast<float>(cache->Dh));
  a.causal = causal;
  a.window = window;
  const int rt_rows = rows_of(a.group, max_q, type);
  a.sms = current_sm_count();
  a.warps = grid_warps(B, a.Hkv, a.group, a.Dh, max_q, max_kv, type, a.sms);
  const size_t pb = part_bytes(a.warps, rt_rows, a.Dh);
  if (!workspace || workspace_bytes < workspace_bytes_of(B, a.Hkv, a.group, a.Dh, max_q, max_kv, type))
    return set_status(ROUGE_B200_ETOOBIG);
  a.part = static_cast<float *>(workspace);
  a.joins = reinterpret_cast<int4 *>(static_cast<uint8_t *>(workspace) + pb);
  a.row_tiles = static_cast<int>((rows + rt_rows - 1) / rt_rows);
  a.by_unit = static_cast<double>(B) * a.Hkv * a.row_tiles < a.warps ? 1 : 0;
  a.by_group = Divisor(a.group);
  a.by_page = Divisor(a.page);
  a.by_heads = Divisor(a.Hkv);
  a.by_tiles = Divisor(a.row_tiles);
  a.err = device_error_word();
  if (!a.err) return set_status(ROUGE_B200_ENOMEM);
  cudaStream_t st = as_stream(stream);
  if (kv4_tiles_apply(a, type)) return launch_attention_kv4_tiles(a, type, st);
  if (a.Dh <= 64) return launch_dt<64>(a, type, rt_rows, st);
  if (a.Dh <= 128) return launch_dt<128>(a, type, rt_rows, st);
  return launch_dt<256>(a, type, rt_rows, st);
}

}  // extern "C"
