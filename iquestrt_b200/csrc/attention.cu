// Attention of a few new tokens over a paged key/value cache (iq_attn_decode).
//
// Mathematics.  For one query row with keys k_j and values v_j, x_j = scale log2(e) q.k_j:
//   M = max_j x_j,  l = sum_j 2^(x_j - M),  o = sum_j 2^(x_j - M) v_j / l,
//   lse = (M + log2 l) ln 2,
// and two partial results (M1, l1, O1), (M2, l2, O2) over disjoint keys join as
//   M = max(M1, M2),  l = l1 2^(M1-M) + l2 2^(M2-M),  O likewise.
//
// What bounds it: the cache is read once, 2 D bytes (e4m3) or 4 D (bf16) a key and key/value
// head, and all the query rows that share a key/value head (group x q_len of them) use what
// was read: HBM, until about 32 rows share a head.
//
// Split.  The keys every row of a step sees ("common" keys) are cut into tiles of TK; the
// tiles of all (sequence, head, block of query rows) units form one list that is dealt to
// the CTAs in equal contiguous shares, whatever the lengths are.  A unit that falls into
// one share is finished there; one that spans several leaves partial results that
// attn_join_kernel adds.  The at most 14 "edge" keys that only some rows of a step see (the
// step's own keys, and the rim of a sliding window) are one more tile of the unit, done in
// scalar arithmetic on exactly the visible keys: a value that a row must not see (an
// infinity or a NaN among them) never meets that row, not even multiplied by zero.
//
// Layout.  S^T = K Q^T and O^T = V^T P^T on the warp MMA (m16n8k16): the cache is the
// 16-row operand and eight query rows the columns, so a group of eight heads fills the
// tile that would otherwise be padded to sixteen rows.  A warp owns the sixteen keys it
// copied (cp.async ring, no block barrier in the loop) and all of D; warps join at the end
// of a unit.
#include <math.h>
#include <stdio.h>

#include <mutex>
#include <unordered_set>

#include <cuda_fp16.h>

#include "paged.cuh"

namespace iqb {

constexpr int kAttnMaxBatch = 1024;
constexpr int kEdgeMax = 16;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLog2e = 1.4426950408889634f;

struct AttnParams {
  const __nv_bfloat16* q;
  long long q_b, q_r, q_h;                       // strides, elements
  const uint8_t *k, *v;
  long long k_row, k_head, v_row, v_head;        // strides, bytes
  PageTable pages;
  const int* lengths;
  int max_rows;                                  // rows the page table covers
  __nv_bfloat16* out;
  long long o_b, o_r, o_h;
  float* lse;                                    // [batch, q_len, q_heads] or null
  float* part;                                   // [2 grid][RB][DP] unnormalised O
  float2* part_ml;                               // [2 grid][RB] (M, l)
  int2* units;                                   // [units] first and last CTA of a split unit
  float* scores;                                 // [batch * kv_heads][score_rows][rows_all] x_j, or null
  float* lse2;                                   // [batch, q_len, q_heads] M + log2 l (with scores)
  int score_rows;
  float* weights;
  long long w_b, w_h;
  int* positions;
  long long p_b, p_h;
  const int* seen;
  int* status;
  int batch, q_len, q_heads, kv_heads, group, dim, window;
  int rows_all;                                  // group * q_len
  int rows_pad;                                  // rows_all rounded up to eight
  int n_rb;                                      // blocks of RB rows
  float scale_log2;
};

// One sequence's keys: common [lo, hi), edges [lo0, lo) and [hi, n) (hi clamped to lo).
struct SeqSpan {
  int n, lo0, lo, hi;
};
__device__ __forceinline__ SeqSpan seq_span(int n, int q_len, int window) {
  SeqSpan s;
  s.n = n;
  const int first = n - q_len;                   // the first row's position
  s.lo0 = window ? max(0, first - window + 1) : 0;
  s.lo = window ? max(0, n - window) : 0;
  s.hi = max(first + 1, 0);
  s.hi = max(s.hi, s.lo);
  return s;
}
__device__ __forceinline__ int span_edges(const SeqSpan& s) { return s.lo - s.lo0 + s.n - s.hi; }
template <int TK>
__device__ __forceinline__ int span_tiles(const SeqSpan& s) {
  return (s.hi - s.lo + TK - 1) / TK + (span_edges(s) > 0 ? 1 : 0);
}

__device__ __forceinline__ int clamp_length(const AttnParams& p, int b, bool report) {
  const int n = __ldg(p.lengths + b);
  if (n < 0 || n > p.max_rows) {
    if (report && p.status) atomicCAS(p.status, 0, IQ_ERR_ROUTE);
    return n < 0 ? 0 : p.max_rows;
  }
  return n;
}

// floor(total c / grid), and the share that owns tile i.
__device__ __forceinline__ int share_begin(int total, int grid, int c) {
  return static_cast<int>(static_cast<long long>(total) * c / grid);
}
__device__ __forceinline__ int share_owner(int total, int grid, int i) {
  return static_cast<int>((static_cast<long long>(i + 1) * grid - 1) / total);
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(two)));
  return h;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}

// KV: IQ_ACT_E4M3 or IQ_ACT_BF16.  DP: head dim rounded up (64, 128, 256).  NBW: blocks of
// eight query rows a warp holds; WR: warps that share a key group's copies, each with its
// own rows; W warps.
template <int KV_, int DP_, int NBW_, int WR_, int W_, int CTAS_>
struct AttnGeo {
  static constexpr int KV = KV_, DP = DP_, NBW = NBW_, WR = WR_, W = W_, CTAS = CTAS_;
  static constexpr int WK = W / WR;
  static constexpr int TK = 16 * WK;             // keys a tile
  static constexpr int RB = 8 * NBW * WR;        // query rows a block
  static constexpr int THREADS = 32 * W;
  static constexpr int ELT = KV == IQ_ACT_BF16 ? 2 : 1;
  static constexpr int DPB = DP * ELT;
  static constexpr int CPR = DPB / 16;           // 16-byte pieces a row
  static constexpr int STAGE = 2 * 16 * DPB;     // one key group's keys and values
  static constexpr int MT = DP / 16;             // m-tiles of O^T
  static constexpr int NREG = MT * 4 + 4;      // one block of eight rows: O, M, l of a lane
  static constexpr int TREE = WK > 1 ? (W / 2) * 32 * NREG * 4 : 0;
  static constexpr int EDGE = RB * (DP + 2) * 4;
  static constexpr int JOIN = TREE > EDGE ? TREE : EDGE;
  static constexpr int FIXED = JOIN + kEdgeMax * 4 + (2 * kAttnMaxBatch + 64) * 4;
  static constexpr int BUDGET = (CTAS == 1 ? 227 : CTAS == 2 ? 113 : 75) * 1024;
  static constexpr int FIT = (BUDGET - FIXED) / (WK * STAGE);
  static constexpr int STAGES = FIT > 8 ? 8 : FIT;
  static constexpr int SMEM = WK * STAGES * STAGE + FIXED;
  static_assert(STAGES >= 2, "the ring needs two stages");
};

// Walks the list of tiles: the unit of the current tile and the tile's place in it.
struct TileIter {
  int b, hb, tile, tiles;
  SeqSpan s;
};

template <class G>
__device__ __forceinline__ void iter_seq(TileIter& it, const AttnParams& p, const int* prefix,
                                         const int* lens) {
  it.tiles = prefix[it.b + 1] - prefix[it.b];
  it.s = seq_span(lens[it.b], p.q_len, p.window);
}
template <class G>
__device__ __forceinline__ void iter_init(TileIter& it, const AttnParams& p, const int* prefix,
                                          const int* lens, int i) {
  const int per = p.kv_heads * p.n_rb;
  int lo = 0, hi = p.batch;                      // prefix[lo] * per <= i < prefix[hi] * per
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] * per <= i) lo = mid; else hi = mid;
  }
  it.b = lo;
  iter_seq<G>(it, p, prefix, lens);
  const int rem = i - prefix[lo] * per;
  it.hb = rem / it.tiles;
  it.tile = rem - it.hb * it.tiles;
}
template <class G>
__device__ __forceinline__ void iter_next(TileIter& it, const AttnParams& p, const int* prefix,
                                          const int* lens) {
  if (++it.tile < it.tiles) return;
  it.tile = 0;
  if (++it.hb < p.kv_heads * p.n_rb) return;
  it.hb = 0;
  do {
    ++it.b;
  } while (it.b < p.batch && prefix[it.b + 1] == prefix[it.b]);
  if (it.b < p.batch) iter_seq<G>(it, p, prefix, lens);
}

template <class G>
__global__ void __launch_bounds__(G::THREADS, G::CTAS) attn_kernel(const __grid_constant__ AttnParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem;
  float* join = reinterpret_cast<float*>(smem + G::WK * G::STAGES * G::STAGE);
  int* edge_rows = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(join) + G::JOIN);
  int* prefix = edge_rows + kEdgeMax;            // [batch + 1]
  int* lens = prefix + kAttnMaxBatch + 4;        // [batch]
  int* warp_sums = lens + kAttnMaxBatch;         // [W]

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int wr = warp % G::WR, kg = warp / G::WR;
  const int g = lane >> 2, t = lane & 3;
  const int cta = blockIdx.x;

  pdl_wait();
  pdl_launch_dependents();

  // ---- the list of tiles: exclusive prefix over the sequences
  {
    const int each = (p.batch + G::THREADS - 1) / G::THREADS;
    const int b0 = min(tid * each, p.batch), b1 = min(b0 + each, p.batch);
    int sum = 0;
    for (int b = b0; b < b1; ++b) {
      const int n = clamp_length(p, b, cta == 0);
      lens[b] = n;
      sum += span_tiles<G::TK>(seq_span(n, p.q_len, p.window));
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    int at = incl - sum;
    for (int w = 0; w < warp; ++w) at += warp_sums[w];
    for (int b = b0; b < b1; ++b) {
      prefix[b] = at;
      at += span_tiles<G::TK>(seq_span(lens[b], p.q_len, p.window));
    }
    if (tid == G::THREADS - 1) prefix[p.batch] = at;
    __syncthreads();
  }
  const int per = p.kv_heads * p.n_rb;
  const int total = prefix[p.batch] * per;
  // at least one tile for each CTA that takes part: no CTA between two that share a unit is
  // without a part of it
  const int grid = min(static_cast<int>(gridDim.x), total);

  // ---- which CTAs a unit spans; rows of empty sequences
  for (int u = cta; u < p.batch * per; u += gridDim.x) {
    const int b = u / per, hb = u - b * per;
    const int tiles = prefix[b + 1] - prefix[b];
    if (tiles > 0) {
      if (tid == 0) {
        const int first = prefix[b] * per + hb * tiles;
        p.units[u] = make_int2(share_owner(total, grid, first),
                               share_owner(total, grid, first + tiles - 1));
      }
      continue;
    }
    if (tid == 0) p.units[u] = make_int2(0, 0);
    const int h = hb / p.n_rb, r0 = (hb - h * p.n_rb) * G::RB;
    const int rows = min(G::RB, p.rows_all - r0);
    for (int i = tid; i < rows * p.dim; i += G::THREADS) {
      const int r = r0 + i / p.dim, d = i % p.dim;
      const int tok = r / p.group, head = h * p.group + r % p.group;
      p.out[b * p.o_b + tok * p.o_r + head * p.o_h + d] = __float2bfloat16_rn(0.f);
      if (d == 0) {
        const long long o = (static_cast<long long>(b) * p.q_len + tok) * p.q_heads + head;
        if (p.lse) p.lse[o] = -INFINITY;
        if (p.lse2) p.lse2[o] = -INFINITY;
      }
    }
  }

  if (cta >= grid) return;
  const int i0 = share_begin(total, grid, cta), i1 = share_begin(total, grid, cta + 1);

  // ---- copies: this warp's part of its key group's ring
  const uint32_t ring_g = smem_u32(ring) + kg * G::STAGES * G::STAGE;
  constexpr int GT = 32 * G::WR;
  const int gtid = wr * 32 + lane;
  TileIter ld;
  iter_init<G>(ld, p, prefix, lens, i0);
  auto look_up = [&]() -> int {                  // lanes 0..15: the cache row of key `lane`
    const int j = ld.s.lo + ld.tile * G::TK + kg * 16 + lane;
    if (lane >= 16 || j >= ld.s.hi) return -1;
    const int row = cache_row(p.pages, ld.b, j);
    if (row < 0 && p.status) atomicCAS(p.status, 0, IQ_ERR_ROUTE);
    return row;
  };
  int row_next = look_up();
  auto issue = [&](int stage) {
    const int h = ld.hb / p.n_rb;
    const uint32_t dst_k = ring_g + stage * G::STAGE, dst_v = dst_k + 16 * G::DPB;
#pragma unroll
    for (int i = 0; i < (16 * G::CPR + GT - 1) / GT; ++i) {
      const int idx = gtid + i * GT;
      const int r = idx / G::CPR, c = idx % G::CPR;
      const int row = __shfl_sync(0xffffffffu, row_next, r & 15);
      if (16 * G::CPR % GT == 0 || idx < 16 * G::CPR) {
        const bool ok = row >= 0 && c * 16 < p.dim * G::ELT;
        const long long rr = ok ? row : 0;
        const int cc = ok ? c * 16 : 0;
        int ck, cv;
        if (G::KV == IQ_ACT_BF16) {
          ck = cv = c ^ (r & 7);
        } else {
          ck = G::DPB >= 128 ? c ^ ((r & 1) << 2) : c;
          cv = G::DPB >= 128 ? c ^ (((r >> 1) & 3) << 1) : c ^ ((r >> 1) & 3);
        }
        cp_async16(dst_k + r * G::DPB + ck * 16, p.k + rr * p.k_row + h * p.k_head + cc, ok);
        cp_async16(dst_v + r * G::DPB + cv * 16, p.v + rr * p.v_row + h * p.v_head + cc, ok);
      }
    }
  };
  int ld_at = i0;
  auto feed = [&](int stage) {                   // the next tile's copies, and one group always
    if (ld_at < i1) {
      issue(stage);
      if (++ld_at < i1) {
        iter_next<G>(ld, p, prefix, lens);
        row_next = look_up();
      }
    }
    cp_async_commit();
  };
  auto group_sync = [&]() {
    if (G::WR == 1) __syncwarp();
    else if (G::WK == 1) __syncthreads();
    else named_bar_sync(1 + kg, GT);
  };

#pragma unroll
  for (int s = 0; s < G::STAGES - 1; ++s) feed(s);

  // ---- state of the unit being computed
  constexpr int QREG = G::DP / 8;                // packed registers of q a block of eight rows
  uint32_t qf[G::NBW][QREG];
  float xs[G::NBW][2];                           // score factor of this lane's two columns
  float m[G::NBW][2], l[G::NBW][2], acc[G::NBW][G::MT][4];
  bool have_edges = false;

  // P relative to 2^14 in half precision (e4m3 caches): the weights that a fixed-point
  // format would lose lie fourteen bits lower; bf16 has fp32's range and needs no shift.
  constexpr float kShift = G::KV == IQ_ACT_BF16 ? 0.f : 14.f;

  TileIter it;
  iter_init<G>(it, p, prefix, lens, i0);
  bool fresh = true;
  int seg_first_tile = it.tile;                  // place of the segment's first tile in its unit

  for (int i = i0; i < i1; ++i) {
    const int slot = (i - i0) % G::STAGES;
    cp_async_wait<G::STAGES - 2>();
    group_sync();
    feed((i - i0 + G::STAGES - 1) % G::STAGES);

    const int h = it.hb / p.n_rb, r0 = (it.hb - h * p.n_rb) * G::RB;
    if (fresh) {
      fresh = false;
      have_edges = false;
      seg_first_tile = it.tile;
#pragma unroll
      for (int nb = 0; nb < G::NBW; ++nb) {
        const int r = r0 + (wr * G::NBW + nb) * 8 + g;
        const bool live = r < p.rows_all;
        const int tok = live ? r / p.group : 0, head = h * p.group + (live ? r % p.group : 0);
        const __nv_bfloat16* src = p.q + it.b * p.q_b + tok * p.q_r + head * p.q_h;
        if (G::KV == IQ_ACT_BF16) {
          // fragment order of the MMA: registers 2i, 2i+1 are channels 16i + 2t, 16i + 8 + 2t
#pragma unroll
          for (int x = 0; x < QREG; ++x) {
            const int d = x * 8 + 2 * t;
            qf[nb][x] = live && d < p.dim ? *reinterpret_cast<const uint32_t*>(src + d) : 0u;
          }
          xs[nb][0] = xs[nb][1] = p.scale_log2;
        } else {
          // lane t holds channels 64 k + 16 t .. + 15; bf16 values scaled by a power of two
          // so that the row's largest lies in [1, 2): exact in half precision but for
          // values 2^-14 below the row's largest
          float big = 0.f;
#pragma unroll
          for (int x = 0; x < QREG; ++x) {
            const int d = (x / 8) * 64 + t * 16 + (x % 8) * 2;
            const uint32_t w = live && d < p.dim ? *reinterpret_cast<const uint32_t*>(src + d) : 0u;
            qf[nb][x] = w;
            big = fmaxf(big, fmaxf(fabsf(__uint_as_float(w << 16)),
                                   fabsf(__uint_as_float(w & 0xffff0000u))));
          }
          big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
          big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
          int e = static_cast<int>(__float_as_uint(big) >> 23) - 127;
          if (big == 0.f || e > 127) e = 0;
          e = max(-126, min(126, e));
          const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
          const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
          for (int x = 0; x < QREG; ++x) {
            const uint32_t w = qf[nb][x];
            qf[nb][x] = pack_f16(__uint_as_float(w << 16) * down,
                                 __uint_as_float(w & 0xffff0000u) * down);
          }
          const float f = p.scale_log2 * up;
          xs[nb][0] = __shfl_sync(0xffffffffu, f, (2 * t) * 4);
          xs[nb][1] = __shfl_sync(0xffffffffu, f, (2 * t + 1) * 4);
        }
        m[nb][0] = m[nb][1] = -INFINITY;
        l[nb][0] = l[nb][1] = 0.f;
#pragma unroll
        for (int x = 0; x < G::MT; ++x)
          acc[nb][x][0] = acc[nb][x][1] = acc[nb][x][2] = acc[nb][x][3] = 0.f;
      }
    }

    const int common = (it.s.hi - it.s.lo + G::TK - 1) / G::TK;
    const int j0 = it.s.lo + it.tile * G::TK + kg * 16;
    if (it.tile < common && j0 < it.s.hi) {
      const uint32_t sk = ring_g + slot * G::STAGE, sv = sk + 16 * G::DPB;
      float sc[G::NBW][4];
#pragma unroll
      for (int nb = 0; nb < G::NBW; ++nb) sc[nb][0] = sc[nb][1] = sc[nb][2] = sc[nb][3] = 0.f;
      if (G::KV == IQ_ACT_BF16) {
        const int r = (lane & 7) + ((lane >> 3) & 1) * 8;       // matrices: keys 0-7, 8-15
#pragma unroll
        for (int x = 0; x < G::MT; ++x) {
          uint32_t a[4];
          ldmatrix_x4(a, sk + r * G::DPB + (((2 * x + (lane >> 4)) ^ (r & 7)) * 16));
#pragma unroll
          for (int nb = 0; nb < G::NBW; ++nb)
            mma_bf16(sc[nb], a[0], a[1], a[2], a[3], qf[nb][2 * x], qf[nb][2 * x + 1]);
        }
      } else {
#pragma unroll
        for (int kk = 0; kk < G::DP / 64; ++kk) {
          const int c = G::DPB >= 128 ? (kk * 4 + t) ^ ((g & 1) << 2) : kk * 4 + t;
          const uint4 lo = lds128(sk + g * G::DPB + c * 16);
          const uint4 hi = lds128(sk + (g + 8) * G::DPB + c * 16);
          const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint32_t a0 = e4m3x2_to_f16x2(wl[x]), a2 = e4m3x2_to_f16x2(wl[x] >> 16);
            const uint32_t a1 = e4m3x2_to_f16x2(wh[x]), a3 = e4m3x2_to_f16x2(wh[x] >> 16);
#pragma unroll
            for (int nb = 0; nb < G::NBW; ++nb)
              mma_f16(sc[nb], a0, a1, a2, a3, qf[nb][kk * 8 + 2 * x], qf[nb][kk * 8 + 2 * x + 1]);
          }
        }
      }
      // ---- softmax of this lane's columns (query rows 2t, 2t+1), keys g and g + 8
      uint32_t pb[G::NBW][2];
      const bool lo_ok = j0 + g < it.s.hi, hi_ok = j0 + g + 8 < it.s.hi;
#pragma unroll
      for (int nb = 0; nb < G::NBW; ++nb) {
        float x0 = sc[nb][0] * xs[nb][0], x1 = sc[nb][1] * xs[nb][1];
        float x2 = sc[nb][2] * xs[nb][0], x3 = sc[nb][3] * xs[nb][1];
        if (p.scores) {
          const int r = r0 + (wr * G::NBW + nb) * 8 + 2 * t;
          if (r < p.rows_pad) {
            float* dst = p.scores +
                         ((static_cast<long long>(it.b) * p.kv_heads + h) * p.score_rows + j0 + g) *
                             p.rows_pad + r;
            if (lo_ok) *reinterpret_cast<float2*>(dst) = make_float2(x0, x1);
            if (hi_ok) *reinterpret_cast<float2*>(dst + 8 * p.rows_pad) = make_float2(x2, x3);
          }
        }
        if (!lo_ok) x0 = x1 = -INFINITY;
        if (!hi_ok) x2 = x3 = -INFINITY;
        float t0 = fmaxf(x0, x2), t1 = fmaxf(x1, x3);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, o));
          t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, o));
        }
        t0 = fmaxf(t0 - kShift, m[nb][0]);
        t1 = fmaxf(t1 - kShift, m[nb][1]);
        const float u0 = t0 == -INFINITY ? 0.f : t0, u1 = t1 == -INFINITY ? 0.f : t1;
        const bool moved = t0 != m[nb][0] || t1 != m[nb][1];
        if (__any_sync(0xffffffffu, moved)) {
          const float c0 = ex2(m[nb][0] - u0), c1 = ex2(m[nb][1] - u1);
          l[nb][0] *= c0;
          l[nb][1] *= c1;
#pragma unroll
          for (int x = 0; x < G::MT; ++x) {
            acc[nb][x][0] *= c0;
            acc[nb][x][1] *= c1;
            acc[nb][x][2] *= c0;
            acc[nb][x][3] *= c1;
          }
          m[nb][0] = t0;
          m[nb][1] = t1;
        }
        x0 = ex2(x0 - u0);
        x1 = ex2(x1 - u1);
        x2 = ex2(x2 - u0);
        x3 = ex2(x3 - u1);
        // the normaliser adds the weights as computed; the products below take them rounded
        // to the MMA's type (half: 2^-11, bf16: 2^-8 relative at most, of random sign)
        l[nb][0] += x0 + x2;
        l[nb][1] += x1 + x3;
        if (G::KV == IQ_ACT_BF16) {
          pb[nb][0] = transpose8x8(pack_bf16(x0, x1));
          pb[nb][1] = transpose8x8(pack_bf16(x2, x3));
        } else {
          pb[nb][0] = transpose8x8(pack_f16(x0, x1));
          pb[nb][1] = transpose8x8(pack_f16(x2, x3));
        }
      }
      // ---- O^T += V^T P^T
      if (G::KV == IQ_ACT_BF16) {
        const int r = (lane & 7) + (lane >> 4) * 8;             // matrices: d 0-7, d 8-15 of keys 0-7; of keys 8-15
#pragma unroll
        for (int x = 0; x < G::MT; ++x) {
          uint32_t a[4];
          ldmatrix_x4_trans(a, sv + r * G::DPB + (((2 * x + ((lane >> 3) & 1)) ^ (r & 7)) * 16));
#pragma unroll
          for (int nb = 0; nb < G::NBW; ++nb)
            mma_bf16(acc[nb][x], a[0], a[1], a[2], a[3], pb[nb][0], pb[nb][1]);
        }
      } else {
        // lane g holds channels 128 dd + 16 g .. + 15 (8 g .. + 7 for D = 64) of the keys
        // 2t, 2t+1, 2t+8, 2t+9; pairs of keys are interleaved bytewise, then widened
        constexpr int WORDS = G::DP >= 128 ? 4 : 2;
#pragma unroll
        for (int dd = 0; dd < (G::DP + 127) / 128; ++dd) {
          uint32_t v[4][WORDS];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int r = 2 * t + (y & 1) + (y >> 1) * 8;
            if (G::DP >= 128) {
              const uint4 w = lds128(sv + r * G::DPB + (((dd * 8 + g) ^ (((r >> 1) & 3) << 1)) * 16));
              v[y][0] = w.x; v[y][1] = w.y; v[y][WORDS - 2] = w.z; v[y][WORDS - 1] = w.w;
            } else {
              const uint2 w = lds64(sv + r * G::DPB + (((g >> 1) ^ ((r >> 1) & 3)) * 16) + (g & 1) * 8);
              v[y][0] = w.x; v[y][1] = w.y;
            }
          }
#pragma unroll
          for (int w = 0; w < WORDS; ++w) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t p01 = __byte_perm(v[0][w], v[1][w], half ? 0x7362 : 0x5140);
              const uint32_t p89 = __byte_perm(v[2][w], v[3][w], half ? 0x7362 : 0x5140);
              const uint32_t a0 = e4m3x2_to_f16x2(p01), a1 = e4m3x2_to_f16x2(p01 >> 16);
              const uint32_t a2 = e4m3x2_to_f16x2(p89), a3 = e4m3x2_to_f16x2(p89 >> 16);
              const int x = dd * 8 + 2 * w + half;
#pragma unroll
              for (int nb = 0; nb < G::NBW; ++nb)
                mma_f16(acc[nb][x], a0, a1, a2, a3, pb[nb][0], pb[nb][1]);
            }
          }
        }
      }
    }

    const bool edge_tile = it.tile >= common;
    const bool unit_end = it.tile == it.tiles - 1;
    if (unit_end || i == i1 - 1) {
      // ---- the unit ends here, or the share does: join the warps' keys
#pragma unroll
      for (int nb = 0; nb < G::NBW; ++nb)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) l[nb][c] += __shfl_xor_sync(0xffffffffu, l[nb][c], o);
#pragma unroll
      for (int nb = 0; nb < G::NBW; ++nb) {
#pragma unroll 1
        for (int half = G::WK / 2; half >= 1; half >>= 1) {
          float* mine = join + (((kg & (half - 1)) * G::WR + wr) * G::NREG) * 32 + lane;
          if (kg >= half && kg < 2 * half) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              mine[64 * c] = m[nb][c];
              mine[64 * c + 32] = l[nb][c];
            }
#pragma unroll
            for (int x = 0; x < G::MT; ++x)
#pragma unroll
              for (int y = 0; y < 4; ++y) mine[32 * (4 + 4 * x + y)] = acc[nb][x][y];
          }
          __syncthreads();
          if (kg < half) {
            float f[2], e[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const float om = mine[64 * c], ol = mine[64 * c + 32];
              const float top = fmaxf(m[nb][c], om), u = top == -INFINITY ? 0.f : top;
              f[c] = ex2(m[nb][c] - u);
              e[c] = ex2(om - u);
              m[nb][c] = top;
              l[nb][c] = l[nb][c] * f[c] + ol * e[c];
            }
#pragma unroll
            for (int x = 0; x < G::MT; ++x)
#pragma unroll
              for (int y = 0; y < 4; ++y)
                acc[nb][x][y] = acc[nb][x][y] * f[y & 1] + mine[32 * (4 + 4 * x + y)] * e[y & 1];
          }
          __syncthreads();
        }
      }
      // ---- the edge keys, row by row, on the keys that row sees
      if (edge_tile) {
        const SeqSpan& s = it.s;
        const int n_edge = span_edges(s), n_low = s.lo - s.lo0;
        if (tid < n_edge) {
          const int j = tid < n_low ? s.lo0 + tid : s.hi + tid - n_low;
          const int row = cache_row(p.pages, it.b, j);
          if (row < 0 && p.status) atomicCAS(p.status, 0, IQ_ERR_ROUTE);
          edge_rows[tid] = row;
        }
        __syncthreads();
        constexpr int PER = G::DP / 32;
        float* edge_o = join;                    // [RB][DP]
        float* edge_ml = join + G::RB * G::DP;   // [RB][2]
        for (int rr = warp; rr < G::RB; rr += G::W) {
          const int r = r0 + rr;
          if (r >= p.rows_all) break;
          const int tok = r / p.group, head = h * p.group + r % p.group;
          const int pos = s.n - p.q_len + tok;
          const __nv_bfloat16* src = p.q + it.b * p.q_b + tok * p.q_r + head * p.q_h;
          float qv[PER], ov[PER];
#pragma unroll
          for (int x = 0; x < PER; ++x) {
            const int d = lane * PER + x;
            qv[x] = d < p.dim ? __bfloat162float(src[d]) : 0.f;
            ov[x] = 0.f;
          }
          float em = -INFINITY, el = 0.f;
          for (int e = 0; e < n_edge; ++e) {
            const int j = e < n_low ? s.lo0 + e : s.hi + e - n_low;
            const bool visible = j <= pos && (p.window == 0 || j > pos - p.window);
            float x = -INFINITY;
            const int row = edge_rows[e];
            if (visible) {
              float dot = 0.f;
              const uint8_t* kr = p.k + static_cast<long long>(max(row, 0)) * p.k_row + h * p.k_head;
#pragma unroll
              for (int y = 0; y < PER; ++y) {
                const int d = lane * PER + y;
                if (d < p.dim && row >= 0)
                  dot += qv[y] * (G::KV == IQ_ACT_BF16
                                      ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(kr)[d])
                                      : e4m3_to_f32(kr[d]));
              }
              x = warp_sum(dot) * p.scale_log2;
              const float top = fmaxf(em, x), u = top == -INFINITY ? 0.f : top;
              const float f = ex2(em - u), w = ex2(x - u);
              em = top;
              el = el * f + w;
              const uint8_t* vr = p.v + static_cast<long long>(max(row, 0)) * p.v_row + h * p.v_head;
#pragma unroll
              for (int y = 0; y < PER; ++y) {
                const int d = lane * PER + y;
                const float val = d < p.dim && row >= 0
                                      ? (G::KV == IQ_ACT_BF16
                                             ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(vr)[d])
                                             : e4m3_to_f32(vr[d]))
                                      : 0.f;
                ov[y] = ov[y] * f + w * val;
              }
            }
            if (p.scores && lane == 0)
              p.scores[((static_cast<long long>(it.b) * p.kv_heads + h) * p.score_rows + j) *
                           p.rows_pad + r] = x;
          }
#pragma unroll
          for (int x = 0; x < PER; ++x) edge_o[rr * G::DP + lane * PER + x] = ov[x];
          if (lane == 0) {
            edge_ml[2 * rr] = em;
            edge_ml[2 * rr + 1] = el;
          }
        }
        __syncthreads();
        have_edges = true;
      }
      if (kg == 0) {
        const bool whole = unit_end && seg_first_tile == 0;
        const int slot_out = 2 * cta + (seg_first_tile == 0 ? 1 : 0);
#pragma unroll
        for (int nb = 0; nb < G::NBW; ++nb) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int rr = (wr * G::NBW + nb) * 8 + 2 * t + c, r = r0 + rr;
            if (r >= p.rows_all) continue;
            float f = 1.f, e = 0.f;
            if (have_edges) {
              const float om = join[G::RB * G::DP + 2 * rr], ol = join[G::RB * G::DP + 2 * rr + 1];
              const float top = fmaxf(m[nb][c], om), uu = top == -INFINITY ? 0.f : top;
              f = ex2(m[nb][c] - uu);
              e = ex2(om - uu);
              m[nb][c] = top;
              l[nb][c] = l[nb][c] * f + ol * e;
            }
            const float inv = l[nb][c] > 0.f ? 1.f / l[nb][c] : (l[nb][c] == 0.f ? 0.f : l[nb][c]);
            const int tok = r / p.group, head = h * p.group + r % p.group;
            __nv_bfloat16* o = p.out + it.b * p.o_b + tok * p.o_r + head * p.o_h;
            float* po = p.part + (static_cast<size_t>(slot_out) * G::RB + rr) * G::DP;
#pragma unroll
            for (int x = 0; x < G::MT; ++x) {
#pragma unroll
              for (int y = 0; y < 2; ++y) {      // rows g and g + 8 of the m-tile
                int d;
                if (G::KV == IQ_ACT_BF16) d = 16 * x + 8 * y + g;
                else d = G::DP >= 128 ? (x / 8) * 128 + g * 16 + 2 * (x % 8) + y : g * 8 + 2 * x + y;
                float val = acc[nb][x][2 * y + c];
                if (have_edges) val = val * f + e * join[rr * G::DP + d];
                if (whole) {
                  if (d < p.dim) o[d] = __float2bfloat16_rn(val * inv);
                } else {
                  po[d] = val;
                }
              }
            }
            if (g == 0) {
              if (whole) {
                const float z = l[nb][c] > 0.f ? m[nb][c] + log2f(l[nb][c])
                                               : (l[nb][c] == 0.f ? -INFINITY : l[nb][c]);
                const long long at = (static_cast<long long>(it.b) * p.q_len + tok) * p.q_heads + head;
                if (p.lse) p.lse[at] = z * kLn2;
                if (p.lse2) p.lse2[at] = z;
              } else {
                p.part_ml[static_cast<size_t>(slot_out) * G::RB + rr] = make_float2(m[nb][c], l[nb][c]);
              }
            }
          }
        }
      }
      __syncthreads();                           // the join buffer is free again
      fresh = true;
    }
    iter_next<G>(it, p, prefix, lens);
  }
  cp_async_wait<0>();
}

// ------------------------------------------------------------------------------------
// Adds the partial results of the units that several CTAs shared: slot 2c + 1 of the first
// CTA, slot 2c of the others, in that order.  `wide`: a block of eight warps a query row
// (many partials a unit); else a warp a row.
constexpr int kJoinThreads = 256;

template <int DP, int RB>
__global__ void __launch_bounds__(kJoinThreads) attn_join_kernel(const __grid_constant__ AttnParams p,
                                                                int wide) {
  __shared__ float red_ml[8][2];
  __shared__ float red_o[8][DP];
  constexpr int PER = DP / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = p.kv_heads * p.n_rb;
  const int u = blockIdx.x;
  const int b = u / per, hb = u - b * per, h = hb / p.n_rb, r0 = (hb - h * p.n_rb) * RB;
  const int rr = wide ? blockIdx.y : blockIdx.y * 8 + warp;
  const int r = r0 + rr;
  pdl_wait();
  pdl_launch_dependents();
  const int2 c = p.units[u];
  if (c.y <= c.x || (wide && r >= p.rows_all)) return;
  const bool live = rr < RB && r < p.rows_all;
  float M = -INFINITY, L = 0.f, o[PER];
#pragma unroll
  for (int x = 0; x < PER; ++x) o[x] = 0.f;
  if (live) {
    const int step = wide ? 8 : 1, n = c.y - c.x + 1;
    for (int base = wide ? warp : 0; base < n; base += 32 * step) {
      const int mine = base + lane * step;
      auto slot_of = [&](int k) { return static_cast<size_t>(2 * (c.x + k) + (k == 0 ? 1 : 0)) * RB + rr; };
      float2 ml = make_float2(-INFINITY, 0.f);
      if (mine < n) ml = __ldcg(p.part_ml + slot_of(mine));
      const float top = fmaxf(M, warp_max(ml.x)), uu = top == -INFINITY ? 0.f : top;
      const float old = ex2(M - uu), f = ex2(ml.x - uu);
      M = top;
      L = L * old + warp_sum(ml.y * f);
#pragma unroll
      for (int x = 0; x < PER; ++x) o[x] *= old;
      const int cnt = min(32, (n - base + step - 1) / step);
#pragma unroll 8
      for (int k = 0; k < cnt; ++k) {
        const float fk = __shfl_sync(0xffffffffu, f, k);
        const float* src = p.part + slot_of(base + k * step) * DP + lane * PER;
        float v[PER];
        if constexpr (PER >= 4) {
#pragma unroll
          for (int x = 0; x < PER; x += 4) {
            const float4 w = __ldcg(reinterpret_cast<const float4*>(src + x));
            v[x] = w.x; v[x + 1] = w.y; v[x + 2] = w.z; v[x + 3] = w.w;
          }
        } else {
          const float2 w = __ldcg(reinterpret_cast<const float2*>(src));
          v[0] = w.x; v[1] = w.y;
        }
#pragma unroll
        for (int x = 0; x < PER; ++x) o[x] += fk * v[x];
      }
    }
  }
  if (wide) {
    if (lane == 0) { red_ml[warp][0] = M; red_ml[warp][1] = L; }
#pragma unroll
    for (int x = 0; x < PER; ++x) red_o[warp][lane * PER + x] = o[x];
    __syncthreads();
    if (warp) return;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < 8; ++w) top = fmaxf(top, red_ml[w][0]);
    const float uu = top == -INFINITY ? 0.f : top;
    L = 0.f;
#pragma unroll
    for (int x = 0; x < PER; ++x) o[x] = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const float f = ex2(red_ml[w][0] - uu);
      L += f * red_ml[w][1];
#pragma unroll
      for (int x = 0; x < PER; ++x) o[x] += f * red_o[w][lane * PER + x];
    }
    M = top;
  }
  if (!live) return;
  const int tok = r / p.group, head = h * p.group + r % p.group;
  __nv_bfloat16* dst = p.out + b * p.o_b + tok * p.o_r + head * p.o_h;
  const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
#pragma unroll
  for (int x = 0; x < PER; ++x)
    if (lane * PER + x < p.dim) dst[lane * PER + x] = __float2bfloat16_rn(o[x] * inv);
  if (lane == 0) {
    const float z = L > 0.f ? M + log2f(L) : (L == 0.f ? -INFINITY : L);
    const long long at = (static_cast<long long>(b) * p.q_len + tok) * p.q_heads + head;
    if (p.lse) p.lse[at] = z * kLn2;
    if (p.lse2) p.lse2[at] = z;
  }
}

// ------------------------------------------------------------------------------------
// weights[b, h, j] += sum over the head's query rows of 2^(x_j - lse2): a thread a key, the
// scores the split kernel left behind (L2 holds most of them) against the joined lse.
// The step's own rows are set, not added to, and get their positions.
__global__ void __launch_bounds__(256) attn_weights_kernel(const __grid_constant__ AttnParams p) {
  __shared__ float z[512];
  const int b = blockIdx.z, h = blockIdx.y;
  pdl_wait();
  pdl_launch_dependents();
  const SeqSpan s = seq_span(clamp_length(p, b, false), p.q_len, p.window);
  for (int r = threadIdx.x; r < p.rows_pad; r += blockDim.x) {
    float v = INFINITY;                          // a padded or empty row adds nothing
    if (r < p.rows_all) {
      const int tok = r / p.group, head = h * p.group + r % p.group;
      v = __ldcg(p.lse2 + (static_cast<long long>(b) * p.q_len + tok) * p.q_heads + head);
      if (v == -INFINITY) v = INFINITY;
    }
    z[r] = v;
  }
  __syncthreads();
  for (int j = s.lo0 + blockIdx.x * blockDim.x + threadIdx.x; j < s.n; j += gridDim.x * blockDim.x) {
    const float* src = p.scores +
                       ((static_cast<long long>(b) * p.kv_heads + h) * p.score_rows + j) * p.rows_pad;
    float w = 0.f;
    for (int r = 0; r < p.rows_pad; r += 4) {
      const float4 x4 = __ldcg(reinterpret_cast<const float4*>(src + r));
      const float x[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
      for (int y = 0; y < 4; ++y) w += z[r + y] == INFINITY ? 0.f : ex2(x[y] - z[r + y]);
    }
    float* dst = p.weights + b * p.w_b + h * p.w_h + j;
    const bool is_new = j >= s.n - p.q_len;
    *dst = is_new ? w : *dst + w;
    if (is_new && p.positions) p.positions[b * p.p_b + h * p.p_h + j] = __ldg(p.seen + b) - s.n + j;
  }
}

// ------------------------------------------------------------------------------------
// host side
static std::mutex g_attn_mutex;

static int attn_sms() {
  static int per_device[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  std::lock_guard<std::mutex> lock(g_attn_mutex);
  if (per_device[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    per_device[dev] = n;
  }
  return per_device[dev];
}

static bool attn_smem_optin(const void* fn, int bytes) {
  static std::unordered_set<uint64_t> done;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t key = (reinterpret_cast<uint64_t>(fn) << 6) ^ static_cast<uint64_t>(dev);
  std::lock_guard<std::mutex> lock(g_attn_mutex);
  if (done.count(key)) return true;
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return false;
  done.insert(key);
  return true;
}

template <class K, class... Args>
static int attn_launch(K kernel, dim3 grid, int threads, int smem, void* stream, bool pdl,
                       const Args&... args) {
  if (smem > 48 * 1024 && !attn_smem_optin(reinterpret_cast<const void*>(kernel), smem))
    return IQ_ERR_CUDA;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1] = {};
  if (pdl) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (err != cudaSuccess) {
    fprintf(stderr, "iqb200: launch failed: %s\n", cudaGetErrorString(err));
    return IQ_ERR_CUDA;
  }
  return IQ_OK;
}

// The work area: partial results of the largest grid, the units' table, then (with weights)
// the joined lse and the scores.
struct AttnWork {
  size_t part, part_ml, units, lse2, scores, total;
};
constexpr int kAttnMaxCtas = 2 * 160;            // CTAs of the split kernel, at most

static int pad_dim(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }
static int block_rows(int rows) { return rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

static AttnWork attn_work(int batch, int q_len, int q_heads, int kv_heads, int dim, int rows,
                          bool weights) {
  const int all = q_heads / kv_heads * q_len;
  const int rb = block_rows(all), n_rb = (all + rb - 1) / rb;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  AttnWork w{};
  size_t at = 0;
  w.part = at;
  at += up(static_cast<size_t>(2 * kAttnMaxCtas) * rb * pad_dim(dim) * 4);
  w.part_ml = at;
  at += up(static_cast<size_t>(2 * kAttnMaxCtas) * rb * 8);
  w.units = at;
  at += up(static_cast<size_t>(batch) * kv_heads * n_rb * 8);
  if (weights) {
    w.lse2 = at;
    at += up(static_cast<size_t>(batch) * q_len * q_heads * 4);
    w.scores = at;
    at += up(static_cast<size_t>(batch) * kv_heads * rows * ((all + 7) / 8 * 8) * 4);
  }
  w.total = at;
  return w;
}

static bool attn_shape_ok(int batch, int q_len, int q_heads, int kv_heads, int dim, int rows) {
  return batch >= 1 && batch <= kAttnMaxBatch && q_len >= 1 && q_len <= 8 && kv_heads >= 1 &&
         q_heads >= kv_heads && q_heads % kv_heads == 0 && q_heads / kv_heads * q_len <= 512 &&
         dim >= 16 && dim <= 256 && dim % 16 == 0 && rows >= 1 && kv_heads <= 65535;
}

template <class G>
static int attn_run(AttnParams& p, int n_sm, bool pdl, void* stream) {
  const long long tiles = static_cast<long long>(p.batch) * p.kv_heads * p.n_rb *
                          ((p.max_rows + G::TK - 1) / G::TK + 1);
  if (tiles > 0x7fffffffLL) return IQ_ERR_UNSUPPORTED;
  const int grid = static_cast<int>(tiles < n_sm * G::CTAS ? tiles : n_sm * G::CTAS);
  int rc = attn_launch(attn_kernel<G>, dim3(grid), G::THREADS, G::SMEM, stream, pdl, p);
  if (rc != IQ_OK) return rc;
  const int units = p.batch * p.kv_heads * p.n_rb;
  // a unit's share of the CTAs: above eight, its partial results are worth a block a row
  const int wide = grid > 8 * units;
  const int y = wide ? (p.rows_all < G::RB ? p.rows_all : G::RB)
                     : ((p.rows_all < G::RB ? p.rows_all : G::RB) + 7) / 8;
  return attn_launch(attn_join_kernel<G::DP, G::RB>, dim3(units, y), kJoinThreads, 0, stream, true,
                     p, wide);
}

template <int KV, int DP>
static int attn_pick(AttnParams& p, int n_sm, bool pdl, void* stream) {
  constexpr int W = KV == IQ_ACT_BF16 && DP == 256 ? 4 : 8;
  if (p.rows_all <= 8) return attn_run<AttnGeo<KV, DP, 1, 1, W, 1>>(p, n_sm, pdl, stream);
  if constexpr (DP <= 128) {
    if (p.rows_all <= 16) return attn_run<AttnGeo<KV, DP, 2, 1, 8, 1>>(p, n_sm, pdl, stream);
    if (p.rows_all <= 32) return attn_run<AttnGeo<KV, DP, 2, 2, 8, 1>>(p, n_sm, pdl, stream);
    return attn_run<AttnGeo<KV, DP, 2, 4, 8, 1>>(p, n_sm, pdl, stream);
  } else {
    if (p.rows_all <= 16) return attn_run<AttnGeo<KV, DP, 1, 2, W, 1>>(p, n_sm, pdl, stream);
    if (p.rows_all <= 32) return attn_run<AttnGeo<KV, DP, 1, 4, 8, 1>>(p, n_sm, pdl, stream);
    return attn_run<AttnGeo<KV, DP, 1, 8, 8, 1>>(p, n_sm, pdl, stream);
  }
}

}  // namespace iqb

using namespace iqb;

extern "C" size_t iq_attn_work_bytes(int batch, int q_len, int q_heads, int kv_heads, int head_dim,
                                     int rows, int weights) {
  if (!attn_shape_ok(batch, q_len, q_heads, kv_heads, head_dim, rows)) return 0;
  return attn_work(batch, q_len, q_heads, kv_heads, head_dim, rows, weights != 0).total;
}

extern "C" int iq_attn_decode(const iq_attn_args* a, void* stream) {
  if (!a || !a->q || !a->k_cache || !a->v_cache || !a->page_table || !a->lengths || !a->out ||
      !a->work)
    return IQ_ERR_ARG;
  if (a->page_size < 1 || a->max_pages < 1 || a->capacity < 1 || a->window < 0) return IQ_ERR_ARG;
  if (a->kv_kind != IQ_ACT_BF16 && a->kv_kind != IQ_ACT_E4M3) return IQ_ERR_ARG;
  const long long rows = static_cast<long long>(a->page_size) * a->max_pages;
  if (rows > 0x3fffffffLL) return IQ_ERR_UNSUPPORTED;
  if (!attn_shape_ok(a->batch, a->q_len, a->q_heads, a->kv_heads, a->head_dim,
                     static_cast<int>(rows)))
    return IQ_ERR_UNSUPPORTED;
  const bool weights = a->weights != nullptr;
  if (weights && a->weights_rows < rows) return IQ_ERR_ARG;
  if ((a->positions != nullptr) != (a->seen != nullptr) || (a->positions && !weights))
    return IQ_ERR_ARG;
  const AttnWork w = attn_work(a->batch, a->q_len, a->q_heads, a->kv_heads, a->head_dim,
                               static_cast<int>(rows), weights);
  if (a->work_bytes < w.total) return IQ_ERR_ARG;
  // 16-byte copies of cache rows, 4-byte loads of q
  const int64_t elt = a->kv_kind == IQ_ACT_BF16 ? 2 : 1;
  const uint64_t al = reinterpret_cast<uint64_t>(a->k_cache) | reinterpret_cast<uint64_t>(a->v_cache) |
                      static_cast<uint64_t>(a->k_row * elt) | static_cast<uint64_t>(a->k_head * elt) |
                      static_cast<uint64_t>(a->v_row * elt) | static_cast<uint64_t>(a->v_head * elt) |
                      reinterpret_cast<uint64_t>(a->work);
  if (al & 15) return IQ_ERR_ARG;
  if ((reinterpret_cast<uint64_t>(a->q) & 3) || ((a->q_b | a->q_r | a->q_h) & 1)) return IQ_ERR_ARG;
  const int n_sm = attn_sms();
  if (n_sm == 0 || n_sm * 2 > kAttnMaxCtas) return IQ_ERR_CUDA;

  AttnParams p{};
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.q_b = a->q_b; p.q_r = a->q_r; p.q_h = a->q_h;
  p.k = static_cast<const uint8_t*>(a->k_cache);
  p.v = static_cast<const uint8_t*>(a->v_cache);
  p.k_row = a->k_row * elt; p.k_head = a->k_head * elt;
  p.v_row = a->v_row * elt; p.v_head = a->v_head * elt;
  p.pages.table = a->page_table;
  p.pages.stride = a->table_stride;
  p.pages.page = a->page_size;
  p.pages.shift = -1;
  for (int s = 0; s < 30; ++s)
    if (a->page_size == 1 << s) p.pages.shift = s;
  p.pages.capacity = a->capacity;
  p.lengths = a->lengths;
  p.max_rows = static_cast<int>(rows);
  p.out = static_cast<__nv_bfloat16*>(a->out);
  p.o_b = a->o_b; p.o_r = a->o_r; p.o_h = a->o_h;
  p.lse = a->lse;
  uint8_t* work = static_cast<uint8_t*>(a->work);
  p.part = reinterpret_cast<float*>(work + w.part);
  p.part_ml = reinterpret_cast<float2*>(work + w.part_ml);
  p.units = reinterpret_cast<int2*>(work + w.units);
  p.status = a->status;
  p.batch = a->batch; p.q_len = a->q_len; p.q_heads = a->q_heads; p.kv_heads = a->kv_heads;
  p.group = a->q_heads / a->kv_heads;
  p.dim = a->head_dim;
  // a window that reaches past the whole table is none
  p.window = a->window >= rows ? 0 : a->window;
  p.rows_all = p.group * p.q_len;
  p.rows_pad = (p.rows_all + 7) / 8 * 8;
  const int rb = block_rows(p.rows_all);
  p.n_rb = (p.rows_all + rb - 1) / rb;
  p.scale_log2 = a->scale * kLog2e;
  if (weights) {
    p.lse2 = reinterpret_cast<float*>(work + w.lse2);
    p.scores = reinterpret_cast<float*>(work + w.scores);
    p.score_rows = static_cast<int>(rows);
    p.weights = a->weights;
    p.w_b = a->w_b; p.w_h = a->w_h;
    p.positions = a->positions;
    p.p_b = a->p_b; p.p_h = a->p_h;
    p.seen = a->seen;
  }
  const bool bf16 = a->kv_kind == IQ_ACT_BF16, pdl = a->pdl != 0;
  int rc;
  switch (pad_dim(a->head_dim)) {
    case 64:
      rc = bf16 ? attn_pick<IQ_ACT_BF16, 64>(p, n_sm, pdl, stream)
                : attn_pick<IQ_ACT_E4M3, 64>(p, n_sm, pdl, stream);
      break;
    case 128:
      rc = bf16 ? attn_pick<IQ_ACT_BF16, 128>(p, n_sm, pdl, stream)
                : attn_pick<IQ_ACT_E4M3, 128>(p, n_sm, pdl, stream);
      break;
    default:
      rc = bf16 ? attn_pick<IQ_ACT_BF16, 256>(p, n_sm, pdl, stream)
                : attn_pick<IQ_ACT_E4M3, 256>(p, n_sm, pdl, stream);
  }
  if (rc != IQ_OK || !weights) return rc;
  // enough blocks for four waves of the chip, never more than the rows need
  const int by_rows = static_cast<int>((rows + 255) / 256);
  const int units = a->batch * a->kv_heads;
  int x = (n_sm * 8 + units - 1) / units;
  if (x > by_rows) x = by_rows;
  return attn_launch(attn_weights_kernel, dim3(x, a->kv_heads, a->batch), 256, 0, stream, true, p);
}
