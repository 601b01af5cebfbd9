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
// Split.  A unit is a sequence, a group of HG key/value heads and a block of query rows; its
// keys are cut into tiles of TK.  The tiles of all units form one list that is dealt to the
// CTAs in equal contiguous shares, whatever the lengths are.  A unit that falls into one
// share is finished there; one that spans several leaves partial results that
// attn_join_kernel adds.  The HG heads of a group are neighbours in memory and are read at the
// same time by the warps of one CTA, so that DRAM sees pieces of HG rows, not of one.
//
// What a row must not see (later tokens of its step, keys that slid out of its window, rows
// past the end) never meets it: its score is replaced, and its value, which the product
// would multiply by zero, is zeroed in shared memory where it is outside the unit or, for the
// few keys that only some rows see, where it is not finite (0 x NaN); those rows then get the
// infinities and NaNs they do see added at the end.
//
// Layout.  S^T = K Q^T and O^T = V^T P^T on the warp MMA (m16n8k16): the cache is the
// 16-row operand and eight query rows the columns, so a group of eight heads fills the
// tile that would otherwise be padded to sixteen rows.  A warp (with more than sixteen
// query rows: a group of warps) owns KPW keys of a tile, one head and all of D.  The warps of
// the same keys share a ring, one stage for all HG heads, which a copying warp fills with
// tiled TMA copies (128-byte swizzle; one box a page piece), or four copying warps gather
// where pages are so small that a tile takes more than sixteen boxes; there is no block
// barrier in the loop, and the warps' keys join at the end of a unit.  Keys sit at absolute
// multiples of KPW, so that a box never leaves its page; the rows of a box that lie outside
// the unit's keys get no weight, and their values are zeroed in shared memory first.
//
// Measured (one B200, both launches, pages of 64 unless said, 128 channels, 8 rows a head):
// e4m3, 64 / 8 heads, 131071 keys: 51.7 us, 5.2 TB/s; 32768 keys, one 8 / 1 shard: 9.9 us;
// 32 sequences of 8192: 90 us, 6.0 TB/s; bf16, 48 sequences of 1 to 8192 keys, pages of 16:
// 146 us, 6.3 TB/s (96 % of a copy's rate).  32 rows a head (four tokens) over 32k keys of
// e4m3: 32.8 us, there the warp MMA and its feeding are the limit.  About 8 us of a call are
// fixed: two launches, the lengths -> page table -> keys chain, the joins.
#include <math.h>
#include <stdio.h>

#include <atomic>
#include <type_traits>

#include <cuda_fp16.h>

#include "paged.cuh"

namespace iqb {

constexpr int kAttnMaxBatch = 1024;
constexpr int kCopyThreads = 128;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLog2e = 1.4426950408889634f;

struct AttnParams {
  CUtensorMap k_map, v_map;                      // bytes: (head_dim, capacity, kv_heads)
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
  float* part;                                   // [2 grid][HG][RB][DP] unnormalised O
  float2* part_ml;                               // [2 grid][HG][RB] (M, l)
  int2* units;                                   // [units] first and last CTA of a split unit
  float* scores;                                 // [batch * kv_heads][score_rows][rows_all] x_j, or null
  float* lse2;                                   // [batch, q_len, q_heads] M + log2 l (with scores)
  int score_rows;
  float* weights;
  long long w_b, w_h;
  int* positions;
  long long p_b, p_h;
  const int* seen;
  const long long* slot;                         // of the step's rows, or null
  unsigned joins;                                // blocks along x that join
  unsigned weight_chunks, weight_blocks;         // blocks a (sequence, head)'s weights take; all of them
  int* status;
  int batch, q_len, q_heads, kv_heads, group, dim, window;
  int rows_all;                                  // group * q_len
  int rows_pad;                                  // rows_all rounded up to eight
  int n_rb;                                      // blocks of RB rows
  int box_rows, box_heads;                       // of a TMA copy: divide a page and KPW; 1 or HG
  int gather;                                    // copy by threads, 16 bytes at a time, instead
  float scale_log2;
};

// One sequence's keys: [lo, n) are seen by some row of the step, [lo_all, hi_all) by all.
struct SeqSpan {
  int n, lo, lo_all, hi_all;
};
__device__ __forceinline__ SeqSpan seq_span(int n, int q_len, int window) {
  SeqSpan s;
  s.n = n;
  s.lo = window ? max(0, n - q_len - window + 1) : 0;
  s.lo_all = window ? max(0, n - window) : 0;
  s.hi_all = max(n - q_len + 1, 0);
  return s;
}
// Tiles start at `lo` rounded down to the keys a warp copies.
template <class G>
__device__ __forceinline__ int span_tiles(const SeqSpan& s) {
  return (s.n - s.lo / G::KPW * G::KPW + G::TK - 1) / G::TK;
}

__device__ __forceinline__ int clamp_length(const AttnParams& p, int b, bool report) {
  const int n = __ldg(p.lengths + b);
  if (n < 0 || n > p.max_rows) {
    if (report && p.status) atomicCAS(p.status, 0, IQ_ERR_ROUTE);
    return n < 0 ? 0 : p.max_rows;
  }
  return n;
}

// D(16x8, fp32) += A(16x16) B(16x8), operands half (e4m3 caches) or bf16.
template <int KV>
__device__ __forceinline__ void mma_k16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  if (KV == IQ_ACT_BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
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
__device__ __forceinline__ void tma_3d_g2s(uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                           uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}

// KV: IQ_ACT_E4M3 or IQ_ACT_BF16.  DP: head dim rounded up (64, 128, 256).  NBW: blocks of
// eight query rows a warp holds; WR warps share a head's keys, each with its own rows; HG
// heads a unit; W warps that compute.  The W / WR / HG = KG groups of warps have a ring each,
// of stages of KPW keys of all HG heads; KPW is what makes a stage of all rings 64 KB.
template <int KV_, int DP_, int NBW_, int WR_, int HG_, int W_>
struct AttnGeo {
  static constexpr int KV = KV_, DP = DP_, NBW = NBW_, WR = WR_, HG = HG_, W = W_;
  static constexpr int ELT = KV == IQ_ACT_BF16 ? 2 : 1;
  static constexpr int DPB = DP * ELT;
  static constexpr int WK = W / WR;
  static constexpr int KG = WK / HG;
  static constexpr int KPW = 32768 / (WK * DPB) < 16 ? 16 : 32768 / (WK * DPB);
  static constexpr int SUB = KPW / 16;
  // Tiles of sixteen keys in flight together: independent sums where a warp has one block of
  // rows; with more, half the code is worth more (whole calls in a graph, 32 rows a head over
  // 32749 keys, 64 / 8 heads: e4m3 32.1 us against 33.7 for two tiles, bf16 36.2 against 39.9)
  static constexpr int SUBI = NBW == 1 && SUB > 1 ? 2 : 1;
  static constexpr int TK = KPW * KG;            // keys a tile
  static constexpr int RB = 8 * NBW * WR;        // query rows a block
  static constexpr int CONSUMERS = 32 * W;
  static constexpr int THREADS = CONSUMERS + kCopyThreads;
  // Registers move from the copying warps to the others (eight of those: 12 warps share the
  // file at 168 a thread; the shares add up to what the block was launched with)
  static constexpr bool MOVE_REGS = W == 8;
  static constexpr int REGS = 168, REGS_COPY = 72, REGS_COMPUTE = 216;
  static_assert(REGS_COPY * kCopyThreads + REGS_COMPUTE * CONSUMERS <= REGS * THREADS || !MOVE_REGS,
                "the register shares are those of the launch");
  static constexpr int PITCH = DPB < 128 ? DPB : 128;   // bytes of a row in one box
  static constexpr int BOXES = DPB / PITCH;      // boxes side by side that make a row
  static constexpr int HEAD = KPW * PITCH;       // one head of one box
  static constexpr int BOX = HG * HEAD;          // a stage: [keys, values][box][head][row]
  static constexpr int HALF = BOXES * BOX;
  static constexpr int STAGE = 2 * HALF;
  static constexpr int MT = DP / 16;             // m-tiles of O^T
  static constexpr int QREG = DP / 8;            // packed registers of q a block of eight rows
  static constexpr bool QS = NBW * DP >= 512;    // q's fragments live in shared memory
  // joining warps exchange one block of eight rows: a lane's M, l and O, in XP parts
  static constexpr int XP = W == 16 ? 2 : 1;
  static constexpr int NREG = MT / XP * 4 + 4;
  static constexpr int JOIN = KG > 1 ? (W / 2) * 32 * NREG * 4 : 0;
  static constexpr int QBYTES = QS ? HG * WR * NBW * QREG * 128 : 0;
  static constexpr int MAX_STAGES = 8;
  static constexpr int FIXED = 1024 + JOIN + QBYTES + 2 * KG * MAX_STAGES * 8 + (2 * kAttnMaxBatch + 64) * 4;
  static constexpr int FIT = (227 * 1024 - FIXED) / (KG * STAGE);
  static constexpr int STAGES = FIT > MAX_STAGES ? MAX_STAGES : FIT;
  static constexpr int SMEM = KG * STAGES * STAGE + FIXED;
  static_assert(STAGES >= 2, "the ring needs two stages");
  static_assert(HEAD % 1024 == 0, "swizzled boxes start on their pattern's period");
  static_assert(KPW <= 256, "a box has at most 256 rows");
  static_assert(WK % HG == 0, "every head has the same number of rings");
};

// The key of a sixteen-key tile that sits in row i (of eight) of the MMA operand.  e4m3: a
// permutation under which the 16-byte (8-byte at D = 64) loads of both the keys' and the
// values' fragments touch every bank once on rows that TMA swizzled.  bf16 (ldmatrix): none.
template <class G>
__device__ __forceinline__ int key_of(int i) {
  if (G::KV == IQ_ACT_BF16) return i;
  if (G::DPB >= 128) return i & 1 ? i ^ 4 : i;   // 0 5 2 7 4 1 6 3
  return (0x65742130 >> (4 * i)) & 7;            // 0 3 1 2 4 7 5 6
}
// Byte offset of 16-byte piece c of row r inside a box.
template <class G>
__device__ __forceinline__ int swizzled(int r, int c) {
  return G::PITCH == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
}
// The channel of rows g (y = 0) and g + 8 (y = 1) of m-tile x of O^T.
template <class G>
__device__ __forceinline__ int channel_of(int x, int y, int g) {
  if (G::KV == IQ_ACT_BF16) return 16 * x + 8 * y + g;
  return G::DP >= 128 ? (x / 8) * 128 + g * 16 + 2 * (x % 8) + y : g * 8 + 2 * x + y;
}

// A place in the list of tiles.
template <class G>
struct Walk {
  int b, hb;                                     // sequence; head group and block of rows
  int left;                                      // tiles of the unit from here on
  int j;                                         // the tile's first key
  int lo, n;                                     // the unit's keys
  int h0, r0;                                    // first head, first query row

  __device__ __forceinline__ void unit(const AttnParams& p, const int* prefix, const int* lens, int tile) {
    const SeqSpan s = seq_span(lens[b], p.q_len, p.window);
    lo = s.lo;
    n = s.n;
    left = prefix[b + 1] - prefix[b] - tile;
    j = s.lo / G::KPW * G::KPW + tile * G::TK;
    const int hg = p.n_rb == 1 ? hb : hb / p.n_rb;
    h0 = hg * G::HG;
    r0 = (hb - hg * p.n_rb) * G::RB;
  }
  // Returns the tile's place in its unit.
  __device__ __forceinline__ int start(const AttnParams& p, const int* prefix, const int* lens, int per, int i) {
    int first = 0, end = p.batch;                // prefix[first] * per <= i < prefix[end] * per
    while (end - first > 1) {
      const int mid = (first + end) >> 1;
      if (prefix[mid] * per <= i) first = mid; else end = mid;
    }
    b = first;
    const int tiles = prefix[b + 1] - prefix[b], rem = i - prefix[b] * per;
    hb = rem / tiles;
    unit(p, prefix, lens, rem - hb * tiles);
    return rem - hb * tiles;
  }
  __device__ __forceinline__ void next(const AttnParams& p, const int* prefix, const int* lens, int per) {
    j += G::TK;
    if (--left > 0) return;
    if (++hb == per) {
      hb = 0;
      do {
        if (++b == p.batch) return;
      } while (prefix[b + 1] == prefix[b]);
    }
    unit(p, prefix, lens, 0);
  }
};

// Zeroes what is not finite among sixteen bytes of values; whether there was any.
template <int KV>
__device__ __forceinline__ bool strip(uint4& v) {
  uint32_t* w = &v.x;
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (KV == IQ_ACT_BF16) {
#pragma unroll
      for (int x = 0; x < 32; x += 16)
        if ((w[i] >> x & 0x7f80u) == 0x7f80u) { w[i] &= ~(0xffffu << x); any = true; }
    } else {
#pragma unroll
      for (int x = 0; x < 32; x += 8)
        if ((w[i] >> x & 0x7fu) == 0x7fu) { w[i] &= ~(0xffu << x); any = true; }
    }
  }
  return any;
}

// Adds to the segment's results, which its warps have just written (to `out`, or to partial
// results `slot`), the infinities and NaNs that `strip` took out of the values of the keys
// [from, to) that only some rows see.  (Their weight is positive, so it does not matter.)
// All consumer threads of the CTA call it.
template <class G>
__device__ __noinline__ void add_not_finite(const AttnParams& p, int b, int n, int h0, int r0, int from,
                                            int to, bool whole, int slot) {
  const SeqSpan s = seq_span(n, p.q_len, p.window);
  const int rows = min(G::RB, p.rows_all - r0);
  for (int i = threadIdx.x; i < G::HG * rows * p.dim; i += G::CONSUMERS) {
    const int d = i % p.dim, rr = i / p.dim % rows, hg = i / p.dim / rows;
    const int h = h0 + hg, tok = (r0 + rr) / p.group, head = h * p.group + (r0 + rr) % p.group;
    const int pos = n - p.q_len + tok;
    float sum = 0.f;
    for (int j = max(from, p.window ? pos - p.window + 1 : 0); j < min(to, pos + 1); ++j) {
      if (j < 0 || (j >= s.lo_all && j < s.hi_all)) continue;   // seen by all: in the product already
      const int row = cache_row(p.pages, b, j);
      if (row < 0) continue;
      const uint8_t* v = p.v + row * p.v_row + h * p.v_head;
      const float x = G::KV == IQ_ACT_BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(v)[d])
                                           : e4m3_to_f32(v[d]);
      if (!isfinite(x)) sum += x;
    }
    if (sum == 0.f) continue;
    if (whole) {
      __nv_bfloat16* o = p.out + b * p.o_b + tok * p.o_r + head * p.o_h + d;
      *o = __float2bfloat16_rn(__bfloat162float(*o) + sum);
    } else {
      // the place of (rr, d) in the fragments
      int x, y, g;
      if (G::KV == IQ_ACT_BF16) { x = d / 16; y = d / 8 % 2; g = d % 8; }
      else if (G::DP >= 128) { x = d / 128 * 8 + d % 16 / 2; y = d % 2; g = d % 128 / 16; }
      else { x = d % 8 / 2; y = d % 2; g = d / 8; }
      const size_t block = (static_cast<size_t>(slot) * G::HG + hg) * (G::RB / 8) + rr / 8;
      p.part[((block * G::MT + x) * 32 + 4 * g + rr % 8 / 2) * 4 + 2 * y + rr % 2] += sum;
    }
  }
}

template <class G>
__global__ void __launch_bounds__(G::THREADS, 1) attn_kernel(const __grid_constant__ AttnParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* ring = smem;
  float* join = reinterpret_cast<float*>(smem + G::KG * G::STAGES * G::STAGE);
  uint32_t* q_smem = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(join) + G::JOIN);
  uint64_t* bar_full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(q_smem) + G::QBYTES);
  uint64_t* bar_free = bar_full + G::KG * G::MAX_STAGES;                // both [ring][stage]
  int* prefix = reinterpret_cast<int*>(bar_free + G::KG * G::MAX_STAGES);   // [batch + 1]
  int* lens = prefix + kAttnMaxBatch + 4;        // [batch]
  int* warp_sums = lens + kAttnMaxBatch;         // [W]
  int* not_finite = warp_sums + 32;              // a value that only some rows see is not finite

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // rows, head of the unit, ring
  const int wr = warp % G::WR, hg = warp / G::WR % G::HG, kg = warp / (G::WR * G::HG);
  const int g = lane >> 2, t = lane & 3;
  const int cta = blockIdx.x;

  if (tid < G::KG * G::STAGES) {
    mbar_init(bar_full + (tid / G::STAGES) * G::MAX_STAGES + tid % G::STAGES, p.gather ? kCopyThreads : 1);
    mbar_init(bar_free + (tid / G::STAGES) * G::MAX_STAGES + tid % G::STAGES, G::HG * G::WR);
  }
  mbar_fence_init();
  if (tid == 0) {
    *not_finite = 0;
    if (!p.gather) {
      prefetch_tensormap(&p.k_map);
      prefetch_tensormap(&p.v_map);
    }
  }
  pdl_wait();
  pdl_launch_dependents();

  // ---- the list of tiles: exclusive prefix over the sequences
  {
    const int each = (p.batch + G::THREADS - 1) / G::THREADS;
    const int b0 = min(tid * each, p.batch), b1 = min(b0 + each, p.batch);
    int sum = 0;
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
      const int n = clamp_length(p, b, cta == 0);
      lens[b] = n;
      sum += span_tiles<G>(seq_span(n, p.q_len, p.window));
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
#pragma unroll 4
    for (int w = 0; w < G::THREADS / 32; ++w) at += w < warp ? warp_sums[w] : 0;
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
      prefix[b] = at;
      at += span_tiles<G>(seq_span(lens[b], p.q_len, p.window));
    }
    if (tid == G::THREADS - 1) prefix[p.batch] = at;
    __syncthreads();
  }
  const int per = p.kv_heads / G::HG * p.n_rb;
  const int total = prefix[p.batch] * per;
  // the first `total % gridDim` CTAs take one tile more; some none, behind all others
  const int share = total / static_cast<int>(gridDim.x), more = total % static_cast<int>(gridDim.x);
  const int i0 = share * cta + min(cta, more), i1 = i0 + share + (cta < more ? 1 : 0);

  // ---- the copying warps: all rings, a tile at a time.  Their instructions per tile are what
  // a small stage would be bound by (one dependent instruction after another)
  if (warp >= G::W) {
    if (G::MOVE_REGS) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::REGS_COPY));
    if (i0 >= i1 || (!p.gather && warp > G::W)) return;
    Walk<G> ld;
    ld.start(p, prefix, lens, per, i0);
    if (p.gather) {
      // Pages too small for boxes: thread t copies piece t % CPR of every (128 / CPR)-th row,
      // for all heads of the unit.  Arrives at `full` when its copies have.
      constexpr int CPR = G::DPB / 16, ROWS = kCopyThreads / CPR, PIECES = G::PITCH / 16;
      static_assert((G::KPW < 32 ? G::KPW : 32) % ROWS == 0, "whole passes");
      const int ct = tid - G::CONSUMERS, c = ct % CPR;
      const bool in_row = c * 16 < p.dim * G::ELT;
      int stage = 0;
      uint32_t parity = 1;
#pragma unroll 1
      for (int i = i0; i < i1; ++i) {
#pragma unroll 1
        for (int kgr = 0; kgr < G::KG; ++kgr) {
          if (!mbar_wait(bar_free + kgr * G::MAX_STAGES + stage, parity)) {
            if (p.status) atomicCAS(p.status, 0, IQ_ERR_PIPE_TIMEOUT);
            i = i1;
            break;
          }
          const uint32_t to = smem_u32(ring) + (kgr * G::STAGES + stage) * G::STAGE + c / PIECES * G::BOX;
          const uint8_t* k0 = p.k + ld.h0 * p.k_head + c * 16;
          const uint8_t* v0 = p.v + ld.h0 * p.v_head + c * 16;
#pragma unroll 1
          for (int base = 0; base < G::KPW; base += 32) {
            // a lane looks up one row of thirty-two
            const int j = ld.j + kgr * G::KPW + base + lane;
            int mine = -1;
            if (j >= ld.lo && j < ld.n && base + lane < G::KPW) {
              mine = cache_row(p.pages, ld.b, j);
              if (mine < 0 && p.status) atomicCAS(p.status, 0, IQ_ERR_ROUTE);
            }
#pragma unroll
            for (int pass = 0; pass < (G::KPW < 32 ? G::KPW : 32) / ROWS; ++pass) {
              const int r = ct / CPR + pass * ROWS;
              const int row = __shfl_sync(0xffffffffu, mine, r);
              const bool ok = row >= 0 && in_row;  // else zeros, and nothing is read
              const uint8_t* k = ok ? k0 + row * p.k_row : p.k;
              const uint8_t* v = ok ? v0 + row * p.v_row : p.v;
              const long long k_step = ok ? p.k_head : 0, v_step = ok ? p.v_head : 0;
              uint32_t dst = to + swizzled<G>(base + r, c % PIECES);
#pragma unroll
              for (int hd = 0; hd < G::HG; ++hd) {
                cp_async16(dst, k, ok);
                cp_async16(dst + G::HALF, v, ok);
                dst += G::HEAD;
                k += k_step;
                v += v_step;
              }
            }
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(
                           smem_u32(bar_full + kgr * G::MAX_STAGES + stage))
                       : "memory");
        }
        if (++stage == G::STAGES) {
          stage = 0;
          parity ^= 1;
        }
        if (i + 1 < i1) ld.next(p, prefix, lens, per);
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      return;
    }
    // A copy is a box of one page: box_rows rows of box_heads heads, of the keys or the values
    // of one ring.  A lane makes the same copy of every tile, and has its page read one tile
    // ahead.
    const int boxes = G::KPW / p.box_rows, groups = G::HG / p.box_heads;
    const int copies = 2 * G::BOXES * boxes * groups * G::KG;
    const int x = (lane >> 1) % G::BOXES, r = (lane >> 1) / G::BOXES, box = r % boxes;
    const int head = r / boxes % groups * p.box_heads, kgr = r / boxes / groups;
    const int key = kgr * G::KPW + box * p.box_rows;
    const uint32_t dst = smem_u32(ring) + kgr * G::STAGES * G::STAGE + (lane & 1) * G::HALF +
                         x * G::BOX + head * G::HEAD + box * p.box_rows * G::PITCH;
    auto look_up = [&]() -> int {                // -1 where the box holds no key of the unit
      const int j = ld.j + key;
      return j < ld.n && j + p.box_rows > ld.lo ? page_id(p.pages, ld.b, j) : -1;
    };
    const CUtensorMap* map = lane & 1 ? &p.v_map : &p.k_map;
    int id_next = lane < copies ? look_up() : -1, stage = 0;
    uint32_t parity = 1;
#pragma unroll 1
    for (int i = i0; i < i1; ++i) {
      bool ok = true;
      if (lane < G::KG) {
        ok = mbar_wait(bar_free + lane * G::MAX_STAGES + stage, parity);
        if (ok) mbar_arrive_expect_tx(bar_full + lane * G::MAX_STAGES + stage, G::STAGE);
      }
      if (!__all_sync(0xffffffffu, ok)) {        // the consumers gave up, or are stuck
        if (lane == 0 && p.status) atomicCAS(p.status, 0, IQ_ERR_PIPE_TIMEOUT);
        break;
      }
      if (lane < copies) {
        // a box without keys of the unit, or of a page outside the cache, is read past the
        // cache's end, which fills it with zeros; so are the last rows of a page that straddles
        // that end
        const int j = ld.j + key;
        int at = p.pages.capacity;
        if (j < ld.n && j + p.box_rows > ld.lo) {
          const int row = page_row(p.pages, id_next, j);
          if (row >= 0) at = row;
          if (p.pages.capacity - at < min(p.box_rows, ld.n - j) && p.status)
            atomicCAS(p.status, 0, IQ_ERR_ROUTE);
        }
        tma_3d_g2s(dst + stage * G::STAGE, map, x * G::PITCH, at, ld.h0 + head,
                   bar_full + kgr * G::MAX_STAGES + stage);
      }
      if (++stage == G::STAGES) {
        stage = 0;
        parity ^= 1;
      }
      if (i + 1 < i1) {
        ld.next(p, prefix, lens, per);
        if (lane < copies) id_next = look_up();
      }
    }
    // shared memory must outlive the copies: the last of each stage
    if (lane < G::KG)
      for (int s = 0; s < min(G::STAGES, i1 - i0); ++s) {
        const int rounds = (i1 - i0 - 1 - s) / G::STAGES;   // of this stage before its last
        mbar_wait(bar_full + lane * G::MAX_STAGES + s, rounds & 1);
      }
    return;
  }

  if (G::MOVE_REGS) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G::REGS_COMPUTE));

  auto sync_all = [&]() { named_bar_sync(1, G::CONSUMERS); };
  constexpr int GT = 32 * G::WR;
  const int gtid = wr * 32 + lane;
  const uint32_t ring_g = smem_u32(ring) + kg * G::STAGES * G::STAGE + hg * G::HEAD;
  uint64_t* full = bar_full + kg * G::MAX_STAGES;
  uint64_t* free_ = bar_free + kg * G::MAX_STAGES;

  // ---- rows of empty sequences: some CTAs a sequence, 16 bytes a store
  {
    const int team = max(1, static_cast<int>(gridDim.x) / p.batch);
#pragma unroll 1
    for (int b = cta / team; b < p.batch; b += (gridDim.x + team - 1) / team) {
      if (prefix[b + 1] != prefix[b]) continue;
      for (int u = tid; u < per; u += G::CONSUMERS) p.units[b * per + u] = make_int2(0, 0);
      const int pieces = p.dim / 8, heads = p.q_len * p.q_heads;
#pragma unroll 1
      for (int i = cta % team * G::CONSUMERS + tid; i < heads * pieces; i += team * G::CONSUMERS) {
        const int th = i / pieces, d = i - th * pieces, tok = th / p.q_heads, head = th - tok * p.q_heads;
        *reinterpret_cast<uint4*>(p.out + b * p.o_b + tok * p.o_r + head * p.o_h + d * 8) =
            make_uint4(0, 0, 0, 0);
        if (d == 0) {
          const long long o = static_cast<long long>(b) * heads + th;
          if (p.lse) p.lse[o] = -INFINITY;
          if (p.lse2) p.lse2[o] = -INFINITY;
        }
      }
    }
  }
  if (i0 >= i1) return;
  Walk<G> it;
  bool from_start = it.start(p, prefix, lens, per, i0) == 0;   // the segment begins where its unit begins

  // ---- state of the unit being computed
  uint32_t qf[G::QS ? 1 : G::NBW][G::QREG];
  uint32_t* q_mine = q_smem + ((hg * G::WR + wr) * G::NBW) * G::QREG * 32 + 2 * lane;   // [nb][reg / 2][lane][2]
  float xs[G::NBW][2];                           // score factor of this lane's two columns
  // m: the reference the weights are relative to; mu: the same, 0 while there is none; thr:
  // how far above it a score may lie before the reference moves
  float m[G::NBW][2], mu[G::NBW][2], thr[G::NBW][2], l[G::NBW][2], acc[G::NBW][G::MT][4];
  int last_key[G::NBW][2];

  // The reference only has to keep the weights inside their type's range, so it follows the
  // maximum lazily: it moves when a score lies more than kLimit above it, to kShift below
  // that score.  Half precision (e4m3 caches): weights up to 2^15; what is 2^-22 of the
  // largest starts to lose bits.  bf16 has fp32's range.
  constexpr float kShift = G::KV == IQ_ACT_BF16 ? 0.f : 8.f;
  constexpr float kLimit = G::KV == IQ_ACT_BF16 ? 8.f : 15.f;
  const int key_lo = key_of<G>(g);               // this lane's keys of a tile of 16: key_lo, + 8
  // Where this lane's fragment loads of a tile start; the others lie at fixed distances, or
  // (other pieces of a swizzled row) at the address with a constant xored in.  bf16: ldmatrix
  // of the keys (matrices: keys 0-7, 8-15, then their next eight channels) and transposed of
  // the values (channels 0-7, 8-15 of keys 0-7, then of keys 8-15).  e4m3: 16 bytes (values at
  // D = 64: 8) of a row a load.
  uint32_t k_lane, v_lane, v_odd = 0;
  if (G::KV == IQ_ACT_BF16) {
    k_lane = ring_g + swizzled<G>(lane & 15, lane >> 4);
    v_lane = ring_g + G::HALF + swizzled<G>((lane & 7) + (lane >> 4) * 8, lane >> 3 & 1);
  } else {
    k_lane = ring_g + swizzled<G>(key_lo, t);
    const int c = G::DP >= 128 ? g : g >> 1, in = G::DP >= 128 ? 0 : (g & 1) * 8;
    v_lane = ring_g + G::HALF + swizzled<G>(key_of<G>(2 * t), c) + in;
    v_odd = swizzled<G>(key_of<G>(2 * t + 1), c) - swizzled<G>(key_of<G>(2 * t), c);
  }

  bool fresh = true, dead = false;
  int seg_key = 0;                               // the segment's first key
  int slot = 0;
  uint32_t parity = 0;

#pragma unroll 1
  for (int i = i0; i < i1; ++i) {
    const int h = it.h0 + hg, r0 = it.r0;
    if (fresh) {
      fresh = false;
      seg_key = it.j;
      if (from_start && tid == 0) p.units[it.b * per + it.hb].x = cta;
#pragma unroll
      for (int nb = 0; nb < G::NBW; ++nb) {
        // the last key each of this lane's two columns sees
        const int rc = r0 + (wr * G::NBW + nb) * 8 + 2 * t;
#pragma unroll
        for (int y = 0; y < 2; ++y)
          last_key[nb][y] = it.n - p.q_len + (p.q_len == 1 ? 0 : min((rc + y) / p.group, p.q_len - 1));
      }
      auto load_q = [&](int nb, uint32_t(&qr)[G::QREG]) {
        const int r = r0 + (wr * G::NBW + nb) * 8 + g;
        const bool live = r < p.rows_all;
        const int tok = live && p.q_len > 1 ? r / p.group : 0, head = h * p.group + (live ? r - tok * p.group : 0);
        const __nv_bfloat16* src = p.q + it.b * p.q_b + tok * p.q_r + head * p.q_h;
        if (G::KV == IQ_ACT_BF16) {
          // fragment order of the MMA: registers 2i, 2i+1 are channels 16i + 2t, 16i + 8 + 2t
#pragma unroll
          for (int x = 0; x < G::QREG; ++x) {
            const int d = x * 8 + 2 * t;
            qr[x] = live && d < p.dim ? *reinterpret_cast<const uint32_t*>(src + d) : 0u;
          }
        } else {
          // lane t holds channels 64 k + 16 t .. + 15
#pragma unroll
          for (int x = 0; x < G::QREG; x += 4) {
            const int d = (x / 8) * 64 + t * 16 + (x % 8) * 2;
            uint4 w = make_uint4(0, 0, 0, 0);
            if (live && d < p.dim) w = *reinterpret_cast<const uint4*>(src + d);
            qr[x] = w.x; qr[x + 1] = w.y; qr[x + 2] = w.z; qr[x + 3] = w.w;
          }
        }
      };
      if (!G::QS)
#pragma unroll
        for (int nb = 0; nb < G::NBW; ++nb) load_q(nb, qf[G::QS ? 0 : nb]);
#pragma unroll
      for (int nb = 0; nb < G::NBW; ++nb) {
        uint32_t(&qr)[G::QREG] = qf[G::QS ? 0 : nb];
        if (G::QS) load_q(nb, qr);
        if (G::KV == IQ_ACT_BF16) {
          xs[nb][0] = xs[nb][1] = p.scale_log2;
        } else {
          // bf16 values scaled by a power of two so that the row's largest lies in [1, 2): of
          // eight significant bits, so exact in half precision (steps of 2^-24) down to 2^-17;
          // smaller ones are rounded to that step, off by at most 2^-25
          float big = 0.f;
#pragma unroll
          for (int x = 0; x < G::QREG; ++x)
            big = fmaxf(big, fmaxf(fabsf(__uint_as_float(qr[x] << 16)),
                                   fabsf(__uint_as_float(qr[x] & 0xffff0000u))));
          big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
          big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
          int e = static_cast<int>(__float_as_uint(big) >> 23) - 127;
          if (big == 0.f || e > 127) e = 0;
          e = max(-126, min(126, e));
          const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
          const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
          for (int x = 0; x < G::QREG; ++x)
            qr[x] = pack_f16(__uint_as_float(qr[x] << 16) * down,
                             __uint_as_float(qr[x] & 0xffff0000u) * down);
          const float f = p.scale_log2 * up;
          xs[nb][0] = __shfl_sync(0xffffffffu, f, (2 * t) * 4);
          xs[nb][1] = __shfl_sync(0xffffffffu, f, (2 * t + 1) * 4);
        }
        if (G::QS && kg == 0)
#pragma unroll
          for (int x = 0; x < G::QREG; x += 2)
            *reinterpret_cast<uint2*>(q_mine + (nb * G::QREG + x) * 32) = make_uint2(qr[x], qr[x + 1]);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          m[nb][c] = -INFINITY;
          mu[nb][c] = 0.f;
          thr[nb][c] = -INFINITY;
          l[nb][c] = 0.f;
        }
#pragma unroll
        for (int x = 0; x < G::MT; ++x)
          acc[nb][x][0] = acc[nb][x][1] = acc[nb][x][2] = acc[nb][x][3] = 0.f;
      }
      if (G::QS) sync_all();
    }

    const int j0 = it.j + kg * G::KPW;
    // some key of these is not seen by every row
    const int lo_all = p.window ? max(0, it.n - p.window) : 0, hi_all = max(it.n - p.q_len + 1, 0);
    const bool partial = j0 < lo_all || j0 + G::KPW > hi_all;
    const uint32_t sv = ring_g + slot * G::STAGE + G::HALF;
    if (!dead && __any_sync(0xffffffffu, !mbar_wait(full + slot, parity))) {
      dead = true;                               // (the whole warp: it waits no more)
      if (lane == 0 && p.status) atomicCAS(p.status, 0, IQ_ERR_PIPE_TIMEOUT);
    }
    if (partial) {
      // values outside the unit: zeros; values that only some rows see: finite ones stay
      constexpr int PIECES = G::PITCH / 16;
#pragma unroll 1
      for (int x = gtid; x < G::KPW * PIECES; x += GT) {
        const int j = j0 + x / PIECES;
        if (j >= lo_all && j < hi_all) continue;
#pragma unroll
        for (int box = 0; box < G::BOXES; ++box) {
          const uint32_t at = sv + box * G::BOX + x * 16;
          uint4 w = make_uint4(0, 0, 0, 0);
          if (j >= it.lo && j < it.n) {
            w = lds128(at);
            if (!strip<G::KV>(w)) continue;
            *not_finite = 1;
          }
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(w.x), "r"(w.y),
                       "r"(w.z), "r"(w.w)
                       : "memory");
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      if (G::WR == 1) __syncwarp();
      else named_bar_sync(2 + warp / G::WR, GT);
    }

    // The tiles of sixteen keys, SUBI at a time.  EDGE: some row does not see some key; SCORES:
    // the scores may be kept.  With neither, nearly all tiles', there is no branch but the
    // reference's.
    auto tiles = [&](auto edge, auto keep) {
      constexpr bool EDGE = decltype(edge)::value, SCORES = decltype(keep)::value;
#pragma unroll 1
      for (int s0 = 0; s0 < G::SUB; s0 += G::SUBI) {
        if (EDGE && (j0 + s0 * 16 >= it.n || j0 + (s0 + G::SUBI) * 16 <= it.lo)) continue;
        const uint32_t tk = k_lane + slot * G::STAGE + s0 * 16 * G::PITCH;
        const uint32_t tv = v_lane + slot * G::STAGE + s0 * 16 * G::PITCH;
        float sc[G::SUBI][G::NBW][4];
#pragma unroll
        for (int sub = 0; sub < G::SUBI; ++sub)
#pragma unroll
          for (int nb = 0; nb < G::NBW; ++nb)
            sc[sub][nb][0] = sc[sub][nb][1] = sc[sub][nb][2] = sc[sub][nb][3] = 0.f;
        // ---- S^T = K Q^T (the tiles interleaved: independent sums)
        auto q_frag = [&](int nb, int x) {       // registers 2x, 2x + 1
          if (!G::QS) return make_uint2(qf[nb][2 * x], qf[nb][2 * x + 1]);
          return lds64(smem_u32(q_mine + (nb * G::QREG + 2 * x) * 32));
        };
        if (G::KV == IQ_ACT_BF16) {
#pragma unroll
          for (int x = 0; x < G::MT; ++x) {
            uint2 b[G::NBW];
#pragma unroll
            for (int nb = 0; nb < G::NBW; ++nb) b[nb] = q_frag(nb, x);
#pragma unroll
            for (int sub = 0; sub < G::SUBI; ++sub) {
              uint32_t a[4];
              ldmatrix_x4(a, (tk ^ (x % 4 * 32)) + x / 4 * G::BOX + sub * 16 * G::PITCH);
#pragma unroll
              for (int nb = 0; nb < G::NBW; ++nb)
                mma_k16<G::KV>(sc[sub][nb], a[0], a[1], a[2], a[3], b[nb].x, b[nb].y);
            }
          }
        } else {
#pragma unroll
          for (int kk = 0; kk < G::DP / 64; ++kk) {
            const uint32_t box = (tk ^ (kk % 2 * 64)) + kk / 2 * G::BOX;
            uint32_t wl[G::SUBI][4], wh[G::SUBI][4];
#pragma unroll
            for (int sub = 0; sub < G::SUBI; ++sub) {
              const uint4 lo = lds128(box + sub * 16 * G::PITCH);
              const uint4 hi = lds128(box + (sub * 16 + 8) * G::PITCH);
              wl[sub][0] = lo.x; wl[sub][1] = lo.y; wl[sub][2] = lo.z; wl[sub][3] = lo.w;
              wh[sub][0] = hi.x; wh[sub][1] = hi.y; wh[sub][2] = hi.z; wh[sub][3] = hi.w;
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              uint2 b[G::NBW];
#pragma unroll
              for (int nb = 0; nb < G::NBW; ++nb) b[nb] = q_frag(nb, kk * 4 + x);
#pragma unroll
              for (int sub = 0; sub < G::SUBI; ++sub) {
                const uint32_t a0 = e4m3x2_to_f16x2(wl[sub][x]), a2 = e4m3x2_to_f16x2(wl[sub][x] >> 16);
                const uint32_t a1 = e4m3x2_to_f16x2(wh[sub][x]), a3 = e4m3x2_to_f16x2(wh[sub][x] >> 16);
#pragma unroll
                for (int nb = 0; nb < G::NBW; ++nb)
                  mma_k16<G::KV>(sc[sub][nb], a0, a1, a2, a3, b[nb].x, b[nb].y);
              }
            }
          }
        }
        // ---- softmax of this lane's columns (query rows 2t, 2t+1) and two keys a tile
        const int jt = j0 + s0 * 16 + key_lo;
        float x[G::NBW][G::SUBI][4];
        auto masked = [&](int nb) {              // -infinity for what this lane's rows do not see
          if constexpr (EDGE) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int to = last_key[nb][y], from = p.window ? to - p.window : -1;
#pragma unroll
              for (int sub = 0; sub < G::SUBI; ++sub)
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                  const int key = jt + sub * 16 + z * 8;
                  if (key <= from || key > to) x[nb][sub][2 * z + y] = -INFINITY;
                }
            }
          }
        };
        if (SCORES && (!EDGE || p.scores)) {
#pragma unroll
          for (int nb = 0; nb < G::NBW; ++nb) {
            const int r = r0 + (wr * G::NBW + nb) * 8 + 2 * t;
            if (r >= p.rows_pad) continue;
#pragma unroll
            for (int sub = 0; sub < G::SUBI; ++sub)
#pragma unroll
              for (int y = 0; y < 4; ++y) x[nb][sub][y] = sc[sub][nb][y] * xs[nb][y & 1];
            masked(nb);
#pragma unroll
            for (int sub = 0; sub < G::SUBI; ++sub) {
              const int j = jt + sub * 16;
              float* dst = p.scores +
                           ((static_cast<long long>(it.b) * p.kv_heads + h) * p.score_rows + j) *
                               p.rows_pad + r;
              const float(&z)[4] = x[nb][sub];
              if (!EDGE || (j >= it.lo && j < it.n)) *reinterpret_cast<float2*>(dst) = make_float2(z[0], z[1]);
              if (!EDGE || (j + 8 >= it.lo && j + 8 < it.n))
                *reinterpret_cast<float2*>(dst + 8 * p.rows_pad) = make_float2(z[2], z[3]);
            }
          }
        }
        float top[G::NBW][2];
        bool above = false;
        auto shifted = [&](int nb) {
#pragma unroll
          for (int sub = 0; sub < G::SUBI; ++sub)
#pragma unroll
            for (int y = 0; y < 4; ++y)
              x[nb][sub][y] = fmaf(sc[sub][nb][y], xs[nb][y & 1], -mu[nb][y & 1]);
          masked(nb);
        };
#pragma unroll
        for (int nb = 0; nb < G::NBW; ++nb) {
          shifted(nb);
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            top[nb][y] = fmaxf(x[nb][0][y], x[nb][0][y + 2]);
#pragma unroll
            for (int sub = 1; sub < G::SUBI; ++sub)
              top[nb][y] = fmaxf(top[nb][y], fmaxf(x[nb][sub][y], x[nb][sub][y + 2]));
            above |= top[nb][y] > thr[nb][y];
          }
        }
        if (__any_sync(0xffffffffu, above)) {    // the references move
#pragma unroll
          for (int nb = 0; nb < G::NBW; ++nb) {
            float c[2];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              float best = top[nb][y] + mu[nb][y];
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
              best = fmaxf(best - kShift, m[nb][y]);
              const float u = best == -INFINITY ? 0.f : best;
              c[y] = ex2(m[nb][y] - u);
              m[nb][y] = best;
              mu[nb][y] = u;
              thr[nb][y] = best == -INFINITY ? -INFINITY : kLimit;
              l[nb][y] *= c[y];
            }
#pragma unroll
            for (int y = 0; y < G::MT; ++y) {
              acc[nb][y][0] *= c[0];
              acc[nb][y][1] *= c[1];
              acc[nb][y][2] *= c[0];
              acc[nb][y][3] *= c[1];
            }
            shifted(nb);
          }
        }
        uint32_t pb[G::SUBI][G::NBW][2];
#pragma unroll
        for (int sub = 0; sub < G::SUBI; ++sub) {
#pragma unroll
          for (int nb = 0; nb < G::NBW; ++nb) {
            float(&z)[4] = x[nb][sub];
#pragma unroll
            for (int y = 0; y < 4; ++y) z[y] = ex2(z[y]);
            // the normaliser adds the weights as computed; the products below take them
            // rounded to the MMA's type (half: 2^-11, bf16: 2^-8 relative at most)
            l[nb][0] += z[0] + z[2];
            l[nb][1] += z[1] + z[3];
            if (G::KV == IQ_ACT_BF16) {
              pb[sub][nb][0] = transpose8x8(pack_bf16(z[0], z[1]));
              pb[sub][nb][1] = transpose8x8(pack_bf16(z[2], z[3]));
            } else {
              pb[sub][nb][0] = transpose8x8(pack_f16(z[0], z[1]));
              pb[sub][nb][1] = transpose8x8(pack_f16(z[2], z[3]));
            }
          }
        }
        // ---- O^T += V^T P^T
#pragma unroll
        for (int sub = 0; sub < G::SUBI; ++sub) {
          if (G::KV == IQ_ACT_BF16) {
#pragma unroll
            for (int x_ = 0; x_ < G::MT; ++x_) {
              uint32_t a[4];
              ldmatrix_x4_trans(a, (tv ^ (x_ % 4 * 32)) + x_ / 4 * G::BOX + sub * 16 * G::PITCH);
#pragma unroll
              for (int nb = 0; nb < G::NBW; ++nb)
                mma_k16<G::KV>(acc[nb][x_], a[0], a[1], a[2], a[3], pb[sub][nb][0], pb[sub][nb][1]);
            }
          } else {
            // lane g holds channels 128 dd + 16 g .. + 15 (8 g .. + 7 for D = 64) of the keys
            // in rows 2t, 2t+1, 2t+8, 2t+9; pairs of keys are interleaved bytewise, then widened
            constexpr int WORDS = G::DP >= 128 ? 4 : 2;
#pragma unroll
            for (int dd = 0; dd < (G::DP + 127) / 128; ++dd) {
              uint32_t v[4][WORDS];
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                const uint32_t at = (y & 1 ? tv + v_odd : tv) + dd * G::BOX + (sub * 16 + (y >> 1) * 8) * G::PITCH;
                if (G::DP >= 128) {
                  const uint4 w = lds128(at);
                  v[y][0] = w.x; v[y][1] = w.y; v[y][WORDS - 2] = w.z; v[y][WORDS - 1] = w.w;
                } else {
                  const uint2 w = lds64(at);
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
                  const int x_ = dd * 8 + 2 * w + half;
#pragma unroll
                  for (int nb = 0; nb < G::NBW; ++nb)
                    mma_k16<G::KV>(acc[nb][x_], a0, a1, a2, a3, pb[sub][nb][0], pb[sub][nb][1]);
                }
              }
            }
          }
        }
      }
    };
    if (!partial) {
      if (p.scores) tiles(std::false_type{}, std::true_type{});
      else tiles(std::false_type{}, std::false_type{});
    } else if (j0 < it.n && j0 + G::KPW > it.lo) {
      tiles(std::true_type{}, std::true_type{});
    }

    // the stage is free: one arrival a warp that reads it
    __syncwarp();
    if (lane == 0) mbar_arrive(free_ + slot);
    if (++slot == G::STAGES) {
      slot = 0;
      parity ^= 1;
    }

    const bool unit_end = it.left == 1;
    if (unit_end || i == i1 - 1) {
      // ---- the unit ends here, or the share does: join the warps' keys
#pragma unroll
      for (int nb = 0; nb < G::NBW; ++nb) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) l[nb][c] += __shfl_xor_sync(0xffffffffu, l[nb][c], o);
        if constexpr (G::KG > 1)
#pragma unroll 1
        for (int half = G::KG / 2; half >= 1; half >>= 1) {
          float* mine = join + ((((kg & (half - 1)) * G::HG + hg) * G::WR + wr) * G::NREG) * 32 + 4 * lane;
          constexpr int MX = G::MT / G::XP;
          float f[2], e[2];
#pragma unroll
          for (int part = 0; part < G::XP; ++part) {
            if (kg >= half && kg < 2 * half) {
              if (part == 0)
                *reinterpret_cast<float4*>(mine) = make_float4(m[nb][0], m[nb][1], l[nb][0], l[nb][1]);
#pragma unroll
              for (int x = 0; x < MX; ++x) {
                const float(&a)[4] = acc[nb][part * MX + x];
                *reinterpret_cast<float4*>(mine + 128 * (x + 1)) = make_float4(a[0], a[1], a[2], a[3]);
              }
            }
            sync_all();
            if (kg < half) {
              if (part == 0) {
                const float4 o4 = *reinterpret_cast<const float4*>(mine);
                const float om[2] = {o4.x, o4.y}, ol[2] = {o4.z, o4.w};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                  const float top = fmaxf(m[nb][c], om[c]), u = top == -INFINITY ? 0.f : top;
                  f[c] = ex2(m[nb][c] - u);
                  e[c] = ex2(om[c] - u);
                  m[nb][c] = top;
                  l[nb][c] = l[nb][c] * f[c] + ol[c] * e[c];
                }
              }
#pragma unroll
              for (int x = 0; x < MX; ++x) {
                const float4 v = *reinterpret_cast<const float4*>(mine + 128 * (x + 1));
                float(&a)[4] = acc[nb][part * MX + x];
                a[0] = a[0] * f[0] + v.x * e[0];
                a[1] = a[1] * f[1] + v.y * e[1];
                a[2] = a[2] * f[0] + v.z * e[0];
                a[3] = a[3] * f[1] + v.w * e[1];
              }
            }
            sync_all();
          }
        }
      }
      const bool whole = unit_end && from_start;
      const int slot_out = 2 * cta + (from_start ? 1 : 0);
      if (unit_end && tid == 0) p.units[it.b * per + it.hb].y = cta;
      if (kg == 0) {
#pragma unroll
        for (int nb = 0; nb < G::NBW; ++nb) {
          const int block = wr * G::NBW + nb;    // rows 8 block .. + 7 of the unit
          float inv[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            inv[c] = l[nb][c] > 0.f ? 1.f / l[nb][c] : (l[nb][c] == 0.f ? 0.f : l[nb][c]);
            const int r = r0 + block * 8 + 2 * t + c;
            if (g != 0 || r >= p.rows_all) continue;
            if (whole) {
              const float z = l[nb][c] > 0.f ? m[nb][c] + log2f(l[nb][c])
                                             : (l[nb][c] == 0.f ? -INFINITY : l[nb][c]);
              const int tok = r / p.group, head = h * p.group + r - tok * p.group;
              const long long at = (static_cast<long long>(it.b) * p.q_len + tok) * p.q_heads + head;
              if (p.lse) p.lse[at] = z * kLn2;
              if (p.lse2) p.lse2[at] = z;
            } else {
              p.part_ml[(static_cast<size_t>(slot_out) * G::HG + hg) * G::RB + block * 8 + 2 * t + c] =
                  make_float2(m[nb][c], l[nb][c]);
            }
          }
          if (!whole) {                          // fragments as they are
            float4* dst = reinterpret_cast<float4*>(p.part) +
                          ((static_cast<size_t>(slot_out) * G::HG + hg) * (G::RB / 8) + block) * G::MT * 32 + lane;
#pragma unroll
            for (int x = 0; x < G::MT; ++x)
              dst[x * 32] = make_float4(acc[nb][x][0], acc[nb][x][1], acc[nb][x][2], acc[nb][x][3]);
          } else if (G::KV == IQ_ACT_BF16) {
            // transposed back: lane (g, t) writes channels 2t, 2t + 1 of row g of each 8 x 8
            const int r = r0 + block * 8 + g, tok = r / p.group, head = h * p.group + r - tok * p.group;
            __nv_bfloat16* o = p.out + it.b * p.o_b + tok * p.o_r + head * p.o_h + 2 * t;
#pragma unroll
            for (int x = 0; x < G::MT; ++x) {
              const uint32_t lo = transpose8x8(pack_bf16(acc[nb][x][0] * inv[0], acc[nb][x][1] * inv[1]));
              const uint32_t hi = transpose8x8(pack_bf16(acc[nb][x][2] * inv[0], acc[nb][x][3] * inv[1]));
              if (r < p.rows_all && 16 * x < p.dim) {
                *reinterpret_cast<uint32_t*>(o + 16 * x) = lo;
                *reinterpret_cast<uint32_t*>(o + 16 * x + 8) = hi;
              }
            }
          } else {
            // lane (g, t) holds runs of 16 (D = 64: 8) channels of rows 2t and 2t + 1
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int r = r0 + block * 8 + 2 * t + c;
              if (r >= p.rows_all) continue;
              const int tok = r / p.group, head = h * p.group + r - tok * p.group;
              __nv_bfloat16* o = p.out + it.b * p.o_b + tok * p.o_r + head * p.o_h;
#pragma unroll
              for (int x = 0; x < G::MT; x += 4) {
                const int d = channel_of<G>(x, 0, g);
                uint4 w;
                w.x = pack_bf16(acc[nb][x][c] * inv[c], acc[nb][x][2 + c] * inv[c]);
                w.y = pack_bf16(acc[nb][x + 1][c] * inv[c], acc[nb][x + 1][2 + c] * inv[c]);
                w.z = pack_bf16(acc[nb][x + 2][c] * inv[c], acc[nb][x + 2][2 + c] * inv[c]);
                w.w = pack_bf16(acc[nb][x + 3][c] * inv[c], acc[nb][x + 3][2 + c] * inv[c]);
                if (d < p.dim) *reinterpret_cast<uint4*>(o + d) = w;
              }
            }
          }
        }
      }
      if (p.q_len > 1) {
        sync_all();
        if (*not_finite) {
          add_not_finite<G>(p, it.b, it.n, it.h0, r0, seg_key, it.j + G::TK, whole, slot_out);
          sync_all();
          if (tid == 0) *not_finite = 0;
        }
      }
      if (G::KG > 1 || G::QS || p.q_len > 1) sync_all();   // the shared buffers are free again
      fresh = true;
      from_start = true;
    }
    it.next(p, prefix, lens, per);
  }
}

// ------------------------------------------------------------------------------------
// Adds the partial results of the units that several CTAs shared: slot 2c + 1 of the first
// CTA, slot 2c of the others, in that order.  A block joins eight query rows of a head, a
// thread the four values of one lane of an m-tile; WIDE (many partial results a unit): a
// block joins one m-tile, its eight warps every eighth partial result.  It is all latency
// (the unit's place, then its partial results), so a thread has all its loads in flight at
// once, those of the maxima and sums among them.  Measured: 5 to 6 us alone with
// cold caches, most of it hidden behind the split kernel's end; a join by the unit's last CTA inside the split kernel saved the
// launch and lost more (9.0 -> 11.6 us a call at a window of 4096 keys, 147 -> 160 for the
// ragged batch), being serial in one CTA.
constexpr int kJoinThreads = 256;
constexpr int kJoinParts = 160;                  // partial results of a unit, at most (one a CTA)

// weights[b, h, j] += sum over the head's query rows of 2^(x_j - lse2): a thread a key, on the
// scores the split kernel left behind (L2 holds most of them).  Each block works out the rows'
// lse2 from the partial results for itself, so these blocks need not wait for those that join.
// The step's own rows are set, not added to, and get their positions; a sequence that had no room
// for them (slot < 0) keeps its weights and positions.  64 / 8 heads over 32768
// keys of e4m3: 26.6 us with the weights, 8 MB of scores written and read once more.
constexpr int kWeightKeys = 1024;                // keys a block (512: 27.5 us; 81.9 over 128k, 1024 74.6)

template <class G>
__device__ __forceinline__ void add_weights(const AttnParams& p, int chunk, int bh, float* z /* [512] */) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = bh / p.kv_heads, h = bh - b * p.kv_heads;
  if (p.slot && __ldg(p.slot + static_cast<long long>(b) * p.q_len) < 0) return;
  const SeqSpan s = seq_span(clamp_length(p, b, false), p.q_len, p.window);
  const int from = max(s.lo, chunk * kWeightKeys), to = min(s.n, (chunk + 1) * kWeightKeys);
  if (from >= to) return;
  for (int r = warp; r < p.rows_pad; r += kJoinThreads / 32) {
    float v = INFINITY;                          // a padded or empty row adds nothing
    if (r < p.rows_all) {
      const int rb = r / G::RB;
      const int2 c = __ldcg(p.units + (static_cast<long long>(b) * (p.kv_heads / G::HG) + h / G::HG) * p.n_rb + rb);
      const int n = c.y - c.x + 1;
      if (n <= 1) {
        const int tok = r / p.group, head = h * p.group + r - tok * p.group;
        v = __ldcg(p.lse2 + (static_cast<long long>(b) * p.q_len + tok) * p.q_heads + head);
      } else {
        float2 ml[kJoinParts / 32];
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int i = 0; i < kJoinParts / 32; ++i) {
          const int k = lane + 32 * i;
          ml[i] = make_float2(-INFINITY, 0.f);
          if (k < n)
            ml[i] = __ldcg(p.part_ml + (static_cast<size_t>(2 * (c.x + k) + (k == 0 ? 1 : 0)) * G::HG + h % G::HG) *
                                           G::RB + r % G::RB);
          top = fmaxf(top, ml[i].x);
        }
        top = warp_max(top);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int i = 0; i < kJoinParts / 32; ++i) sum += ex2(ml[i].x - base) * ml[i].y;
        sum = warp_sum(sum);
        v = sum > 0.f ? top + log2f(sum) : (sum == 0.f ? -INFINITY : sum);
      }
      if (v == -INFINITY) v = INFINITY;
    }
    if (lane == 0) z[r] = v;
  }
  __syncthreads();
  // a thread's four keys are all in flight
  constexpr int EACH = kWeightKeys / kJoinThreads;
  const long long row = static_cast<long long>(b) * p.kv_heads + h;
  float w[EACH], old[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int j = chunk * kWeightKeys + tid + i * kJoinThreads;
    w[i] = old[i] = 0.f;
    if (j >= from && j < to && j < s.n - p.q_len) old[i] = p.weights[b * p.w_b + h * p.w_h + j];
  }
#pragma unroll 2
  for (int r = 0; r < p.rows_pad; r += 4) {
    float4 x[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int j = chunk * kWeightKeys + tid + i * kJoinThreads;
      if (j >= from && j < to)
        x[i] = __ldcg(reinterpret_cast<const float4*>(p.scores + (row * p.score_rows + j) * p.rows_pad + r));
    }
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const float zr = z[r + y];
      if (zr == INFINITY) continue;
#pragma unroll
      for (int i = 0; i < EACH; ++i) w[i] += ex2((y == 0 ? x[i].x : y == 1 ? x[i].y : y == 2 ? x[i].z : x[i].w) - zr);
    }
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int j = chunk * kWeightKeys + tid + i * kJoinThreads;
    if (j < from || j >= to) continue;
    p.weights[b * p.w_b + h * p.w_h + j] = old[i] + w[i];
    if (j >= s.n - p.q_len && p.positions)
      p.positions[b * p.p_b + h * p.p_h + j] = __ldg(p.seen + b) - s.n + j;
  }
}

template <class G, bool WIDE>
__global__ void __launch_bounds__(kJoinThreads) attn_join_kernel(const __grid_constant__ AttnParams p) {
  __shared__ float fac[8][kJoinParts];
  __shared__ float stat[8];
  __shared__ float4 red[8][32];
  constexpr int BATCH = WIDE ? kJoinParts / 8 : 8;   // loads of a thread in flight
  constexpr int EACH = kJoinParts / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int per = p.kv_heads / G::HG * p.n_rb;
  pdl_wait();
  pdl_launch_dependents();
  if (blockIdx.x >= p.joins) {
    const unsigned i = (blockIdx.z * gridDim.y + blockIdx.y) * (gridDim.x - p.joins) + blockIdx.x - p.joins;
    if (i < p.weight_blocks)
      add_weights<G>(p, i % p.weight_chunks, i / p.weight_chunks, reinterpret_cast<float*>(red));
    return;
  }
  const int u = blockIdx.x / G::HG, hg = blockIdx.x % G::HG;
  const int b = u / per, hb = u - b * per, h = hb / p.n_rb * G::HG + hg;
  const int block = blockIdx.y, r0 = hb % p.n_rb * G::RB + block * 8;
  const int2 c = __ldcg(p.units + u);
  const int n = c.y - c.x + 1;
  if (n <= 1 || r0 >= p.rows_all) return;
  auto slot_of = [&](int k) { return (2 * (c.x + k) + (k == 0 ? 1 : 0)) * G::HG + hg; };
  const float4* part = reinterpret_cast<const float4*>(p.part) + block * G::MT * 32 + lane;
  auto load = [&](int x, int k) {
    return __ldcg(part + static_cast<size_t>(slot_of(k)) * (G::RB / 8) * G::MT * 32 + x * 32);
  };
  const int step = WIDE ? 8 : 1, first = WIDE ? warp : 0;
  float4 v[BATCH];
  const int x0 = WIDE ? blockIdx.z : warp;
#pragma unroll
  for (int i = 0; i < BATCH; ++i)
    if (x0 < G::MT && first + i * step < n) v[i] = load(x0, first + i * step);
  // ---- warp w: row w's maximum, sum and each partial result's factor
  {
    const bool live = r0 + warp < p.rows_all;
    const float2* ml = p.part_ml + block * 8 + warp;
    float2 z[EACH];
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      z[i] = make_float2(-INFINITY, 0.f);
      if (live && lane + 32 * i < n) z[i] = __ldcg(&ml[static_cast<size_t>(slot_of(lane + 32 * i)) * G::RB]);
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) top = fmaxf(top, z[i].x);
    top = warp_max(top);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const float f = ex2(z[i].x - base);
      fac[warp][lane + 32 * i] = f;
      sum += f * z[i].y;
    }
    sum = warp_sum(sum);
    if (lane == 0) {
      stat[warp] = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
      if (live && (!WIDE || blockIdx.z == 0)) {
        const float y = sum > 0.f ? top + log2f(sum) : (sum == 0.f ? -INFINITY : sum);
        const int r = r0 + warp, tok = r / p.group, head = h * p.group + r - tok * p.group;
        const long long at = (static_cast<long long>(b) * p.q_len + tok) * p.q_heads + head;
        if (p.lse) p.lse[at] = y * kLn2;
        if (p.lse2) p.lse2[at] = y;
      }
    }
  }
  __syncthreads();
  auto put = [&](int x, float4 o) {
    const float val[2][2] = {{o.x, o.z}, {o.y, o.w}};
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int r = r0 + 2 * t + y;
      if (r >= p.rows_all) continue;
      const int tok = r / p.group, head = h * p.group + r - tok * p.group;
      __nv_bfloat16* dst = p.out + b * p.o_b + tok * p.o_r + head * p.o_h;
      const float inv = stat[2 * t + y];
      const int d0 = channel_of<G>(x, 0, g), d1 = channel_of<G>(x, 1, g);
      if (d0 < p.dim) dst[d0] = __float2bfloat16_rn(val[y][0] * inv);
      if (d1 < p.dim) dst[d1] = __float2bfloat16_rn(val[y][1] * inv);
    }
  };
#pragma unroll 1
  for (int x = x0; x < G::MT; x += WIDE ? G::MT : 8) {
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int k0 = first; k0 < n; k0 += BATCH * step) {
      if (x != x0 || k0 != first)
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
          if (k0 + i * step < n) v[i] = load(x, k0 + i * step);
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int k = k0 + i * step;
        if (k < n) {
          const float f0 = fac[2 * t][k], f1 = fac[2 * t + 1][k];
          o.x += f0 * v[i].x;
          o.y += f1 * v[i].y;
          o.z += f0 * v[i].z;
          o.w += f1 * v[i].w;
        }
      }
    }
    if (!WIDE) put(x, o);
    else red[warp][lane] = o;
  }
  if (!WIDE) return;
  __syncthreads();
  if (warp) return;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const float4 a = red[w][lane];
    o.x += a.x; o.y += a.y; o.z += a.z; o.w += a.w;
  }
  put(x0, o);
}

// ------------------------------------------------------------------------------------
// host side
// SMs of the current device, and which it is; 0 where that fails.
static int attn_sms(int* dev) {
  static std::atomic<int> per_device[64];
  if (cudaGetDevice(dev) != cudaSuccess || *dev < 0 || *dev >= 64) return 0;
  int n = per_device[*dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *dev) != cudaSuccess) return 0;
    per_device[*dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Per kernel and device, once: the opt-in to its shared memory, and (where registers move
// between its warps) that it was compiled for as many as they share.
template <class K>
static bool attn_ready(K kernel, std::atomic<uint64_t>& done, int dev, int smem, int regs) {
  const uint64_t bit = uint64_t{1} << dev;       // dev < 64, see attn_sms
  if (done.load(std::memory_order_acquire) & bit) return true;
  if (regs > 0) {
    cudaFuncAttributes at{};
    if (cudaFuncGetAttributes(&at, kernel) != cudaSuccess || at.numRegs < regs) return false;
  }
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return false;
  done.fetch_or(bit, std::memory_order_release);
  return true;
}

template <class K, class... Args>
static int attn_launch(K kernel, dim3 grid, int threads, int smem, void* stream, bool pdl,
                       const Args&... args) {
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
constexpr int kAttnMaxCtas = 160;                // CTAs of the split kernel, at most

// (64-byte rows are copied in boxes of two rows at least: a box starts on 128 bytes)
static int pad_dim(int d, int elt, int page) {
  return d <= 64 && (elt == 2 || page % 2 == 0) ? 64 : d <= 128 ? 128 : 256;
}
static int block_rows(int rows) { return rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

// Heads a unit.  Neighbouring heads' rows are one piece of DRAM: against one head a unit, four
// took a ragged bf16 batch (32 / 8 heads) from 205 to 150 us and 32 x 8192 rows of e4m3 from
// 135 to 91; eight leave as many more partial results to join (128k rows of e4m3: 54 us, four
// 51).  No more than the rings of the geometry that the rows take.
static int head_group(int kv_heads, int rb, int dim) {
  int g = dim > 128 ? (rb <= 16 ? 4 : rb <= 32 ? 2 : 1) : (rb <= 32 ? 4 : 2);
  while (kv_heads % g) g /= 2;
  return g;
}

static AttnWork attn_work(int batch, int q_len, int q_heads, int kv_heads, int dim, int rows,
                          bool weights) {
  const int all = q_heads / kv_heads * q_len;
  const int rb = block_rows(all), n_rb = (all + rb - 1) / rb, rows_cta = rb * head_group(kv_heads, rb, dim);
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  AttnWork w{};
  size_t at = 0;
  w.part = at;
  at += up(static_cast<size_t>(2 * kAttnMaxCtas) * rows_cta * (dim <= 128 ? 128 : 256) * 4);
  w.part_ml = at;
  at += up(static_cast<size_t>(2 * kAttnMaxCtas) * rows_cta * 8);
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

// The cache as (bytes of a head's row, rows, heads), in boxes of `pitch` bytes x box_rows x
// box_heads with the swizzle whose width the box has.  Encoded anew for every call (a few hundred
// nanoseconds on the host): nothing is kept by address.
static int attn_map(CUtensorMap* out, const void* base, const AttnParams& p, long long row,
                    long long head, int elt, int pitch) {
  typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                    const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                    const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                    CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<EncodeTiledFn> known{nullptr};
  EncodeTiledFn encode = known.load();
  if (!encode) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) !=
            cudaSuccess || q != cudaDriverEntryPointSuccess || !fn)
      return IQ_ERR_CUDA;
    encode = reinterpret_cast<EncodeTiledFn>(fn);
    known.store(encode);
  }
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(p.dim * elt),
                              static_cast<cuuint64_t>(p.pages.capacity),
                              static_cast<cuuint64_t>(p.kv_heads)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(p.pages.capacity > 1 ? row : p.dim * elt),
                                 static_cast<cuuint64_t>(p.kv_heads > 1 ? head : p.dim * elt)};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(pitch), static_cast<cuuint32_t>(p.box_rows),
                             static_cast<cuuint32_t>(p.box_heads)};
  const cuuint32_t ones[3] = {1, 1, 1};
  const CUresult r = encode(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims,
                            strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            pitch == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    fprintf(stderr, "iqb200: cuTensorMapEncodeTiled failed (%d)\n", static_cast<int>(r));
    return IQ_ERR_CUDA;
  }
  return IQ_OK;
}

template <class G>
static int attn_run(AttnParams& p, int n_sm, int dev, bool pdl, void* stream) {
  const long long tiles = static_cast<long long>(p.batch) * (p.kv_heads / G::HG) * p.n_rb *
                          ((p.max_rows + G::TK - 1) / G::TK + 2);
  if (tiles > 0x7fffffffLL) return IQ_ERR_UNSUPPORTED;
  int box = G::KPW;
  while (p.pages.page % box) box /= 2;
  p.box_rows = box;
  p.box_heads = box == G::KPW ? G::HG : 1;       // (a stage's heads lie KPW rows apart)
  // One warp issues the boxes, at some 60 ns each: past sixteen a tile the threads are faster
  // (pages of 16 rows, 128k rows of e4m3: 54 us against 58; pages of one row need 64 a head).
  // Boxes leave less to do per tile where there are few (4096 rows: 8.9 us against 11.4).
  p.gather = 2 * G::BOXES * (G::KPW / box) * (G::HG / p.box_heads) * G::KG > 16;
  static std::atomic<uint64_t> done{0};          // (a launch with fewer registers would wait for good)
  if (!attn_ready(attn_kernel<G>, done, dev, G::SMEM, G::MOVE_REGS ? G::REGS : 0)) return IQ_ERR_CUDA;
  int rc = IQ_OK;
  if (!p.gather) rc = attn_map(&p.k_map, p.k, p, p.k_row, p.k_head, G::ELT, G::PITCH);
  if (!p.gather && rc == IQ_OK) rc = attn_map(&p.v_map, p.v, p, p.v_row, p.v_head, G::ELT, G::PITCH);
  if (rc != IQ_OK) return rc;
  const int grid = static_cast<int>(tiles < n_sm ? tiles : n_sm);
  rc = attn_launch(attn_kernel<G>, dim3(grid), G::THREADS, G::SMEM, stream, pdl, p);
  if (rc != IQ_OK) return rc;
  const int heads = p.batch * p.kv_heads * p.n_rb;   // units x heads of a unit
  const int blocks = ((p.rows_all < G::RB ? p.rows_all : G::RB) + 7) / 8;
  // the CTAs that share a unit: from nine on its partial results are worth a block an m-tile
  const int wide = static_cast<long long>(grid) * G::HG > 8LL * heads;
  p.joins = static_cast<unsigned>(heads);
  p.weight_chunks = p.scores ? static_cast<unsigned>((p.max_rows + kWeightKeys - 1) / kWeightKeys) : 0;
  p.weight_blocks = p.weight_chunks * static_cast<unsigned>(p.batch * p.kv_heads);
  // the weights' blocks fill the grid's other axes too: empty blocks cost (64 / 8 heads over
  // 32k keys: 28.1 us with them, 26.6 without; over 128k 80.8 and 74.6)
  const unsigned layers = static_cast<unsigned>(blocks * (wide ? G::MT : 1));
  const unsigned x = p.joins + (p.weight_blocks + layers - 1) / layers;
  return wide ? attn_launch(attn_join_kernel<G, true>, dim3(x, blocks, G::MT), kJoinThreads, 0, stream,
                            true, p)
              : attn_launch(attn_join_kernel<G, false>, dim3(x, blocks), kJoinThreads, 0, stream, true, p);
}

// Sixteen rows a warp: their fragments of K and V are read and widened once.  Thirty-two (with
// q in shared memory) left too few registers: 67 us against 37 for 32 rows over 32k keys of
// e4m3, sixteen warps of eight rows 42.
template <int KV, int DP, int HG>
static int attn_pick_rows(AttnParams& p, int n_sm, int dev, bool pdl, void* stream) {
  if constexpr (DP <= 128) {
    if (p.rows_all <= 8) return attn_run<AttnGeo<KV, DP, 1, 1, HG, 8>>(p, n_sm, dev, pdl, stream);
    if (p.rows_all <= 16) return attn_run<AttnGeo<KV, DP, 2, 1, HG, 8>>(p, n_sm, dev, pdl, stream);
    if (p.rows_all <= 32) return attn_run<AttnGeo<KV, DP, 2, 2, HG, 8>>(p, n_sm, dev, pdl, stream);
    if constexpr (HG <= 2) return attn_run<AttnGeo<KV, DP, 2, 4, HG, 8>>(p, n_sm, dev, pdl, stream);
  } else {
    constexpr int W = KV == IQ_ACT_BF16 ? 4 : 8;     // (two stages of eight rings do not fit)
    if (p.rows_all <= 8) return attn_run<AttnGeo<KV, DP, 1, 1, HG, W>>(p, n_sm, dev, pdl, stream);
    if (p.rows_all <= 16) return attn_run<AttnGeo<KV, DP, 2, 1, HG, W>>(p, n_sm, dev, pdl, stream);
    if constexpr (HG <= 2) {
      if (p.rows_all <= 32) return attn_run<AttnGeo<KV, DP, 2, 2, HG, 8>>(p, n_sm, dev, pdl, stream);
    }
    if constexpr (HG == 1) return attn_run<AttnGeo<KV, DP, 2, 4, 1, 8>>(p, n_sm, dev, pdl, stream);
  }
  return IQ_ERR_UNSUPPORTED;
}

template <int KV, int DP>
static int attn_pick(AttnParams& p, int n_sm, int dev, bool pdl, void* stream) {
  switch (head_group(p.kv_heads, block_rows(p.rows_all), p.dim)) {
    case 4: return attn_pick_rows<KV, DP, 4>(p, n_sm, dev, pdl, stream);
    case 2: return attn_pick_rows<KV, DP, 2>(p, n_sm, dev, pdl, stream);
    default: return attn_pick_rows<KV, DP, 1>(p, n_sm, dev, pdl, stream);
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
  if ((a->positions != nullptr) != (a->seen != nullptr) || ((a->positions || a->slot) && !weights))
    return IQ_ERR_ARG;
  const AttnWork w = attn_work(a->batch, a->q_len, a->q_heads, a->kv_heads, a->head_dim,
                               static_cast<int>(rows), weights);
  if (a->work_bytes < w.total) return IQ_ERR_ARG;
  // 16-byte loads and stores
  const int64_t elt = a->kv_kind == IQ_ACT_BF16 ? 2 : 1;
  const uint64_t al = reinterpret_cast<uint64_t>(a->k_cache) | reinterpret_cast<uint64_t>(a->v_cache) |
                      static_cast<uint64_t>(a->k_row * elt) | static_cast<uint64_t>(a->k_head * elt) |
                      static_cast<uint64_t>(a->v_row * elt) | static_cast<uint64_t>(a->v_head * elt) |
                      reinterpret_cast<uint64_t>(a->work);
  if (al & 15) return IQ_ERR_ARG;
  const int64_t far = int64_t{1} << 40;          // a tensor map's strides, bytes
  for (const int64_t st : {a->k_row, a->k_head, a->v_row, a->v_head})
    if (st < 0 || st * elt >= far) return IQ_ERR_ARG;
  if (((reinterpret_cast<uint64_t>(a->q) | reinterpret_cast<uint64_t>(a->out)) & 15) ||
      ((a->q_b | a->q_r | a->q_h | a->o_b | a->o_r | a->o_h) & 7))
    return IQ_ERR_ARG;
  int dev = 0;
  const int n_sm = attn_sms(&dev);
  if (n_sm == 0 || n_sm > kAttnMaxCtas) return IQ_ERR_CUDA;

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
    p.slot = reinterpret_cast<const long long*>(a->slot);
  }
  const bool bf16 = a->kv_kind == IQ_ACT_BF16, pdl = a->pdl != 0;
  int rc;
  switch (pad_dim(a->head_dim, static_cast<int>(elt), a->page_size)) {
    case 64:
      rc = bf16 ? attn_pick<IQ_ACT_BF16, 64>(p, n_sm, dev, pdl, stream)
                : attn_pick<IQ_ACT_E4M3, 64>(p, n_sm, dev, pdl, stream);
      break;
    case 128:
      rc = bf16 ? attn_pick<IQ_ACT_BF16, 128>(p, n_sm, dev, pdl, stream)
                : attn_pick<IQ_ACT_E4M3, 128>(p, n_sm, dev, pdl, stream);
      break;
    default:
      rc = bf16 ? attn_pick<IQ_ACT_BF16, 256>(p, n_sm, dev, pdl, stream)
                : attn_pick<IQ_ACT_E4M3, 256>(p, n_sm, dev, pdl, stream);
  }
  return rc;
}
