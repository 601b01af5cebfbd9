// Bookkeeping of the paged key/value cache: eviction by accumulated attention weight
// (iq_kv_evict) and the next tokens' rows (iq_kv_advance).
//
// Eviction is a selection and a movement.  The selection finds the budget-th largest of a
// (sequence, head)'s weights exactly: order-preserving integers of the weights, histogram
// passes of 11, 11 and 10 bits (it stops at the pass whose bin is kept whole).  One cluster
// holds all of a head's weights in the shared memory of its CTAs, so global memory is read
// once; a pass costs a histogram of local words, one barrier and the sum of the CTAs' bins
// through distributed shared memory.  The movement fills the freed places below the budget
// with the kept rows above it: sources and destinations are disjoint, so it runs in place, in
// any order and on all SMs, and moves the fewest rows there are to move.
// What bounds it: latency (barriers, passes) for a step's few rows, HBM for a long prompt's.
// Measured (one B200, pages of 64, 8 heads, 128 channels of e4m3): one row of 4097 out: 10.3
// us; 32768 rows to 8192: 22.7 us, 0.19 of the copy rate, half of it the selection; 24 ragged
// sequences of bf16 to 2048 rows: 33 to 39 us with where the pages lie, 3.3 to 3.9 TB/s.
#include <math.h>
#include <stdio.h>

#include <mutex>
#include <unordered_set>

#include <cooperative_groups.h>

#include "paged.cuh"

namespace iqb {

namespace cg = cooperative_groups;

// Threads of a selecting CTA: the many for long sequences, the few (eight CTAs an SM) where a
// CTA of those holds all of a sequence's rows (65 x 16 heads of 256 rows: 39 us against 13).
constexpr int kEvictMany = 1024, kEvictFew = 256;
constexpr int kEvictChunk = 32768;               // weights a CTA of a cluster holds at most
constexpr int kEvictCluster = 8;
constexpr int kEvictRows = kEvictChunk * kEvictCluster;
constexpr int kMoveThreads = 256;
constexpr int kMovesInFlight = 2;
// Moves a (sequence, head) can have at most for the selecting cluster to make them itself.
constexpr int kEvictFusedMoves = 256;

struct EvictParams {
  uint8_t *k, *v;
  long long k_row, k_head, v_row, v_head;        // bytes
  PageTable pages;
  int max_rows;
  const int *lengths, *seen;
  const float* w;
  long long w_b, w_h;
  const int* pos;
  long long p_b, p_h;
  float* w_out;
  long long wo_b, wo_h;
  int* pos_out;
  long long po_b, po_h;
  int* lengths_out;
  int* count;                                    // [batch * kv_heads] moves
  int2* moves;                                   // [batch * kv_heads][move_rows] (to, from)
  int move_rows;
  int* status;
  int kv_heads, row_bytes, budget, keep_first, keep_last;
  int chunk;                                     // key words of shared memory a CTA has
  int fused;
};

__device__ __forceinline__ int evict_length(const EvictParams& p, int b, bool report) {
  const int n = __ldg(p.lengths + b);
  if (n < 0 || n > p.max_rows) {
    if (report && p.status) atomicCAS(p.status, 0, IQ_ERR_ROUTE);
    return n < 0 ? 0 : p.max_rows;
  }
  return n;
}

// Larger weight, larger word; +0 and -0 alike; NaN lowest.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (isnan(w)) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive sum of `x` over the block's threads in thread order; *all gets the total.
template <int T>
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t* sums /* [32] */, uint32_t* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto inclusive = [&](uint32_t v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += y;
    }
    return v;
  };
  const uint32_t incl = inclusive(x);
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  const uint32_t warps = inclusive(lane < T / 32 ? sums[lane] : 0);   // (every warp for itself)
  const uint32_t before = __shfl_sync(0xffffffffu, warps, warp ? warp - 1 : 0);
  *all = __shfl_sync(0xffffffffu, warps, 31);
  __syncthreads();                               // `sums` is free again
  return incl - x + (warp ? before : 0u);
}

// Moves [i0, i0 + step, ..) of `total`, a cache row of K and of V each, by groups of `width`
// threads (16 bytes a thread), two moves in flight a group: a move is a chain of its list
// entry, two page lookups and the row itself, and more moves in flight cost more in resident
// warps than they hide (24 x 8 heads, some 1500 of
// 256 bytes each: two 33 to 39 us with where the pages lie, four 45, one 43).
__device__ __forceinline__ void move_rows(const EvictParams& p, int b, int h, const int2* moves, int i0,
                                          int step, int total, int at, int width) {
  constexpr int U = kMovesInFlight;
#pragma unroll 1
  for (int i = i0; i < total; i += U * step) {
    int to[U], from[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      to[u] = from[u] = -1;
      if (i + u * step < total) {
        const int2 mv = __ldcg(moves + i + u * step);
        to[u] = cache_row(p.pages, b, mv.x);
        from[u] = cache_row(p.pages, b, mv.y);
        if ((to[u] < 0 || from[u] < 0) && p.status) atomicCAS(p.status, 0, IQ_ERR_ROUTE);
      }
    }
#pragma unroll 1
    for (int c = at * 16; c < p.row_bytes; c += width * 16) {
      uint4 k[U], v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (to[u] < 0 || from[u] < 0) continue;
        k[u] = *reinterpret_cast<const uint4*>(p.k + from[u] * p.k_row + h * p.k_head + c);
        v[u] = *reinterpret_cast<const uint4*>(p.v + from[u] * p.v_row + h * p.v_head + c);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (to[u] < 0 || from[u] < 0) continue;
        *reinterpret_cast<uint4*>(p.k + to[u] * p.k_row + h * p.k_head + c) = k[u];
        *reinterpret_cast<uint4*>(p.v + to[u] * p.v_row + h * p.v_head + c) = v[u];
      }
    }
  }
}

template <int T>
__global__ void __launch_bounds__(T) evict_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ uint32_t keys[];             // [chunk]
  __shared__ uint32_t hist[3][2048];
  __shared__ uint32_t sums[32];
  constexpr int WARPS = T / 32;
  __shared__ uint32_t places[T];     // a warp's flags in a round of keys; then what lies before
  __shared__ uint32_t equals[T];
  __shared__ uint32_t found[3];                  // the digit, what is needed inside it, and all it has
  __shared__ uint32_t counts[2];                 // this CTA's keys at the edge; free places | moved rows << 16
  cg::cluster_group cluster = cg::this_cluster();
  const int cs = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int unit = blockIdx.x / cs, b = unit / p.kv_heads, h = unit - b * p.kv_heads;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto sync = [&]() {
    if (cs == 1) __syncthreads();
    else cluster.sync();
  };

#pragma unroll
  for (int i = tid; i < 3 * 2048; i += T) hist[0][i] = 0;
  pdl_wait();
  pdl_launch_dependents();
  // This CTA's rows; their weights and positions are on their way before the length is known
  // (rows past it are inside the arrays).
  const int i0 = rank * p.chunk, end = min(p.max_rows, i0 + p.chunk) - i0;
  const float* w = p.w + b * p.w_b + h * p.w_h;
  const int* pos = p.pos + b * p.p_b + h * p.p_h;
  float* w_out = p.w_out + b * p.wo_b + h * p.wo_h;
  int* pos_out = p.pos_out + b * p.po_b + h * p.po_h;
  constexpr int AHEAD = 8;
  float wv[AHEAD];
  int pv[AHEAD];
#pragma unroll
  for (int x = 0; x < AHEAD; ++x) {
    const int i = tid + x * T;
    if (i < end) {
      wv[x] = w[i0 + i];
      pv[x] = pos[i0 + i];
    }
  }
  const int n = evict_length(p, b, h == 0 && rank == 0 && tid == 0);
  const int last = __ldg(p.seen + b) - p.keep_last;
  const int keep = min(n, p.budget), mine = max(0, min(n - i0, end));
  if (h == 0 && rank == 0 && tid == 0) p.lengths_out[b] = keep;
  // The keys, and (out of place) the copies of what may stay below the budget; the places
  // about to be filled get their old values too, before the moves below
  auto take = [&](int i, float x, int at) {
    keys[i] = at < p.keep_first || at >= last ? 0xffffffffu : weight_key(x);
    if (i0 + i < keep) {
      if (w_out != w) w_out[i0 + i] = x;
      if (pos_out != pos) pos_out[i0 + i] = at;
    }
  };
#pragma unroll
  for (int x = 0; x < AHEAD; ++x)
    if (tid + x * T < mine) take(tid + x * T, wv[x], pv[x]);
#pragma unroll 4
  for (int i = tid + AHEAD * T; i < mine; i += T) take(i, w[i0 + i], pos[i0 + i]);
  if (n <= p.budget) {                           // (the whole cluster)
    if (rank == 0 && tid == 0) p.count[unit] = 0;
    return;
  }
  __syncthreads();

  // ---- the budget-th largest key
  uint32_t prefix = 0, need = p.budget;
  int shift = 32;
  bool ties = true;                              // of the keys at the edge only the first `need` stay
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int above = shift, width = pass < 2 ? 11 : 10;
    shift -= width;
#pragma unroll 4
    for (int i = tid; i < mine; i += T) {
      const uint32_t key = keys[i];
      if (pass == 0 || key >> above == prefix) atomicAdd(&hist[pass][key >> shift & ((1u << width) - 1)], 1u);
    }
    sync();
    // thread t: BINS bins from 2047 - BINS t down, so that the sums run from the top
    constexpr int BINS = 2048 / T;
    uint32_t c[BINS] = {}, mine_of = 0;
#pragma unroll
    for (int other = 0; other < kEvictCluster; ++other) {
      if (other >= cs) break;
      const uint2* v = reinterpret_cast<const uint2*>(cluster.map_shared_rank(&hist[pass][0], other) +
                                                      2048 - BINS * (tid + 1));
#pragma unroll
      for (int x = 0; x < BINS; x += 2) {
        const uint2 two = v[(BINS - 2 - x) / 2];
        c[x] += two.y;
        c[x + 1] += two.x;
      }
    }
#pragma unroll
    for (int x = 0; x < BINS; ++x) mine_of += c[x];
    uint32_t all, before = block_scan<T>(mine_of, sums, &all);
#pragma unroll
    for (int x = 0; x < BINS; ++x) {
      if (before < need && need <= before + c[x]) {
        found[0] = 2047 - BINS * tid - x;
        found[1] = need - before;
        found[2] = c[x];
      }
      before += c[x];
    }
    __syncthreads();
    prefix = prefix << width | found[0];
    need = found[1];
    if (need == found[2]) {                      // (the same in every CTA) all of them stay
      ties = false;
      break;
    }
  }
  // kept: keys whose bits from `shift` up are above `prefix`, or equal to it and, with ties
  // (shift is 0 then), among the first `need`

  // ---- ranks, by rounds of a key a thread: a warp's flags are one ballot, and the counts of
  // (round, warp) are summed in the order of the keys
  const int rounds = (p.chunk + T - 1) / T;   // <= 32
  const uint32_t below_me = (1u << lane) - 1;
  uint32_t all;
  if (ties) {
    for (int x = 0; x < rounds; ++x) {
      const int i = x * T + tid;
      const uint32_t eq = __ballot_sync(0xffffffffu, i < mine && keys[i] == prefix);
      if (lane == 0) equals[x * WARPS + warp] = __popc(eq);
    }
    __syncthreads();
    uint32_t before = block_scan<T>(tid < rounds * WARPS ? equals[tid] : 0, sums, &all);
    if (cs > 1) {
      if (tid == 0) counts[0] = all;
      cluster.sync();
      for (int c = 0; c < rank; ++c) before += cluster.map_shared_rank(counts, c)[0];
    }
    if (tid < rounds * WARPS) equals[tid] = before;
    __syncthreads();
  }
  uint32_t free_place = 0, moved = 0;            // this round's ballots
  auto flags = [&](int x) {
    const int i = x * T + tid;
    const bool live = i < mine;
    const uint32_t key = live ? keys[i] : 0, top = key >> shift;
    bool kept = top > prefix || top == prefix;
    if (ties) {
      const bool eq = live && key == prefix;
      const uint32_t eqs = __ballot_sync(0xffffffffu, eq);
      if (eq) kept = equals[x * WARPS + warp] + __popc(eqs & below_me) < need;
    }
    const bool low = i0 + i < p.budget;
    free_place = __ballot_sync(0xffffffffu, live && low && !kept);
    moved = __ballot_sync(0xffffffffu, live && !low && kept);
  };
  for (int x = 0; x < rounds; ++x) {
    flags(x);
    if (lane == 0) places[x * WARPS + warp] = __popc(free_place) | __popc(moved) << 16;
  }
  __syncthreads();
  uint32_t before = block_scan<T>(tid < rounds * WARPS ? places[tid] : 0, sums, &all);
  int total = static_cast<int>(all >> 16), free_at = 0, move_at = 0;
  if (cs > 1) {
    if (tid == 0) counts[1] = all;
    cluster.sync();
    total = 0;
#pragma unroll
    for (int c = 0; c < kEvictCluster; ++c) {
      if (c >= cs) break;
      const uint32_t other = cluster.map_shared_rank(counts, c)[1];
      if (c < rank) {
        free_at += static_cast<int>(other & 0xffff);
        move_at += static_cast<int>(other >> 16);
      }
      total += static_cast<int>(other >> 16);
    }
  }
  if (tid < rounds * WARPS) places[tid] = before;
  __syncthreads();
  int2* moves = p.moves + static_cast<long long>(unit) * p.move_rows;
  for (int x = 0; x < rounds; ++x) {
    flags(x);
    const uint32_t base = places[x * WARPS + warp];
    const int at = i0 + x * T + tid;
    if (free_place >> lane & 1) moves[free_at + (base & 0xffff) + __popc(free_place & below_me)].x = at;
    if (moved >> lane & 1) moves[move_at + (base >> 16) + __popc(moved & below_me)].y = at;
  }
  if (rank == 0 && tid == 0) p.count[unit] = total;
  sync();                                        // the list is complete; no CTA's memory is read any more
  for (int i = rank * T + tid; i < total; i += cs * T) {
    const int2 mv = __ldcg(moves + i);
    w_out[mv.x] = w[mv.y];
    pos_out[mv.x] = pos[mv.y];
  }
  if (p.fused) {
    const int width = p.row_bytes <= 128 ? 8 : 32, per = T / width;
    move_rows(p, b, h, moves, rank * per + tid / width, cs * per, total, tid % width, width);
  }
}

__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ EvictParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int unit = blockIdx.y, b = unit / p.kv_heads, h = unit - b * p.kv_heads;
  const int total = __ldcg(p.count + unit);
  const int2* moves = p.moves + static_cast<long long>(unit) * p.move_rows;
  const int width = p.row_bytes <= 128 ? 8 : p.row_bytes <= 256 ? 16 : 32, per = kMoveThreads / width;
  move_rows(p, b, h, moves, blockIdx.x * per + threadIdx.x / width, gridDim.x * per, total,
            threadIdx.x % width, width);
}

struct AdvanceParams {
  PageTable pages;
  int max_rows;
  const int *lengths, *seen;
  int *lengths_out, *seen_out;
  long long *slot, *pos;
  int batch, q_len, max_positions;
  int* status;
};

// A thread a sequence: it reads the sequence's length and count before it writes them.  All
// latency, 1.4 us; 2.3 us for 256 sequences of four tokens.
__global__ void __launch_bounds__(128) advance_kernel(const __grid_constant__ AdvanceParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= p.batch) return;
  const int n = p.lengths[b], seen = p.seen[b];
  bool ok = n >= 0 && n <= p.max_rows - p.q_len &&
            (p.max_positions == 0 || (seen >= 0 && seen <= p.max_positions - p.q_len));
  int row[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    row[r] = ok && r < p.q_len ? cache_row(p.pages, b, n + r) : 0;
  }
#pragma unroll
  for (int r = 0; r < 8; ++r) ok = ok && row[r] >= 0;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    if (r < p.q_len) {
      p.slot[b * p.q_len + r] = ok ? row[r] : -1;
      p.pos[b * p.q_len + r] = ok ? seen + r : 0;
    }
  }
  p.lengths_out[b] = ok ? n + p.q_len : n;
  p.seen_out[b] = ok ? seen + p.q_len : seen;
  if (!ok && p.status) atomicCAS(p.status, 0, IQ_ERR_ROUTE);
}

// ------------------------------------------------------------------------------------
// host side
static int kv_sms() {
  static std::mutex mutex;
  static int per_device[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  std::lock_guard<std::mutex> lock(mutex);
  if (per_device[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    if (cudaFuncSetAttribute(evict_kernel<kEvictMany>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kEvictChunk * 4) != cudaSuccess)
      return 0;
    per_device[dev] = n;
  }
  return per_device[dev];
}

static int page_shift(int page) {
  for (int s = 0; s < 30; ++s)
    if (page == 1 << s) return s;
  return -1;
}

template <class P>
static int kv_launch(void (*kernel)(const P), const P& p, dim3 grid, int threads, int smem,
                     int cluster, void* stream, bool pdl) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2] = {};
  int n = 0;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = static_cast<unsigned>(n);
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, p);
  if (err != cudaSuccess) {
    fprintf(stderr, "iqb200: launch failed: %s\n", cudaGetErrorString(err));
    return IQ_ERR_CUDA;
  }
  return IQ_OK;
}

// Whether two arrays of n ints share memory.
static bool overlap(const int* a, const int* b, long long n) {
  const uint64_t x = reinterpret_cast<uint64_t>(a), y = reinterpret_cast<uint64_t>(b);
  return (x < y ? y - x : x - y) < static_cast<uint64_t>(n) * 4;
}

static size_t evict_count_bytes(long long units) { return static_cast<size_t>((units * 4 + 255) / 256 * 256); }

static bool evict_shape_ok(int batch, int kv_heads, long long rows) {
  return batch >= 1 && kv_heads >= 1 && rows >= 1 && rows <= kEvictRows &&
         static_cast<long long>(batch) * kv_heads <= 65535;
}

}  // namespace iqb

using namespace iqb;

extern "C" size_t iq_evict_work_bytes(int batch, int kv_heads, int rows) {
  if (!evict_shape_ok(batch, kv_heads, rows)) return 0;
  const long long units = static_cast<long long>(batch) * kv_heads;
  // at most half of the rows move: a moved row lies above the budget, its place below
  return evict_count_bytes(units) + static_cast<size_t>(units) * (rows / 2 + 1) * sizeof(int2);
}

extern "C" int iq_kv_evict(const iq_evict_args* a, void* stream) {
  if (!a || !a->k_cache || !a->v_cache || !a->page_table || !a->lengths || !a->seen ||
      !a->weights || !a->positions || !a->weights_out || !a->positions_out || !a->lengths_out ||
      !a->work)
    return IQ_ERR_ARG;
  if (a->page_size < 1 || a->max_pages < 1 || a->capacity < 1) return IQ_ERR_ARG;
  if (a->kv_kind != IQ_ACT_BF16 && a->kv_kind != IQ_ACT_E4M3) return IQ_ERR_ARG;
  if (a->budget < 1 || a->keep_first < 0 || a->keep_last < 0 ||
      static_cast<long long>(a->keep_first) + a->keep_last > a->budget)
    return IQ_ERR_ARG;
  const long long rows = static_cast<long long>(a->page_size) * a->max_pages;
  if (!evict_shape_ok(a->batch, a->kv_heads, rows)) return IQ_ERR_UNSUPPORTED;
  // every head reads both; in place means element on element
  if (overlap(a->lengths_out, a->lengths, a->batch) || overlap(a->lengths_out, a->seen, a->batch) ||
      (a->weights_out == a->weights && (a->wo_b != a->w_b || a->wo_h != a->w_h)) ||
      (a->positions_out == a->positions && (a->po_b != a->p_b || a->po_h != a->p_h)))
    return IQ_ERR_ARG;
  const int elt = a->kv_kind == IQ_ACT_BF16 ? 2 : 1;
  if (a->head_dim < 1 || a->head_dim > 1024 || a->head_dim * elt % 16) return IQ_ERR_UNSUPPORTED;
  if (a->work_bytes < iq_evict_work_bytes(a->batch, a->kv_heads, static_cast<int>(rows)))
    return IQ_ERR_ARG;
  const uint64_t al = reinterpret_cast<uint64_t>(a->k_cache) | reinterpret_cast<uint64_t>(a->v_cache) |
                      static_cast<uint64_t>(a->k_row * elt) | static_cast<uint64_t>(a->k_head * elt) |
                      static_cast<uint64_t>(a->v_row * elt) | static_cast<uint64_t>(a->v_head * elt) |
                      reinterpret_cast<uint64_t>(a->work);
  if (al & 15) return IQ_ERR_ARG;
  const int n_sm = kv_sms();
  if (n_sm == 0) return IQ_ERR_CUDA;

  EvictParams p{};
  p.k = static_cast<uint8_t*>(a->k_cache);
  p.v = static_cast<uint8_t*>(a->v_cache);
  p.k_row = a->k_row * elt; p.k_head = a->k_head * elt;
  p.v_row = a->v_row * elt; p.v_head = a->v_head * elt;
  p.pages = PageTable{a->page_table, a->table_stride, a->page_size, page_shift(a->page_size), a->capacity};
  p.max_rows = static_cast<int>(rows);
  p.lengths = a->lengths; p.seen = a->seen;
  p.w = a->weights; p.w_b = a->w_b; p.w_h = a->w_h;
  p.pos = a->positions; p.p_b = a->p_b; p.p_h = a->p_h;
  p.w_out = a->weights_out; p.wo_b = a->wo_b; p.wo_h = a->wo_h;
  p.pos_out = a->positions_out; p.po_b = a->po_b; p.po_h = a->po_h;
  p.lengths_out = a->lengths_out;
  const long long units = static_cast<long long>(a->batch) * a->kv_heads;
  p.count = static_cast<int*>(a->work);
  p.moves = reinterpret_cast<int2*>(static_cast<uint8_t*>(a->work) + evict_count_bytes(units));
  p.move_rows = static_cast<int>(rows / 2 + 1);
  p.status = a->status;
  p.kv_heads = a->kv_heads;
  p.row_bytes = a->head_dim * elt;
  p.budget = a->budget; p.keep_first = a->keep_first; p.keep_last = a->keep_last;
  const long long spare = rows - a->budget;
  const long long most = spare < a->budget ? (spare > 0 ? spare : 0) : a->budget;
  p.fused = most <= kEvictFusedMoves;
  // CTAs a cluster: eight keys a thread and pass where that many CTAs run at once (two an SM);
  // 32768 rows x 8 heads: four CTAs 25.9 us, eight 27.2, two 32.4; 52283 rows x 56 heads, which
  // eight each would make two waves: four 33, eight 62
  int cluster = 1;
  while (cluster < kEvictCluster &&
         (rows > static_cast<long long>(kEvictChunk) * cluster ||
          (rows > 8LL * kEvictMany * cluster && units * cluster <= n_sm)))
    cluster *= 2;
  p.chunk = static_cast<int>((rows + cluster - 1) / cluster);
  const dim3 grid(static_cast<unsigned>(units * cluster));
  const int rc = rows <= 8 * kEvictFew
                     ? kv_launch(evict_kernel<kEvictFew>, p, grid, kEvictFew, p.chunk * 4, 1, stream, a->pdl != 0)
                     : kv_launch(evict_kernel<kEvictMany>, p, grid, kEvictMany, p.chunk * 4, cluster, stream,
                                 a->pdl != 0);
  if (rc != IQ_OK || p.fused) return rc;
  // two rows for every group of lanes, twice the chip's threads at most
  const int per = kMoveThreads / (p.row_bytes <= 128 ? 8 : p.row_bytes <= 256 ? 16 : 32);
  long long x = (most + kMovesInFlight * per - 1) / (kMovesInFlight * per);
  const long long cap = (n_sm * 16 + units - 1) / units;
  if (x > cap) x = cap;
  return kv_launch(evict_move_kernel, p, dim3(static_cast<unsigned>(x), static_cast<unsigned>(units)),
                   kMoveThreads, 0, 1, stream, true);
}

extern "C" int iq_kv_advance(const iq_advance_args* a, void* stream) {
  if (!a || !a->page_table || !a->lengths || !a->seen || !a->lengths_out || !a->seen_out ||
      !a->slot || !a->pos)
    return IQ_ERR_ARG;
  if (a->page_size < 1 || a->max_pages < 1 || a->capacity < 1 || a->batch < 1 || a->q_len < 1 ||
      a->q_len > 8 || a->max_positions < 0)
    return IQ_ERR_ARG;
  const long long rows = static_cast<long long>(a->page_size) * a->max_pages;
  if (rows > 0x3fffffffLL || a->batch > (1 << 24)) return IQ_ERR_UNSUPPORTED;
  // in place means element on element: another thread's element is not to be written
  for (const int* out : {a->lengths_out, a->seen_out})
    for (const int* in : {a->lengths, a->seen})
      if (out != in && overlap(out, in, a->batch)) return IQ_ERR_ARG;
  if (overlap(a->lengths_out, a->seen_out, a->batch)) return IQ_ERR_ARG;
  AdvanceParams p{};
  p.pages = PageTable{a->page_table, a->table_stride, a->page_size, page_shift(a->page_size), a->capacity};
  p.max_rows = static_cast<int>(rows);
  p.lengths = a->lengths; p.seen = a->seen;
  p.lengths_out = a->lengths_out; p.seen_out = a->seen_out;
  p.slot = reinterpret_cast<long long*>(a->slot);
  p.pos = reinterpret_cast<long long*>(a->pos);
  p.batch = a->batch; p.q_len = a->q_len; p.max_positions = a->max_positions;
  p.status = a->status;
  return kv_launch(advance_kernel, p, dim3(static_cast<unsigned>((a->batch + 127) / 128)), 128, 0, 1,
                   stream, a->pdl != 0);
}
