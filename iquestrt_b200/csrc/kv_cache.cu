// Bookkeeping of the paged key/value cache: eviction by accumulated attention weight
// (iq_kv_evict) and the next tokens' rows (iq_kv_advance).
//
// Eviction is a selection and a movement.  The selection finds the budget-th largest of a
// (sequence, head)'s weights exactly: order-preserving integers of the weights, four
// histogram passes of eight bits each.  One cluster holds all of a head's weights in the
// shared memory of its CTAs, so global memory is read once; a pass costs a histogram of
// local words, one cluster barrier and the sum of the CTAs' 256 bins through distributed
// shared memory.  The movement fills the freed places below the budget with the kept rows
// above it: sources and destinations are disjoint, so it runs in place, in any order and on
// all SMs, and moves the fewest rows there are to move.
// What bounds it: latency (barriers, passes) for a step's few rows, HBM for a long prompt's.
#include <math.h>
#include <stdio.h>

#include <mutex>
#include <unordered_set>

#include <cooperative_groups.h>

#include "paged.cuh"

namespace iqb {

namespace cg = cooperative_groups;

constexpr int kEvictThreads = 512;
constexpr int kEvictChunk = 32768;               // weights a CTA of a cluster holds at most
constexpr int kEvictCluster = 8;
constexpr int kEvictRows = kEvictChunk * kEvictCluster;
constexpr int kMoveThreads = 256;
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
__device__ __forceinline__ int block_scan(int x, int* sums /* [33] */, int* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int incl = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  __syncthreads();                               // `sums` may still be read by an earlier scan
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    const int v = lane < warps ? sums[lane] : 0;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    if (lane < warps) sums[lane] = s - v;
    if (lane == 31) sums[32] = s;
  }
  __syncthreads();
  *all = sums[32];
  return incl - x + sums[warp];
}

// One cache row of K and of V, 16 bytes a thread of `width` threads.
__device__ __forceinline__ void move_row(const EvictParams& p, int b, int h, int2 mv, int at, int width) {
  const int to = cache_row(p.pages, b, mv.x), from = cache_row(p.pages, b, mv.y);
  if (to < 0 || from < 0) {
    if (p.status) atomicCAS(p.status, 0, IQ_ERR_ROUTE);
    return;
  }
  for (int c = at * 16; c < p.row_bytes; c += width * 16) {
    const uint4 k = *reinterpret_cast<const uint4*>(p.k + from * p.k_row + h * p.k_head + c);
    const uint4 v = *reinterpret_cast<const uint4*>(p.v + from * p.v_row + h * p.v_head + c);
    *reinterpret_cast<uint4*>(p.k + to * p.k_row + h * p.k_head + c) = k;
    *reinterpret_cast<uint4*>(p.v + to * p.v_row + h * p.v_head + c) = v;
  }
}

__global__ void __launch_bounds__(kEvictThreads) evict_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ uint32_t keys[];             // [chunk]
  __shared__ uint32_t hist[4][256];
  __shared__ uint32_t bins[2][256];
  __shared__ int sums[33];
  __shared__ int found[2];                       // the digit, and what is still needed inside it
  __shared__ int counts[3];                      // this CTA's equal keys, free places, moved rows
  cg::cluster_group cluster = cg::this_cluster();
  const int cs = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int unit = blockIdx.x / cs, b = unit / p.kv_heads, h = unit - b * p.kv_heads;
  const int tid = threadIdx.x;

  pdl_wait();
  pdl_launch_dependents();
  const int n = evict_length(p, b, h == 0 && rank == 0 && tid == 0);
  const int keep = min(n, p.budget);
  if (h == 0 && rank == 0 && tid == 0) p.lengths_out[b] = keep;
  const float* w = p.w + b * p.w_b + h * p.w_h;
  const int* pos = p.pos + b * p.p_b + h * p.p_h;
  float* w_out = p.w_out + b * p.wo_b + h * p.wo_h;
  int* pos_out = p.pos_out + b * p.po_b + h * p.po_h;
  if (n <= p.budget) {                           // (the whole cluster)
    if (rank == 0 && tid == 0) p.count[unit] = 0;
    for (int i = rank * kEvictThreads + tid; i < n; i += cs * kEvictThreads) {
      if (w_out != w) w_out[i] = w[i];
      if (pos_out != pos) pos_out[i] = pos[i];
    }
    return;
  }

  const int share = (n + cs - 1) / cs;           // <= p.chunk
  const int i0 = min(rank * share, n), mine = min(i0 + share, n) - i0;
  for (int x = tid; x < 4 * 256; x += kEvictThreads) hist[x >> 8][x & 255] = 0;
  const int last = __ldg(p.seen + b) - p.keep_last;
  for (int i = tid; i < mine; i += kEvictThreads) {
    const int at = pos[i0 + i];
    keys[i] = at < p.keep_first || at >= last ? 0xffffffffu : weight_key(w[i0 + i]);
  }
  __syncthreads();

  // ---- the budget-th largest key: eight bits a pass
  uint32_t prefix = 0;
  int need = p.budget;
#pragma unroll 1
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    for (int i = tid; i < mine; i += kEvictThreads) {
      const uint32_t key = keys[i];
      if (pass == 0 || (key >> (shift + 8)) == prefix) atomicAdd(&hist[pass][(key >> shift) & 255], 1u);
    }
    cluster.sync();
    {
      // two threads a bin, each half of the CTAs
      const int bin = tid & 255, half = tid >> 8;
      uint32_t s = 0;
      for (int c = half; c < cs; c += 2) s += cluster.map_shared_rank(&hist[pass][0], c)[bin];
      bins[half][bin] = s;
    }
    __syncthreads();
    if (tid < 32) {                              // lane l: bins 255 - 8 l down to 248 - 8 l
      int s = 0;
      int c[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const int bin = 255 - 8 * tid - x;
        c[x] = static_cast<int>(bins[0][bin] + bins[1][bin]);
        s += c[x];
      }
      int incl = s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (tid >= o) incl += y;
      }
      int above = incl - s;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        if (above < need && need <= above + c[x]) {
          found[0] = 255 - 8 * tid - x;
          found[1] = need - above;
        }
        above += c[x];
      }
    }
    __syncthreads();
    prefix = prefix << 8 | static_cast<uint32_t>(found[0]);
    need = found[1];
  }
  // kept: keys above `prefix`, and the first `need` of those equal to it

  // ---- ranks.  A thread owns `each` consecutive keys (an odd number: no bank conflicts)
  const int each = ((mine + kEvictThreads - 1) / kEvictThreads) | 1;
  const int a0 = min(tid * each, mine), a1 = min(a0 + each, mine);
  int eq = 0;
  for (int i = a0; i < a1; ++i) eq += keys[i] == prefix;
  int all;
  int eq_at = block_scan(eq, sums, &all);
  if (tid == 0) counts[0] = all;
  cluster.sync();
  for (int c = 0; c < rank; ++c) eq_at += cluster.map_shared_rank(counts, c)[0];
  int holes = 0, moved = 0, e = eq_at;
  for (int i = a0; i < a1; ++i) {
    const bool kept = keys[i] > prefix || (keys[i] == prefix && e++ < need);
    if (i0 + i < p.budget) holes += !kept; else moved += kept;
  }
  int n_holes, n_moved;
  int hole_at = block_scan(holes, sums, &n_holes);
  int move_at = block_scan(moved, sums, &n_moved);
  if (tid == 0) {
    counts[1] = n_holes;
    counts[2] = n_moved;
  }
  cluster.sync();
  int total = 0;
  for (int c = 0; c < cs; ++c) {
    const int* other = cluster.map_shared_rank(counts, c);
    if (c < rank) {
      hole_at += other[1];
      move_at += other[2];
    }
    total += other[2];
  }
  int2* moves = p.moves + static_cast<long long>(unit) * p.move_rows;
  e = eq_at;
  for (int i = a0; i < a1; ++i) {
    const int at = i0 + i;
    const bool kept = keys[i] > prefix || (keys[i] == prefix && e++ < need);
    if (at < p.budget) {
      if (!kept) moves[hole_at++].x = at;
    } else if (kept) {
      moves[move_at++].y = at;
    }
  }
  if (w_out != w || pos_out != pos) {
    for (int i = tid; i < mine && i0 + i < p.budget; i += kEvictThreads) {
      // (places about to be filled get their old values first; the moves below come after
      // the barrier)
      if (w_out != w) w_out[i0 + i] = w[i0 + i];
      if (pos_out != pos) pos_out[i0 + i] = pos[i0 + i];
    }
  }
  if (rank == 0 && tid == 0) p.count[unit] = total;
  cluster.sync();                                // the list is complete; no CTA's counts are read any more
  for (int i = rank * kEvictThreads + tid; i < total; i += cs * kEvictThreads) {
    const int2 mv = __ldcg(moves + i);
    w_out[mv.x] = w[mv.y];
    pos_out[mv.x] = pos[mv.y];
  }
  if (p.fused) {
    const int width = p.row_bytes <= 128 ? 8 : 32;
    const int per = kEvictThreads / width;
    for (int i = rank * per + tid / width; i < total; i += cs * per)
      move_row(p, b, h, __ldcg(moves + i), tid % width, width);
  }
}

__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ EvictParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int unit = blockIdx.y, b = unit / p.kv_heads, h = unit - b * p.kv_heads;
  const int total = __ldcg(p.count + unit);
  const int2* moves = p.moves + static_cast<long long>(unit) * p.move_rows;
  const int width = p.row_bytes <= 128 ? 8 : p.row_bytes <= 256 ? 16 : 32;
  const int per = kMoveThreads / width;
  for (int i = blockIdx.x * per + threadIdx.x / width; i < total; i += gridDim.x * per)
    move_row(p, b, h, __ldcg(moves + i), threadIdx.x % width, width);
}

struct AdvanceParams {
  PageTable pages;
  int max_rows;
  const int *lengths, *seen;
  int *lengths_out, *seen_out;
  long long *slot, *pos;
  int batch, q_len;
  int* status;
};

// A thread a sequence: it reads the sequence's length and count before it writes them.
__global__ void __launch_bounds__(128) advance_kernel(const __grid_constant__ AdvanceParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= p.batch) return;
  const int n = p.lengths[b], seen = p.seen[b];
  bool ok = n >= 0 && n <= p.max_rows - p.q_len;
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
      p.pos[b * p.q_len + r] = seen + r;
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
    if (cudaFuncSetAttribute(evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
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
  if (a->lengths_out == a->lengths) return IQ_ERR_ARG;
  const long long rows = static_cast<long long>(a->page_size) * a->max_pages;
  if (!evict_shape_ok(a->batch, a->kv_heads, rows)) return IQ_ERR_UNSUPPORTED;
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
  // CTAs a cluster: about eight keys a thread and pass
  int cluster = 1;
  while (cluster < kEvictCluster && rows > 4096LL * cluster) cluster *= 2;
  p.chunk = static_cast<int>((rows + cluster - 1) / cluster);
  const int rc = kv_launch(evict_kernel, p, dim3(static_cast<unsigned>(units * cluster)), kEvictThreads,
                           p.chunk * 4, cluster, stream, a->pdl != 0);
  if (rc != IQ_OK || p.fused) return rc;
  // eight rows of work for every group of lanes, the whole chip at most
  const int per = kMoveThreads / (p.row_bytes <= 128 ? 8 : p.row_bytes <= 256 ? 16 : 32);
  long long x = (most + 4 * per - 1) / (4 * per);
  const long long cap = (n_sm * 8 + units - 1) / units;
  if (x > cap) x = cap;
  return kv_launch(evict_move_kernel, p, dim3(static_cast<unsigned>(x), static_cast<unsigned>(units)),
                   kMoveThreads, 0, 1, stream, true);
}

extern "C" int iq_kv_advance(const iq_advance_args* a, void* stream) {
  if (!a || !a->page_table || !a->lengths || !a->seen || !a->lengths_out || !a->seen_out ||
      !a->slot || !a->pos)
    return IQ_ERR_ARG;
  if (a->page_size < 1 || a->max_pages < 1 || a->capacity < 1 || a->batch < 1 || a->q_len < 1 ||
      a->q_len > 8)
    return IQ_ERR_ARG;
  const long long rows = static_cast<long long>(a->page_size) * a->max_pages;
  if (rows > 0x3fffffffLL || a->batch > (1 << 24)) return IQ_ERR_UNSUPPORTED;
  AdvanceParams p{};
  p.pages = PageTable{a->page_table, a->table_stride, a->page_size, page_shift(a->page_size), a->capacity};
  p.max_rows = static_cast<int>(rows);
  p.lengths = a->lengths; p.seen = a->seen;
  p.lengths_out = a->lengths_out; p.seen_out = a->seen_out;
  p.slot = reinterpret_cast<long long*>(a->slot);
  p.pos = reinterpret_cast<long long*>(a->pos);
  p.batch = a->batch; p.q_len = a->q_len;
  p.status = a->status;
  return kv_launch(advance_kernel, p, dim3(static_cast<unsigned>((a->batch + 127) / 128)), 128, 0, 1,
                   stream, a->pdl != 0);
}
