// What the kernels over the paged key/value cache share: the cache's geometry.
#pragma once

#include "common.cuh"

namespace iqb {

// A row index of the cache from a row index of a sequence; -1 where the page table holds
// no page of the cache.
struct PageTable {
  const int* table;        // [batch, stride]
  long long stride;
  int page;                // rows a page
  int shift;               // log2(page), or -1
  int capacity;            // rows of the cache
};

// The page that holds row j of sequence b, and the cache row of row j given its page.
__device__ __forceinline__ int page_id(const PageTable& t, int b, int j) {
  return __ldg(t.table + b * t.stride + (t.shift >= 0 ? j >> t.shift : j / t.page));
}
__device__ __forceinline__ int page_row(const PageTable& t, int id, int j) {
  const int off = t.shift >= 0 ? j & (t.page - 1) : j % t.page;
  const long long row = static_cast<long long>(id) * t.page + off;
  return id >= 0 && row < t.capacity ? static_cast<int>(row) : -1;
}
__device__ __forceinline__ int cache_row(const PageTable& t, int b, int j) {
  return page_row(t, page_id(t, b, j), j);
}

// 16 bytes global -> shared; `ok` false fills with zeros and reads nothing.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  const int n = ok ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n)
               : "memory");
}

// 2^x, flushing results below the smallest normal number (relative error <= 2^-22).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace iqb
