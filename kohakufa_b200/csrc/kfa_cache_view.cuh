// A cache of keys and values in pages as its kernels see it, and how kernels that follow one another in a stream are chained.
#pragma once

#include "kfa_ptx.cuh"

namespace kfa {

constexpr int DEV_BAD_CACHE = 90;  // KFA_DEV_BAD_CACHE

struct CacheView {
  uint8_t *k, *v;                               // pages
  long long k_sn, k_sh, k_ss, v_sn, v_sh, v_ss;  // strides of page, head, slot, in bytes
  const int* table;                             // or nullptr: page b is sequence b's
  long long table_stride;
  const int* lengths;
  FastDiv by_page;
  int page, n_pages, capacity, batch, heads, cols;
};

// Which rows of new tokens a call takes (see KfaRows).
struct RowsView {
  const int* index;
  long long index_stride;
  const int* counts;
  int steps, T;
  __device__ __forceinline__ int count(int b) const { return counts ? min(max(counts[b], 0), steps) : steps; }
  __device__ __forceinline__ int row(int b, int i) const { return index ? index[b * index_stride + i] : i; }
};

// Kernels here are launched while the one before them in the stream may still run: each sets up what touches no global memory, then
// waits for that one's end (its writes are visible then), and lets the next be launched as soon as all its own CTAs have come that far.
// One that uses tensor memory lets it only when it has its own: the next one's CTAs keep theirs while they wait.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

__device__ __forceinline__ void report(int* status, int code) { atomicCAS(status, 0, code); }

// The length of sequence b; one that the cache has no room for is cut off (and reported by the caller's check).
__device__ __forceinline__ int cache_length(const CacheView& c, int b) { return min(max(c.lengths[b], 0), c.capacity); }
__device__ __forceinline__ bool length_ok(const CacheView& c, int b) { return c.lengths[b] >= 0 && c.lengths[b] <= c.capacity; }
// Page and slot of a position inside the capacity; false: the table names a page that the cache does not have.
__device__ __forceinline__ bool cache_place(const CacheView& c, int b, int pos, int& page, int& slot) {
  if (c.table == nullptr) {
    page = b;
    slot = pos;
    return true;
  }
  const int at = static_cast<int>(c.by_page.div(pos));
  slot = pos - at * c.page;
  page = c.table[b * c.table_stride + at];
  return page >= 0 && page < c.n_pages;
}

}  // namespace kfa
