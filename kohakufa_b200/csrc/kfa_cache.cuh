// A cache of keys and values in pages, and what copies on it: append, eviction. (Attention: kfa_attend.cuh; accumulated weights: kfa_weigh.cuh.)
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

// ---- append --------------------------------------------------------------------------------------------------------------
struct AppendParams {
  CacheView c;
  RowsView r;
  const uint8_t *k, *v;
  long long k_sb, k_sh, k_ss, v_sb, v_sh, v_ss;  // bytes
  FastDiv by_piece, by_head, by_step;
  unsigned total;
  int* status;
};

// A thread moves 16 bytes of a key and 16 of the value: pieces of a row fastest, then heads, then rows.
__global__ void __launch_bounds__(256) kfa_cache_append_kernel(const AppendParams p) {
  const unsigned at = blockIdx.x * 256u + threadIdx.x;
  if (at >= p.total) return;
  const unsigned row = p.by_piece.div(at), piece = at - row * p.by_piece.d;
  const unsigned rest = p.by_head.div(row), g = row - rest * p.by_head.d;
  const unsigned b = p.by_step.div(rest), i = rest - b * p.by_step.d;
  if (static_cast<int>(i) >= p.r.count(b)) return;
  const int t = p.r.row(b, i);
  const long long pos = static_cast<long long>(p.c.lengths[b]) + i;
  int page = -1, slot = 0;
  if (t < 0 || t >= p.r.T || p.c.lengths[b] < 0 || pos >= p.c.capacity || !cache_place(p.c, b, static_cast<int>(pos), page, slot)) {
    report(p.status, DEV_BAD_CACHE);
    return;
  }
  const uint4 k = *reinterpret_cast<const uint4*>(p.k + b * p.k_sb + g * p.k_sh + t * p.k_ss + 16 * piece);
  const uint4 v = *reinterpret_cast<const uint4*>(p.v + b * p.v_sb + g * p.v_sh + t * p.v_ss + 16 * piece);
  *reinterpret_cast<uint4*>(p.c.k + page * p.c.k_sn + g * p.c.k_sh + slot * p.c.k_ss + 16 * piece) = k;
  *reinterpret_cast<uint4*>(p.c.v + page * p.c.v_sn + g * p.c.v_sh + slot * p.c.v_ss + 16 * piece) = v;
}

// ---- eviction ------------------------------------------------------------------------------------------------------------
struct EvictParams {
  CacheView c, out;
  const float* w;
  long long w_sb, w_sh;
  int keep, recent, clear;
  float* w_out;
  int* kept;
  int* lengths_out;
  FastDiv by_slot, by_head, by_piece;
  unsigned total;
  int* status;
};

constexpr int SELECT_THREADS = 512;

// Numbers whose order as unsigned integers is the weights' order: -0 and 0 are equal, NaN is the largest.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Which positions stay, per (sequence, K / V head). The key of the last one that stays is found digit by digit (8 bits, from the
// top): a histogram of the digit among the positions that agree in the digits before it. Then one pass in ascending order: all
// above that key stay, of those equal to it the first ones, until there are enough.
__global__ void __launch_bounds__(SELECT_THREADS) kfa_cache_select_kernel(const EvictParams p) {
  const int g = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __shared__ int hist[256], warp_gt[SELECT_THREADS / 32], warp_eq[SELECT_THREADS / 32], s_digit, s_need;
  const int len = cache_length(p.c, b);
  if (tid == 0 && !length_ok(p.c, b)) report(p.status, DEV_BAD_CACHE);
  const float* w = p.w + b * p.w_sb + g * p.w_sh;
  const long long row = static_cast<long long>(b) * p.c.heads + g;
  int* kept = p.kept + row * p.keep;
  float* w_out = p.w_out + row * p.keep;
  const int left = min(len, p.keep);
  if (g == 0 && tid == 0) p.lengths_out[b] = left;
  for (int i = left + tid; i < p.keep; i += SELECT_THREADS) {
    kept[i] = -1;
    w_out[i] = 0.f;
  }
  if (len <= p.keep) {
    for (int i = tid; i < len; i += SELECT_THREADS) {
      kept[i] = i;
      w_out[i] = w[i];
    }
    return;
  }
  const int old = len - p.recent, want = p.keep - p.recent;  // 0 <= want < old
  for (int i = tid; i < p.recent; i += SELECT_THREADS) {
    kept[want + i] = old + i;
    w_out[want + i] = w[old + i];
  }
  if (want == 0) return;
  uint32_t prefix = 0, mask = 0;
  int need = want;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += SELECT_THREADS) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < old; i += SELECT_THREADS) {
      const uint32_t key = weight_key(w[i]);
      if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int d = 255, above = 0;
      while (above + hist[d] < need) above += hist[d--];
      s_digit = d;
      s_need = need - above;
    }
    __syncthreads();
    need = s_need;
    prefix |= static_cast<uint32_t>(s_digit) << shift;
    mask |= 255u << shift;
    __syncthreads();
  }
  int done_gt = 0, done_eq = 0;  // before this stretch of positions
  for (int i0 = 0; i0 < old; i0 += SELECT_THREADS) {
    const int i = i0 + tid;
    const float x = i < old ? w[i] : 0.f;
    const uint32_t key = weight_key(x);
    const bool gt = i < old && key > prefix, eq = i < old && key == prefix;
    const unsigned bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) warp_gt[warp] = __popc(bg), warp_eq[warp] = __popc(be);
    __syncthreads();
    int gts = done_gt, eqs = done_eq;
    for (int o = 0; o < SELECT_THREADS / 32; ++o) {
      if (o < warp) gts += warp_gt[o], eqs += warp_eq[o];
      done_gt += warp_gt[o];
      done_eq += warp_eq[o];
    }
    const unsigned below = (1u << lane) - 1u;
    gts += __popc(bg & below);
    eqs += __popc(be & below);
    if (gt || (eq && eqs < need)) {
      const int at = gts + min(eqs, need);
      kept[at] = i;
      w_out[at] = x;
    }
    __syncthreads();
  }
}

// Moves the rows that stay: a thread 16 bytes of a key and of its value.
__global__ void __launch_bounds__(256) kfa_cache_gather_kernel(const EvictParams p) {
  const unsigned at = blockIdx.x * 256u + threadIdx.x;
  if (at >= p.total) return;
  const unsigned row = p.by_piece.div(at), piece = at - row * p.by_piece.d;
  const unsigned rest = p.by_head.div(row), g = row - rest * p.by_head.d;
  const unsigned b = p.by_slot.div(rest), i = rest - b * p.by_slot.d;
  const int pos = p.kept[(static_cast<long long>(b) * p.c.heads + g) * p.keep + i];
  if (pos < 0 && !p.clear) return;
  int page = 0, slot = 0, page_o, slot_o;
  if ((pos >= 0 && !cache_place(p.c, b, pos, page, slot)) || !cache_place(p.out, b, i, page_o, slot_o)) {
    report(p.status, DEV_BAD_CACHE);
    return;
  }
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  if (pos >= 0) {
    k = *reinterpret_cast<const uint4*>(p.c.k + page * p.c.k_sn + g * p.c.k_sh + slot * p.c.k_ss + 16 * piece);
    v = *reinterpret_cast<const uint4*>(p.c.v + page * p.c.v_sn + g * p.c.v_sh + slot * p.c.v_ss + 16 * piece);
  }
  *reinterpret_cast<uint4*>(p.out.k + page_o * p.out.k_sn + g * p.out.k_sh + slot_o * p.out.k_ss + 16 * piece) = k;
  *reinterpret_cast<uint4*>(p.out.v + page_o * p.out.v_sn + g * p.out.v_sh + slot_o * p.out.v_ss + 16 * piece) = v;
}

}  // namespace kfa
