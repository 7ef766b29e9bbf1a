// A cache of keys and values in pages, and what copies on it: append, eviction. (Attention: kfa_attend.cuh; accumulated weights: kfa_weigh.cuh.)
#pragma once

#include "kfa_cache_view.cuh"

namespace kfa {

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
  wait_for_previous();
  let_next_begin();
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
  int room;                  // positions of w_out; with clear also of out that get zeros behind the kept ones
  float* w_out;
  int* kept;
  int* lengths_out;
  FastDiv by_slot, by_head;  // 32 slots of a (sequence, head) at a time (clear: up to room, else up to keep); heads
  unsigned total;            // such groups
  int* status;
};

constexpr int SELECT_HELD = 8;  // positions of a thread that stay in registers

// Numbers whose order as unsigned integers is the weights' order: -0 and 0 are equal, NaN is the largest.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Which positions stay, per (sequence, K / V head). The key of the last one that stays is found digit by digit (11, 11 and 10 bits, from the
// top): a histogram of the digit among the positions that agree in the digits before it. It ends early when all that agree stay. Then every
// warp takes a stretch of the positions, counts those above that key and those equal to it, and lists them in ascending order: all above it
// stay, of the equal ones the first, until there are enough. Bound by latency; a thread's first 8 positions are read once and held.
// SELECT_THREADS: 512 for caches of up to 2048 positions, else 1024. (The whole call in us with 256, 512, 1024: 2 x 4 heads over 320
// positions 10.7, 10.0, 11.1; 16 x 8 over 1500 to 8192 93.7, 76.8, 57.4.) A long row is one CTA's as well: 8 heads over 8192, 32768, 131072 positions
// take 21, 45, 193.
template <int SELECT_THREADS>
__global__ void __launch_bounds__(SELECT_THREADS) kfa_cache_select_kernel(const EvictParams p) {
  constexpr int WARPS = SELECT_THREADS / 32, BINS = 2048, PER = BINS / SELECT_THREADS;
  const int g = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __shared__ int hist[BINS], warp_gt[WARPS], warp_eq[WARPS], s_digit, s_need, s_all;
  wait_for_previous();
  let_next_begin();
  const int len = cache_length(p.c, b);
  if (tid == 0 && !length_ok(p.c, b)) report(p.status, DEV_BAD_CACHE);
  const float* w = p.w + b * p.w_sb + g * p.w_sh;
  const long long row = static_cast<long long>(b) * p.c.heads + g;
  int* kept = p.kept + row * p.keep;
  float* w_out = p.w_out + row * p.room;
  const int left = min(len, p.keep);
  if (g == 0 && tid == 0) p.lengths_out[b] = left;
  for (int i = left + tid; i < p.keep; i += SELECT_THREADS) kept[i] = -1;
  for (int i = left + tid; i < p.room; i += SELECT_THREADS) w_out[i] = 0.f;
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
  float held[SELECT_HELD];
#pragma unroll
  for (int k = 0; k < SELECT_HELD; ++k) {
    const int i = k * SELECT_THREADS + tid;
    held[k] = i < old ? w[i] : 0.f;
  }
  for (int shift = 21;; shift = shift == 21 ? 10 : 0) {
    const uint32_t digits = shift == 0 ? 1023u : 2047u;
    for (int i = tid; i < BINS; i += SELECT_THREADS) hist[i] = 0;
    __syncthreads();
    auto tally = [&](int i, float x) {
      const uint32_t key = weight_key(x), digit = (key >> shift) & digits;
      const bool in = i < old && (key & mask) == prefix;
      // (many equal weights: one addition a warp)
      const unsigned act = __ballot_sync(0xffffffffu, in);
      if (act == 0) return;
      const uint32_t lead = __shfl_sync(0xffffffffu, digit, __ffs(act) - 1);
      if (__all_sync(0xffffffffu, !in || digit == lead)) {
        if (lane == 0) atomicAdd(&hist[lead], __popc(act));
      } else if (in) {
        atomicAdd(&hist[digit], 1);
      }
    };
#pragma unroll
    for (int k = 0; k < SELECT_HELD; ++k)
      if (k * SELECT_THREADS < old) tally(k * SELECT_THREADS + tid, held[k]);
#pragma unroll 4
    for (int i0 = SELECT_HELD * SELECT_THREADS; i0 < old; i0 += SELECT_THREADS) tally(i0 + tid, i0 + tid < old ? w[i0 + tid] : 0.f);
    __syncthreads();
    // bins from the top, PER a thread: in whose are the last ones that are needed?
    int mine = 0, upto;
#pragma unroll
    for (int k = 0; k < PER; ++k) mine += hist[BINS - 1 - (PER * tid + k)];
    upto = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += up;
    }
    if (lane == 31) warp_gt[warp] = upto;
    __syncthreads();
    for (int o = 0; o < warp; ++o) upto += warp_gt[o];
    int above = upto - mine;
    if (above < need && upto >= need) {
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int n = hist[BINS - 1 - (PER * tid + k)];
        if (above < need && above + n >= need) {
          s_digit = BINS - 1 - (PER * tid + k);
          s_need = need - above;
          s_all = n == need - above;
        }
        above += n;
      }
    }
    __syncthreads();
    need = s_need;
    prefix |= static_cast<uint32_t>(s_digit) << shift;
    mask |= digits << shift;
    if (s_all || shift == 0) break;
  }
  // (above the prefix and equal to it in the digits looked at; where all that are equal stay, the other digits do not matter)
  const int stretch = (old + 32 * WARPS - 1) / (32 * WARPS) * 32, i_first = warp * stretch, i_last = min(i_first + stretch, old);
  int gts = 0, eqs = 0;
#pragma unroll 4
  for (int i0 = i_first; i0 < i_last; i0 += 32) {
    const uint32_t key = i0 + lane < i_last ? weight_key(w[i0 + lane]) & mask : 0u;
    gts += __popc(__ballot_sync(0xffffffffu, i0 + lane < i_last && key > prefix));
    eqs += __popc(__ballot_sync(0xffffffffu, i0 + lane < i_last && key == prefix));
  }
  __syncthreads();
  if (lane == 0) warp_gt[warp] = gts, warp_eq[warp] = eqs;
  __syncthreads();
  gts = eqs = 0;
  for (int o = 0; o < warp; ++o) gts += warp_gt[o], eqs += warp_eq[o];
  const unsigned below = (1u << lane) - 1u;
#pragma unroll 2
  for (int i0 = i_first; i0 < i_last; i0 += 32) {
    const int i = i0 + lane;
    const float x = i < i_last ? w[i] : 0.f;
    const uint32_t key = weight_key(x) & mask;
    const bool gt = i < i_last && key > prefix, eq = i < i_last && key == prefix;
    const unsigned bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
    const int my_eq = eqs + __popc(be & below);
    if (gt || (eq && my_eq < need)) {
      const int at = gts + __popc(bg & below) + min(my_eq, need);
      kept[at] = i;
      w_out[at] = x;
    }
    gts += __popc(bg);
    eqs += __popc(be);
  }
}

// Moves the rows that stay. A warp takes 32 slots of a (sequence, K / V head): each lane finds where one of them comes from and goes to, then
// lanes 0 - 15 move the key's 16-byte pieces and lanes 16 - 31 the value's, row after row (short rows several at once), GATHER_ROWS
// loads in flight. Bound by memory: 2 x 2 D bytes read and written a row. A row whose page is not there reads as NaN.
constexpr int GATHER_ROWS = 4;
__global__ void __launch_bounds__(256) kfa_cache_gather_kernel(const EvictParams p) {
  wait_for_previous();
  let_next_begin();
  const unsigned group = blockIdx.x * 8u + (threadIdx.x >> 5);
  if (group >= p.total) return;
  const int lane = threadIdx.x & 31;
  const unsigned row = p.by_slot.div(group), first = (group - row * p.by_slot.d) * 32u;  // (sequence, head); first slot
  const unsigned b = p.by_head.div(row), g = row - b * p.by_head.d;
  const int i = static_cast<int>(first) + lane;
  int pos = -1, page = 0, slot = 0, page_o = -1, slot_o = 0;
  bool lost = false;
  if (i < (p.clear ? p.room : p.keep)) {
    if (i < p.keep) pos = p.kept[static_cast<long long>(row) * p.keep + i];
    lost = pos >= 0 && !cache_place(p.c, b, pos, page, slot);
    const bool nowhere = (pos >= 0 || p.clear) && !cache_place(p.out, b, i, page_o, slot_o);
    if (nowhere) page_o = -1;
    if (lost) pos = -1;
    if (lost || nowhere) report(p.status, DEV_BAD_CACHE);
  }
  const unsigned all_lost = __ballot_sync(0xffffffffu, lost);
  const unsigned live = __ballot_sync(0xffffffffu, page_o >= 0);
  if (live == 0) return;
  const bool values = lane >= 16;
  const int pieces = p.c.cols / 8, span = pieces > 8 ? 16 : (pieces > 4 ? 8 : 4), at_once = 16 / span;  // rows at once
  const int mine = (lane & 15) / span, piece = (lane & 15) % span;
  const uint8_t* from = (values ? p.c.v + g * p.c.v_sh : p.c.k + g * p.c.k_sh) + 16 * piece;
  uint8_t* to = (values ? p.out.v + g * p.out.v_sh : p.out.k + g * p.out.k_sh) + 16 * piece;
  const long long f_n = values ? p.c.v_sn : p.c.k_sn, f_s = values ? p.c.v_ss : p.c.k_ss;
  const long long t_n = values ? p.out.v_sn : p.out.k_sn, t_s = values ? p.out.v_ss : p.out.k_ss;
  for (int r0 = 0; r0 < 32; r0 += GATHER_ROWS * at_once) {
    uint4 x[GATHER_ROWS];
    uint8_t* dst[GATHER_ROWS];
#pragma unroll
    for (int k = 0; k < GATHER_ROWS; ++k) {
      const int r = (r0 + k * at_once + mine) & 31;
      const int at = __shfl_sync(0xffffffffu, pos, r), pg = __shfl_sync(0xffffffffu, page, r), sl = __shfl_sync(0xffffffffu, slot, r);
      const int pg_o = __shfl_sync(0xffffffffu, page_o, r), sl_o = __shfl_sync(0xffffffffu, slot_o, r);
      const uint32_t fill = (all_lost >> r) & 1u ? 0x7fff7fffu : 0u;
      dst[k] = nullptr;
      x[k] = make_uint4(fill, fill, fill, fill);
      if (pg_o < 0 || piece >= pieces || r0 + k * at_once + mine >= 32) continue;
      if (at >= 0) x[k] = *reinterpret_cast<const uint4*>(from + pg * f_n + sl * f_s);
      dst[k] = to + pg_o * t_n + sl_o * t_s;
    }
#pragma unroll
    for (int k = 0; k < GATHER_ROWS; ++k)
      if (dst[k] != nullptr) *reinterpret_cast<uint4*>(dst[k]) = x[k];
  }
}

}  // namespace kfa
