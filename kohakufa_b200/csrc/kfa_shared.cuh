// Attention behind shared prefixes: sequences of a batch that go on from a few prefixes, which are stored, and read, once.
//
//   a row's softmax over (its prefix, its sequence's cache, the new tokens) is that of two parts:
//   m = max(m1, m2),  l = l1 2^(m1 - m) + l2 2^(m2 - m),  O = (O1 2^(m1 - m) + O2 2^(m2 - m)) / l
//
// with P = 2^(S c - m). The reference m is the largest score when it was taken times c = scale * log2 e, rounded: P, l and O of a part belong to it as it is
// stored, so that its rounding cancels, and an exponent is one multiply-add. P goes into the second product in the values' 16-bit type, which a product has for both
// operands: each is off by at most u = eps / 2 of itself, the output by u sum p |v| besides its own rounding. l is the sum of the P before that. (Outputs against
// 64 bits, norm of the difference over the norm: bf16 2.4e-3, fp16 2.7e-4 to 2.9e-4; P in fp32 and rounded once at the end 1.7e-3 and 2.1e-4.)
//
// What bounds it: the keys and values, each read once; and where many rows share a long prefix the two products and the exponentials. One kernel does both
// parts side by side: its CTAs have two halves, each a stream of its own, and a CTA takes either two stretches of the prefixes' work or two of the
// sequences' own, as many CTAs as each has of the work (lengths are known on the device only). (Not one half of each: the two loops do not fit into an
// SM's instruction cache together. A prefix' tile took 4000 clk beside an own one and that 3800, two of a kind take 1900 and 2800.) Both kinds are cut
// by keys as in kfa_attend.cuh. A prefix's row tile has the rows of several sequences (sequences, tokens, heads of a K / V head, up to 256), whose queries one TMA box
// brings; a prefix is read once for each of them, out of L2 but the first time.
// Graph time with 32 / 8 heads, D = 128: 64 sequences behind 8192 positions, 1 to 1024 of their own, one token 50 us (floor 28, memory; the prefix first, its join, then
// the own part 76); 32 behind 8192, trees of 8 tokens 71 (floor 17); 256 behind 32768, 200 to 2048 of their own 280 (floor 208). A tile of 256 rows x 64 keys takes
// 2030 clk, an own one of 128 keys 2800 to 3300 (0.9 of the copy rate), what lies between two own items 7000.
//
// More than 128 rows of a prefix: a tile has up to 256, half of them in each half of the CTA, which share its keys and values. (They are
// copied once a CTA then: two halves with tiles of their own ask L2 for 30 bytes a clock and SM.) Where there is one prefix, the row tiles of a K / V head are cut at the same
// keys, and CTAs that run together read the same.
//
// What a part leaves is fp32: O before the division, m, l and the largest score per row. Items that one CTA has whole go to the carry, rows (sequence,
// head, token); parts of cut ones to the CTA's slots; the item's entry in a directory says which. A second kernel gives every row a warp, which
// takes its prefix' parts and its own in the order of the keys: results repeat bit for bit.
//
// The halves know nothing of one another (kfa_attend.cuh's two streams share their items): an item's end and the next one's beginning pass while the other half
// works. Up to 32 rows (N = 16, 32): keys as matrix rows, tiles of 128 keys. More (N = 128): rows as matrix rows, tiles of 64 keys, P in tensor memory.
//
//   warps 0-3 of a half's eight  softmax, O
//   warp 4                       MMA issue
//   warps 5, 6                   TMA producers: keys and queries, values
#pragma once

#include <type_traits>

#include "kfa_attend.cuh"

namespace kfa {

constexpr int SH_THREADS = 256, SH_SMEM = 115712;  // of a half
// Registers per thread: 128 at the start (65536 / 512); the issuing warps' go to the softmax warps.
constexpr int SH_REGS = 128, SH_REGS_STREAM = 176, SH_REGS_ISSUE = 80;
static_assert(128 * (SH_REGS_STREAM + SH_REGS_ISSUE) <= SH_THREADS * SH_REGS, "register budgets exceed the CTA's allocation");
constexpr int SH_TMEM = 256;  // columns of a half

struct SharedParams {
  AttendParams pre, own;
  float weight;   // what a unit of the prefixes, of a CTA, counts beside one of the sequences' own, of a half
  int pre_items;  // where there is one prefix: its items; else 0
  int pre_pair;   // whether a prefix' row tile takes both halves of a CTA
  int halves;     // of all CTAs
};

// Shared memory and barriers of a half, whichever work it has: 1 KB of barriers and control, then its rings. N = 256: of the whole CTA, whose first half
// has the rings and their barriers.
template <int NC_, int N>
struct ShCfg {
  static constexpr int NC = NC_;
  static constexpr bool ROWS = N >= 128, PAIR = N == 256, KEYS_FIRST = true;
  static constexpr int KEYS = ROWS ? 64 : 128, UNITS = KEYS / ATT_UNIT;
  static constexpr int CHUNK = KEYS * 128, STAGE = NC * CHUNK;  // KEYS keys x 64 columns
  static constexpr int Q_CHUNK = N * 128, Q_BYTES = NC * Q_CHUNK, NQ = ROWS ? 1 : 2;
  static constexpr int NP = ROWS ? 2 : 1;                  // buffers for P
  static constexpr int P_BYTES = ROWS ? 0 : 128 * N * 2;   // in shared memory
  // column maxima of two tiles, shifts, sums and maxima of two segments; rows on their way out
  static constexpr int OTHER = ROWS ? (PAIR ? 8 : 4) * 2048 : (2 * 4 * N + 4 * N + 2 * 6 * N) * 4;
  static constexpr int FIXED = 1024 * (PAIR ? 3 : 2) + NQ * Q_BYTES + P_BYTES + OTHER;
  static constexpr int FIT = ((PAIR ? 2 * SH_SMEM : SH_SMEM) - FIXED) / STAGE;
  static constexpr int DV = (FIT + 1) / 2 < 4 ? (FIT + 1) / 2 : 4;  // (of three stages two: values stay until a tile is done with, keys only until its scores are made)
  static constexpr int DK = FIT - DV < 4 ? FIT - DV : 4;
  static_assert(DV >= 1 && DK >= 1, "no room for a tile of keys and one of values");
  static constexpr int RINGS = 1, NS = DK + DV;
  static constexpr int SMEM = FIXED + NS * STAGE;
  __device__ static __forceinline__ int k_stage(int T) { return T % DK; }
  __device__ static __forceinline__ int v_stage(int T) { return DK + T % DV; }
  __device__ static __forceinline__ int k_turn(int T) { return T / DK; }
  __device__ static __forceinline__ int v_turn(int T) { return T / DV; }
  // barriers, the same for both kinds of work: see AttRings
  static constexpr int B_Q = 0, B_S = 2, B_P = 4, B_PV = 6, B_QFREE = 8, B_OFREE = 10, B_DRAIN = 11, B_KV = 12, B_KVFREE = 20, N_BARS = 28;
};

// Sum over the CTA's threads; s: 16 numbers of shared memory. Synchronises.
__device__ __forceinline__ long long sh_sum(long long x, long long* s) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = x;
  __syncthreads();
  long long all = 0;
#pragma unroll
  for (int i = 0; i < 2 * SH_THREADS / 32; ++i) all += s[i];
  return all;
}

// What b has of the work, as it is counted.
template <int MODE>
__device__ __forceinline__ int sh_counted(const AttendParams& p, int b) {
  using W = WalkOf<MODE>;
  return b < p.c.batch ? (W::units_of(p, b) + p.extra) * W::items_of(p, b) : 0;
}

// The stretch of half (or CTA) `index` of `count` that share this work, `total` as it is counted. s_i: 32 ints of shared memory. Synchronises the CTA,
// whose halves both come here. split: of one prefix: every item is cut into so many stretches; 0: all stretches have the same length.
template <int MODE>
__device__ __forceinline__ bool sh_work(const AttendParams& p, int* s_i, int index, int count, int total, int split, WalkOf<MODE>& w, int& chunk,
                                        int& end) {
  using W = WalkOf<MODE>;
  const int tid = threadIdx.x & (SH_THREADS - 1), warp = tid >> 5, lane = tid & 31;
  chunk = 0;
  if (split > 0) {
    const int items = W::items_of(p, 0), each = total / items, long_ones = each % split, length = each / split;
    auto unit = [&](int i) { return max(length * i + min(i, long_ones) - p.extra, 0); };
    w.b = 0;
    w.item = index / split;
    const int k = index - w.item * split;
    w.unit = unit(k);
    w.end_b = 0;
    w.end_item = k + 1 < split ? w.item : w.item + 1;
    w.end_unit = k + 1 < split ? unit(k + 1) : 0;
    if (w.end_item == items) w.end_b = p.c.batch, w.end_item = 0;
    end = 0;
    __syncthreads();
    return w.item < items && w.start(p);
  }
  chunk = max((total + count - 1) / count, p.least);
  const int at[2] = {chunk * index, chunk * index + chunk};
  end = at[1];
  int before = 0;
  for (int b0 = 0; b0 < p.c.batch; b0 += SH_THREADS) {
    const int own = sh_counted<MODE>(p, b0 + tid);
    int upto = own;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += up;
    }
    __syncthreads();
    if (lane == 31) s_i[8 + warp] = upto;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int i = 0; i < SH_THREADS / 32; ++i) {
      const int x = s_i[8 + i];
      if (i < warp) upto += x;
      all += x;
    }
    upto += before;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (at[i] >= upto - own && at[i] < upto) {
        const int b = b0 + tid, off = at[i] - (upto - own), each = own / W::items_of(p, b), item = off / each;
        s_i[3 * i] = b;
        s_i[3 * i + 1] = item;
        s_i[3 * i + 2] = max(off - item * each - p.extra, 0);
      }
    before += all;
  }
  __syncthreads();
  const bool inside[2] = {at[0] < total, at[1] < total};
  w.b = inside[0] ? s_i[0] : p.c.batch;
  w.item = inside[0] ? s_i[1] : 0;
  w.unit = inside[0] ? s_i[2] : 0;
  w.end_b = inside[1] ? s_i[3] : p.c.batch;
  w.end_item = inside[1] ? s_i[4] : 0;
  w.end_unit = inside[1] ? s_i[5] : 0;
  return w.b < p.c.batch && w.start(p);
}

// See part_factor, for references that are scaled.
__device__ __forceinline__ float sh_factor(float m, float l, float m_all) {
  if (m == -INFINITY) return l == 0.f ? -1.f : 1.f;
  return ex2(m - m_all);
}
constexpr float SH_SLACK = 8.f;  // how far a maximum may grow before O is rescaled: a factor of 2^8

// How many CTAs the prefixes' work gets, and into how many stretches each of its items is cut (0: wherever stretches end).
template <bool PAIR>
__device__ __forceinline__ void sh_share(const SharedParams& p, int total_pre, int total_own, int grid, int& pre_ctas, int& split) {
  split = 0;
  const float pre = total_pre * p.weight, own = 0.5f * total_own;  // a CTA's time for all of it (own: two halves work at once)
  const float most = static_cast<float>(grid - 1);                 // (the own work is never nothing)
  pre_ctas = total_pre == 0 ? 0 : static_cast<int>(fminf(fmaxf(grid * __fdividef(pre, pre + own) + 0.5f, 1.f), most));
  if (total_pre == 0 || p.pre_items == 0) return;
  // one prefix: so many stretches an item that what ends last ends first
  const float per = PAIR ? 1.f : 0.5f;  // CTAs of a stretch
  const float stretch = per * p.pre_items, ideal = __fdividef(static_cast<float>(pre_ctas), stretch);
  float best = 0.f;
  const float continuous = pre_ctas;
  const int each = total_pre / p.pre_items;  // (a stretch has a unit at least)
  for (int s = max(static_cast<int>(ideal), 1); s <= min(static_cast<int>(ideal) + 1, max(each / p.pre.least, 1)); ++s) {
    const float ctas = ceilf(s * stretch);
    if (ctas > most) break;
    const float time = fmaxf(__fdividef(pre, s * stretch), __fdividef(own, grid - ctas));
    if (split == 0 || time < best) {
      best = time;
      split = s;
      pre_ctas = static_cast<int>(ctas);
    }
  }
  // Fewer CTAs than items: cut where stretches end. Where they are few less every item gets a stretch all the same, so that those of a K / V head read the same keys.
  // us with a stretch an item, and cut anywhere: 256 sequences behind 4096 positions with 300 of their own (ideal 0.94) 89, 101, 400 (0.84) 98, 111, 500 (0.75)
  // 110, 123, 600 (0.69) 125, 130, 800 (0.59) 155, 162; 128 sequences with 1400 (0.81) 132, 134. (So whole items would pay below 0.8 as well.)
  if (split > 0 && ideal < 0.8f) {
    split = 0;
    pre_ctas = static_cast<int>(continuous);
  }
}

// Where a segment's rows go: the carry, or one of the half's two slots of parts.
struct ShOut {
  float* o;       // rows of 128
  float* ml;      // m; l and the largest score `plane` further each
  long long plane;
  bool whole;
  template <class W>
  __device__ __forceinline__ ShOut(const AttendParams& p, const W& w, int half) {
    whole = w.begins() && w.ends();
    const long long slot = 2ll * half + (w.begins() ? 1 : 0);
    o = whole ? p.carry_o : p.part_o + slot * p.rows * 128;
    ml = whole ? p.carry_ml : p.part_ml + slot * 3 * p.rows;
    plane = whole ? p.carry_rows : p.rows;
  }
  __device__ __forceinline__ long long row(const AttendParams& p, int r, int b, int h, int t) const {
    return whole ? (static_cast<long long>(b) * p.H + h) * p.T + t : r;
  }
};

struct ShHalf {
  uint32_t sKV, sQ, sP, bar0, tmem;
  uint32_t ring0;       // the barriers of keys, values and queries (of a pair: the first half's)
  uint8_t* other;       // OTHER bytes
  int half, index;      // among all halves; among those (of a pair: the CTAs) that have this kind of work
  int chunk, end, split;  // see sh_work
  int *kv_issued, *q_issued;
  __device__ __forceinline__ void meet() const { asm volatile("bar.sync %0, 128;" ::"r"(1 + (half & 1)) : "memory"); }  // of the softmax warps
};

// The directory's entry of the item that begins here.
template <int MODE, class W>
__device__ __forceinline__ void sh_note(const AttendParams& p, const W& w, const RowMapOf<MODE>& rows, const ShHalf& x) {
  if (!w.begins()) return;
  int parts = 0;
  if (!w.ends()) parts = x.split > 0 ? x.split - x.index % x.split : (x.end - w.n + w.units - 1) / x.chunk - x.index + 1;
  p.dir[(static_cast<long long>(rows.g) * p.row_tiles + rows.rt) * p.seqs + rows.s0] = make_int2(x.half, parts);
}

// Values behind the end may be anything, and 0 * NaN is no 0: see clean_values of kfa_attend.cuh. Here the row of a new token is looked at where it has landed:
// a look into global memory ahead of the scores cost 4700 clk a segment. Whether any of its values were left out.
template <class R, bool BF16>
__device__ __forceinline__ bool sh_clean(uint32_t stage, int key, bool valid, bool fresh) {
  const uint32_t row = stage + key * 128;
  bool odd = false;
  if (!valid) {
#pragma unroll
    for (int i = 0; i < R::NC * 8; ++i)  // (rows begin at the same bank: each thread in an order of its own)
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(row + (i >> 3) * R::CHUNK + (((i ^ key) & 7) << 4)), "r"(0) : "memory");
  } else if (fresh) {
#pragma unroll 4
    for (int i = 0; i < R::NC * 8; ++i) {
      const uint32_t at = row + (i >> 3) * R::CHUNK + ((i & 7) << 4);
      uint32_t q[4];
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]) : "r"(at) : "memory");
      bool here = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (odd_half<BF16>(q[j])) q[j] &= 0xffff0000u, here = true;
        if (odd_half<BF16>(q[j] >> 16)) q[j] &= 0xffffu, here = true;
      }
      if (here) asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3]) : "memory");
      odd |= here;
    }
  }
  return odd;
}

// Suspended until the phase is over, or for about 100 ns.
__device__ __forceinline__ void mbar_nap(uint32_t bar, uint32_t parity) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%0], %1, %2;\n\t}" ::"r"(bar), "r"(parity), "r"(100u)
      : "memory");
}
// The issuing warps' loop: see att_issue. Scores of tile i as soon as their keys (and queries) are there and the values of tile i - 2 have been issued, values
// of tile j as soon as P and V are there, whichever comes first. Where nothing can go the warp is suspended: one that polls takes issue slots from those that
// compute.
template <class R, class W, typename FS, typename FP>
__device__ __forceinline__ void sh_issue(const AttendParams& p, const W& first, const ShHalf& x, const AttCtl& ac, FS issue_S, FP issue_PV) {
  uint32_t held = 0, held_parity = 0;  // what the last test failed at
  auto ready = [&](uint32_t bar, uint32_t parity) {
    const bool there = __all_sync(0xffffffffu, mbar_test(bar, parity));
    if (!there) held = bar, held_parity = parity;
    return there;
  };
  auto ring = [&](int i) { return x.ring0 + 8u * i; };
  auto bar = [&](int i) { return x.bar0 + 8u * i; };
  AttTiles<true, R::UNITS, W> tiles{first, 0};
  AttTile ahead = {0, 0, 0, false, false}, even = ahead, odd = ahead;  // the next to get scores; those that have, by tile (at most two wait for values)
  bool have = tiles.take(p, ahead);
  int i_s = 0, i_p = 0;  // tiles whose scores and whose values are issued
  long long t0 = clock64();
  while (have || i_p < i_s) {
    bool went = false;
    if (have && i_s <= i_p + 1 && ready(ring(R::B_KV + R::k_stage(ahead.T)), R::k_turn(ahead.T) & 1) &&
        (!ahead.opens || ready(ring(R::B_Q + ahead.s % R::NQ), (ahead.s / R::NQ) & 1))) {
      tc_fence_after();
      issue_S(ahead, i_s);
      if (i_s & 1) odd = ahead;
      else even = ahead;
      ++i_s;
      went = true;
      have = tiles.take(p, ahead);
    }
    if (i_p < i_s) {
      const AttTile now = (i_p & 1) ? odd : even;
      if (ready(bar(R::B_P + i_p % R::NP), (i_p / R::NP) & 1) && ready(ring(R::B_KV + R::v_stage(now.T)), R::v_turn(now.T) & 1) &&
          (!now.opens || now.uses == 0 || ready(bar(R::B_OFREE), (now.uses - 1) & 1))) {
        tc_fence_after();
        issue_PV(now, i_p);
        ++i_p;
        went = true;
      }
    }
    if (went) {
      t0 = clock64();
    } else if (*ac.abort != 0) {
      break;
    } else if (clock64() - t0 > KFA_WAIT_CYCLES) {
      *ac.abort = KFA_DEV_TIMEOUT_BASE + 73;
      break;
    } else {
      mbar_nap(held, held_parity);
    }
  }
  // what was issued has retired before tensor memory is freed
  const bool lead = elect_one();
  umma_commit_lead(lead, bar(R::B_DRAIN));
  mbar_drain(bar(R::B_DRAIN), 0);
}

// ---- up to 32 rows: keys as matrix rows ---------------------------------------------------------------------------------------
template <int NC, int N, bool BF16, int MODE>
__device__ __forceinline__ void sh_columns(const AttendParams& p, const WalkOf<MODE>& first, const ShHalf& x, const AttCtl& ac, const CUtensorMap* tmQ,
                                           const CUtensorMap* tmK, const CUtensorMap* tmV, const CUtensorMap* tmKn, const CUtensorMap* tmVn) {
  using R = ShCfg<NC, N>;
  const int tid = threadIdx.x & (SH_THREADS - 1), warp = warp_index() & 7, lane = tid & 31;
  auto bar = [&](int i) { return x.bar0 + 8u * i; };
  const Ctl ctl{ac.abort};
  const uint32_t tmS = x.tmem, tmO = x.tmem + 2 * N;
  if (warp > 4) {
    reg_budget<SH_REGS_ISSUE, SH_REGS>();
    if (warp < 7) {
      const bool values = warp == 6;
      att_produce<R>(p, first, values, x.sKV, x.sQ, x.bar0, ac, tmQ, values ? tmV : tmK, values ? tmVn : tmKn, *x.kv_issued, *x.q_issued);
    }
  } else if (warp == 4) {
    reg_budget<SH_REGS_ISSUE, SH_REGS>();
    const bool lead = elect_one();
    constexpr uint32_t IDESC_S = make_idesc(BF16, false, 128, N), IDESC_O = make_idesc(BF16, true, 128, N) | (1u << 15);
    constexpr uint32_t HI_P = sdesc_hi_for(N);
    const int k_steps = (p.c.cols + 15) / 16;
    sh_issue<R>(
        p, first, x, ac,
        [&](const AttTile& t, int c) {
          const uint32_t k_lo = sdesc_lo(x.sKV + R::k_stage(t.T) * R::STAGE, 16), q_lo = sdesc_lo(x.sQ + (t.s % R::NQ) * R::Q_BYTES, 16);
#pragma unroll 2
          for (int kk = 0; kk < k_steps; ++kk)
            umma_ss_lead2(lead, tmS + (c & 1) * N, k_lo + (((kk >> 2) * R::CHUNK + (kk & 3) * 32) >> 4), SDESC_HI,
                          q_lo + (((kk >> 2) * R::Q_CHUNK + (kk & 3) * 32) >> 4), SDESC_HI, IDESC_S, kk > 0 ? 1u : 0u);
          umma_commit_lead(lead, bar(R::B_S + (c & 1)));
          umma_commit_lead(lead, bar(R::B_KVFREE + R::k_stage(t.T)));
          if (t.closes) umma_commit_lead(lead, bar(R::B_QFREE + t.s % R::NQ));
        },
        [&](const AttTile& t, int) {
          // (64 columns or fewer: the matrix' rows 64 .. 127 repeat the first ones, and nobody reads them)
          const uint32_t v_lo = sdesc_lo(x.sKV + R::v_stage(t.T) * R::STAGE, NC == 2 ? R::CHUNK : 0), p_lo = sdesc_lo(x.sP, 16);
#pragma unroll 2
          for (int kk = 0; kk < 8; ++kk)
            umma_ss_lead2(lead, tmO, v_lo + ((kk * 16 * 128) >> 4), SDESC_HI, p_lo + ((kk * 16 * 2 * N) >> 4), HI_P, IDESC_O,
                          (!t.opens || kk > 0) ? 1u : 0u);
          umma_commit_lead(lead, bar(R::B_PV));
          umma_commit_lead(lead, bar(R::B_KVFREE + R::v_stage(t.T)));
        });
  } else {
    // (After a wait that ran out the role goes on without waiting: its warps meet at barriers.)
    reg_budget<SH_REGS_STREAM, SH_REGS>();
    const uint32_t lane_base = static_cast<uint32_t>(warp * 32) << 16;
    const int col = lane & (N - 1);                           // whose maximum a lane keeps
    float* s_max = reinterpret_cast<float*>(x.other);         // [tile & 1][warp][N]
    float* shift = s_max + 8 * N + warp * N;                  // [N]
    float* s_fin = s_max + 12 * N;                            // [segment & 1]: l of four warps, m, largest score, each [N]
    const float c_log2 = p.c_log2;
    const float2 c2 = make_float2(c_log2, c_log2);
    WalkOf<MODE> w = first;
    bool more = true, ok = true;
    int c = 0, s = 0;  // tiles and segments
    while (more) {
      const RowMapOf<MODE> rows(p, w.b, w.item);
      float l[N], m_ref = -INFINITY, m_top = -INFINITY;
#pragma unroll
      for (int i = 0; i < N; ++i) l[i] = 0.f;
      // the new tokens that see token `lane`, a bit each; all of them lie in the item's last unit (no more tokens than rows). Asked for ahead of the tiles.
      uint32_t see_new = 0u;
      if (MODE == ATT_OWN && w.ud > 0) {
        const int n = min(min(p.tt, p.T - rows.t0), w.count - rows.t0);
        see_new = n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u);
        if (p.tree == nullptr) {
          if (lane > rows.t0) see_new &= lane - rows.t0 >= 32 ? 0u : 0xffffffffu << (lane - rows.t0);
        } else if (n > 0 && lane < w.count) {
          see_new = tree_bits(p.tree + w.b * p.tree_sb + rows.t0 * p.tree_st + lane * p.tree_sj, p.tree_st, n);
        }
      }
      const int tiles = w.template tiles<R::UNITS>(), c0 = c;
      const int t_full = max(min(w.n, min(w.len / ATT_UNIT, w.uc) - w.unit), 0) / R::UNITS;  // tiles below hold cached keys only
      // (The masked tiles, an item's last ones, have code of their own: it does not share the instruction cache with the loop over the others.)
      auto tile = [&](auto masked, int t) {
        constexpr bool full = !decltype(masked)::value;
        int fresh = -1;
        const bool valid = full || which_key(w, w.unit + R::UNITS * t, tid & 127, fresh);
        const uint32_t see = !valid ? 0u : (fresh >= 0 ? see_new : 0xffffffffu);
        if (ok) ok = wait_warp(bar(R::B_S + (c & 1)), (c >> 1) & 1, ctl, 78);
        tc_fence_after();
        float e[N];
        tmem_ld_cols<N>(tmS + lane_base + (c & 1) * N, e);
        tmem_wait_ld();
        if constexpr (!full) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const int dt = fresh >= 0 ? static_cast<int>(p.by_gt.div(i)) : 0;
            if (!((see >> (dt & 31)) & 1u)) e[i] = -INFINITY;
          }
        }
        // ---- column maxima ----
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float y = warp_max(e[i]);
          if (col == i) top = y;
        }
        float* mx = s_max + (c & 1) * 4 * N;
        if (lane < N) mx[warp * N + lane] = top;
        x.meet();
        const float raw = fmaxf(fmaxf(mx[col], mx[N + col]), fmaxf(mx[2 * N + col], mx[3 * N + col])), y = raw * c_log2;
        m_top = fmaxf(m_top, raw);
        const bool move = m_ref == -INFINITY ? y > -INFINITY : y > m_ref + SH_SLACK;
        float alpha = 1.f;
        if (move) {
          alpha = m_ref == -INFINITY ? 0.f : ex2(m_ref - y);
          m_ref = y;
        }
        if (lane < N) shift[col] = m_ref == -INFINITY ? 0.f : -m_ref;
        const bool grew = __any_sync(0xffffffffu, move);  // the same in all warps
        __syncwarp();
        if (c > 0 && ok) ok = wait_warp(bar(R::B_PV), (c - 1) & 1, ctl, 80);  // P and O are free
        if (__builtin_expect(grew && c > c0, 0)) {
          // sums and O of the earlier tiles, to the new maxima
          tc_fence_after();
#pragma unroll
          for (int i = 0; i < N; i += 16) {
            float o[16];
            tmem_ld16(tmO + lane_base + i, reinterpret_cast<uint32_t*>(o));
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float a = __shfl_sync(0xffffffffu, alpha, i + j);
              o[j] *= a;
              l[i + j] *= a;
            }
            tmem_st16(tmO + lane_base + i, reinterpret_cast<const uint32_t*>(o));
          }
          tmem_wait_st();
        }
        // ---- P ----
#pragma unroll
        for (int i = 0; i < N; i += 8) {
          const float4 a = *reinterpret_cast<const float4*>(shift + i), b = *reinterpret_cast<const float4*>(shift + i + 4);
          const float2 mm[4] = {make_float2(a.x, a.y), make_float2(a.z, a.w), make_float2(b.x, b.y), make_float2(b.z, b.w)};
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            const float2 z = __ffma2_rn(make_float2(e[i + j], e[i + j + 1]), c2, mm[j / 2]);
            e[i + j] = ex2(z.x);
            e[i + j + 1] = ex2(z.y);
            const float2 sum = __fadd2_rn(make_float2(l[i + j], l[i + j + 1]), make_float2(e[i + j], e[i + j + 1]));
            l[i + j] = sum.x;
            l[i + j + 1] = sum.y;
          }
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(x.sP + p_piece<N>(tid & 127, i / 8)), "r"(pack16<BF16>(e[i], e[i + 1])),
                       "r"(pack16<BF16>(e[i + 2], e[i + 3])), "r"(pack16<BF16>(e[i + 4], e[i + 5])), "r"(pack16<BF16>(e[i + 6], e[i + 7]))
                       : "memory");
        }
        if constexpr (!full) {
          if (ok) ok = wait_warp(bar(R::B_KV + R::v_stage(c)), R::v_turn(c) & 1, ctl, 82);
          if (sh_clean<R, BF16>(x.sKV + R::v_stage(c) * R::STAGE, tid & 127, valid, fresh >= 0)) ac.odd[0] = s + 1;
        }
        fence_async_smem();
        tc_fence_before();
        mbar_arrive(bar(R::B_P));
      };
#pragma unroll 1
      for (int t = 0; t < min(t_full, tiles); ++t, ++c) tile(std::false_type{}, t);
#pragma unroll 1
      for (int t = t_full; t < tiles; ++t, ++c) tile(std::true_type{}, t);
      // ---- the segment's end ----
      const ShOut to(p, w, x.half);
      columns_over_lanes<N>(l, lane);
      float* fin = s_fin + (s & 1) * 6 * N;
      if constexpr (N == 32) {
        fin[warp * N + lane] = l[0];
      } else {
        if (!(lane & 1)) fin[warp * N + lane / 2] = l[0];
      }
      if (warp == 0 && lane < N) {
        fin[4 * N + lane] = m_ref;
        fin[5 * N + lane] = m_top;
      }
      int h, tk, sq;
      const bool exists = rows.row(p, col, h, tk, sq);
      const long long at = exists ? to.row(p, col, sq, h, tk) : -1;
      if (tid == 0) sh_note<MODE>(p, w, rows, x);
      if (ok) ok = wait_warp(bar(R::B_PV), (c - 1) & 1, ctl, 83);
      tc_fence_before();
      x.meet();
      tc_fence_after();
      float o[N];
      tmem_ld_cols<N>(tmO + lane_base, o);
      const float m = fin[4 * N + col], l_all = (fin[col] + fin[N + col]) + (fin[2 * N + col] + fin[3 * N + col]);
      if (warp == 0 && lane < N && exists) {
        to.ml[at] = m;
        to.ml[to.plane + at] = l_all;
        to.ml[2 * to.plane + at] = fin[5 * N + col];
      }
      const bool none = sh_factor(m, l_all, m) < 0.f;  // nothing was seen: O is not defined
      tmem_wait_ld();
      tc_fence_before();
      mbar_arrive(bar(R::B_OFREE));
      const int d = tid & 127;
      const bool odd = ac.odd[0] >= s + 1;
      const int j0 = max(w.unit - w.uc, 0) * ATT_UNIT, j1 = odd ? min((w.unit + w.n - w.uc) * ATT_UNIT, w.count) : 0;
      const unsigned nothing = __ballot_sync(0xffffffffu, none);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if ((nothing >> i) & 1u) o[i] = 0.f;
      if (d < p.c.cols) {
        for (int j = j0; j < j1; ++j) {
          const float y = load16<BF16>(p.v + w.b * p.v_sb + rows.g * p.v_sh + j * p.v_ss + 2 * d);
          if (fabsf(y) < INFINITY) continue;
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (sees_new(p, w, rows.t0 + static_cast<int>(p.by_gt.div(i)), j)) o[i] += y;
        }
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const long long r = __shfl_sync(0xffffffffu, at, i);
        if (r >= 0 && d < p.c.cols) to.o[r * 128 + d] = o[i];
      }
      ++s;
      more = w.next(p);
    }
  }
}

// ---- more rows: rows as matrix rows -------------------------------------------------------------------------------------------
// Tiles of 64 keys, scores and P in two buffers of 64 columns in turn: P (16-bit) lies over the first 32 columns of its scores, and while one tile's values are
// multiplied and its next scores made, the threads work on the other's.
template <int NC, int N, bool BF16, int MODE>
__device__ __forceinline__ void sh_rows(const AttendParams& p, const WalkOf<MODE>& first, const ShHalf& x, const AttCtl& ac, const CUtensorMap* tmQ,
                                        const CUtensorMap* tmK, const CUtensorMap* tmV, const CUtensorMap* tmKn, const CUtensorMap* tmVn) {
  using R = ShCfg<NC, N>;
  const int side = R::PAIR ? x.half & 1 : 0;
  constexpr int D = 64 * NC;  // columns of O (those that the head dim does not have are zeros)
  const int tid = threadIdx.x & (SH_THREADS - 1), warp = warp_index() & 7, lane = tid & 31;
  auto bar = [&](int i) { return x.bar0 + 8u * i; };
  auto ring = [&](int i) { return x.ring0 + 8u * i; };
  const Ctl ctl{ac.abort};
  if (warp > 4) {
    reg_budget<SH_REGS_ISSUE, SH_REGS>();
    if (warp < 7 && side == 0) {
      const bool values = warp == 6;
      att_produce<R>(p, first, values, x.sKV, x.sQ, x.bar0, ac, tmQ, values ? tmV : tmK, values ? tmVn : tmKn, *x.kv_issued, *x.q_issued);
    }
  } else if (warp == 4) {
    reg_budget<SH_REGS_ISSUE, SH_REGS>();
    const bool lead = elect_one();
    constexpr uint32_t IDESC_S = make_idesc(BF16, false, 128, 64), IDESC_O = make_idesc(BF16, true, 128, D);
    const uint32_t tS = x.tmem, tO = x.tmem + 128;
    const int k_steps = (p.c.cols + 15) / 16;
    sh_issue<R>(
        p, first, x, ac,
        [&](const AttTile& t, int c) {
          const uint32_t q_lo = sdesc_lo(x.sQ + (t.s % R::NQ) * R::Q_BYTES + side * 128 * 128, 16), k_lo = sdesc_lo(x.sKV + R::k_stage(t.T) * R::STAGE, 16);
#pragma unroll 2
          for (int kk = 0; kk < k_steps; ++kk)
            umma_ss_lead(lead, tS + 64 * (c & 1), q_lo + (((kk >> 2) * R::Q_CHUNK + (kk & 3) * 32) >> 4),
                         k_lo + (((kk >> 2) * R::CHUNK + (kk & 3) * 32) >> 4), IDESC_S, kk > 0 ? 1u : 0u);
          umma_commit_lead(lead, bar(R::B_S + (c & 1)));
          umma_commit_lead(lead, ring(R::B_KVFREE + R::k_stage(t.T)));
          if (t.closes) umma_commit_lead(lead, ring(R::B_QFREE + t.s % R::NQ));
        },
        [&](const AttTile& t, int c) {
          const uint32_t v_lo = sdesc_lo(x.sKV + R::v_stage(t.T) * R::STAGE, R::CHUNK);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_ts_lead(lead, tO, tS + 64 * (c & 1) + kk * 8, v_lo + ((kk * 16 * 128) >> 4), IDESC_O, (!t.opens || kk > 0) ? 1u : 0u);
          umma_commit_lead(lead, bar(R::B_PV + (c & 1)));
          umma_commit_lead(lead, ring(R::B_KVFREE + R::v_stage(t.T)));
        });
  } else {
    // (After a wait that ran out the role goes on without waiting.)
    reg_budget<SH_REGS_STREAM, SH_REGS>();
    const int r = tid & 127, tile_row = side * 128 + r;  // the thread's row of the half, of the tile
    const uint32_t lane_base = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t tS = x.tmem + lane_base, tO = x.tmem + 128 + lane_base;
    const float c_log2 = p.c_log2;
    const float2 c2 = make_float2(c_log2, c_log2);
    WalkOf<MODE> w = first;
    bool more = true, ok = true;
    int c = 0, s = 0;  // tiles and segments
    while (more) {
      const RowMapOf<MODE> rows(p, w.b, w.item);
      int h, tk, sq;
      const bool exists = rows.row(p, tile_row, h, tk, sq);
      float l = 0.f, m_ref = -INFINITY, m_top = -INFINITY;
      const int tiles = w.template tiles<R::UNITS>();
      const int t_full = max(min(w.n, min(w.len / ATT_UNIT, w.uc) - w.unit), 0) / R::UNITS;  // tiles below hold cached keys only
      float2 e[32];
      bool loaded = false;
      // (The masked tiles, an item's last ones, have code of their own: it does not share the instruction cache with the loop over the others.)
      auto tile = [&](auto masked, int t) {
        constexpr bool full = !decltype(masked)::value;
        uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
        if constexpr (!full) {
          const int ub = w.unit + R::UNITS * t;
          seen[0] = exists ? seen_word(p, w, ub, tk) : 0u;
          seen[1] = exists ? seen_word(p, w, ub + 1, tk) : 0u;
        }
        if (!loaded) {
          if (ok) ok = wait_warp(bar(R::B_S + (c & 1)), (c >> 1) & 1, ctl, 78);
          tc_fence_after();
          tmem_ld_cols<64>(tS + 64 * (c & 1), reinterpret_cast<float*>(e));
          tmem_wait_ld();
        }
        if constexpr (!full) {
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if (!((seen[j / 16] >> (2 * j & 31)) & 1u)) e[j].x = -INFINITY;
            if (!((seen[j / 16] >> ((2 * j + 1) & 31)) & 1u)) e[j].y = -INFINITY;
          }
        }
        float y[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < 32; ++j) y[j & 3] = fmaxf(y[j & 3], fmaxf(e[j].x, e[j].y));
        const float top = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
        m_top = fmaxf(m_top, top);
        const float y_top = top * c_log2;
        const bool move = m_ref == -INFINITY ? y_top > -INFINITY : y_top > m_ref + SH_SLACK;
        if (__builtin_expect(__any_sync(0xffffffffu, move), 0)) {
          const float alpha = !move ? 1.f : (m_ref == -INFINITY ? 0.f : ex2(m_ref - y_top));
          if (t > 0) {  // every product issued so far has to have retired
            if (ok) ok = wait_warp(bar(R::B_PV + ((c - 1) & 1)), ((c - 1) >> 1) & 1, ctl, 79);
            tc_fence_after();
#pragma unroll 1
            for (int k = 0; k < D; k += 16) {
              float o[16];
              tmem_ld16(tO + k, reinterpret_cast<uint32_t*>(o));
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] *= alpha;
              tmem_st16(tO + k, reinterpret_cast<const uint32_t*>(o));
            }
            tmem_wait_st();
            l *= alpha;
          }
          if (move) m_ref = y_top;
        }
        const float sh = m_ref == -INFINITY ? 0.f : -m_ref;
        const float2 s2 = make_float2(sh, sh);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int k = 0; k < 32; k += 16) {  // (stored by the half: fewer registers at once)
          uint32_t pk[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float2 z = __ffma2_rn(e[k + j], c2, s2);
            z.x = ex2(z.x);
            z.y = ex2(z.y);
            sum[j & 1] = __fadd2_rn(sum[j & 1], z);
            pk[j] = pack16<BF16>(z.x, z.y);
          }
          tmem_st16(tS + 64 * (c & 1) + k, pk);
        }
        const bool early = mbar_test(bar(R::B_S + ((c + 1) & 1)), ((c + 1) >> 1) & 1);  // the next tile's scores are there already
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        if constexpr (!full) {
          // (The tile before has to be done with: until then the barrier of this one's stage may be a turn behind.)
          if (c > 0 && ok) ok = wait_warp(bar(R::B_PV + ((c - 1) & 1)), ((c - 1) >> 1) & 1, ctl, 81);
          if (ok) ok = wait_warp(ring(R::B_KV + R::v_stage(c)), R::v_turn(c) & 1, ctl, 82);
          if (r < R::KEYS) {
            int fresh = -1;
            const bool valid = which_key(w, w.unit + R::UNITS * t, r, fresh);
            if (sh_clean<R, BF16>(x.sKV + R::v_stage(c) * R::STAGE, r, valid, fresh >= 0)) ac.odd[0] = s + 1;
          }
          fence_async_smem();
        }
        // The next tile's scores are fetched while P is on its way into tensor memory. (A wait costs 300 clk even for what is there, the way
        // in 200.)
        loaded = t + 1 < tiles && __all_sync(0xffffffffu, early);
        auto announce = [&] {
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(bar(R::B_P + (c & 1)));
        };
        if (loaded) {  // (load and wait in one piece of straight code: nothing moves the registers in between)
          tc_fence_after();
          tmem_ld_cols<64>(tS + 64 * ((c + 1) & 1), reinterpret_cast<float*>(e));
          announce();
          tmem_wait_ld();
        } else {
          announce();
        }
      };
#pragma unroll 1
      for (int t = 0; t < min(t_full, tiles); ++t, ++c) tile(std::false_type{}, t);
#pragma unroll 1
      for (int t = t_full; t < tiles; ++t, ++c) tile(std::true_type{}, t);
      // ---- the segment's end ----
      const ShOut to(p, w, x.half);
      const long long at = exists ? to.row(p, r, sq, h, tk) : -1;
      if (tid == 0 && side == 0) sh_note<MODE>(p, w, rows, x);
      if (exists) {
        to.ml[at] = m_ref;
        to.ml[to.plane + at] = l;
        to.ml[2 * to.plane + at] = m_top;
      }
      const bool none = sh_factor(m_ref, l, m_ref) < 0.f;  // nothing was seen: O is not defined
      if (ok) ok = wait_warp(bar(R::B_PV + ((c - 1) & 1)), ((c - 1) >> 1) & 1, ctl, 83);
      tc_fence_before();
      x.meet();  // (what the threads have met of values that are not finite)
      tc_fence_after();
      const bool odd = ac.odd[0] >= s + 1;
      const int j0 = max(w.unit - w.uc, 0) * ATT_UNIT, j1 = odd ? min((w.unit + w.n - w.uc) * ATT_UNIT, w.count) : 0;
      // A thread holds a row, and a store of 16 bytes by each of 32 rows touches 32 lines: through 2 KB a warp of shared memory pieces of 64 bytes of 8
      // rows are written at once.
      const uint32_t turn = (lane >> 1) & 3;
      const uint32_t out_stage = smem_u32(x.other) + warp * 2048;  // 32 rows of 64 bytes
#pragma unroll 1
      for (int i = 0; i < D; i += 16) {
        if (i >= p.c.cols) break;
        float o[16];
        tmem_ld16(tO + i, reinterpret_cast<uint32_t*>(o));
        tmem_wait_ld();
        if (none) {
#pragma unroll
          for (int j = 0; j < 16; ++j) o[j] = 0.f;
        }
        for (int j = j0; j < j1; ++j) {
          if (!exists || !sees_new(p, w, tk, j)) continue;
          const uint8_t* v = p.v + w.b * p.v_sb + rows.g * p.v_sh + j * p.v_ss + 2 * i;
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            if (i + k >= p.c.cols) break;
            const float z = load16<BF16>(v + 2 * k);
            if (!(fabsf(z) < INFINITY)) o[k] += z;
          }
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j)
          asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(out_stage + lane * 64 + ((j ^ turn) << 4)), "f"(o[4 * j]), "f"(o[4 * j + 1]),
                       "f"(o[4 * j + 2]), "f"(o[4 * j + 3])
                       : "memory");
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = 8 * k + (lane >> 2), piece = lane & 3;
          const long long to_row = __shfl_sync(0xffffffffu, at, row);
          float4 z;
          asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(z.x), "=f"(z.y), "=f"(z.z), "=f"(z.w)
                       : "r"(out_stage + row * 64 + ((piece ^ ((row >> 1) & 3)) << 4))
                       : "memory");
          if (to_row >= 0) *reinterpret_cast<float4*>(to.o + to_row * 128 + i + 4 * piece) = z;
        }
      }
      tc_fence_before();
      mbar_arrive(bar(R::B_OFREE));
      ++s;
      more = w.next(p);
    }
  }
}

template <int NC, int N_PRE, int N_OWN, bool BF16>
__global__ void __launch_bounds__(2 * SH_THREADS, 1)
kfa_shared_kernel(const __grid_constant__ CUtensorMap tmQp, const __grid_constant__ CUtensorMap tmKp, const __grid_constant__ CUtensorMap tmVp,
                  const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ CUtensorMap tmKn, const __grid_constant__ CUtensorMap tmVn, const __grid_constant__ SharedParams p) {
  using RP = ShCfg<NC, N_PRE>;
  using RO = ShCfg<NC, N_OWN>;
  extern __shared__ uint8_t smem_raw[];
  const int tid = threadIdx.x & (SH_THREADS - 1), warp = warp_index() & 7, lane = tid & 31, side = warp_index() >> 3;
  const uint32_t base0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem0 = smem_raw + (base0 - smem_u32(smem_raw));  // the halves' barriers and control, 1 KB each; what they have of their own, or what both have
  const AttCtl ac(reinterpret_cast<uint64_t*>(smem0 + 1024 * side) + RP::N_BARS);
  long long* s_sum = reinterpret_cast<long long*>(smem0 + 512);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem0 + 768);
  if (threadIdx.x == 32 * 7) {
    for (const CUtensorMap* map : {&tmQp, &tmKp, &tmVp, &tmQ, &tmK, &tmV, &tmKn, &tmVn}) asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
  }
  ShHalf x;
  x.half = 2 * static_cast<int>(blockIdx.x) + side;
  x.bar0 = base0 + 1024 * side;
  if (warp == 5) {
    for (int i = lane; i < RP::N_BARS; i += 32) {
      const bool streams = (i >= RP::B_P && i < RP::B_PV) || i == RP::B_OFREE, frees = i >= RP::B_KVFREE || (i >= RP::B_QFREE && i < RP::B_OFREE);
      if (!frees) mbar_init(x.bar0 + 8u * i, streams ? 128 : 1);
    }
    if (lane == 0) *ac.abort = ac.odd[0] = ac.odd[1] = 0;
    fence_mbar_init();
    fence_async_smem();
  }
  if (warp == 4 && side == 0) {
    tmem_alloc(smem_u32(s_tmem), 2 * SH_TMEM);
    tmem_relinquish();
  }
  wait_for_previous();
  if (warp == 5 && lane == 0) *ac.bad = load_status(p.pre.status) != 0;
  // starts that do not ascend inside the batch: prefixes would have sequences in common, and more work than the host's limit on its units allows for. There is
  // none of it then, in any CTA, and the joining kernel sees the status word.
  bool wrong = false;
  if (p.pre.starts) {
    for (int i = threadIdx.x; i <= p.pre.groups; i += 2 * SH_THREADS)
      wrong |= p.pre.starts[i] < 0 || p.pre.starts[i] > p.pre.seqs || (i > 0 && p.pre.starts[i] < p.pre.starts[i - 1]);
  }
  wrong = __syncthreads_or(wrong) != 0;
  if (wrong && blockIdx.x == 0 && threadIdx.x == 0) report(p.pre.status, DEV_BAD_CACHE);
  tc_fence_before();
  // ---- how much there is of both kinds of work, and which is this CTA's ----
  int total_pre = 0, total_own = 0;
  for (int b = threadIdx.x; b < (wrong ? 0 : p.pre.c.batch); b += 2 * SH_THREADS) total_pre += sh_counted<ATT_PREFIX>(p.pre, b);
  for (int b = threadIdx.x; b < p.own.c.batch; b += 2 * SH_THREADS) total_own += sh_counted<ATT_OWN>(p.own, b);
  const long long both = sh_sum((static_cast<long long>(total_pre) << 32) + total_own, s_sum);
  total_pre = static_cast<int>(both >> 32);
  total_own = static_cast<int>(both & 0xffffffffll);
  const int grid = static_cast<int>(gridDim.x);
  int pre_ctas, split;
  sh_share<RP::PAIR>(p, total_pre, total_own, grid, pre_ctas, split);
  const bool pre = static_cast<int>(blockIdx.x) < pre_ctas;
  x.index = pre ? (RP::PAIR ? static_cast<int>(blockIdx.x) : x.half) : x.half - 2 * pre_ctas;
  x.split = pre ? split : 0;
  if (warp == 5) {  // (Rings that both halves read are freed by both. The others see these barriers behind those of sh_work.)
    for (int i = lane; i < RP::N_BARS; i += 32)
      if (i >= RP::B_KVFREE || (i >= RP::B_QFREE && i < RP::B_OFREE)) mbar_init(x.bar0 + 8u * i, RP::PAIR && pre ? 2 : 1);
    fence_mbar_init();
    fence_async_smem();
  }
  WalkOf<ATT_PREFIX> wp;
  WalkOf<ATT_OWN> wo;
  bool work;
  if (pre) work = sh_work<ATT_PREFIX>(p.pre, ac.ints, x.index, RP::PAIR ? pre_ctas : 2 * pre_ctas, total_pre, split, wp, x.chunk, x.end);
  else work = sh_work<ATT_OWN>(p.own, ac.ints, x.index, 2 * (grid - pre_ctas), total_own, 0, wo, x.chunk, x.end);
  let_next_begin();
  tc_fence_after();
  x.tmem = *s_tmem + side * SH_TMEM;
  x.sKV = base0 + 2048 + side * (SH_SMEM - 1024);
  x.ring0 = x.bar0;
  int kv_issued = 0, q_issued = 0;
  x.kv_issued = &kv_issued;
  x.q_issued = &q_issued;
  if (work && pre) {
    if (RP::PAIR) {
      x.ring0 = base0;
      x.sKV = base0 + 2048;
    }
    x.sQ = x.sKV + RP::NS * RP::STAGE;
    x.sP = x.sQ + RP::NQ * RP::Q_BYTES;
    x.other = smem0 + (x.sP - base0) + RP::P_BYTES + (RP::PAIR ? side * 4 * 2048 : 0);
    if constexpr (RP::ROWS) sh_rows<NC, N_PRE, BF16, ATT_PREFIX>(p.pre, wp, x, ac, &tmQp, &tmKp, &tmVp, &tmKp, &tmVp);
    else sh_columns<NC, N_PRE, BF16, ATT_PREFIX>(p.pre, wp, x, ac, &tmQp, &tmKp, &tmVp, &tmKp, &tmVp);
  } else if (work) {
    x.sQ = x.sKV + RO::NS * RO::STAGE;
    x.sP = x.sQ + RO::NQ * RO::Q_BYTES;
    x.other = smem0 + (x.sP - base0) + RO::P_BYTES;
    if constexpr (RO::ROWS) sh_rows<NC, N_OWN, BF16, ATT_OWN>(p.own, wo, x, ac, &tmQ, &tmK, &tmV, &tmKn, &tmVn);
    else sh_columns<NC, N_OWN, BF16, ATT_OWN>(p.own, wo, x, ac, &tmQ, &tmK, &tmV, &tmKn, &tmVn);
  }

  // ---- teardown (every thread gets here, also after an abort; the joining kernel sees the status word) ----
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *ac.bad) report(p.pre.status, DEV_BAD_CACHE);
  if (*ac.abort) {
    if (tid == 0) report_abort(ac.abort, p.pre.status);
    if ((warp == 5 || warp == 6) && lane == 0) {  // the copies that were started land
      auto drain = [&](auto cfg) {
        using R = decltype(cfg);
        for (int s = max(q_issued - R::NQ, 0); s < q_issued; ++s) mbar_drain(x.bar0 + 8u * (R::B_Q + s % R::NQ), (s / R::NQ) & 1);
        for (int T = max(kv_issued - (warp == 5 ? R::DK : R::DV), 0); T < kv_issued; ++T)
          mbar_drain(x.bar0 + 8u * (R::B_KV + (warp == 5 ? R::k_stage(T) : R::v_stage(T))), (warp == 5 ? R::k_turn(T) : R::v_turn(T)) & 1);
      };
      if (pre) drain(RP{});
      else drain(RO{});
    }
  }
  if (warp == 4 && side == 0) {
    tc_fence_after();
    tmem_dealloc(*s_tmem, 2 * SH_TMEM);
  }
}

// Joins what the prefixes and the sequences' own keys have left of a row: a warp a row, a lane four columns. 32 sources at a time: a lane has the
// factor of one, and all add up their columns; AHEAD of them are on their way at once.
template <bool BF16>
__global__ void __launch_bounds__(256) kfa_shared_join_kernel(const __grid_constant__ SharedParams p, const FastDiv by_head, const FastDiv by_token) {
  constexpr int AHEAD = 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned row = blockIdx.x * 8u + warp;  // (sequence, token, head): the rows of a tile of sequences one after the other
  const unsigned bt = by_head.div(row), b = by_token.div(bt);
  const int h = static_cast<int>(row - bt * by_head.d), t = static_cast<int>(bt - b * by_token.d);
  wait_for_previous();
  let_next_begin();
  const AttendParams &own = p.own, &pre = p.pre;
  if (row >= own.carry_rows) return;
  bool bad = false;
  const int count = own.counts ? min(max(own.counts[b], 0), own.T) : own.T;
  const int g = h / own.group, dh = h - g * own.group;
  const long long at = (static_cast<long long>(b) * own.H + h) * own.T + t;
  // the row's tile of its own
  int2 mine, before = make_int2(0, -1);  // -1: no prefix
  int r_own, r_pre = 0, pair = 0;
  {
    const int th = dh / own.gt, tt = t / own.tt;
    mine = own.dir[(static_cast<long long>(g) * own.row_tiles + tt * own.head_tiles + th) * own.seqs + b];
    r_own = (t - tt * own.tt) * own.gt + dh - th * own.gt;
  }
  int group = -1;
  if (!pre.starts) {
    group = 0;
  } else {  // the last prefix that begins at b or before, if it has b
    int lo = 0, hi = pre.groups;  // starts[lo] <= b < starts[hi]
    if (static_cast<int>(b) >= pre.starts[0] && static_cast<int>(b) < pre.starts[pre.groups]) {
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre.starts[mid] <= static_cast<int>(b)) lo = mid;
        else hi = mid;
      }
      group = lo;
    }
  }
  if (group >= 0) {
    int s0, s1;
    prefix_group(pre, group, s0, s1);
    const int ds = static_cast<int>(pre.by_ts.div(max(static_cast<int>(b) - s0, 0))), th = dh / pre.gt, tt = t / pre.tt, first = s0 + ds * pre.ts;
    before = pre.dir[(static_cast<long long>(g) * pre.row_tiles + tt * pre.head_tiles + th) * pre.seqs + first];
    r_pre = ((static_cast<int>(b) - first) * pre.tt + t - tt * pre.tt) * pre.gt + dh - th * pre.gt;
    pair = p.pre_pair;  // rows 128 .. 255 are the second half's, and a part's CTA has both
    if (before.y > 0) before.x += r_pre >> 7;
    r_pre &= 127;
  }
  // (Lengths that another stream changes while the kernel before this one runs may leave anything there; it stays inside the scratch.)
  mine.y = min(max(mine.y, 0), p.halves);
  before.y = min(before.y, p.halves);
  if (load_status(own.status) != 0) {  // (the directory may not have been written)
    bad = true;
    mine = make_int2(0, 0);
    before = make_int2(0, -1);
  }
  const int n_pre = before.y < 0 ? 0 : max(before.y, 1), n = n_pre + max(mine.y, 1);
  // source i: the prefix' parts, then the row's own. Parts: the first in slot 1 of its half, the others in slot 0 of theirs.
  auto find = [&](int i, const float*& o, const float*& ml, long long& plane) {
    const AttendParams& q = i < n_pre ? pre : own;
    const int2 d = i < n_pre ? before : mine;
    const int j = i < n_pre ? i : i - n_pre, r = i < n_pre ? r_pre : r_own;
    if (d.y == 0) {
      o = q.carry_o + at * 128;
      ml = q.carry_ml + at;
      plane = q.carry_rows;
    } else {
      const int half = min(max(d.x, 0) + (i < n_pre && pair ? 2 * j : j), p.halves - 1);
      const long long slot = 2ll * half + (j == 0 ? 1 : 0);
      o = q.part_o + (slot * q.rows + r) * 128;
      ml = q.part_ml + slot * 3 * q.rows + r;
      plane = q.rows;
    }
  };
  float m = -INFINITY, top = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int k = min(32, n - i0);
    const float *from = nullptr, *ml = nullptr;
    long long plane = 0;
    float mi = -INFINITY, li = 0.f, ti = -INFINITY;
    if (lane < k) {
      find(i0 + lane, from, ml, plane);
      mi = ml[0];
      li = ml[plane];
      ti = ml[2 * plane];
    }
    auto part = [&](int i) {
      const float* src = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(from), i));
      return 4 * lane < own.c.cols ? *reinterpret_cast<const float4*>(src + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    float4 y[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) y[i] = part(min(i, k - 1));
    const float m_new = fmaxf(m, warp_max(mi));
    top = fmaxf(top, warp_max(ti));
    if (i0) {
      const float old = sh_factor(m, l, m_new), a = old < 0.f ? 0.f : old;
      l *= a;
      o = make_float4(o.x * a, o.y * a, o.z * a, o.w * a);
    }
    m = m_new;
    const float a = lane < k ? sh_factor(mi, li, m) : -1.f;
    li *= a;
    auto add = [&](int i, const float4& z) {
      const float ai = __shfl_sync(0xffffffffu, a, i);
      l += __shfl_sync(0xffffffffu, li, i);
      if (!(ai < 0.f)) {
        o.x += ai * z.x;
        o.y += ai * z.y;
        o.z += ai * z.z;
        o.w += ai * z.w;
      }
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (i < k) add(i, y[i]);
    for (int j0 = AHEAD; j0 < k; j0 += AHEAD) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) y[i] = part(min(j0 + i, k - 1));
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (j0 + i < k) add(j0 + i, y[i]);
    }
  }
  const bool some = t < count && l != 0.f;
  const float nan = __int_as_float(0x7fc00000), inv = some ? 1.f / l : 0.f;
  if (bad) o = make_float4(nan, nan, nan, nan);
  else if (!some) o = make_float4(0.f, 0.f, 0.f, 0.f);
  else o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  if (4 * lane < own.c.cols)
    *reinterpret_cast<uint2*>(own.o + b * own.o_sb + h * own.o_sh + t * own.o_ss + 8 * lane) = make_uint2(pack16<BF16>(o.x, o.y), pack16<BF16>(o.z, o.w));
  if (own.stats && lane == 0) {
    float* to = own.stats + (static_cast<long long>(b) * own.H + h) * 2 * own.T + t;
    to[0] = bad ? nan : (some ? top : INFINITY);
    to[own.T] = bad ? nan : (some ? log2f(l) + __fmaf_rn(-top, own.c_log2, m) : 0.f);
  }
}

}  // namespace kfa
