// Attention of a sequence's newest tokens (one, a tree of drafted ones, a chunk of a prompt) to its cached keys and to one another.
//
//   S = q K^T,  m = max S,  P = exp2((S - m) c),  l = sum P,  out = P V / l,  c = scale * log2(e)
//
// What bounds it: the keys and values, read once each (2 x 2 D bytes a position and K / V head). All query rows that share them, the
// query heads of a K / V head times the new tokens, are one tile of rows. There are two kernels.
//
// Up to 64 rows (kfa_cache_attend_kernel): far below what makes the tensor core the limit, so the tile is turned around: the KEYS are the
// 128 rows of the matrix instructions, the query rows their N columns (16, 32 or 64), and little is computed for rows that are not there:
//   S^T [128 keys x N] = K Q^T                 A = K from shared memory as copied, B = Q
//   O^T [D x N]       += V^T P^T               A = V as copied (the transposed, MN-major, operand), B = P^T from shared memory
// A thread holds one key's scores. The maximum over keys is a warp reduction per column and an exchange between four warps; the sum
// over keys stays in the thread until the end.
// More rows (kfa_cache_attend_rows_kernel): rows on the matrix rows, a thread a row, P from tensor memory, as in the forward of whole
// sequences. (A thread of the first kernel would spend 6800 clk on 256 rows x 128 keys, one of this kernel spends 4400.)
// In both O is rescaled only when a row's maximum grew by more than a factor of 2^8 (the numerators may be up to 2^8 then, which 16-bit P
// takes at the same relative precision).
//
// Work is cut by keys, not by sequences: the keys of all (sequence, K / V head, row tile) items are counted in units of 32 and every CTA
// takes an equal stretch, whatever the lengths (which only the device knows). An item counts some units more than it has, for what its
// beginning and its end take. An item that one CTA has whole is written by it; of the others the CTA leaves its part (unnormalised O in
// fp32, m, l) in scratch and a second kernel joins them in the order of the keys, so that results repeat bit for bit.
//
//   warps 0-3, 4-7  two streams: tiles of 128 keys go to the two in turn, each with its own maxima, sums and O, joined at the item's end
//                   (with more than 128 rows both see every tile, each with half of the rows)
//   warps 8, 9      MMA issue for the two streams
//   warps 10, 11    TMA producers: keys (and queries), values; a lane per box of up to 32 rows inside a page
#pragma once

#include "kfa_cache_view.cuh"

namespace kfa {

constexpr int ATT_THREADS = 384;
constexpr int ATT_UNIT = 32;  // keys: what work is counted in
// Registers per thread: 168 at the start (65536 / 384, in eights); with 64 columns the streams, which hold two numbers a column, take what the
// issuing warps do not need. (A CTA owns what it was launched with: budgets beyond that would wait for ever.)
constexpr int ATT_REGS = 168, ATT_REGS_STREAM = 208, ATT_REGS_ISSUE = 88;
static_assert(2 * 128 * ATT_REGS_STREAM + 128 * ATT_REGS_ISSUE <= ATT_THREADS * ATT_REGS, "register budgets exceed the CTA's allocation");

enum { ATT_PLAIN = 0, ATT_PREFIX = 1, ATT_OWN = 2 };  // (the last two: kfa_shared.cuh)

struct AttendParams {
  CacheView c;
  const uint8_t *k, *v;  // new tokens' (null: none): element access for values that are not finite
  long long v_sb, v_sh, v_ss;  // bytes
  const uint8_t* tree;
  long long tree_sb, tree_st, tree_sj;
  const int* counts;
  uint8_t* o;
  long long o_sb, o_sh, o_ss;  // bytes
  float* stats;
  int H, T, group;
  int gt, tt, head_tiles, row_tiles;  // a row tile: gt heads x tt tokens, head_tiles x token tiles = row_tiles of them per K / V head
  FastDiv by_gt, by_items, by_row_tiles, by_head_tiles;
  FastDiv by_grid;
  int items;       // per sequence: K / V heads x row tiles
  int whole;       // every item is one CTA's (short caches: nothing is cut)
  int least;       // the shortest stretch of a CTA, in units
  int extra;       // units that an item counts more than it has
  int box;         // rows of a page's TMA box
  int rows;        // of scratch per part
  int appended;    // the new tokens are in the cache already (cache_weights): positions lengths .. lengths + counts - 1
  float c_log2, slack;  // scale * log2 e; how far a maximum may grow before O is rescaled
  float* part_o;   // [slot][rows][128]; of the kernel for more rows [slot][rows / 32][128 / 4][32][4]
  float* part_ml;  // [slot][3][rows]: m, l, largest score
  int4* part_meta; // [CTA]: parts of the item that begins in it and ends in another (0: none), sequence, item
  int* status;
  // shared prefixes. ATT_PREFIX: c has the prefixes, its batch is their number; `items` are those of one tile of sequences
  const int* starts;  // sequences starts[i] .. starts[i + 1] - 1 go on from prefix i; or nullptr: all from the only one
  int groups, seqs;   // prefixes, sequences
  int ts;             // sequences of a row tile
  FastDiv by_ts, by_seq_rows;  // by_seq_rows: rows of a sequence in a tile, gt x tt
  float* carry_o;     // [(sequence, head, token)][128]
  float* carry_ml;    // [3][(sequence, head, token)]: m, l, largest score
  long long carry_rows;
  int2* dir;          // [(K / V head, row tile)][first sequence of the tile]: the half CTA in which the item begins, its parts (0: in the carry)
};

// The sequences that go on from prefix i: first and behind the last, inside the batch whatever `starts` says.
__device__ __forceinline__ void prefix_group(const AttendParams& p, int i, int& s0, int& s1) {
  s0 = 0;
  s1 = p.seqs;
  if (p.starts) {
    s0 = min(max(p.starts[i], 0), p.seqs);
    s1 = min(max(p.starts[i + 1], s0), p.seqs);
  }
}

// The stretch of work of a CTA, from (b, item, unit) to (end_b, end_item, end_unit), walked item by item; every role walks for itself.
// (ATT_PREFIX: b is a prefix.)
template <int MODE>
struct WalkOf {
  int b, item, unit, end_b, end_item, end_unit;
  int units, uc, ud, len, count;  // of the item; uc, ud: units of cached and of new keys
  int n;                          // units of the current segment, the part of the item that is this CTA's
  int items;                      // of b
  __device__ __forceinline__ static void size(const AttendParams& p, int b, int& len, int& count, int& uc, int& ud) {
    len = cache_length(p.c, b);
    if constexpr (MODE == ATT_PREFIX) {
      count = 0;
      uc = (len + ATT_UNIT - 1) / ATT_UNIT;
      ud = 0;
      return;
    }
    count = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
    if (p.appended) len = count ? min(len + count, p.c.capacity) : 0;
    uc = count ? (len + ATT_UNIT - 1) / ATT_UNIT : 0;
    ud = count && p.k ? (count + ATT_UNIT - 1) / ATT_UNIT : 0;
  }
  __device__ __forceinline__ static int units_of(const AttendParams& p, int b) {
    int len, count, uc, ud;
    size(p, b, len, count, uc, ud);
    return max(uc + ud, 1);
  }
  __device__ __forceinline__ static int items_of(const AttendParams& p, int b) {
    if constexpr (MODE != ATT_PREFIX) return p.items;
    int s0, s1;
    prefix_group(p, b, s0, s1);
    return p.items * static_cast<int>(p.by_ts.div(s1 - s0 + p.ts - 1));
  }
  __device__ __forceinline__ bool last() const { return b == end_b && item == end_item; }
  __device__ __forceinline__ void load(const AttendParams& p) {
    size(p, b, len, count, uc, ud);
    units = max(uc + ud, 1);
    items = items_of(p, b);
  }
  __device__ __forceinline__ void cut() { n = (last() ? min(units, end_unit) : units) - unit; }
  __device__ __forceinline__ bool start(const AttendParams& p) {  // false: nothing to do
    if (b == end_b && (item > end_item || (item == end_item && unit >= end_unit))) return false;
    load(p);
    cut();
    return true;
  }
  __device__ __forceinline__ bool next(const AttendParams& p) {  // false: that was the last segment, and it stays the current one
    if (last()) return false;
    const bool other = item + 1 == items;
    int b2 = b + (other ? 1 : 0);
    const int item2 = other ? 0 : item + 1;
    if constexpr (MODE == ATT_PREFIX) {  // (prefixes that nobody goes on from have no items)
      while (other && b2 < end_b && items_of(p, b2) == 0) ++b2;
    }
    if (b2 == end_b && item2 == end_item && end_unit == 0) return false;
    b = b2;
    item = item2;
    unit = 0;
    if (other) load(p);
    cut();
    return true;
  }
  template <int UNITS = 4>
  __device__ __forceinline__ int tiles() const {
    return (n + UNITS - 1) / UNITS;
  }
  __device__ __forceinline__ bool begins() const { return unit == 0; }
  __device__ __forceinline__ bool ends() const { return unit + n == units; }
};
using Walk = WalkOf<ATT_PLAIN>;

// Shares out the whole batch's work, counted(b) of it sequence b's (0 or more), equally: at[0] .. at[1] is this CTA's stretch, found(i, b, off,
// counted(b)) is called by one thread for each of the two ends that lies inside sequence b, off into it. All threads of the CTA; s_i: 32 ints of
// shared memory, of which the first 8 are found's. Returns the length of a stretch.
template <typename F, typename G>
__device__ __forceinline__ int att_share(const AttendParams& p, int* s_i, F counted, int (&at)[2], int& total, G found) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto of = [&](int b) { return b < p.c.batch ? counted(b) : 0; };
  auto warp_scan = [&](int x) {
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, x, off);
      if (lane >= off) x += up;
    }
    return x;
  };
  // 384 sequences at a time; then the sequences in which this CTA's stretch begins and ends
  total = 0;
  const int own0 = of(tid), scan0 = warp_scan(own0);
  for (int b0 = 0; b0 < p.c.batch; b0 += ATT_THREADS) {
    const int s = b0 == 0 ? scan0 : warp_scan(of(b0 + tid));
    if (b0 > 0) __syncthreads();
    if (lane == 31) s_i[8 + warp] = s;
    __syncthreads();
    for (int i = 0; i < ATT_THREADS / 32; ++i) total += s_i[8 + i];
  }
  const int chunk = max(static_cast<int>(p.by_grid.div(total + gridDim.x - 1)), p.least);
  at[0] = chunk * static_cast<int>(blockIdx.x);
  at[1] = at[0] + chunk;
  int before = 0;
  for (int b0 = 0; b0 < p.c.batch; b0 += ATT_THREADS) {
    const int own = b0 == 0 ? own0 : of(b0 + tid);
    int upto = b0 == 0 ? scan0 : warp_scan(own);
    if (p.c.batch > ATT_THREADS) {
      __syncthreads();
      if (lane == 31) s_i[8 + warp] = upto;
      __syncthreads();
    }
    int all = 0;
    for (int i = 0; i < ATT_THREADS / 32; ++i) {
      const int x = s_i[8 + i];
      if (i < warp) upto += x;
      all += x;
    }
    upto += before;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (at[i] >= upto - own && at[i] < upto) found(i, b0 + tid, at[i] - (upto - own), own);
    before += all;
  }
  __syncthreads();
  return chunk;
}

// Which work is this CTA's (all its threads; s_i: 32 ints of shared memory). Synchronises the CTA. chunk, end: units per CTA and where this
// one's stretch ends, both as they are counted.
__device__ __forceinline__ bool my_work(const AttendParams& p, int* s_i, Walk& w, int& chunk, int& end) {
  chunk = end = 0;
  if (p.whole) {
    const unsigned all = static_cast<unsigned>(p.c.batch) * p.items;
    const unsigned i0 = p.by_grid.div(static_cast<unsigned>(all)) * blockIdx.x + min(blockIdx.x, all - p.by_grid.div(all) * gridDim.x);
    const unsigned i1 = i0 + p.by_grid.div(all) + (blockIdx.x < all - p.by_grid.div(all) * gridDim.x ? 1 : 0);
    w.b = static_cast<int>(p.by_items.div(i0));
    w.item = static_cast<int>(i0 - w.b * p.items);
    w.end_b = static_cast<int>(p.by_items.div(i1));
    w.end_item = static_cast<int>(i1 - w.end_b * p.items);
    w.unit = w.end_unit = 0;
    __syncthreads();
    return w.start(p);
  }
  int at[2], total;
  chunk = att_share(p, s_i, [&](int b) { return (Walk::units_of(p, b) + p.extra) * p.items; }, at, total, [&](int i, int b, int off, int own) {
    const int each = own / p.items, item = off / each;
    s_i[3 * i] = b;
    s_i[3 * i + 1] = item;
    s_i[3 * i + 2] = max(off - item * each - p.extra, 0);
  });
  const bool inside[2] = {at[0] < total, at[1] < total};
  w.b = inside[0] ? s_i[0] : p.c.batch;
  w.item = inside[0] ? s_i[1] : 0;
  w.unit = inside[0] ? s_i[2] : 0;
  w.end_b = inside[1] ? s_i[3] : p.c.batch;
  w.end_item = inside[1] ? s_i[4] : 0;
  w.end_unit = inside[1] ? s_i[5] : 0;
  end = at[1];
  return w.b < p.c.batch && w.start(p);
}

// mbar_wait_warp for kernels in which many warps wait at the same time: the hardware may suspend a thread for up to 10 us (the hint)
// instead of the default, and suspended warps take no issue slots from those that compute.
__device__ __forceinline__ bool mbar_suspend(uint32_t bar, uint32_t parity) {
  if constexpr (KFA_SHORT_WAITS) {
    return mbar_try_wait(bar, parity);
  } else {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(10000u)
        : "memory");
    return ok != 0;
  }
}
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, const Ctl& ctl, int site) {
  bool ok = mbar_suspend(bar, parity);
  if (__builtin_expect(__all_sync(0xffffffffu, ok), 1)) return true;
  if (!ok) {
    const long long t0 = clock64();
#pragma unroll 1
    while (!(ok = mbar_suspend(bar, parity))) {
      if (*ctl.s_abort != 0) break;
      if (clock64() - t0 > KFA_WAIT_CYCLES) {
        *ctl.s_abort = KFA_DEV_TIMEOUT_BASE + site;
        break;
      }
    }
  }
  return __all_sync(0xffffffffu, ok);
}

// Shared memory and rings that both kernels lay out alike. NC: chunks of 64 columns of the head dim; Q_ROWS: rows of the query buffer;
// BOTH: both streams see every tile (else they take turns); OTHER: bytes beside keys, values and queries.
template <int NC_, int Q_ROWS_, int NQ_, bool BOTH_, int OTHER_>
struct AttRings {
  static constexpr int NC = NC_, Q_ROWS = Q_ROWS_, NQ = NQ_;
  static constexpr bool BOTH = BOTH_, KEYS_FIRST = false;  // KEYS_FIRST: whether the first values wait for the first keys' scores
  static constexpr int UNITS = 4;                          // of a tile
  static constexpr int CHUNK = 128 * 64 * 2;  // 128 keys x 64 columns
  static constexpr int STAGE = NC * CHUNK;
  static constexpr int Q_CHUNK = Q_ROWS * 128, Q_BYTES = NC * Q_CHUNK;
  static constexpr int FIXED = 1024 + NQ * Q_BYTES + OTHER_;
  static constexpr int FIT = (232448 - FIXED) / STAGE;
  // Rings of key tiles and of value tiles, in turn for each stream (BOTH: one of each for both). A stage has one producer and the
  // same consumers every time: who waits for a phase of its barrier has waited for the one before, so that a parity means one phase.
  static constexpr int RINGS = BOTH ? 1 : 2;
  static constexpr int DEEP = FIT / RINGS, MOST = BOTH ? 4 : 2;
  static constexpr int DV = DEEP / 2 < MOST ? DEEP / 2 : MOST;
  static constexpr int DK = DEEP - DV < MOST ? DEEP - DV : MOST;
  static_assert(DV >= 1 && DK >= 1, "no room for a tile of keys and one of values");
  static constexpr int NS = RINGS * (DK + DV);
  static constexpr int SMEM = FIXED + NS * STAGE;
  __device__ static __forceinline__ int k_stage(int T) { return BOTH ? T % DK : (T & 1) * DK + (T >> 1) % DK; }
  __device__ static __forceinline__ int v_stage(int T) { return RINGS * DK + (BOTH ? T % DV : (T & 1) * DV + (T >> 1) % DV); }
  __device__ static __forceinline__ int k_turn(int T) { return (BOTH ? T : T >> 1) / DK; }
  __device__ static __forceinline__ int v_turn(int T) { return (BOTH ? T : T >> 1) / DV; }
  // barriers: tiles there and free, queries there, scores there, P there, P V done, a segment is finished, a stream's O has been read (in the
  // segments in which the stream had tiles), all done
  static constexpr int B_KV = 0, B_KVFREE = NS, B_Q = 2 * NS, B_S = B_Q + NQ, B_P = B_S + 4, B_PV = B_P + 4, B_QFREE = B_PV + 4,
                       B_OFREE = B_QFREE + NQ, B_DRAIN = B_OFREE + 2, N_BARS = B_DRAIN + 2;
  static_assert(N_BARS * 8 + 256 <= 1024, "barrier block");
};

__device__ __forceinline__ float warp_max(float x) {  // NaN counts as nothing
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
template <int ID, int COUNT>
__device__ __forceinline__ void named_sync() {
  asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(COUNT) : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
template <int W>
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, float* r) {
  if constexpr (W == 8) tmem_ld8(taddr, reinterpret_cast<uint32_t*>(r));
  else if constexpr (W == 16) tmem_ld16(taddr, reinterpret_cast<uint32_t*>(r));
  else if constexpr (W == 32) tmem_ld32(taddr, reinterpret_cast<uint32_t*>(r));
  else {
    tmem_ld32(taddr, reinterpret_cast<uint32_t*>(r));
    tmem_ld32(taddr + 32, reinterpret_cast<uint32_t*>(r + 32));
  }
}
// A and B with high descriptor words of their own.
__device__ __forceinline__ void umma_ss_lead2(bool lead, uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                              uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %2};\n\t"
      "mov.b64 db, {%3, %4};\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "setp.ne.b32 q, %7, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t}"
      ::"r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(static_cast<uint32_t>(lead))
      : "memory");
}

// Where the 16-byte piece `i` of row `row` of a P^T tile lies: rows of 2 N bytes with the swizzle that spans one.
template <int N>
__device__ __forceinline__ uint32_t p_piece(int row, int i) {
  constexpr int SPREAD = N == 64 ? 1 : (N == 32 ? 2 : 4);  // rows that share a pattern
  return static_cast<uint32_t>(row * 2 * N + ((i ^ ((row / SPREAD) & (N / 8 - 1))) << 4));
}

// Sums over the 32 lanes of V values per lane at once: afterwards lane i holds the sums of columns i * V / 32 .. (V = 64: 2, 32: 1), V = 16:
// lanes 2 i and 2 i + 1 that of column i.
template <int V>
__device__ __forceinline__ void columns_over_lanes(float* x, int lane) {
  int width = V;
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    if (width > 1) {
      width >>= 1;
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        if (i < width) {
          const bool up = (lane & off) != 0;
          const float give = up ? x[i] : x[i + width], keep = up ? x[i + width] : x[i];
          x[i] = keep + __shfl_xor_sync(0xffffffffu, give, off);
        }
      }
    } else {
      x[0] += __shfl_xor_sync(0xffffffffu, x[0], off);
    }
  }
}

// What a part with maximum m and sum l counts beside the maximum of all parts: < 0 if it saw no key (its O is not defined then, its l is 0);
// a sum that is NaN without any maximum (all its scores were NaN) counts, as NaN. A part that counts 0 because its scores are far below the others' is
// multiplied like the rest: 0 * NaN of a value that is seen is NaN, whatever part the value lies in.
__device__ __forceinline__ float part_factor(float m, float l, float m_all, float c_log2) {
  if (m == -INFINITY) return l == 0.f ? -1.f : 1.f;
  return ex2((m - m_all) * c_log2);
}

// The heads and tokens (ATT_PREFIX: and sequences) of a row tile's rows.
template <int MODE>
struct RowMapOf {
  int g, h0, heads, t0;  // K / V head; first head, heads that exist, first token
  int s0, s1;            // first sequence, behind the last of the group (else the sequence)
  int rt;                // row tile of the K / V head
  __device__ __forceinline__ RowMapOf(const AttendParams& p, int b, int item) {
    s0 = b;
    s1 = b + 1;
    if constexpr (MODE == ATT_PREFIX) {  // items of a K / V head one after the other: CTAs that run together read the same keys
      prefix_group(p, b, s0, s1);
      const int tiles = static_cast<int>(p.by_ts.div(s1 - s0 + p.ts - 1)), per = p.row_tiles * tiles;
      g = item / per;
      const int rest = item - g * per, tile_s = static_cast<int>(p.by_row_tiles.div(rest));
      s0 += tile_s * p.ts;
      rt = rest - tile_s * p.row_tiles;
    } else {
      g = static_cast<int>(p.by_row_tiles.div(item));
      rt = item - g * p.row_tiles;
    }
    const int tile_t = static_cast<int>(p.by_head_tiles.div(rt)), tile_h = rt - tile_t * p.head_tiles;
    h0 = g * p.group + tile_h * p.gt;
    heads = min(p.gt, p.group - tile_h * p.gt);
    t0 = tile_t * p.tt;
  }
  __device__ __forceinline__ bool row(const AttendParams& p, int r, int& h, int& t) const {
    int s;
    return row(p, r, h, t, s);
  }
  __device__ __forceinline__ bool row(const AttendParams& p, int r, int& h, int& t, int& s) const {
    s = s0;
    bool in = true;
    if constexpr (MODE == ATT_PREFIX) {
      const int ds = static_cast<int>(p.by_seq_rows.div(r));
      s += ds;
      in = ds < p.ts && s < s1;
      r -= ds * static_cast<int>(p.by_seq_rows.d);
    }
    const int dt = static_cast<int>(p.by_gt.div(r)), dh = r - dt * p.gt;
    h = h0 + dh;
    t = t0 + dt;
    return in && dt < p.tt && dh < heads && t < p.T;
  }
};
using RowMap = RowMapOf<ATT_PLAIN>;
// Rows of a tile that may exist.
template <int MODE>
__device__ __forceinline__ int tile_rows(const AttendParams& p) {
  return MODE == ATT_PREFIX ? p.gt * p.tt * p.ts : p.gt * p.tt;
}

// Control block of a CTA behind its barriers.
struct AttCtl {
  uint32_t* tmem;
  volatile int *abort, *bad;  // bad: the cache says something that is not so, or an earlier kernel failed
  volatile int* odd;          // [stream] 1 + the last segment in which it met new values that are not finite
  int* ints;                  // 32, for my_work
  __device__ __forceinline__ explicit AttCtl(uint64_t* behind) {
    tmem = reinterpret_cast<uint32_t*>(behind);
    abort = reinterpret_cast<volatile int*>(tmem + 1);
    bad = abort + 1;
    odd = abort + 2;
    ints = reinterpret_cast<int*>(tmem + 8);
  }
};

// Both kernels' beginning: barriers, tensor memory, the CTA's work.
template <class R>
__device__ __forceinline__ bool att_setup(const AttendParams& p, uint32_t bar0, const AttCtl& ctl, int tmem_cols, Walk& first, int& chunk,
                                          int& end) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 10) {
    for (int i = lane; i < R::N_BARS; i += 32) {
      int count = 1;
      if (i >= R::B_KVFREE && i < R::B_Q) count = R::BOTH ? 2 : 1;
      if (i >= R::B_P && i < R::B_PV) count = 128;
      if (i >= R::B_QFREE && i < R::B_OFREE) count = R::BOTH ? 2 : 256;
      if (i >= R::B_OFREE && i < R::B_DRAIN) count = R::BOTH ? 128 : 256;
      mbar_init(bar0 + 8u * i, count);
    }
    if (lane == 0) *ctl.abort = ctl.odd[0] = ctl.odd[1] = 0;
    fence_mbar_init();
    fence_async_smem();
  }
  if (warp == 8) {
    tmem_alloc(smem_u32(ctl.tmem), tmem_cols);
    tmem_relinquish();
  }
  wait_for_previous();
  if (warp == 10 && lane == 0) *ctl.bad = load_status(p.status) != 0;
  tc_fence_before();
  const bool work = my_work(p, ctl.ints, first, chunk, end);
  let_next_begin();
  tc_fence_after();
  return work;
}

// The producers' role: warp 10 queries and keys, warp 11 values. Leaves how many tiles and segments' queries it has started.
template <class R, int MODE>
__device__ __forceinline__ void att_produce(const AttendParams& p, const WalkOf<MODE>& first, bool values, uint32_t sKV, uint32_t sQ, uint32_t bar0,
                                            const AttCtl& ac, const CUtensorMap* q_map, const CUtensorMap* map, const CUtensorMap* map_new,
                                            int& kv_issued, int& q_issued) {
  const int lane = threadIdx.x & 31;
  const Ctl ctl{ac.abort};
  auto bar = [&](int i) { return bar0 + 8u * i; };
  WalkOf<MODE> w = first;
  const int per_unit = ATT_UNIT / p.box, boxes = R::UNITS * per_unit;
  bool ok = true, more = true;
  int T = 0, s = 0;  // tiles and segments so far
  if constexpr (KFA_LATE_VALUES > 0) {
    const long long t0 = clock64();
    while (values && clock64() - t0 < KFA_LATE_VALUES) {}
  }
  // (At the start all CTAs ask for all that their rings hold: the first keys, which everything waits for, go ahead of the values. What is waited for are the first
  // scores, not the keys' own barrier: a key stage is filled again as soon as its scores are made, so that a warp which is held up could come to that barrier a
  // phase or two late, and wait for what only its own values bring about. The phase behind that of the first scores belongs to the third tile's, which are made
  // when the first values have been multiplied: it cannot be over before this wait.)
  if (R::KEYS_FIRST && values) ok = wait_warp(bar(R::B_S), 0, ctl, 77);
  while (more && ok) {
    const RowMapOf<MODE> rows(p, w.b, w.item);
    if (lane == 0 && !length_ok(p.c, w.b)) *ac.bad = 1;
    if (!values) {
      if (s >= R::NQ) {  // both streams are done with the segment that used this buffer
        ok = wait_warp(bar(R::B_QFREE + s % R::NQ), (s / R::NQ - 1) & 1, ctl, 70);
        if (!ok) break;
      }
      if (lane == 0) {
        mbar_expect_tx(bar(R::B_Q + s % R::NQ), R::NC * tile_rows<MODE>(p) * 128);
        for (int ch = 0; ch < R::NC; ++ch)
          tma_load_4d(sQ + (s % R::NQ) * R::Q_BYTES + ch * R::Q_CHUNK, q_map, bar(R::B_Q + s % R::NQ), ch * 64, rows.h0, rows.t0, rows.s0);
      }
      q_issued = s + 1;
    }
    const int tiles = w.template tiles<R::UNITS>();
    for (int t = 0; t < tiles && ok; ++t, ++T) {
      // this lane's box
      const int in_unit = (lane % per_unit) * p.box, unit = w.unit + R::UNITS * t + lane / per_unit;
      const bool mine = lane < boxes && unit < w.unit + w.n;
      const int row = (lane / per_unit) * ATT_UNIT + in_unit;
      int c1 = 0, c3 = w.b, kind = 0;  // 1: cached rows, 2: new ones
      if (mine && unit < w.uc) {
        const int pos = unit * ATT_UNIT + in_unit;
        if (pos < w.len) {
          if (cache_place(p.c, w.b, pos, c3, c1)) kind = 1;
          else *ac.bad = 1;
        }
      } else if (mine && in_unit == 0) {
        c1 = (unit - w.uc) * ATT_UNIT;
        if (c1 < w.count && w.ud > 0) kind = 2;
      }
      const unsigned cached = __ballot_sync(0xffffffffu, kind == 1), fresh = __ballot_sync(0xffffffffu, kind == 2);
      const int stage = values ? R::v_stage(T) : R::k_stage(T), turn = values ? R::v_turn(T) : R::k_turn(T);
      if (turn > 0) {
        ok = wait_warp(bar(R::B_KVFREE + stage), (turn - 1) & 1, ctl, values ? 71 : 72);
        if (!ok) break;
      }
      if (lane == 0) mbar_expect_tx(bar(R::B_KV + stage), R::NC * 128 * (__popc(cached) * p.box + __popc(fresh) * ATT_UNIT));
      __syncwarp();
      if (kind != 0) {
        const uint32_t dst = sKV + stage * R::STAGE + row * 128;
        for (int ch = 0; ch < R::NC; ++ch) tma_load_4d(dst + ch * R::CHUNK, kind == 1 ? map : map_new, bar(R::B_KV + stage), ch * 64, c1, rows.g, c3);
      }
      kv_issued = T + 1;
    }
    if (ok) {
      ++s;
      more = w.next(p);
    }
  }
}

// A stream's tiles one after the other, over all segments.
struct AttTile {
  int T, s;
  int uses;    // segments before in which the stream had tiles
  bool opens;  // the stream's first tile of segment s
  bool closes; // the segment's last tile
};
template <bool ALL, int UNITS = 4, class W = Walk>
struct AttTiles {
  W w;
  int st, at = 0, T = 0, s = 0, uses = 0;
  bool more = true, opens = true;
  __device__ __forceinline__ bool take(const AttendParams& p, AttTile& t) {
    while (more) {
      const int tiles = w.template tiles<UNITS>();
      while (at < tiles) {
        ++at;
        const int now = T++;
        if (ALL || (now & 1) == st) {
          t = {now, s, uses, opens, at == tiles};
          opens = false;
          return true;
        }
      }
      at = 0;
      ++s;
      uses += opens ? 0 : 1;
      opens = true;
      more = w.next(p);
    }
    return false;
  }
};

// The issuing warps' loop: scores of piece i as soon as their keys (and queries) are there and the columns free, which they are once the
// values of piece i - 2 have been issued, values of piece j as soon as P and V are there, whichever comes first: neither holds the other up
// (keys that are late would delay values whose results others wait for). PIECES of a tile: 1, or 2 halves of 64 keys.
// issue_S(tile, c, piece), issue_PV(tile, c, piece) issue and commit; c counts the stream's tiles.
template <class R, int PIECES, int NP, typename FS, typename FP>
__device__ __forceinline__ void att_issue(const AttendParams& p, const Walk& first, int st, uint32_t bar0, const AttCtl& ac, FS issue_S, FP issue_PV) {
  auto ready = [&](int i, uint32_t parity) { return __all_sync(0xffffffffu, mbar_test(bar0 + 8u * i, parity)); };
  AttTiles<R::BOTH> tiles{first, st};
  AttTile ahead = {0, 0, 0, false, false}, even = ahead, odd = ahead;  // the next to get scores; those that have, by c (at most two wait for values)
  bool have = tiles.take(p, ahead);
  int i_s = 0, i_p = 0;  // pieces of scores and of values issued
  long long t0 = clock64();
  while (have || i_p < i_s) {
    bool went = false;
    if (have && i_s <= i_p + 1) {
      const int c = i_s / PIECES, piece = i_s % PIECES;
      if (piece > 0 || (ready(R::B_KV + R::k_stage(ahead.T), R::k_turn(ahead.T) & 1) &&
                        (!ahead.opens || ready(R::B_Q + ahead.s % R::NQ, (ahead.s / R::NQ) & 1)))) {
        tc_fence_after();
        issue_S(ahead, c, piece);
        ++i_s;
        went = true;
        if (piece == PIECES - 1) {
          if (c & 1) odd = ahead;
          else even = ahead;
          have = tiles.take(p, ahead);
        }
      }
    }
    if (i_p < i_s) {
      const int c = i_p / PIECES, piece = i_p % PIECES;
      // (nothing else can go before these values: no need to look at both)
      if ((!have || i_s > i_p + 1) &&
          !wait_warp(bar0 + 8u * (R::B_P + 2 * st + (PIECES == 2 ? piece : c % NP)), (PIECES == 2 ? c : c / NP) & 1, Ctl{ac.abort}, 74))
        break;
      const AttTile now = (c * PIECES + PIECES > i_s) ? ahead : ((c & 1) ? odd : even);  // (its second half may have no scores yet)
      if (ready(R::B_P + 2 * st + (PIECES == 2 ? piece : c % NP), (PIECES == 2 ? c : c / NP) & 1) &&
          (piece > 0 || (ready(R::B_KV + R::v_stage(now.T), R::v_turn(now.T) & 1) &&
                         (!now.opens || now.uses == 0 || ready(R::B_OFREE + st, (now.uses - 1) & 1))))) {
        tc_fence_after();
        issue_PV(now, c, piece);
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
    }
  }
  // what was issued has retired before tensor memory is freed
  const bool lead = elect_one();
  umma_commit_lead(lead, bar0 + 8u * (R::B_DRAIN + st));
  mbar_drain(bar0 + 8u * (R::B_DRAIN + st), 0);
}

// A bit for each of the first n (at most 32) bytes `stride` apart that are not 0. (The loads do not wait for one another.)
__device__ __forceinline__ uint32_t tree_bits(const uint8_t* at, long long stride, int n) {
  uint32_t bits = 0;
#pragma unroll 1
  for (int i0 = 0; i0 < min(n, 32); i0 += 8) {
    uint8_t x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = at[min(i0 + i, n - 1) * stride];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i0 + i < n && x[i] != 0) bits |= 1u << (i0 + i);
  }
  return bits;
}

// Which keys of a unit the row of token t sees, a bit each (the first pass of a masked tile).
template <class W>
__device__ __forceinline__ uint32_t seen_word(const AttendParams& p, const W& w, int unit, int t) {
  if (unit >= w.unit + w.n) return 0u;
  if (unit < w.uc) {
    const int left = w.len - unit * ATT_UNIT;
    return left >= ATT_UNIT ? 0xffffffffu : (1u << left) - 1u;
  }
  if (w.ud == 0 || t >= w.count) return 0u;
  const int j0 = (unit - w.uc) * ATT_UNIT, left = w.count - j0;
  if (left <= 0) return 0u;
  uint32_t there = left >= ATT_UNIT ? 0xffffffffu : (1u << left) - 1u;
  if (p.tree == nullptr) {
    const int upto = t - j0;  // tokens 0 .. t
    return upto < 0 ? 0u : (upto >= ATT_UNIT - 1 ? there : there & ((2u << upto) - 1u));
  }
  return there & tree_bits(p.tree + w.b * p.tree_sb + t * p.tree_st + j0 * p.tree_sj, p.tree_sj, left);
}

// Values behind the end may be anything, and 0 * NaN is no 0: in a tile that is not full of cached keys, the thread of key `key` zeroes
// its row of the tile. So it does with the values of a new token that are not finite, which would otherwise reach rows that do not see it; the
// epilogue hands them to those that do. odd_values looks for them in memory, ahead of the scores: which 16-byte pieces hold any.
template <bool BF16>
__device__ __forceinline__ bool odd_half(uint32_t x) {  // all exponent bits: infinity or NaN
  constexpr uint32_t E = BF16 ? 0x7f80u : 0x7c00u;
  return (x & E) == E;
}
template <bool BF16>
__device__ __forceinline__ uint32_t odd_values(const AttendParams& p, const Walk& w, int g, int fresh) {
  if (fresh < 0) return 0u;
  const uint8_t* row = p.v + w.b * p.v_sb + g * p.v_sh + fresh * p.v_ss;
  uint32_t found = 0;
#pragma unroll 8
  for (int i = 0; i < p.c.cols / 8; ++i) {
    const uint4 q = *reinterpret_cast<const uint4*>(row + 16 * i);
    const bool odd = odd_half<BF16>(q.x) || odd_half<BF16>(q.x >> 16) || odd_half<BF16>(q.y) || odd_half<BF16>(q.y >> 16) ||
                     odd_half<BF16>(q.z) || odd_half<BF16>(q.z >> 16) || odd_half<BF16>(q.w) || odd_half<BF16>(q.w >> 16);
    found |= (odd ? 1u : 0u) << i;
  }
  return found;
}
template <int NC, bool BF16>
__device__ __forceinline__ void clean_values(const AttendParams& p, const Walk& w, int g, uint32_t stage, int key, bool valid, int fresh, uint32_t odd) {
  const uint32_t row = stage + key * 128;
  if (!valid) {
#pragma unroll
    for (int i = 0; i < NC * 8; ++i)  // (rows begin at the same bank: each thread in an order of its own)
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(row + (i >> 3) * (128 * 128) + (((i ^ key) & 7) << 4)), "r"(0) : "memory");
  }
  while (odd != 0) {
    const int i = __ffs(odd) - 1;
    odd &= odd - 1;
    const uint4 q4 = *reinterpret_cast<const uint4*>(p.v + w.b * p.v_sb + g * p.v_sh + fresh * p.v_ss + 16 * i);
    uint32_t q[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (odd_half<BF16>(q[j])) q[j] &= 0xffff0000u;
      if (odd_half<BF16>(q[j] >> 16)) q[j] &= 0xffffu;
    }
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row + (i >> 3) * (128 * 128) + (((i ^ key) & 7) << 4)), "r"(q[0]), "r"(q[1]),
                 "r"(q[2]), "r"(q[3])
                 : "memory");
  }
}
// What key `key` of the tile at unit ub is: whether it exists; the new token that it is, < 0: a cached one.
template <class W>
__device__ __forceinline__ bool which_key(const W& w, int ub, int key, int& fresh) {
  const int unit = ub + (key >> 5);
  fresh = -1;
  if (unit >= w.unit + w.n) return false;
  if (unit < w.uc) return unit * ATT_UNIT + (key & 31) < w.len;
  const int j = (unit - w.uc) * ATT_UNIT + (key & 31);
  if (w.ud == 0 || j >= w.count) return false;
  fresh = j;
  return true;
}
// Whether the row of token t sees new token j.
template <class W>
__device__ __forceinline__ bool sees_new(const AttendParams& p, const W& w, int t, int j) {
  return t < w.count && (p.tree ? p.tree[w.b * p.tree_sb + t * p.tree_st + j * p.tree_sj] != 0 : j <= t);
}

// After a wait that ran out: the copies that the producers have started land, and the rows of what the CTA had whole read as NaN (what
// was cut, the joining kernel sees to). All threads, behind a barrier.
template <class R>
__device__ __forceinline__ void att_give_up(const AttendParams& p, const Walk& first, bool work, uint32_t bar0, const AttCtl& ac, int kv_issued,
                                            int q_issued) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) report_abort(ac.abort, p.status);
  if (warp >= 10 && lane == 0) {
    for (int s = max(q_issued - R::NQ, 0); s < q_issued; ++s) mbar_drain(bar0 + 8u * (R::B_Q + s % R::NQ), (s / R::NQ) & 1);
    for (int T = max(kv_issued - R::RINGS * (warp == 10 ? R::DK : R::DV), 0); T < kv_issued; ++T)
      mbar_drain(bar0 + 8u * (R::B_KV + (warp == 10 ? R::k_stage(T) : R::v_stage(T))), (warp == 10 ? R::k_turn(T) : R::v_turn(T)) & 1);
  }
  Walk w = first;
  bool more = work;
  while (more) {
    if (w.begins() && w.ends()) {
      const RowMap rows(p, w.b, w.item);
      const int pieces = p.c.cols / 8;
      for (int i = tid; i < p.gt * p.tt * pieces; i += ATT_THREADS) {
        int h, t;
        if (!rows.row(p, i / pieces, h, t)) continue;
        *reinterpret_cast<uint4*>(p.o + w.b * p.o_sb + h * p.o_sh + t * p.o_ss + 16 * (i % pieces)) =
            make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
        if (p.stats && i % pieces == 0) {
          float* at = p.stats + (static_cast<long long>(w.b) * p.H + h) * 2 * p.T + t;
          at[0] = at[p.T] = __int_as_float(0x7fc00000);
        }
      }
    }
    more = w.next(p);
  }
}

// What begins in this CTA and ends in another, for the joining kernel: only its last item can. w: the walk at its end.
__device__ __forceinline__ void note_parts(const AttendParams& p, const Walk& w, bool work, int chunk, int end) {
  int4 meta = make_int4(0, 0, 0, 0);
  if (work && w.begins() && !w.ends()) meta = make_int4((end - w.n + w.units - 1) / chunk - static_cast<int>(blockIdx.x) + 1, w.b, w.item, 0);
  p.part_meta[blockIdx.x] = meta;
}

// ---- up to 64 rows --------------------------------------------------------------------------------------------------------
template <int NC, int N>
struct AttCfg : AttRings<NC, N, 2, false, 2 * (N <= 32 ? 2 : 1) * 128 * N * 2 + 1024 + 16 * N * 4 + 8 * N * 4 + 24 * N * 4> {
  static constexpr int NP = N <= 32 ? 2 : 1;  // buffers for P per stream (each with barriers of its own: a stream may be a buffer ahead)
  static constexpr int P_BYTES = 128 * N * 2;
  static constexpr int TMEM = N == 64 ? 512 : (N == 32 ? 256 : 128);  // 6 N columns: S 2 x 2, O 2
};

template <int NC, int N, bool BF16>
__global__ void __launch_bounds__(ATT_THREADS, 1)
kfa_cache_attend_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                        const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmKn,
                        const __grid_constant__ CUtensorMap tmVn, const AttendParams p) {
  using R = AttCfg<NC, N>;
  constexpr int NP = R::NP;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t sKV = base, sQ = sKV + R::NS * R::STAGE, sP = sQ + R::NQ * R::Q_BYTES;
  uint8_t* small = smem + R::NS * R::STAGE + R::NQ * R::Q_BYTES + 2 * NP * R::P_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(small);
  float* s_max = reinterpret_cast<float*>(small + 1024);  // [stream][tile & 1][warp][N]
  float* s_shift = s_max + 16 * N;                        // [warp][N]
  float* s_fin = s_shift + 8 * N;                         // [segment & 1][stream]: l of four warps, m, largest score, each [N]
  const AttCtl ac(bars + R::N_BARS);
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](int i) { return bar0 + 8u * i; };
  const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31;
  if (tid == 32 * 11) {
    for (const CUtensorMap* map : {&tmQ, &tmK, &tmV, &tmKn, &tmVn}) asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
  }
  Walk first;
  int chunk, end;
  const bool work = att_setup<R>(p, bar0, ac, R::TMEM, first, chunk, end);
  const uint32_t tmem = *ac.tmem;
  const Ctl ctl{ac.abort};
  const uint32_t tmS = tmem, tmO = tmem + 4 * N;
  int kv_issued = 0, q_issued = 0;

  if (!work) {
    if (tid == 0 && !p.whole) note_parts(p, first, false, 1, 0);
  } else if (warp >= 10) {
    if constexpr (N == 64) reg_budget<ATT_REGS_ISSUE, ATT_REGS>();
    const bool values = warp == 11;
    att_produce<R>(p, first, values, sKV, sQ, bar0, ac, &tmQ, values ? &tmV : &tmK, values ? &tmVn : &tmKn, kv_issued, q_issued);
  } else if (warp >= 8) {
    if constexpr (N == 64) reg_budget<ATT_REGS_ISSUE, ATT_REGS>();
    const int st = warp - 8;
    const bool lead = elect_one();
    constexpr uint32_t IDESC_S = make_idesc(BF16, false, 128, N), IDESC_O = make_idesc(BF16, true, 128, N) | (1u << 15);
    constexpr uint32_t HI_P = sdesc_hi_for(N);
    const int k_steps = (p.c.cols + 15) / 16;
    att_issue<R, 1, NP>(
        p, first, st, bar0, ac,
        [&](const AttTile& t, int c, int) {
          const uint32_t k_lo = sdesc_lo(sKV + R::k_stage(t.T) * R::STAGE, 16), q_lo = sdesc_lo(sQ + (t.s % R::NQ) * R::Q_BYTES, 16);
          for (int kk = 0; kk < k_steps; ++kk)
            umma_ss_lead2(lead, tmS + (2 * st + (c & 1)) * N, k_lo + (((kk >> 2) * R::CHUNK + (kk & 3) * 32) >> 4), SDESC_HI,
                          q_lo + (((kk >> 2) * R::Q_CHUNK + (kk & 3) * 32) >> 4), SDESC_HI, IDESC_S, kk > 0 ? 1u : 0u);
          umma_commit_lead(lead, bar(R::B_S + 2 * st + (c & 1)));
          umma_commit_lead(lead, bar(R::B_KVFREE + R::k_stage(t.T)));
        },
        [&](const AttTile& t, int c, int) {
          // (64 columns or fewer: the matrix' rows 64 .. 127 repeat the first ones, and nobody reads them)
          const uint32_t v_lo = sdesc_lo(sKV + R::v_stage(t.T) * R::STAGE, NC == 2 ? R::CHUNK : 0);
          const uint32_t p_lo = sdesc_lo(sP + (st * NP + c % NP) * R::P_BYTES, 16);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            umma_ss_lead2(lead, tmO + st * N, v_lo + ((kk * 16 * 128) >> 4), SDESC_HI, p_lo + ((kk * 16 * 2 * N) >> 4), HI_P, IDESC_O,
                          (!t.opens || kk > 0) ? 1u : 0u);
          umma_commit_lead(lead, bar(R::B_PV + 2 * st + c % NP));
          umma_commit_lead(lead, bar(R::B_KVFREE + R::v_stage(t.T)));
        });
  } else {
    // =========================== softmax, output ===========================
    // (After a wait that ran out the role goes on without waiting: the warps of a stream meet at barriers.)
    if constexpr (N == 64) reg_budget<ATT_REGS_STREAM, ATT_REGS>();
    const int st = warp >> 2, wl = warp & 3, key = tid & 127;
    const uint32_t lane_base = static_cast<uint32_t>(wl * 32) << 16;
    constexpr int PER = N / 32 > 0 ? N / 32 : 1;  // columns whose maximum a lane keeps: lane, lane + 32
    float* shift = s_shift + warp * N;
    const float c_log2 = p.c_log2;
    const float2 c2 = make_float2(c_log2, c_log2);
    Walk w = first;
    bool more = true, ok = true;
    int c = 0, T0 = 0, s = 0;  // the stream's tiles; tiles and segments before
    while (more) {
      const RowMap rows(p, w.b, w.item);
      float l[N], m_ref[PER], m_top[PER];
#pragma unroll
      for (int i = 0; i < N; ++i) l[i] = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) m_ref[i] = m_top[i] = -INFINITY;
      bool opens = true;
      const int tiles = w.tiles();
      for (int t = 0; t < tiles; ++t) {
        const int T = T0 + t;
        if ((T & 1) != st) continue;
        const int ub = w.unit + 4 * t;
        const bool full = 4 * t + 4 <= w.n && (ub + 4) * ATT_UNIT <= w.len && ub + 4 <= w.uc;
        int fresh = -1;
        const bool valid = full || which_key(w, ub, key, fresh);
        // ahead of the scores: a bit per token of the row tile that sees this new token (N rows hold at most N tokens)
        uint32_t see[PER], odd = 0u;
        if (!full) {
#pragma unroll
          for (int k = 0; k < PER; ++k) {
            see[k] = valid ? 0xffffffffu : 0u;
            if (fresh >= 0) {
              const int t0 = rows.t0 + 32 * k, n = min(min(p.tt - 32 * k, p.T - t0), w.count - t0);  // tokens that there are
              see[k] = n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u);
              if (n > 0 && p.tree != nullptr) see[k] = tree_bits(p.tree + w.b * p.tree_sb + t0 * p.tree_st + fresh * p.tree_sj, p.tree_st, n);
              if (p.tree == nullptr && fresh > t0) see[k] &= fresh - t0 >= 32 ? 0u : 0xffffffffu << (fresh - t0);
            }
          }
          odd = odd_values<BF16>(p, w, rows.g, fresh);
        }
        if (ok) ok = wait_warp(bar(R::B_S + 2 * st + (c & 1)), (c >> 1) & 1, ctl, 78);
        tc_fence_after();
        float x[N];
        tmem_ld_cols<N>(tmS + lane_base + (2 * st + (c & 1)) * N, x);
        tmem_wait_ld();
        if (!full) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const int dt = fresh >= 0 ? static_cast<int>(p.by_gt.div(i)) : 0;
            const uint32_t word = PER == 1 || dt < 32 ? see[0] : see[PER - 1];
            if (!((word >> (dt & 31)) & 1u)) x[i] = -INFINITY;
          }
        }
        // ---- column maxima ----
        float top[PER];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float y = warp_max(x[i]);
          if (N < 32 ? (lane & (N - 1)) == i : lane == (i & 31)) top[i / 32] = y;
        }
        float* mx = s_max + (2 * st + (c & 1)) * 4 * N;
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (lane + 32 * i < N) mx[wl * N + lane + 32 * i] = top[i];
        if (st == 0) named_sync<1, 128>();
        else named_sync<2, 128>();
        bool grew = false;
        float alpha[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int col = (lane & (N < 32 ? N - 1 : 31)) + 32 * i;
          const float y = fmaxf(fmaxf(mx[col], mx[N + col]), fmaxf(mx[2 * N + col], mx[3 * N + col]));
          m_top[i] = fmaxf(m_top[i], y);
          const bool move = m_ref[i] == -INFINITY ? y > -INFINITY : y > m_ref[i] + p.slack;
          alpha[i] = 1.f;
          if (move) {
            alpha[i] = m_ref[i] == -INFINITY ? 0.f : ex2((m_ref[i] - y) * c_log2);
            m_ref[i] = y;
          }
          grew |= move;
          if (lane + 32 * i < N) shift[col] = m_ref[i] == -INFINITY ? 0.f : -m_ref[i];
        }
        grew = __any_sync(0xffffffffu, grew);  // the same in all warps of the stream
        __syncwarp();
        if (grew && !opens) {
          // sums and O of the earlier tiles, to the new maxima
          if (ok) ok = wait_warp(bar(R::B_PV + 2 * st + (c - 1) % NP), ((c - 1) / NP) & 1, ctl, 79);
          tc_fence_after();
#pragma unroll
          for (int i = 0; i < N; i += 16) {
            float o[16];
            tmem_ld16(tmO + lane_base + st * N + i, reinterpret_cast<uint32_t*>(o));
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float a = __shfl_sync(0xffffffffu, alpha[(i + j) / 32], (i + j) & 31);
              o[j] *= a;
              l[i + j] *= a;
            }
            tmem_st16(tmO + lane_base + st * N + i, reinterpret_cast<const uint32_t*>(o));
          }
          tmem_wait_st();
        }
        // ---- P ----
        if (c >= NP && ok) ok = wait_warp(bar(R::B_PV + 2 * st + c % NP), (c / NP - 1) & 1, ctl, 80);  // its buffer has been read
        const uint32_t sp = sP + (st * NP + c % NP) * R::P_BYTES;
#pragma unroll
        for (int i = 0; i < N; i += 8) {
          const float4 a = *reinterpret_cast<const float4*>(shift + i), b = *reinterpret_cast<const float4*>(shift + i + 4);
          const float2 mm[4] = {make_float2(a.x, a.y), make_float2(a.z, a.w), make_float2(b.x, b.y), make_float2(b.z, b.w)};
          float e[8];
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            const float2 y = __fmul2_rn(__fadd2_rn(make_float2(x[i + j], x[i + j + 1]), mm[j / 2]), c2);
            e[j] = ex2(y.x);
            e[j + 1] = ex2(y.y);
            const float2 sum = __fadd2_rn(make_float2(l[i + j], l[i + j + 1]), make_float2(e[j], e[j + 1]));
            l[i + j] = sum.x;
            l[i + j + 1] = sum.y;
          }
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(sp + p_piece<N>(key, i / 8)), "r"(pack16<BF16>(e[0], e[1])),
                       "r"(pack16<BF16>(e[2], e[3])), "r"(pack16<BF16>(e[4], e[5])), "r"(pack16<BF16>(e[6], e[7]))
                       : "memory");
        }
        if (!full) {
          // (The tile before has to be done with: until then the barrier of this one's stage may be a turn behind.)
          if (c > 0 && ok) ok = wait_warp(bar(R::B_PV + 2 * st + (c - 1) % NP), ((c - 1) / NP) & 1, ctl, 81);
          if (ok) ok = wait_warp(bar(R::B_KV + R::v_stage(T)), R::v_turn(T) & 1, ctl, 82);
          clean_values<NC, BF16>(p, w, rows.g, sKV + R::v_stage(T) * R::STAGE, key, valid, fresh, odd);
          if (odd != 0) ac.odd[st] = s + 1;
        }
        fence_async_smem();
        tc_fence_before();
        mbar_arrive(bar(R::B_P + 2 * st + c % NP));
        opens = false;
        ++c;
      }
      T0 += tiles;
      // ---- the segment's end ----
      columns_over_lanes<N>(l, lane);
      float* fin = s_fin + ((s & 1) * 2 + st) * 6 * N;
      if constexpr (N == 64) {
        fin[wl * N + 2 * lane] = l[0];
        fin[wl * N + 2 * lane + 1] = l[1];
      } else if constexpr (N == 32) {
        fin[wl * N + lane] = l[0];
      } else {
        if (!(lane & 1)) fin[wl * N + lane / 2] = l[0];
      }
      if (wl == 0) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (lane + 32 * i < N) {
            fin[4 * N + lane + 32 * i] = m_ref[i];
            fin[5 * N + lane + 32 * i] = m_top[i];
          }
      }
      if (!opens && ok) ok = wait_warp(bar(R::B_PV + 2 * st + (c - 1) % NP), ((c - 1) / NP) & 1, ctl, 83);
      tc_fence_before();
      named_sync<3, 256>();
      tc_fence_after();
      const bool bad = *ac.bad != 0;
      const bool whole = w.begins() && w.ends();
      const long long slot = 2ll * blockIdx.x + (w.begins() ? 1 : 0);
      // new tokens of the segment, where some of their values were left out (a stream may be one segment ahead: >=)
      const bool odd = ac.odd[0] >= s + 1 || ac.odd[1] >= s + 1;
      const int j0 = max(w.unit - w.uc, 0) * ATT_UNIT, j1 = odd ? min((w.unit + w.n - w.uc) * ATT_UNIT, w.count) : 0;
      const int d = wl * 32 + lane;
      constexpr int W = N / 2;  // columns of a thread
      const int c0 = st * W;
      // lane i (i < W): column i's factors and statistics
      const float* f0 = s_fin + (s & 1) * 12 * N + c0 + (lane & (W - 1));
      const float* f1 = f0 + 6 * N;
      const float m0 = f0[4 * N], m1 = f1[4 * N], m = fmaxf(m0, m1), top = fmaxf(f0[5 * N], f1[5 * N]);
      const float l0 = (f0[0] + f0[N]) + (f0[2 * N] + f0[3 * N]), l1 = (f1[0] + f1[N]) + (f1[2 * N] + f1[3 * N]);
      float a0 = part_factor(m0, l0, m, c_log2), a1 = part_factor(m1, l1, m, c_log2);
      const float l_all = l0 * a0 + l1 * a1;
      int h, tk;
      const bool exists = rows.row(p, c0 + (lane & (W - 1)), h, tk);
      const long long off = exists ? w.b * p.o_sb + h * p.o_sh + tk * p.o_ss : -1;
      const bool some = exists && tk < w.count && l_all != 0.f;
      const float nan = __int_as_float(0x7fc00000);
      if (whole) {
        const float inv = some ? 1.f / l_all : 0.f;
        if (p.stats && wl == 0 && exists && lane < W) {
          float* at = p.stats + (static_cast<long long>(w.b) * p.H + h) * 2 * p.T + tk;
          at[0] = bad ? nan : (some ? top : INFINITY);
          at[p.T] = bad ? nan : (some ? log2f(l_all) + (m - top) * c_log2 : 0.f);
        }
        a0 = some ? a0 * inv : -1.f;
        a1 = some ? a1 * inv : -1.f;
      } else if (wl == 0 && lane < W) {
        float* at = p.part_ml + slot * 3 * p.rows + c0 + lane;
        at[0] = m;
        at[p.rows] = l_all;
        at[2 * p.rows] = top;
      }
      float o0[W], o1[W];
      tmem_ld_cols<W>(tmO + lane_base + c0, o0);
      tmem_ld_cols<W>(tmO + lane_base + N + c0, o1);
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float x0 = __shfl_sync(0xffffffffu, a0, i), x1 = __shfl_sync(0xffffffffu, a1, i);
        o0[i] = (x0 < 0.f ? 0.f : o0[i] * x0) + (x1 < 0.f ? 0.f : o1[i] * x1);  // (a stream without tiles has left nothing there)
      }
      if (d < p.c.cols) {
        for (int j = j0; j < j1; ++j) {
          const float y = load16<BF16>(p.v + w.b * p.v_sb + rows.g * p.v_sh + j * p.v_ss + 2 * d);
          if (fabsf(y) < INFINITY) continue;
#pragma unroll
          for (int i = 0; i < W; ++i)
            if (sees_new(p, w, rows.t0 + static_cast<int>(p.by_gt.div(c0 + i)), j)) o0[i] += y;
        }
      }
      if (whole) {
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const long long at = __shfl_sync(0xffffffffu, off, i);
          if (at >= 0 && d < p.c.cols) {
            const uint32_t y = pack16<BF16>(bad ? nan : o0[i], 0.f);
            *reinterpret_cast<uint16_t*>(p.o + at + 2 * d) = static_cast<uint16_t>(y);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < W; ++i)
          if (c0 + i < p.gt * p.tt) p.part_o[(slot * p.rows + c0 + i) * 128 + d] = o0[i];
      }
      tc_fence_before();
      if (tiles > 1 || ((T0 - 1) & 1) == 0) mbar_arrive(bar(R::B_OFREE));
      if (tiles > 1 || ((T0 - 1) & 1) == 1) mbar_arrive(bar(R::B_OFREE + 1));
      mbar_arrive(bar(R::B_QFREE + s % R::NQ));
      ++s;
      more = w.next(p);
    }
    if (tid == 0 && !p.whole) note_parts(p, w, true, chunk, end);
  }

  // ---- teardown (every thread gets here, also after an abort) ----
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *ac.bad) report(p.status, DEV_BAD_CACHE);
  if (*ac.abort) att_give_up<R>(p, first, work, bar0, ac, kv_issued, q_issued);
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, R::TMEM);
  }
}

// ---- more rows ------------------------------------------------------------------------------------------------------------
// HALVES: 1: up to 128 rows, tiles to the streams in turn; 2: up to 256 rows, a half of them to each stream.
template <int NC, int HALVES>
struct AttRowsCfg : AttRings<NC, 128 * HALVES, HALVES == 1 ? 2 : 1, HALVES == 2, 1024 + 2 * 2 * 128 * 3 * 4 + 8 * 2048> {
  static constexpr int TMEM = 512;  // S 2 x 128; O 2 x 128
};

// A tile's 128 score columns are made and used as two halves of 64 keys, each with its own barriers: P (16-bit) lies over the first 32
// of its half's columns, and while one half's values are multiplied and its next scores made, the thread works on the other.
template <int NC, int HALVES, bool BF16>
__global__ void __launch_bounds__(ATT_THREADS, 1)
kfa_cache_attend_rows_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                             const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmKn,
                             const __grid_constant__ CUtensorMap tmVn, const AttendParams p) {
  using R = AttRowsCfg<NC, HALVES>;
  constexpr bool BOTH = R::BOTH;
  constexpr int D = 64 * NC;  // columns of O (those that the head dim does not have are zeros)

  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t sKV = base, sQ = sKV + R::NS * R::STAGE;
  uint8_t* small = smem + R::NS * R::STAGE + R::NQ * R::Q_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(small);
  float* s_fin = reinterpret_cast<float*>(small + 1024);  // [segment & 1][stream][m, l, largest score][128 rows]
  const AttCtl ac(bars + R::N_BARS);
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](int i) { return bar0 + 8u * i; };
  const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31;
  if (tid == 32 * 11) {
    for (const CUtensorMap* map : {&tmQ, &tmK, &tmV, &tmKn, &tmVn}) asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
  }
  Walk first;
  int chunk, end;
  const bool work = att_setup<R>(p, bar0, ac, R::TMEM, first, chunk, end);
  const uint32_t tmem = *ac.tmem;
  const Ctl ctl{ac.abort};
  int kv_issued = 0, q_issued = 0;

  if (!work) {
    if (tid == 0 && !p.whole) note_parts(p, first, false, 1, 0);
  } else if (warp >= 10) {
    reg_budget<ATT_REGS_ISSUE, ATT_REGS>();
    const bool values = warp == 11;
    att_produce<R>(p, first, values, sKV, sQ, bar0, ac, &tmQ, values ? &tmV : &tmK, values ? &tmVn : &tmKn, kv_issued, q_issued);
  } else if (warp >= 8) {
    reg_budget<ATT_REGS_ISSUE, ATT_REGS>();
    const int st = warp - 8;
    const bool lead = elect_one();
    constexpr uint32_t IDESC_S = make_idesc(BF16, false, 128, 64), IDESC_O = make_idesc(BF16, true, 128, D);
    const uint32_t tS = tmem + 128 * st, tO = tmem + 256 + 128 * st;
    const int k_steps = (p.c.cols + 15) / 16;
    att_issue<R, 2, 1>(
        p, first, st, bar0, ac,
        [&](const AttTile& t, int, int half) {
          const uint32_t q_lo = sdesc_lo(sQ + (t.s % R::NQ) * R::Q_BYTES + (BOTH ? st * 128 * 128 : 0), 16);
          const uint32_t k_lo = sdesc_lo(sKV + R::k_stage(t.T) * R::STAGE + half * 64 * 128, 16);
          for (int kk = 0; kk < k_steps; ++kk)
            umma_ss_lead(lead, tS + 64 * half, q_lo + (((kk >> 2) * R::Q_CHUNK + (kk & 3) * 32) >> 4),
                         k_lo + (((kk >> 2) * R::CHUNK + (kk & 3) * 32) >> 4), IDESC_S, kk > 0 ? 1u : 0u);
          umma_commit_lead(lead, bar(R::B_S + 2 * st + half));
          if (half == 1) umma_commit_lead(lead, bar(R::B_KVFREE + R::k_stage(t.T)));
          if (BOTH && half == 1 && t.closes) umma_commit_lead(lead, bar(R::B_QFREE + t.s % R::NQ));  // (one buffer: the next queries come as soon as may be)
        },
        [&](const AttTile& t, int, int half) {
          const uint32_t v_lo = sdesc_lo(sKV + R::v_stage(t.T) * R::STAGE + half * 64 * 128, R::CHUNK);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_ts_lead(lead, tO, tS + 64 * half + kk * 8, v_lo + ((kk * 16 * 128) >> 4), IDESC_O, (!t.opens || half > 0 || kk > 0) ? 1u : 0u);
          umma_commit_lead(lead, bar(R::B_PV + 2 * st + half));
          if (half == 1) umma_commit_lead(lead, bar(R::B_KVFREE + R::v_stage(t.T)));
        });
  } else {
    // =========================== softmax, output ===========================
    // (After a wait that ran out the role goes on without waiting: the streams meet at barriers.)
    reg_budget<ATT_REGS_STREAM, ATT_REGS>();
    const int st = warp >> 2, wl = warp & 3, r_in = tid & 127;
    const uint32_t lane_base = static_cast<uint32_t>(wl * 32) << 16;
    const uint32_t tS = tmem + 128 * st + lane_base, tO = tmem + 256 + 128 * st + lane_base;
    const float c_log2 = p.c_log2;
    const float2 c2 = make_float2(c_log2, c_log2);
    const int r = (BOTH ? 128 * st : 0) + r_in;  // the thread's row of the tile
    Walk w = first;
    bool more = true, ok = true;
    int c = 0, T0 = 0, s = 0;  // the stream's tiles; tiles and segments before
    while (more) {
      const RowMap rows(p, w.b, w.item);
      int h, tk;
      const bool exists = rows.row(p, r, h, tk);
      float l = 0.f, m_ref = -INFINITY, m_top = -INFINITY;
      const int tiles = w.tiles();
      // the stream's tiles of the segment, every STEP-th from t_first on, as pieces of 64 keys; those below t_full hold cached keys only
      constexpr int STEP = BOTH ? 1 : 2;
      const int t_first = BOTH || (T0 & 1) == st ? 0 : 1, pieces = 2 * ((tiles - t_first + STEP - 1) / STEP);
      const int t_full = max(min(w.n, min(w.len / ATT_UNIT, w.uc) - w.unit), 0) / 4;
      const int c0 = c;
      float2 x[32];
      bool loaded = false;
      int fresh = -1;
      bool valid = true;
      uint32_t odd_bits = 0u;
#pragma unroll 1
      for (int i = 0; i < pieces; ++i) {
        const int half = i & 1, t = t_first + (i >> 1) * STEP;
        c = c0 + (i >> 1);
        const bool full = t < t_full;
        uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
        if (!full) {
          const int ub = w.unit + 4 * t;
          if (half == 0) {
            valid = which_key(w, ub, r_in, fresh);
            odd_bits = odd_values<BF16>(p, w, rows.g, fresh);
          }
          seen[0] = exists ? seen_word(p, w, ub + 2 * half, tk) : 0u;
          seen[1] = exists ? seen_word(p, w, ub + 2 * half + 1, tk) : 0u;
        }
        if (!loaded) {
          if (ok) ok = wait_warp(bar(R::B_S + 2 * st + half), c & 1, ctl, 78);
          tc_fence_after();
          tmem_ld_cols<64>(tS + 64 * half, reinterpret_cast<float*>(x));
          tmem_wait_ld();
        }
        if (!full) {
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if (!((seen[j / 16] >> (2 * j & 31)) & 1u)) x[j].x = -INFINITY;
            if (!((seen[j / 16] >> ((2 * j + 1) & 31)) & 1u)) x[j].y = -INFINITY;
          }
        }
        float y[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < 32; ++j) y[j & 3] = fmaxf(y[j & 3], fmaxf(x[j].x, x[j].y));
        const float top = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
        m_top = fmaxf(m_top, top);
        const bool move = m_ref == -INFINITY ? top > -INFINITY : top > m_ref + p.slack;
        if (__any_sync(0xffffffffu, move)) {
          const float alpha = !move ? 1.f : (m_ref == -INFINITY ? 0.f : ex2((m_ref - top) * c_log2));
          if (i > 0) {  // every product issued so far has to have retired
            const int before = 2 * c + half - 1;
            if (ok) ok = wait_warp(bar(R::B_PV + 2 * st + (before & 1)), (before >> 1) & 1, ctl, 79);
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < D; k += 32) {
              float o[32];
              tmem_ld32(tO + k, reinterpret_cast<uint32_t*>(o));
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] *= alpha;
              tmem_st32(tO + k, reinterpret_cast<const uint32_t*>(o));
            }
            tmem_wait_st();
            l *= alpha;
          }
          if (move) m_ref = top;
        }
        const float sh = m_ref == -INFINITY ? 0.f : -m_ref;
        const float2 s2 = make_float2(sh, sh);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int k = 0; k < 32; k += 16) {  // (stored by the half: fewer registers at once)
          uint32_t pk[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float2 e = __fmul2_rn(__fadd2_rn(x[k + j], s2), c2);
            e.x = ex2(e.x);
            e.y = ex2(e.y);
            sum[j & 1] = __fadd2_rn(sum[j & 1], e);
            pk[j] = pack16<BF16>(e.x, e.y);
          }
          tmem_st16(tS + 64 * half + k, pk);
        }
        const bool early = mbar_test(bar(R::B_S + 2 * st + (half ^ 1)), (c + half) & 1);  // the next piece's scores are there already
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        if (!full && half == 0) {
          // (The tile before has to be done with: until then the barrier of this one's stage may be a turn behind.)
          const int stage = R::v_stage(T0 + t), turn = R::v_turn(T0 + t);
          if (c > 0 && ok) ok = wait_warp(bar(R::B_PV + 2 * st + 1), (c - 1) & 1, ctl, 81);
          if (ok) ok = wait_warp(bar(R::B_KV + stage), turn & 1, ctl, 82);
          clean_values<NC, BF16>(p, w, rows.g, sKV + stage * R::STAGE, r_in, valid, fresh, odd_bits);
          if (odd_bits != 0) ac.odd[st] = s + 1;
          fence_async_smem();
        }
        // The next piece's scores are fetched while P is on its way into tensor memory. (A wait costs 300 clk even for what is there, the way
        // in 200.)
        loaded = i + 1 < pieces && __all_sync(0xffffffffu, early);
        auto announce = [&] {
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(bar(R::B_P + 2 * st + half));
        };
        if (loaded) {  // (load and wait in one piece of straight code: nothing moves the registers in between)
          tc_fence_after();
          tmem_ld_cols<64>(tS + 64 * (half ^ 1), reinterpret_cast<float*>(x));
          announce();
          tmem_wait_ld();
        } else {
          announce();
        }
      }
      const bool opens = pieces == 0;  // the stream had no tile
      c = c0 + pieces / 2;
      T0 += tiles;
      // ---- the segment's end ----
      if (!opens && ok) ok = wait_warp(bar(R::B_PV + 2 * st + 1), (c - 1) & 1, ctl, 83);
      float a0 = 1.f, a1 = 0.f, m = m_ref, top = m_top, l_all = l;  // factors of the streams' O, the row's statistics
      tc_fence_before();
      if constexpr (BOTH) {
        if (st == 0) named_sync<1, 128>();  // (what the stream's threads have met of values that are not finite)
        else named_sync<2, 128>();
        a0 = part_factor(m, l, m, c_log2);
      } else {
        float* fin = s_fin + (s & 1) * 768 + st * 384 + r_in;
        fin[0] = m_ref;
        fin[128] = l;
        fin[256] = m_top;
        named_sync<3, 256>();
        const float* f = s_fin + (s & 1) * 768 + r_in;
        const float m0 = f[0], m1 = f[384], l0 = f[128], l1 = f[512];
        m = fmaxf(m0, m1);
        top = fmaxf(f[256], f[640]);
        a0 = part_factor(m0, l0, m, c_log2);
        a1 = part_factor(m1, l1, m, c_log2);
        l_all = l0 * a0 + l1 * a1;
      }
      tc_fence_after();
      const bool bad = *ac.bad != 0;
      const bool whole = w.begins() && w.ends();
      const long long slot = 2ll * blockIdx.x + (w.begins() ? 1 : 0);
      const bool odd = ac.odd[st] >= s + 1 || (!BOTH && ac.odd[1 - st] >= s + 1);
      const int j0 = max(w.unit - w.uc, 0) * ATT_UNIT, j1 = odd ? min((w.unit + w.n - w.uc) * ATT_UNIT, w.count) : 0;
      const bool some = exists && tk < w.count && l_all != 0.f;
      const float nan = __int_as_float(0x7fc00000);
      const bool writes = BOTH || st == 0;  // of the row's statistics
      if (whole) {
        const float inv = some ? 1.f / l_all : 0.f;
        if (p.stats && exists && writes) {
          float* at = p.stats + (static_cast<long long>(w.b) * p.H + h) * 2 * p.T + tk;
          at[0] = bad ? nan : (some ? top : INFINITY);
          at[p.T] = bad ? nan : (some ? log2f(l_all) + (m - top) * c_log2 : 0.f);
        }
        a0 = some ? a0 * inv : -1.f;
        a1 = some ? a1 * inv : -1.f;
      } else if (writes && r < p.gt * p.tt) {
        float* at = p.part_ml + slot * 3 * p.rows + r;
        at[0] = m;
        at[p.rows] = l_all;
        at[2 * p.rows] = top;
      }
      // Columns: all of the stream's own rows (BOTH), or every second 32 of the shared ones. A thread holds a row, and a store of 16 bytes by
      // each of 32 rows touches 32 lines: through 2 KB a warp of shared memory whole pieces of rows are written one after the other. A part
      // lies as the threads have it, 4 columns of 32 rows after 4 columns of 32 rows: each store is 512 bytes in one piece.
      const uint32_t turn = (lane >> 1) & 3;
      const uint32_t out_stage = smem_u32(s_fin) + 6144 + warp * 2048;  // 32 rows of 64 bytes
      const long long off = exists ? w.b * p.o_sb + static_cast<long long>(h) * p.o_sh + tk * p.o_ss : -1;
      const int r_warp = r - lane;
#pragma unroll 1
      for (int i = BOTH ? 0 : 32 * st; i < D; i += BOTH ? 32 : 64) {
        float o0[32];
        tmem_ld32((BOTH ? tO : tmem + 256 + lane_base) + i, reinterpret_cast<uint32_t*>(o0));
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j) o0[j] = a0 < 0.f ? 0.f : o0[j] * a0;
        if constexpr (!BOTH) {
          float o1[32];
          tmem_ld32(tmem + 384 + lane_base + i, reinterpret_cast<uint32_t*>(o1));
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) o0[j] += a1 < 0.f ? 0.f : o1[j] * a1;
        }
        for (int j = j0; j < j1; ++j) {
          if (!exists || !sees_new(p, w, tk, j)) continue;
          const uint8_t* v = p.v + w.b * p.v_sb + rows.g * p.v_sh + j * p.v_ss + 2 * i;
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            if (i + k >= p.c.cols) break;
            const float y = load16<BF16>(v + 2 * k);
            if (!(fabsf(y) < INFINITY)) o0[k] += y;
          }
        }
        __syncwarp();
        if (whole) {
#pragma unroll
          for (int j = 0; j < 4; ++j)  // rows of 64 bytes: 4 pieces
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(out_stage + lane * 64 + ((j ^ turn) << 4)),
                         "r"(pack16<BF16>(o0[8 * j], o0[8 * j + 1])), "r"(pack16<BF16>(o0[8 * j + 2], o0[8 * j + 3])),
                         "r"(pack16<BF16>(o0[8 * j + 4], o0[8 * j + 5])), "r"(pack16<BF16>(o0[8 * j + 6], o0[8 * j + 7]))
                         : "memory");
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int row = 8 * k + (lane >> 2), piece = lane & 3;
            const long long at = __shfl_sync(0xffffffffu, off, row);
            uint4 y;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(y.x), "=r"(y.y), "=r"(y.z), "=r"(y.w)
                         : "r"(out_stage + row * 64 + ((piece ^ ((row >> 1) & 3)) << 4))
                         : "memory");
            if (bad) y = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
            if (at >= 0 && i + 8 * piece < p.c.cols) *reinterpret_cast<uint4*>(p.o + at + 2 * i + 16 * piece) = y;
          }
        } else if (r_warp < p.gt * p.tt) {
          float4* at = reinterpret_cast<float4*>(p.part_o + (slot * p.rows + r_warp) * 128) + 8 * i + lane;
#pragma unroll
          for (int j = 0; j < 8; ++j) at[32 * j] = make_float4(o0[4 * j], o0[4 * j + 1], o0[4 * j + 2], o0[4 * j + 3]);
        }
      }
      tc_fence_before();
      if (BOTH) {
        mbar_arrive(bar(R::B_OFREE + st));  // (its queries were freed by the last scores)
      } else {
        mbar_arrive(bar(R::B_QFREE + s % R::NQ));
        if (tiles > 1 || ((T0 - 1) & 1) == 0) mbar_arrive(bar(R::B_OFREE));
        if (tiles > 1 || ((T0 - 1) & 1) == 1) mbar_arrive(bar(R::B_OFREE + 1));
      }
      ++s;
      more = w.next(p);
    }
    if (tid == 0 && !p.whole) note_parts(p, w, true, chunk, end);
  }

  // ---- teardown (every thread gets here, also after an abort) ----
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *ac.bad) report(p.status, DEV_BAD_CACHE);
  if (*ac.abort) att_give_up<R>(p, first, work, bar0, ac, kv_issued, q_issued);
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, R::TMEM);
  }
}

// Joins the parts of the items that were cut: CTA x has the item that begins in CTA x of the kernel above, a warp a row, a lane four
// columns. Starts while that kernel ends and waits for it. 32 parts at a time: a lane has the factor of one, and all add up their columns; the
// first AHEAD parts' columns are on their way while the factors are found (drafts of 7 tokens 15.2 -> 14.2 us).
template <bool BF16>
__global__ void __launch_bounds__(256) kfa_cache_join_kernel(const AttendParams p) {
  constexpr int AHEAD = 4;
  wait_for_previous();
  let_next_begin();
  const int4 meta = p.part_meta[blockIdx.x];
  if (meta.x == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = blockIdx.y * 8 + warp;
  const RowMap rows(p, meta.y, meta.z);
  int h, t;
  if (!rows.row(p, r, h, t)) return;
  const bool bad = *reinterpret_cast<const volatile int*>(p.status) != 0;
  const int count = p.counts ? min(max(p.counts[meta.y], 0), p.T) : p.T;
  // part i: the first in slot 1 of its CTA, the others in slot 0 of theirs
  auto slot = [&](int i) { return 2ll * (blockIdx.x + i) + (i == 0 ? 1 : 0); };
  const float* o_row = p.part_o + r * 128 + 4 * lane;
  float m = -INFINITY, top = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < meta.x; i0 += 32) {
    const int n = min(32, meta.x - i0);
    auto part = [&](int i) { return *reinterpret_cast<const float4*>(o_row + slot(i0 + i) * p.rows * 128); };
    float4 x[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) x[i] = part(min(i, n - 1));
    float mi = -INFINITY, li = 0.f, ti = -INFINITY;
    if (lane < n) {
      const float* ml = p.part_ml + slot(i0 + lane) * 3 * p.rows + r;
      mi = ml[0];
      li = ml[p.rows];
      ti = ml[2 * p.rows];
    }
    const float m_new = fmaxf(m, warp_max(mi));
    top = fmaxf(top, warp_max(ti));
    if (i0) {
      const float before = part_factor(m, l, m_new, p.c_log2), a = before < 0.f ? 0.f : before;
      l *= a;
      o = make_float4(o.x * a, o.y * a, o.z * a, o.w * a);
    }
    m = m_new;
    const float a = lane < n ? part_factor(mi, li, m, p.c_log2) : -1.f;
    li *= a;
    auto add = [&](int i, const float4& y) {
      const float ai = __shfl_sync(0xffffffffu, a, i);
      l += __shfl_sync(0xffffffffu, li, i);
      if (!(ai < 0.f)) {
        o.x += ai * y.x;
        o.y += ai * y.y;
        o.z += ai * y.z;
        o.w += ai * y.w;
      }
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (i < n) add(i, x[i]);
#pragma unroll 4
    for (int i = AHEAD; i < n; ++i) add(i, part(i));
  }
  const bool some = t < count && l != 0.f;
  const float nan = __int_as_float(0x7fc00000), inv = some ? 1.f / l : 0.f;
  if (bad) o = make_float4(nan, nan, nan, nan);
  else if (!some) o = make_float4(0.f, 0.f, 0.f, 0.f);
  else o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  if (4 * lane < p.c.cols)
    *reinterpret_cast<uint2*>(p.o + meta.y * p.o_sb + h * p.o_sh + t * p.o_ss + 8 * lane) = make_uint2(pack16<BF16>(o.x, o.y), pack16<BF16>(o.z, o.w));
  if (p.stats && lane == 0) {
    float* at = p.stats + (static_cast<long long>(meta.y) * p.H + h) * 2 * p.T + t;
    at[0] = bad ? nan : (some ? top : INFINITY);
    at[p.T] = bad ? nan : (some ? log2f(l) + (m - top) * p.c_log2 : 0.f);
  }
}

// The same for the kernel for more rows, whose parts lie by columns: a lane a row, a warp 16 columns of 32 rows, nothing exchanged. One pass:
// what is there is scaled down when a part has a larger maximum. (16 trees of 64 tokens, 256 rows mostly in two parts: 102.9 us with parts by
// rows and a warp a row, 96.4 with 8 lanes a row, 93.7 so.)
template <bool BF16>
__global__ void __launch_bounds__(256) kfa_cache_join_rows_kernel(const AttendParams p) {
  wait_for_previous();
  let_next_begin();
  const int4 meta = p.part_meta[blockIdx.x];
  if (meta.x == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = blockIdx.y * 32 + lane;
  const RowMap rows(p, meta.y, meta.z);
  int h, t;
  if (16 * warp >= p.c.cols || !rows.row(p, r, h, t)) return;
  const bool bad = *reinterpret_cast<const volatile int*>(p.status) != 0;
  const int count = p.counts ? min(max(p.counts[meta.y], 0), p.T) : p.T;
  const float* ml = p.part_ml + (2ll * blockIdx.x + 1) * 3 * p.rows + r;  // the first part in slot 1 of its CTA, the others in slot 0 of theirs
  const float4* from = reinterpret_cast<const float4*>(p.part_o + ((2ll * blockIdx.x + 1) * p.rows + 32 * blockIdx.y) * 128) + 128 * warp + lane;
  float m = -INFINITY, top = -INFINITY, l = 0.f, o[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) o[k] = 0.f;
#pragma unroll 2
  for (int i = 0; i < meta.x; ++i) {
    const float mi = ml[0], li = ml[p.rows], ti = ml[2 * p.rows];
    float4 x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = from[32 * k];
    const int next = i == 0 ? 1 : 2;  // slots
    ml += next * 3 * p.rows;
    from += next * p.rows * 32;
    const float m_new = fmaxf(m, mi), f = part_factor(m, l, m_new, p.c_log2), fi = part_factor(mi, li, m_new, p.c_log2);
    top = fmaxf(top, ti);
    m = m_new;
    l = l * f + li * fi;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float y[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
      for (int q = 0; q < 4; ++q) o[4 * k + q] = o[4 * k + q] * f + (fi < 0.f ? 0.f : y[q] * fi);
    }
  }
  const bool some = t < count && l != 0.f;
  const float nan = __int_as_float(0x7fc00000), inv = some ? 1.f / l : 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) o[k] = bad ? nan : (some ? o[k] * inv : 0.f);
  unsigned char* out = p.o + meta.y * p.o_sb + h * p.o_sh + t * p.o_ss + 32 * warp;
#pragma unroll
  for (int k = 0; k < 16; k += 8)
    if (16 * warp + k < p.c.cols)
      *reinterpret_cast<uint4*>(out + 2 * k) = make_uint4(pack16<BF16>(o[k], o[k + 1]), pack16<BF16>(o[k + 2], o[k + 3]),
                                                          pack16<BF16>(o[k + 4], o[k + 5]), pack16<BF16>(o[k + 6], o[k + 7]));
  if (p.stats && warp == 0) {
    float* at = p.stats + (static_cast<long long>(meta.y) * p.H + h) * 2 * p.T + t;
    at[0] = bad ? nan : (some ? top : INFINITY);
    at[p.T] = bad ? nan : (some ? log2f(l) + (m - top) * p.c_log2 : 0.f);
  }
}

}  // namespace kfa
