// Attention of a sequence's newest tokens (one, a tree of drafted ones, a chunk of a prompt) to its cached keys and to one another.
//
//   S = q K^T,  m = max S,  P = exp2((S - m) c),  l = sum P,  out = P V / l,  c = scale * log2(e)
//
// What bounds it: the keys and values, read once each (2 x 2 D bytes a position and K / V head). All query rows that share them, the
// query heads of a K / V head times the new tokens, are one tile; with few rows that is far below what makes the tensor core
// the limit, so the tile is turned around: the KEYS are the 128 rows of the matrix instructions, the query rows their N columns
// (16, 32 or 64), and nothing is computed for rows that are not there:
//   S^T [128 keys x N] = K Q^T                 A = K from shared memory as copied, B = Q
//   O^T [D x N]       += V^T P^T               A = V as copied (the transposed, MN-major, operand), B = P^T from shared memory
// A thread holds one key's scores. The maximum over keys is a warp reduction per column and an exchange between four warps; the sum
// over keys stays in the thread until the end. O^T is rescaled only when a row's maximum grew by more than a factor of 2^8
// (the numerators may be up to 2^8 then, which 16-bit P takes at the same relative precision).
//
// Work is cut by keys, not by sequences: the keys of all (sequence, K / V head, row tile) items are counted in units of 32 and every CTA
// takes an equal stretch, whatever the lengths (which only the device knows). An item that one CTA has whole is written by it;
// of the others the CTA leaves its part (unnormalised O in fp32, m, l) in scratch and a second kernel joins them in the order of the keys, so
// that results repeat bit for bit.
//
//   warps 0-3, 4-7  two streams. N <= 64: tiles of 128 keys go to the two in turn, each with its own maxima, sums and O, joined at the
//                   item's end; 128 rows: both see every tile, each with 64 of the rows.
//   warps 8, 9      MMA issue for the two streams
//   warps 10, 11    TMA producers: keys (and queries), values; a lane per box of up to 32 rows inside a page
#pragma once

#include "kfa_cache.cuh"

namespace kfa {

constexpr int ATT_THREADS = 384;
constexpr int ATT_UNIT = 32;  // keys: what work is counted in
// Registers per thread: 168 at the start (65536 / 384, in eights); with 64 columns the streams, which hold two numbers a column, take what the
// issuing warps do not need. (A CTA owns what it was launched with: budgets beyond that would wait for ever.)
constexpr int ATT_REGS = 168, ATT_REGS_STREAM = 208, ATT_REGS_ISSUE = 88;
static_assert(2 * 128 * ATT_REGS_STREAM + 128 * ATT_REGS_ISSUE <= ATT_THREADS * ATT_REGS, "register budgets exceed the CTA's allocation");

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
  int items;       // per sequence: K / V heads x row tiles
  int whole;       // every item is one CTA's (short caches: nothing is cut)
  int box;         // rows of a page's TMA box
  float c_log2, slack;  // scale * log2 e; how far a maximum may grow before O is rescaled
  float* part_o;   // [slot][NR][128]
  float* part_ml;  // [slot][3][NR]: m, l, largest score
  int4* part_meta; // [CTA]: parts of the item that begins in it and ends in another (0: none), sequence, item
  int* status;
};

// The stretch of work of a CTA, walked item by item; every role walks for itself.
struct Walk {
  int b, item, unit, units, uc, ud, len, count;  // unit: first of the current segment; uc, ud: units of cached and of new keys
  int n;                                         // units of the current segment
  long long left;                                // units (whole: items) left, the current segment's included
  __device__ __forceinline__ static void size(const AttendParams& p, int b, int& len, int& count, int& uc, int& ud) {
    len = cache_length(p.c, b);
    count = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
    uc = count ? (len + ATT_UNIT - 1) / ATT_UNIT : 0;
    ud = count && p.k ? (count + ATT_UNIT - 1) / ATT_UNIT : 0;
  }
  __device__ __forceinline__ void load(const AttendParams& p) {
    size(p, b, len, count, uc, ud);
    units = max(uc + ud, 1);
  }
  __device__ __forceinline__ void cut(const AttendParams& p) {
    n = units - unit;
    if (!p.whole && n > left) n = static_cast<int>(left);
  }
  __device__ __forceinline__ bool next(const AttendParams& p) {  // false: that was the last segment
    left -= p.whole ? 1 : n;
    if (left <= 0) return false;
    unit = 0;
    if (++item == p.items) {
      item = 0;
      ++b;
      load(p);
    }
    cut(p);
    return true;
  }
  __device__ __forceinline__ int tiles() const { return (n + 3) >> 2; }
  __device__ __forceinline__ bool begins() const { return unit == 0; }
  __device__ __forceinline__ bool ends() const { return unit + n == units; }
};

template <int NC, int NR>
struct AttCfg {
  static constexpr bool BY_ROWS = NR == 128;        // the streams share the rows, not the tiles
  static constexpr int N = BY_ROWS ? 64 : NR;       // columns of a stream
  static constexpr int NQ = BY_ROWS ? 1 : 2;        // buffers for queries
  static constexpr int NP = N <= 32 ? 2 : 1;        // buffers for P per stream
  static constexpr int CHUNK = 128 * 64 * 2;        // 128 keys x 64 columns
  static constexpr int STAGE = NC * CHUNK;
  static constexpr int Q_BYTES = NC * NR * 128;
  static constexpr int P_BYTES = 128 * N * 2;
  static constexpr int SMALL = 1024 + 2 * 2 * 4 * N * 4 + 8 * N * 4 + 2 * 2 * 6 * N * 4;  // barriers; maxima; shifts; final sums
  static constexpr int FIXED = 1024 + NQ * Q_BYTES + 2 * NP * P_BYTES + SMALL;
  static constexpr int FIT = (232448 - FIXED) / STAGE;
  // Rings of key tiles and of value tiles, in turn for each stream (BY_ROWS: one of each for both). A stage has one producer and the
  // same consumers every time: who waits for a phase of its barrier has waited for the one before, and a parity means one phase.
  static constexpr int RINGS = BY_ROWS ? 1 : 2;
  static constexpr int DEEP = FIT / RINGS, MOST = BY_ROWS ? 4 : 2;
  static constexpr int DV = DEEP / 2 < MOST ? DEEP / 2 : MOST;
  static constexpr int DK = DEEP - DV < MOST ? DEEP - DV : MOST;
  static_assert(DV >= 1 && DK >= 1, "no room for a tile of keys and one of values");
  static constexpr int NS = RINGS * (DK + DV);
  static_assert(NS <= FIT, "ring too long");
  static constexpr int SMEM = FIXED + NS * STAGE;
  __device__ static __forceinline__ int k_stage(int T) { return BY_ROWS ? T % DK : (T & 1) * DK + (T >> 1) % DK; }
  __device__ static __forceinline__ int v_stage(int T) { return RINGS * DK + (BY_ROWS ? T % DV : (T & 1) * DV + (T >> 1) % DV); }
  __device__ static __forceinline__ int k_turn(int T) { return (BY_ROWS ? T : T >> 1) / DK; }
  __device__ static __forceinline__ int v_turn(int T) { return (BY_ROWS ? T : T >> 1) / DV; }
  static constexpr uint32_t TMEM = N == 64 ? 512 : (N == 32 ? 256 : 128);  // 6 N columns: S 2 x 2, O 2
  // (P and "P V has retired" have a barrier per buffer: a stream may be a buffer ahead of what waits for it.)
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

// What a part with maximum m and sum l counts beside the maximum of all parts: nothing if it saw no key (its O is not defined
// then); a sum that is NaN without any maximum (all its scores were NaN) counts, as NaN.
__device__ __forceinline__ float part_factor(float m, float l, float m_all, float c_log2) {
  if (m == -INFINITY) return l == 0.f ? 0.f : 1.f;
  return ex2((m - m_all) * c_log2);
}

// The heads and tokens of a row tile's rows, and where a row's output lies (bytes), < 0: there is no such row.
struct RowMap {
  int h0, heads, t0;  // first head, heads that exist, first token
  __device__ __forceinline__ RowMap(const AttendParams& p, int item) {
    const int g = static_cast<int>(p.by_row_tiles.div(item)), rt = item - g * p.row_tiles;
    const int tile_t = static_cast<int>(p.by_head_tiles.div(rt)), tile_h = rt - tile_t * p.head_tiles;
    h0 = g * p.group + tile_h * p.gt;
    heads = min(p.gt, p.group - tile_h * p.gt);
    t0 = tile_t * p.tt;
  }
  __device__ __forceinline__ bool row(const AttendParams& p, int r, int& h, int& t) const {
    const int dt = static_cast<int>(p.by_gt.div(r)), dh = r - dt * p.gt;
    h = h0 + dh;
    t = t0 + dt;
    return dt < p.tt && dh < heads && t < p.T;
  }
};

template <int NC, int NR, bool BF16>
__global__ void __launch_bounds__(ATT_THREADS, 1)
kfa_cache_attend_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                        const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmKn,
                        const __grid_constant__ CUtensorMap tmVn, const AttendParams p) {
  using Cfg = AttCfg<NC, NR>;
  constexpr int N = Cfg::N, NS = Cfg::NS, NQ = Cfg::NQ, NP = Cfg::NP;
  constexpr bool BY_ROWS = Cfg::BY_ROWS;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t sKV = base, sQ = sKV + NS * Cfg::STAGE, sP = sQ + NQ * Cfg::Q_BYTES;
  uint8_t* small = smem + NS * Cfg::STAGE + NQ * Cfg::Q_BYTES + 2 * NP * Cfg::P_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(small);
  float* s_max = reinterpret_cast<float*>(small + 1024);  // [stream][tile & 1][warp][N]
  float* s_shift = s_max + 2 * 2 * 4 * N;                 // [warp][N]
  float* s_fin = s_shift + 8 * N;                         // [segment & 1][stream]: l of four warps, m, largest score, each [N]
  constexpr int B_KV = 0, B_KVFREE = NS, B_Q = 2 * NS, B_S = B_Q + NQ, B_P = B_S + 4, B_PV = B_P + 4, B_OFREE = B_PV + 4,
                B_DRAIN = B_OFREE + 2, N_BARS = B_DRAIN + 2;
  static_assert(N_BARS * 8 + 256 <= 1024, "barrier block");
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(bars + N_BARS);
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
  volatile int* s_bad = s_abort + 1;  // the cache says something that is not so, or an earlier kernel failed
  volatile int* s_odd = s_abort + 2;  // [stream] 1 + the last segment in which it met new values that are not finite
  int* s_b = reinterpret_cast<int*>(s_tmem + 5);                        // first sequence
  long long* s_work = reinterpret_cast<long long*>(bars + N_BARS + 4);  // first unit in it; from [2]: warps' sums
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](int i) { return bar0 + 8u * i; };

  const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31;

  // ---- setup; which work is this CTA's ----
  if (warp == 10) {
    for (int i = lane; i < N_BARS; i += 32) {
      int count = 1;
      if (i >= B_KVFREE && i < B_Q) count = BY_ROWS ? 2 : 1;
      if (i >= B_P && i < B_PV) count = 128;
      if (i >= B_OFREE && i < B_DRAIN) count = BY_ROWS ? 128 : 256;
      mbar_init(bar(i), count);
    }
    if (lane == 0) {
      *s_abort = 0;
      *s_bad = load_status(p.status) != 0;
      s_odd[0] = s_odd[1] = 0;
    }
    fence_mbar_init();
    fence_async_smem();
  }
  if (warp == 8) {
    tmem_alloc(smem_u32(s_tmem), Cfg::TMEM);
    tmem_relinquish();
  }
  Walk first;
  long long chunk = 0, u1 = 0;  // units per CTA, the end of this one's
  if (p.whole) {
    const long long all = static_cast<long long>(p.c.batch) * p.items;
    const long long i0 = all * blockIdx.x / gridDim.x, i1 = all * (blockIdx.x + 1) / gridDim.x;
    first.b = static_cast<int>(p.by_items.div(static_cast<uint32_t>(i0)));
    first.item = static_cast<int>(i0 - static_cast<long long>(first.b) * p.items);
    first.left = i1 - i0;
    first.unit = 0;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  } else {
    // units of the whole batch, 384 sequences at a time; then the sequence in which this CTA's stretch begins
    auto units_of = [&](int b) {
      if (b >= p.c.batch) return 0ll;
      int len, count, uc, ud;
      Walk::size(p, b, len, count, uc, ud);
      return static_cast<long long>(max(uc + ud, 1)) * p.items;
    };
    auto warp_scan = [&](long long x) {
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, x, off);
        if (lane >= off) x += up;
      }
      return x;
    };
    long long total = 0;
    const long long mine0 = units_of(tid), scan0 = warp_scan(mine0);
    for (int b0 = 0; b0 < p.c.batch; b0 += ATT_THREADS) {
      const long long s = b0 == 0 ? scan0 : warp_scan(units_of(b0 + tid));
      if (b0 > 0) __syncthreads();
      if (lane == 31) s_work[2 + warp] = s;
      __syncthreads();
      for (int w = 0; w < ATT_THREADS / 32; ++w) total += s_work[2 + w];
    }
    chunk = max((total + gridDim.x - 1) / gridDim.x, 4ll);
    const long long u0 = chunk * blockIdx.x;
    u1 = min(u0 + chunk, total);
    long long before = 0;
    for (int b0 = 0; b0 < p.c.batch; b0 += ATT_THREADS) {
      const long long own = b0 == 0 ? mine0 : units_of(b0 + tid);
      long long end = b0 == 0 ? scan0 : warp_scan(own);
      if (p.c.batch > ATT_THREADS) {
        __syncthreads();
        if (lane == 31) s_work[2 + warp] = end;
        __syncthreads();
      }
      for (int w = 0; w < ATT_THREADS / 32; ++w) {
        if (w < warp) end += s_work[2 + w];
      }
      if (u0 >= before + end - own && u0 < before + end) {
        *s_b = b0 + tid;
        s_work[0] = u0 - (before + end - own);
      }
      for (int w = 0; w < ATT_THREADS / 32; ++w) before += s_work[2 + w];
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    first.left = max(u1 - u0, 0ll);
    first.b = first.item = first.unit = 0;
    if (first.left > 0) {
      first.b = *s_b;
      int len, count, uc, ud;
      Walk::size(p, first.b, len, count, uc, ud);
      const int units = max(uc + ud, 1);
      first.item = static_cast<int>(s_work[0] / units);
      first.unit = static_cast<int>(s_work[0] - static_cast<long long>(first.item) * units);
    }
  }
  const bool work = first.left > 0;
  if (work) {
    first.load(p);
    first.cut(p);
  }
  const uint32_t tmem = *s_tmem;
  const Ctl ctl{s_abort};
  const uint32_t tmS = tmem, tmO = tmem + 4 * N;
  int kv_issued = 0, q_issued = 0;  // producers: ring slots filled, segments' queries

  if (!work) {
    if (tid == 0 && !p.whole) p.part_meta[blockIdx.x] = make_int4(0, 0, 0, 0);
  } else if (warp >= 10) {
    // =========================== TMA producers ===========================
    if constexpr (N == 64) reg_budget<ATT_REGS_ISSUE, ATT_REGS>();
    const bool values = warp == 11;
    const CUtensorMap *map = values ? &tmV : &tmK, *map_new = values ? &tmVn : &tmKn;
    Walk w = first;
    const int per_unit = ATT_UNIT / p.box, boxes = 4 * per_unit;
    bool ok = true, more = true;
    int T = 0, s = 0;  // tiles and segments so far
    while (more && ok) {
      const RowMap rows(p, w.item);
      const int g = static_cast<int>(p.by_row_tiles.div(w.item));
      if (lane == 0 && w.unit == 0 && !length_ok(p.c, w.b)) *s_bad = 1;
      if (!values) {
        if (s >= NQ) {
          ok = mbar_wait_warp(bar(B_OFREE), ((s - NQ) & 1), ctl, 70) && mbar_wait_warp(bar(B_OFREE + 1), ((s - NQ) & 1), ctl, 71);
          if (!ok) break;
        }
        if (lane == 0) {
          mbar_expect_tx(bar(B_Q + s % NQ), NC * p.gt * p.tt * 128);
          for (int ch = 0; ch < NC; ++ch)
            tma_load_4d(sQ + (s % NQ) * Cfg::Q_BYTES + ch * NR * 128, &tmQ, bar(B_Q + s % NQ), ch * 64, rows.h0, rows.t0, w.b);
        }
        q_issued = s + 1;
      }
      const int tiles = w.tiles();
      for (int t = 0; t < tiles && ok; ++t, ++T) {
        // this lane's box
        const int in_unit = (lane % per_unit) * p.box, unit = w.unit + 4 * t + lane / per_unit;
        const bool mine = lane < boxes && unit < w.unit + w.n;
        const int row = (lane / per_unit) * ATT_UNIT + in_unit;
        int c1 = 0, c3 = w.b, kind = 0;  // 1: cached rows, 2: new ones
        if (mine && unit < w.uc) {
          const int pos = unit * ATT_UNIT + in_unit;
          if (pos < w.len) {
            if (cache_place(p.c, w.b, pos, c3, c1)) kind = 1;
            else *s_bad = 1;
          }
        } else if (mine && in_unit == 0) {
          c1 = (unit - w.uc) * ATT_UNIT;
          if (c1 < w.count && w.ud > 0) kind = 2;
        }
        const unsigned cached = __ballot_sync(0xffffffffu, kind == 1), fresh = __ballot_sync(0xffffffffu, kind == 2);
        const int stage = values ? Cfg::v_stage(T) : Cfg::k_stage(T), turn = values ? Cfg::v_turn(T) : Cfg::k_turn(T);
        if (turn > 0) {
          ok = mbar_wait_warp(bar(B_KVFREE + stage), (turn - 1) & 1, ctl, 72);
          if (!ok) break;
        }
        if (lane == 0) mbar_expect_tx(bar(B_KV + stage), NC * 128 * (__popc(cached) * p.box + __popc(fresh) * ATT_UNIT));
        __syncwarp();
        if (kind != 0) {
          const uint32_t dst = sKV + stage * Cfg::STAGE + row * 128;
          for (int ch = 0; ch < NC; ++ch)
            tma_load_4d(dst + ch * Cfg::CHUNK, kind == 1 ? map : map_new, bar(B_KV + stage), ch * 64, c1, g, c3);
        }
        kv_issued = T + 1;
      }
      if (ok) {
        ++s;
        more = w.next(p);
      }
    }
  } else if (warp >= 8) {
    // =========================== MMA issue ===========================
    if constexpr (N == 64) reg_budget<ATT_REGS_ISSUE, ATT_REGS>();
    const int st = warp - 8;
    const bool lead = elect_one();
    constexpr uint32_t IDESC_S = make_idesc(BF16, false, 128, N), IDESC_O = make_idesc(BF16, true, 128, N) | (1u << 15);
    constexpr uint32_t HI_P = sdesc_hi_for(N);
    const int k_steps = (p.c.cols + 15) / 16;
    bool ok = true;
    struct Tile {
      int T, s;
      bool opens;  // the stream's first tile of the segment
    };
    Walk w = first;
    int at = 0, T_next = 0, s_next = 0;  // inside the segment; over all
    bool more = true, opens = true;
    auto take = [&](Tile& t) {  // the stream's next tile
      while (more) {
        while (at < w.tiles()) {
          ++at;
          const int T = T_next++;
          if (BY_ROWS || (T & 1) == st) {
            t = {T, s_next, opens};
            opens = false;
            return true;
          }
        }
        at = 0;
        ++s_next;
        opens = true;
        more = w.next(p);
      }
      return false;
    };
    auto issue_S = [&](const Tile& t, int c) {
      const int stage = Cfg::k_stage(t.T);
      ok = mbar_wait_warp(bar(B_KV + stage), Cfg::k_turn(t.T) & 1, ctl, 73);
      if (ok && t.opens) ok = mbar_wait_warp(bar(B_Q + t.s % NQ), (t.s / NQ) & 1, ctl, 74);
      if (!ok) return;
      tc_fence_after();
      const uint32_t k_lo = sdesc_lo(sKV + stage * Cfg::STAGE, 16);
      const uint32_t q_lo = sdesc_lo(sQ + (t.s % NQ) * Cfg::Q_BYTES + (BY_ROWS ? st * 64 * 128 : 0), 16);
      for (int kk = 0; kk < k_steps; ++kk)
        umma_ss_lead2(lead, tmS + (2 * st + (c & 1)) * N, k_lo + (((kk >> 2) * Cfg::CHUNK + (kk & 3) * 32) >> 4), SDESC_HI,
                      q_lo + (((kk >> 2) * (NR * 128) + (kk & 3) * 32) >> 4), SDESC_HI, IDESC_S, kk > 0 ? 1u : 0u);
      umma_commit_lead(lead, bar(B_S + 2 * st + (c & 1)));
      umma_commit_lead(lead, bar(B_KVFREE + stage));
    };
    auto issue_PV = [&](const Tile& t, int c) {
      const int stage = Cfg::v_stage(t.T);
      ok = mbar_wait_warp(bar(B_KV + stage), Cfg::v_turn(t.T) & 1, ctl, 75) && mbar_wait_warp(bar(B_P + 2 * st + c % NP), (c / NP) & 1, ctl, 76);
      if (ok && t.opens && t.s > 0) ok = mbar_wait_warp(bar(B_OFREE + st), (t.s - 1) & 1, ctl, 77);
      if (!ok) return;
      tc_fence_after();
      const uint32_t v_lo = sdesc_lo(sKV + stage * Cfg::STAGE, NC == 2 ? Cfg::CHUNK : 0);
      const uint32_t p_lo = sdesc_lo(sP + (st * NP + c % NP) * Cfg::P_BYTES, 16);
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)
        umma_ss_lead2(lead, tmO + st * N, v_lo + ((kk * 16 * 128) >> 4), SDESC_HI, p_lo + ((kk * 16 * 2 * N) >> 4), HI_P, IDESC_O,
                      (!t.opens || kk > 0) ? 1u : 0u);
      umma_commit_lead(lead, bar(B_PV + 2 * st + c % NP));
      umma_commit_lead(lead, bar(B_KVFREE + stage));
    };
    Tile now, then;
    int c = 0;
    bool have = take(now);
    if (have) issue_S(now, 0);
    while (have && ok) {
      const bool again = take(then);
      // (A segment's queries are only loaded once the segment NQ before it is finished, for which this tile's values may be needed.)
      const bool ahead = again && then.s - now.s < NQ;
      if (ahead) issue_S(then, c + 1);
      if (ok) issue_PV(now, c);
      if (ok && again && !ahead) issue_S(then, c + 1);
      now = then;
      have = again;
      ++c;
    }
    umma_commit_lead(lead, bar(B_DRAIN + st));  // what was issued has retired before tensor memory is freed
    mbar_drain(bar(B_DRAIN + st), 0);
  } else {
    // =========================== softmax, output ===========================
    // (After a wait that ran out the role goes on without waiting: the warps of a stream meet at barriers.)
    if constexpr (N == 64) reg_budget<ATT_REGS_STREAM, ATT_REGS>();
    const int st = warp >> 2, wl = warp & 3, key = tid & 127;
    const uint32_t lane_base = static_cast<uint32_t>(wl * 32) << 16;
    constexpr int PER = N / 32 > 0 ? N / 32 : 1;  // columns whose maximum a lane keeps: lane, lane + 32
    float* shift = s_shift + warp * N;
    const float c_log2 = p.c_log2;
    Walk w = first;
    bool more = true, ok = true;
    int c = 0, T0 = 0, s = 0;  // the stream's tiles; tiles and segments before
    while (more) {
      const RowMap rows(p, w.item);
      float l[N], m_ref[PER], m_top[PER];
#pragma unroll
      for (int i = 0; i < N; ++i) l[i] = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) m_ref[i] = m_top[i] = -INFINITY;
      bool opens = true;
      const int tiles = w.tiles();
      for (int t = 0; t < tiles; ++t) {
        const int T = T0 + t;
        if (!BY_ROWS && (T & 1) != st) continue;
        const int ub = w.unit + 4 * t;
        const bool full = 4 * t + 4 <= w.n && (ub + 4) * ATT_UNIT <= w.len && ub + 4 <= w.uc;
        if (ok) ok = mbar_wait_warp(bar(B_S + 2 * st + (c & 1)), (c >> 1) & 1, ctl, 78);
        tc_fence_after();
        float x[N];
        tmem_ld_cols<N>(tmS + lane_base + (2 * st + (c & 1)) * N, x);
        tmem_wait_ld();
        int fresh = -1;  // the new token that this key is
        bool valid = true;
        if (!full) {
          const int unit = ub + (key >> 5);
          if (unit >= w.unit + w.n) valid = false;
          else if (unit < w.uc) valid = unit * ATT_UNIT + (key & 31) < w.len;
          else {
            fresh = (unit - w.uc) * ATT_UNIT + (key & 31);
            valid = w.ud > 0 && fresh < w.count;
            if (!valid) fresh = -1;
          }
          const uint8_t* tree = p.tree ? p.tree + w.b * p.tree_sb + static_cast<long long>(max(fresh, 0)) * p.tree_sj : nullptr;
          const int r0 = BY_ROWS ? st * 64 : 0;
          bool sees = true;
          int t_last = -1;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            if (fresh >= 0) {
              const int row_t = rows.t0 + static_cast<int>(p.by_gt.div(r0 + i));
              if (row_t != t_last) {
                t_last = row_t;
                sees = row_t < w.count && (tree ? tree[row_t * p.tree_st] != 0 : fresh <= row_t);
              }
            }
            if (!valid || !sees) x[i] = -INFINITY;
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
          if (lane + 32 * i < N) shift[col] = m_ref[i] == -INFINITY ? 0.f : m_ref[i];
        }
        grew = __any_sync(0xffffffffu, grew);  // the same in all warps of the stream
        __syncwarp();
        if (grew && !opens) {
          // sums and O of the earlier tiles, to the new maxima
          if (ok) ok = mbar_wait_warp(bar(B_PV + 2 * st + (c - 1) % NP), ((c - 1) / NP) & 1, ctl, 79);
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
        if (c >= NP && ok) ok = mbar_wait_warp(bar(B_PV + 2 * st + c % NP), (c / NP - 1) & 1, ctl, 80);  // its buffer has been read
        const uint32_t sp = sP + (st * NP + c % NP) * Cfg::P_BYTES;
#pragma unroll
        for (int i = 0; i < N; i += 8) {
          const float4 a = *reinterpret_cast<const float4*>(shift + i), b = *reinterpret_cast<const float4*>(shift + i + 4);
          const float mm[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
          float e[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            e[j] = ex2((x[i + j] - mm[j]) * c_log2);
            l[i + j] += e[j];
          }
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(sp + p_piece<N>(key, i / 8)), "r"(pack16<BF16>(e[0], e[1])),
                       "r"(pack16<BF16>(e[2], e[3])), "r"(pack16<BF16>(e[4], e[5])), "r"(pack16<BF16>(e[6], e[7]))
                       : "memory");
        }
        if (!full) {
          // Values behind the end may be anything, and 0 * NaN is no 0: their rows become zeros. So do a new token's values that
          // are not finite, which would otherwise reach rows that do not see it; the epilogue hands them to those that do.
          // (The tile before has to be done with: until then the barrier of this one's stage may be a turn behind.)
          const int stage = Cfg::v_stage(T);
          if (c > 0 && ok) ok = mbar_wait_warp(bar(B_PV + 2 * st + (c - 1) % NP), ((c - 1) / NP) & 1, ctl, 81);
          if (ok) ok = mbar_wait_warp(bar(B_KV + stage), Cfg::v_turn(T) & 1, ctl, 83);
          const uint32_t row = sKV + stage * Cfg::STAGE + key * 128;
          if (!valid) {
#pragma unroll
            for (int i = 0; i < NC * 8; ++i)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(row + (i >> 3) * Cfg::CHUNK + (i & 7) * 16), "r"(0) : "memory");
          } else if (fresh >= 0) {
            const uint8_t* g_row = p.v + w.b * p.v_sb + static_cast<long long>(p.by_row_tiles.div(w.item)) * p.v_sh + fresh * p.v_ss;
            for (int i = 0; i < p.c.cols / 8; ++i) {
              const uint4 q4 = *reinterpret_cast<const uint4*>(g_row + 16 * i);
              uint32_t q[4] = {q4.x, q4.y, q4.z, q4.w};
              bool odd = false;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                constexpr uint32_t E = BF16 ? 0x7f80u : 0x7c00u;  // all exponent bits: infinity or NaN
                if ((q[j] & E) == E) q[j] &= 0xffff0000u, odd = true;
                if ((q[j] >> 16 & E) == E) q[j] &= 0xffffu, odd = true;
              }
              if (odd) {
                s_odd[st] = s + 1;
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row + (i >> 3) * Cfg::CHUNK + (((i & 7) ^ (key & 7)) << 4)),
                             "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3])
                             : "memory");
              }
            }
          }
        }
        fence_async_smem();
        tc_fence_before();
        mbar_arrive(bar(B_P + 2 * st + c % NP));
        opens = false;
        ++c;
      }
      T0 += tiles;
      // ---- the segment's end ----
      if (!opens && ok) ok = mbar_wait_warp(bar(B_PV + 2 * st + (c - 1) % NP), ((c - 1) / NP) & 1, ctl, 82);
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
      tc_fence_before();
      if constexpr (BY_ROWS) {
        if (st == 0) named_sync<1, 128>();
        else named_sync<2, 128>();
      } else {
        named_sync<3, 256>();
      }
      tc_fence_after();
      const bool bad = *s_bad != 0;
      const bool whole = w.begins() && w.ends();
      const long long slot = 2ll * blockIdx.x + (w.begins() ? 1 : 0);
      // new tokens of the segment, where some of their values were left out (a stream may be one segment ahead: >=)
      const bool odd = s_odd[st] >= s + 1 || (!BY_ROWS && s_odd[1 - st] >= s + 1);
      const int j0 = max(w.unit - w.uc, 0) * ATT_UNIT, j1 = odd ? min((w.unit + w.n - w.uc) * ATT_UNIT, w.count) : 0;
      const int d = wl * 32 + lane;
      constexpr int W = BY_ROWS ? 32 : N / 2;  // columns a thread writes at a time
      for (int part = 0; part < (BY_ROWS ? 2 : 1); ++part) {
        const int c0 = BY_ROWS ? 32 * part : st * W;  // in the stream's columns
        const int r0 = BY_ROWS ? 64 * st + c0 : c0;   // in the tile's rows
        // lane i (i < W): column i's factors and statistics
        const int col = c0 + (lane & (W - 1));
        const float* f0 = s_fin + ((s & 1) * 2 + (BY_ROWS ? st : 0)) * 6 * N + col;
        float l0 = f0[0] + f0[N] + f0[2 * N] + f0[3 * N], m0 = f0[4 * N], top0 = f0[5 * N];
        float a0 = 1.f, a1 = 0.f;
        if constexpr (!BY_ROWS) {
          const float* f1 = f0 + 6 * N;
          const float l1 = f1[0] + f1[N] + f1[2 * N] + f1[3 * N], m1 = f1[4 * N];
          const float mm = fmaxf(m0, m1);
          a0 = part_factor(m0, l0, mm, c_log2);
          a1 = part_factor(m1, l1, mm, c_log2);
          l0 = l0 * a0 + l1 * a1;
          m0 = mm;
          top0 = fmaxf(top0, f1[5 * N]);
        } else if (m0 == -INFINITY) {
          a0 = part_factor(m0, l0, m0, c_log2);
        }
        int h, tk;
        const bool exists = rows.row(p, r0 + (lane & (W - 1)), h, tk);
        const bool counts = exists && tk < w.count;
        long long off = exists ? w.b * p.o_sb + h * p.o_sh + tk * p.o_ss : -1;
        const bool some = counts && l0 != 0.f;
        const float nan = __int_as_float(0x7fc00000);
        if (whole) {
          const float inv = some ? 1.f / l0 : 0.f;
          if (p.stats && wl == 0 && exists && lane < W) {
            float* at = p.stats + (static_cast<long long>(w.b) * p.H + h) * 2 * p.T + tk;
            at[0] = bad ? nan : (some ? top0 : INFINITY);
            at[p.T] = bad ? nan : (some ? log2f(l0) + (m0 - top0) * c_log2 : 0.f);
          }
          a0 = some ? a0 * inv : 0.f;
          a1 = some ? a1 * inv : 0.f;
        } else if (wl == 0 && lane < W) {
          float* at = p.part_ml + slot * 3 * NR + r0 + lane;
          at[0] = m0;
          at[NR] = l0;
          at[2 * NR] = top0;
        }
        float o0[W], o1[W];
        tmem_ld_cols<W>(tmO + lane_base + (BY_ROWS ? st * N : 0) + c0, o0);
        if constexpr (!BY_ROWS) tmem_ld_cols<W>(tmO + lane_base + N + c0, o1);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float x0 = __shfl_sync(0xffffffffu, a0, i), x1 = __shfl_sync(0xffffffffu, a1, i);
          float y = x0 == 0.f ? 0.f : o0[i] * x0;  // (a stream without tiles has left nothing there)
          if constexpr (!BY_ROWS) y += x1 == 0.f ? 0.f : o1[i] * x1;
          o0[i] = y;
        }
        if (d < p.c.cols) {
          for (int j = j0; j < j1; ++j) {
            const float y = load16<BF16>(p.v + w.b * p.v_sb + static_cast<long long>(p.by_row_tiles.div(w.item)) * p.v_sh + j * p.v_ss + 2 * d);
            if (fabsf(y) < INFINITY) continue;
#pragma unroll
            for (int i = 0; i < W; ++i) {
              const int row_t = rows.t0 + static_cast<int>(p.by_gt.div(r0 + i));
              if (row_t < w.count && (p.tree ? p.tree[w.b * p.tree_sb + row_t * p.tree_st + j * p.tree_sj] != 0 : j <= row_t)) o0[i] += y;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const long long at = __shfl_sync(0xffffffffu, off, i);
          if (whole) {
            if (at >= 0 && d < p.c.cols) {
              const uint32_t y = pack16<BF16>(bad ? nan : o0[i], 0.f);
              *reinterpret_cast<uint16_t*>(p.o + at + 2 * d) = static_cast<uint16_t>(y);
            }
          } else {
            p.part_o[(slot * NR + r0 + i) * 128 + d] = o0[i];
          }
        }
      }
      tc_fence_before();
      mbar_arrive(bar(B_OFREE + st));
      if constexpr (!BY_ROWS) mbar_arrive(bar(B_OFREE + 1 - st));
      ++s;
      more = w.next(p);
    }
    if (tid == 0 && !p.whole) {  // only the last item can begin here and end in another CTA
      int4 meta = make_int4(0, 0, 0, 0);
      if (w.begins() && !w.ends()) meta = make_int4(static_cast<int>((u1 - w.n + w.units - 1) / chunk - blockIdx.x) + 1, w.b, w.item, 0);
      p.part_meta[blockIdx.x] = meta;
    }
  }

  // ---- teardown (every thread gets here, also after an abort) ----
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *s_bad) report(p.status, DEV_BAD_CACHE);
  if (*s_abort) {
    if (tid == 0) report_abort(s_abort, p.status);
    if (warp >= 10 && lane == 0) {  // the copies it has started land before the CTA leaves its shared memory
      for (int s = max(q_issued - NQ, 0); s < q_issued; ++s) mbar_drain(bar(B_Q + s % NQ), (s / NQ) & 1);
      for (int T = max(kv_issued - Cfg::RINGS * (warp == 10 ? Cfg::DK : Cfg::DV), 0); T < kv_issued; ++T)
        mbar_drain(bar(B_KV + (warp == 10 ? Cfg::k_stage(T) : Cfg::v_stage(T))), (warp == 10 ? Cfg::k_turn(T) : Cfg::v_turn(T)) & 1);
    }
    Walk w = first;
    bool more = work;
    while (more) {  // the rows of what it had whole read as NaN; what was cut, the joining kernel sees to
      if (w.begins() && w.ends()) {
        const RowMap rows(p, w.item);
        for (int i = tid; i < NR * (p.c.cols / 8); i += ATT_THREADS) {
          int h, t;
          if (!rows.row(p, i / (p.c.cols / 8), h, t)) continue;
          const uint4 nan8 = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
          *reinterpret_cast<uint4*>(p.o + w.b * p.o_sb + h * p.o_sh + t * p.o_ss + 16 * (i % (p.c.cols / 8))) = nan8;
          if (p.stats && i % (p.c.cols / 8) == 0) {
            float* at = p.stats + (static_cast<long long>(w.b) * p.H + h) * 2 * p.T + t;
            at[0] = at[p.T] = __int_as_float(0x7fc00000);
          }
        }
      }
      more = w.next(p);
    }
  }
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::TMEM);
  }
}

// Joins the parts of the items that were cut: CTA x has the item that begins in CTA x of the kernel above, a warp a row, a lane four
// columns. Starts while that kernel ends and waits for it.
template <int NR, bool BF16>
__global__ void __launch_bounds__(256) kfa_cache_join_kernel(const AttendParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 meta = p.part_meta[blockIdx.x];
  if (meta.x == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = blockIdx.y * 8 + warp;
  const RowMap rows(p, meta.z);
  int h, t;
  if (!rows.row(p, r, h, t)) return;
  const bool bad = *reinterpret_cast<const volatile int*>(p.status) != 0;
  const int count = p.counts ? min(max(p.counts[meta.y], 0), p.T) : p.T;
  // part i: the first in slot 1 of its CTA, the others in slot 0 of theirs
  auto slot = [&](int i) { return 2ll * (blockIdx.x + i) + (i == 0 ? 1 : 0); };
  float m = -INFINITY, top = -INFINITY;
  for (int i = lane; i < meta.x; i += 32) {
    const float* ml = p.part_ml + slot(i) * 3 * NR + r;
    m = fmaxf(m, ml[0]);
    top = fmaxf(top, ml[2 * NR]);
  }
  m = warp_max(m);
  top = warp_max(top);
  float l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < meta.x; i0 += 32) {
    float a = 0.f, li = 0.f;
    if (i0 + lane < meta.x) {
      const float* ml = p.part_ml + slot(i0 + lane) * 3 * NR + r;
      a = part_factor(ml[0], ml[NR], m, p.c_log2);
      li = a * ml[NR];
    }
    const int n = min(32, meta.x - i0);
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float ai = __shfl_sync(0xffffffffu, a, i);
      l += __shfl_sync(0xffffffffu, li, i);
      const float4 x = *reinterpret_cast<const float4*>(p.part_o + (slot(i0 + i) * NR + r) * 128 + 4 * lane);
      if (ai != 0.f) {
        o.x += ai * x.x;
        o.y += ai * x.y;
        o.z += ai * x.z;
        o.w += ai * x.w;
      }
    }
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

}  // namespace kfa
