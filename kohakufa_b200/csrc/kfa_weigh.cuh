// How much attention the newest tokens gave to every cached position: w[p] = sum over rows of exp2((q k_p - m) c - log2 l), the rows' m
// and log2 l from the attention call. The keys are the rows of the matrix instructions, as in kfa_cache_attend_kernel: a thread holds a key
// and sums over the columns, the query rows, so that nothing crosses threads.
//
// Up to 64 rows (kfa_cache_weigh_kernel, a decoding step): bound by the keys, read once; work cut by keys as in the attention, every
// position is one CTA's. (With small pages by the warp that issues their copies: 16 sequences of 300 to 4096 with 5 tokens, 8 heads of 128, take 30.7, 21.7, 17.6
// us in a graph with pages of 8, 16, 32 positions, 15.8 without pages; the bytes 12.9.) More rows (kfa_cache_weigh_rows_kernel, a prompt): bound by the exponentials; an item is a tile of 128 keys and a block of
// 128 tokens, whose rows stream past the keys in tiles of 128. Items are shared out equally; a key tile whose items fall to several CTAs is
// joined from their sums in order.
#pragma once

#include "kfa_attend.cuh"

namespace kfa {

struct WeighParams {
  RowsView r;
  const uint8_t* q;
  long long q_sb, q_sh, q_ss;  // bytes
  const float* stats;          // [B, H, 2, T]
  float* w;
  long long w_sb, w_sh;
  int room, add;
  FastDiv by_piece;            // 16-byte pieces of a row
  // many rows: tokens and heads of a row tile; sums of the key tiles that a CTA has a part of [slot][128]; [CTA]: parts of the key tile that
  // begins in it and ends in another (0: none), sequence, K / V head, tile
  int tile_t, tile_h, head_tiles;
  FastDiv by_tile_h, by_tile_t;
  float* part;
  int4* part_meta;
  // rows picked by an index, gathered
  uint8_t* q_to;
  float* stats_to;
};

// m and log2 l of row r of a (sequence, K / V head): token i of those that count, head h. What is not there: +inf, which gives 0.
__device__ __forceinline__ float2 row_stats(const AttendParams& a, const WeighParams& p, int b, int h, int t) {
  const float* at = p.stats + (static_cast<long long>(b) * a.H + h) * 2 * p.r.T + t;
  return make_float2(at[0], at[p.r.T]);
}

// How many of a tile's rows, `heads` a token, stand before a key that lies `ahead` positions behind the tile's first token: those do not see it.
// (Most keys lie far before the token: the product of that distance would pass 32 bits in a long cache. Behind the token are less than 256, what is left of its tile and of the rows' tile.)
__device__ __forceinline__ int rows_before(int ahead, int heads) { return max(ahead, 0) * heads; }

// The weights of a key, summed: N scores against N rows, whose -m and -log2 l stand one after the other (two at a time in the packed
// instructions). Rows that are not there (-m = -inf; their scores may be anything) and those that do not see the key (below r_min) count nothing.
template <int N>
__device__ __forceinline__ float weigh_scores(const float* x, const float* neg_m, const float* neg_l, float c_log2, int r_min) {
  const float2 c2 = make_float2(c_log2, c_log2);
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const float4 m = *reinterpret_cast<const float4*>(neg_m + i), l = *reinterpret_cast<const float4*>(neg_l + i);
    float2 e0 = __ffma2_rn(__fadd2_rn(make_float2(x[i], x[i + 1]), make_float2(m.x, m.y)), c2, make_float2(l.x, l.y));
    float2 e1 = __ffma2_rn(__fadd2_rn(make_float2(x[i + 2], x[i + 3]), make_float2(m.z, m.w)), c2, make_float2(l.z, l.w));
    e0 = make_float2(ex2(e0.x), ex2(e0.y));
    e1 = make_float2(ex2(e1.x), ex2(e1.y));
    if (m.x == -INFINITY || i < r_min) e0.x = 0.f;
    if (m.y == -INFINITY || i + 1 < r_min) e0.y = 0.f;
    if (m.z == -INFINITY || i + 2 < r_min) e1.x = 0.f;
    if (m.w == -INFINITY || i + 3 < r_min) e1.y = 0.f;
    sum[0] = __fadd2_rn(sum[0], e0);
    sum[1] = __fadd2_rn(sum[1], e1);
  }
  return (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
}

// The same for rows that are all there and see the key, and whose two numbers may be one, -(m c + log2 l): half the loads, which is what bounds
// a prompt (a float for every lane of a warp takes a cycle of the shared memory, whether lanes differ or not).
template <int N>
__device__ __forceinline__ float weigh_scores_one(const float* x, const float* neg, float c_log2) {
  const float2 c2 = make_float2(c_log2, c_log2);
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const float4 t = *reinterpret_cast<const float4*>(neg + i);
    const float2 e0 = __ffma2_rn(make_float2(x[i], x[i + 1]), c2, make_float2(t.x, t.y));
    const float2 e1 = __ffma2_rn(make_float2(x[i + 2], x[i + 3]), c2, make_float2(t.z, t.w));
    sum[0] = __fadd2_rn(sum[0], make_float2(ex2(e0.x), ex2(e0.y)));
    sum[1] = __fadd2_rn(sum[1], make_float2(ex2(e1.x), ex2(e1.y)));
  }
  return (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
}

// ---- up to 64 rows -------------------------------------------------------------------------------------------------------------
template <int NC, int N>
struct WeighCfg {
  static constexpr int CHUNK = 128 * 64 * 2, STAGE = NC * CHUNK, Q_CHUNK = N * 128, Q_BYTES = NC * Q_CHUNK;
  static constexpr int DK = 3;  // key tiles per stream
  static constexpr int NS = 2 * DK;
  static constexpr int SMALL = 1024 + 2 * N * 8;
  static constexpr int SMEM = 1024 + NS * STAGE + 2 * Q_BYTES + SMALL;
  static constexpr int TMEM = N == 64 ? 256 : (N == 32 ? 128 : 64);  // S 2 x 2
  static constexpr int B_K = 0, B_KFREE = NS, B_Q = 2 * NS, B_QFREE = B_Q + 2, B_S = B_QFREE + 2, B_SFREE = B_S + 4, B_DRAIN = B_SFREE + 4,
                       N_BARS = B_DRAIN + 2;
  static_assert(SMEM <= 232448 && N_BARS * 8 + 256 <= 1024, "shared memory");
};

template <int NC, int N, bool BF16>
__global__ void __launch_bounds__(ATT_THREADS, 1)
kfa_cache_weigh_kernel(const __grid_constant__ CUtensorMap tmK, const AttendParams a, const WeighParams p) {
  using R = WeighCfg<NC, N>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t sK = base, sQ = sK + R::NS * R::STAGE;
  uint8_t* small = smem + R::NS * R::STAGE + 2 * R::Q_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(small);
  float* s_rows = reinterpret_cast<float*>(small + 1024);  // [segment & 1][-m, -log2 l][N]
  const AttCtl ac(bars + R::N_BARS);
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](int i) { return bar0 + 8u * i; };
  const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31;
  if (tid == 32 * 11) asm volatile("prefetch.tensormap [%0];" ::"l"(&tmK) : "memory");
  if (warp == 10) {
    for (int i = lane; i < R::N_BARS; i += 32) {
      int count = 1;
      if (i >= R::B_Q && i < R::B_QFREE) count = 32;
      if (i >= R::B_QFREE && i < R::B_S) count = 256;
      if (i >= R::B_SFREE && i < R::B_DRAIN) count = 128;
      mbar_init(bar(i), count);
    }
    if (lane == 0) *ac.abort = 0;
    fence_mbar_init();
    fence_async_smem();
  }
  if (warp == 8) {
    tmem_alloc(smem_u32(ac.tmem), R::TMEM);
    tmem_relinquish();
  }
  wait_for_previous();
  if (warp == 10 && lane == 0) *ac.bad = load_status(a.status) != 0;
  tc_fence_before();
  Walk first;
  int chunk, end;
  const bool work = my_work(a, ac.ints, first, chunk, end);
  let_next_begin();
  tc_fence_after();
  const uint32_t tmem = *ac.tmem;
  const Ctl ctl{ac.abort};
  int issued = 0;
  auto stage_of = [](int T) { return (T & 1) * R::DK + (T >> 1) % R::DK; };
  auto turn_of = [](int T) { return (T >> 1) / R::DK; };

  if (!work) {
  } else if (warp == 10) {
    // =========================== TMA producer: keys ===========================
    Walk w = first;
    const int per_unit = ATT_UNIT / a.box, boxes = 4 * per_unit;
    bool ok = true, more = true;
    int T = 0;
    while (more && ok) {
      const int tiles = w.tiles();
      for (int t = 0; t < tiles && ok; ++t, ++T) {
        const int unit = w.unit + 4 * t + lane / per_unit, row = (lane / per_unit) * ATT_UNIT + (lane % per_unit) * a.box;
        const int pos = (w.unit + 4 * t) * ATT_UNIT + row;
        int page = 0, slot = 0;
        bool mine = lane < boxes && unit < w.unit + w.n && pos < w.len;
        if (mine && !cache_place(a.c, w.b, pos, page, slot)) {
          mine = false;
          *ac.bad = 1;
        }
        const unsigned there = __ballot_sync(0xffffffffu, mine);
        const int stage = stage_of(T);
        if (turn_of(T) > 0) {
          ok = wait_warp(bar(R::B_KFREE + stage), (turn_of(T) - 1) & 1, ctl, 84);
          if (!ok) break;
        }
        if (lane == 0) mbar_expect_tx(bar(R::B_K + stage), NC * 128 * a.box * __popc(there));
        __syncwarp();
        if (mine)
          for (int ch = 0; ch < NC; ++ch)
            tma_load_4d(sK + stage * R::STAGE + ch * R::CHUNK + row * 128, &tmK, bar(R::B_K + stage), ch * 64, slot,
                        static_cast<int>(a.by_row_tiles.div(w.item)), page);
        issued = T + 1;
      }
      if (ok) more = w.next(a);
    }
  } else if (warp == 11) {
    // =========================== queries and their statistics, a segment at a time ===========================
    Walk w = first;
    bool ok = true, more = true;
    int s = 0;
    const int pieces = a.c.cols / 8;
    while (more && ok) {
      const int g = static_cast<int>(a.by_row_tiles.div(w.item));
      if (s >= 2) ok = wait_warp(bar(R::B_QFREE + (s & 1)), ((s >> 1) - 1) & 1, ctl, 85);
      if (!ok) break;
      if (lane == 0) {
        const int len = a.c.lengths[w.b];
        if (w.count > 0 && (len < 0 || static_cast<long long>(len) + w.count > a.c.capacity)) *ac.bad = 1;
      }
      for (int r = lane; r < N; r += 32) {
        const int i = static_cast<int>(a.by_gt.div(r)), h = g * a.group + (r - i * a.gt);
        float2 st = make_float2(INFINITY, 0.f);
        if (i < w.count) {
          const int t = p.r.row(w.b, i);
          if (t >= 0 && t < p.r.T) st = row_stats(a, p, w.b, h, t);
          else *ac.bad = 1;
        }
        s_rows[(s & 1) * 2 * N + r] = -st.x;
        s_rows[(s & 1) * 2 * N + N + r] = -st.y;
      }
      const uint32_t dst = sQ + (s & 1) * R::Q_BYTES;
      const int total = w.count * a.gt * pieces;
#pragma unroll 1
      for (int n0 = 0; n0 < total; n0 += 256) {
        uint4 x[8];
        uint32_t at[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int n = n0 + 32 * k + lane;
          const int r = static_cast<int>(p.by_piece.div(n)), piece = n - r * pieces;
          const int i = static_cast<int>(a.by_gt.div(r)), h = g * a.group + (r - i * a.gt);
          at[k] = dst + (piece >> 3) * R::Q_CHUNK + r * 128 + (((piece & 7) ^ (r & 7)) << 4);
          const int t = n < total ? p.r.row(w.b, i) : 0;
          x[k] = make_uint4(0, 0, 0, 0);
          if (n < total && t >= 0 && t < p.r.T)
            x[k] = *reinterpret_cast<const uint4*>(p.q + w.b * p.q_sb + static_cast<long long>(h) * p.q_sh + t * p.q_ss + 16 * piece);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (n0 + 32 * k + lane < total)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at[k]), "r"(x[k].x), "r"(x[k].y), "r"(x[k].z), "r"(x[k].w) : "memory");
      }
      // columns up to the next 16 that the rows do not have: zeros (the keys' are)
      if (pieces & 1)
        for (int r = lane; r < w.count * a.gt; r += 32)
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst + (pieces >> 3) * R::Q_CHUNK + r * 128 + (((pieces & 7) ^ (r & 7)) << 4)),
                       "r"(0)
                       : "memory");
      fence_async_smem();
      mbar_arrive(bar(R::B_Q + (s & 1)));
      ++s;
      more = w.next(a);
    }
  } else if (warp >= 8) {
    // =========================== MMA issue ===========================
    const int st = warp - 8;
    const bool lead = elect_one();
    constexpr uint32_t IDESC = make_idesc(BF16, false, 128, N);
    const int k_steps = (a.c.cols + 15) / 16;
    AttTiles<false> tiles{first, st};
    AttTile t = {0, 0, 0, false};
    bool ok = true;
    for (int c = 0; ok && tiles.take(a, t); ++c) {
      const int stage = stage_of(t.T);
      ok = wait_warp(bar(R::B_K + stage), turn_of(t.T) & 1, ctl, 86) && wait_warp(bar(R::B_Q + (t.s & 1)), (t.s >> 1) & 1, ctl, 87);
      if (ok && c >= 2) ok = wait_warp(bar(R::B_SFREE + 2 * st + (c & 1)), ((c >> 1) - 1) & 1, ctl, 88);
      if (!ok) break;
      tc_fence_after();
      const uint32_t k_lo = sdesc_lo(sK + stage * R::STAGE, 16), q_lo = sdesc_lo(sQ + (t.s & 1) * R::Q_BYTES, 16);
      for (int kk = 0; kk < k_steps; ++kk)
        umma_ss_lead(lead, tmem + (2 * st + (c & 1)) * N, k_lo + (((kk >> 2) * R::CHUNK + (kk & 3) * 32) >> 4),
                     q_lo + (((kk >> 2) * R::Q_CHUNK + (kk & 3) * 32) >> 4), IDESC, kk > 0 ? 1u : 0u);
      umma_commit_lead(lead, bar(R::B_S + 2 * st + (c & 1)));
      umma_commit_lead(lead, bar(R::B_KFREE + stage));
    }
    umma_commit_lead(lead, bar(R::B_DRAIN + st));
    mbar_drain(bar(R::B_DRAIN + st), 0);
  } else {
    // =========================== weights ===========================
    const int st = warp >> 2, key = tid & 127;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    Walk w = first;
    bool more = true, ok = true;
    int c = 0, T0 = 0, s = 0;
    while (more) {
      const int g = static_cast<int>(a.by_row_tiles.div(w.item)), tiles = w.tiles();
      const int old = w.len - w.count;  // positions before the first of these tokens
      float* out = p.w + w.b * p.w_sb + g * p.w_sh;
      // Both streams wait for every segment's queries, with a tile in it or not: neither says twice that a buffer is free before the other has.
      if (ok) ok = wait_warp(bar(R::B_Q + (s & 1)), (s >> 1) & 1, ctl, 89);
      for (int t = 0; t < tiles; ++t) {
        if (((T0 + t) & 1) != st) continue;
        const int pos0 = (w.unit + 4 * t) * ATT_UNIT, pos = pos0 + key;
        const bool mine = pos < w.len && (key >> 5) < w.n - 4 * t;
        const float before = p.add && mine ? out[pos] : 0.f;
        if (ok) ok = wait_warp(bar(R::B_S + 2 * st + (c & 1)), (c >> 1) & 1, ctl, 90);
        tc_fence_after();
        float x[N];
        tmem_ld_cols<N>(tmem + lane_base + (2 * st + (c & 1)) * N, x);
        tmem_wait_ld();
        tc_fence_before();
        mbar_arrive(bar(R::B_SFREE + 2 * st + (c & 1)));
        // (tokens that are not there have m = +inf; their scores come from what the buffer held before)
        const float* rows = s_rows + (s & 1) * 2 * N;
        const float sum = weigh_scores<N>(x, rows, rows + N, a.c_log2, rows_before(pos - old, a.gt));  // (token i sees positions up to old + i)
        if (mine) out[pos] = *ac.bad != 0 ? __int_as_float(0x7fc00000) : before + sum;
        ++c;
      }
      T0 += tiles;
      if (w.ends() && !p.add)  // behind the last position
        for (int i = w.len + tid; i < p.room; i += 256) out[i] = 0.f;
      mbar_arrive(bar(R::B_QFREE + (s & 1)));
      ++s;
      more = w.next(a);
    }
  }

  // ---- teardown ----
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *ac.bad) report(a.status, DEV_BAD_CACHE);
  if (*ac.abort) {
    if (tid == 0) report_abort(ac.abort, a.status);
    if (warp == 10 && lane == 0)
      for (int T = max(issued - R::NS, 0); T < issued; ++T) mbar_drain(bar(R::B_K + stage_of(T)), turn_of(T) & 1);
    Walk w = first;
    bool more = work;
    while (more) {
      float* out = p.w + w.b * p.w_sb + a.by_row_tiles.div(w.item) * p.w_sh;
      for (int i = w.unit * ATT_UNIT + tid; i < min((w.unit + w.n) * ATT_UNIT, w.len); i += ATT_THREADS) out[i] = __int_as_float(0x7fc00000);
      more = w.next(a);
    }
  }
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, R::TMEM);
  }
}

// ---- more rows -------------------------------------------------------------------------------------------------------------------
// Rows picked by an index, as rows of their own: q [B, steps, H, D], statistics [B, H, 2, steps].
__global__ void __launch_bounds__(256) kfa_cache_take_rows_kernel(const AttendParams a, const WeighParams p, FastDiv by_piece, FastDiv by_head,
                                                                  FastDiv by_step, unsigned total) {
  const unsigned at = blockIdx.x * 256u + threadIdx.x;
  wait_for_previous();
  let_next_begin();
  if (at >= total) return;
  const unsigned row = by_piece.div(at), piece = at - row * by_piece.d;
  const unsigned rest = by_head.div(row), h = row - rest * by_head.d;
  const unsigned b = by_step.div(rest), i = rest - b * by_step.d;
  const int t = p.r.row(b, i);
  const bool there = static_cast<int>(i) < p.r.count(b);
  const bool fine = there && t >= 0 && t < p.r.T;
  if (there && !fine) report(a.status, DEV_BAD_CACHE);
  uint4 x = make_uint4(0, 0, 0, 0);
  if (fine) x = *reinterpret_cast<const uint4*>(p.q + b * p.q_sb + h * p.q_sh + t * p.q_ss + 16 * piece);
  *reinterpret_cast<uint4*>(p.q_to + 16ll * at) = x;
  if (piece == 0) {
    const float2 st = fine ? row_stats(a, p, b, h, t) : make_float2(INFINITY, 0.f);
    float* to = p.stats_to + (static_cast<long long>(b) * a.H + h) * 2 * p.r.steps + i;
    to[0] = st.x;
    to[p.r.steps] = st.y;
  }
}

template <int NC>
struct WeighRowsCfg {
  static constexpr int CHUNK = 128 * 64 * 2, STAGE = NC * CHUNK;  // 128 keys, 128 rows
  static constexpr int DQ = 2, DS = 3;  // row tiles; their statistics (two CTAs an SM: what one waits for, the other fills)
  static constexpr int SLOT = 3 * 128 + 4;  // floats: -(m c + log2 l), -m, -log2 l of 128 rows; whether they need two numbers, or are not all there
  static constexpr int SMALL = 1024 + DS * SLOT * 4 + 2 * 128 * 4;
  static constexpr int SMEM = 1024 + STAGE + DQ * STAGE + SMALL;
  static constexpr int TMEM = 256;  // S 2 x 128
  static constexpr int B_K = 0, B_KFREE = 1, B_Q = 2, B_QFREE = B_Q + DQ, B_ST = B_QFREE + DQ, B_STFREE = B_ST + DS, B_S = B_STFREE + DS,
                       B_SFREE = B_S + 2, B_DRAIN = B_SFREE + 2, N_BARS = B_DRAIN + 1;
  static_assert(2 * (SMEM + 1024) <= 233472 && N_BARS * 8 + 256 <= 1024, "shared memory");
  // (4096 tokens, 32 / 8 heads of 128: 109 us; 142 with scores ten times larger, where tiles take two numbers.)
  // Up to here one number per row will do: its rounding moves a weight by 2^-20 / 2 * ln 2 = 3.3e-7 at most, no more than the exponent's own.
  static constexpr float ONE_NUMBER = 16.f;
};

// Items of a sequence: K / V head slowest, then tile of 128 keys, then block of 128 tokens, from the first that sees one of the keys. The
// items of a key tile that a CTA has are a run: its keys stay, and its sums are written once.
constexpr int WEIGH_BLOCK = 128;
struct ItemWalk {
  int b, g, kt, blk, left;  // left: items, this one included
  int len, count;           // positions before the first token; tokens
  // whether length and count say something that is so; otherwise the sequence has no items
  __device__ __forceinline__ static bool load(const AttendParams& a, const WeighParams& p, int b, int& len, int& count) {
    count = p.r.count(b);
    len = a.c.lengths[b];
    if (count == 0 || (len >= 0 && static_cast<long long>(len) + count <= a.c.capacity)) return true;
    count = 0;
    return false;
  }
  __device__ __forceinline__ static int items_of(int len, int count) {
    int n = 0;
    for (int i = 0; i < count; i += WEIGH_BLOCK) n += (len + min(count, i + WEIGH_BLOCK) + 127) / 128;  // tiles that the block sees
    return n;
  }
  __device__ __forceinline__ int blocks() const { return (count + WEIGH_BLOCK - 1) / WEIGH_BLOCK; }
  __device__ __forceinline__ int tiles() const { return (len + count + 127) / 128; }
  __device__ __forceinline__ int first_block() const { return max(kt * 128 - len, 0) / WEIGH_BLOCK; }
  __device__ __forceinline__ void find(int off) {  // off items into the (sequence, head)
    const int nb = blocks(), full = min((len + WEIGH_BLOCK + 127) / 128, tiles());  // tiles that all blocks see
    if (off < full * nb) {
      kt = off / nb;
      blk = off - kt * nb;
      return;
    }
    off -= full * nb;
    for (kt = full;; ++kt) {
      blk = first_block();
      if (off < nb - blk) break;
      off -= nb - blk;
    }
    blk += off;
  }
  __device__ __forceinline__ bool last_of_tile() const { return blk + 1 == blocks(); }
  // the next item of the run, or false: it is over (left: 0 if all is)
  __device__ __forceinline__ bool next() {
    --left;
    if (left <= 0 || last_of_tile()) return false;
    ++blk;
    return true;
  }
  // behind the end of a run: to the next key tile
  __device__ __forceinline__ bool next_run(const AttendParams& a, const WeighParams& p) {
    if (left <= 0) return false;
    if (++kt == tiles()) {
      kt = 0;
      if (++g == a.c.heads) {
        g = 0;
        do {
          ++b;
          (void)load(a, p, b, len, count);
        } while (count == 0);
      }
    }
    blk = first_block();
    return true;
  }
  __device__ __forceinline__ int last_token() const { return min(count, (blk + 1) * WEIGH_BLOCK); }
  // the block's first token that sees one of the keys, in whole row tiles; row tiles of the item
  __device__ __forceinline__ int first_token(const WeighParams& p) const {
    const int i0 = blk * WEIGH_BLOCK, lowest = max(kt * 128 - len, i0);
    return i0 + static_cast<int>(p.by_tile_t.div(lowest - i0)) * p.tile_t;
  }
  __device__ __forceinline__ int row_tiles(const WeighParams& p) const {
    return static_cast<int>(p.by_tile_t.div(last_token() - first_token(p) + p.tile_t - 1)) * p.head_tiles;
  }
};

template <int NC, bool BF16>
__global__ void __launch_bounds__(ATT_THREADS, 2)
kfa_cache_weigh_rows_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const AttendParams a,
                            const WeighParams p) {
  using R = WeighRowsCfg<NC>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t sK = base, sQ = sK + R::STAGE;
  uint8_t* small = smem + R::STAGE + R::DQ * R::STAGE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(small);
  float* s_rows = reinterpret_cast<float*>(small + 1024);  // [slot]
  float* s_sum = s_rows + R::DS * R::SLOT;                 // [run & 1][128]: the second warpgroup's
  const AttCtl ac(bars + R::N_BARS);
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](int i) { return bar0 + 8u * i; };
  const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31;
  if (tid == 32 * 11) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmK) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmQ) : "memory");
  }
  if (warp == 10) {
    for (int i = lane; i < R::N_BARS; i += 32) {
      int count = 1;
      if (i >= R::B_ST && i < R::B_STFREE) count = 32;
      if (i >= R::B_STFREE && i < R::B_S) count = 256;
      if (i >= R::B_SFREE && i < R::B_DRAIN) count = 256;
      mbar_init(bar(i), count);
    }
    if (lane == 0) *ac.abort = 0;
    fence_mbar_init();
    fence_async_smem();
  }
  if (warp == 8) {
    tmem_alloc(smem_u32(ac.tmem), R::TMEM);
    tmem_relinquish();
  }
  wait_for_previous();
  if (warp == 10 && lane == 0) *ac.bad = load_status(a.status) != 0;
  tc_fence_before();
  // which items: an equal number for each CTA
  ItemWalk first;
  int share[2], total;
  auto items = [&](int b) {
    int len, count;
    (void)ItemWalk::load(a, p, b, len, count);
    return ItemWalk::items_of(len, count) * a.c.heads;
  };
  const int chunk = att_share(a, ac.ints, items, share, total,
            [&](int i, int b, int off, int) {
              ac.ints[3 * i] = b;
              ac.ints[3 * i + 1] = off;
            });
  let_next_begin();
  tc_fence_after();
  first.left = min(share[1], total) - share[0];
  const bool work = first.left > 0;
  if (work) {
    first.b = ac.ints[0];
    (void)ItemWalk::load(a, p, first.b, first.len, first.count);
    const int each = ItemWalk::items_of(first.len, first.count);
    first.g = ac.ints[1] / each;
    first.find(ac.ints[1] - first.g * each);
  }
  const uint32_t tmem = *ac.tmem;
  const Ctl ctl{ac.abort};
  int k_issued = 0, q_issued = 0;
  // row tile number T (over all items): its rows lie in stage T % DQ, their statistics in slot T % DS, its scores in buffer T & 1
  if (!work) {
    if (tid == 0) p.part_meta[blockIdx.x] = make_int4(0, 0, 0, 0);
  } else if (warp == 10) {
    // =========================== keys ===========================
    ItemWalk w = first;
    const int per_tile = 128 / a.box;
    bool more = true;
    for (int n = 0; more; ++n) {
      const int row = lane * a.box, pos = w.kt * 128 + row;
      int page = 0, slot = 0;
      bool mine = lane < per_tile && pos < w.len + w.count;
      if (mine && !cache_place(a.c, w.b, pos, page, slot)) {
        mine = false;
        *ac.bad = 1;
      }
      const unsigned there = __ballot_sync(0xffffffffu, mine);
      if (n > 0 && !wait_warp(bar(R::B_KFREE), (n - 1) & 1, ctl, 84)) break;
      if (lane == 0) mbar_expect_tx(bar(R::B_K), NC * 128 * a.box * __popc(there));
      __syncwarp();
      if (mine)
        for (int ch = 0; ch < NC; ++ch) tma_load_4d(sK + ch * R::CHUNK + row * 128, &tmK, bar(R::B_K), ch * 64, slot, w.g, page);
      k_issued = n + 1;
      while (w.next()) {
      }
      more = w.next_run(a, p);
    }
  } else if (warp == 11) {
    // =========================== rows and their statistics ===========================
    ItemWalk w = first;
    bool ok = true, more = true;
    int T = 0;
    while (more && ok) {
      const int tiles = w.row_tiles(p), i1 = w.last_token();
      int token = w.first_token(p), head = 0;  // of the tile
      for (int j = 0; j < tiles && ok; ++j, ++T) {
        float2 st[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = 32 * k + lane, dt = static_cast<int>(p.by_tile_h.div(r)), dh = r - dt * p.tile_h;
          const bool there = dt < p.tile_t && head + dh < a.group && token + dt < i1;
          st[k] = there ? row_stats(a, p, w.b, w.g * a.group + head + dh, token + dt) : make_float2(INFINITY, 0.f);
        }
        const int stage = T % R::DQ, slot = T % R::DS;
        if (T >= R::DQ) ok = wait_warp(bar(R::B_QFREE + stage), (T / R::DQ - 1) & 1, ctl, 85);
        if (!ok) break;
        if (lane == 0) {
          mbar_expect_tx(bar(R::B_Q + stage), NC * p.tile_t * p.tile_h * 128);
          for (int ch = 0; ch < NC; ++ch)
            tma_load_4d(sQ + stage * R::STAGE + ch * R::CHUNK, &tmQ, bar(R::B_Q + stage), ch * 64, w.g * a.group + head, token, w.b);
        }
        q_issued = T + 1;
        if (T >= R::DS) ok = wait_warp(bar(R::B_STFREE + slot), (T / R::DS - 1) & 1, ctl, 76);
        if (!ok) break;
        bool two = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float* to = s_rows + slot * R::SLOT + 32 * k + lane;
          const float t = fmaf(st[k].x, a.c_log2, st[k].y);
          to[0] = -t;
          to[128] = -st[k].x;
          to[256] = -st[k].y;
          two |= !(fabsf(t) <= R::ONE_NUMBER);  // (also where there is no row: infinity)
        }
        two = __any_sync(0xffffffffu, two);
        if (lane == 0) s_rows[slot * R::SLOT + 384] = two ? 1.f : 0.f;
        mbar_arrive(bar(R::B_ST + slot));
        if ((head += p.tile_h) >= a.group) {
          head = 0;
          token += p.tile_t;
        }
      }
      if (ok) more = w.next() || w.next_run(a, p);
    }
  } else if (warp == 9) {
    // (nothing: one warp issues for both halves of the rows)
  } else if (warp == 8) {
    // =========================== MMA issue ===========================
    const bool lead = elect_one();
    constexpr uint32_t IDESC = make_idesc(BF16, false, 128, 128);
    const int k_steps = (a.c.cols + 15) / 16;
    ItemWalk w = first;
    bool ok = true, more = true;
    int T = 0;
    for (int n = 0; more && ok; ++n) {
      ok = wait_warp(bar(R::B_K), n & 1, ctl, 86);
      bool run = true;
      while (run && ok) {
        const int tiles = w.row_tiles(p);
        for (int j = 0; j < tiles && ok; ++j, ++T) {
          const int stage = T % R::DQ;
          ok = wait_warp(bar(R::B_Q + stage), (T / R::DQ) & 1, ctl, 87);
          if (ok && T >= 2) ok = wait_warp(bar(R::B_SFREE + (T & 1)), ((T >> 1) - 1) & 1, ctl, 88);
          if (!ok) break;
          tc_fence_after();
          const uint32_t k_lo = sdesc_lo(sK, 16), q_lo = sdesc_lo(sQ + stage * R::STAGE, 16);
          for (int kk = 0; kk < k_steps; ++kk) {
            const uint32_t off = ((kk >> 2) * R::CHUNK + (kk & 3) * 32) >> 4;
            umma_ss_lead(lead, tmem + (T & 1) * 128, k_lo + off, q_lo + off, IDESC, kk > 0 ? 1u : 0u);
          }
          umma_commit_lead(lead, bar(R::B_S + (T & 1)));
          umma_commit_lead(lead, bar(R::B_QFREE + stage));
        }
        run = w.next();
      }
      if (ok) {
        umma_commit_lead(lead, bar(R::B_KFREE));
        more = w.next_run(a, p);
      }
    }
    umma_commit_lead(lead, bar(R::B_DRAIN));
    mbar_drain(bar(R::B_DRAIN), 0);
  } else {
    // =========================== weights ===========================
    // Each warpgroup 64 of a tile's 128 rows. (After a wait that ran out the role goes on without waiting: they meet at a barrier.)
    const int half = warp >> 2, key = tid & 127;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    ItemWalk w = first;
    bool ok = true, more = true;
    int T = 0;
    int4 meta = make_int4(0, 0, 0, 0);
    for (int n = 0; more; ++n) {
      const int pos = w.kt * 128 + key;
      const bool begins = w.blk == w.first_block();
      float* out = p.w + w.b * p.w_sb + w.g * p.w_sh;
      const bool mine = half == 0 && pos < w.len + w.count;
      const float before = p.add && mine ? out[pos] : 0.f;
      float sum = 0.f;
      bool run = true;
      while (run) {
        const int tiles = w.row_tiles(p);
        int token = w.first_token(p), head = 0;
        float part = 0.f;
        for (int j = 0; j < tiles; ++j, ++T) {
          const int slot = T % R::DS;
          const bool hidden = w.kt * 128 + 127 > w.len + token;  // some key from some row
          if (ok) ok = wait_warp(bar(R::B_ST + slot), (T / R::DS) & 1, ctl, 89);
          const float* rows = s_rows + slot * R::SLOT + 64 * half;
          const bool one = !hidden && s_rows[slot * R::SLOT + 384] == 0.f;
          if (ok) ok = wait_warp(bar(R::B_S + (T & 1)), (T >> 1) & 1, ctl, 90);
          tc_fence_after();
#pragma unroll
          for (int i = 0; i < 64; i += 32) {
            float x[32];
            tmem_ld32(tmem + lane_base + (T & 1) * 128 + 64 * half + i, reinterpret_cast<uint32_t*>(x));
            tmem_wait_ld();
            if (i == 32) {
              tc_fence_before();
              mbar_arrive(bar(R::B_SFREE + (T & 1)));
            }
            if (one) {
              part += weigh_scores_one<32>(x, rows + i, a.c_log2);
            } else {  // (token t sees positions up to len + t)
              part += weigh_scores<32>(x, rows + 128 + i, rows + 256 + i, a.c_log2, rows_before(pos - w.len - token, p.tile_h) - 64 * half - i);
            }
          }
          mbar_arrive(bar(R::B_STFREE + slot));
          if ((head += p.tile_h) >= a.group) {
            head = 0;
            token += p.tile_t;
          }
        }
        sum += part;
        run = w.next();
      }
      if (half == 1) s_sum[(n & 1) * 128 + key] = sum;
      named_sync<3, 256>();  // (the buffer is written again two runs on, behind the next one's barrier)
      const bool ends = w.last_of_tile();
      if (half == 0) {
        sum += s_sum[(n & 1) * 128 + key];
        if (begins && ends) {
          if (mine) out[pos] = *ac.bad != 0 ? __int_as_float(0x7fc00000) : before + sum;
        } else {
          p.part[(2ll * blockIdx.x + (begins ? 1 : 0)) * 128 + key] = sum;
        }
      }
      if (ends && !p.add && w.kt + 1 == w.tiles())  // behind the last position
        for (int i = w.len + w.count + tid; i < p.room; i += 256) out[i] = 0.f;
      if (begins && !ends) meta = make_int4(1 + (w.blocks() - w.blk - 1 + chunk - 1) / chunk, w.b, w.g, w.kt);
      more = w.next_run(a, p);
    }
    if (tid == 0) p.part_meta[blockIdx.x] = meta;
  }

  // ---- teardown ---- (what a CTA that gives up had whole reads as NaN; what it had a part of, the joining kernel sees to)
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *ac.bad) report(a.status, DEV_BAD_CACHE);
  if (*ac.abort) {
    if (tid == 0) report_abort(ac.abort, a.status);
    if (warp == 10 && lane == 0 && k_issued > 0) mbar_drain(bar(R::B_K), (k_issued - 1) & 1);
    if (warp == 11 && lane == 0)
      for (int T = max(q_issued - R::DQ, 0); T < q_issued; ++T) mbar_drain(bar(R::B_Q + T % R::DQ), (T / R::DQ) & 1);
    ItemWalk w = first;
    bool more = work;
    while (more) {
      const bool begins = w.blk == w.first_block();
      while (w.next()) {
      }
      const int pos = w.kt * 128 + tid;
      if (begins && w.last_of_tile() && tid < 128 && pos < w.len + w.count) p.w[w.b * p.w_sb + w.g * p.w_sh + pos] = __int_as_float(0x7fc00000);
      more = w.next_run(a, p);
    }
  }
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, R::TMEM);
  }
}

// Key tiles that were cut, CTA x the one that begins in CTA x of the kernel above: w (+)= the parts, in order. The CTAs behind those: a
// sequence each that has no items, whose weights are 0 (add: left), or NaN if its length or count says something that is not so.
__global__ void __launch_bounds__(256) kfa_cache_join_weights_kernel(const AttendParams a, const WeighParams p, int cut) {
  wait_for_previous();
  let_next_begin();
  const float nan = __int_as_float(0x7fc00000);
  int len, count;
  if (static_cast<int>(blockIdx.x) >= cut) {
    const int b = static_cast<int>(blockIdx.x) - cut;
    const bool fine = ItemWalk::load(a, p, b, len, count);
    if (count > 0 || (fine && p.add)) return;
    if (!fine && threadIdx.x == 0) report(a.status, DEV_BAD_CACHE);
    for (int g = 0; g < a.c.heads; ++g)
      for (int i = threadIdx.x; i < (p.add ? a.c.capacity : p.room); i += 256) p.w[b * p.w_sb + g * p.w_sh + i] = !fine && i < a.c.capacity ? nan : 0.f;
    return;
  }
  const int4 meta = p.part_meta[blockIdx.x];
  if (meta.x == 0) return;
  (void)ItemWalk::load(a, p, meta.y, len, count);
  const int pos = meta.w * 128 + threadIdx.x;
  if (threadIdx.x >= 128 || pos >= len + count) return;
  float* out = p.w + meta.y * p.w_sb + meta.z * p.w_sh + pos;
  float sum = 0.f;
  for (int i = 0; i < meta.x; ++i) sum += p.part[(2ll * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * 128 + threadIdx.x];
  const bool bad = *reinterpret_cast<const volatile int*>(a.status) != 0;
  *out = bad ? nan : (p.add ? *out + sum : sum);
}

}  // namespace kfa
