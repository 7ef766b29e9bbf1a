// How much attention the newest tokens gave to every cached position: w[p] = sum over rows of exp2((q k_p - m) c - log2 l), the rows' m
// and log2 l from the attention call. The keys are the rows of the matrix instructions, as in kfa_cache_attend_kernel: a thread holds a key
// and sums over the columns, the query rows, so that nothing crosses threads.
//
// Up to 64 rows (kfa_cache_weigh_kernel, a decoding step): bound by the keys, read once; work cut by keys as in the attention, every
// position is one CTA's. More rows (kfa_cache_weigh_rows_kernel, a prompt): bound by the exponentials; an item is a tile of 128 keys and a block of
// the tokens, whose rows stream past the keys in tiles of 64; the blocks' sums go to scratch and are added in order.
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
  // many rows: tokens per block, blocks; tokens and heads of a row tile; their sums [block][B * Hkv][capacity]
  int block, blocks, tile_t, tile_h, head_tiles;
  FastDiv by_tile_h, by_piece;  // (pieces: 16 bytes of a row)
  float* part;
  // rows picked by an index, gathered
  uint8_t* q_to;
  float* stats_to;
};

// m and log2 l of row r of a (sequence, K / V head): token i of those that count, head h. What is not there: +inf, which gives 0.
__device__ __forceinline__ float2 row_stats(const AttendParams& a, const WeighParams& p, int b, int h, int t) {
  const float* at = p.stats + (static_cast<long long>(b) * a.H + h) * 2 * p.r.T + t;
  return make_float2(at[0], at[p.r.T]);
}

// The weights of a key, summed: N scores against N rows, whose -m and -log2 l stand one after the other (two at a time in the packed
// instructions). slow: some rows are not there (-m = -inf, and their scores may be anything), or do not see the key: those below r_min.
template <int N>
__device__ __forceinline__ float weigh_scores(const float* x, const float* neg_m, const float* neg_l, float c_log2, bool slow, int r_min) {
  const float2 c2 = make_float2(c_log2, c_log2);
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const float4 m = *reinterpret_cast<const float4*>(neg_m + i), l = *reinterpret_cast<const float4*>(neg_l + i);
    float2 e0 = __ffma2_rn(__fadd2_rn(make_float2(x[i], x[i + 1]), make_float2(m.x, m.y)), c2, make_float2(l.x, l.y));
    float2 e1 = __ffma2_rn(__fadd2_rn(make_float2(x[i + 2], x[i + 3]), make_float2(m.z, m.w)), c2, make_float2(l.z, l.w));
    e0 = make_float2(ex2(e0.x), ex2(e0.y));
    e1 = make_float2(ex2(e1.x), ex2(e1.y));
    if (slow) {
      if (m.x == -INFINITY || i < r_min) e0.x = 0.f;
      if (m.y == -INFINITY || i + 1 < r_min) e0.y = 0.f;
      if (m.z == -INFINITY || i + 2 < r_min) e1.x = 0.f;
      if (m.w == -INFINITY || i + 3 < r_min) e1.y = 0.f;
    }
    sum[0] = __fadd2_rn(sum[0], e0);
    sum[1] = __fadd2_rn(sum[1], e1);
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
  static constexpr int B_K = 0, B_KFREE = NS, B_Q = 2 * NS, B_QFREE = B_Q + 2, B_S = B_QFREE + 1, B_SFREE = B_S + 4, B_DRAIN = B_SFREE + 4,
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
      if (i == R::B_QFREE) count = 256;
      if (i >= R::B_SFREE && i < R::B_DRAIN) count = 128;
      mbar_init(bar(i), count);
    }
    if (lane == 0) {
      *ac.abort = 0;
      *ac.bad = load_status(a.status) != 0;
    }
    fence_mbar_init();
    fence_async_smem();
  }
  if (warp == 8) {
    tmem_alloc(smem_u32(ac.tmem), R::TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  Walk first;
  int chunk, end;
  const bool work = my_work(a, ac.ints, first, chunk, end);
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
          ok = mbar_wait_warp(bar(R::B_KFREE + stage), (turn_of(T) - 1) & 1, ctl, 84);
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
      if (s >= 2) ok = mbar_wait_warp(bar(R::B_QFREE), (s - 2) & 1, ctl, 85);
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
      ok = mbar_wait_warp(bar(R::B_K + stage), turn_of(t.T) & 1, ctl, 86) && mbar_wait_warp(bar(R::B_Q + (t.s & 1)), (t.s >> 1) & 1, ctl, 87);
      if (ok && c >= 2) ok = mbar_wait_warp(bar(R::B_SFREE + 2 * st + (c & 1)), ((c >> 1) - 1) & 1, ctl, 88);
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
      // (its statistics are there: the keys' scores are waited for below, but a stream without tiles in the segment looks at nothing)
      for (int t = 0; t < tiles; ++t) {
        if (((T0 + t) & 1) != st) continue;
        const int pos0 = (w.unit + 4 * t) * ATT_UNIT, pos = pos0 + key;
        const bool mine = pos < w.len && (key >> 5) < w.n - 4 * t;
        const float before = p.add && mine ? out[pos] : 0.f;
        if (ok) ok = mbar_wait_warp(bar(R::B_Q + (s & 1)), (s >> 1) & 1, ctl, 89);
        if (ok) ok = mbar_wait_warp(bar(R::B_S + 2 * st + (c & 1)), (c >> 1) & 1, ctl, 90);
        tc_fence_after();
        float x[N];
        tmem_ld_cols<N>(tmem + lane_base + (2 * st + (c & 1)) * N, x);
        tmem_wait_ld();
        tc_fence_before();
        mbar_arrive(bar(R::B_SFREE + 2 * st + (c & 1)));
        // (tokens that are not there have m = +inf; their scores come from what the buffer held before)
        const float* rows = s_rows + (s & 1) * 2 * N;
        const float sum = weigh_scores<N>(x, rows, rows + N, a.c_log2, true, (pos - old) * a.gt);  // (token i sees positions up to old + i)
        if (mine) out[pos] = *ac.bad != 0 ? __int_as_float(0x7fc00000) : before + sum;
        ++c;
      }
      T0 += tiles;
      if (w.ends() && !p.add)  // behind the last position
        for (int i = w.len + tid; i < p.room; i += 256) out[i] = 0.f;
      mbar_arrive(bar(R::B_QFREE));
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
  static constexpr int CHUNK = 128 * 64 * 2, STAGE = NC * CHUNK;
  static constexpr int Q_CHUNK = 64 * 128, Q_BYTES = NC * Q_CHUNK;
  static constexpr int DK = 1, DQ = 2;  // key tiles; row tiles per stream (two CTAs an SM: what one waits for, the other fills)
  static constexpr int SMALL = 1024 + 2 * DQ * 64 * 8 + 2 * 128 * 4 * 2;
  static constexpr int SMEM = 1024 + DK * STAGE + 2 * DQ * Q_BYTES + SMALL;
  static constexpr int TMEM = 256;  // S 2 x 2 x 64
  static constexpr int B_K = 0, B_KFREE = DK, B_Q = 2 * DK, B_QFREE = B_Q + 2 * DQ, B_S = B_QFREE + 2 * DQ, B_SFREE = B_S + 4,
                       B_DRAIN = B_SFREE + 4, N_BARS = B_DRAIN + 2;
  static_assert(2 * (SMEM + 1024) <= 233472 && N_BARS * 8 + 256 <= 1024, "shared memory");
};

// Items of a sequence: K / V head slowest, then block of tokens, then tile of 128 keys: those that some token of the block sees.
struct ItemWalk {
  int b, g, blk, kt, left;      // left: items, this one included
  int len, count;               // positions before the first token; tokens
  int i0, i1, keys, tiles;      // of the block: tokens i0 .. i1 - 1, positions they see, tiles of them
  __device__ __forceinline__ static int tiles_of(const WeighParams& p, int len, int count, int blk) {
    const int upto = min(count, (blk + 1) * p.block);
    return blk * p.block < upto ? (len + upto + 127) / 128 : 0;
  }
  __device__ __forceinline__ static int items_of(const AttendParams& a, const WeighParams& p, int b, int& len, int& count) {
    count = p.r.count(b);
    len = a.c.lengths[b];
    if (len < 0 || static_cast<long long>(len) + count > a.c.capacity) count = 0;  // (reported where the sums are joined)
    int n = 0;
    for (int k = 0; k < p.blocks; ++k) n += tiles_of(p, len, count, k);
    return n;
  }
  __device__ __forceinline__ void block(const WeighParams& p) {
    i0 = blk * p.block;
    i1 = min(count, i0 + p.block);
    keys = len + i1;
    tiles = tiles_of(p, len, count, blk);
  }
  __device__ __forceinline__ bool next(const AttendParams& a, const WeighParams& p) {
    if (--left <= 0) return false;
    if (++kt < tiles) return true;
    kt = 0;
    do {
      if (++blk == p.blocks) {
        blk = 0;
        if (++g == a.c.heads) {
          g = 0;
          ++b;
          (void)items_of(a, p, b, len, count);
        }
      }
      block(p);
    } while (tiles == 0);
    return true;
  }
  // row tiles of the item: of the block's tokens, from the first that sees one of its keys
  __device__ __forceinline__ int first_token(const WeighParams& p) const {
    const int lowest = max(kt * 128 - len, i0);
    return i0 + (lowest - i0) / p.tile_t * p.tile_t;
  }
  __device__ __forceinline__ int row_tiles(const WeighParams& p) const {
    return (i1 - first_token(p) + p.tile_t - 1) / p.tile_t * p.head_tiles;
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
  const uint32_t sK = base, sQ = sK + R::DK * R::STAGE;
  uint8_t* small = smem + R::DK * R::STAGE + 2 * R::DQ * R::Q_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(small);
  float* s_rows = reinterpret_cast<float*>(small + 1024);                                // [stage][-m, -log2 l][64]
  float* s_sum = reinterpret_cast<float*>(small + 1024 + 2 * R::DQ * 64 * 8);            // [item & 1][128]: the second stream's
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
      if (i >= R::B_KFREE && i < R::B_Q) count = 2;
      if (i >= R::B_Q && i < R::B_QFREE) count = 33;
      if (i >= R::B_QFREE && i < R::B_S) count = 129;  // a stream's threads (statistics) and its products
      if (i >= R::B_SFREE && i < R::B_DRAIN) count = 128;
      mbar_init(bar(i), count);
    }
    if (lane == 0) {
      *ac.abort = 0;
      *ac.bad = load_status(a.status) != 0;
    }
    fence_mbar_init();
    fence_async_smem();
  }
  if (warp == 8) {
    tmem_alloc(smem_u32(ac.tmem), R::TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  // which items: an equal number for each CTA
  ItemWalk first;
  int share[2], total;
  int unused_len, unused_count;
  att_share(a, ac.ints, [&](int b) { return ItemWalk::items_of(a, p, b, unused_len, unused_count) * a.c.heads; }, share, total,
            [&](int i, int b, int off, int) {
              ac.ints[3 * i] = b;
              ac.ints[3 * i + 1] = off;
            });
  tc_fence_after();
  first.left = min(share[1], total) - share[0];
  const bool work = first.left > 0;
  if (work) {
    first.b = ac.ints[0];
    int off = ac.ints[1];
    const int each = ItemWalk::items_of(a, p, first.b, first.len, first.count);
    first.g = off / each;
    off -= first.g * each;
    first.blk = 0;
    first.block(p);
    while (off >= first.tiles) {
      off -= first.tiles;
      ++first.blk;
      first.block(p);
    }
    first.kt = off;
  }
  const uint32_t tmem = *ac.tmem;
  const Ctl ctl{ac.abort};
  int k_issued = 0, q_issued = 0;
  // row tile number T (over all items) is stream T & 1's, in its stage (T >> 1) % DQ
  auto q_stage = [](int T) { return (T & 1) * R::DQ + (T >> 1) % R::DQ; };
  auto q_turn = [](int T) { return (T >> 1) / R::DQ; };

  if (!work) {
  } else if (warp == 10) {
    // =========================== keys ===========================
    ItemWalk w = first;
    const int per_tile = 128 / a.box;
    bool ok = true, more = true;
    for (int n = 0; more && ok; ++n) {
      const int row = lane * a.box, pos = w.kt * 128 + row;
      int page = 0, slot = 0;
      bool mine = lane < per_tile && pos < w.keys;
      if (mine && !cache_place(a.c, w.b, pos, page, slot)) {
        mine = false;
        *ac.bad = 1;
      }
      const unsigned there = __ballot_sync(0xffffffffu, mine);
      if (n >= R::DK) ok = mbar_wait_warp(bar(R::B_KFREE + n % R::DK), (n / R::DK - 1) & 1, ctl, 84);
      if (!ok) break;
      if (lane == 0) mbar_expect_tx(bar(R::B_K + n % R::DK), NC * 128 * a.box * __popc(there));
      __syncwarp();
      if (mine)
        for (int ch = 0; ch < NC; ++ch)
          tma_load_4d(sK + n % R::DK * R::STAGE + ch * R::CHUNK + row * 128, &tmK, bar(R::B_K + n % R::DK), ch * 64, slot, w.g, page);
      k_issued = n + 1;
      more = w.next(a, p);
    }
  } else if (warp == 11) {
    // =========================== rows and their statistics ===========================
    ItemWalk w = first;
    bool ok = true, more = true;
    int T = 0;
    while (more && ok) {
      const int tiles = w.row_tiles(p), t0 = w.first_token(p);
      int token = t0, head = 0;  // of the tile
      for (int j = 0; j < tiles && ok; ++j, ++T) {
        float2 st[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int r = 32 * k + lane, dt = static_cast<int>(p.by_tile_h.div(r)), dh = r - dt * p.tile_h;
          const bool there = dt < p.tile_t && head + dh < a.group && token + dt < w.i1;
          st[k] = there ? row_stats(a, p, w.b, w.g * a.group + head + dh, token + dt) : make_float2(INFINITY, 0.f);
        }
        const int stage = q_stage(T);
        if (q_turn(T) > 0) ok = mbar_wait_warp(bar(R::B_QFREE + stage), (q_turn(T) - 1) & 1, ctl, 85);
        if (!ok) break;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          s_rows[stage * 128 + 32 * k + lane] = -st[k].x;
          s_rows[stage * 128 + 64 + 32 * k + lane] = -st[k].y;
        }
        if (lane == 0) {
          mbar_expect_tx(bar(R::B_Q + stage), NC * p.tile_t * p.tile_h * 128);
          for (int ch = 0; ch < NC; ++ch)
            tma_load_4d(sQ + stage * R::Q_BYTES + ch * R::Q_CHUNK, &tmQ, bar(R::B_Q + stage), ch * 64, w.g * a.group + head, token, w.b);
        }
        mbar_arrive(bar(R::B_Q + stage));
        q_issued = T + 1;
        if ((head += p.tile_h) >= a.group) {
          head = 0;
          token += p.tile_t;
        }
      }
      if (ok) more = w.next(a, p);
    }
  } else if (warp >= 8) {
    // =========================== MMA issue ===========================
    const int st = warp - 8;
    const bool lead = elect_one();
    constexpr uint32_t IDESC = make_idesc(BF16, false, 128, 64);
    const int k_steps = (a.c.cols + 15) / 16;
    ItemWalk w = first;
    bool ok = true, more = true;
    int T = 0, c = 0;
    for (int n = 0; more && ok; ++n) {
      const int tiles = w.row_tiles(p);
      ok = mbar_wait_warp(bar(R::B_K + n % R::DK), (n / R::DK) & 1, ctl, 86);
      for (int j = 0; j < tiles && ok; ++j, ++T) {
        if ((T & 1) != st) continue;
        const int stage = q_stage(T);
        ok = mbar_wait_warp(bar(R::B_Q + stage), q_turn(T) & 1, ctl, 87);
        if (ok && c >= 2) ok = mbar_wait_warp(bar(R::B_SFREE + 2 * st + (c & 1)), ((c >> 1) - 1) & 1, ctl, 88);
        if (!ok) break;
        tc_fence_after();
        const uint32_t k_lo = sdesc_lo(sK + n % R::DK * R::STAGE, 16), q_lo = sdesc_lo(sQ + stage * R::Q_BYTES, 16);
        for (int kk = 0; kk < k_steps; ++kk)
          umma_ss_lead(lead, tmem + (2 * st + (c & 1)) * 64, k_lo + (((kk >> 2) * R::CHUNK + (kk & 3) * 32) >> 4),
                       q_lo + (((kk >> 2) * R::Q_CHUNK + (kk & 3) * 32) >> 4), IDESC, kk > 0 ? 1u : 0u);
        umma_commit_lead(lead, bar(R::B_S + 2 * st + (c & 1)));
        umma_commit_lead(lead, bar(R::B_QFREE + stage));
        ++c;
      }
      if (ok) {
        umma_commit_lead(lead, bar(R::B_KFREE + n % R::DK));
        more = w.next(a, p);
      }
    }
    umma_commit_lead(lead, bar(R::B_DRAIN + st));
    mbar_drain(bar(R::B_DRAIN + st), 0);
  } else {
    // =========================== weights ===========================
    // (After a wait that ran out the role goes on without waiting: the streams meet at a barrier.)
    const int st = warp >> 2, key = tid & 127;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    ItemWalk w = first;
    bool ok = true, more = true;
    int T = 0, c = 0;
    for (int n = 0; more; ++n) {
      const int tiles = w.row_tiles(p), pos = w.kt * 128 + key;
      int token = w.first_token(p), head = 0;
      float sum = 0.f;
      for (int j = 0; j < tiles; ++j, ++T) {
        if ((T & 1) == st) {
          const int stage = q_stage(T);
          const bool slow = w.kt * 128 + 127 > w.len + token || token + p.tile_t > w.i1 || p.tile_t * p.tile_h < 64 || head + p.tile_h > a.group;
          if (ok) ok = mbar_wait_warp(bar(R::B_Q + stage), q_turn(T) & 1, ctl, 89);
          if (ok) ok = mbar_wait_warp(bar(R::B_S + 2 * st + (c & 1)), (c >> 1) & 1, ctl, 90);
          tc_fence_after();
          const float* rows = s_rows + stage * 128;
          const bool odd = slow || __any_sync(0xffffffffu, rows[lane] == -INFINITY || rows[lane + 32] == -INFINITY);
          const int r_min = (pos - w.len - token) * p.tile_h;  // (token t sees positions up to len + t)
#pragma unroll
          for (int i = 0; i < 64; i += 32) {
            float x[32];
            tmem_ld32(tmem + lane_base + (2 * st + (c & 1)) * 64 + i, reinterpret_cast<uint32_t*>(x));
            tmem_wait_ld();
            if (i == 32) {
              tc_fence_before();
              mbar_arrive(bar(R::B_SFREE + 2 * st + (c & 1)));
            }
            if (odd) sum += weigh_scores<32>(x, rows + i, rows + 64 + i, a.c_log2, true, r_min - i);
            else sum += weigh_scores<32>(x, rows + i, rows + 64 + i, a.c_log2, false, 0);
          }
          mbar_arrive(bar(R::B_QFREE + stage));
          ++c;
        }
        if ((head += p.tile_h) >= a.group) {
          head = 0;
          token += p.tile_t;
        }
      }
      if (st == 1) s_sum[(n & 1) * 128 + key] = sum;
      named_sync<3, 256>();  // (the buffer is written again two items on, behind the next one's barrier)
      if (st == 0 && pos < w.keys)
        p.part[(static_cast<long long>(w.blk) * a.c.batch * a.c.heads + static_cast<long long>(w.b) * a.c.heads + w.g) * a.c.capacity + pos] =
            sum + s_sum[(n & 1) * 128 + key];
      more = w.next(a, p);
    }
  }

  // ---- teardown ---- (what a CTA that gives up has not written, the joining kernel replaces: it sees the status)
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *ac.bad) report(a.status, DEV_BAD_CACHE);
  if (*ac.abort) {
    if (tid == 0) report_abort(ac.abort, a.status);
    if (warp == 10 && lane == 0)
      for (int n = max(k_issued - R::DK, 0); n < k_issued; ++n) mbar_drain(bar(R::B_K + n % R::DK), (n / R::DK) & 1);
    if (warp == 11 && lane == 0)
      for (int T = max(q_issued - 2 * R::DQ, 0); T < q_issued; ++T) mbar_drain(bar(R::B_Q + q_stage(T)), q_turn(T) & 1);
  }
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, R::TMEM);
  }
}

// w (+)= the blocks' sums, in order; 0 behind the last position (add: left).
__global__ void __launch_bounds__(256) kfa_cache_sum_blocks_kernel(const AttendParams a, const WeighParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int g = blockIdx.y, b = blockIdx.z;
  const int count = p.r.count(b), len = a.c.lengths[b];
  const bool wrong = count > 0 && (len < 0 || static_cast<long long>(len) + count > a.c.capacity);
  if (wrong && threadIdx.x == 0) report(a.status, DEV_BAD_CACHE);
  const bool bad = wrong || *reinterpret_cast<const volatile int*>(a.status) != 0;
  const int seen = wrong ? a.c.capacity : (count > 0 ? len + count : 0);
  float* out = p.w + b * p.w_sb + g * p.w_sh;
  for (int pos = blockIdx.x * 256 + threadIdx.x; pos < p.room; pos += gridDim.x * 256) {
    if (p.add && pos >= seen) return;
    float w = p.add ? out[pos] : 0.f;
    if (!wrong)
      for (int k = 0; k < p.blocks; ++k)
        if (k * p.block < count && pos < len + min(count, (k + 1) * p.block))
          w += p.part[(static_cast<long long>(k) * a.c.batch * a.c.heads + static_cast<long long>(b) * a.c.heads + g) * a.c.capacity + pos];
    out[pos] = bad && pos < seen ? __int_as_float(0x7fc00000) : w;
  }
}

}  // namespace kfa
