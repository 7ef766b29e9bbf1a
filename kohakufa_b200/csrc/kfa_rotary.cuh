// Rotary positions: pairs of a row's columns turned by angles that grow with the row's position, as a pass of its own or on the way into a
// cache of keys and values.
//
//   (y1, y2) = a (x1 cos - x2 sin, x2 cos + x1 sin),   angle = position * f_pair      (the gradient: the same with -sin)
//
// Bound by memory: every row is read once and written once. What has to be kept out of the way are the angles. They are not read from a
// table of positions: f is given in turns as a 64-bit fraction, position * f modulo 2^64 is the angle's fraction of a turn without any error but the position
// times that of the fraction (2^-65 turns at best; made of a frequency in radians in 64-bit floats 2^-52 of it), for positions of any size, and sine and cosine are taken of a remainder within an eighth of a turn. A CTA takes a stretch of
// rows, token by token and head by head, so that one token's sines and cosines, in shared memory, serve all its heads (40 of 32 query and 8 key
// heads), and asks for its rows before it makes them: what a sine costs (some 40 instructions) passes while the rows are on their way.
//
// A thread's unit is a cell: two pieces (of up to 16 bytes) of a row that hold each other's partners. Half layout (columns i and i + R / 2 are a
// pair): pieces R / 2 apart; interleaved (2 i and 2 i + 1): adjacent ones. Both ways cell j has the pairs j * V .. (j + 1) * V - 1, V columns a piece. Cells behind
// the turned columns are copied as they are.
#pragma once

#include "kfa_cache_view.cuh"

namespace kfa {

constexpr int ROT_THREADS = 256;
constexpr int ROT_CELLS = 2;  // of a thread (the pass of its own)

struct RotaryStream {  // queries, keys, values
  const uint8_t* in;
  long long in_b, in_h, in_s;  // bytes
  uint8_t* out;                // or nullptr (append: only the pages get it)
  long long out_b, out_h, out_s;
};

struct RotaryParams {
  RotaryStream x[3];
  int q_heads, qk_heads;          // heads before the keys', before the values'
  int heads;                      // of a token, all streams'
  // cells of a row; heads of a token (append: groups of heads, a thread has one head of each); tokens of a sequence; pairs of a row
  FastDiv by_cell, by_group, by_step, by_pair;
  int pairs, pair_cells, columns;  // pair_cells: cells with turned columns
  unsigned total;                  // cells of all heads (groups)
  const uint64_t* turns;
  float amplitude, sine;          // of cosine; of sine (negative: the gradient)
  const void* positions;
  long long pos_b, pos_s;
  int pos_wide;                   // int64
  const int* offset;
  // append
  CacheView c;
  RowsView r;
  int* status;
};

__device__ __forceinline__ long long rotary_position(const RotaryParams& p, int b, int i, int t, bool append) {
  long long at;
  if (p.positions) {
    const long long where = b * p.pos_b + t * p.pos_s;
    at = p.pos_wide ? static_cast<const long long*>(p.positions)[where] : static_cast<const int*>(p.positions)[where];
  } else {
    at = append ? static_cast<long long>(p.c.lengths[b]) + i : t;
  }
  return p.offset ? at + p.offset[b] : at;
}

// cos and sin of a position's angle: the fraction of a turn is cut into a quarter and what is left, within an eighth on both sides, of which 32 bits
// are taken (2^-34 turns; fp32 rounds them by 2^-24 of themselves).
__device__ __forceinline__ float2 rotary_turn(uint64_t turns, long long position, float amplitude, float sine) {
  const uint64_t angle = turns * static_cast<uint64_t>(position);
  const uint64_t quarter = (angle + (1ull << 61)) >> 62;
  const long long left = static_cast<long long>(angle - (quarter << 62));
  float s, c;
  sincospif(static_cast<float>(static_cast<int>(left >> 30)) * 0x1p-33f, &s, &c);
  const float x = quarter & 1 ? -s : c, y = quarter & 1 ? c : s;
  const float sign = quarter & 2 ? -1.f : 1.f;
  return make_float2(x * sign * amplitude, y * sign * sine);
}

template <int BYTES>
struct RotaryPiece;
template <>
struct RotaryPiece<16> { using type = uint4; };
template <>
struct RotaryPiece<8> { using type = uint2; };
template <>
struct RotaryPiece<4> { using type = uint32_t; };
template <>
struct RotaryPiece<2> { using type = uint16_t; };

template <typename T, int BYTES>
union RotaryHalf {
  typename RotaryPiece<BYTES>::type piece;
  T x[BYTES / sizeof(T)];
  __device__ RotaryHalf() {}
};

__device__ __forceinline__ float rotary_float(float x) { return x; }
__device__ __forceinline__ float rotary_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float rotary_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void rotary_round(float x, float& y) { y = x; }
__device__ __forceinline__ void rotary_round(float x, __half& y) { y = __float2half_rn(x); }
__device__ __forceinline__ void rotary_round(float x, __nv_bfloat16& y) { y = __float2bfloat16_rn(x); }
// One pair, y = (cos, sin). (The roundings are written out: both kernels give the same bits.)
template <typename T>
__device__ __forceinline__ void rotary_pair(float x1, float x2, float2 y, T& lo, T& hi) {
  rotary_round(__fmaf_rn(x1, y.x, -__fmul_rn(x2, y.y)), lo);
  rotary_round(__fmaf_rn(x2, y.x, __fmul_rn(x1, y.y)), hi);
}

// The pass of its own. Six CTAs an SM: a training step of 4 x 8192 tokens, 32 / 8 heads, D 128 (two launches) takes 195 us in a graph, what a copy of as many
// bytes takes at 6880 GB/s; with five 208, with one cell a thread 224, with two heads of a cell a thread as below 222 to 250.
template <typename T, int BYTES, bool INTERLEAVED>
__global__ void __launch_bounds__(ROT_THREADS, 6) kfa_rotary_kernel(const RotaryParams p) {
  constexpr int V = BYTES / sizeof(T), CHUNK = V < 2 ? 1 : 2, CHUNKS = V / CHUNK;  // pairs of a cell; of a 16-byte piece of them in shared memory
  using Piece = typename RotaryPiece<BYTES>::type;
  extern __shared__ float4 rotary_smem[];
  float2* cs = reinterpret_cast<float2*>(rotary_smem);  // [token][chunk][cell][CHUNK]
  const unsigned first = blockIdx.x * static_cast<unsigned>(ROT_THREADS * ROT_CELLS);
  const unsigned last = min(first + ROT_THREADS * ROT_CELLS, p.total) - 1;
  const unsigned token0 = p.by_group.div(p.by_cell.div(first)), tokens = p.by_group.div(p.by_cell.div(last)) - token0 + 1;
  wait_for_previous();
  let_next_begin();

  // ---- this thread's cells are asked for ----
  RotaryHalf<T, BYTES> a[ROT_CELLS], b[ROT_CELLS];
  unsigned where[ROT_CELLS];  // token, counted from the CTA's first; head; cell
  uint8_t* to[ROT_CELLS];
  bool two[ROT_CELLS];
  int second[ROT_CELLS];  // bytes from a to b
#pragma unroll
  for (int u = 0; u < ROT_CELLS; ++u) {
    const unsigned at = first + u * ROT_THREADS + threadIdx.x;
    to[u] = nullptr;
    two[u] = false;
    second[u] = 0;
    where[u] = 0;
    if (at >= p.total) continue;
    const unsigned row = p.by_cell.div(at), cell = at - row * p.by_cell.d;
    const unsigned token = p.by_group.div(row);
    int head = static_cast<int>(row - token * p.by_group.d);
    const unsigned seq = p.by_step.div(token);
    const int i = static_cast<int>(token - seq * p.by_step.d);
    const int kind = head < p.q_heads ? 0 : 1;
    const RotaryStream& x = p.x[kind];
    head -= kind == 0 ? 0 : p.q_heads;
    // the first column, and how far the second piece is
    int column = static_cast<int>(cell) * 2 * V, apart = V;
    const bool turned = static_cast<int>(cell) < p.pair_cells;
    if (!INTERLEAVED) {
      if (turned) column = static_cast<int>(cell) * V, apart = p.pairs;
      else column = 2 * p.pairs + (static_cast<int>(cell) - p.pair_cells) * 2 * V;
    }
    two[u] = column + apart < p.columns;
    second[u] = apart * static_cast<int>(sizeof(T));
    where[u] = (token - token0) << 17 | (turned ? 1u << 16 : 0u) | cell;
    const int bytes = column * static_cast<int>(sizeof(T));
    const uint8_t* from = x.in + seq * x.in_b + head * x.in_h + i * x.in_s + bytes;
    a[u].piece = *reinterpret_cast<const Piece*>(from);
    if (two[u]) b[u].piece = *reinterpret_cast<const Piece*>(from + second[u]);
    to[u] = x.out + seq * x.out_b + head * x.out_h + i * x.out_s + bytes;
  }

  // ---- the CTA's tokens' angles ----
  for (unsigned at = threadIdx.x; at < tokens * p.pairs; at += ROT_THREADS) {
    const unsigned token = p.by_pair.div(at), pair = at - token * p.pairs;
    const unsigned seq = p.by_step.div(token0 + token);
    const int i = static_cast<int>(token0 + token - seq * p.by_step.d);
    const unsigned cell = pair / V, in = pair % V;
    cs[((token * CHUNKS + in / CHUNK) * p.pair_cells + cell) * CHUNK + in % CHUNK] =
        rotary_turn(p.turns[pair], rotary_position(p, static_cast<int>(seq), i, i, false), p.amplitude, p.sine);
  }
  __syncthreads();

#pragma unroll
  for (int u = 0; u < ROT_CELLS; ++u) {
    if (to[u] == nullptr) continue;
    const unsigned token = where[u] >> 17, cell = where[u] & 0xffffu;
    if (where[u] & 1u << 16) {
      const float2* angles = cs + (token * CHUNKS * p.pair_cells + cell) * CHUNK;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float2 y = angles[(k / CHUNK) * p.pair_cells * CHUNK + k % CHUNK];
        // (pair k of the cell; interleaved: the first half of them lies in the first piece)
        T& lo = INTERLEAVED ? (2 * k < V ? a[u].x[2 * k % V] : b[u].x[2 * k % V]) : a[u].x[k];
        T& hi = INTERLEAVED ? (2 * k + 1 < V ? a[u].x[(2 * k + 1) % V] : b[u].x[(2 * k + 1) % V]) : b[u].x[k];
        if (INTERLEAVED && static_cast<int>(cell) * V + k >= p.pairs) continue;
        const float x1 = rotary_float(lo), x2 = rotary_float(hi);
        rotary_pair(x1, x2, y, lo, hi);
      }
    }
    *reinterpret_cast<Piece*>(to[u]) = a[u].piece;
    if (two[u]) *reinterpret_cast<Piece*>(to[u] + second[u]) = b[u].piece;
  }
}

// On the way into a cache. A thread has the same cell of HEADS heads of a token: what is looked up for the token (its count, row, page, angles) and what the
// indices' divisions take, which bound this kernel where a thread had two cells anywhere, are once a thread. Prompts of 4 x 4096 tokens, 32 / 8 heads,
// D 128, keys twice, in a graph: 70.2 us with three heads a thread, 77.0 with two, 86 with one, 84 with two cells anywhere (a copy of as many bytes takes 67);
// 64 tokens 3.5, 3.0, 2.7: one head a thread where the GPU is not filled.
template <typename T, int BYTES, bool INTERLEAVED, int HEADS>
__global__ void __launch_bounds__(ROT_THREADS, 4) kfa_rotary_append_kernel(const RotaryParams p) {
  constexpr int V = BYTES / sizeof(T), CHUNK = V < 2 ? 1 : 2, CHUNKS = V / CHUNK;  // pairs of a cell; of a 16-byte piece of them in shared memory
  using Piece = typename RotaryPiece<BYTES>::type;
  extern __shared__ float4 rotary_smem[];
  float2* cs = reinterpret_cast<float2*>(rotary_smem);  // [token][chunk][cell][CHUNK]
  const unsigned first = blockIdx.x * static_cast<unsigned>(ROT_THREADS), last = min(first + ROT_THREADS, p.total) - 1, at = first + threadIdx.x;
  const unsigned token0 = p.by_group.div(p.by_cell.div(first)), tokens = p.by_group.div(p.by_cell.div(last)) - token0 + 1;
  const unsigned row = p.by_cell.div(at), cell = at - row * p.by_cell.d, token = p.by_group.div(row);
  const int group = static_cast<int>(row - token * p.by_group.d);
  const unsigned seq = p.by_step.div(token);
  const int i = static_cast<int>(token - seq * p.by_step.d);
  // the first column of queries and keys, and how far the second piece is; values have adjacent ones
  const bool turned = static_cast<int>(cell) < p.pair_cells;
  int column = static_cast<int>(cell) * 2 * V, apart = V;
  if (!INTERLEAVED) {
    if (turned) column = static_cast<int>(cell) * V, apart = p.pairs;
    else column = 2 * p.pairs + (static_cast<int>(cell) - p.pair_cells) * 2 * V;
  }
  wait_for_previous();
  let_next_begin();

  // ---- this thread's cells are asked for ----
  RotaryHalf<T, BYTES> a[HEADS], b[HEADS];
  int t = i;
  bool there = at < p.total;
  const bool mine = there;
  there = there && i < p.r.count(static_cast<int>(seq));
  if (there) {
    t = p.r.row(static_cast<int>(seq), i);
    if (t < 0 || t >= p.r.T) {
      report(p.status, DEV_BAD_CACHE);
      there = false;
    }
  }
#pragma unroll
  for (int u = 0; u < HEADS; ++u) {
    a[u].piece = b[u].piece = Piece{};
    int head = group + u * static_cast<int>(p.by_group.d);
    if (!there || head >= p.heads) continue;
    const int kind = head < p.q_heads ? 0 : (head < p.qk_heads ? 1 : 2);
    const RotaryStream& x = p.x[kind];
    head -= kind == 0 ? 0 : (kind == 1 ? p.q_heads : p.qk_heads);
    const int col = kind < 2 ? column : static_cast<int>(cell) * 2 * V, far = kind < 2 ? apart : V;
    const uint8_t* from = x.in + seq * x.in_b + head * x.in_h + t * x.in_s + col * static_cast<int>(sizeof(T));
    a[u].piece = *reinterpret_cast<const Piece*>(from);
    if (col + far < p.columns) b[u].piece = *reinterpret_cast<const Piece*>(from + far * static_cast<int>(sizeof(T)));
  }
  // where the token's keys and values go
  uint8_t *k_to = nullptr, *v_to = nullptr;
  if (there && group + (HEADS - 1) * static_cast<int>(p.by_group.d) >= p.q_heads) {
    const int length = p.c.lengths[seq];
    const long long pos = static_cast<long long>(length) + i;
    int page = -1, slot = 0;
    if (length < 0 || pos >= p.c.capacity || !cache_place(p.c, static_cast<int>(seq), static_cast<int>(pos), page, slot)) {
      report(p.status, DEV_BAD_CACHE);
    } else {
      k_to = p.c.k + page * p.c.k_sn + slot * p.c.k_ss;
      v_to = p.c.v + page * p.c.v_sn + slot * p.c.v_ss;
    }
  }

  // ---- the CTA's tokens' angles ----
  for (unsigned n = threadIdx.x; n < tokens * p.pairs; n += ROT_THREADS) {
    const unsigned of = p.by_pair.div(n), pair = n - of * p.pairs;
    const unsigned b_of = p.by_step.div(token0 + of);
    const int i_of = static_cast<int>(token0 + of - b_of * p.by_step.d);
    if (i_of >= p.r.count(static_cast<int>(b_of))) continue;
    const int t_of = p.r.row(static_cast<int>(b_of), i_of);
    if (t_of < 0 || t_of >= p.r.T) continue;
    const unsigned to_cell = pair / V, in = pair % V;
    cs[((of * CHUNKS + in / CHUNK) * p.pair_cells + to_cell) * CHUNK + in % CHUNK] =
        rotary_turn(p.turns[pair], rotary_position(p, static_cast<int>(b_of), i_of, t_of, true), p.amplitude, p.sine);
  }
  __syncthreads();
  if (!mine) return;

  // (a thread's heads have the same angles)
  float2 y[V];
  if (turned && there) {
    const unsigned from = ((token - token0) * CHUNKS * p.pair_cells + cell) * CHUNK;
#pragma unroll
    for (int k = 0; k < V; k += CHUNK) {
      if constexpr (CHUNK == 2) {
        const float4 z = reinterpret_cast<const float4*>(cs)[(from >> 1) + (k / 2) * p.pair_cells];
        y[k] = make_float2(z.x, z.y);
        y[k + 1] = make_float2(z.z, z.w);
      } else {
        y[k] = cs[from + k * p.pair_cells];
      }
    }
  }
#pragma unroll
  for (int u = 0; u < HEADS; ++u) {
    int head = group + u * static_cast<int>(p.by_group.d);
    if (head >= p.heads) continue;
    const int kind = head < p.q_heads ? 0 : (head < p.qk_heads ? 1 : 2);
    const RotaryStream& x = p.x[kind];
    head -= kind == 0 ? 0 : (kind == 1 ? p.q_heads : p.qk_heads);
    const int col = kind < 2 ? column : static_cast<int>(cell) * 2 * V, far = (kind < 2 ? apart : V) * static_cast<int>(sizeof(T));
    if (turned && there && kind < 2) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        // (pair k of the cell; interleaved: the first half of them lies in the first piece)
        T& lo = INTERLEAVED ? (2 * k < V ? a[u].x[2 * k % V] : b[u].x[2 * k % V]) : a[u].x[k];
        T& hi = INTERLEAVED ? (2 * k + 1 < V ? a[u].x[(2 * k + 1) % V] : b[u].x[(2 * k + 1) % V]) : b[u].x[k];
        if (INTERLEAVED && static_cast<int>(cell) * V + k >= p.pairs) continue;
        const float x1 = rotary_float(lo), x2 = rotary_float(hi);
        rotary_pair(x1, x2, y[k], lo, hi);
      }
    }
    const bool two = col + far / static_cast<int>(sizeof(T)) < p.columns;
    const int bytes = col * static_cast<int>(sizeof(T));
    if (x.out != nullptr) {
      uint8_t* to = x.out + seq * x.out_b + head * x.out_h + i * x.out_s + bytes;
      *reinterpret_cast<Piece*>(to) = a[u].piece;
      if (two) *reinterpret_cast<Piece*>(to + far) = b[u].piece;
    }
    if (kind > 0 && k_to != nullptr) {
      uint8_t* to = (kind == 1 ? k_to + head * p.c.k_sh : v_to + head * p.c.v_sh) + bytes;
      *reinterpret_cast<Piece*>(to) = a[u].piece;
      if (two) *reinterpret_cast<Piece*>(to + far) = b[u].piece;
    }
  }
}

}  // namespace kfa
