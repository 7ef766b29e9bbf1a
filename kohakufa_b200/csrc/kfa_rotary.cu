// C ABI of rotary positions (declared in include/kfa.h): argument checks and launches.
#include "kfa_cache_call.cuh"
#include "kfa_rotary.cuh"

namespace {

// A tensor of rows [B, H, S, D]: last dimension contiguous, other strides not negative, base and strides whole elements.
int check_rows_of(const KfaTensor4* t, int size, const char* name) {
  if (!t || !t->ptr) return fail(KFA_ERR_ARG, "%s: null tensor", name);
  if (reinterpret_cast<uintptr_t>(t->ptr) % size) return fail(KFA_ERR_ARG, "%s: base not aligned", name);
  if (t->shape[3] > 1 && t->stride[3] != 1) return fail(KFA_ERR_ARG, "%s: last dimension must be contiguous", name);
  for (int i = 0; i < 4; ++i) {
    if (t->shape[i] < 1 || t->shape[i] > 0x7fffffff) return fail(KFA_ERR_ARG, "%s: bad shape[%d]", name, i);
    if (t->shape[i] > 1 && t->stride[i] < 0) return fail(KFA_ERR_ARG, "%s: stride[%d] is negative", name, i);
  }
  return KFA_OK;
}

// Written: rows of their own.
int check_rows_out(const KfaTensor4* t, int size, const char* name) {
  int rc = check_rows_of(t, size, name);
  if (rc) return rc;
  for (int i = 0; i < 3; ++i)
    if (t->shape[i] > 1 && t->stride[i] < t->shape[3]) return fail(KFA_ERR_ARG, "%s: rows overlap", name);
  return KFA_OK;
}

int check_rotary(const KfaRotary* r, int64_t D) {
  if (!r || !r->turns) return fail(KFA_ERR_ARG, "rotary: null");
  if (r->pairs < 1 || 2 * r->pairs > D) return fail(KFA_ERR_ARG, "rotary: %lld pairs: 1 .. %lld, half the head dim", (long long)r->pairs, (long long)(D / 2));
  if (!std::isfinite(r->amplitude)) return fail(KFA_ERR_ARG, "rotary: amplitude %g", r->amplitude);
  return KFA_OK;
}

void fill_stream(kfa::RotaryStream& x, const KfaTensor4* in, const KfaTensor4* out, int size) {
  x.in = static_cast<const uint8_t*>(in->ptr);
  x.in_b = size * in->stride[0], x.in_h = size * in->stride[1], x.in_s = size * in->stride[2];
  if (out) {
    x.out = static_cast<uint8_t*>(out->ptr);
    x.out_b = size * out->stride[0], x.out_h = size * out->stride[1], x.out_s = size * out->stride[2];
  }
}

// The largest piece that `t`'s base, rows and strides are whole numbers of.
int piece_of(const KfaTensor4* t, int size, int piece) {
  if (!t) return piece;
  uint64_t all = reinterpret_cast<uintptr_t>(t->ptr) | static_cast<uint64_t>(t->shape[3] * size);
  for (int i = 0; i < 3; ++i)
    if (t->shape[i] > 1) all |= static_cast<uint64_t>(t->stride[i] * size);
  while (piece > size && all % piece) piece >>= 1;
  return piece;
}

void fill_angles(kfa::RotaryParams& p, const KfaRotary* r, bool inverse) {
  p.turns = reinterpret_cast<const uint64_t*>(r->turns);
  p.pairs = static_cast<int>(r->pairs);
  p.by_pair = kfa::FastDiv::by(p.pairs);
  p.amplitude = r->amplitude;
  p.sine = inverse ? -r->amplitude : r->amplitude;
  p.positions = r->positions;
  p.pos_b = r->position_stride[0];
  p.pos_s = r->position_stride[1];
  p.pos_wide = r->wide_positions != 0;
  p.offset = r->offset;
}

// APPEND: 0: the pass of its own; else into a cache, so many heads a thread.
template <typename T, int BYTES, bool INTERLEAVED, int APPEND>
int launch_pieces(kfa::RotaryParams& p, int64_t batch, int64_t heads, int64_t steps, cudaStream_t s) {
  constexpr int V = BYTES / static_cast<int>(sizeof(T));
  const int cells = (p.columns + 2 * V - 1) / (2 * V);  // of a row (half layout: the turned ones and the others are whole cells up to a last single piece)
  p.pair_cells = (p.pairs + V - 1) / V;
  constexpr int HEADS = APPEND ? APPEND : 1;
  constexpr int64_t PER = kfa::ROT_THREADS * (APPEND ? 1 : kfa::ROT_CELLS);  // cells of a CTA
  const int64_t groups = (heads + HEADS - 1) / HEADS, all_tokens = batch * steps, total = all_tokens * groups * cells;
  if (total > 0xfffff000ll) return fail(KFA_ERR_ARG, "rotary: too many rows in one call");
  p.heads = static_cast<int>(heads);
  p.by_cell = kfa::FastDiv::by(cells);
  p.by_group = kfa::FastDiv::by(static_cast<uint32_t>(groups));
  p.by_step = kfa::FastDiv::by(static_cast<uint32_t>(steps));
  p.total = static_cast<unsigned>(total);
  // tokens that a CTA's stretch of cells can touch
  const int64_t touched = std::min<int64_t>((PER + groups * cells - 2) / (groups * cells) + 1, all_tokens);
  const int smem = static_cast<int>(touched) * p.pair_cells * V * 8;
  const dim3 grid(static_cast<unsigned>((total + PER - 1) / PER));
  if constexpr (APPEND) return launch(kfa::kfa_rotary_append_kernel<T, BYTES, INTERLEAVED, APPEND>, grid, kfa::ROT_THREADS, smem, s, p);
  else return launch(kfa::kfa_rotary_kernel<T, BYTES, INTERLEAVED>, grid, kfa::ROT_THREADS, smem, s, p);
}

template <typename T>
int launch_rotary(kfa::RotaryParams& p, bool interleaved, int piece, int64_t batch, int64_t heads, int64_t steps, cudaStream_t s) {
  if (interleaved) {
    switch (piece) {
      case 16: return launch_pieces<T, 16, true, 0>(p, batch, heads, steps, s);
      case 8: return launch_pieces<T, 8, true, 0>(p, batch, heads, steps, s);
      case 4: return launch_pieces<T, 4, true, 0>(p, batch, heads, steps, s);
      default: return launch_pieces<T, sizeof(T), true, 0>(p, batch, heads, steps, s);
    }
  }
  switch (piece) {
    case 16: return launch_pieces<T, 16, false, 0>(p, batch, heads, steps, s);
    case 8: return launch_pieces<T, 8, false, 0>(p, batch, heads, steps, s);
    case 4: return launch_pieces<T, 4, false, 0>(p, batch, heads, steps, s);
    default: return launch_pieces<T, sizeof(T), false, 0>(p, batch, heads, steps, s);
  }
}

template <typename T, int HEADS>
int launch_append(kfa::RotaryParams& p, bool interleaved, int64_t batch, int64_t heads, int64_t steps, cudaStream_t s) {
  if (interleaved) return launch_pieces<T, 16, true, HEADS>(p, batch, heads, steps, s);  // (tensors and pages: rows of whole 16 bytes)
  int piece = 16;
  while (p.pairs * 2 % piece) piece >>= 1;
  switch (piece) {
    case 16: return launch_pieces<T, 16, false, HEADS>(p, batch, heads, steps, s);
    case 8: return launch_pieces<T, 8, false, HEADS>(p, batch, heads, steps, s);
    case 4: return launch_pieces<T, 4, false, HEADS>(p, batch, heads, steps, s);
    default: return launch_pieces<T, 2, false, HEADS>(p, batch, heads, steps, s);
  }
}
template <typename T>
int launch_append(kfa::RotaryParams& p, bool interleaved, int64_t batch, int64_t heads, int64_t steps, cudaStream_t s) {
  // (one head a thread where that leaves room on the GPU: four CTAs an SM of 32-byte cells)
  const bool few = batch * steps * heads * ((p.columns + 15) / 16) <= 4ll * SMS * kfa::ROT_THREADS;
  return few ? launch_append<T, 1>(p, interleaved, batch, heads, steps, s) : launch_append<T, 3>(p, interleaved, batch, heads, steps, s);
}

}  // namespace

extern "C" {

int kfa_rotary(const KfaTensor4* q, const KfaTensor4* k, const KfaTensor4* q_out, const KfaTensor4* k_out, const KfaRotary* rotary,
               int inverse, int dtype, void* stream) {
  kfa::RotaryParams p;
  std::memset(&p, 0, sizeof(p));
  if (dtype != KFA_F16 && dtype != KFA_BF16 && dtype != KFA_F32) return fail(KFA_ERR_ARG, "dtype %d: KFA_F16, KFA_BF16 or KFA_F32", dtype);
  const int size = dtype == KFA_F32 ? 4 : 2;
  int rc;
  if ((rc = check_rows_of(q, size, "q")) || (rc = check_rows_out(q_out, size, "q_out")) || (rc = check_rotary(rotary, q->shape[3]))) return rc;
  if (q->shape[3] > 1024) return fail(KFA_ERR_ARG, "head_dim %lld: up to 1024", (long long)q->shape[3]);
  if (!k != !k_out) return fail(KFA_ERR_ARG, "k and k_out: both or neither");
  for (int i = 0; i < 4; ++i)
    if (q_out->shape[i] != q->shape[i]) return fail(KFA_ERR_ARG, "q_out: shape differs from q");
  if (k) {
    if ((rc = check_rows_of(k, size, "k")) || (rc = check_rows_out(k_out, size, "k_out"))) return rc;
    for (int i = 0; i < 4; ++i)
      if (k_out->shape[i] != k->shape[i] || (i != 1 && k->shape[i] != q->shape[i])) return fail(KFA_ERR_ARG, "k: batch, tokens and head dim of q");
  }
  fill_angles(p, rotary, inverse != 0);
  fill_stream(p.x[0], q, q_out, size);
  if (k) fill_stream(p.x[1], k, k_out, size);
  const int64_t heads = q->shape[1] + (k ? k->shape[1] : 0);
  if (heads > 0x7fffffff || q->shape[0] * q->shape[2] > 0x7fffffff) return fail(KFA_ERR_ARG, "rotary: too many rows in one call");
  p.q_heads = static_cast<int>(q->shape[1]);
  p.qk_heads = static_cast<int>(heads);
  p.columns = static_cast<int>(q->shape[3]);
  int piece = piece_of(k_out, size, piece_of(q_out, size, piece_of(k, size, piece_of(q, size, 16))));
  while (!rotary->interleaved && piece > size && rotary->pairs * size % piece) piece >>= 1;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool inter = rotary->interleaved != 0;
  if (dtype == KFA_F32) return launch_rotary<float>(p, inter, piece, q->shape[0], heads, q->shape[2], s);
  if (dtype == KFA_BF16) return launch_rotary<__nv_bfloat16>(p, inter, piece, q->shape[0], heads, q->shape[2], s);
  return launch_rotary<__half>(p, inter, piece, q->shape[0], heads, q->shape[2], s);
}

int kfa_cache_append_rotary(const KfaCache* cache, const KfaTensor4* q, const KfaTensor4* k, const KfaTensor4* v, const KfaRows* rows,
                            const KfaRotary* rotary, const KfaTensor4* q_out, const KfaTensor4* k_out, int dtype, int* dev_status,
                            void* stream) {
  kfa::RotaryParams p;
  std::memset(&p, 0, sizeof(p));
  int rc;
  if ((rc = check_dtype(dtype)) || (rc = check_cache(cache, &p.c)) || (rc = check_new(k, p.c, p.c.heads, "k")) || (rc = check_new(v, p.c, p.c.heads, "v")) ||
      (rc = check_rotary(rotary, p.c.cols)))
    return rc;
  if (k->shape[2] != v->shape[2]) return fail(KFA_ERR_ARG, "k, v: different numbers of tokens");
  if ((rc = check_rows(rows, k->shape[2], &p.r))) return rc;
  if (!dev_status) return fail(KFA_ERR_ARG, "dev_status: null pointer");
  if (!q != !q_out) return fail(KFA_ERR_ARG, "q and q_out: both or neither");
  if ((q || k_out) && (rows->index || rows->steps != k->shape[2])) return fail(KFA_ERR_ARG, "q, k_out: only where all the tokens are taken in order");
  const KfaTensor4* pairs[2][2] = {{q, q_out}, {k_out ? k : nullptr, k_out}};
  const char* names[2][2] = {{"q", "q_out"}, {"k", "k_out"}};
  for (int i = 0; i < 2; ++i) {
    if (!pairs[i][0]) continue;
    if ((rc = check_new(pairs[i][0], p.c, i ? p.c.heads : 0, names[i][0])) || (rc = check_new(pairs[i][1], p.c, i ? p.c.heads : 0, names[i][1])) ||
        (rc = check_rows_out(pairs[i][1], 2, names[i][1])))
      return rc;
    for (int j = 0; j < 4; ++j)
      if (pairs[i][0]->shape[j] != pairs[i][1]->shape[j]) return fail(KFA_ERR_ARG, "%s: shape differs", names[i][1]);
    if (pairs[i][0]->shape[2] != k->shape[2]) return fail(KFA_ERR_ARG, "q: as many tokens as k");
  }
  fill_angles(p, rotary, false);
  if (q) fill_stream(p.x[0], q, q_out, 2);
  fill_stream(p.x[1], k, k_out, 2);
  fill_stream(p.x[2], v, nullptr, 2);
  p.q_heads = q ? static_cast<int>(q->shape[1]) : 0;
  p.qk_heads = p.q_heads + p.c.heads;
  p.columns = p.c.cols;
  p.status = dev_status;
  const int64_t heads = p.qk_heads + static_cast<int64_t>(p.c.heads);
  if (static_cast<int64_t>(p.c.batch) * p.r.steps > 0x7fffffff) return fail(KFA_ERR_ARG, "rotary: too many rows in one call");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == KFA_BF16) return launch_append<__nv_bfloat16>(p, rotary->interleaved != 0, p.c.batch, heads, p.r.steps, s);
  return launch_append<__half>(p, rotary->interleaved != 0, p.c.batch, heads, p.r.steps, s);
}

}  // extern "C"
