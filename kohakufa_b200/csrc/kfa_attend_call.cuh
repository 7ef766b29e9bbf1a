// What the C entry points of attention over a cache share: how a call is cut up, its checks, parameters and launches. For the sources of
// libkfa.so only.
#pragma once

#include "kfa_attend.cuh"
#include "kfa_cache_call.cuh"

namespace {

// How an attention call is cut up: a function of the shapes alone, so that the scratch it needs is known beforehand.
struct AttendPlan {
  int rows, tile_rows, gt, tt, head_tiles, row_tiles, grid, extra, least;
  bool whole;
  int64_t most_units, meta_bytes, ml_bytes, bytes;
};

AttendPlan plan_attend(int64_t batch, int64_t heads, int64_t kv_heads, int64_t T, int64_t capacity, bool fresh) {
  AttendPlan a;
  const int64_t group = heads / kv_heads;
  // Rows that share a K / V head, up to 256 of them in a tile: whole groups of heads, the tokens in equal parts.
  const int64_t gt = std::min<int64_t>(group, 256), most = 256 / gt;
  const int64_t token_tiles = (T + most - 1) / most;
  const int64_t tt = (T + token_tiles - 1) / token_tiles;
  a.gt = static_cast<int>(gt);
  a.tt = static_cast<int>(tt);
  a.head_tiles = static_cast<int>((group + gt - 1) / gt);
  a.row_tiles = static_cast<int>(a.head_tiles * ((T + tt - 1) / tt));
  a.tile_rows = static_cast<int>(gt * tt);
  a.rows = gt * tt <= 16 ? 16 : (gt * tt <= 32 ? 32 : (gt * tt <= 64 ? 64 : (gt * tt <= 128 ? 128 : 256)));
  const int64_t items = batch * kv_heads * a.row_tiles;
  const int64_t units = std::max<int64_t>((capacity + 31) / 32 + (fresh ? (T + 31) / 32 : 0), 1);
  a.whole = units <= 8;
  // What an item's beginning and end take, in units of 32 keys. Graph time per call in us with 8, 10, 12, 14: 64 sequences of 1 to 4096 positions,
  // one token each (D = 128) 104.6, 100.0, 98.6, 99.5; 32 x 12 heads over 0 to 1500 (D = 80) 34.8, 32.4, 30.2, 29.6; 8 sequences of 300 to 2048,
  // 7 tokens (D = 64) 15.4, 14.3, 14.1, 14.2. With 10, 13, 16, 20: 16 sequences of 2048 to 4096, 256 rows 94.1, 94.3, 93.7, 93.7.
  a.extra = a.rows > 64 ? 16 : 12;
  a.least = 4;
  a.most_units = items * (units + a.extra);
  a.grid = static_cast<int>(std::min<int64_t>(SMS, a.whole ? items : (items * units + 3) / 4));
  a.meta_bytes = a.ml_bytes = a.bytes = 0;
  if (!a.whole) {
    a.meta_bytes = (16 * a.grid + 255) / 256 * 256;
    a.ml_bytes = 2ll * a.grid * 3 * a.rows * 4;
    a.bytes = a.meta_bytes + a.ml_bytes + 2ll * a.grid * a.rows * 128 * 4;
  }
  return a;
}

template <bool BF16, class R, typename K>
int launch_attend(K kern, const CUtensorMap (&m)[5], const kfa::AttendParams& p, const AttendPlan& plan, cudaStream_t s) {
  static std::atomic<uint64_t> allowed{0};
  int rc = allow_smem(allowed, reinterpret_cast<const void*>(kern), R::SMEM);
  if (rc) return rc;
  if ((rc = launch(kern, dim3(plan.grid), kfa::ATT_THREADS, R::SMEM, s, m[0], m[1], m[2], m[3], m[4], p)) || plan.whole) return rc;
  if (plan.rows > 64) return launch(kfa::kfa_cache_join_rows_kernel<BF16>, dim3(plan.grid, (plan.tile_rows + 31) / 32), 256, 0, s, p);
  return launch(kfa::kfa_cache_join_kernel<BF16>, dim3(plan.grid, (plan.tile_rows + 7) / 8), 256, 0, s, p);
}

template <int NC, bool BF16>
int launch_attend_rows(const CUtensorMap (&m)[5], const kfa::AttendParams& p, const AttendPlan& plan, cudaStream_t s) {
  switch (plan.rows) {
    case 16: return launch_attend<BF16, kfa::AttCfg<NC, 16>>(kfa::kfa_cache_attend_kernel<NC, 16, BF16>, m, p, plan, s);
    case 32: return launch_attend<BF16, kfa::AttCfg<NC, 32>>(kfa::kfa_cache_attend_kernel<NC, 32, BF16>, m, p, plan, s);
    case 64: return launch_attend<BF16, kfa::AttCfg<NC, 64>>(kfa::kfa_cache_attend_kernel<NC, 64, BF16>, m, p, plan, s);
    case 128: return launch_attend<BF16, kfa::AttRowsCfg<NC, 1>>(kfa::kfa_cache_attend_rows_kernel<NC, 1, BF16>, m, p, plan, s);
    default: return launch_attend<BF16, kfa::AttRowsCfg<NC, 2>>(kfa::kfa_cache_attend_rows_kernel<NC, 2, BF16>, m, p, plan, s);
  }
}

int launch_attend_call(const CUtensorMap (&m)[5], const kfa::AttendParams& p, const AttendPlan& plan, int dtype, cudaStream_t s) {
  if (dtype == KFA_BF16) return p.c.cols > 64 ? launch_attend_rows<2, true>(m, p, plan, s) : launch_attend_rows<1, true>(m, p, plan, s);
  return p.c.cols > 64 ? launch_attend_rows<2, false>(m, p, plan, s) : launch_attend_rows<1, false>(m, p, plan, s);
}

// What a plan's rows, items and scratch are, in the kernels' parameters.
void fill_plan(kfa::AttendParams& p, const AttendPlan& plan, void* scratch) {
  p.gt = plan.gt;
  p.tt = plan.tt;
  p.head_tiles = plan.head_tiles;
  p.row_tiles = plan.row_tiles;
  p.items = p.c.heads * plan.row_tiles;
  p.by_gt = kfa::FastDiv::by(p.gt);
  p.by_items = kfa::FastDiv::by(p.items);
  p.by_row_tiles = kfa::FastDiv::by(p.row_tiles);
  p.by_head_tiles = kfa::FastDiv::by(p.head_tiles);
  p.by_grid = kfa::FastDiv::by(plan.grid);
  p.whole = plan.whole;
  p.least = plan.least;
  p.extra = plan.extra;
  p.rows = plan.rows;
  p.box = page_box(p.c);
  if (!plan.whole) {
    uint8_t* at = static_cast<uint8_t*>(scratch);
    p.part_meta = reinterpret_cast<int4*>(at);
    p.part_ml = reinterpret_cast<float*>(at + plan.meta_bytes);
    p.part_o = reinterpret_cast<float*>(at + plan.meta_bytes + plan.ml_bytes);
  }
}

int pages_map(const KfaTensor4* t, const kfa::AttendParams& p, int dtype, CUtensorMap* map, const char* name) {
  return make_box_map(t->ptr, p.c.cols, t->shape[2], t->stride[2], t->shape[1], t->stride[1], t->shape[0], t->stride[0], p.box, 1, 1, dtype, map, name);
}

// Rows of new tokens' keys or values, in boxes of a unit.
int new_map(const KfaTensor4* t, const kfa::AttendParams& p, int dtype, CUtensorMap* map, const char* name) {
  return make_box_map(t->ptr, p.c.cols, p.T, t->stride[2], p.c.heads, t->stride[1], p.c.batch, t->stride[0], kfa::ATT_UNIT, 1, 1, dtype, map, name);
}

// The checks of an attention call to a cache, and the parameters that do not depend on how it is cut up.
int check_attend(const KfaTensor4* q, const KfaCache* cache, const KfaTensor4* k, const KfaTensor4* v, const uint8_t* tree,
                 const int64_t* tree_stride, const int32_t* counts, const KfaTensor4* out, float* stats, float scale, int dtype,
                 int* dev_status, kfa::AttendParams& p) {
  std::memset(&p, 0, sizeof(p));
  int rc;
  if ((rc = check_cache(cache, &p.c)) || (rc = check_new(q, p.c, 0, "q")) || (rc = check_new(out, p.c, 0, "out")) ||
      (rc = check_scale(scale)) || (rc = check_dtype(dtype)))
    return rc;
  for (int i = 0; i < 4; ++i)
    if (out->shape[i] != q->shape[i]) return fail(KFA_ERR_ARG, "out: shape differs from q");
  if (!k != !v) return fail(KFA_ERR_ARG, "k and v: both or neither");
  if (tree && (!k || !tree_stride)) return fail(KFA_ERR_ARG, "tree: needs k, v and its strides");
  if (!dev_status) return fail(KFA_ERR_ARG, "dev_status: null pointer");
  if (k) {
    if ((rc = check_new(k, p.c, p.c.heads, "k")) || (rc = check_new(v, p.c, p.c.heads, "v"))) return rc;
    if (k->shape[2] != q->shape[2] || v->shape[2] != q->shape[2]) return fail(KFA_ERR_ARG, "k, v: as many new tokens as q");
    p.k = static_cast<const uint8_t*>(k->ptr);
    p.v = static_cast<const uint8_t*>(v->ptr);
    p.v_sb = 2 * v->stride[0], p.v_sh = 2 * v->stride[1], p.v_ss = 2 * v->stride[2];
  }
  p.o = static_cast<uint8_t*>(out->ptr);
  p.o_sb = 2 * out->stride[0], p.o_sh = 2 * out->stride[1], p.o_ss = 2 * out->stride[2];
  p.tree = tree;
  if (tree) p.tree_sb = tree_stride[0], p.tree_st = tree_stride[1], p.tree_sj = tree_stride[2];
  p.counts = counts;
  p.stats = stats;
  p.H = static_cast<int>(q->shape[1]);
  p.T = static_cast<int>(q->shape[2]);
  p.group = p.H / p.c.heads;
  // (a scale of 0 makes all scores equal: so does this one, and hidden scores of -inf stay what they are)
  p.c_log2 = std::max(scale * LOG2E, 1e-30f);
  p.slack = 8.f / p.c_log2;
  p.status = dev_status;
  return KFA_OK;
}

// The same with its plan and tensor maps.
int prepare_attend(const KfaTensor4* q, const KfaCache* cache, const KfaTensor4* k, const KfaTensor4* v, const uint8_t* tree,
                   const int64_t* tree_stride, const int32_t* counts, const KfaTensor4* out, float* stats, void* scratch, float scale, int dtype,
                   int* dev_status, kfa::AttendParams& p, AttendPlan& plan, CUtensorMap (&m)[5]) {
  int rc = check_attend(q, cache, k, v, tree, tree_stride, counts, out, stats, scale, dtype, dev_status, p);
  if (rc) return rc;
  plan = plan_attend(p.c.batch, p.H, p.c.heads, p.T, p.c.capacity, k != nullptr);
  if (plan.most_units > 0x3fffffff) return fail(KFA_ERR_ARG, "too many rows in one call");
  if (plan.bytes && (!scratch || reinterpret_cast<uintptr_t>(scratch) % 16)) return fail(KFA_ERR_ARG, "scratch: null or not 16-byte aligned");
  fill_plan(p, plan, scratch);
  const int64_t D = p.c.cols;
  if ((rc = make_box_map(q->ptr, D, p.H, q->stride[1], p.T, q->stride[2], p.c.batch, q->stride[0], p.gt, p.tt, 1, dtype, &m[0], "q")) ||
      (rc = pages_map(&cache->k, p, dtype, &m[1], "cache keys")) || (rc = pages_map(&cache->v, p, dtype, &m[2], "cache values")))
    return rc;
  m[3] = m[1];
  m[4] = m[2];
  if (k && ((rc = new_map(k, p, dtype, &m[3], "k")) || (rc = new_map(v, p, dtype, &m[4], "v")))) return rc;
  return KFA_OK;
}

}  // namespace
