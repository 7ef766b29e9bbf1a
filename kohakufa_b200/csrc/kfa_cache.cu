// C ABI of the operators on a cache of keys and values (declared in include/kfa.h): argument checks and launches.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>

#include "kfa_attend.cuh"
#include "kfa_cache.cuh"
#include "kfa_call.cuh"
#include "kfa_weigh.cuh"

namespace {

constexpr float LOG2E = 1.4426950408889634f;

int check_dim(int64_t D) {
  if (D < 8 || D > 128 || D % 8) return fail(KFA_ERR_ARG, "head_dim %lld: a multiple of 8 up to 128", (long long)D);
  return KFA_OK;
}

int check_cache(const KfaCache* c, kfa::CacheView* view, const char* name = "cache") {
  if (!c || !c->lengths) return fail(KFA_ERR_ARG, "%s: null", name);
  int rc;
  if ((rc = check_tensor(&c->k, "cache keys")) || (rc = check_tensor(&c->v, "cache values")) || (rc = check_dim(c->k.shape[3]))) return rc;
  for (int i = 0; i < 4; ++i)
    if (c->k.shape[i] != c->v.shape[i]) return fail(KFA_ERR_ARG, "%s: pages of keys and values differ in shape", name);
  if (c->batch < 1 || c->batch > 65535) return fail(KFA_ERR_ARG, "%s: batch %lld: 1 .. 65535", name, (long long)c->batch);
  const int64_t pages = c->k.shape[0], heads = c->k.shape[1], page = c->k.shape[2];
  if (heads > 65535) return fail(KFA_ERR_ARG, "%s: K / V heads %lld: up to 65535", name, (long long)heads);
  if (c->table) {
    if (page % 8) return fail(KFA_ERR_ARG, "%s: pages of %lld positions: a multiple of 8", name, (long long)page);
    if (c->table_cols < 1 || c->table_stride < 0) return fail(KFA_ERR_ARG, "%s: empty table", name);
  } else if (pages != c->batch) {
    return fail(KFA_ERR_ARG, "%s: without a table page b is sequence b's: %lld pages for a batch of %lld", name, (long long)pages,
                (long long)c->batch);
  }
  const int64_t capacity = c->table ? c->table_cols * page : page;
  if (capacity > 0x7fff0000) return fail(KFA_ERR_ARG, "%s: capacity above 2^31 positions", name);
  view->k = static_cast<uint8_t*>(c->k.ptr);
  view->v = static_cast<uint8_t*>(c->v.ptr);
  view->k_sn = 2 * c->k.stride[0];
  view->k_sh = 2 * c->k.stride[1];
  view->k_ss = 2 * c->k.stride[2];
  view->v_sn = 2 * c->v.stride[0];
  view->v_sh = 2 * c->v.stride[1];
  view->v_ss = 2 * c->v.stride[2];
  view->table = c->table;
  view->table_stride = c->table_stride;
  view->lengths = c->lengths;
  view->page = static_cast<int>(page);
  view->by_page = kfa::FastDiv::by(static_cast<uint32_t>(page));
  view->n_pages = static_cast<int>(pages);
  view->capacity = static_cast<int>(capacity);
  view->batch = static_cast<int>(c->batch);
  view->heads = static_cast<int>(heads);
  view->cols = static_cast<int>(c->k.shape[3]);
  return KFA_OK;
}

// New tokens' keys and values, or queries (heads: how many, 0 for any multiple): [B, heads, T, D] as the cache has it.
int check_new(const KfaTensor4* t, const kfa::CacheView& c, int heads, const char* name) {
  int rc = check_tensor(t, name);
  if (rc) return rc;
  if (t->shape[0] != c.batch || t->shape[3] != c.cols || (heads ? t->shape[1] != heads : t->shape[1] % c.heads != 0))
    return fail(KFA_ERR_ARG, "%s: [%lld, %lld, %lld, %lld] does not fit the cache's batch %d, %d heads, head dim %d", name,
                (long long)t->shape[0], (long long)t->shape[1], (long long)t->shape[2], (long long)t->shape[3], c.batch, c.heads, c.cols);
  return KFA_OK;
}

int check_rows(const KfaRows* r, int64_t T, kfa::RowsView* view) {
  if (!r || r->steps < 1 || r->steps > 0x7fffffff || (!r->index && r->steps > T) || (r->index && r->index_stride < 0))
    return fail(KFA_ERR_ARG, "rows: 1 .. T of them, or an index");
  *view = {r->index, r->index_stride, r->counts, static_cast<int>(r->steps), static_cast<int>(T)};
  return KFA_OK;
}

int check_scale(float scale) {
  return std::isfinite(scale) && scale >= 0.f ? KFA_OK : fail(KFA_ERR_ARG, "scale %g: finite, not negative", scale);
}

int check_dtype(int dtype) {
  return dtype == KFA_F16 || dtype == KFA_BF16 ? KFA_OK : fail(KFA_ERR_ARG, "dtype %d: KFA_F16 or KFA_BF16", dtype);
}

// 4-D tiled map over rows of D 16-bit columns: dims (D, n1, n2, n3) with element strides s1, s2, s3, boxes of 64 columns (128 bytes,
// swizzled) x b1 x b2; what is out of range reads as zeros.
int make_box_map(void* ptr, int64_t D, int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t n3, int64_t s3, int b1, int b2, int dtype,
                 CUtensorMap* map, const char* name) {
  EncodeFn enc = encode_fn();
  if (!enc) return fail(KFA_ERR_CUDA, "cuTensorMapEncodeTiled not available from the driver");
  auto st = [&](int64_t n, int64_t s) { return static_cast<cuuint64_t>(n > 1 ? s : D) * 2; };  // (an extent of 1 never advances)
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(n1), static_cast<cuuint64_t>(n2), static_cast<cuuint64_t>(n3)};
  const cuuint64_t strides[3] = {st(n1, s1), st(n2, s2), st(n3, s3)};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(b1), static_cast<cuuint32_t>(b2), 1}, one[4] = {1, 1, 1, 1};
  const CUresult r = enc(map, dtype == KFA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, ptr, dims, strides, box,
                         one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(KFA_ERR_CUDA, "cuTensorMapEncodeTiled(%s) failed with CUresult %d", name, static_cast<int>(r));
  return KFA_OK;
}

constexpr int SMS = 148;  // (what this library is built for)

// A kernel's dynamic shared memory is allowed once per device (the runtime call costs a small problem's launch about as much as its checks).
// done: the kernel's own, a bit per device.
int allow_smem(std::atomic<uint64_t>& done, const void* kern, int bytes) {
  int dev = 0;
  KFA_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return KFA_OK;
  KFA_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done.fetch_or(bit, std::memory_order_relaxed);
  return KFA_OK;
}

// How an attention call is cut up: a function of the shapes alone, so that the scratch it needs is known beforehand.
struct AttendPlan {
  int rows, gt, tt, head_tiles, row_tiles, grid, extra, least;
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

// A launch that need not wait for the kernel before it in the stream to end: the kernels here wait for that themselves, behind what they
// set up first. (One call after the other: decoding of a short sequence 7.5 -> 6.3 us,
// drafts of 7 tokens 15.4 -> 15.2.)
template <typename... P>
int launch(void (*kern)(P...), dim3 grid, int threads, int smem, cudaStream_t s, const P&... params) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = s;
  cudaLaunchAttribute early[1];
  early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = early;
  config.numAttrs = 1;
  KFA_CUDA(cudaLaunchKernelEx(&config, kern, params...));
  return KFA_OK;
}

template <bool BF16, class R, typename K>
int launch_attend(K kern, const CUtensorMap (&m)[5], const kfa::AttendParams& p, const AttendPlan& plan, cudaStream_t s) {
  static std::atomic<uint64_t> allowed{0};
  int rc = allow_smem(allowed, reinterpret_cast<const void*>(kern), R::SMEM);
  if (rc) return rc;
  if ((rc = launch(kern, dim3(plan.grid), kfa::ATT_THREADS, R::SMEM, s, m[0], m[1], m[2], m[3], m[4], p)) || plan.whole) return rc;
  if (plan.rows > 64) return launch(kfa::kfa_cache_join_rows_kernel<BF16>, dim3(plan.grid, (plan.gt * plan.tt + 31) / 32), 256, 0, s, p);
  return launch(kfa::kfa_cache_join_kernel<BF16>, dim3(plan.grid, (plan.gt * plan.tt + 7) / 8), 256, 0, s, p);
}

// Rows of a TMA box that a page holds whole numbers of (without a table: the last box may end behind the page, and reads zeros there).
int page_box(const kfa::CacheView& c) { return c.table ? (c.page % 32 == 0 ? 32 : (c.page % 16 == 0 ? 16 : 8)) : 32; }

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

struct WeighPlan {
  int64_t rows, work, bytes, meta_floats, part_floats, stats_floats;
  int grid, least, extra, tile_h, tile_t;
};

WeighPlan plan_weigh(int64_t batch, int64_t heads, int64_t kv_heads, int64_t steps, int64_t capacity, int64_t D, bool index) {
  WeighPlan w;
  std::memset(&w, 0, sizeof(w));
  const int64_t group = heads / kv_heads;
  w.rows = std::min<int64_t>(group * steps, 1 << 30);
  if (w.rows <= 64) {
    const int64_t units = (capacity + 31) / 32;
    // (See plan_attend. us with 0, 4, 8, 16: 64 x 8 heads over 1 to 4096 positions 64, 58, 54, 53; 32 x 12 over 0 to 900 25, 15, 11.8, 10.5; 16 x 8
    // over 300 to 4096 with 5 tokens 21.1, 20.8, 21.7, 23.5.)
    w.extra = 8;
    w.least = 4;
    w.work = batch * kv_heads * (units + w.extra);
    w.grid = static_cast<int>(std::min<int64_t>(SMS, (batch * kv_heads * units + 3) / 4));
    return w;
  }
  // Whole tokens a tile: with a group that is no power of two some of the 128 rows do not exist, the tile takes two numbers a row and there are more
  // of them. 4096 tokens, 8 K / V heads, D = 128, us with groups of 3, 4, 5, 6, 7, 8 heads: 142, 109, 206, 238, 271, 204.
  w.tile_h = static_cast<int>(std::min<int64_t>(group, 128));
  w.tile_t = 128 / w.tile_h;
  w.least = 1;
  const int64_t blocks = (steps + kfa::WEIGH_BLOCK - 1) / kfa::WEIGH_BLOCK;
  w.work = batch * kv_heads * blocks * ((capacity + 127) / 128);
  w.grid = static_cast<int>(std::min<int64_t>(2 * SMS, w.work));
  w.meta_floats = (4 * w.grid + 63) / 64 * 64;
  w.part_floats = 2ll * w.grid * 128;
  if (index) w.stats_floats = (2 * batch * heads * steps + 63) / 64 * 64;
  w.bytes = 4 * (w.meta_floats + w.part_floats + w.stats_floats) + (index ? 2 * batch * heads * steps * D : 0);
  return w;
}

template <bool BF16, class R, typename K>
int launch_weigh_few(K kern, const CUtensorMap& mk, const kfa::AttendParams& a, const kfa::WeighParams& p, const WeighPlan& plan, cudaStream_t s) {
  static std::atomic<uint64_t> allowed{0};
  int rc = allow_smem(allowed, reinterpret_cast<const void*>(kern), R::SMEM);
  if (rc) return rc;
  return launch(kern, dim3(plan.grid), kfa::ATT_THREADS, R::SMEM, s, mk, a, p);
}
template <int NC, bool BF16>
int launch_weigh_few(const CUtensorMap& mk, const kfa::AttendParams& a, const kfa::WeighParams& p, const WeighPlan& plan, cudaStream_t s) {
  if (plan.rows <= 16) return launch_weigh_few<BF16, kfa::WeighCfg<NC, 16>>(kfa::kfa_cache_weigh_kernel<NC, 16, BF16>, mk, a, p, plan, s);
  if (plan.rows <= 32) return launch_weigh_few<BF16, kfa::WeighCfg<NC, 32>>(kfa::kfa_cache_weigh_kernel<NC, 32, BF16>, mk, a, p, plan, s);
  return launch_weigh_few<BF16, kfa::WeighCfg<NC, 64>>(kfa::kfa_cache_weigh_kernel<NC, 64, BF16>, mk, a, p, plan, s);
}

template <int NC, bool BF16>
int launch_weigh_many(const CUtensorMap& mq, const CUtensorMap& mk, const kfa::AttendParams& a, const kfa::WeighParams& p, const WeighPlan& plan,
                      cudaStream_t s) {
  using R = kfa::WeighRowsCfg<NC>;
  auto kern = kfa::kfa_cache_weigh_rows_kernel<NC, BF16>;
  static std::atomic<uint64_t> allowed{0};
  int rc = allow_smem(allowed, reinterpret_cast<const void*>(kern), R::SMEM);
  if (rc) return rc;
  if ((rc = launch(kern, dim3(plan.grid), kfa::ATT_THREADS, R::SMEM, s, mq, mk, a, p))) return rc;
  return launch(kfa::kfa_cache_join_weights_kernel, dim3(plan.grid + a.c.batch), 256, 0, s, a, p, plan.grid);
}

}  // namespace

extern "C" {

int64_t kfa_cache_attend_bytes(const KfaTensor4* q, const KfaCache* cache, const KfaTensor4* k) {
  if (!q || !cache) return 0;
  const int64_t page = cache->k.shape[2], kv_heads = cache->k.shape[1];
  if (q->shape[0] < 1 || q->shape[1] < 1 || q->shape[2] < 1 || kv_heads < 1 || q->shape[1] < kv_heads || page < 1) return 0;  // (refused by the call)
  return plan_attend(q->shape[0], q->shape[1], kv_heads, q->shape[2], cache->table ? cache->table_cols * page : page, k != nullptr).bytes;
}

int kfa_cache_attend(const KfaTensor4* q, const KfaCache* cache, const KfaTensor4* k, const KfaTensor4* v, const uint8_t* tree,
                     const int64_t* tree_stride, const int32_t* counts, const KfaTensor4* out, float* stats, void* scratch,
                     float scale, int dtype, int* dev_status, void* stream) {
  kfa::AttendParams p;
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
  const AttendPlan plan = plan_attend(p.c.batch, p.H, p.c.heads, p.T, p.c.capacity, k != nullptr);
  if (plan.most_units > 0x3fffffff) return fail(KFA_ERR_ARG, "too many rows in one call");
  if (plan.bytes && (!scratch || reinterpret_cast<uintptr_t>(scratch) % 16)) return fail(KFA_ERR_ARG, "scratch: null or not 16-byte aligned");
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
  CUtensorMap m[5];
  const KfaTensor4 *ck = &cache->k, *cv = &cache->v;
  const int64_t D = p.c.cols;
  auto pages = [&](const KfaTensor4* t, CUtensorMap* map, const char* name) {
    return make_box_map(t->ptr, D, t->shape[2], t->stride[2], t->shape[1], t->stride[1], t->shape[0], t->stride[0], p.box, 1, dtype, map, name);
  };
  if ((rc = make_box_map(q->ptr, D, p.H, q->stride[1], p.T, q->stride[2], p.c.batch, q->stride[0], p.gt, p.tt, dtype, &m[0], "q")) ||
      (rc = pages(ck, &m[1], "cache keys")) || (rc = pages(cv, &m[2], "cache values")))
    return rc;
  m[3] = m[1];
  m[4] = m[2];
  auto fresh = [&](const KfaTensor4* t, CUtensorMap* map, const char* name) {
    return make_box_map(t->ptr, D, p.T, t->stride[2], p.c.heads, t->stride[1], p.c.batch, t->stride[0], kfa::ATT_UNIT, 1, dtype, map, name);
  };
  if (k && ((rc = fresh(k, &m[3], "k")) || (rc = fresh(v, &m[4], "v")))) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == KFA_BF16) return D > 64 ? launch_attend_rows<2, true>(m, p, plan, s) : launch_attend_rows<1, true>(m, p, plan, s);
  return D > 64 ? launch_attend_rows<2, false>(m, p, plan, s) : launch_attend_rows<1, false>(m, p, plan, s);
}

int kfa_cache_append(const KfaCache* cache, const KfaTensor4* k, const KfaTensor4* v, const KfaRows* rows, int* dev_status,
                     void* stream) {
  kfa::AppendParams p;
  std::memset(&p, 0, sizeof(p));
  int rc;
  if ((rc = check_cache(cache, &p.c)) || (rc = check_new(k, p.c, p.c.heads, "k")) || (rc = check_new(v, p.c, p.c.heads, "v"))) return rc;
  if (k->shape[2] != v->shape[2]) return fail(KFA_ERR_ARG, "k, v: different numbers of tokens");
  if ((rc = check_rows(rows, k->shape[2], &p.r))) return rc;
  if (!dev_status) return fail(KFA_ERR_ARG, "dev_status: null pointer");
  p.k = static_cast<const uint8_t*>(k->ptr);
  p.v = static_cast<const uint8_t*>(v->ptr);
  p.k_sb = 2 * k->stride[0], p.k_sh = 2 * k->stride[1], p.k_ss = 2 * k->stride[2];
  p.v_sb = 2 * v->stride[0], p.v_sh = 2 * v->stride[1], p.v_ss = 2 * v->stride[2];
  const long long total = static_cast<long long>(p.c.batch) * p.r.steps * p.c.heads * (p.c.cols / 8);
  if (total > 0xffffff00ll) return fail(KFA_ERR_ARG, "kfa_cache_append: more than 64 GB in one call");
  p.by_piece = kfa::FastDiv::by(p.c.cols / 8);
  p.by_head = kfa::FastDiv::by(p.c.heads);
  p.by_step = kfa::FastDiv::by(p.r.steps);
  p.total = static_cast<unsigned>(total);
  p.status = dev_status;
  return launch(kfa::kfa_cache_append_kernel, dim3(static_cast<unsigned>((total + 255) / 256)), 256, 0, static_cast<cudaStream_t>(stream), p);
}

int64_t kfa_cache_weigh_bytes(const KfaTensor4* q, const KfaCache* cache, const KfaRows* rows) {
  if (!q || !cache || !rows) return 0;
  const int64_t page = cache->k.shape[2], kv_heads = cache->k.shape[1];
  if (q->shape[1] < kv_heads || kv_heads < 1 || rows->steps < 1) return 0;  // (refused by the call)
  return plan_weigh(cache->batch, q->shape[1], kv_heads, rows->steps, cache->table ? cache->table_cols * page : page, cache->k.shape[3],
                    rows->index != nullptr)
      .bytes;
}

int kfa_cache_weigh(const KfaTensor4* q, const float* stats, const KfaCache* cache, const KfaRows* rows, float* weights,
                    const int64_t* weights_stride, int64_t room, int add, void* scratch, float scale, int dtype, int* dev_status,
                    void* stream) {
  kfa::AttendParams a;
  kfa::WeighParams p;
  std::memset(&a, 0, sizeof(a));
  std::memset(&p, 0, sizeof(p));
  int rc;
  if ((rc = check_cache(cache, &a.c)) || (rc = check_new(q, a.c, 0, "q")) || (rc = check_rows(rows, q->shape[2], &p.r)) ||
      (rc = check_scale(scale)) || (rc = check_dtype(dtype)))
    return rc;
  if (!stats || !weights || !weights_stride || !dev_status) return fail(KFA_ERR_ARG, "kfa_cache_weigh: null pointer");
  if (room < a.c.capacity || room > 0x7fff0000) return fail(KFA_ERR_ARG, "weights: at least the cache's %d positions", a.c.capacity);
  const int64_t D = a.c.cols;
  a.H = static_cast<int>(q->shape[1]);
  a.group = a.H / a.c.heads;
  a.T = p.r.steps;
  a.counts = p.r.counts;
  a.appended = 1;
  a.c_log2 = std::max(scale * LOG2E, 1e-30f);  // (see kfa_cache_attend)
  a.status = dev_status;
  a.row_tiles = a.head_tiles = 1;
  a.items = a.c.heads;
  a.gt = a.group;
  a.by_gt = kfa::FastDiv::by(a.gt);
  a.by_items = kfa::FastDiv::by(a.items);
  a.by_row_tiles = a.by_head_tiles = kfa::FastDiv::by(1);
  a.box = page_box(a.c);
  p.q = static_cast<const uint8_t*>(q->ptr);
  p.q_sb = 2 * q->stride[0], p.q_sh = 2 * q->stride[1], p.q_ss = 2 * q->stride[2];
  p.stats = stats;
  p.w = weights;
  p.w_sb = weights_stride[0];
  p.w_sh = weights_stride[1];
  p.room = static_cast<int>(room);
  p.add = add != 0;
  p.by_piece = kfa::FastDiv::by(static_cast<uint32_t>(D / 8));
  const WeighPlan plan = plan_weigh(a.c.batch, a.H, a.c.heads, p.r.steps, a.c.capacity, D, p.r.index != nullptr);
  if (plan.work > 0x3fffffff) return fail(KFA_ERR_ARG, "too many rows in one call");
  if (plan.bytes && (!scratch || reinterpret_cast<uintptr_t>(scratch) % 16)) return fail(KFA_ERR_ARG, "scratch: null or not 16-byte aligned");
  a.by_grid = kfa::FastDiv::by(plan.grid);
  a.least = plan.least;
  a.extra = plan.extra;
  CUtensorMap mk, mq;
  const KfaTensor4* ck = &cache->k;
  if ((rc = make_box_map(ck->ptr, D, ck->shape[2], ck->stride[2], ck->shape[1], ck->stride[1], ck->shape[0], ck->stride[0], a.box, 1, dtype, &mk,
                         "cache keys")))
    return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (plan.rows <= 64) {
    if (dtype == KFA_BF16) return D > 64 ? launch_weigh_few<2, true>(mk, a, p, plan, s) : launch_weigh_few<1, true>(mk, a, p, plan, s);
    return D > 64 ? launch_weigh_few<2, false>(mk, a, p, plan, s) : launch_weigh_few<1, false>(mk, a, p, plan, s);
  }
  p.tile_h = plan.tile_h;
  p.tile_t = plan.tile_t;
  p.head_tiles = (a.group + p.tile_h - 1) / p.tile_h;
  p.by_tile_h = kfa::FastDiv::by(p.tile_h);
  p.by_tile_t = kfa::FastDiv::by(p.tile_t);
  p.part_meta = static_cast<int4*>(scratch);
  p.part = static_cast<float*>(scratch) + plan.meta_floats;
  KfaTensor4 rows_q = *q;
  if (p.r.index) {
    p.stats_to = p.part + plan.part_floats;
    p.q_to = reinterpret_cast<uint8_t*>(p.stats_to + plan.stats_floats);
    const int64_t total = static_cast<int64_t>(a.c.batch) * p.r.steps * a.H * (D / 8);
    if (total > 0xffffff00ll) return fail(KFA_ERR_ARG, "too many rows in one call");
    if ((rc = launch(kfa::kfa_cache_take_rows_kernel, dim3(static_cast<unsigned>((total + 255) / 256)), 256, 0, s, a, p, p.by_piece,
                     kfa::FastDiv::by(a.H), kfa::FastDiv::by(p.r.steps), static_cast<unsigned>(total))))
      return rc;
    rows_q.ptr = p.q_to;
    rows_q.shape[2] = p.r.steps;
    rows_q.stride[2] = a.H * D;
    rows_q.stride[1] = D;
    rows_q.stride[0] = static_cast<int64_t>(p.r.steps) * a.H * D;
    p.stats = p.stats_to;
    p.r.index = nullptr;
    p.r.T = p.r.steps;
  }
  if ((rc = make_box_map(rows_q.ptr, D, a.H, rows_q.stride[1], rows_q.shape[2], rows_q.stride[2], a.c.batch, rows_q.stride[0], p.tile_h, p.tile_t,
                         dtype, &mq, "q")))
    return rc;
  if (dtype == KFA_BF16) return D > 64 ? launch_weigh_many<2, true>(mq, mk, a, p, plan, s) : launch_weigh_many<1, true>(mq, mk, a, p, plan, s);
  return D > 64 ? launch_weigh_many<2, false>(mq, mk, a, p, plan, s) : launch_weigh_many<1, false>(mq, mk, a, p, plan, s);
}

int kfa_cache_evict(const KfaCache* cache, const float* weights, const int64_t* weights_stride, int64_t keep, int64_t recent,
                    const KfaCache* out, float* weights_out, int32_t* kept, int32_t* lengths_out, int clear, int* dev_status,
                    void* stream) {
  return kfa_cache_evict_room(cache, weights, weights_stride, keep, recent, keep, out, weights_out, kept, lengths_out, clear, dev_status, stream);
}

int kfa_cache_evict_room(const KfaCache* cache, const float* weights, const int64_t* weights_stride, int64_t keep, int64_t recent, int64_t room,
                         const KfaCache* out, float* weights_out, int32_t* kept, int32_t* lengths_out, int clear, int* dev_status,
                         void* stream) {
  kfa::EvictParams p;
  std::memset(&p, 0, sizeof(p));
  int rc;
  if ((rc = check_cache(cache, &p.c)) || (rc = check_cache(out, &p.out, "out"))) return rc;
  if (p.out.batch != p.c.batch || p.out.heads != p.c.heads || p.out.cols != p.c.cols)
    return fail(KFA_ERR_ARG, "out: batch, heads or head dim differ from the cache's");
  if (keep < 1 || recent < 0 || recent > keep || keep > p.out.capacity)
    return fail(KFA_ERR_ARG, "keep %lld, recent %lld: 0 <= recent <= keep, 1 <= keep <= %d, the room of out", (long long)keep,
                (long long)recent, p.out.capacity);
  if (room < keep || room > 0x7fff0000 || (clear && room > p.out.capacity))
    return fail(KFA_ERR_ARG, "room %lld: at least keep, up to 2^31 - 65536 (with clear up to %d, the room of out)", (long long)room, p.out.capacity);
  if (!weights || !weights_stride || !weights_out || !kept || !lengths_out || !dev_status)
    return fail(KFA_ERR_ARG, "kfa_cache_evict: null pointer");
  p.w = weights;
  p.w_sb = weights_stride[0];
  p.w_sh = weights_stride[1];
  p.keep = static_cast<int>(keep);
  p.recent = static_cast<int>(recent);
  p.clear = clear != 0;
  p.room = static_cast<int>(room);
  p.w_out = weights_out;
  p.kept = kept;
  p.lengths_out = lengths_out;
  const long long groups = ((clear ? room : keep) + 31) / 32, total = static_cast<long long>(p.c.batch) * p.c.heads * groups;
  if (total > 0x7fffffffll) return fail(KFA_ERR_ARG, "kfa_cache_evict: too many rows in one call");
  p.by_slot = kfa::FastDiv::by(static_cast<uint32_t>(groups));
  p.by_head = kfa::FastDiv::by(p.c.heads);
  p.total = static_cast<unsigned>(total);
  p.status = dev_status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 heads(p.c.heads, p.c.batch);
  rc = p.c.capacity <= 2048 ? launch(kfa::kfa_cache_select_kernel<512>, heads, 512, 0, s, p) : launch(kfa::kfa_cache_select_kernel<1024>, heads, 1024, 0, s, p);
  if (rc) return rc;
  return launch(kfa::kfa_cache_gather_kernel, dim3(static_cast<unsigned>((total + 7) / 8)), 256, 0, s, p);
}

}  // extern "C"
