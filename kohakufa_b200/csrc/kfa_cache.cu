// C ABI of the operators on a cache of keys and values (declared in include/kfa.h): argument checks and launches.
#include "kfa_attend.cuh"
#include "kfa_attend_call.cuh"
#include "kfa_cache.cuh"
#include "kfa_cache_call.cuh"
#include "kfa_weigh.cuh"

namespace {

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
  AttendPlan plan;
  CUtensorMap m[5];
  int rc = prepare_attend(q, cache, k, v, tree, tree_stride, counts, out, stats, scratch, scale, dtype, dev_status, p, plan, m);
  if (rc) return rc;
  return launch_attend_call(m, p, plan, dtype, static_cast<cudaStream_t>(stream));
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
  if ((rc = make_box_map(ck->ptr, D, ck->shape[2], ck->stride[2], ck->shape[1], ck->stride[1], ck->shape[0], ck->stride[0], a.box, 1, 1, dtype, &mk,
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
  if ((rc = make_box_map(rows_q.ptr, D, a.H, rows_q.stride[1], rows_q.shape[2], rows_q.stride[2], a.c.batch, rows_q.stride[0], p.tile_h, p.tile_t, 1,
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
