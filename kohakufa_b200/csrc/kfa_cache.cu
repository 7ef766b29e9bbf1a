// C ABI of the operators on a cache of keys and values (declared in include/kfa.h): argument checks and launches.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "kfa_cache.cuh"
#include "kfa_call.cuh"

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

}  // namespace

extern "C" {

int64_t kfa_cache_attend_bytes(const KfaTensor4* q, const KfaCache* cache, const KfaTensor4* k) {
  (void)q, (void)cache, (void)k;
  return 0;
}

int kfa_cache_attend(const KfaTensor4* q, const KfaCache* cache, const KfaTensor4* k, const KfaTensor4* v, const uint8_t* tree,
                     const int64_t* tree_stride, const int32_t* counts, const KfaTensor4* out, float* stats, void* scratch,
                     float scale, int dtype, int* dev_status, void* stream) {
  (void)scratch;
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
    p.k_sb = 2 * k->stride[0], p.k_sh = 2 * k->stride[1], p.k_ss = 2 * k->stride[2];
    p.v_sb = 2 * v->stride[0], p.v_sh = 2 * v->stride[1], p.v_ss = 2 * v->stride[2];
  }
  p.q = static_cast<const uint8_t*>(q->ptr);
  p.q_sb = 2 * q->stride[0], p.q_sh = 2 * q->stride[1], p.q_ss = 2 * q->stride[2];
  p.o = static_cast<uint8_t*>(out->ptr);
  p.o_sb = 2 * out->stride[0], p.o_sh = 2 * out->stride[1], p.o_ss = 2 * out->stride[2];
  p.tree = tree;
  if (tree) p.tree_sb = tree_stride[0], p.tree_st = tree_stride[1], p.tree_sj = tree_stride[2];
  p.counts = counts;
  p.stats = stats;
  p.H = static_cast<int>(q->shape[1]);
  p.T = static_cast<int>(q->shape[2]);
  p.group = p.H / p.c.heads;
  p.scale_log2 = scale * LOG2E;
  p.status = dev_status;
  if (p.H > 65535) return fail(KFA_ERR_ARG, "too many heads");
  const dim3 grid(p.T, p.H, p.c.batch);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == KFA_BF16) kfa::kfa_cache_attend_simple_kernel<true><<<grid, 128, 0, s>>>(p);
  else kfa::kfa_cache_attend_simple_kernel<false><<<grid, 128, 0, s>>>(p);
  KFA_CUDA(cudaGetLastError());
  return KFA_OK;
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
  kfa::kfa_cache_append_kernel<<<static_cast<unsigned>((total + 255) / 256), 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
  KFA_CUDA(cudaGetLastError());
  return KFA_OK;
}

int kfa_cache_weigh(const KfaTensor4* q, const float* stats, const KfaCache* cache, const KfaRows* rows, float* weights,
                    const int64_t* weights_stride, int64_t room, int add, float scale, int dtype, int* dev_status, void* stream) {
  kfa::WeighParams p;
  std::memset(&p, 0, sizeof(p));
  int rc;
  if ((rc = check_cache(cache, &p.c)) || (rc = check_new(q, p.c, 0, "q")) || (rc = check_rows(rows, q->shape[2], &p.r)) ||
      (rc = check_scale(scale)) || (rc = check_dtype(dtype)))
    return rc;
  if (!stats || !weights || !weights_stride || !dev_status) return fail(KFA_ERR_ARG, "kfa_cache_weigh: null pointer");
  if (room < p.c.capacity || room > 0x7fff0000) return fail(KFA_ERR_ARG, "weights: at least the cache's %d positions", p.c.capacity);
  p.q = static_cast<const uint8_t*>(q->ptr);
  p.q_sb = 2 * q->stride[0], p.q_sh = 2 * q->stride[1], p.q_ss = 2 * q->stride[2];
  p.stats = stats;
  p.w = weights;
  p.w_sb = weights_stride[0];
  p.w_sh = weights_stride[1];
  p.H = static_cast<int>(q->shape[1]);
  p.group = p.H / p.c.heads;
  p.room = static_cast<int>(room);
  p.add = add != 0;
  p.scale_log2 = scale * LOG2E;
  p.status = dev_status;
  const dim3 grid(static_cast<unsigned>((room + 127) / 128), p.c.heads, p.c.batch);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == KFA_BF16) kfa::kfa_cache_weigh_simple_kernel<true><<<grid, 128, 0, s>>>(p);
  else kfa::kfa_cache_weigh_simple_kernel<false><<<grid, 128, 0, s>>>(p);
  KFA_CUDA(cudaGetLastError());
  return KFA_OK;
}

int kfa_cache_evict(const KfaCache* cache, const float* weights, const int64_t* weights_stride, int64_t keep, int64_t recent,
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
  if (!weights || !weights_stride || !weights_out || !kept || !lengths_out || !dev_status)
    return fail(KFA_ERR_ARG, "kfa_cache_evict: null pointer");
  p.w = weights;
  p.w_sb = weights_stride[0];
  p.w_sh = weights_stride[1];
  p.keep = static_cast<int>(keep);
  p.recent = static_cast<int>(recent);
  p.clear = clear != 0;
  p.w_out = weights_out;
  p.kept = kept;
  p.lengths_out = lengths_out;
  const long long total = static_cast<long long>(p.c.batch) * keep * p.c.heads * (p.c.cols / 8);
  if (total > 0xffffff00ll) return fail(KFA_ERR_ARG, "kfa_cache_evict: more than 64 GB in one call");
  p.by_piece = kfa::FastDiv::by(p.c.cols / 8);
  p.by_head = kfa::FastDiv::by(p.c.heads);
  p.by_slot = kfa::FastDiv::by(static_cast<uint32_t>(keep));
  p.total = static_cast<unsigned>(total);
  p.status = dev_status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  kfa::kfa_cache_select_kernel<<<dim3(p.c.heads, p.c.batch), kfa::SELECT_THREADS, 0, s>>>(p);
  KFA_CUDA(cudaGetLastError());
  kfa::kfa_cache_gather_kernel<<<static_cast<unsigned>((total + 255) / 256), 256, 0, s>>>(p);
  KFA_CUDA(cudaGetLastError());
  return KFA_OK;
}

}  // extern "C"
