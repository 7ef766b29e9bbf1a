// C ABI of attention behind shared prefixes (declared in include/kfa.h): argument checks and launches.
#include "kfa_attend.cuh"
#include "kfa_attend_call.cuh"

namespace {

// How the prefixes' part is cut up: row tiles of up to 256 rows out of the sequences that go on from a prefix, otherwise as plan_attend does it. What each
// prefix has of them only the device knows; the tile is made for twice their mean number (for all where there is one prefix, in equal parts).
AttendPlan plan_prefix(int64_t batch, int64_t heads, int64_t kv_heads, int64_t T, int64_t prefixes, int64_t capacity, int* ts) {
  AttendPlan a = plan_attend(1, heads, kv_heads, T, capacity, false);
  const int64_t per_seq = static_cast<int64_t>(a.gt) * a.tt, mean = (batch + prefixes - 1) / prefixes;
  int64_t n = 1;
  if (a.tt == T) n = std::min(std::max<int64_t>(256 / per_seq, 1), prefixes == 1 ? batch : std::min(batch, 2 * mean));
  if (prefixes == 1) n = (batch + (batch + n - 1) / n - 1) / ((batch + n - 1) / n);
  *ts = static_cast<int>(n);
  a.tile_rows = static_cast<int>(per_seq * n);
  a.rows = a.tile_rows <= 16 ? 16 : (a.tile_rows <= 32 ? 32 : (a.tile_rows <= 64 ? 64 : (a.tile_rows <= 128 ? 128 : 256)));
  a.whole = false;
  a.extra = a.rows > 64 ? 16 : 12;
  const int64_t items = kv_heads * a.row_tiles * ((batch + n - 1) / n + prefixes - 1), units = std::max<int64_t>((capacity + 31) / 32, 1);
  a.most_units = items * (units + a.extra);
  a.grid = static_cast<int>(std::min<int64_t>(SMS, (items * units + 3) / 4));
  a.meta_bytes = (16 * a.grid + 255) / 256 * 256;
  a.ml_bytes = 2ll * a.grid * 3 * a.rows * 4;
  a.bytes = a.meta_bytes + a.ml_bytes + 2ll * a.grid * a.rows * 128 * 4;
  return a;
}

int64_t padded(int64_t bytes) { return (bytes + 255) / 256 * 256; }

}  // namespace

extern "C" {

int64_t kfa_cache_attend_shared_bytes(const KfaTensor4* q, const KfaCache* prefix, const KfaCache* cache, const KfaTensor4* k) {
  if (!q || !prefix || !cache) return 0;
  const int64_t page = prefix->k.shape[2], kv_heads = prefix->k.shape[1], own = cache->k.shape[2], batch = q->shape[0];
  if (batch < 1 || q->shape[1] < 1 || q->shape[2] < 1 || kv_heads < 1 || q->shape[1] < kv_heads || page < 1 || own < 1 || prefix->batch < 1)
    return 0;  // (refused by the call)
  int ts;
  const AttendPlan a = plan_prefix(batch, q->shape[1], kv_heads, q->shape[2], prefix->batch, prefix->table ? prefix->table_cols * page : page, &ts);
  const AttendPlan o = plan_attend(batch, q->shape[1], kv_heads, q->shape[2], cache->table ? cache->table_cols * own : own, k != nullptr, true);
  return padded(a.bytes) + padded(12 * batch * q->shape[1] * q->shape[2]) + 512 * batch * q->shape[1] * q->shape[2] + o.bytes;
}

int kfa_cache_attend_shared(const KfaTensor4* q, const KfaCache* prefix, const int32_t* starts, const KfaCache* cache, const KfaTensor4* k,
                            const KfaTensor4* v, const uint8_t* tree, const int64_t* tree_stride, const int32_t* counts,
                            const KfaTensor4* out, float* stats, void* scratch, float scale, int dtype, int* dev_status, void* stream) {
  kfa::AttendParams p, o;
  AttendPlan plan, own;
  CUtensorMap m[5], mo[5];
  std::memset(&p, 0, sizeof(p));
  int rc;
  if (!scratch || reinterpret_cast<uintptr_t>(scratch) % 16) return fail(KFA_ERR_ARG, "scratch: null or not 16-byte aligned");
  if ((rc = check_cache(prefix, &p.c, "prefix")) || (rc = check_tensor(q, "q"))) return rc;
  if (!starts && p.c.batch != 1) return fail(KFA_ERR_ARG, "starts: needed for %d prefixes", p.c.batch);
  if (q->shape[1] % p.c.heads || q->shape[3] != p.c.cols) return fail(KFA_ERR_ARG, "q: does not fit the prefixes' heads and head dim");
  int ts;
  plan = plan_prefix(q->shape[0], q->shape[1], p.c.heads, q->shape[2], p.c.batch, p.c.capacity, &ts);
  const int64_t rows = q->shape[0] * q->shape[1] * q->shape[2];
  if (plan.most_units > 0x3fffffff || rows > 0x7fffffff) return fail(KFA_ERR_ARG, "too many rows in one call");
  uint8_t* carry = static_cast<uint8_t*>(scratch) + padded(plan.bytes);
  uint8_t* behind = carry + padded(12 * rows) + 512 * rows;
  if ((rc = prepare_attend(q, cache, k, v, tree, tree_stride, counts, out, stats, behind, scale, dtype, dev_status, o, own, mo, true))) return rc;
  if (o.c.heads != p.c.heads || o.c.cols != p.c.cols) return fail(KFA_ERR_ARG, "prefix: heads or head dim differ from the cache's");
  p.H = o.H;
  p.T = o.T;
  p.group = o.group;
  p.c_log2 = o.c_log2;
  p.slack = o.slack;
  p.status = dev_status;
  fill_plan(p, plan, scratch);
  p.seqs = static_cast<int>(q->shape[0]);
  p.ts = ts;
  p.by_ts = kfa::FastDiv::by(ts);
  p.by_seq_rows = kfa::FastDiv::by(p.gt * p.tt);
  p.starts = o.starts = starts;
  p.groups = o.groups = p.c.batch;
  p.carry_rows = o.carry_rows = rows;
  p.carry_ml = o.carry_ml = reinterpret_cast<float*>(carry);
  p.carry_o = o.carry_o = reinterpret_cast<float*>(carry + padded(12 * rows));
  if ((rc = make_box_map(q->ptr, p.c.cols, p.H, q->stride[1], p.T, q->stride[2], p.seqs, q->stride[0], p.gt, p.tt, ts, dtype, &m[0], "q")) ||
      (rc = pages_map(&prefix->k, p, dtype, &m[1], "prefix keys")) || (rc = pages_map(&prefix->v, p, dtype, &m[2], "prefix values")))
    return rc;
  m[3] = m[1];
  m[4] = m[2];
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if ((rc = launch_attend_call<kfa::ATT_PREFIX>(m, p, plan, dtype, s))) return rc;
  return launch_attend_call<kfa::ATT_OWN>(mo, o, own, dtype, s);
}

}  // extern "C"
