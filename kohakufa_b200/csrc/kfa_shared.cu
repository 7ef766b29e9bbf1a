// C ABI of attention behind shared prefixes (declared in include/kfa.h): argument checks and launches.
#include "kfa_attend_call.cuh"
#include "kfa_shared.cuh"

namespace {

int64_t padded(int64_t bytes) { return (bytes + 255) / 256 * 256; }
int matrix_rows(int64_t rows) { return rows <= 16 ? 16 : (rows <= 32 ? 32 : (rows <= 128 ? 128 : 256)); }

// How a call is cut up: a function of the shapes alone, so that the scratch it needs is known beforehand.
struct SharedPlan {
  int gt, tt, head_tiles, row_tiles, ts;  // a row tile: gt heads x tt tokens, of a prefix x ts sequences
  int n_pre, n_own;                       // the kernel's rows
  int grid, extra_pre, extra_own;
  int64_t most_pre, most_own;             // counted units
  int64_t part_ml, part_o, carry_ml, carry_o, dir_pre, dir_own, bytes;  // where each begins in the scratch: [4 grid][3][rows]; [4 grid][rows][128]; ...
  int64_t carry_bytes;                    // of one of the two
};

SharedPlan plan_shared(int64_t batch, int64_t heads, int64_t kv_heads, int64_t T, int64_t prefixes, int64_t prefix_room, int64_t room, bool fresh) {
  SharedPlan a;
  const int64_t group = heads / kv_heads, gt = std::min<int64_t>(group, 128), most = 128 / gt;
  const int64_t token_tiles = (T + most - 1) / most, tt = (T + token_tiles - 1) / token_tiles, per = gt * tt;
  a.gt = static_cast<int>(gt);
  a.tt = static_cast<int>(tt);
  a.head_tiles = static_cast<int>((group + gt - 1) / gt);
  a.row_tiles = static_cast<int>(a.head_tiles * token_tiles);
  // Sequences of a prefix' row tile: what 256 rows hold (128, where all fit), of one prefix in equal parts. How many each prefix has only the device knows: where they are
  // many the tile is made for twice their mean number.
  const int64_t mean = (batch + prefixes - 1) / prefixes, wanted = prefixes == 1 ? batch : std::min(batch, 2 * mean);
  int64_t ts = 1;
  if (token_tiles == 1) {  // (tiles of 256 rows where they are no more CTAs than those of 128, two in one)
    const int64_t half = std::max<int64_t>(128 / per, 1), whole = std::max<int64_t>(256 / per, 1), n = prefixes == 1 ? batch : mean;
    ts = std::min((n + half - 1) / half < 2 * ((n + whole - 1) / whole) ? half : whole, wanted);
  }
  if (prefixes == 1) ts = (batch + (batch + ts - 1) / ts - 1) / ((batch + ts - 1) / ts);
  a.ts = static_cast<int>(ts);
  a.n_own = matrix_rows(per);
  a.n_pre = std::max(matrix_rows(per * ts), a.n_own);
  // What an item's beginning and end count, in units of 32 keys, and in the call below what a unit of the prefixes counts beside one of a sequence's own. No
  // close fit: the 7000 clk between two own items are what 9 units take, and times hardly follow. Graph time in us of 7 prefixes of 96 sequences, drafts of 8 tokens,
  // 64 sequences and 256: own items count 6 units more 32.6, 72.1, 50.2, 282; 10 30.2, 71.0, 50.3, 284; 14 32.8, 70.8, 51.7, 283. With 10, a unit counts 1.0 33.8,
  // 71.0, 50.7, 284; 1.2 30.2, 71.0, 50.3, 284; 1.7 32.6, 70.6, 51.6, 283. (The first is the only one that moves by more than 3 %, both ways: with where its
  // stretches happen to end.)
  a.extra_pre = 8;
  a.extra_own = 10;
  const int64_t pre_items = kv_heads * a.row_tiles * ((batch + ts - 1) / ts + prefixes - 1), own_items = batch * kv_heads * a.row_tiles;
  const int64_t pre_units = std::max<int64_t>((prefix_room + 31) / 32, 1);
  const int64_t own_units = std::max<int64_t>((room + 31) / 32 + (fresh ? (T + 31) / 32 : 0), 1);
  a.most_pre = pre_items * (pre_units + a.extra_pre);
  a.most_own = own_items * (own_units + a.extra_own);
  // (each kind of work has CTAs of its own, of two halves that have at least 4 units each)
  const auto ctas = [](int64_t items, int64_t units) { return (std::min<int64_t>(items, 2 * SMS) * ((units + 3) / 4) + 1) / 2; };
  a.grid = static_cast<int>(std::min<int64_t>(SMS, ctas(pre_items, pre_units) + ctas(own_items, own_units)));
  const int64_t rows = batch * heads * T;
  const int r = std::min(std::max(a.n_pre, a.n_own), 128);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += padded(bytes);
    return here;
  };
  a.part_ml = take(4ll * a.grid * 3 * r * 4);
  a.part_o = take(4ll * a.grid * r * 512);
  a.carry_bytes = padded(12 * rows) + padded(512 * rows);
  a.carry_ml = take(2 * a.carry_bytes);
  a.carry_o = a.carry_ml + padded(12 * rows);
  a.dir_pre = take(8 * kv_heads * a.row_tiles * batch);
  a.dir_own = take(8 * kv_heads * a.row_tiles * batch);
  a.bytes = at;
  return a;
}

void fill_part(kfa::AttendParams& p, const SharedPlan& plan, bool pre, int64_t batch, void* scratch) {
  p.gt = plan.gt;
  p.tt = plan.tt;
  p.head_tiles = plan.head_tiles;
  p.row_tiles = plan.row_tiles;
  p.items = p.c.heads * plan.row_tiles;
  p.by_gt = kfa::FastDiv::by(p.gt);
  p.by_items = kfa::FastDiv::by(p.items);
  p.by_row_tiles = kfa::FastDiv::by(p.row_tiles);
  p.by_head_tiles = kfa::FastDiv::by(p.head_tiles);
  p.least = 4;
  p.extra = pre ? plan.extra_pre : plan.extra_own;
  p.rows = std::min(std::max(plan.n_pre, plan.n_own), 128);
  p.box = page_box(p.c);
  p.seqs = static_cast<int>(batch);
  p.ts = plan.ts;
  p.by_ts = kfa::FastDiv::by(plan.ts);
  p.by_seq_rows = kfa::FastDiv::by(plan.gt * plan.tt);
  uint8_t* at = static_cast<uint8_t*>(scratch);
  p.part_ml = reinterpret_cast<float*>(at + plan.part_ml);
  p.part_o = reinterpret_cast<float*>(at + plan.part_o);
  p.carry_ml = reinterpret_cast<float*>(at + plan.carry_ml + (pre ? 0 : plan.carry_bytes));
  p.carry_o = reinterpret_cast<float*>(at + plan.carry_o + (pre ? 0 : plan.carry_bytes));
  p.dir = reinterpret_cast<int2*>(at + (pre ? plan.dir_pre : plan.dir_own));
}

template <int NC, int N_PRE, int N_OWN, bool BF16>
int launch_shared(const CUtensorMap (&m)[8], const kfa::SharedParams& p, const SharedPlan& plan, cudaStream_t s) {
  auto kern = kfa::kfa_shared_kernel<NC, N_PRE, N_OWN, BF16>;
  constexpr int SMEM = 2 * kfa::SH_SMEM + 1024;
  static_assert(kfa::ShCfg<NC, N_PRE>::SMEM <= (N_PRE == 256 ? 2 : 1) * kfa::SH_SMEM && kfa::ShCfg<NC, N_OWN>::SMEM <= kfa::SH_SMEM && SMEM <= 232448,
                "shared memory");
  static std::atomic<uint64_t> allowed{0};
  int rc = allow_smem(allowed, reinterpret_cast<const void*>(kern), SMEM);
  if (rc) return rc;
  if ((rc = launch(kern, dim3(plan.grid), 2 * kfa::SH_THREADS, SMEM, s, m[0], m[1], m[2], m[3], m[4], m[5], m[6], m[7], p))) return rc;
  return launch(kfa::kfa_shared_join_kernel<BF16>, dim3(static_cast<unsigned>((p.own.carry_rows + 7) / 8)), 256, 0, s, p, kfa::FastDiv::by(p.own.H),
                kfa::FastDiv::by(p.own.T));
}

template <int NC, bool BF16>
int launch_shared_rows(const CUtensorMap (&m)[8], const kfa::SharedParams& p, const SharedPlan& plan, cudaStream_t s) {
  if (plan.n_own == 128) return plan.n_pre == 256 ? launch_shared<NC, 256, 128, BF16>(m, p, plan, s) : launch_shared<NC, 128, 128, BF16>(m, p, plan, s);
  if (plan.n_own == 32) {
    if (plan.n_pre == 256) return launch_shared<NC, 256, 32, BF16>(m, p, plan, s);
    return plan.n_pre == 128 ? launch_shared<NC, 128, 32, BF16>(m, p, plan, s) : launch_shared<NC, 32, 32, BF16>(m, p, plan, s);
  }
  if (plan.n_pre == 256) return launch_shared<NC, 256, 16, BF16>(m, p, plan, s);
  if (plan.n_pre == 128) return launch_shared<NC, 128, 16, BF16>(m, p, plan, s);
  return plan.n_pre == 32 ? launch_shared<NC, 32, 16, BF16>(m, p, plan, s) : launch_shared<NC, 16, 16, BF16>(m, p, plan, s);
}

}  // namespace

extern "C" {

int64_t kfa_cache_attend_shared_bytes(const KfaTensor4* q, const KfaCache* prefix, const KfaCache* cache, const KfaTensor4* k) {
  if (!q || !prefix || !cache) return 0;
  const int64_t page = prefix->k.shape[2], kv_heads = prefix->k.shape[1], own = cache->k.shape[2], batch = q->shape[0];
  if (batch < 1 || q->shape[1] < 1 || q->shape[2] < 1 || kv_heads < 1 || q->shape[1] < kv_heads || page < 1 || own < 1 || prefix->batch < 1)
    return 0;  // (refused by the call)
  return plan_shared(batch, q->shape[1], kv_heads, q->shape[2], prefix->batch, prefix->table ? prefix->table_cols * page : page,
                     cache->table ? cache->table_cols * own : own, k != nullptr)
      .bytes;
}

int kfa_cache_attend_shared(const KfaTensor4* q, const KfaCache* prefix, const int32_t* starts, const KfaCache* cache, const KfaTensor4* k,
                            const KfaTensor4* v, const uint8_t* tree, const int64_t* tree_stride, const int32_t* counts,
                            const KfaTensor4* out, float* stats, void* scratch, float scale, int dtype, int* dev_status, void* stream) {
  kfa::SharedParams p;
  std::memset(&p, 0, sizeof(p));
  int rc;
  if ((rc = check_attend(q, cache, k, v, tree, tree_stride, counts, out, stats, scale, dtype, dev_status, p.own)) ||
      (rc = check_cache(prefix, &p.pre.c, "prefix")))
    return rc;
  kfa::AttendParams &own = p.own, &pre = p.pre;
  if (own.c.heads != pre.c.heads || own.c.cols != pre.c.cols) return fail(KFA_ERR_ARG, "prefix: heads or head dim differ from the cache's");
  if (!starts && pre.c.batch != 1) return fail(KFA_ERR_ARG, "starts: needed for %d prefixes", pre.c.batch);
  if (!scratch || reinterpret_cast<uintptr_t>(scratch) % 16) return fail(KFA_ERR_ARG, "scratch: null or not 16-byte aligned");
  const int64_t batch = own.c.batch, rows = batch * own.H * own.T, D = own.c.cols;
  const SharedPlan plan = plan_shared(batch, own.H, own.c.heads, own.T, pre.c.batch, pre.c.capacity, own.c.capacity, k != nullptr);
  if (plan.most_pre > 0x3fffffff || plan.most_own > 0x3fffffff || rows > 0x7fffff00) return fail(KFA_ERR_ARG, "too many rows in one call");
  pre.H = own.H;
  pre.T = own.T;
  pre.group = own.group;
  pre.c_log2 = own.c_log2;
  pre.status = dev_status;
  pre.starts = own.starts = starts;
  pre.groups = own.groups = pre.c.batch;
  pre.carry_rows = own.carry_rows = rows;
  fill_part(pre, plan, true, batch, scratch);
  fill_part(own, plan, false, batch, scratch);
  p.pre_pair = plan.n_pre == 256;
  p.halves = 2 * plan.grid;
  p.pre_items = pre.c.batch == 1 && !starts ? static_cast<int>(own.c.heads * plan.row_tiles * ((batch + plan.ts - 1) / plan.ts)) : 0;
  p.weight = p.pre_pair ? 1.2f : 0.6f;  // (of a CTA's time: without a pair its halves do two at once)
  CUtensorMap m[8];
  auto queries = [&](int ts, CUtensorMap* map) {
    return make_box_map(q->ptr, D, own.H, q->stride[1], own.T, q->stride[2], batch, q->stride[0], plan.gt, plan.tt, ts, dtype, map, "q");
  };
  if ((rc = queries(plan.ts, &m[0])) || (rc = pages_map(&prefix->k, pre, dtype, &m[1], "prefix keys")) ||
      (rc = pages_map(&prefix->v, pre, dtype, &m[2], "prefix values")) || (rc = queries(1, &m[3])) ||
      (rc = pages_map(&cache->k, own, dtype, &m[4], "cache keys")) || (rc = pages_map(&cache->v, own, dtype, &m[5], "cache values")))
    return rc;
  m[6] = m[4];
  m[7] = m[5];
  if (k && ((rc = new_map(k, own, dtype, &m[6], "k")) || (rc = new_map(v, own, dtype, &m[7], "v")))) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == KFA_BF16) return D > 64 ? launch_shared_rows<2, true>(m, p, plan, s) : launch_shared_rows<1, true>(m, p, plan, s);
  return D > 64 ? launch_shared_rows<2, false>(m, p, plan, s) : launch_shared_rows<1, false>(m, p, plan, s);
}

}  // extern "C"
