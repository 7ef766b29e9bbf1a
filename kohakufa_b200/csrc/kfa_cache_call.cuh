// What the C entry points on a cache share: checks of its descriptors, tensor maps over its rows, launches. For the sources of libkfa.so only.
#pragma once

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>

#include "kfa_cache_view.cuh"
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

// 4-D tiled map over rows of D 16-bit columns: dims (D, n1, n2, n3) with element strides s1, s2, s3, boxes of 64 columns (128 bytes,
// swizzled) x b1 x b2 x b3; what is out of range reads as zeros.
int make_box_map(void* ptr, int64_t D, int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t n3, int64_t s3, int b1, int b2, int b3, int dtype,
                 CUtensorMap* map, const char* name) {
  EncodeFn enc = encode_fn();
  if (!enc) return fail(KFA_ERR_CUDA, "cuTensorMapEncodeTiled not available from the driver");
  auto st = [&](int64_t n, int64_t s) { return static_cast<cuuint64_t>(n > 1 ? s : D) * 2; };  // (an extent of 1 never advances)
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(n1), static_cast<cuuint64_t>(n2), static_cast<cuuint64_t>(n3)};
  const cuuint64_t strides[3] = {st(n1, s1), st(n2, s2), st(n3, s3)};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(b1), static_cast<cuuint32_t>(b2), static_cast<cuuint32_t>(b3)}, one[4] = {1, 1, 1, 1};
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

// Rows of a TMA box that a page holds whole numbers of (without a table: the last box may end behind the page, and reads zeros there).
int page_box(const kfa::CacheView& c) { return c.table ? (c.page % 32 == 0 ? 32 : (c.page % 16 == 0 ? 16 : 8)) : 32; }

}  // namespace
