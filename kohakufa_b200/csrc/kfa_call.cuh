// What the C entry points share: the error message of the calling thread, CUDA errors, the driver's tensor-map encoder
// and the checks of a tensor's descriptor. For the sources of libkfa.so only.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/kfa.h"

namespace kfa {
inline thread_local char g_err[512] = "";  // one for all sources: kfa_last_error reads it
}

namespace {

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(kfa::g_err, sizeof(kfa::g_err), fmt, ap);
  va_end(ap);
  return code;
}

#define KFA_CUDA(expr)                                                                    \
  do {                                                                                    \
    cudaError_t e_ = (expr);                                                              \
    if (e_ != cudaSuccess) return fail(KFA_ERR_CUDA, "%s: %s", #expr, cudaGetErrorString(e_)); \
  } while (0)

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static std::atomic<EncodeFn> cached{nullptr};
  EncodeFn f = cached.load();
  if (f) return f;
  void* sym = nullptr;
  cudaDriverEntryPointQueryResult q;
  if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) != cudaSuccess ||
      q != cudaDriverEntryPointSuccess || !sym)
    return nullptr;
  f = reinterpret_cast<EncodeFn>(sym);
  cached.store(f);
  return f;
}

int check_tensor(const KfaTensor4* t, const char* name) {
  if (!t || !t->ptr) return fail(KFA_ERR_ARG, "%s: null tensor", name);
  if (reinterpret_cast<uintptr_t>(t->ptr) % 16) return fail(KFA_ERR_ARG, "%s: base not 16-byte aligned", name);
  if (t->stride[3] != 1) return fail(KFA_ERR_ARG, "%s: last dimension must be contiguous", name);
  for (int i = 0; i < 3; ++i)
    if (t->shape[i] > 1 && (t->stride[i] % 8 != 0 || t->stride[i] <= 0))
      return fail(KFA_ERR_ARG, "%s: stride[%d]=%lld must be a positive multiple of 8 elements", name, i,
                  static_cast<long long>(t->stride[i]));
  for (int i = 0; i < 4; ++i)
    if (t->shape[i] < 1 || t->shape[i] > 0x7fffffff) return fail(KFA_ERR_ARG, "%s: bad shape[%d]", name, i);
  return KFA_OK;
}

}  // namespace
