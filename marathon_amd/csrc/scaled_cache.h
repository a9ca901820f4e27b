// scaled_cache.h -- what the block-scaled cache's kernels share (include/marathon_kvscaled.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "marathon_kvscaled.h"

// kvshift.hip's: records the reason for mkv_last_error() and returns `code`.
__attribute__((visibility("hidden"))) int mkv_fail(int code, const char* fmt, ...);

namespace mkv_scaled {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// One layer's cache, as the kernels take it.
struct DevCache {
  char* k;
  char* v;
  uint8_t* scales;
  int64_t num_blocks;
  int64_t bstride;
  int32_t hstride;  // bytes; within a block, so 32 bits (checked on the host)
  int32_t tstride;
  int32_t bs_shift;
  int32_t heads;
};

// The step's requests.
struct DevStep {
  const int32_t* starts;
  const int32_t* lens;
  const int32_t* tables;
  int64_t table_stride;
  int32_t table_width;
  int32_t requests;
  int32_t* flags;
};

__device__ __forceinline__ void raise(int32_t* flags, int32_t bit) {
  if (flags != nullptr) atomicOr(flags, bit);
}

// The exponent a scale byte stands for, in the range that the format allows.
__device__ __forceinline__ int scale_exp(uint32_t byte) {
  const int e = static_cast<int>(byte) - 127;
  return min(max(e, MKV_SCALE_MIN_EXP), MKV_SCALE_MAX_EXP);
}

// 2^e for e in [-126, 127].
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// A wave-uniform value as a scalar.
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

// The last i in [0, n) whose value(i) is at most `at`, for values that do not descend; -1 if
// there is none.  n <= 4096: at most two rounds of loads by the whole wave, where a binary
// search takes log2(n) dependent ones (each some 300 ns).  Values that descend give some
// index in [-1, n): callers check what they find there.
template <typename F>
__device__ __forceinline__ int last_at_most(int n, int64_t at, F value) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  if (n > 64) {
    const int i = lane * 64;
    const uint64_t hit = __ballot(i < n && value(i) <= at);
    if (hit == 0) return -1;
    base = (63 - __builtin_clzll(hit)) * 64;
  }
  const int i = base + lane;
  const uint64_t hit = __ballot(i < n && value(i) <= at);
  return hit == 0 ? -1 : base + 63 - __builtin_clzll(hit);
}

// Flags requests whose starts leave the token arrays or descend, whether or not a workgroup
// would come across them (with `rows_held`, also those with more new tokens than tokens).  One
// workgroup of a launch calls it, in front of its own work: what it loads is looked up next.
__device__ __forceinline__ void check_starts(const DevStep& s, int64_t tokens, bool rows_held) {
  if (s.flags == nullptr) return;
  bool bad = false;
  for (int r = threadIdx.x; r < s.requests; r += blockDim.x) {
    const int64_t s0 = s.starts[r], s1 = s.starts[r + 1];
    bad = bad || s0 < 0 || s1 < s0 || s1 > tokens ||
          (rows_held && s1 > s0 && s.lens[r] < s1 - s0);
  }
  if (bad) raise(s.flags, MKV_FLAG_SPAN);
}

// Host: an entry point's cache, checked and translated.
inline int check_cache(const char* who, const mkv_scaled_cache_t& c, bool bases, DevCache* out) {
  if (c.head_size != 64 && c.head_size != 128 && c.head_size != 256)
    return mkv_fail(MKV_ERR_UNSUPPORTED, "%s: head_size %d is not 64, 128 or 256", who,
                    c.head_size);
  if (c.block_size != 16 && c.block_size != 32 && c.block_size != 64 && c.block_size != 128)
    return mkv_fail(MKV_ERR_UNSUPPORTED, "%s: block_size %d is not 16, 32, 64 or 128", who,
                    c.block_size);
  if (c.heads <= 0 || c.heads > 4096) return mkv_fail(MKV_ERR_ARG, "%s: heads %d", who, c.heads);
  if (c.num_blocks < 0) return mkv_fail(MKV_ERR_ARG, "%s: num_blocks < 0", who);
  if (c.block_stride < 0 || c.head_stride < 0 || c.token_stride < 0)
    return mkv_fail(MKV_ERR_ARG, "%s: negative stride", who);
  if (((c.block_stride | c.head_stride | c.token_stride) & 15) != 0)
    return mkv_fail(MKV_ERR_ALIGN, "%s: cache strides (%lld, %lld, %lld) not 16-byte aligned", who,
                    (long long)c.block_stride, (long long)c.head_stride,
                    (long long)c.token_stride);
  // offsets within a block are 32-bit in the kernels
  const int64_t most = INT32_MAX / 2 - 512;
  if (c.head_stride > most / (c.heads > 1 ? c.heads - 1 : 1) ||
      c.token_stride > most / (c.block_size - 1) ||
      c.block_stride > INT64_MAX / 2 / (c.num_blocks > 1 ? c.num_blocks : 1))
    return mkv_fail(MKV_ERR_UNSUPPORTED, "%s: cache strides out of range", who);
  if (bases && c.num_blocks > 0) {
    if (c.k_base == nullptr || c.v_base == nullptr || c.scales == nullptr)
      return mkv_fail(MKV_ERR_ARG, "%s: a cache pointer is NULL", who);
    if (((reinterpret_cast<uintptr_t>(c.k_base) | reinterpret_cast<uintptr_t>(c.v_base)) & 15) != 0)
      return mkv_fail(MKV_ERR_ALIGN, "%s: a cache base is not 16-byte aligned", who);
    if ((reinterpret_cast<uintptr_t>(c.scales) & 1) != 0)
      return mkv_fail(MKV_ERR_ALIGN, "%s: scales are not 2-byte aligned", who);
  }
  out->k = static_cast<char*>(c.k_base);
  out->v = static_cast<char*>(c.v_base);
  out->scales = c.scales;
  out->num_blocks = c.num_blocks;
  out->bstride = c.block_stride;
  out->hstride = static_cast<int32_t>(c.head_stride);
  out->tstride = static_cast<int32_t>(c.token_stride);
  out->bs_shift = __builtin_ctz(static_cast<unsigned>(c.block_size));
  out->heads = c.heads;
  return MKV_OK;
}

// Host: the step's arrays.
inline int check_step(const char* who, int32_t block_size, const int32_t* tables,
                      int64_t table_stride, int32_t table_width, const int32_t* starts, const int32_t* lens,
                      int32_t requests, int32_t* flags, DevStep* out) {
  if (requests < 0 || requests > MKV_MAX_REQUESTS)
    return mkv_fail(MKV_ERR_ARG, "%s: requests %d outside [0, %d]", who, requests,
                    MKV_MAX_REQUESTS);
  if (table_width < 0 || table_stride < 0)
    return mkv_fail(MKV_ERR_ARG, "%s: block table of width %d, stride %lld", who, table_width,
                    (long long)table_stride);
  if (static_cast<int64_t>(table_width) * block_size > (1 << 30))
    return mkv_fail(MKV_ERR_UNSUPPORTED, "%s: block tables of more than 2^30 tokens", who);
  if (requests > 0 &&
      (starts == nullptr || lens == nullptr || (tables == nullptr && table_width > 0)))
    return mkv_fail(MKV_ERR_ARG, "%s: starts, lens or block_tables is NULL", who);
  *out = DevStep{starts, lens, tables, table_stride, table_width, requests, flags};
  return MKV_OK;
}

inline int launched(const char* who) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return mkv_fail(MKV_ERR_HIP, "%s: launch failed: %s", who, hipGetErrorString(e));
  return MKV_OK;
}

}  // namespace mkv_scaled
