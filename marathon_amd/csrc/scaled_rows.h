// scaled_rows.h -- rows on their way into the block-scaled cache: loads, the largest value of a
// block, and its codes under the scale that follows from it (include/marathon_kvscaled.h).
#pragma once

#include "scaled_cache.h"

#include "fp8_e4m3.h"

#pragma clang fp contract(off)

namespace mkv_scaled {

constexpr uint32_t kInfBits = 0x7F800000u;
// 448 * 2^MKV_SCALE_MAX_EXP: beyond it even the largest scale saturates
constexpr uint32_t kTopBits = (static_cast<uint32_t>(MKV_SCALE_MAX_EXP + 8 + 127) << 23) | 0x600000u;

// The exponent of the scale for a largest |x| with these bits (finite): 448 = 1.75 * 2^8.
__device__ __forceinline__ int exponent_for(uint32_t bits) {
  if (bits == 0) return MKV_SCALE_MIN_EXP;
  const int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return min(max(e, MKV_SCALE_MIN_EXP), MKV_SCALE_MAX_EXP);
}

// The largest of a wave's values, in every lane: neighbours exchanged by the vector unit
// itself (quads, halves and whole rows of 16 mirrored, rows broadcast), where __shfl goes
// through LDS six times.
__device__ __forceinline__ uint32_t wave_max(uint32_t m) {
  const auto with = [](uint32_t x, uint32_t y) { return max(x, y); };
#define MKV_DPP(ctrl, rows) \
  with(m, static_cast<uint32_t>(__builtin_amdgcn_update_dpp( \
              static_cast<int>(m), static_cast<int>(m), ctrl, rows, 0xF, false)))
  m = MKV_DPP(0xB1, 0xF);   // quad_perm 1 0 3 2
  m = MKV_DPP(0x4E, 0xF);   // quad_perm 2 3 0 1
  m = MKV_DPP(0x141, 0xF);  // row_half_mirror
  m = MKV_DPP(0x140, 0xF);  // row_mirror
  m = MKV_DPP(0x142, 0xA);  // row_bcast 15, into rows 1 and 3
  m = MKV_DPP(0x143, 0xC);  // row_bcast 31, into rows 2 and 3
#undef MKV_DPP
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(m), 63));
}

// Four values to four codes under 2^e (the conversion divides by it, exactly, and rounds to
// nearest even).  Values fit 448 * 2^e unless `wild`: then infinities and what is larger
// saturate, and NaNs become 0x7F.
__device__ __forceinline__ uint32_t encode4(const float* x, float scale, bool wild) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  float q[4] = {x[0], x[1], x[2], x[3]};
  if (wild) {
    const float top = 448.0f * scale;
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = __builtin_amdgcn_fmed3f(q[j], -top, top);
  }
  s16x2 w = {0, 0};
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, q[0], q[1], scale, false);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, q[2], q[3], scale, true);
  uint32_t c = __builtin_bit_cast(uint32_t, w);
  if (wild) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (x[j] != x[j]) c = mkv_fp8::with_nan(c, j);
  }
  return c;
}

__device__ __forceinline__ u32x4 encode16(const float* x, int e, bool wild) {
  const float s = pow2(e);
  return u32x4{encode4(x, s, wild), encode4(x + 4, s, wild), encode4(x + 8, s, wild),
               encode4(x + 12, s, wild)};
}

// Four codes times the power of two s: the conversion multiplies.
__device__ __forceinline__ void decode4(uint32_t w, float s, float* x) {
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, s, false);
  const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, s, true);
  x[0] = a[0];
  x[1] = a[1];
  x[2] = b[0];
  x[3] = b[1];
}

__device__ __forceinline__ void decode16(u32x4 w, float s, float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) decode4(w[i], s, x + 4 * i);
}

// Where a lane stands in its wave's 16 rows of one (block, head): rows of D values in chunks
// of 16, as many rows a pass as the wave's 64 lanes cover.
template <int D>
struct Rows {
  static constexpr int kChunks = D / 16;
  static constexpr int kPerPass = 64 / kChunks;
  static constexpr int kPasses = 16 / kPerPass;
};

// The largest finite |x| (bits) of the K or V rows of a (block, head), which `parts` waves
// share, and whether any value there needs care: an infinity, a NaN, or one that saturates
// under the largest scale.
struct Largest {
  uint32_t bits, wild;
};

// The largest |x| of a lane's values; a NaN where there is one.
template <int N>
__device__ __forceinline__ uint32_t lane_max(const float* x) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < N; i += 2)  // one v_maximum3 for two values
    m = __builtin_elementwise_maximum(
        __builtin_elementwise_maximum(__builtin_fabsf(x[i]), __builtin_fabsf(x[i + 1])), m);
  return __float_as_uint(m) & 0x7FFFFFFFu;
}

template <int N>
__device__ __forceinline__ uint32_t finite_max(const float* x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t b = __float_as_uint(x[i]) & 0x7FFFFFFFu;
    m = max(m, b >= kInfBits ? 0u : b);
  }
  return m;
}

// Over a wave's values, N a lane.
template <int N>
__device__ __forceinline__ Largest largest(const float* x) {
  Largest m = {wave_max(lane_max<N>(x)), 0};
  if (m.bits > kTopBits) m = {wave_max(finite_max<N>(x)), 1};
  return m;
}

// Exchange between the waves of one (block, head); every wave of the workgroup calls it.
__device__ __forceinline__ Largest across(Largest m, int parts, uint32_t (*lds)[2], int wave) {
  if (parts == 1) return m;
  __syncthreads();  // the last exchange has been read
  if ((threadIdx.x & 63) == 0) {
    lds[wave][0] = m.bits;
    lds[wave][1] = m.wild;
  }
  __syncthreads();
  const int first = wave - wave % parts;
  for (int i = 0; i < parts; ++i) {
    m.bits = max(m.bits, lds[first + i][0]);
    m.wild |= lds[first + i][1];
  }
  return m;
}

// 8 values of element type ET, as they lie in memory.
template <int ET>
struct Raw8 {
  u32x4 w[ET == MKV_F32 ? 2 : 1];
};

template <int ET>
__device__ __forceinline__ Raw8<ET> fetch8(const char* p) {
  Raw8<ET> r;
#pragma unroll
  for (int i = 0; i < (ET == MKV_F32 ? 2 : 1); ++i)
    r.w[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p) + i);
  return r;
}

template <int ET>
__device__ __forceinline__ void unpack8(const Raw8<ET>& r, float* x) {
  if constexpr (ET == MKV_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(r.w[i / 4][i % 4]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t pair = r.w[0][j];  // (a bit cast of an element itself takes element 0)
      if constexpr (ET == MKV_BF16) {
        x[2 * j] = __uint_as_float(pair << 16);
        x[2 * j + 1] = __uint_as_float(pair & 0xFFFF0000u);
      } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const h2 h = __builtin_bit_cast(h2, pair);
        x[2 * j] = static_cast<float>(h[0]);
        x[2 * j + 1] = static_cast<float>(h[1]);
      }
    }
  }
}

// 16 values of element type ET at p.
template <int ET>
__device__ __forceinline__ void load16(const char* p, float* x) {
  const Raw8<ET> a = fetch8<ET>(p), b = fetch8<ET>(p + (ET == MKV_F32 ? 32 : 16));
  unpack8<ET>(a, x);
  unpack8<ET>(b, x + 8);
}

// Host: the tokens that a workgroup of a store looks through, of `each` workgroups if it were one.
// Decode steps want every token, and small stores every block, a workgroup of its own; large
// stores few workgroups that lead nothing, up to one a block.  In us with 1 / 4 / 8 / 16 tokens a
// workgroup, blocks of 16, 8 heads of 128 but where said:
//   1,000 requests of one token 11.8 / 15.7 / 26 / 44, 4,096 39 / 39 / 36 / 52
//   8 requests of 65, 4 heads 5.3 / 7.2;  488 of 16, 4 heads 16.1 with 4, 18.9 with 16
//   one of 1,000 12.9 / 5.9 / 6.6 / 8.5, of 2,000 28 / 9.8 / 7.6 / 9.2, of 4,000 52 / 16.6 / 11.7 /
//   10.5, of 22,000 269 / 76 / 48 / 30
//   13 requests of 5,003 in all, 4 heads of 64 12.8 / 8.1 / 9.3 / 9.4
// and with 4 / 16 / 64: blocks of 64, one of 1,000 8.9 / 8.1 / 10.1, of 8,000 107 / 36 / 15;
// blocks of 128, one of 8,000 217 / 49 / 19, and 17 with 128.
inline int store_group(int64_t tokens, int32_t requests, int64_t each, int32_t block_size) {
  const int64_t ahead = tokens / requests;  // a request's on average
  if (ahead < 16 || (each <= 4096 && ahead < 256))
    return each <= 4096 ? 1 : 4;
  if (each > 24576)
    return block_size;
  if (each > 12288)
    return ahead >= 64 ? 16 : 4;
  return block_size >= 64 && ahead >= 64 ? 16 : each > 4096 && ahead >= 1024 ? 8 : 4;
}

}  // namespace mkv_scaled
