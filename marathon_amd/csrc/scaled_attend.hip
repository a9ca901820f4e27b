// scaled_attend.hip -- causal attention over the block-scaled 8-bit cache for gfx950.
//
// Mathematics.  For a query row q and the tokens j that it sees,
//     s_j = softmax_scale * q . K_j,   out = sum_j exp(s_j - m) V_j / sum_j exp(s_j - m)
// in one pass over the tokens, with the running largest m, the running sum and the running
// output rescaled when m grows.  Here m only grows when some s_j passes it by more than 2^8
// (in powers of two): any m gives the same quotient, and the fp32 sums have room for terms of
// 2^8, so nearly all steps rescale nothing and exchange nothing between lanes.
//
// Operands.  Products run on the bf16 (fp16) matrix instructions with fp32 sums: a code times
// its power of two is exact in bf16, so K and V lose nothing.  (The 8-bit matrix instructions
// would take the codes as they are, at the same cost for bf16 queries cut into two e4m3 terms,
// but they align a step's products to about 13 bits below the largest: measured 2^-12.5 of
// it.)  The one rounding is p's: to bf16 for bf16 queries (half a step is 2^-9 of it, below
// the output's own); for fp16 queries p is cut into two bf16 terms, which leaves 2^-17.
// fp16 queries multiply the bare codes (exact in fp16, where a scaled value may not be) and
// the scale is applied to s_j.
//
// Layout.  Both products are computed transposed, S^T = K Q^T and O^T = V^T P^T: a lane then
// holds scores of one query row, its statistics are one register, and P^T leaves the first
// product in the lanes where the second one wants it.  The order of the tokens within a step
// and of the dimensions is chosen per operand so that no value moves between lanes.

#include "scaled_cache.h"

#include "fp8_e4m3.h"

#pragma clang fp contract(off)

namespace {

using namespace mkv_scaled;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct AttendParams {
  DevCache c;
  DevStep s;
  const char* q;
  char* out;
  float* part_o;   // [tile, kv head, split][rows][head_size], unnormalised
  float* part_ml;  // [tile, kv head, split][rows][2]: m (log2) and l
  int64_t q_token, q_head, out_token, out_head;  // bytes
  int64_t tokens;
  int32_t group;   // query heads a KV head serves
  int32_t splits;  // most parts that a tile's tokens are cut into
  float scale;     // softmax_scale * log2(e)
};

constexpr float kInf = __builtin_inff();
constexpr float kSlack = 8.0f;  // powers of two that a score may pass the running largest by
constexpr int kMinSplit = 256;  // tokens a part has at least

// A tile: `BM` query rows (token, query head of the group) of one request, heads fastest.
// Request r's tiles begin at starts[r] * group / BM + r: that leaves each at least as many as
// it needs, from what the host knows alone, and tiles beyond a request's rows do nothing.
struct Tile {
  int64_t s0;     // the request's first token
  int64_t row0;   // the tile's first row in the request
  int rows;       // rows of the tile, 1 to BM
  int request;
  int64_t first;  // position of the request's first new token
  int64_t full;   // tokens that every row sees
  int64_t keys;   // tokens that some row sees
  int parts;      // parts its tokens are cut into, and the tokens of each
  int64_t per;
};

template <int BM>
__device__ __forceinline__ bool find_tile(const AttendParams& p, int64_t tile, Tile& t) {
  const int32_t* starts = p.s.starts;
  const int group = p.group;
  const auto begin = [starts, group](int i) {
    return static_cast<int64_t>(starts[i]) * group / BM + i;
  };
  const int r = last_at_most(p.s.requests, tile, begin);
  if (r < 0) return false;
  t.request = r;
  t.s0 = starts[r];
  const int64_t s1 = starts[r + 1];
  const int64_t first_tile = t.s0 * group / BM + r;
  if (t.s0 < 0 || s1 < t.s0 || s1 > p.tokens) {
    if (threadIdx.x == 0 && tile == first_tile) raise(p.s.flags, MKV_FLAG_SPAN);
    return false;
  }
  t.row0 = (tile - first_tile) * BM;
  const int64_t rows = (s1 - t.s0) * group - t.row0;
  if (rows <= 0) return false;
  t.rows = static_cast<int>(rows < BM ? rows : BM);
  const int64_t len = p.s.lens[r];
  t.first = len - (s1 - t.s0);
  const int64_t room = static_cast<int64_t>(p.s.table_width) << p.c.bs_shift;
  if (len > room && threadIdx.x == 0) raise(p.s.flags, MKV_FLAG_SRC_RANGE);
  int64_t most = len < room ? len : room;
  if (p.c.num_blocks == 0) {  // no block to read, whatever the table says
    if (most > 0 && threadIdx.x == 0) raise(p.s.flags, MKV_FLAG_SRC_RANGE);
    most = 0;
  }
  const int64_t lo = t.first + t.row0 / group + 1;
  const int64_t hi = t.first + (t.row0 + t.rows - 1) / group + 1;
  t.keys = hi < 0 ? 0 : (hi < most ? hi : most);
  if (t.keys < 0) t.keys = 0;
  t.full = lo < 0 ? 0 : (lo < t.keys ? lo : t.keys);
  int64_t parts = (t.keys + kMinSplit - 1) / kMinSplit;
  parts = parts < 1 ? 1 : (parts > p.splits ? p.splits : parts);
  t.per = ((t.keys + parts - 1) / parts + 63) / 64 * 64;
  t.parts = t.per > 0 ? static_cast<int>((t.keys + t.per - 1) / t.per) : 1;
  if (t.parts < 1) t.parts = 1;
  return true;
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

template <typename T, typename F>
__device__ __forceinline__ T bits_as(F x) { return __builtin_bit_cast(T, x); }

// Two codes (bytes 0 and 1 of w, or 2 and 3) times the power of two s, as a bf16 pair.
template <bool HI>
__device__ __forceinline__ uint32_t bf16_pair(uint32_t w, float s) {
  return bits_as<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(w), s, HI));
}

template <bool HI>
__device__ __forceinline__ uint32_t f16_pair(uint32_t w) {
  return bits_as<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w), 1.0f, HI));
}

__device__ __forceinline__ uint32_t round_pair(float a, float b) {
  const f32x2 x = {a, b};
  return bits_as<uint32_t>(__builtin_convertvector(x, bf16x2));
}

// Whether a dword of codes holds a NaN, as a mask of its bytes (0x80 in each such byte).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
}

// ------------------------------------------------------------------ few rows: decode steps
//
// Bound by the cache's bytes.  A workgroup's four waves share a tile of RT * 16 rows and one
// KV head and take turns at steps of 32 tokens; each reads its rows of K and V straight into
// the registers where the matrix instructions want them (16x16x32: a lane is a token of K or
// 4, 8 or 16 dimensions of V, whose bytes are paired between tokens by v_perm), so nothing
// passes through LDS but the waves' results at the end.

constexpr int kFewWaves = 4;

template <int D>
struct FewRaw {  // one step's codes, as loaded
  u32x4 k[2][D / 64];       // tile of 16 tokens; 16 bytes each
  uint32_t v[8][D / 64];    // token slot; D / 16 bytes
  uint32_t scale[2];
  bool ok[2];               // the tile's block id is one
};

template <bool F16, int D, int RT>
__global__ __launch_bounds__(64 * kFewWaves) void attend_few_kernel(AttendParams p) {
  constexpr int BM = 16 * RT, KS = D / 32, DT = D / 16, NQ = D / 64;
  __shared__ float s_o[2][D * 16];
  __shared__ float s_ml[kFewWaves][BM][2];
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int head = blockIdx.y;
  Tile t;
  if (!find_tile<BM>(p, blockIdx.x, t)) return;
  const int part = blockIdx.z;
  if (part >= t.parts) return;
  const int64_t k0 = part * t.per, k1 = min(t.keys, k0 + t.per);

  // this lane's query rows: operand B of S^T = K Q^T
  u32x4 q[RT][KS];
  int limit[RT];  // tokens the row sees
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int64_t row = t.row0 + rt * 16 + c;
    const bool there = rt * 16 + c < t.rows;
    const int64_t token = row / p.group;
    const int64_t sees = t.first + token + 1;
    limit[rt] = there ? static_cast<int>(sees < 0 ? 0 : (sees < t.keys ? sees : t.keys)) : 0;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[rt][ks] = u32x4{0, 0, 0, 0};
    if (there) {
      const char* at = p.q + (t.s0 + token) * p.q_token +
                       (static_cast<int64_t>(head) * p.group + row % p.group) * p.q_head;
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        q[rt][2 * i] = *reinterpret_cast<const u32x4*>(at + (64 * i + 16 * g) * 2);
        q[rt][2 * i + 1] = *reinterpret_cast<const u32x4*>(at + (64 * i + 16 * g + 8) * 2);
      }
    }
  }

  f32x4 o[RT][DT];
  float m[RT], l[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -kInf;
    l[rt] = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f32x4{0, 0, 0, 0};
  }

  const int32_t* table = p.s.tables + t.request * p.s.table_stride;
  const int bs_mask = (1 << p.c.bs_shift) - 1;
  const auto load = [&](int64_t at, FewRaw<D>& x) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // rows behind the last token seen are read from its block and not used
      const int64_t tok = at + 16 * i;
      const int64_t last = t.keys - 1;
      int64_t id = table[(tok < last ? tok : last) >> p.c.bs_shift];
      x.ok[i] = id >= 0 && id < p.c.num_blocks;
      if (!x.ok[i]) {
        if (lane == 0) raise(p.s.flags, MKV_FLAG_SRC_RANGE);
        id = 0;
      }
      const int row = static_cast<int>(tok) & bs_mask;
      const int64_t block = id * p.c.bstride + head * static_cast<int64_t>(p.c.hstride);
      x.scale[i] = *reinterpret_cast<const uint16_t*>(p.c.scales + (id * p.c.heads + head) * 2);
      const char* kb = p.c.k + block + (row + c) * p.c.tstride + 16 * g;
#pragma unroll
      for (int j = 0; j < NQ; ++j) x.k[i][j] = *reinterpret_cast<const u32x4*>(kb + 64 * j);
      const char* vb = p.c.v + block + (row + 4 * g) * p.c.tstride + (D / 16) * c;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const char* a = vb + j * p.c.tstride;
        if constexpr (D == 64) {
          x.v[4 * i + j][0] = *reinterpret_cast<const uint32_t*>(a);
        } else if constexpr (D == 128) {
          const u32x2 w = *reinterpret_cast<const u32x2*>(a);
          x.v[4 * i + j][0] = w[0];
          x.v[4 * i + j][1] = w[1];
        } else {
          const u32x4 w = *reinterpret_cast<const u32x4*>(a);
#pragma unroll
          for (int u = 0; u < 4; ++u) x.v[4 * i + j][u] = w[u];
        }
      }
    }
  };

  const auto step = [&](int64_t at, FewRaw<D>& x) {
    const bool masked = at + 32 > t.full || !x.ok[0] || !x.ok[1];
    const int ek[2] = {scale_exp(x.scale[0] & 0xFF), scale_exp(x.scale[1] & 0xFF)};
    const float fv[2] = {pow2(scale_exp(x.scale[0] >> 8)), pow2(scale_exp(x.scale[1] >> 8))};
    // S^T: tile i's tokens by this lane's row, tokens 16 i + 4 g + r
    f32x4 s[RT][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[rt][i] = f32x4{0, 0, 0, 0};
      const float fk = pow2(ek[i]);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const uint32_t w0 = x.k[i][ks / 2][2 * (ks & 1)], w1 = x.k[i][ks / 2][2 * (ks & 1) + 1];
        u32x4 a;
        if constexpr (F16)
          a = u32x4{f16_pair<false>(w0), f16_pair<true>(w0), f16_pair<false>(w1),
                    f16_pair<true>(w1)};
        else
          a = u32x4{bf16_pair<false>(w0, fk), bf16_pair<true>(w0, fk), bf16_pair<false>(w1, fk),
                    bf16_pair<true>(w1, fk)};
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          if constexpr (F16)
            s[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                bits_as<f16x8>(a), bits_as<f16x8>(q[rt][ks]), s[rt][i], 0, 0, 0);
          else
            s[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                bits_as<bf16x8>(a), bits_as<bf16x8>(q[rt][ks]), s[rt][i], 0, 0, 0);
        }
      }
    }
    // what lies in rows that nobody sees must not reach the products: NaN codes times 0
    bool odd = false;  // a NaN in V where some rows see a token and others do not
    if (masked) {
      uint32_t any = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t tok = at + 16 * (j >> 2) + 4 * g + (j & 3);
        const bool seen = tok < t.keys && x.ok[j >> 2];
#pragma unroll
        for (int u = 0; u < NQ; ++u) {
          x.v[j][u] = seen ? x.v[j][u] : 0u;
          any |= nan_bytes(x.v[j][u]);
        }
      }
      odd = __any(any != 0);
    }
    uint32_t ph[RT][4], pl[RT][4];  // P^T: pairs of tokens; and what bf16 leaves (F16)
    uint32_t see[RT];               // odd: which of the lane's 8 tokens its row sees
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float y[8];
      see[rt] = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = j >> 2;
        y[j] = s[rt][i][j & 3] * (F16 ? p.scale * pow2(ek[i]) : p.scale);
        if (masked) {
          const int64_t tok = at + 16 * i + 4 * g + (j & 3);
          const bool sees = tok < limit[rt] && x.ok[i];
          y[j] = sees ? y[j] : -kInf;
          see[rt] |= sees ? 1u << j : 0u;
        }
      }
      float top = y[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) top = fmaxf(top, y[j]);
      if (__any(top > m[rt] + kSlack)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float now = fmaxf(m[rt], top);
        const float f = now == -kInf ? 1.0f : fast_exp2(m[rt] - now);
        m[rt] = now;
        l[rt] *= f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[rt][dt] *= f;
      }
      const float base = m[rt] == -kInf ? 0.0f : m[rt];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y[j] = fast_exp2(y[j] - base);
        l[rt] += y[j];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ph[rt][j] = round_pair(y[2 * j], y[2 * j + 1]);
        if constexpr (F16)
          pl[rt][j] = round_pair(y[2 * j] - __uint_as_float(ph[rt][j] << 16),
                                 y[2 * j + 1] - __uint_as_float(ph[rt][j] & 0xFFFF0000u));
      }
    }
    // O^T += V^T P^T: dimension tile dt holds dimensions (D / 16) * c + dt
#pragma unroll
    for (int u = 0; u < NQ; ++u) {
      uint32_t even[4], high[4];  // codes of dimensions 4u, 4u+1 (and 4u+2, 4u+3) by token pair
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t a = x.v[2 * j][u], b = x.v[2 * j + 1][u];
        even[j] = __builtin_amdgcn_perm(b, a, 0x05010400u);
        high[j] = __builtin_amdgcn_perm(b, a, 0x07030602u);
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int dt = 4 * u + w;
        u32x4 a;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t src = w < 2 ? even[j] : high[j];
          a[j] = (w & 1) ? bf16_pair<true>(src, fv[j >> 1]) : bf16_pair<false>(src, fv[j >> 1]);
        }
        u32x4 bad;
        if (odd) {  // NaNs out of the product, and into exactly the rows that see them
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool n0 = (a[j] & 0x7FFFu) > 0x7F80u, n1 = (a[j] & 0x7FFF0000u) > 0x7F800000u;
            bad[j] = (n0 ? 0x3F80u : 0u) | (n1 ? 0x3F800000u : 0u);
            a[j] &= (n0 ? 0u : 0xFFFFu) | (n1 ? 0u : 0xFFFF0000u);
          }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const u32x4 b = {ph[rt][0], ph[rt][1], ph[rt][2], ph[rt][3]};
          o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bits_as<bf16x8>(a),
                                                              bits_as<bf16x8>(b), o[rt][dt], 0, 0, 0);
          if constexpr (F16) {
            const u32x4 b2 = {pl[rt][0], pl[rt][1], pl[rt][2], pl[rt][3]};
            o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                bits_as<bf16x8>(a), bits_as<bf16x8>(b2), o[rt][dt], 0, 0, 0);
          }
          if (odd) {
            u32x4 ones;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              ones[j] = ((see[rt] >> (2 * j)) & 1u ? 0x3F80u : 0u) |
                        ((see[rt] >> (2 * j + 1)) & 1u ? 0x3F800000u : 0u);
            const f32x4 hit = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                bits_as<bf16x8>(bad), bits_as<bf16x8>(ones), f32x4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r)
              o[rt][dt][r] = hit[r] > 0.0f ? __builtin_nanf("") : o[rt][dt][r];
          }
        }
      }
    }
  };

  {
    FewRaw<D> x;
    for (int64_t at = k0 + 32 * wave; at < k1; at += 32 * kFewWaves) {
      load(at, x);
      step(at, x);
    }
  }

  // the four waves' results: their largest, then the sums under it
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    l[rt] += __shfl_xor(l[rt], 16);
    l[rt] += __shfl_xor(l[rt], 32);
    if (g == 0) {
      s_ml[wave][rt * 16 + c][0] = m[rt];
      s_ml[wave][rt * 16 + c][1] = l[rt];
    }
  }
  __syncthreads();
  float* part_o = nullptr;
  float* part_ml = nullptr;
  if (t.parts > 1) {
    const int64_t at = (static_cast<int64_t>(blockIdx.x) * p.c.heads + head) * p.splits + part;
    part_o = p.part_o + at * BM * D;
    part_ml = p.part_ml + at * BM * 2;
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    float top = -kInf, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) top = fmaxf(top, s_ml[w][rt * 16 + c][0]);
    const float base = top == -kInf ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w)
      sum += s_ml[w][rt * 16 + c][1] * fast_exp2(s_ml[w][rt * 16 + c][0] - base);
    const float f = fast_exp2(m[rt] - base);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[rt][dt] *= f;
    const auto put = [&](int slot) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) s_o[slot][(dt * 4 + r) * 64 + lane] = o[rt][dt][r];
    };
    const auto add = [&](int slot) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[rt][dt][r] += s_o[slot][(dt * 4 + r) * 64 + lane];
    };
    if (rt > 0) __syncthreads();
    if (wave >= 2) put(wave - 2);
    __syncthreads();
    if (wave < 2) add(wave);
    __syncthreads();
    if (wave == 1) put(0);
    __syncthreads();
    if (wave == 0) {
      add(0);
      const int i = rt * 16 + c;
      if (i < t.rows) {
        if (part_o != nullptr) {
          if (g == 0) {
            part_ml[2 * i] = top;
            part_ml[2 * i + 1] = sum;
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float* at = part_o + static_cast<int64_t>(i) * D + (D / 16) * (4 * g + r);
#pragma unroll
            for (int dt = 0; dt < DT; dt += 4)
              *reinterpret_cast<f32x4*>(at + dt) =
                  f32x4{o[rt][dt][r], o[rt][dt + 1][r], o[rt][dt + 2][r], o[rt][dt + 3][r]};
          }
        } else {
          const int64_t row = t.row0 + i;
          char* at = p.out + (t.s0 + row / p.group) * p.out_token +
                     (static_cast<int64_t>(head) * p.group + row % p.group) * p.out_head;
          const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
#pragma unroll
            for (int dt = 0; dt < DT; dt += 4) {
              const float a = o[rt][dt][r] * by, b = o[rt][dt + 1][r] * by;
              const float cc = o[rt][dt + 2][r] * by, d = o[rt][dt + 3][r] * by;
              u32x2 w;
              if constexpr (F16)
                w = u32x2{bits_as<uint32_t>(f16x2{static_cast<_Float16>(a), static_cast<_Float16>(b)}),
                          bits_as<uint32_t>(f16x2{static_cast<_Float16>(cc), static_cast<_Float16>(d)})};
              else
                w = u32x2{round_pair(a, b), round_pair(cc, d)};
              *reinterpret_cast<u32x2*>(at + ((D / 16) * (4 * g + r) + dt) * 2) = w;
            }
          }
        }
      }
    }
  }
}

// ------------------------------------------------------------------ the parts' results joined

template <bool F16, int D, int BM>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendParams p) {
  Tile t;
  if (!find_tile<BM>(p, blockIdx.x, t) || t.parts <= 1) return;
  const int head = blockIdx.y;
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * p.c.heads + head) * p.splits;
  for (int i = threadIdx.x; i < t.rows * (D / 4); i += 256) {
    const int row = i / (D / 4), d = i % (D / 4) * 4;
    float top = -kInf;
    for (int s = 0; s < t.parts; ++s) top = fmaxf(top, p.part_ml[((at + s) * BM + row) * 2]);
    const float base = top == -kInf ? 0.0f : top;
    float sum = 0.0f;
    f32x4 o = {0, 0, 0, 0};
    for (int s = 0; s < t.parts; ++s) {
      const float* ml = p.part_ml + ((at + s) * BM + row) * 2;
      const float f = fast_exp2(ml[0] - base);
      sum += ml[1] * f;
      o += *reinterpret_cast<const f32x4*>(p.part_o + ((at + s) * BM + row) * D + d) * f;
    }
    o *= sum == 0.0f ? 0.0f : 1.0f / sum;
    const int64_t r = t.row0 + row;
    char* to = p.out + (t.s0 + r / p.group) * p.out_token +
               (static_cast<int64_t>(head) * p.group + r % p.group) * p.out_head;
    u32x2 w;
    if constexpr (F16)
      w = u32x2{bits_as<uint32_t>(f16x2{static_cast<_Float16>(o[0]), static_cast<_Float16>(o[1])}),
                bits_as<uint32_t>(f16x2{static_cast<_Float16>(o[2]), static_cast<_Float16>(o[3])})};
    else
      w = u32x2{round_pair(o[0], o[1]), round_pair(o[2], o[3])};
    *reinterpret_cast<u32x2*>(to + d * 2) = w;
  }
}

// ------------------------------------------------------------------------------- host

// How a call runs: rows a tile has, tiles, and the parts that a tile's tokens may be cut into.
struct Shape {
  int rows;
  int64_t tiles;
  int splits;
};

int check(const mkv_attend_desc_t& d, AttendParams* p, Shape* shape) {
  const char* who = "mkv_attend_scaled";
  int rc = check_cache(who, d.cache, true, &p->c);
  if (rc == MKV_OK)
    rc = check_step(who, d.block_tables, d.table_stride, d.table_width, d.starts, d.lens,
                    d.requests, d.error_flags, &p->s);
  if (rc != MKV_OK) return rc;
  if (d.dtype != MKV_BF16 && d.dtype != MKV_F16)
    return mkv_fail(MKV_ERR_DTYPE, "%s: dtype %d is not bf16 or fp16", who, d.dtype);
  if (d.q_heads <= 0 || d.q_heads % d.cache.heads != 0)
    return mkv_fail(MKV_ERR_ARG, "%s: %d query heads for %d KV heads", who, d.q_heads,
                    d.cache.heads);
  if (d.tokens < 0 || d.tokens * d.q_heads > INT32_MAX || d.tokens > INT32_MAX)
    return mkv_fail(MKV_ERR_ARG, "%s: tokens %lld", who, (long long)d.tokens);
  if (d.max_new < 0 || d.max_len < 0)
    return mkv_fail(MKV_ERR_ARG, "%s: max_new %d, max_len %d", who, d.max_new, d.max_len);
  if (!(d.softmax_scale > 0.0f) || d.softmax_scale > 65536.0f)
    return mkv_fail(MKV_ERR_ARG, "%s: softmax_scale %g outside (0, 65536]", who, d.softmax_scale);
  const int64_t most = INT64_MAX / 16 / (d.tokens + d.q_heads);
  if (d.q_token_stride < 0 || d.q_head_stride < 0 || d.out_token_stride < 0 ||
      d.out_head_stride < 0 || d.q_token_stride > most || d.q_head_stride > most ||
      d.out_token_stride > most || d.out_head_stride > most)
    return mkv_fail(MKV_ERR_ARG, "%s: a stride of q or out is out of range", who);
  p->q = static_cast<const char*>(d.q);
  p->out = static_cast<char*>(d.out);
  p->q_token = d.q_token_stride * 2;
  p->q_head = d.q_head_stride * 2;
  p->out_token = d.out_token_stride * 2;
  p->out_head = d.out_head_stride * 2;
  p->tokens = d.tokens;
  p->group = d.q_heads / d.cache.heads;
  p->scale = d.softmax_scale * 1.4426950408889634f;

  const int64_t rows = d.tokens * p->group;
  const int64_t each = static_cast<int64_t>(d.max_new > 0 ? d.max_new : d.tokens) * p->group;
  shape->rows = each <= 16 ? 16 : 32;
  shape->tiles = rows / shape->rows + d.requests;
  // parts: enough workgroups for three on each of 256 CUs, none under kMinSplit tokens
  const int64_t room = static_cast<int64_t>(d.table_width) * d.cache.block_size;
  const int64_t longest = d.max_len > 0 && d.max_len < room ? d.max_len : room;
  const int64_t groups = shape->tiles * d.cache.heads;
  int64_t splits = groups > 0 ? (768 + groups - 1) / groups : 1;
  const int64_t most_parts = (longest + kMinSplit - 1) / kMinSplit;
  splits = splits > most_parts ? most_parts : splits;
  splits = splits < 1 ? 1 : splits > 256 ? 256 : splits;
  shape->splits = static_cast<int>(splits);
  p->splits = shape->splits;
  if (shape->tiles > INT32_MAX)
    return mkv_fail(MKV_ERR_UNSUPPORTED, "%s: %lld tiles", who, (long long)shape->tiles);
  return MKV_OK;
}

int64_t parts_of(const mkv_attend_desc_t& d, const Shape& s) {
  return s.splits > 1 ? s.tiles * d.cache.heads * s.splits : 0;
}

template <bool F16, int D, int RT>
void launch_few(const AttendParams& p, const Shape& s, int heads, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(s.tiles), heads, s.splits);
  attend_few_kernel<F16, D, RT><<<grid, 64 * kFewWaves, 0, stream>>>(p);
  if (s.splits > 1)
    attend_join_kernel<F16, D, 16 * RT>
        <<<dim3(static_cast<unsigned>(s.tiles), heads), 256, 0, stream>>>(p);
}

template <bool F16, int D>
void launch(const AttendParams& p, const Shape& s, int heads, hipStream_t stream) {
  if (s.rows == 16)
    launch_few<F16, D, 1>(p, s, heads, stream);
  else
    launch_few<F16, D, 2>(p, s, heads, stream);
}

template <bool F16>
void launch(int d, const AttendParams& p, const Shape& s, int heads, hipStream_t stream) {
  if (d == 64)
    launch<F16, 64>(p, s, heads, stream);
  else if (d == 128)
    launch<F16, 128>(p, s, heads, stream);
  else
    launch<F16, 256>(p, s, heads, stream);
}

}  // namespace

extern "C" int64_t mkv_attend_workspace_size(const mkv_attend_desc_t* d) {
  if (d == nullptr) return -1;
  AttendParams p;
  Shape s;
  if (check(*d, &p, &s) != MKV_OK) return -1;
  return parts_of(*d, s) * s.rows * (d->cache.head_size + 2) * 4;
}

extern "C" int mkv_attend_scaled(const mkv_attend_desc_t* d, void* stream) {
  const char* who = "mkv_attend_scaled";
  if (d == nullptr) return mkv_fail(MKV_ERR_ARG, "%s: desc is NULL", who);
  AttendParams p;
  Shape s;
  const int rc = check(*d, &p, &s);
  if (rc != MKV_OK) return rc;
  if (d->tokens == 0 || d->requests == 0) return MKV_OK;
  if (d->q == nullptr || d->out == nullptr)
    return mkv_fail(MKV_ERR_ARG, "%s: q or out is NULL", who);
  if (((reinterpret_cast<uintptr_t>(d->q) | reinterpret_cast<uintptr_t>(d->out) | p.q_token |
        p.q_head | p.out_token | p.out_head) & 15) != 0)
    return mkv_fail(MKV_ERR_ALIGN, "%s: q or out is not 16-byte aligned", who);
  const int64_t parts = parts_of(*d, s);
  const int64_t need = parts * s.rows * (d->cache.head_size + 2) * 4;
  if (need > 0 && (d->workspace == nullptr || d->workspace_bytes < need))
    return mkv_fail(MKV_ERR_ARG, "%s: workspace of %lld bytes, %lld needed", who,
                    (long long)d->workspace_bytes, (long long)need);
  if ((reinterpret_cast<uintptr_t>(d->workspace) & 15) != 0)
    return mkv_fail(MKV_ERR_ALIGN, "%s: workspace is not 16-byte aligned", who);
  p.part_o = static_cast<float*>(d->workspace);
  p.part_ml = need > 0 ? p.part_o + parts * s.rows * d->cache.head_size : nullptr;
  hipStream_t hs = static_cast<hipStream_t>(stream);
  if (d->dtype == MKV_F16)
    launch<true>(d->cache.head_size, p, s, d->cache.heads, hs);
  else
    launch<false>(d->cache.head_size, p, s, d->cache.heads, hs);
  return launched(who);
}
