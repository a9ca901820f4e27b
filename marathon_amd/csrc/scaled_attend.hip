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
// it.)  The one rounding is p's.  The kernel of few rows cuts it into two bf16 terms, which leaves
// 2^-17: the second product hides behind memory (a batch's next tokens 110.7 -> 111.2 us, one
// request's 19.8 -> 19.9; of 17 to 32 rows 27.4 -> 30.9).  The kernel of many rows does so for
// fp16 queries; for bf16 ones it rounds p to bf16, by half a step of it, 2^-8, as the output
// itself is: a second product would take 2,048 tokens over 22,141 from 1,072 to 1,380 us.
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
typedef float f32x16 __attribute__((ext_vector_type(16)));

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
  int32_t rows_from, rows_to;  // the requests that this launch is for, by their rows
  int32_t per;     // tokens of a part, a multiple of 64 (more where `splits` would not reach)
  float scale;     // softmax_scale * log2(e)
};

constexpr float kInf = __builtin_inff();
constexpr float kSlack = 8.0f;  // powers of two that a score may pass the running largest by
constexpr int kMinSplit = 512;  // tokens a part has at least
constexpr int kMaxSplits = 256;

// A tile: `BM` query rows (token, query head of the group) of one request, heads fastest.
// Request r's tiles begin at starts[r] * group / BM + r: that leaves each at least as many as
// it needs, from what the host knows alone, and tiles beyond a request's rows do nothing.
struct Tile {
  int64_t s0;     // the request's first token
  int64_t row0;   // the tile's first row in the request
  int64_t first;  // position of the request's first new token
  int rows;       // rows of the tile, 1 to BM
  int request;
  int full;       // tokens that every row sees
  int keys;       // tokens that some row sees
  int parts;      // parts its tokens are cut into, and the tokens of each
  int per;
};

template <int BM>
__device__ __forceinline__ bool find_tile(const AttendParams& p, int64_t tile, Tile& t) {
  const int32_t* starts = p.s.starts;
  const int group = p.group;
  const auto begin = [starts, group](int i) {
    return static_cast<int64_t>(starts[i]) * group / BM + i;
  };
  const bool single = p.rows_to <= BM;  // a request has one tile: the grid has one for each
  const int r = single ? static_cast<int>(tile) : last_at_most(p.s.requests, tile, begin);
  if (r < 0) return false;
  t.request = r;
  t.s0 = starts[r];
  const int64_t s1 = starts[r + 1];
  const int64_t first_tile = single ? tile : begin(r);
  if (t.s0 < 0 || s1 < t.s0 || s1 > p.tokens) return false;  // flagged by the first workgroup
  t.row0 = (tile - first_tile) * BM;
  const int64_t all = (s1 - t.s0) * group;
  if (all < p.rows_from || all > p.rows_to) return false;  // another launch's
  const int64_t rows = all - t.row0;
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
  const int64_t keys = hi < most ? hi : most;
  t.keys = keys < 0 ? 0 : static_cast<int>(keys);
  t.full = lo < 0 ? 0 : static_cast<int>(lo < t.keys ? lo : t.keys);
  const int per = (t.keys / p.splits + 64) & ~63;  // at least keys / splits
  t.per = per > p.per ? per : p.per;
  t.parts = t.keys > t.per ? (t.keys + t.per - 1) / t.per : 1;
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

// Two values of the output type.
template <bool F16>
__device__ __forceinline__ uint32_t out_pair(float a, float b) {
  if constexpr (F16)
    return bits_as<uint32_t>(f16x2{static_cast<_Float16>(a), static_cast<_Float16>(b)});
  else
    return round_pair(a, b);
}

// A load of what is read once: past the caches' ordinary replacement.
template <typename T>
__device__ __forceinline__ T once(const char* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const T*>(p));
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
// passes through LDS but the waves' results at the end.  A token for each of 32 requests with
// 8,270 on average, 8 KV heads of 128 (542 MB), takes 106 us, 5.1 TB/s, and as long with its blocks
// in order; a bare linear read of as many bytes 77 to 85.  Heads of 64 67 us, of 256 199.

constexpr int kFewWaves = 4;

template <int D>
struct FewRaw {  // one step's codes, as loaded
  u32x4 k[2][D / 64];       // tile of 16 tokens; 16 bytes each
  uint32_t v[8][D / 64];    // token slot; D / 16 bytes
};

// Waves a SIMD is to hold: what is in flight hides memory's latency.
template <int D, int RT>
constexpr int few_waves() {
  return D == 64 ? (RT == 1 ? 4 : 3) : D == 128 ? (RT == 1 ? 4 : 2) : (RT == 1 ? 2 : 1);
}

template <bool F16, int D, int RT>
__global__ __launch_bounds__(64 * kFewWaves, (few_waves<D, RT>())) void attend_few_kernel(AttendParams p) {
  constexpr int BM = 16 * RT, KS = D / 32, DT = D / 16, NQ = D / 64;
  __shared__ float s_o[2][D * 16];
  __shared__ float s_ml[kFewWaves][BM][2];
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int head = blockIdx.y;
  Tile t;
  // Workgroups go to the eight XCDs in turn: the tiles are turned by the part, so that a long
  // request's parts do not all fall to one (32 ragged requests: 119 -> 112 us).
  const unsigned tile = (blockIdx.x + blockIdx.z) % gridDim.x;
  if (static_cast<int>(blockIdx.z) == p.splits) {  // (a part of its own: no register is held for it)
    if (blockIdx.x + blockIdx.y == 0) check_starts(p.s, p.tokens, false);
    return;
  }
  if (!find_tile<BM>(p, tile, t)) return;
  const int part = blockIdx.z;
  if (part >= t.parts) return;
  const int k0 = part * t.per, k1 = min(t.keys, k0 + t.per);

  // Block ids and scales of this wave's next 64 steps, one step a lane: the loop then waits
  // for no table, and its loads depend on nothing that it loads.
  const int32_t* table = p.s.tables + t.request * p.s.table_stride;
  int ids[2] = {-1, -1};
  int scales[2] = {0, 0};
  const auto look_up = [&](int at) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // tokens behind the last one seen are read from its block and not used
      const int tok = min(at + 32 * kFewWaves * lane + 16 * i, t.keys - 1);
      ids[i] = table[tok >> p.c.bs_shift];
      scales[i] = 127 | (127 << 8);
      if (ids[i] < 0 || ids[i] >= p.c.num_blocks) {
        raise(p.s.flags, MKV_FLAG_SRC_RANGE);
        ids[i] = -1;
      } else {
        scales[i] = *reinterpret_cast<const uint16_t*>(
            p.c.scales + (static_cast<int64_t>(ids[i]) * p.c.heads + head) * 2);
      }
    }
  };
  const int first = k0 + 32 * wave;
  if (first < k1) look_up(first);

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

  const int bs_mask = (1 << p.c.bs_shift) - 1;
  const int lane_k = c * p.c.tstride + 16 * g, lane_v = 4 * g * p.c.tstride + (D / 16) * c;
  const auto load = [&](int at, int n, FewRaw<D>& x) {  // n: the step's lane in ids and scales
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int id = max(__builtin_amdgcn_readlane(ids[i], n), 0);
      const int64_t block = id * p.c.bstride + head * static_cast<int64_t>(p.c.hstride) +
                            ((at + 16 * i) & bs_mask) * static_cast<int64_t>(p.c.tstride);
      const char* kb = p.c.k + block;
      const char* vb = p.c.v + block;
#pragma unroll
      for (int j = 0; j < NQ; ++j) x.k[i][j] = once<u32x4>(kb + lane_k + 64 * j);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const char* a = vb + lane_v + j * p.c.tstride;
        if constexpr (D == 64) {
          x.v[4 * i + j][0] = once<uint32_t>(a);
        } else if constexpr (D == 128) {
          const u32x2 w = once<u32x2>(a);
          x.v[4 * i + j][0] = w[0];
          x.v[4 * i + j][1] = w[1];
        } else {
          const u32x4 w = once<u32x4>(a);
#pragma unroll
          for (int u = 0; u < 4; ++u) x.v[4 * i + j][u] = w[u];
        }
      }
    }
  };

  const auto step = [&](int at, int n, FewRaw<D>& x) {
    const bool ok[2] = {__builtin_amdgcn_readlane(ids[0], n) >= 0,
                        __builtin_amdgcn_readlane(ids[1], n) >= 0};
    const bool masked = at + 32 > t.full || !ok[0] || !ok[1];
    const int sc[2] = {__builtin_amdgcn_readlane(scales[0], n),
                       __builtin_amdgcn_readlane(scales[1], n)};
    const int ek[2] = {scale_exp(sc[0] & 0xFF), scale_exp(sc[1] & 0xFF)};
    const float fv[2] = {pow2(scale_exp(sc[0] >> 8)), pow2(scale_exp(sc[1] >> 8))};
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
    // What lies in rows that nobody sees must not reach the products, NaN codes times 0; nor
    // NaNs in V that only some rows see: those are noted, and marked behind the products.
    bool odd = false;
    if (masked) {
      uint32_t any = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int tok = at + 16 * (j >> 2) + 4 * g + (j & 3);
        const bool seen = tok < t.keys && ok[j >> 2];
#pragma unroll
        for (int u = 0; u < NQ; ++u) {
          x.v[j][u] = seen ? x.v[j][u] : 0u;
          const uint32_t bad = nan_bytes(x.v[j][u]);
          any |= bad;
          x.v[j][u] &= ~((bad >> 7) * 255u);
        }
      }
      odd = __any(any != 0);
    }
    uint32_t ph[RT][4], pl[RT][4];  // P^T: pairs of tokens; and what bf16 leaves of them
    uint32_t see[RT];               // masked: which of the lane's 8 tokens its row sees
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float y[8];
      see[rt] = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = j >> 2;
        y[j] = s[rt][i][j & 3] * (F16 ? p.scale * pow2(ek[i]) : p.scale);
        if (masked) {
          const int tok = at + 16 * i + 4 * g + (j & 3);
          const bool sees = tok < limit[rt] && ok[i];
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
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const u32x4 b = {ph[rt][0], ph[rt][1], ph[rt][2], ph[rt][3]};
          o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bits_as<bf16x8>(a),
                                                              bits_as<bf16x8>(b), o[rt][dt], 0, 0, 0);
          const u32x4 b2 = {pl[rt][0], pl[rt][1], pl[rt][2], pl[rt][3]};
          o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bits_as<bf16x8>(a),
                                                              bits_as<bf16x8>(b2), o[rt][dt], 0, 0, 0);
        }
      }
    }
    if (odd) {  // counted into exactly the rows that see them
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        u32x4 bad = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int i = j >> 2, row = at + 16 * i + 4 * g + (j & 3);
          bool nan = row < t.keys && ok[i];
          if (nan)
            nan = (p.c.v[max(__builtin_amdgcn_readlane(ids[i], n), 0) * p.c.bstride +
                         head * static_cast<int64_t>(p.c.hstride) +
                         (row & bs_mask) * static_cast<int64_t>(p.c.tstride) + DT * c + dt] &
                   0x7F) == 0x7F;
          bad[j >> 1] |= nan ? 0x3F80u << (16 * (j & 1)) : 0u;
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          u32x4 ones = {0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < 8; ++j)
            ones[j >> 1] |= (see[rt] >> j) & 1u ? 0x3F80u << (16 * (j & 1)) : 0u;
          const f32x4 hit = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              bits_as<bf16x8>(bad), bits_as<bf16x8>(ones), f32x4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            o[rt][dt][r] = hit[r] > 0.0f ? __builtin_nanf("") : o[rt][dt][r];
        }
      }
    }
  };

  // One step's codes in registers, and other waves to hide its loads: keeping the next step's
  // as well takes the registers of one wave in three (119 us against 111, the same requests).
  constexpr int kStride = 32 * kFewWaves;
  for (int base = first; base < k1; base += 64 * kStride) {
    if (base != first) look_up(base);
    const int last = min(64, (k1 - base + kStride - 1) / kStride) - 1;
    for (int n = 0; n <= last; ++n) {
      FewRaw<D> x;
      load(base + n * kStride, n, x);
      step(base + n * kStride, n, x);
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
    const int64_t at = (static_cast<int64_t>(tile) * p.c.heads + head) * p.splits + part;
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
              const u32x2 w = {out_pair<F16>(o[rt][dt][r] * by, o[rt][dt + 1][r] * by),
                               out_pair<F16>(o[rt][dt + 2][r] * by, o[rt][dt + 3][r] * by)};
              *reinterpret_cast<u32x2*>(at + ((D / 16) * (4 * g + r) + dt) * 2) = w;
            }
          }
        }
      }
    }
  }
}

// ------------------------------------------------------------- many rows: chunks, prefills
//
// Bound by the matrix products and the softmax's vector work, about even.  A workgroup's four
// waves hold 32 rows each of a tile of 128 and one KV head and walk the tokens together, 64 a
// step (32x32x16 products).  Codes are decoded once for all waves on their way to LDS, V
// transposed besides, so that a lane reads 8 dimensions of a token of K, and 8 tokens of a
// dimension of V, in 16 bytes.  (K kept as codes there halves its reads, but each wave then
// decodes it again, 64 conversions for 32 products: 10% slower.)  Both are read without bank
// conflicts: a row's 16-byte chunks are exchanged by its number, so that 16 rows' chunks of
// one column cover the 64 banks.
// The next step's codes are loaded into registers before a step is computed and written to
// the other of two buffers behind it: one barrier a step.  Two workgroups fit a CU, and one
// computes while the other waits.  (Heads of 64 leave room for three, of 256 for one, which
// spills 41 registers.)  A chunk of 2,048 tokens over 22,141, 40 query heads of 128 (0.97 TFLOP),
// takes 1,050 to 1,130 us with the card: 0.86 to 0.93 PFLOP/s, where a library product of 8,192^3
// reaches 1.22.  Heads of 64 run at 0.8 PFLOP/s, a score's softmax having half the products to
// hide behind; of 256 at 0.53; fp16 queries, with a second product for p, at 0.68.

constexpr int kManyWaves = 4;
constexpr int kManyRows = 32 * kManyWaves;

// Where chunk `ch` (8 values) of K's row r lies: rows of 128, 256 or 512 bytes.
template <int D>
__device__ __forceinline__ int k_place(int r, int ch) {
  return r * (2 * D) + ((ch ^ (D == 64 ? (r >> 1) & 7 : r & 15)) << 4);
}

template <bool F16, int D>
__global__ __launch_bounds__(64 * kManyWaves, (D == 256 ? 1 : 2)) void attend_many_kernel(AttendParams p) {
  constexpr int KS = D / 16, MT = D / 32, W = D / 16, KC = D / 16;
  constexpr int kKLoads = 64 * D / 16 / 256;
  __shared__ __attribute__((aligned(16))) char s_k[2][128 * D];
  __shared__ __attribute__((aligned(16))) char s_v[2][128 * D];
  __shared__ int s_odd[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
  const int c = lane & 31, h = lane >> 5;
  const int head = blockIdx.x;
  Tile t;
  // the last tiles first: of one request they see the most
  const unsigned tile = gridDim.y - 1 - blockIdx.y;
  if (blockIdx.x + blockIdx.y + blockIdx.z == 0) check_starts(p.s, p.tokens, false);
  if (!find_tile<kManyRows>(p, tile, t)) return;
  const int part = blockIdx.z;
  if (part >= t.parts) return;
  const int k0 = part * t.per, k1 = min(t.keys, k0 + t.per);
  if (tid < 2) s_odd[tid] = -1;

  // ids and scales of 64 groups of 16 tokens, one a lane; and those of the 64 behind them
  const int32_t* table = p.s.tables + t.request * p.s.table_stride;
  struct Groups {
    int id, scale;
  };
  const auto look_up = [&](int at) {
    Groups x = {-1, 127 | (127 << 8)};
    if (at < k1) {
      x.id = table[min(at + 16 * lane, t.keys - 1) >> p.c.bs_shift];
      if (x.id < 0 || x.id >= p.c.num_blocks) {
        if (wave == 0) raise(p.s.flags, MKV_FLAG_SRC_RANGE);
        x.id = -1;
      } else {
        x.scale = *reinterpret_cast<const uint16_t*>(
            p.c.scales + (static_cast<int64_t>(x.id) * p.c.heads + head) * 2);
      }
    }
    return x;
  };

  // this wave's rows: operand B of S^T = K Q^T
  const int64_t row = t.row0 + wave * 32 + c;
  const bool there = wave * 32 + c < t.rows;
  u32x4 q[KS];
  int limit = 0;
  {
    const int64_t token = row / p.group;
    const int64_t sees = t.first + token + 1;
    if (there) limit = static_cast<int>(sees < 0 ? 0 : (sees < t.keys ? sees : t.keys));
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[ks] = u32x4{0, 0, 0, 0};
    if (there) {
      const char* at = p.q + (t.s0 + token) * p.q_token +
                       (static_cast<int64_t>(head) * p.group + row % p.group) * p.q_head;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        q[ks] = *reinterpret_cast<const u32x4*>(at + (16 * ks + 8 * h) * 2);
    }
  }
  int most = limit;  // tokens that some row of the wave sees
  for (int x = 16; x > 0; x >>= 1) most = max(most, __shfl_xor(most, x));
  most = uni(most);

  f32x16 o[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[mt][i] = 0.0f;
  float m = -kInf, l = 0.0f;

  // A step's codes on their way to LDS.  K: this thread's 16 bytes of rows tid / KC + ...;
  // V: W dimensions W * (tid % 16) + j of the 4 tokens 4 * (tid / 16) + i.
  u32x4 rk[kKLoads];
  uint32_t rv[4][D / 64];
  const int bs_mask = (1 << p.c.bs_shift) - 1;
  const auto block_of = [&](const Groups& x, int n) {
    return max(__builtin_amdgcn_readlane(x.id, n), 0) * p.c.bstride +
           head * static_cast<int64_t>(p.c.hstride);
  };
  // A wave's rows of a load lie in one group of 16 tokens: a scalar base, and offsets that
  // never change.  K: 16, 8 or 4 rows a load; V: 16 tokens.
  constexpr int kRowsPass = 256 / KC;  // rows that one load of all threads covers
  const uint32_t k_off = (tid / KC % 16) * p.c.tstride + 16 * (tid % KC);
  const uint32_t v_off = 4 * (tid >> 4 & 3) * p.c.tstride + W * (tid & 15);
  const auto k_group = [&](int u) { return (u * kRowsPass + wave * (64 / KC)) >> 4; };
  const auto k_row = [&](int u) { return u * kRowsPass + tid / KC; };
  const auto fetch = [&](int at, const Groups& x, int n) {  // n: the step's first group in x
#pragma unroll
    for (int u = 0; u < kKLoads; ++u) {
      const int g = k_group(u);
      const char* kb = p.c.k + block_of(x, n + g) +
                       ((at + 16 * g) & bs_mask) * static_cast<int64_t>(p.c.tstride);
      rk[u] = *reinterpret_cast<const u32x4*>(kb + k_off);
    }
    const char* vb = p.c.v + block_of(x, n + wave) +
                     ((at + 16 * wave) & bs_mask) * static_cast<int64_t>(p.c.tstride);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const char* a = vb + i * static_cast<int64_t>(p.c.tstride) + v_off;
      if constexpr (D == 64) {
        rv[i][0] = *reinterpret_cast<const uint32_t*>(a);
      } else if constexpr (D == 128) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(a);
        rv[i][0] = w[0];
        rv[i][1] = w[1];
      } else {
        const u32x4 w = *reinterpret_cast<const u32x4*>(a);
#pragma unroll
        for (int u = 0; u < 4; ++u) rv[i][u] = w[u];
      }
    }
  };
  const auto stage = [&](int at, const Groups& x, int n, int buf) {
#pragma unroll
    for (int u = 0; u < kKLoads; ++u) {
      const float f = pow2(scale_exp(__builtin_amdgcn_readlane(x.scale, n + k_group(u)) & 0xFF));
      const int r = k_row(u), ch = 2 * (tid % KC);
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const uint32_t w0 = rk[u][2 * z], w1 = rk[u][2 * z + 1];
        u32x4 w;
        if constexpr (F16)
          w = u32x4{f16_pair<false>(w0), f16_pair<true>(w0), f16_pair<false>(w1), f16_pair<true>(w1)};
        else
          w = u32x4{bf16_pair<false>(w0, f), bf16_pair<true>(w0, f), bf16_pair<false>(w1, f),
                    bf16_pair<true>(w1, f)};
        *reinterpret_cast<u32x4*>(s_k[buf] + k_place<D>(r, ch + z)) = w;
      }
    }
    const bool good = __builtin_amdgcn_readlane(x.id, n + wave) >= 0;
    if (at + 64 > t.full || !good) {
      // what nobody sees must not reach the products, NaN codes times 0; nor NaNs that only
      // some rows see: those are noted, and marked behind the products
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool seen = good && i < t.keys - at - 4 * (tid >> 4);
#pragma unroll
        for (int u = 0; u < D / 64; ++u) {
          rv[i][u] = seen ? rv[i][u] : 0u;
          const uint32_t bad = nan_bytes(rv[i][u]);
          any |= bad;
          rv[i][u] &= ~((bad >> 7) * 255u);
        }
      }
      if (any != 0) s_odd[buf] = at;
    }
    const float f = pow2(scale_exp(__builtin_amdgcn_readlane(x.scale, n + wave) >> 8));
    // tokens 16 t + 4 quad + i: chunk 2 t + (quad & 1), its half quad / 2
    const int quad = (tid >> 4) & 3, chunk = 2 * wave + (quad & 1), half = quad >> 1;
#pragma unroll
    for (int u = 0; u < D / 64; ++u) {
      const uint32_t a01 = __builtin_amdgcn_perm(rv[1][u], rv[0][u], 0x05010400u);
      const uint32_t b01 = __builtin_amdgcn_perm(rv[3][u], rv[2][u], 0x05010400u);
      const uint32_t a23 = __builtin_amdgcn_perm(rv[1][u], rv[0][u], 0x07030602u);
      const uint32_t b23 = __builtin_amdgcn_perm(rv[3][u], rv[2][u], 0x07030602u);
      const u32x2 w[4] = {{bf16_pair<false>(a01, f), bf16_pair<false>(b01, f)},
                          {bf16_pair<true>(a01, f), bf16_pair<true>(b01, f)},
                          {bf16_pair<false>(a23, f), bf16_pair<false>(b23, f)},
                          {bf16_pair<true>(a23, f), bf16_pair<true>(b23, f)}};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = (4 * u + j) * 16 + (tid & 15);  // dimension W * (r % 16) + r / 16
        *reinterpret_cast<u32x2*>(s_v[buf] + r * 128 + ((chunk ^ ((r >> 1) & 7)) << 4) + 8 * half) =
            w[j];
      }
    }
  };

  const auto compute = [&](int at, const Groups& x, int n, int buf) {
    bool masked = at + 64 > t.full;
    int ek[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      masked |= __builtin_amdgcn_readlane(x.id, n + i) < 0;
      ek[i] = scale_exp(__builtin_amdgcn_readlane(x.scale, n + i) & 0xFF);
    }
    f32x16 s[2];
#pragma unroll
    for (int st = 0; st < 2; ++st) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[st][i] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const u32x4 a =
            *reinterpret_cast<const u32x4*>(s_k[buf] + k_place<D>(32 * st + c, 2 * ks + h));
        if constexpr (F16)
          s[st] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bits_as<f16x8>(a), bits_as<f16x8>(q[ks]),
                                                         s[st], 0, 0, 0);
        else
          s[st] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              bits_as<bf16x8>(a), bits_as<bf16x8>(q[ks]), s[st], 0, 0, 0);
      }
    }
    // What the scores of each 16 tokens are multiplied by (fp16: bare codes), as they are
    // used; no less than fp32's smallest, so that masked ones stay -inf.
    float by[4];
#pragma unroll
    for (int g = 0; g < 4; ++g)
      by[g] = F16 ? fmaxf(p.scale * pow2(ek[g]), 0x1p-126f) : p.scale;
    // register i of tile st: token at + 32 st + 8 (i / 4) + 4 h + i % 4
    // (compared with what is left, the places are constants: none is kept in a register)
    if (masked) {
      const int left = limit - at - 4 * h;
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const bool sees = 32 * st + 8 * (i >> 2) + (i & 3) < left &&
                            __builtin_amdgcn_readlane(x.id, n + 2 * st + (i >> 3)) >= 0;
          s[st][i] = sees ? s[st][i] : -kInf;
        }
    }
    float top = -kInf;
    if constexpr (F16) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float most = s[g >> 1][8 * (g & 1)];
#pragma unroll
        for (int j = 1; j < 8; ++j) most = fmaxf(most, s[g >> 1][8 * (g & 1) + j]);
        top = fmaxf(top, most * by[g]);
      }
    } else {
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[st][i]);
      top *= p.scale;
    }
    if (__any(top > m + kSlack)) {
      top = fmaxf(top, __shfl_xor(top, 32));
      const float now = fmaxf(m, top);
      const float f = now == -kInf ? 1.0f : fast_exp2(m - now);
      m = now;
      l *= f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[mt][i] *= f;
    }
    const float base = m == -kInf ? 0.0f : m;
    u32x4 ph[4], pl[4];  // P^T: 16 tokens each; and what bf16 leaves of it (F16)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y[j] = fast_exp2(__builtin_fmaf(s[g >> 1][8 * (g & 1) + j], by[g], -base));
        l += y[j];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ph[g][j] = round_pair(y[2 * j], y[2 * j + 1]);
        if constexpr (F16)
          pl[g][j] = round_pair(y[2 * j] - __uint_as_float(ph[g][j] << 16),
                                y[2 * j + 1] - __uint_as_float(ph[g][j] & 0xFFFF0000u));
      }
    }
    asm volatile("" : "+v"(l));  // summed here: sunk below the products, 32 terms stay live
    const auto v_of = [&](int g, int mt) {
      const int r = 32 * mt + c;
      return *reinterpret_cast<const u32x4*>(s_v[buf] + r * 128 + (((2 * g + h) ^ ((r >> 1) & 7)) << 4));
    };
    const auto times = [&](u32x4 a, u32x4 b, f32x16 z) {
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(bits_as<bf16x8>(a), bits_as<bf16x8>(b), z, 0, 0, 0);
    };
#pragma unroll
    for (int g = 0; g < 4; ++g) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const u32x4 a = v_of(g, mt);
        o[mt] = times(a, ph[g], o[mt]);
        if constexpr (F16) o[mt] = times(a, pl[g], o[mt]);
      }
    }
    if (masked && uni(s_odd[buf]) == at) {
      // NaNs in V that some rows see and others do not: counted into exactly the rows that do
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int r = 32 * mt + c, d = W * (r & 15) + (r >> 4);
        f32x16 hit;
#pragma unroll
        for (int i = 0; i < 16; ++i) hit[i] = 0.0f;
#pragma unroll 1
        for (int g = 0; g < 4; ++g) {
          const char* vb = p.c.v + block_of(x, n + g) + d;
          u32x4 bad = {0, 0, 0, 0}, ones = {0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int tok = at + 16 * g + 8 * (j >> 2) + 4 * h + (j & 3);
            bool nan = tok < t.keys && __builtin_amdgcn_readlane(x.id, n + g) >= 0;
            if (nan) nan = (vb[(tok & bs_mask) * static_cast<int64_t>(p.c.tstride)] & 0x7F) == 0x7F;
            bad[j >> 1] |= nan ? 0x3F80u << (16 * (j & 1)) : 0u;
            ones[j >> 1] |= tok < limit ? 0x3F80u << (16 * (j & 1)) : 0u;
          }
          hit = times(bad, ones, hit);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) o[mt][i] = hit[i] > 0.0f ? __builtin_nanf("") : o[mt][i];
      }
    }
  };

  if (k0 < k1) {
    Groups now = look_up(k0), next = look_up(k0 + 1024);
    fetch(k0, now, 0);
    __syncthreads();  // s_odd is set
    stage(k0, now, 0, 0);
    __syncthreads();
    int n = 0, buf = 0;  // the step's first group in `now`, and its buffer
    for (int at = k0; at < k1; at += 64, buf ^= 1) {
      const bool more = at + 64 < k1;
      const int n1 = (n + 4) & 63;
      const Groups then = n1 == 0 ? next : now;
      if (more) fetch(at + 64, then, n1);
      if (at < most) compute(at, now, n, buf);
      if (more) stage(at + 64, then, n1, buf ^ 1);
      if (n1 == 0) {
        now = next;
        next = look_up(at + 64 + 1024);
      }
      n = n1;
      __syncthreads();
    }
  }

  l += __shfl_xor(l, 32);
  const int i = wave * 32 + c;
  if (!there) return;
  if (t.parts > 1) {
    const int64_t at = (static_cast<int64_t>(tile) * p.c.heads + head) * p.splits + part;
    if (h == 0) {
      p.part_ml[(at * kManyRows + i) * 2] = m;
      p.part_ml[(at * kManyRows + i) * 2 + 1] = l;
    }
    float* to = p.part_o + (at * kManyRows + i) * D;
#pragma unroll
    for (int e = 0; e < 8; ++e) {  // dimensions W * d + 0..W-1, two of each mt
      const int d = 8 * (e >> 2) + 4 * h + (e & 3);
#pragma unroll
      for (int mt = 0; mt < MT; mt += 2)
        *reinterpret_cast<f32x4*>(to + W * d + 2 * mt) =
            f32x4{o[mt][e], o[mt][e + 8], o[mt + 1][e], o[mt + 1][e + 8]};
    }
  } else {
    const float by = l == 0.0f ? 0.0f : 1.0f / l;
    char* to = p.out + (t.s0 + row / p.group) * p.out_token +
               (static_cast<int64_t>(head) * p.group + row % p.group) * p.out_head;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = 8 * (e >> 2) + 4 * h + (e & 3);
#pragma unroll
      for (int mt = 0; mt < MT; mt += 2)
        *reinterpret_cast<u32x2*>(to + (W * d + 2 * mt) * 2) =
            u32x2{out_pair<F16>(o[mt][e] * by, o[mt][e + 8] * by),
                  out_pair<F16>(o[mt + 1][e] * by, o[mt + 1][e + 8] * by)};
    }
  }
}

// ------------------------------------------------------------------ the parts' results joined

// A workgroup joins one row of a tile and KV head where there are many parts and few rows
// (NG > 1: NG groups of D / 4 lanes take turns at the parts), or 256 / (D / 4) rows.

template <bool F16, int D, int BM, bool MANY>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendParams p) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
  __shared__ float s_f[kMaxSplits];
  __shared__ float s_red[4];
  __shared__ f32x4 s_o[kGroups][kLanes];
  Tile t;
  if (!find_tile<BM>(p, blockIdx.x, t) || t.parts <= 1) return;
  const int head = blockIdx.y, d = threadIdx.x % kLanes, grp = threadIdx.x / kLanes;
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * p.c.heads + head) * p.splits;
  const int step = MANY ? gridDim.z : gridDim.z * kGroups;
  for (int row = MANY ? blockIdx.z : blockIdx.z * kGroups + grp; row < t.rows; row += step) {
    f32x4 o = {0, 0, 0, 0};
    float sum = 0.0f;
    if constexpr (MANY) {
      const int tid = threadIdx.x;
      float m = -kInf, l = 0.0f;
      if (tid < t.parts) {
        const float* ml = p.part_ml + ((at + tid) * BM + row) * 2;
        m = ml[0];
        l = ml[1];
      }
      float top = m;
      for (int x = 32; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
      __syncthreads();  // the last row's reads are done
      if ((tid & 63) == 0) s_red[tid >> 6] = top;
      __syncthreads();
      top = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
      const float f = fast_exp2(m - (top == -kInf ? 0.0f : top));
      s_f[tid] = f;
      float part = l * f;
      for (int x = 32; x > 0; x >>= 1) part += __shfl_xor(part, x);
      __syncthreads();
      if ((tid & 63) == 0) s_red[tid >> 6] = part;
#pragma unroll 4
      for (int s = grp; s < t.parts; s += kGroups)
        o += *reinterpret_cast<const f32x4*>(p.part_o + ((at + s) * BM + row) * D + 4 * d) * s_f[s];
      s_o[grp][d] = o;
      __syncthreads();
      sum = s_red[0] + s_red[1] + s_red[2] + s_red[3];
      if (grp != 0) continue;
#pragma unroll
      for (int i = 1; i < kGroups; ++i) o += s_o[i][d];
    } else {
      float top = -kInf;
      for (int s = 0; s < t.parts; s += 4) {  // four parts' loads at once
        float m[4], l[4];
        f32x4 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t from = (at + min(s + j, t.parts - 1)) * BM + row;
          m[j] = s + j < t.parts ? p.part_ml[from * 2] : -kInf;
          l[j] = p.part_ml[from * 2 + 1];
          x[j] = *reinterpret_cast<const f32x4*>(p.part_o + from * D + 4 * d);
        }
        const float now = fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), top);
        const float base = now == -kInf ? 0.0f : now;
        const float old = fast_exp2(top - base);
        sum *= old;
        o *= old;
        top = now;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float f = fast_exp2(m[j] - base);
          sum += l[j] * f;
          o += x[j] * f;
        }
      }
    }
    o *= sum == 0.0f ? 0.0f : 1.0f / sum;
    const int64_t r = t.row0 + row;
    char* to = p.out + (t.s0 + r / p.group) * p.out_token +
               (static_cast<int64_t>(head) * p.group + r % p.group) * p.out_head;
    *reinterpret_cast<u32x2*>(to + d * 8) =
        u32x2{out_pair<F16>(o[0], o[1]), out_pair<F16>(o[2], o[3])};
  }
}

// ------------------------------------------------------------------------------- host

// How a call's requests run: rows a tile has, tiles, the parts that a tile's tokens may be cut
// into and the tokens of one, and the requests (by their rows) that it is for.
struct Shape {
  int rows;
  int64_t each;  // rows of the largest request
  int64_t tiles;
  int splits;
  int per;
  int32_t from, to;

  int64_t parts(int heads) const { return splits > 1 ? tiles * heads * splits : 0; }
  int64_t bytes(int heads, int head_size) const {
    return parts(heads) * rows * (head_size + 2) * 4;
  }
};

// One launch for all requests, or one for the few rows of most and one for the many of others.
struct Plan {
  Shape shape[2];
  int count;
};

constexpr int64_t kWantFew = 4096;
constexpr int64_t kMostParts = 8;  // times as many parts as wanted that a workspace has room for

// A tile's rows by those of the largest request, and the parts: of one size for all requests,
// so that long and short histories fill the chip alike, about `want` workgroups if every
// request were the longest.
Shape shape_for(const mkv_attend_desc_t& d, int64_t each, int32_t from, int32_t to) {
  Shape s;
  const int64_t rows = d.tokens * (d.q_heads / d.cache.heads);
  s.each = each;
  s.rows = each <= 16 ? 16 : each <= 32 ? 32 : kManyRows;
  s.tiles = to <= s.rows ? d.requests : rows / s.rows + d.requests;
  s.from = from;
  s.to = to;
  const int64_t room = static_cast<int64_t>(d.table_width) * d.cache.block_size;
  const int64_t longest = d.max_len > 0 && d.max_len < room ? d.max_len : room;
  const int64_t largest = (each + s.rows - 1) / s.rows * d.requests;  // if all were the largest
  const int64_t groups = (s.tiles < largest ? s.tiles : largest) * d.cache.heads;
  const auto per_of = [&](int64_t want) {  // tokens of a part
    int64_t per = longest * (groups > 0 ? groups : 1) / want;
    if (per < longest / kMaxSplits + 64) per = longest / kMaxSplits + 64;
    return ((per < kMinSplit ? kMinSplit : per) + 63) / 64 * 64;
  };
  const auto parts_of = [&](int64_t per) { return longest > per ? (longest + per - 1) / per : 1; };
  int64_t want = kWantFew, per = per_of(want);
  if (s.rows == kManyRows && (d.requests > 1 || d.cache.head_size == 64)) {
    // Requests differ in length: short parts fill the chip alike.  Eight requests with 1,024 / 1,536
    // wanted, heads of 128: 576 tiles 114.7 / 114.1 us, 808 301 / 287, 1,064 280 / 256; of 64: 808
    // 183 / 187, 1,064 166 / 148; of 256: 1,064 823 / 764.  Fewer tiles want fewer: 200 of seven
    // requests (heads of 64) 47.8 / 50.7.  One request, heads of 64: 512 over 22,000 tokens
    // 539 / 506, 976 over 8,000 462 / 416; 348 over 1,835 73.7 / 80.9, 1,080 over 2,000 204 / 215.
    want = groups >= 512 && (groups < 1024 || d.requests > 1) ? 1536 : 1024;
    per = per_of(want);
  } else if (s.rows == kManyRows) {
    // One request: as few parts as fill nine tenths of the slots that they take in turns (as many as
    // run at once, by the kernel's registers and LDS), one or two; otherwise twice as many parts as
    // run at once, or three times where those fill less and are long.  Measured as 1,024 or (512 to
    // 1,023 tiles) 1,536 wanted / this rule, heads of 128: 256 tiles over 2,000 tokens 92.2 / 83.1 us,
    // over 22,000 465 / 445; 376 over 22,000 708 / 655; 512 over 2,000 173 / 135, over 8,000 379 /
    // 343; 640 over 2,000 203 / 202; 856 over 8,000 630 / 633; 976 over 8,000 741 / 703; 1,080 over
    // 22,000 2,143 / 1,899.  Of 256: 128 over 8,000 336 / 283, 512 over 8,000 1,292 / 1,108, 640 over
    // 22,141 3,798 / 3,708.  Not where one turn takes long unequal tiles (two heads' 8,192 tokens
    // from nothing: one part 218, two 204), nor, of more tiles than two turns take, where the history
    // is short (1,256 over 1,000 tokens: one part 335, two 375).
    const int64_t resident = d.cache.head_size == 256 ? 256 : 512;
    want = 2 * resident;
    per = per_of(want);
    const int64_t fresh = each / (d.q_heads / d.cache.heads);
    const bool wedge = 2 * fresh > longest && longest >= 4096;  // first tiles see little, last ones much
    const auto fills = [&](int64_t n) {  // nine tenths of the slots that n parts a tile take in turns
      const int64_t all = groups * n, turns = (all + resident - 1) / resident;
      return 10 * all >= 9 * turns * resident && !(wedge && turns == 1);
    };
    const int64_t shorter = per_of(3 * resident);
    const bool cut = groups < 2 * resident || (longest >= 8192 && !wedge);
    if (fills(1)) {
      per = (longest + 64) / 64 * 64;
    } else if (cut && fills(2)) {
      per = ((longest + 1) / 2 + 63) / 64 * 64;
      if (per < kMinSplit) per = kMinSplit;
    } else if (cut && !fills(parts_of(per)) && (groups >= resident || shorter >= 2048)) {
      want = 3 * resident;
      per = shorter;
    }
  }
  s.splits = static_cast<int>(parts_of(per));
  // Every tile has room for its parts' results, also where the hints promise fewer tiles than the
  // token array has room for (a padded batch, a wrong hint): a token for one request of an array
  // of 8,192 would ask for 31 GB.  Parts of such a call are fewer and longer.
  const int64_t all = s.tiles * d.cache.heads;
  if (all * s.splits > kMostParts * want)
    s.splits = static_cast<int>(all < kMostParts * want ? kMostParts * want / all : 1);
  s.per = static_cast<int>(per < 1 << 30 ? per : 1 << 30);  // (no request has more tokens)
  return s;
}

int check(const mkv_attend_desc_t& d, AttendParams* p, Plan* plan) {
  const char* who = "mkv_attend_scaled";
  int rc = check_cache(who, d.cache, true, &p->c);
  if (rc == MKV_OK)
    rc = check_step(who, d.cache.block_size, d.block_tables, d.table_stride, d.table_width,
                    d.starts, d.lens, d.requests, d.error_flags, &p->s);
  if (rc != MKV_OK) return rc;
  if (d.dtype != MKV_BF16 && d.dtype != MKV_F16)
    return mkv_fail(MKV_ERR_DTYPE, "%s: dtype %d is not bf16 or fp16", who, d.dtype);
  if (d.q_heads <= 0 || d.q_heads % d.cache.heads != 0)
    return mkv_fail(MKV_ERR_ARG, "%s: %d query heads for %d KV heads", who, d.q_heads,
                    d.cache.heads);
  if (d.tokens < 0 || d.tokens > INT32_MAX || d.tokens * d.q_heads > INT32_MAX)
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

  const int64_t new_most = d.max_new > 0 && d.max_new < d.tokens ? d.max_new : d.tokens;
  const int64_t each = new_most * p->group;
  // A long chunk beside decoding requests: where those behind the largest have 16 rows or
  // fewer on average, the requests of up to 16 rows get a launch of their own, of 16 rows a
  // tile in place of 128. Measured as one launch / two, 4 query heads a KV head: a chunk of
  // 1,024 tokens beside 31 requests at 16,000 tokens 535 / 440 us, 1,000 beside 255 at 4,000
  // 400 / 348, 1,000 beside one at 16,000 314 / 306, 512 beside 3 143 / 145; with a chunk of
  // 129 beside 31 149 / 173, of 13 beside one 41 / 59: there the one launch has room for both.
  const int64_t rest = (d.tokens - new_most) * p->group;
  if (each >= 2048 && d.requests > 1 && rest <= 16 * static_cast<int64_t>(d.requests - 1)) {
    plan->shape[0] = shape_for(d, 16, 0, 16);
    plan->shape[1] = shape_for(d, each, 17, INT32_MAX);
    plan->count = 2;
  } else {
    plan->shape[0] = shape_for(d, each, 0, INT32_MAX);
    plan->count = 1;
  }
  for (int i = 0; i < plan->count; ++i) {  // the grid's limits
    const Shape& s = plan->shape[i];
    if (s.tiles > (s.rows == kManyRows ? 65535 : UINT32_MAX / (64 * kFewWaves)))
      return mkv_fail(MKV_ERR_UNSUPPORTED, "%s: %lld query rows", who,
                      (long long)(d.tokens * p->group));
  }
  return MKV_OK;
}

template <bool F16, int D, int RT>
void launch_few(const AttendParams& p, const Shape& s, int heads, hipStream_t stream) {
  // one part more, which looks through the starts
  const dim3 grid(static_cast<unsigned>(s.tiles), heads, s.splits + (p.s.flags != nullptr ? 1 : 0));
  attend_few_kernel<F16, D, RT><<<grid, 64 * kFewWaves, 0, stream>>>(p);
  if (s.splits > 1) {
    const unsigned rows = static_cast<unsigned>(s.each < 16 * RT ? (s.each > 0 ? s.each : 1) : 16 * RT);
    attend_join_kernel<F16, D, 16 * RT, true>
        <<<dim3(static_cast<unsigned>(s.tiles), heads, rows), 256, 0, stream>>>(p);
  }
}

template <bool F16, int D>
void launch(const AttendParams& p, const Shape& s, int heads, hipStream_t stream) {
  if (s.rows == 16) return launch_few<F16, D, 1>(p, s, heads, stream);
  if (s.rows == 32) return launch_few<F16, D, 2>(p, s, heads, stream);
  const unsigned tiles = static_cast<unsigned>(s.tiles);
  attend_many_kernel<F16, D><<<dim3(heads, tiles, s.splits), 64 * kManyWaves, 0, stream>>>(p);
  if (s.splits > 1)
    attend_join_kernel<F16, D, kManyRows, false>
        <<<dim3(tiles, heads, kManyRows * D / 1024), 256, 0, stream>>>(p);
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
  Plan plan;
  if (check(*d, &p, &plan) != MKV_OK) return -1;
  int64_t bytes = 0;
  for (int i = 0; i < plan.count; ++i)
    bytes += plan.shape[i].bytes(d->cache.heads, d->cache.head_size);
  return bytes;
}

extern "C" int mkv_attend_scaled(const mkv_attend_desc_t* d, void* stream) {
  const char* who = "mkv_attend_scaled";
  if (d == nullptr) return mkv_fail(MKV_ERR_ARG, "%s: desc is NULL", who);
  AttendParams p;
  Plan plan;
  const int rc = check(*d, &p, &plan);
  if (rc != MKV_OK) return rc;
  if (d->tokens == 0 || d->requests == 0) return MKV_OK;
  if (d->q == nullptr || d->out == nullptr)
    return mkv_fail(MKV_ERR_ARG, "%s: q or out is NULL", who);
  if (((reinterpret_cast<uintptr_t>(d->q) | reinterpret_cast<uintptr_t>(d->out) | p.q_token |
        p.q_head | p.out_token | p.out_head) & 15) != 0)
    return mkv_fail(MKV_ERR_ALIGN, "%s: q or out is not 16-byte aligned", who);
  // out's rows: the smaller stride passes a row, the larger one all that the smaller reaches
  const bool heads_first = d->out_head_stride <= d->out_token_stride;
  int64_t reach = d->cache.head_size;
  for (const bool heads : {heads_first, !heads_first}) {
    const int64_t n = heads ? d->q_heads : d->tokens;
    const int64_t step = heads ? d->out_head_stride : d->out_token_stride;
    if (n > 1 && step < reach) return mkv_fail(MKV_ERR_ARG, "%s: out's rows overlap", who);
    reach += step * (n - 1);
  }
  const int64_t need = mkv_attend_workspace_size(d);
  if (need > 0 && (d->workspace == nullptr || d->workspace_bytes < need))
    return mkv_fail(MKV_ERR_ARG, "%s: workspace of %lld bytes, %lld needed", who,
                    (long long)d->workspace_bytes, (long long)need);
  if ((reinterpret_cast<uintptr_t>(d->workspace) & 15) != 0)
    return mkv_fail(MKV_ERR_ALIGN, "%s: workspace is not 16-byte aligned", who);
  char* room = static_cast<char*>(d->workspace);
  for (int i = 0; i < plan.count; ++i) {
    const Shape& s = plan.shape[i];
    p.splits = s.splits;
    p.per = s.per;
    p.rows_from = s.from;
    p.rows_to = s.to;
    p.part_o = reinterpret_cast<float*>(room);
    p.part_ml = p.part_o + s.parts(d->cache.heads) * s.rows * d->cache.head_size;
    room += s.bytes(d->cache.heads, d->cache.head_size);
    hipStream_t hs = static_cast<hipStream_t>(stream);
    if (d->dtype == MKV_F16)
      launch<true>(d->cache.head_size, p, s, d->cache.heads, hs);
    else
      launch<false>(d->cache.head_size, p, s, d->cache.heads, hs);
  }
  return launched(who);
}
