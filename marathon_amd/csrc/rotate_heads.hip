// rotate_heads.hip -- query and key heads normalised and turned to their positions for gfx950,
// for any cache (norm_rotate) and on the way into the block-scaled one (store_rotated).
//
// Mathematics.  A head x of D values at position p:
//     y = x * rsqrt(mean(x^2) + eps) * w
//     (y_i, y_{i+R/2}) turned by a_i = p * inv_freq_i,  i < R/2
// in fp32, rounded once.
//
// Layout.  Both sums and pairs stay within a few lanes: D / 16 lanes hold a head, each 8 values
// at a_off and 8 at b_off, the two halves of 8 pairs (behind the first R values: 16 that are
// not turned).  The sum of squares then takes 2 to 4 exchanges between neighbours by the vector
// unit (DPP), a pair none, and every access moves 16 bytes a lane.
//
// Angles.  cos and sin are the same for all heads of a token, so a wave makes each once, a
// frequency a lane, and hands them over through LDS.  p * inv_freq is taken in quarter turns
// in 64 bits (a position of a million times an fp32 frequency loses 16 bits in 32), split
// into the nearest whole one and what is left, |u| <= 1/2; of that fp32 holds enough, and the
// Taylor series of sin and cos at u * pi/2 <= pi/4, to the terms of u^11 and u^12, are below
// fp32's rounding.
//
// No matrix work, a dozen operations a value: bound by memory, small calls by their latency.

#include "marathon_kvstep.h"
#include "scaled_rows.h"

#include <algorithm>
#include <numeric>
#include <type_traits>

#pragma clang fp contract(off)

namespace {

using namespace mkv_scaled;

struct Turn {
  const float* inv_freq;
  const char* weight[2];  // q's, k's; null: ones
  int32_t half;           // rotary / 2
  int32_t weight_type;
  float eps;
  int32_t norm;
};

struct HeadRows {
  const char* x;
  char* out;
  int64_t token, head, out_token, out_head;  // bytes
  int32_t heads;
  int32_t stream;  // the output past the caches
};

// Quarter turns of an angle a position, in 64 bits.
__device__ __forceinline__ double quarters(float inv_freq) {
  return static_cast<double>(inv_freq) * 0x1.45f306dc9c883p-1;
}

// (cos, sin) of `q` quarter turns, |q| < 2^51.
__device__ __forceinline__ f32x2 cos_sin(double q) {
  // 1.5 * 2^52 leaves no room for a fraction: the sum's last bits are the nearest whole number
  constexpr double kWhole = 0x1.8p52;
  const double sum = q + kWhole;
  const uint32_t quadrant = static_cast<uint32_t>(__builtin_bit_cast(uint64_t, sum));
  const float u = static_cast<float>(q - (sum - kWhole)), u2 = u * u;
  // (pi/2)^n / n! with the signs of the series; pi/2 itself in two terms
  float s = __builtin_fmaf(u2, -0x1.e307500000000p-19f, 0x1.5078340000000p-13f);
  s = __builtin_fmaf(u2, s, -0x1.32d2cc0000000p-8f);
  s = __builtin_fmaf(u2, s, 0x1.466bc60000000p-4f);
  s = __builtin_fmaf(u2, s, -0x1.4abbce0000000p-1f);
  s = __builtin_fmaf(u2, s, -0x1.777a5c0000000p-25f);
  s = __builtin_fmaf(u, 0x1.921fb60000000p+0f, u * s);
  float c = __builtin_fmaf(u2, 0x1.f9d38a0000000p-22f, -0x1.a6d1f20000000p-16f);
  c = __builtin_fmaf(u2, c, 0x1.e1f5060000000p-11f);
  c = __builtin_fmaf(u2, c, -0x1.55d3c80000000p-6f);
  c = __builtin_fmaf(u2, c, 0x1.03c1f00000000p-2f);
  c = __builtin_fmaf(u2, c, -0x1.3bd3cc0000000p+0f);
  c = __builtin_fmaf(u2, c, 1.0f);
  const bool odd = quadrant & 1;
  const float x = odd ? s : c, y = odd ? c : s;
  const uint32_t flip = quadrant << 30;  // bit 31: quadrants 2 and 3
  return f32x2{__uint_as_float(__float_as_uint(x) ^ ((flip ^ (quadrant << 31)) & 0x80000000u)),
               __uint_as_float(__float_as_uint(y) ^ (flip & 0x80000000u))};
}

// Where a lane's 16 values of a head lie.
template <int D>
struct Place {
  static constexpr int kLanes = D / 16;         // lanes of a head
  static constexpr int kHeads = 64 / kLanes;    // heads (or rows) a wave holds at once
  int a, b;     // first values of the two eights
  bool turned;
  __device__ __forceinline__ Place(int piece, int half) {
    turned = 8 * piece < half;
    a = turned ? 8 * piece : 16 * piece;  // 2 half + 16 (piece - half / 8)
    b = turned ? a + half : a + 8;
  }
};

// The sum over a head's lanes, in each of them; the order is the same in every lane.
template <int D>
__device__ __forceinline__ float head_sum(float x) {
#define MKV_DPP(ctrl) \
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), ctrl, 0xF, 0xF, true))
  MKV_DPP(0xB1);   // quad_perm 1 0 3 2
  MKV_DPP(0x4E);   // quad_perm 2 3 0 1
  if constexpr (D >= 128) MKV_DPP(0x141);  // row_half_mirror
  if constexpr (D >= 256) MKV_DPP(0x140);  // row_mirror
#undef MKV_DPP
  return x;
}

// 8 weights; ones where there are none.
__device__ __forceinline__ void weights8(const char* w, int type, int at, float* x) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = 1.0f;
  if (w == nullptr) return;
  if (type == MKV_F32) {
    const u32x4* p = reinterpret_cast<const u32x4*>(w + 4 * at);
    unpack8<MKV_F32>(Raw8<MKV_F32>{{p[0], p[1]}}, x);
  } else {
    const u32x4 p = *reinterpret_cast<const u32x4*>(w + 2 * at);
    if (type == MKV_BF16)
      unpack8<MKV_BF16>(Raw8<MKV_BF16>{{p}}, x);
    else
      unpack8<MKV_F16>(Raw8<MKV_F16>{{p}}, x);
  }
}

template <int ET>
__device__ __forceinline__ void put8(char* p, const float* x, bool stream) {
  if constexpr (ET == MKV_F32) {
    reinterpret_cast<u32x4*>(p)[0] = u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]),
                                           __float_as_uint(x[2]), __float_as_uint(x[3])};
    reinterpret_cast<u32x4*>(p)[1] = u32x4{__float_as_uint(x[4]), __float_as_uint(x[5]),
                                           __float_as_uint(x[6]), __float_as_uint(x[7])};
  } else {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (ET == MKV_BF16)
        w[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x[2 * j], x[2 * j + 1]}), b2));
      else
        w[j] = __builtin_bit_cast(uint32_t, h2{static_cast<_Float16>(x[2 * j]), static_cast<_Float16>(x[2 * j + 1])});
    }
    if (stream) {
      asm volatile("" ::: "memory");  // (else the two stores become one, an ordinary one)
      __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(p));
      asm volatile("" ::: "memory");
    } else {
      *reinterpret_cast<u32x4*>(p) = w;
    }
  }
}

// A lane's 16 values of a head: normalised and weighted, then the pairs turned.
template <int D>
__device__ __forceinline__ void normalise(float* x, const float* w, const Turn& t) {
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) sum = __builtin_fmaf(x[i], x[i], sum);
  const float r = rsqrtf(__builtin_fmaf(head_sum<D>(sum), 1.0f / D, t.eps));
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = x[i] * r * w[i];
}

// (Values that are not turned are left alone, not turned by nothing: an infinity or a NaN would
// reach its neighbour as 0 * inf.  Chosen behind the products: a branch costs calls that turn all
// of a head up to 4%.)
__device__ __forceinline__ void rotate(float* x, const f32x2* turn, bool turned) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = x[i], b = x[8 + i], c = turn[i][0], s = turn[i][1];
    x[i] = turned ? __builtin_fmaf(a, c, -(b * s)) : a;
    x[8 + i] = turned ? __builtin_fmaf(b, c, a * s) : b;
  }
}

// The (cos, sin) of a lane's 8 pairs.
template <int D>
__device__ __forceinline__ void turns8(const f32x2* lds, const Place<D>& place, f32x2* turn) {
#pragma unroll
  for (int i = 0; i < 8; ++i) turn[i] = place.turned ? lds[place.a + i] : f32x2{1.0f, 0.0f};
}

// A wave's share of one side: heads [h0, h1) of one token; or (SEVERAL) all heads of `count` tokens
// from `token` on.  As many at once as a wave holds, in the order (token, head).
struct Share {
  int64_t token;
  int count, h0, h1;
};

// The share's heads: the next heads' loads are in flight while these are worked on.  `own` says which
// of the tokens are somebody's (a bit each): the others' rows are not read, which a caller may not
// have.  Behind the first loads, `angles` makes the wave's (cos, sin) in LDS, [token][half], and
// leaves out tokens of requests that do not fit: positions are waited for beside the rows.
template <int ET, int D, bool SEVERAL, typename O, typename F>
__device__ __forceinline__ void turn_heads(const HeadRows& rows, const Turn& t, int side,
                                           const Share& s, const f32x2* lds, O own, F angles) {
  constexpr int kBytes = ET == MKV_F32 ? 4 : 2, kHeads = Place<D>::kHeads;
  const int lane = threadIdx.x & 63, sub = lane / Place<D>::kLanes;
  const Place<D> place(lane % Place<D>::kLanes, t.half);
  const int heads = s.h1 - s.h0, count = SEVERAL ? s.count : 1;
  const int skip = SEVERAL ? kHeads / heads : 0, step = kHeads - skip * heads;  // tokens, heads a round
  int mine = SEVERAL ? sub / heads : 0, h = s.h0 + sub - mine * heads;
  const char* in = rows.x + s.token * rows.token;
  char* out = rows.out + s.token * rows.out_token;
  Raw8<ET> a{}, b{};
  uint32_t owned = own();
  if (owned == 0) return;
  const auto held = [&](int token, int h) {
    return token < count && h < s.h1 && (!SEVERAL || (owned >> token & 1));
  };
  const auto fetch = [&](int token, int h) {
    const char* at = in + h * rows.head;
    if constexpr (SEVERAL) at += token * rows.token;
    a = fetch8<ET>(at + place.a * kBytes);
    b = fetch8<ET>(at + place.b * kBytes);
  };
  if (held(mine, h)) fetch(mine, h);
  float w[16];
  if (t.norm) {
    weights8(t.weight[side], t.weight_type, place.a, w);
    weights8(t.weight[side], t.weight_type, place.b, w + 8);
  }
  owned = angles(owned);
  if (owned == 0) return;
  f32x2 turn[8];
  if constexpr (!SEVERAL) turns8(lds, place, turn);
  for (int first = 0; first < count * heads; first += kHeads) {
    if constexpr (SEVERAL) turns8(lds + min(mine, count - 1) * t.half, place, turn);
    float x[16];
    unpack8<ET>(a, x);
    unpack8<ET>(b, x + 8);
    int next = mine + skip, h_next = h + step;
    if (SEVERAL && h_next >= s.h1) ++next, h_next -= heads;
    if (held(next, h_next)) fetch(next, h_next);
    if (t.norm) normalise<D>(x, w, t);
    if (t.half > 0) rotate(x, turn, place.turned);
    if (held(mine, h)) {
      char* to = out + h * rows.out_head;
      if constexpr (SEVERAL) to += mine * rows.out_token;
      put8<ET>(to + place.a * kBytes, x, rows.stream);
      put8<ET>(to + place.b * kBytes, x + 8, rows.stream);
    }
    mine = next;
    h = h_next;
  }
}

// (cos, sin) of `count` tokens at position(i), i < count, into the wave's LDS.
template <typename F>
__device__ __forceinline__ void make_angles(f32x2* lds, const Turn& t, int count, F position) {
  const int lane = threadIdx.x & 63;
  wave_fence();  // the last ones have been read
  if (count == 1) {
    const double at = position(0);
    for (int f = lane; f < t.half; f += 64) lds[f] = cos_sin(at * quarters(t.inv_freq[f]));
  } else {
    for (int e = lane; e < count * t.half; e += 64)
      lds[e] = cos_sin(position(e / t.half) * quarters(t.inv_freq[e % t.half]));
  }
  wave_fence();
}

// Host: how many times as many heads as it holds at once a wave takes, of `all` that there are: one
// while so many waves fill the chip less than once, two while they fill it once or twice, then as
// many as share a token's angles and have the next heads' loads in flight.  (With 1 / 2 / 6: 800
// tokens of 32 + 8 heads of 128 5.1 / 5.1 / 5.8 us, 1,600 9.1 / 7.7 / 8.3, 4,000 20.5 / 18.6 / 17.3;
// 22,141 of 40 + 8 109 / 93 / 87.)
int passes_for(int64_t all) { return all >= 8192 ? 6 : all >= 3500 ? 2 : 1; }

// Host: how a side's heads are shared out: tokens and heads that a wave takes, and waves of as many
// tokens.
struct Cut {
  int32_t tokens, each, parts;
};

Cut cut_heads(int heads, int at_once, int most) {
  // the fewest tokens whose heads leave no lane idle (at most as many as heads at once), against a
  // token a wave or as many as fit in one round: 22,141 tokens of 5 + 1 heads of 128 19.6 to 24.4 us,
  // of 10 + 2 29.5 to 34.6, of 5 + 1 into the cache 25.3 to 34.8; six rounds for all sides: 2,000
  // tokens of 40 + 8 fp32 heads 27.6 to 22.5
  const int tokens = heads > 0 ? std::min(at_once / std::gcd(heads, at_once), at_once * most / heads) : 1;
  if (tokens > 1) return {tokens, heads, 1};
  const int passes = (heads + at_once - 1) / at_once, waves = (passes + most - 1) / most;
  const int each = at_once * (waves > 0 ? (passes + waves - 1) / waves : 1);
  return {1, each, (heads + each - 1) / each};
}

// ------------------------------------------------------------------------- norm and rotate

struct RotateParams {
  HeadRows side[2];  // q, k
  Turn turn;
  const void* positions;
  int64_t tokens;
  int32_t wide;  // positions of 64 bits
  Cut cut[2];
  uint32_t q_waves, waves;  // of the queries, and in all
};

constexpr int kWaves = 4;

// Queries' waves first, then the keys'.  SEVERAL: of one side or both, waves have several tokens (the
// code for that costs the others 2%).
template <int ET, int D, bool SEVERAL>
__global__ __launch_bounds__(64 * kWaves) void norm_rotate_kernel(RotateParams p) {
  __shared__ f32x2 s_turn[kWaves][Place<D>::kHeads * D / 2];
  const int wave = uni(threadIdx.x >> 6);
  uint32_t unit = blockIdx.x * kWaves + wave;
  if (unit >= p.waves) return;
  const int side = unit >= p.q_waves;
  if (side) unit -= p.q_waves;
  const HeadRows rows = side ? p.side[1] : p.side[0];
  const Cut cut = side ? p.cut[1] : p.cut[0];
  Share s;
  s.token = static_cast<int64_t>(unit / cut.parts) * cut.tokens;
  s.count = static_cast<int>(min(static_cast<int64_t>(cut.tokens), p.tokens - s.token));
  s.h0 = unit % cut.parts * cut.each;
  s.h1 = min(s.h0 + cut.each, rows.heads);
  const auto own = []() { return 0xFFFFFFFFu; };
  const auto angles = [&](uint32_t owned) {
    if (p.turn.half > 0)
      make_angles(s_turn[wave], p.turn, SEVERAL ? s.count : 1, [&](int i) {
        return p.wide ? static_cast<double>(static_cast<const int64_t*>(p.positions)[s.token + i])
                      : static_cast<double>(static_cast<const int32_t*>(p.positions)[s.token + i]);
      });
    return owned;
  };
  if (SEVERAL && cut.tokens > 1)
    turn_heads<ET, D, SEVERAL>(rows, p.turn, side, s, s_turn[wave], own, angles);
  else
    turn_heads<ET, D, false>(rows, p.turn, side, s, s_turn[wave], own, angles);
}

// ------------------------------------------------------------- into the block-scaled cache

struct PutParams {
  DevCache c;
  DevStep s;
  HeadRows q;
  Turn turn;
  const char* k;
  const char* v;
  int64_t k_token, k_head, v_token, v_head;  // bytes
  int64_t tokens;
  int32_t group;   // tokens a workgroup looks through
  int32_t planes;  // of the grid's y that store keys and values; those behind them turn queries
  Cut cut;         // of the queries
};

constexpr int kMaxWaves = 8;

// Keys and values: a workgroup's waves take `heads_here` heads of the blocks that begin, for
// their request and step, among `group` consecutive tokens, 16 rows of a block and head a wave,
// as the cache's plain store does.  The block's angles are made by all of its waves together.
template <int ET, int D>
__device__ __forceinline__ void put_keys(const PutParams& p, f32x2* s_turn, uint32_t (*s_max)[2]) {
  using R = Rows<D>;
  constexpr int P = R::kPasses, kBytes = ET == MKV_F32 ? 4 : 2;
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const int bs = 1 << p.c.bs_shift, parts = bs >> 4;
  const int heads_here = (blockDim.x >> 6) / parts;
  const int head = blockIdx.y * heads_here + wave / parts, part = wave % parts;
  const bool active = head < p.c.heads;
  const int piece = lane % R::kChunks, sub = lane / R::kChunks;
  const Place<D> place(piece, p.turn.half);
  const int half = p.turn.half;
  if (blockIdx.x == 0 && blockIdx.y == 0) check_starts(p.s, p.tokens, true);
  float w[16];
  if (p.turn.norm) {
    weights8(p.turn.weight[1], p.turn.weight_type, place.a, w);
    weights8(p.turn.weight[1], p.turn.weight_type, place.b, w + 8);
  }
  int64_t t = static_cast<int64_t>(blockIdx.x) * p.group;
  const int64_t end = min(t + p.group, p.tokens);
  while (t < end) {  // the same steps in every wave of the workgroup
    const int32_t* starts = p.s.starts;
    const int r = last_at_most(p.s.requests, t, [starts](int i) { return starts[i]; });
    if (r < 0) {  // before the first request
      const int64_t first = p.s.requests > 0 ? starts[0] : end;
      t = first > t ? first : end;
      continue;
    }
    const int64_t s0 = starts[r], s1 = starts[r + 1];
    if (t < s0 || t >= s1) break;  // behind the last request, or starts that descend
    const int64_t first_pos = p.s.lens[r] - (s1 - s0);
    const int64_t pos = first_pos + (t - s0);
    if (s0 < 0 || s1 > p.tokens || first_pos < 0) {  // flagged by the first workgroup
      t = s1;
      continue;
    }
    const int off = static_cast<int>(pos & (bs - 1)), base = static_cast<int>(pos) - off;
    if (t != s0 && off != 0) {  // a block that an earlier token leads
      t = min(t + bs - off, s1);
      continue;
    }
    const int n = static_cast<int>(min(static_cast<int64_t>(bs - off), s1 - t));
    const int64_t col = pos >> p.c.bs_shift;
    int64_t id = -1;
    if (col < p.s.table_width) id = p.s.tables[r * p.s.table_stride + col];
    // this wave's new rows of the block
    Raw8<ET> ka[P], kb[P], va[P], vb[P];
#pragma unroll
    for (int u = 0; u < P; ++u) {
      const int row = part * 16 + u * R::kPerPass + sub;
      const bool fresh = active && row >= off && row < off + n;
      ka[u] = kb[u] = va[u] = vb[u] = Raw8<ET>{};
      if (fresh) {
        const int64_t at = t + row - off;
        const char* k = p.k + at * p.k_token + head * p.k_head;
        const char* v = p.v + at * p.v_token + head * p.v_head + piece * 16 * kBytes;
        ka[u] = fetch8<ET>(k + place.a * kBytes);
        kb[u] = fetch8<ET>(k + place.b * kBytes);
        va[u] = fetch8<ET>(v);
        vb[u] = fetch8<ET>(v + 8 * kBytes);
      }
    }
    if (id < 0 || id >= p.c.num_blocks) {  // (the rows are on their way while it is looked up)
      if (lane == 0 && wave == 0) raise(p.s.flags, MKV_FLAG_DST_RANGE);
      t += n;
      continue;
    }
    if (half > 0) {
      __syncthreads();  // the last block's have been read
      for (int f = lane; f < half; f += 64) {
        const double each = quarters(p.turn.inv_freq[f]);
        for (int row = off + wave; row < off + n; row += blockDim.x >> 6)
          s_turn[row * half + f] = cos_sin(static_cast<double>(base + row) * each);
      }
      __syncthreads();
    }
    uint8_t* scale = p.c.scales + (id * p.c.heads + head) * 2;
    const int64_t block = id * p.c.bstride + head * static_cast<int64_t>(p.c.hstride);
    const int old = active && off > 0 ? *reinterpret_cast<const uint16_t*>(scale) : 0;
    // rows [0, off) stay, under the larger scale
    const auto keep = [&](char* at, int was, int e) {
      if (e <= was) return;
#pragma unroll
      for (int u = 0; u < P; ++u) {
        const int row = part * 16 + u * R::kPerPass + sub;
        if (row >= off) continue;
        u32x4* codes = reinterpret_cast<u32x4*>(at + row * p.c.tstride + piece * 16);
        float x[16];
        decode16(*codes, 1.0f, x);
        *codes = encode16(x, min(e - was, 100), true);
      }
    };
    // a pass none of whose rows is new (most of a decode step's) has nothing to work on
    const auto idle = [&](int u) {
      const int first = part * 16 + u * R::kPerPass;
      return first + R::kPerPass <= off || first >= off + n;
    };
    int ek, ev;
    {
      float x[P][16];
#pragma unroll
      for (int u = 0; u < P; ++u) {
        const int row = part * 16 + u * R::kPerPass + sub;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[u][i] = 0.0f;
        if (idle(u)) continue;
        unpack8<ET>(ka[u], x[u]);
        unpack8<ET>(kb[u], x[u] + 8);
        if (p.turn.norm) normalise<D>(x[u], w, p.turn);
        if (half > 0) {
          f32x2 turn[8];
          turns8(s_turn + row * half, place, turn);
          rotate(x[u], turn, place.turned);
        }
        if (!(active && row >= off && row < off + n)) {  // (eps 0 makes NaNs of no row at all)
#pragma unroll
          for (int i = 0; i < 16; ++i) x[u][i] = 0.0f;
        }
      }
      const Largest most = across(largest<16 * P>(x[0]), parts, s_max, wave);
      ek = exponent_for(most.bits);
      if (active) {
        char* to = p.c.k + block;
        if (off > 0) {
          const int was = scale_exp(old & 0xFF);
          keep(to, was, ek);
          ek = max(ek, was);
        }
        // Neighbours exchange eights, so that each holds 16 values in a row: a lane of even
        // number its own first eight and its neighbour's, one of odd number the second ones.
        const bool odd = piece & 1;
        const int at = place.turned && odd ? place.b - 8 : place.a;
#pragma unroll
        for (int u = 0; u < P; ++u) {
          if (idle(u)) continue;
          const int row = part * 16 + u * R::kPerPass + sub;
          const auto other = [](uint32_t c) {
            return static_cast<uint32_t>(
                __builtin_amdgcn_update_dpp(0, static_cast<int>(c), 0xB1, 0xF, 0xF, true));
          };
          u32x4 c = encode16(x[u], ek, most.wild);
          const uint32_t g0 = other(odd ? c[0] : c[2]), g1 = other(odd ? c[1] : c[3]);
          if (place.turned) c = odd ? u32x4{g0, g1, c[2], c[3]} : u32x4{c[0], c[1], g0, g1};
          if (row >= off && row < off + n)
            __builtin_nontemporal_store(c, reinterpret_cast<u32x4*>(to + row * p.c.tstride + at));
        }
      }
    }
    {
      float x[P][16];
#pragma unroll
      for (int u = 0; u < P; ++u) {
        unpack8<ET>(va[u], x[u]);
        unpack8<ET>(vb[u], x[u] + 8);
      }
      const Largest most = across(largest<16 * P>(x[0]), parts, s_max, wave);
      ev = exponent_for(most.bits);
      if (active) {
        char* to = p.c.v + block;
        if (off > 0) {
          const int was = scale_exp(old >> 8);
          keep(to, was, ev);
          ev = max(ev, was);
        }
#pragma unroll
        for (int u = 0; u < P; ++u) {
          if (idle(u)) continue;
          const int row = part * 16 + u * R::kPerPass + sub;
          const u32x4 c = encode16(x[u], ev, most.wild);
          if (row >= off && row < off + n)
            __builtin_nontemporal_store(c, reinterpret_cast<u32x4*>(to + row * p.c.tstride + piece * 16));
        }
      }
    }
    if (parts > 1) __syncthreads();  // every wave has read the old scale
    if (active && part == 0 && lane == 0)
      *reinterpret_cast<uint16_t*>(scale) = static_cast<uint16_t>((ek + 127) | ((ev + 127) << 8));
    t += n;
  }
}

// Queries: the waves of a workgroup, and of the planes beside it, take turns at the tokens and
// at their heads.
template <int ET, int D, bool SEVERAL>
__device__ __forceinline__ void put_queries(const PutParams& p, f32x2* s_turn) {
  const int waves = blockDim.x >> 6, wave = uni(threadIdx.x >> 6);
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.group;
  const int here = static_cast<int>(min(static_cast<int64_t>(p.group), p.tokens - t0));
  const int units = (here + p.cut.tokens - 1) / p.cut.tokens * p.cut.parts;
  f32x2* lds = s_turn + wave * p.cut.tokens * p.turn.half;
  // The step's rows among them: those in front of and behind the requests are not read.  (Looked up
  // by the two outer starts: each token's request in front of its rows cost 121 us in place of 119
  // for 22,141 tokens, and 16.6 of 15.5 for 16 requests of 100; this 119.2 and 15.5, and 12.3 of 11.8
  // for 5,003 ragged ones with heads of 64.)
  const auto within = [&](int64_t row) {
    return static_cast<int>(max(int64_t{0}, min(row - t0, static_cast<int64_t>(here))));
  };
  const int lo = within(p.s.starts[0]), hi = within(p.s.starts[p.s.requests]);
  for (int i = (blockIdx.y - p.planes) * waves + wave; i < units; i += (gridDim.y - p.planes) * waves) {
    Share s;
    const int first = i / p.cut.parts * p.cut.tokens;
    s.token = t0 + first;
    s.count = min(p.cut.tokens, here - first);
    s.h0 = i % p.cut.parts * p.cut.each;
    s.h1 = min(s.h0 + p.cut.each, p.q.heads);
    const auto own = [&]() {
      // the bits of the tokens in front of the group's row n
      const auto below = [&](int n) { return (1u << max(0, min(n - first, s.count))) - 1; };
      return below(hi) & ~below(lo);
    };
    turn_heads<ET, D, SEVERAL>(p.q, p.turn, 0, s, lds, own, [&](uint32_t held) {
      // each token's position, in the lane of its number; a request is looked up once for all of
      // its tokens
      uint32_t owned = 0;
      int at = 0;
      int64_t shift = 0, s1 = -1;
      const int32_t* starts = p.s.starts;
      for (int j = 0; j < s.count; ++j) {
        const int64_t t = s.token + j;
        if (t >= s1) {
          s1 = -1;
          const int r = last_at_most(p.s.requests, t, [starts](int x) { return starts[x]; });
          if (r < 0) continue;
          const int64_t s0 = starts[r], end = starts[r + 1];
          shift = p.s.lens[r] - end;  // from a row to its position
          if (s0 < 0 || t < s0 || t >= end || end > p.tokens || shift + s0 < 0) continue;
          s1 = end;
        }
        owned |= 1u << j;
        at = static_cast<int>(threadIdx.x & 63) == j ? static_cast<int>(t + shift) : at;
      }
      owned &= held;
      // (a lane may ask another: `half` is a multiple of 16, so the last round of make_angles has at
      // least 16 lanes, and no wave has more tokens)
      if (owned != 0 && p.turn.half > 0)
        make_angles(lds, p.turn, s.count, [&](int j) { return static_cast<double>(__shfl(at, j)); });
      return owned;
    });
  }
}

template <int ET, int D>
__global__ __launch_bounds__(64 * kMaxWaves) void put_kernel(PutParams p) {
  extern __shared__ f32x2 s_turn[];  // [half] of a block's rows, or of each wave's tokens
  __shared__ uint32_t s_max[kMaxWaves][2];
  if (static_cast<int>(blockIdx.y) < p.planes)
    put_keys<ET, D>(p, s_turn, s_max);
  else if (p.cut.tokens > 1)
    put_queries<ET, D, true>(p, s_turn);
  else
    put_queries<ET, D, false>(p, s_turn);
}

// ------------------------------------------------------------------------- host

int check_turn(const char* who, const mkv_turn_t& t, int32_t head_size, Turn* out) {
  if (t.rotary < 0 || t.rotary > head_size || t.rotary % 32 != 0)
    return mkv_fail(MKV_ERR_ARG, "%s: rotary %d is not a multiple of 32 up to %d", who, t.rotary,
                    head_size);
  if (t.rotary > 0 && t.inv_freq == nullptr)
    return mkv_fail(MKV_ERR_ARG, "%s: inv_freq is NULL", who);
  if ((reinterpret_cast<uintptr_t>(t.inv_freq) & 3) != 0)
    return mkv_fail(MKV_ERR_ALIGN, "%s: inv_freq is not 4-byte aligned", who);
  if (t.norm && !(t.eps >= 0.0f && t.eps < __builtin_inff()))
    return mkv_fail(MKV_ERR_ARG, "%s: eps %g", who, t.eps);
  const bool weighted = t.q_weight != nullptr || t.k_weight != nullptr;
  if (weighted && !t.norm) return mkv_fail(MKV_ERR_ARG, "%s: weights without a norm", who);
  if (weighted && t.weight_dtype != MKV_BF16 && t.weight_dtype != MKV_F16 && t.weight_dtype != MKV_F32)
    return mkv_fail(MKV_ERR_DTYPE, "%s: weight dtype %d is not bf16, fp16 or fp32", who,
                    t.weight_dtype);
  if (((reinterpret_cast<uintptr_t>(t.q_weight) | reinterpret_cast<uintptr_t>(t.k_weight)) & 15) != 0)
    return mkv_fail(MKV_ERR_ALIGN, "%s: a weight is not 16-byte aligned", who);
  out->inv_freq = t.inv_freq;
  out->weight[0] = static_cast<const char*>(t.q_weight);
  out->weight[1] = static_cast<const char*>(t.k_weight);
  out->half = t.rotary / 2;
  out->weight_type = t.weight_dtype;
  out->eps = t.eps;
  out->norm = t.norm != 0;
  return MKV_OK;
}

// The rows that are read and written; those written lie apart.
int check_rows(const char* who, const char* name, const mkv_head_rows_t& r, int64_t tokens,
               int32_t head_size, int64_t eb, HeadRows* out) {
  if (r.heads < 0 || r.heads > 65536)
    return mkv_fail(MKV_ERR_ARG, "%s: %d heads of %s", who, r.heads, name);
  const int64_t most = INT64_MAX / 64 / (tokens + r.heads + 1);
  for (const int64_t s : {r.token_stride, r.head_stride, r.out_token_stride, r.out_head_stride})
    if (s < 0 || s > most) return mkv_fail(MKV_ERR_ARG, "%s: a stride of %s is out of range", who, name);
  *out = HeadRows{static_cast<const char*>(r.x), static_cast<char*>(r.out), r.token_stride * eb,
                  r.head_stride * eb, r.out_token_stride * eb, r.out_head_stride * eb, r.heads, 0};
  if (tokens == 0 || r.heads == 0) return MKV_OK;
  if (r.x == nullptr || r.out == nullptr) return mkv_fail(MKV_ERR_ARG, "%s: %s is NULL", who, name);
  if (((reinterpret_cast<uintptr_t>(r.x) | reinterpret_cast<uintptr_t>(r.out) | out->token |
        out->head | out->out_token | out->out_head) & 15) != 0)
    return mkv_fail(MKV_ERR_ALIGN, "%s: %s is not 16-byte aligned", who, name);
  // the smaller stride passes a row, the larger one all that the smaller reaches
  const bool heads_first = r.out_head_stride <= r.out_token_stride;
  int64_t reach = head_size;
  for (const bool heads : {heads_first, !heads_first}) {
    const int64_t n = heads ? r.heads : tokens, step = heads ? r.out_head_stride : r.out_token_stride;
    if (n > 1 && step < reach) return mkv_fail(MKV_ERR_ARG, "%s: the rows of %s overlap", who, name);
    reach += step * (n - 1);
  }
  return MKV_OK;
}

// Whether outputs of `bytes` go past the caches: where they would not stay in them (256 MB) till they
// are read, and a store of a wave writes whole lines of 128 bytes (other types, smaller heads and
// parts of heads lose 2 to 13%).  Calls that write in turns to two outputs, without / with: 12,000
// tokens of 40 + 8 heads of 128 (147 MB) 52.4 / 55.4 us, 14,000 67.0 / 64.3, 16,000 74.4 / 71.6, 22,141
// 102.5 / 97.5; into the cache 12,000 63.0 / 66.0, 16,000 89.6 / 87.5, 22,141 125 / 119; in place over
// three projections 110 / 102 and 127 / 121.  One output over and over, which the caches absorb, is the
// price: 16,000 62.6 / 71.6, 22,141 85 / 97.5, into the cache 111 / 119.  Between a projection and the
// attention, as in a model's layer of 22,141 tokens, 89 / 97 us of 6.5 ms; the whole does not differ by
// more than it varies (0.3%).
int streams(int64_t bytes, int head_size, int rotary, int64_t eb) {
  return bytes >= int64_t{150} << 20 && eb == 2 && head_size >= 128 && rotary == head_size;
}

template <int ET>
void rotate_launch(int d, dim3 grid, const RotateParams& p, hipStream_t s) {
  const auto launch = [&](auto several) {
    constexpr bool kSeveral = decltype(several)::value;
    if (d == 64)
      norm_rotate_kernel<ET, 64, kSeveral><<<grid, 64 * kWaves, 0, s>>>(p);
    else if (d == 128)
      norm_rotate_kernel<ET, 128, kSeveral><<<grid, 64 * kWaves, 0, s>>>(p);
    else
      norm_rotate_kernel<ET, 256, kSeveral><<<grid, 64 * kWaves, 0, s>>>(p);
  };
  if (p.cut[0].tokens > 1 || p.cut[1].tokens > 1)
    launch(std::true_type());
  else
    launch(std::false_type());
}

template <int ET>
int put_launch(int d, dim3 grid, int threads, int lds, const PutParams& p, hipStream_t s) {
  void (*kernel)(PutParams) =
      d == 64 ? put_kernel<ET, 64> : d == 128 ? put_kernel<ET, 128> : put_kernel<ET, 256>;
  // More than a launch has unasked, with the kernel's own: heads of 256 in blocks of 64 and of 128, of
  // 128 in blocks of 128.  Asked for is always the most that heads of this size need, so that no call
  // takes from another thread's what it has just asked for.
  constexpr int kOwn = kMaxWaves * 2 * sizeof(uint32_t), kMostRows = 128;
  if (lds + kOwn > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, kMostRows * d / 2 * 8);
    if (e != hipSuccess)
      return mkv_fail(MKV_ERR_HIP, "mkv_store_rotated: %d bytes of LDS: %s", lds, hipGetErrorString(e));
  }
  kernel<<<grid, threads, lds, s>>>(p);
  return launched("mkv_store_rotated");
}

}  // namespace

extern "C" int mkv_norm_rotate(const mkv_norm_rotate_desc_t* d, void* stream) {
  const char* who = "mkv_norm_rotate";
  if (d == nullptr) return mkv_fail(MKV_ERR_ARG, "%s: desc is NULL", who);
  if (d->head_size != 64 && d->head_size != 128 && d->head_size != 256)
    return mkv_fail(MKV_ERR_UNSUPPORTED, "%s: head_size %d is not 64, 128 or 256", who, d->head_size);
  if (d->dtype != MKV_BF16 && d->dtype != MKV_F16 && d->dtype != MKV_F32)
    return mkv_fail(MKV_ERR_DTYPE, "%s: dtype %d is not bf16, fp16 or fp32", who, d->dtype);
  if (d->tokens < 0 || d->tokens > INT32_MAX)
    return mkv_fail(MKV_ERR_ARG, "%s: tokens %lld", who, (long long)d->tokens);
  RotateParams p;
  const int64_t eb = d->dtype == MKV_F32 ? 4 : 2;
  int rc = check_turn(who, d->turn, d->head_size, &p.turn);
  if (rc == MKV_OK) rc = check_rows(who, "q", d->q, d->tokens, d->head_size, eb, &p.side[0]);
  if (rc == MKV_OK) rc = check_rows(who, "k", d->k, d->tokens, d->head_size, eb, &p.side[1]);
  if (rc != MKV_OK) return rc;
  if (d->tokens == 0 || d->q.heads + d->k.heads == 0) return MKV_OK;
  if (d->turn.rotary > 0) {
    if (d->positions == nullptr) return mkv_fail(MKV_ERR_ARG, "%s: positions is NULL", who);
    if (d->position_bytes != 4 && d->position_bytes != 8)
      return mkv_fail(MKV_ERR_ARG, "%s: positions of %d bytes", who, d->position_bytes);
    if ((reinterpret_cast<uintptr_t>(d->positions) & (d->position_bytes - 1)) != 0)
      return mkv_fail(MKV_ERR_ALIGN, "%s: positions are not aligned", who);
  }
  p.side[0].stream = p.side[1].stream =
      streams(d->tokens * (d->q.heads + d->k.heads) * d->head_size * eb, d->head_size, d->turn.rotary, eb);
  p.positions = d->positions;
  p.wide = d->position_bytes == 8;
  p.tokens = d->tokens;
  const int at_once = 64 / (d->head_size / 16);
  const int passes = passes_for(d->tokens * (d->q.heads + d->k.heads) / at_once);
  int64_t waves[2];
  for (int i = 0; i < 2; ++i) {
    p.cut[i] = cut_heads(p.side[i].heads, at_once, passes);
    waves[i] = (d->tokens + p.cut[i].tokens - 1) / p.cut[i].tokens * p.cut[i].parts;
  }
  if (waves[0] + waves[1] > UINT32_MAX / 64)
    return mkv_fail(MKV_ERR_UNSUPPORTED, "%s: %lld tokens", who, (long long)d->tokens);
  p.q_waves = static_cast<uint32_t>(waves[0]);
  p.waves = static_cast<uint32_t>(waves[0] + waves[1]);
  const dim3 grid((p.waves + kWaves - 1) / kWaves);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (d->dtype == MKV_BF16)
    rotate_launch<MKV_BF16>(d->head_size, grid, p, s);
  else if (d->dtype == MKV_F16)
    rotate_launch<MKV_F16>(d->head_size, grid, p, s);
  else
    rotate_launch<MKV_F32>(d->head_size, grid, p, s);
  return launched(who);
}

extern "C" int mkv_store_rotated(const mkv_store_rotated_desc_t* d, void* stream) {
  const char* who = "mkv_store_rotated";
  if (d == nullptr) return mkv_fail(MKV_ERR_ARG, "%s: desc is NULL", who);
  PutParams p;
  const mkv_scaled_cache_t& c = d->cache;
  int rc = check_cache(who, c, true, &p.c);
  if (rc == MKV_OK)
    rc = check_step(who, c.block_size, d->block_tables, d->table_stride, d->table_width, d->starts,
                    d->lens, d->requests, d->error_flags, &p.s);
  if (rc != MKV_OK) return rc;
  if (d->dtype != MKV_BF16 && d->dtype != MKV_F16 && d->dtype != MKV_F32)
    return mkv_fail(MKV_ERR_DTYPE, "%s: dtype %d is not bf16, fp16 or fp32", who, d->dtype);
  if (d->tokens < 0 || d->tokens > INT32_MAX)
    return mkv_fail(MKV_ERR_ARG, "%s: tokens %lld", who, (long long)d->tokens);
  const int64_t eb = d->dtype == MKV_F32 ? 4 : 2;
  rc = check_turn(who, d->turn, c.head_size, &p.turn);
  if (rc == MKV_OK) rc = check_rows(who, "q", d->q, d->tokens, c.head_size, eb, &p.q);
  if (rc != MKV_OK) return rc;
  if (d->tokens == 0 || d->requests == 0) return MKV_OK;
  if (d->k == nullptr || d->v == nullptr) return mkv_fail(MKV_ERR_ARG, "%s: k or v is NULL", who);
  const int64_t most = INT64_MAX / 16 / (d->tokens + c.heads);
  for (const int64_t s : {d->k_token_stride, d->k_head_stride, d->v_token_stride, d->v_head_stride})
    if (s < 0 || s > most)
      return mkv_fail(MKV_ERR_ARG, "%s: a stride of k or v is out of range", who);
  p.k = static_cast<const char*>(d->k);
  p.v = static_cast<const char*>(d->v);
  p.k_token = d->k_token_stride * eb;
  p.k_head = d->k_head_stride * eb;
  p.v_token = d->v_token_stride * eb;
  p.v_head = d->v_head_stride * eb;
  if (((reinterpret_cast<uintptr_t>(d->k) | reinterpret_cast<uintptr_t>(d->v) | p.k_token |
        p.k_head | p.v_token | p.v_head) & 15) != 0)
    return mkv_fail(MKV_ERR_ALIGN, "%s: k or v is not 16-byte aligned", who);
  p.tokens = d->tokens;
  const int parts = c.block_size / 16;
  p.group = store_group(d->tokens, d->requests, d->tokens * ((c.heads + 1) / 2), c.block_size);
  // A block's angles serve the heads of a workgroup: four where there is much to do, two where
  // latency counts (measured with 2 / 4: 32 tokens 6.2 / 6.5 us, 4,000 25.8 / 23.5, 22,141 116 / 113).
  const int want = (p.group == 1 ? 2 : 4) / parts;
  const int heads_here = want < 1 ? 1 : c.heads < want ? c.heads : want;
  const int waves = parts * heads_here;
  p.planes = (c.heads + heads_here - 1) / heads_here;
  const int at_once = 64 / (c.head_size / 16);
  p.cut = cut_heads(d->q.heads, at_once, passes_for(d->tokens * d->q.heads / at_once));
  p.q.stream = streams(d->tokens * d->q.heads * c.head_size * eb, c.head_size, d->turn.rotary, eb);
  const int units = (p.group + p.cut.tokens - 1) / p.cut.tokens * p.cut.parts;
  const int q_planes = (units + waves - 1) / waves;
  if ((d->tokens + p.group - 1) / p.group > UINT32_MAX / (64 * waves) || p.planes + q_planes > 65535)
    return mkv_fail(MKV_ERR_UNSUPPORTED, "%s: %lld tokens", who, (long long)d->tokens);
  const dim3 grid(static_cast<unsigned>((d->tokens + p.group - 1) / p.group),
                  static_cast<unsigned>(p.planes + q_planes));
  const int rows = waves * p.cut.tokens;  // (cos, sin) of a block's rows, or of the waves' tokens
  const int lds = (c.block_size > rows ? c.block_size : rows) * p.turn.half * 8;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (d->dtype == MKV_BF16) return put_launch<MKV_BF16>(c.head_size, grid, 64 * waves, lds, p, s);
  if (d->dtype == MKV_F16) return put_launch<MKV_F16>(c.head_size, grid, 64 * waves, lds, p, s);
  return put_launch<MKV_F32>(c.head_size, grid, 64 * waves, lds, p, s);
}
