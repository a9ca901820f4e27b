// scaled_attend.h -- the kernels of causal attention over the block-scaled 8-bit cache for gfx950:
// a tile of query rows over a range of tokens.  Over a request's whole history for
// scaled_attend.hip; over what a group of requests shares, and over what a request has of its
// own, for shared_attend.hip.
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
// fp16 queries, and for tiles of requests of few rows that share tokens (K::kTwoTerms): these keep
// what they have alone, however many they are (32 of them 34.1 -> 37.9 us, 96 99 -> 117, 32 of
// heads of 64 28 -> 29, of 256 60 -> 64; 31 beside a chunk of 1,024 386 -> 407).  For other bf16
// queries it rounds p to bf16, by half a step of it, 2^-8, as the output itself is: a second
// product would take 2,048 tokens over 22,141 from 1,072 to 1,380 us.
// fp16 queries multiply the bare codes (exact in fp16, where a scaled value may not be) and
// the scale is applied to s_j.
//
// Layout.  Both products are computed transposed, S^T = K Q^T and O^T = V^T P^T: a lane then
// holds scores of one query row, its statistics are one register, and P^T leaves the first
// product in the lanes where the second one wants it.  The order of the tokens within a step
// and of the dimensions is chosen per operand so that no value moves between lanes.

#pragma once

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

// What a tile goes over: a request's whole history, what a group of requests shares, or what a
// request has behind that.
enum Over { kHistory, kShared, kOwn };

// A batch whose requests begin, in groups, with the same tokens: requests [groups[g], groups[g + 1])
// with the first shared[g], in whole blocks, of groups[g]'s table.
struct DevGroups {
  const int32_t* groups;
  const int32_t* shared;
  int32_t count;
};

// Where a row's results lie: row `at` of all tiles of a launch, in `parts` parts.
struct RowPlace {
  int32_t shared_at, shared_parts, own_at, own_parts;
};

struct GroupedParams : AttendParams {
  DevGroups g;
  RowPlace* places;     // of each (token, query head of a KV head's group)
  int32_t shared_rows;  // of the tiles over what is shared: their rows, the least tokens of a part
  int32_t shared_per;   // and the most parts
  int32_t shared_splits;
  int32_t launch;       // this launch among those over the own tokens, 0 or 1
};

// A tile: `BM` query rows (token, query head of the group) of one request, heads fastest.
// Request r's tiles begin at starts[r] * group / BM + r: that leaves each at least as many as
// it needs, from what the host knows alone, and tiles beyond a request's rows do nothing.
// (Over what is shared: of one group of requests, from its first one's row on, in the same way.)
struct Tile {
  Over over;
  int64_t s0;     // the request's first token
  int64_t row0;   // the tile's first row in the request
  int64_t first;  // position of the request's first new token
  int rows;       // rows of the tile, 1 to BM
  int request;    // whose table is read
  int from;       // the first token of the range
  int full;       // tokens that every row sees
  int keys;       // tokens that some row sees
  int parts;      // parts its tokens are cut into, and the tokens of each
  int per;
  int last;       // shared: the group's last request
  // own: the request's first row in its group, the group's first tile and the parts of what it
  // shares (0: nothing, or no group)
  int64_t shared_row, shared_tile;
  int shared_parts;
};

// `n` tokens in parts of at least `least` each and at most `splits` of them: the tokens of one.
__device__ __forceinline__ int part_size(int n, int splits, int least) {
  const int per = (n / splits + 64) & ~63;  // at least n / splits
  return per > least ? per : least;
}
__device__ __forceinline__ int part_count(int n, int per) { return n > per ? (n + per - 1) / per : 1; }

// The tokens that a table of the cache has room for, of `len`; flagged where that is not all.
__device__ __forceinline__ int64_t within(const DevCache& c, const DevStep& s, int64_t len) {
  const int64_t room = static_cast<int64_t>(s.table_width) << c.bs_shift;
  if (len > room && threadIdx.x == 0) raise(s.flags, MKV_FLAG_SRC_RANGE);
  int64_t most = len < room ? len : room;
  if (c.num_blocks == 0) {  // no block to read, whatever the table says
    if (most > 0 && threadIdx.x == 0) raise(s.flags, MKV_FLAG_SRC_RANGE);
    most = 0;
  }
  return most;
}

// A group of requests: its first and last (exclusive), its tokens' rows and what it shares.
struct Group {
  int index, a, b, shared;
  int64_t s0, s1;
};

// The last group with value(its first request, its number) at most `at`, as last_at_most finds it; -1 if
// there is none.  Groups that begin behind or in front of the batch, and those with value -1, are
// passed over wherever they stand, so that they lead nobody away from the others: where one is a
// probe, the next that is none of them stands for its 64.
template <typename F>
__device__ __forceinline__ int last_group(const DevGroups& d, int requests, int64_t at, F value) {
  const int lane = threadIdx.x & 63;
  const auto value_of = [&](int i) {
    const int a = d.groups[i];
    return a >= 0 && a < requests ? value(a, i) : int64_t{-1};
  };
  int base = 0;
  if (d.count > 64) {
    int i = lane * 64;
    const int end = min(i + 64, d.count);
    int64_t x = -1;
    while (i < end && (x = value_of(i)) < 0) ++i;
    const uint64_t hit = __ballot(x >= 0 && x <= at);
    if (hit == 0) return -1;
    base = (63 - __builtin_clzll(hit)) * 64;
  }
  const int i = base + lane;
  const int64_t x = i < d.count ? value_of(i) : -1;
  const uint64_t hit = __ballot(x >= 0 && x <= at);
  return hit == 0 ? -1 : base + 63 - __builtin_clzll(hit);
}

// Group `g`; what a valid one shares is 0 or more whole blocks.
__device__ __forceinline__ bool read_group(const DevCache& c, const DevStep& s, const DevGroups& d,
                                           int64_t tokens, int g, Group& out) {
  out.index = g;
  out.a = d.groups[g];
  out.b = d.groups[g + 1];
  const int shared = d.shared[g];
  if (out.a < 0 || out.b <= out.a || out.b > s.requests) return false;
  out.s0 = s.starts[out.a];
  out.s1 = s.starts[out.b];
  if (out.s0 < 0 || out.s1 < out.s0 || out.s1 > tokens) return false;
  const int64_t n = within(c, s, shared);
  out.shared = n <= 0 ? 0 : static_cast<int>(n >> c.bs_shift << c.bs_shift);
  return true;
}

// The group of request r with the rows [s0, s1), one wave; false where it is in none.
__device__ __forceinline__ bool group_of(const DevCache& c, const DevStep& s, const DevGroups& d,
                                         int64_t tokens, int r, int64_t s0, int64_t s1, Group& out) {
  const int g = last_group(d, s.requests, r, [](int a, int) { return static_cast<int64_t>(a); });
  return g >= 0 && read_group(c, s, d, tokens, g, out) && r >= out.a && r < out.b &&
         s0 >= out.s0 && s1 <= out.s1;
}

// The first tile of group g, whose rows begin at `row`, in a launch of `rows` rows a tile: rounded
// up with the group's number, which leaves each group exactly as many as its rows may need and
// one group none too many.  (An empty tile's workgroups end early, but where the chip is filled
// once they leave others two to a CU: 32 parts of one tile 26.9 us, beside as many empty 37.4.)
__device__ __forceinline__ int64_t shared_begin(int64_t row, int rows, int g) {
  return (row + static_cast<int64_t>(g) * (rows - 1)) / rows;
}

// The group that a tile over what is shared may be of.
template <typename P>
__device__ __forceinline__ int shared_group(const P& p, int64_t tile, int rows) {
  const int32_t* starts = p.s.starts;
  const int64_t group = p.group, tokens = p.tokens;
  return last_group(p.g, p.s.requests, tile, [=](int a, int i) {
    const int64_t s0 = starts[a];
    return s0 >= 0 && s0 <= tokens ? shared_begin(s0 * group, rows, i) : int64_t{-1};
  });
}

// (GROUPED: over what `t.over` says; otherwise over histories.)
template <bool GROUPED, int BM, typename P>
__device__ __forceinline__ bool find_tile(const P& p, int64_t tile, Tile& t) {
  const int32_t* starts = p.s.starts;
  const int group = p.group;
  if constexpr (GROUPED) if (t.over == kShared) {
    const int g = p.g.count == 1 ? 0 : shared_group(p, tile, BM);
    Group of;
    if (g < 0 || !read_group(p.c, p.s, p.g, p.tokens, g, of)) return false;
    t.request = of.a;
    t.last = of.b - 1;
    t.s0 = of.s0;
    t.row0 = (tile - shared_begin(of.s0 * group, BM, g)) * BM;
    const int64_t rows = (of.s1 - of.s0) * group - t.row0;
    if (t.row0 < 0 || rows <= 0 || of.shared == 0) return false;
    t.rows = static_cast<int>(rows < BM ? rows : BM);
    t.keys = of.shared;
    t.from = 0;
    t.first = 0;
    t.per = part_size(t.keys, p.splits, p.per);
    t.parts = part_count(t.keys, t.per);
    return true;
  }
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
  const int64_t most = within(p.c, p.s, len);
  const int64_t lo = t.first + t.row0 / group + 1;
  const int64_t hi = t.first + (t.row0 + t.rows - 1) / group + 1;
  const int64_t keys = hi < most ? hi : most;
  t.keys = keys < 0 ? 0 : static_cast<int>(keys);
  t.full = lo < 0 ? 0 : static_cast<int>(lo < t.keys ? lo : t.keys);
  t.from = 0;
  if constexpr (GROUPED) {
    Group of;
    t.shared_parts = 0;
    bool found = group_of(p.c, p.s, p.g, p.tokens, r, t.s0, s1, of) && of.shared > 0;
    if (found) {
      t.shared_row = (t.s0 - of.s0) * group + t.row0;
      t.shared_tile = shared_begin(of.s0 * group, p.shared_rows, of.index);
      if (p.g.count > 64) {
        // Do the tiles that have the rows find the group?  With up to 64 groups always; beyond, starts
        // that descend may hide it from them, and its parts would be read and never written.  (100
        // groups of four requests 53.2 -> 55.1 us, 1,000 of two 127 -> 135.)
        const int64_t first = t.shared_tile + t.shared_row / p.shared_rows;
        const int64_t last = t.shared_tile + (t.shared_row + t.rows - 1) / p.shared_rows;
        found = shared_group(p, first, p.shared_rows) == of.index &&
                (last == first || shared_group(p, last, p.shared_rows) == of.index);
      }
    }
    if (found) {
      t.from = of.shared;
      t.shared_parts = part_count(of.shared, part_size(of.shared, p.shared_splits, p.shared_per));
      if (t.keys < t.from) t.keys = t.full = t.from;  // nothing of its own
    }
  }
  t.per = part_size(t.keys - t.from, p.splits, p.per);
  t.parts = part_count(t.keys - t.from, t.per);
  return true;
}

// Over what is shared: whether every row sees all of it, as nearly always, those that stand behind
// it.  The requests' lengths are waited for here, not before the tile's table is looked up.
template <typename P>
__device__ __forceinline__ void find_full(const P& p, Tile& t) {
  int64_t least = t.keys;
  for (int r = t.request + (threadIdx.x & 63); r <= t.last; r += 64) {
    const int64_t n = static_cast<int64_t>(p.s.starts[r + 1]) - p.s.starts[r];
    const int64_t sees = n > 0 ? p.s.lens[r] - n + 1 : t.keys;
    least = sees < least ? sees : least;
  }
  t.full = __all(least >= t.keys) ? t.keys : 0;
}

// Rows of a request beside a long chunk, at most, that has a launch of its own with others of so few.
constexpr int kBesideRows = 16;

// Over what is shared: whether a row of the tile is of such a request.
template <typename P>
__device__ __forceinline__ bool of_few_rows(const P& p, const Tile& t) {
  const int64_t from = t.s0 * p.group + t.row0, to = from + t.rows;
  bool few = false;
  for (int r = t.request + (threadIdx.x & 63); r <= t.last; r += 64) {
    const int64_t a = static_cast<int64_t>(p.s.starts[r]) * p.group;
    const int64_t b = static_cast<int64_t>(p.s.starts[r + 1]) * p.group;
    few = few || (b - a <= kBesideRows && a < to && b > from);
  }
  return __any(few);
}

// Tokens that a row of the tile sees, at most t.keys.
template <bool GROUPED, typename P>
__device__ __forceinline__ int row_sees(const P& p, const Tile& t, int64_t token) {
  int64_t sees = t.first + token + 1;
  if constexpr (GROUPED) if (t.over == kShared) {
    if (t.full == t.keys) return t.keys;
    int lo = t.request, hi = t.last;  // the last request that begins at or before the row
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (p.s.starts[mid] <= t.s0 + token)
        lo = mid;
      else
        hi = mid - 1;
    }
    sees = static_cast<int64_t>(p.s.lens[lo]) - p.s.starts[lo + 1] + t.s0 + token + 1;
  }
  return static_cast<int>(sees < 0 ? 0 : (sees < t.keys ? sees : t.keys));
}

// Notes where the results of a tile's rows will lie.
template <int BM>
__device__ __forceinline__ void note_places(const GroupedParams& p, const Tile& t, int64_t tile) {
  RowPlace* to = p.places + t.s0 * p.group + t.row0;
  for (int i = threadIdx.x; i < t.rows; i += blockDim.x) {
    RowPlace x = {0, t.shared_parts, static_cast<int32_t>(tile * BM + i), t.parts | p.launch << 16};
    if (t.shared_parts > 0) {
      const int64_t row = t.shared_row + i;
      x.shared_at = static_cast<int32_t>((t.shared_tile + row / p.shared_rows) * p.shared_rows +
                                         row % p.shared_rows);
    }
    to[i] = x;
  }
}

// Flags groups that leave the requests or descend, and tokens shared below zero.
__device__ __forceinline__ void check_groups(const DevStep& s, const DevGroups& d) {
  if (s.flags == nullptr) return;
  bool bad = false;
  for (int g = threadIdx.x; g < d.count; g += blockDim.x)
    bad = bad || d.groups[g] < 0 || d.groups[g + 1] < d.groups[g] || d.groups[g + 1] > s.requests ||
          d.shared[g] < 0;
  if (bad) raise(s.flags, MKV_FLAG_SPAN);
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
// spills 44 registers; beside tiles of few rows over own tokens 42 to 87.)  A chunk of 2,048 tokens over 22,141, 40 query heads of 128 (0.97 TFLOP),
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

// -------------------------------------------------------------------------------- kernels
//
// One body for both, so that a launch may hold tiles of both (K::kFew: row tiles of 16 of the one,
// 0 without; K::kMany) and a launch of one of them is compiled as if it stood alone.  (As two
// functions that kernels call, one for few rows and one for many, the same code held more registers,
// spilled some and ran up to 12% slower.)  K::pick says which tile, KV head and part a workgroup has, in which section, if any,
// and (K::kGrouped) over what.  The body is a text of its own, included: called as a function by every
// kernel, the same code took 127 us for a batch's next tokens in place of 111.5.

enum Section { kNothing, kFewRows, kManyRowsTile };

template <int D, int RT>
struct FewLds {
  __attribute__((aligned(16))) float o[kFewWaves][D * 16];
  float ml[kFewWaves][16 * RT][2];
};

template <int D>
struct ManyLds {
  __attribute__((aligned(16))) char k[2][128 * D];
  __attribute__((aligned(16))) char v[2][128 * D];
  int odd[2];
};

// A launch's LDS: of one section, or either's.
template <int D, int RT, bool MANY>
union Lds {
  FewLds<D, RT> few;
  ManyLds<D> many;
};
template <int D, int RT>
union Lds<D, RT, false> {
  FewLds<D, RT> few;
};
template <int D>
union Lds<D, 0, true> {
  ManyLds<D> many;
};

template <typename K, int D>
constexpr int min_waves() {
  constexpr int few = K::kFew == 0 ? 8 : few_waves<D, K::kFew == 0 ? 1 : K::kFew>();
  constexpr int many = !K::kMany ? 8 : D == 256 ? 1 : 2;
  return few < many ? few : many;
}

template <typename K, bool F16, int D>
__global__ __launch_bounds__(256, (min_waves<K, D>())) void attend_kernel(typename K::Params params) {
  __shared__ Lds<D, K::kFew, K::kMany> lds;
#include "scaled_attend_body.h"
}

// The same for a kernel that chooses between two K.
template <typename K, bool F16, int D>
__device__ __forceinline__ void attend_tile(const typename K::Params& params, Lds<D, K::kFew, K::kMany>& lds) {
#include "scaled_attend_body.h"
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

constexpr int64_t kWantFew = 4096;
constexpr int64_t kMostParts = 8;  // times as many parts as wanted that a workspace has room for

// A tile's rows by those of the largest request, and the parts: of one size for all requests,
// so that long and short histories fill the chip alike, about `want` workgroups if every
// request were the longest.
inline Shape shape_for(const mkv_attend_desc_t& d, int64_t each, int32_t from, int32_t to) {
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

// An attention call's cache, requests, queries and outputs, but for their addresses.
inline int check_attend(const char* who, const mkv_attend_desc_t& d, AttendParams* p) {
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
  return MKV_OK;
}

// And their addresses: out's rows lie apart, and the workspace has `need` bytes.
inline int check_attend_rows(const char* who, const mkv_attend_desc_t& d, const AttendParams& p,
                             int64_t need) {
  if (d.q == nullptr || d.out == nullptr)
    return mkv_fail(MKV_ERR_ARG, "%s: q or out is NULL", who);
  if (((reinterpret_cast<uintptr_t>(d.q) | reinterpret_cast<uintptr_t>(d.out) | p.q_token |
        p.q_head | p.out_token | p.out_head) & 15) != 0)
    return mkv_fail(MKV_ERR_ALIGN, "%s: q or out is not 16-byte aligned", who);
  // out's rows: the smaller stride passes a row, the larger one all that the smaller reaches
  const bool heads_first = d.out_head_stride <= d.out_token_stride;
  int64_t reach = d.cache.head_size;
  for (const bool heads : {heads_first, !heads_first}) {
    const int64_t n = heads ? d.q_heads : d.tokens;
    const int64_t step = heads ? d.out_head_stride : d.out_token_stride;
    if (n > 1 && step < reach) return mkv_fail(MKV_ERR_ARG, "%s: out's rows overlap", who);
    reach += step * (n - 1);
  }
  if (need > 0 && (d.workspace == nullptr || d.workspace_bytes < need))
    return mkv_fail(MKV_ERR_ARG, "%s: workspace of %lld bytes, %lld needed", who,
                    (long long)d.workspace_bytes, (long long)need);
  if ((reinterpret_cast<uintptr_t>(d.workspace) & 15) != 0)
    return mkv_fail(MKV_ERR_ALIGN, "%s: workspace is not 16-byte aligned", who);
  return MKV_OK;
}

}  // namespace
