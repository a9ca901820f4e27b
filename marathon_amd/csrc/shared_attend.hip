// shared_attend.hip -- attention of a batch whose requests begin, in groups, with the same
// cached tokens, for gfx950: what a group shares is read once for all of its rows.
//
// Mathematics.  A row's softmax over the tokens [0, shared) and [shared, len) is joined from the
// two ranges' largest score m, sum l and unnormalised output o:
//     out = sum_i o_i 2^(m_i - m) / sum_i l_i 2^(m_i - m),   m = max m_i.
// Over the first range the rows of all requests of a group are one matrix against one matrix:
// a launch over (group, KV head) with the rows of up to 128 (token, query head) a tile, where
// attention for each request alone would read those tokens once a request.  Over the second a
// launch over the requests.  Both are scaled_attend.h's kernels over a range of tokens, and leave
// parts; one more launch joins every row's.
//
// The launch over own tokens notes where each row's parts lie, so that the join waits for one
// lookup in front of its data and not for the chain that finds a row's request, group and tiles.

#include "marathon_kvstep.h"
#include "scaled_attend.h"

#include <algorithm>
#include <cmath>

#pragma clang fp contract(off)

namespace {

// ----------------------------------------------------------------- both ranges, one launch
//
// The two ranges' tiles run side by side: over what is shared a tile is bound by the matrix
// instructions and, over own tokens, a few rows by memory's latency.

struct BothParams {
  GroupedParams own;
  // of the tiles over what is shared
  float* part_o;
  float* part_ml;
  int64_t shared_units, own_units;  // workgroups
  int32_t shared_tiles, own_tiles;
};

// Tiles of SHARED rows over what is shared and of OWN rows over own tokens: 16 or 32 take the
// section of few rows, 128 that of many, there with p of bf16 queries in two terms (TWO) or one.
template <int SHARED, int OWN, bool TWO = (OWN < kManyRows)>
struct Both {
  typedef BothParams Params;
  static constexpr bool kGrouped = true, kMany = SHARED == kManyRows, kTwoTerms = TWO;
  static constexpr int kFew = OWN == kManyRows ? 0 : OWN / 16;
  static_assert(kMany || SHARED == OWN, "one section of few rows");

  static __device__ __forceinline__ Section pick(const Params& p, unsigned& tile, int& head, int& part,
                                                 Over& over) {
    uint32_t unit = blockIdx.x;
    const uint32_t heads = p.own.c.heads;
    if (unit < p.shared_units) {
      // the tiles of one (part, head) go to one XCD, whose L2 then serves all of them but the first
      const uint32_t in = unit % (8 * p.shared_tiles), pair = unit / (8 * p.shared_tiles) * 8 + in % 8;
      tile = in / 8;
      head = pair % heads;
      part = pair / heads;
      over = kShared;
      if (part >= p.own.shared_splits) return kNothing;
      return kMany ? kManyRowsTile : kFewRows;
    }
    unit -= p.shared_units;
    if (unit >= p.own_units) {  // (a workgroup of its own: no register is held for it)
      check_starts(p.own.s, p.own.tokens, false);
      check_groups(p.own.s, p.own.g);
      return kNothing;
    }
    const uint32_t tiles = p.own_tiles, y = unit / tiles;
    head = y % heads;
    part = y / heads;
    tile = (unit + part) % tiles;  // turned by the part, as over whole histories
    over = kOwn;
    return OWN == kManyRows ? kManyRowsTile : kFewRows;
  }

  static __device__ __forceinline__ GroupedParams params(const Params& p, Over over) {
    GroupedParams x = p.own;
    if (over == kShared) {
      x.part_o = p.part_o;
      x.part_ml = p.part_ml;
      x.splits = x.shared_splits;
      x.per = x.shared_per;
    }
    return x;
  }
};

// bf16 chunks beside another launch over the own tokens of requests of few rows, whose rows over what
// is shared are here: their tiles take two terms of p, the chunks' one.
template <int D>
__global__ __launch_bounds__(256, (min_waves<Both<kManyRows, kManyRows>, D>())) void chunks_beside_kernel(
    BothParams params) {
  typedef Both<kManyRows, kManyRows, false> One;
  __shared__ Lds<D, One::kFew, One::kMany> lds;
  bool few = false;
  if (blockIdx.x < params.shared_units) {
    unsigned tile;
    int head, part;
    Tile t;
    One::pick(params, tile, head, part, t.over);
    const auto& p = One::params(params, t.over);
    few = find_tile<true, kManyRows>(p, tile, t) && of_few_rows(p, t);
  }
  if (uni(few))
    attend_tile<Both<kManyRows, kManyRows, true>, false, D>(params, lds);
  else
    attend_tile<One, false, D>(params, lds);
}

// ------------------------------------------------------------------ the parts' results joined

// Parts of a launch: results of `rows` rows a tile, tiles by KV heads by parts.
struct PartSet {
  float* o;
  float* ml;
  int32_t rows;
  int32_t splits;
  int64_t tiles;
};

struct JoinParams {
  const int32_t* starts;
  int32_t requests;
  int64_t tokens;
  const RowPlace* places;
  PartSet sets[3];  // shared, own (few rows, or all), own (many rows)
  char* out;
  int64_t out_token, out_head;  // bytes
  int32_t heads, group;
};

// WAVES waves join a row, or one wave each of four rows: the parts' m and l, one a lane, then
// their outputs, D / 4 lanes a part.  What the places say is kept within the parts, whatever was
// changed between the launches.
template <bool F16, int D, int WAVES>
__global__ __launch_bounds__(256) void shared_join_kernel(JoinParams p) {
  constexpr int kLanes = D / 4, kGroups = 64 / kLanes * WAVES;  // groups of lanes at a row's parts
  __shared__ f32x4 s_o[WAVES][kLanes];
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const int q_heads = p.heads * p.group;
  const uint32_t unit = WAVES > 1 ? blockIdx.x : blockIdx.x * 4 + wave;
  const int64_t token = unit / q_heads;
  if (token >= p.tokens) return;
  const int h = unit % q_heads, head = h / p.group;
  const RowPlace at = p.places[token * p.group + h % p.group];
  const int32_t* starts = p.starts;
  const int r = last_at_most(p.requests, token, [starts](int i) { return starts[i]; });
  if (r < 0) return;
  const int64_t s0 = starts[r], s1 = starts[r + 1];
  if (s0 < 0 || token < s0 || token >= s1 || s1 > p.tokens) return;  // nobody's
  const PartSet shared = p.sets[0], mine = (at.own_parts >> 16) & 1 ? p.sets[2] : p.sets[1];
  const auto first_of = [&](const PartSet& s, int32_t place) {
    int64_t tile = place / s.rows;
    tile = tile < 0 ? 0 : tile < s.tiles ? tile : s.tiles - 1;
    const int row = place < 0 ? 0 : place % s.rows;
    return (tile * p.heads + head) * s.splits * s.rows + row;
  };
  const int ns = min(max(at.shared_parts, 0), shared.splits);
  const int no = min(max(at.own_parts & 0xFFFF, 0), mine.splits);
  const int64_t from_s = ns > 0 ? first_of(shared, at.shared_at) : 0;
  const int64_t from_o = first_of(mine, at.own_at);
  const int d = lane % kLanes, grp = lane / kLanes + (WAVES > 1 ? wave * (64 / kLanes) : 0), n = ns + no;
  f32x4 o = {0, 0, 0, 0};
  float top = -kInf, sum = 0.0f;
  for (int base = 0; base < n; base += 64) {
    const int i = base + lane, here = min(64, n - base);
    float m = -kInf, l = 0.0f;
    if (i < n) {
      const float* ml = i < ns ? shared.ml + 2 * (from_s + static_cast<int64_t>(i) * shared.rows)
                               : mine.ml + 2 * (from_o + static_cast<int64_t>(i - ns) * mine.rows);
      m = ml[0];
      l = ml[1];
    }
    // the first outputs are on their way while m and l are
    const auto part_o = [&](int j) {
      const int k = base + min(j, here - 1);
      const float* x = k < ns ? shared.o + (from_s + static_cast<int64_t>(k) * shared.rows) * D
                              : mine.o + (from_o + static_cast<int64_t>(k - ns) * mine.rows) * D;
      return *reinterpret_cast<const f32x4*>(x + 4 * d);
    };
    f32x4 x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = part_o(grp + u * kGroups);
    float now = m;
    for (int y = 32; y > 0; y >>= 1) now = fmaxf(now, __shfl_xor(now, y));
    now = fmaxf(now, top);
    const float b = now == -kInf ? 0.0f : now, old = fast_exp2(top - b), f = fast_exp2(m - b);
    float part = l * f;
    for (int y = 32; y > 0; y >>= 1) part += __shfl_xor(part, y);
    sum = sum * old + part;
    o *= old;
    top = now;
    for (int j = grp; j - grp < here; j += 4 * kGroups) {  // (alike in every lane)
      if (j != grp) {
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = part_o(j + u * kGroups);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int k = j + u * kGroups;
        const float w = __shfl(f, min(k, 63));
        if (k < here) o += x[u] * w;
      }
    }
  }
#pragma unroll
  for (int x = kLanes; x < 64; x <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], x);
  if constexpr (WAVES > 1) {
    if (lane < kLanes) s_o[wave][d] = o;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) o += s_o[w][d];
  }
  if (lane >= kLanes) return;
  o *= sum == 0.0f ? 0.0f : 1.0f / sum;
  *reinterpret_cast<u32x2*>(p.out + token * p.out_token + h * p.out_head + d * 8) =
      u32x2{out_pair<F16>(o[0], o[1]), out_pair<F16>(o[2], o[3])};
}

// ------------------------------------------------------------------------------- host

// The launches of a call: over what is shared (none without groups), and over own tokens one or
// two (scaled_attend.hip's rule: a long chunk beside decoding requests has one of its own).
struct Plan {
  Shape shared;
  Shape own[2];
  int owns;
};

// What a kernel's steps take, in us: of `tokens` by a workgroup that is alone on its CU, and of a
// CU's time where it has as many as fit; and how many workgroups run at once.  Measured on whole
// calls, for 16 rows a tile, 32 and 128.
struct Cost {
  int tokens;
  double alone, full;
  int slots;
};

Cost cost_of(int rows, int head_size, bool f16) {
  const int i = head_size == 64 ? 0 : head_size == 128 ? 1 : 2;
  if (rows == kManyRows) {
    constexpr double kAlone[] = {1.35, 1.6, 5.5}, kFull[] = {0.85, 1.06, 5.0};
    constexpr int kSlots[] = {768, 512, 256};
    // p's second product, and scores scaled one by one (bf16's second product alone as none: with 1.4
    // 32 requests took 41.0 us against 37.9, heads of 256 60.4 against 63.5, 13 other batches the same)
    const double more = f16 ? 1.4 : 1.0;
    return {64, kAlone[i] * more, kFull[i] * more, kSlots[i]};
  }
  constexpr double kAlone[] = {1.1, 1.6, 3.4}, kFull[] = {0.8, 1.5, 3.4};
  constexpr int kSlots[2][3] = {{1024, 1024, 512}, {768, 512, 256}};
  const double more = rows == 32 ? 1.6 : 1.0;
  return {32 * kFewWaves, kAlone[i] * more, kFull[i] * more, kSlots[rows == 32][i]};
}

// The parts of both ranges, by the time that they are expected to take: the longest workgroup of
// either, or all of the work over the chip, whichever is more, and the join, which reads a row's
// results once for each part.  Against a sweep of the parts over 16 batches (2 to 96 requests, 1 to 8
// KV heads) its choice is within 8% of the best for 13 of them, and 10 to 30% off where groups differ
// most in what they share, own histories are the longer ones, or heads are of 256.
void choose_parts(const mkv_attend_shared_desc_t& d, int64_t shared_most, int64_t own_most, Shape* s,
                  Shape* o) {
  constexpr double kCus = 256, kStart = 5.0, kStartFull = 1.2, kJoin = 1.5e-6;  // (a value of a part)
  const mkv_attend_desc_t& a = d.attend;
  const bool f16 = a.dtype == MKV_F16;
  const Cost cs = cost_of(s->rows, a.cache.head_size, f16), co = cost_of(o->rows, a.cache.head_size, f16);
  const double heads = a.cache.heads;
  const double part = 0.05 + kJoin * static_cast<double>(a.tokens) * a.q_heads * a.cache.head_size;
  // Tiles that have work, if groups and requests are alike.  Own histories, whose lengths only the GPU
  // knows, are taken to be 0.55 of the longest on average: one of 8,000 tokens beside 31 of 200 77.6 us,
  // where 0.8 or 1 took 98 or 143; the price is paid by those that are alike, 24 of 4,000 behind 2,000
  // shared 55.8 (47.4 both), 8 of 8,000 behind 4,000 50.5 (50.5 and 40.2).
  const auto alike = [](const Shape& x, int64_t each, int64_t count) {
    return static_cast<double>(std::min((each + x.rows - 1) / x.rows * count, x.tiles));
  };
  // Groups may share lengths that differ, which only the GPU knows: one has the longest range, the
  // others are taken to have three quarters of it.  Against the longest for all: 46 us to 51.5 for
  // 3 groups of 14,693 to 30,000 tokens, 67.3 to 71.7 for 8 of 3,721 to 12,000, 16.0 to 15.3 for 3 of
  // 1,457 to 3,000; four alike or nearly so, the same.
  const double mean = 0.75 + (d.n_groups > 0 ? 0.25 / d.n_groups : 0.25);
  const double st = mean * alike(*s, s->each, d.n_groups) * heads, ot = alike(*o, o->each, a.requests) * heads;
  const double spare = 0.3 * (static_cast<double>(o->tiles) * heads - ot);  // (these end early)
  const int64_t ss = (shared_most + cs.tokens - 1) / cs.tokens, os = (own_most + co.tokens - 1) / co.tokens;
  const auto most = [](int64_t n) { return n < kMaxSplits ? n < 1 ? 1 : static_cast<int>(n) : kMaxSplits; };
  const int most_s = d.n_groups > 0 ? most(shared_most / 128) : 1, most_o = most(own_most / 128);
  double best = 1e30;
  int n = 1, m = 1;
  for (int i = 1; i <= most_s; i += (i + 3) / 4) {
    const double units = st * i, steps = static_cast<double>((ss + i - 1) / i);
    const double load = units <= kCus ? 1.0 : std::min(std::ceil(units / kCus), cs.slots / kCus);
    const double path = ss > 0 ? kStart + steps * std::max(cs.alone, load * cs.full) : 0.0;
    const double work = ss > 0 ? units * (kStartFull + steps * cs.full) : 0.0;
    for (int j = 1; j <= most_o; j += (j + 3) / 4) {
      const double own = ot * (j * kStartFull + 0.55 * static_cast<double>(os) * co.full);
      const double own_path = kStart + static_cast<double>((os + j - 1) / j) * co.alone;
      // where they do not all run at once, the chip waits for a quarter of a last one
      const double wait = units > cs.slots ? path : units + (ot + spare) * j > cs.slots ? own_path : 0.0;
      const double time = std::max(std::max(path, own_path), (work + own) / kCus + 0.25 * wait) + (i + j) * part;
      if (time < best) best = time, n = i, m = j;
    }
  }
  const auto cut = [heads](int64_t tokens, int parts, Shape* x) {
    const int64_t per = (tokens / parts + 64) / 64 * 64;
    x->per = static_cast<int>(per < 1 << 30 ? per : 1 << 30);
    x->splits = static_cast<int>(tokens > per ? (tokens + per - 1) / per : 1);
    // Every tile has room for its parts, also those that hints or a padded batch leave without
    // work: a workspace is bounded as that of whole histories is, by fewer and longer parts.
    const int64_t all = x->tiles * static_cast<int64_t>(heads);
    const int64_t most = kMostParts * (x->rows == kManyRows ? 1536 : kWantFew);
    if (all * x->splits > most) x->splits = static_cast<int>(all < most ? most / all : 1);
  };
  cut(shared_most, n, s);
  cut(own_most, m, o);
}

int check(const mkv_attend_shared_desc_t& d, GroupedParams* p, Plan* plan) {
  const char* who = "mkv_attend_shared";
  const mkv_attend_desc_t& a = d.attend;
  int rc = check_attend(who, a, p);
  if (rc != MKV_OK) return rc;
  if (d.n_groups < 0 || d.n_groups > MKV_MAX_REQUESTS)
    return mkv_fail(MKV_ERR_ARG, "%s: groups %d outside [0, %d]", who, d.n_groups, MKV_MAX_REQUESTS);
  if (d.n_groups > 0 && (d.groups == nullptr || d.shared == nullptr))
    return mkv_fail(MKV_ERR_ARG, "%s: groups or shared is NULL", who);
  if (d.max_shared < 0) return mkv_fail(MKV_ERR_ARG, "%s: max_shared %d", who, d.max_shared);
  p->g = DevGroups{d.groups, d.shared, d.n_groups};

  const int64_t new_most = a.max_new > 0 && a.max_new < a.tokens ? a.max_new : a.tokens;
  const int64_t each = new_most * p->group;
  const int64_t rest = (a.tokens - new_most) * p->group;
  if (each >= 2048 && a.requests > 1 && rest <= kBesideRows * static_cast<int64_t>(a.requests - 1)) {
    plan->own[0] = shape_for(a, kBesideRows, 0, kBesideRows);
    plan->own[1] = shape_for(a, each, kBesideRows + 1, INT32_MAX);
    plan->owns = 2;
  } else {
    plan->own[0] = shape_for(a, each, 0, INT32_MAX);
    plan->owns = 1;
  }
  mkv_attend_desc_t s = a;  // a group's rows as one request's
  s.requests = d.n_groups > 0 ? d.n_groups : 1;
  s.max_len = d.max_shared;
  const int64_t rows = a.tokens * p->group;
  plan->shared = shape_for(s, (rows + s.requests - 1) / s.requests, 0, INT32_MAX);
  // one section of few rows, and many own rows beside many shared ones
  Shape& own = plan->own[plan->owns - 1];
  if (own.rows > plan->shared.rows)
    plan->shared.rows = own.rows;
  else if (plan->shared.rows == 32 && own.rows == 16)
    own = shape_for(a, 32, 0, INT32_MAX);
  plan->shared.tiles = (rows + static_cast<int64_t>(s.requests) * (plan->shared.rows - 1)) / plan->shared.rows;
  const int64_t room = static_cast<int64_t>(a.table_width) * a.cache.block_size;
  const auto known = [room](int32_t most) { return most > 0 && most < room ? most : room; };
  if (plan->owns == 1)
    choose_parts(d, d.n_groups > 0 ? known(d.max_shared) : 0, known(a.max_len), &plan->shared, &plan->own[0]);
  // the grid's limits, and 32 bits for a row's place
  int64_t units = 1;
  for (const Shape* x : {&plan->shared, &plan->own[0], &plan->own[plan->owns - 1]}) {
    units += x->tiles * (a.cache.heads * x->splits + 7);
    if (x->tiles * x->rows > INT32_MAX) units = INT64_MAX / 2;
  }
  if (units > UINT32_MAX / 256 || a.tokens * a.q_heads > UINT32_MAX / 256)
    return mkv_fail(MKV_ERR_UNSUPPORTED, "%s: %lld query rows", who, (long long)(a.tokens * a.q_heads));
  return MKV_OK;
}

// Every launch leaves parts, also where one is all.
int64_t part_rows(const Shape& s, int heads) { return s.tiles * heads * s.splits * s.rows; }

constexpr int64_t kFewJoins = 8192;  // rows that are joined by four waves each

int64_t up16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

int64_t workspace_of(const mkv_attend_shared_desc_t& d, const Plan& plan) {
  const mkv_scaled_cache_t& c = d.attend.cache;
  int64_t rows = 0;
  rows += part_rows(plan.shared, c.heads);
  for (int i = 0; i < plan.owns; ++i) rows += part_rows(plan.own[i], c.heads);
  return d.attend.tokens * (d.attend.q_heads / c.heads) * static_cast<int64_t>(sizeof(RowPlace)) +
         rows * (c.head_size + 2) * 4 + 64;
}

unsigned units_of(const BothParams& p) {
  return static_cast<unsigned>(p.shared_units + p.own_units + (p.own.s.flags != nullptr ? 1 : 0));
}

template <typename K, bool F16, int D>
void launch(const BothParams& p, hipStream_t stream) {
  attend_kernel<K, F16, D><<<units_of(p), 256, 0, stream>>>(p);
}

// (with_few: chunks beside another launch over the own tokens of requests of few rows)
template <bool F16, int D>
void launch(int shared_rows, int own_rows, bool with_few, const BothParams& p, hipStream_t stream) {
  if (with_few && !F16) {
    chunks_beside_kernel<D><<<units_of(p), 256, 0, stream>>>(p);
  } else if (shared_rows == kManyRows) {
    if (own_rows == 16)
      launch<Both<kManyRows, 16>, F16, D>(p, stream);
    else if (own_rows == 32)
      launch<Both<kManyRows, 32>, F16, D>(p, stream);
    else
      launch<Both<kManyRows, kManyRows>, F16, D>(p, stream);
  } else if (shared_rows == 16) {
    launch<Both<16, 16>, F16, D>(p, stream);
  } else {
    launch<Both<32, 32>, F16, D>(p, stream);
  }
}

template <bool F16, int D>
void run(const GroupedParams& base, const Plan& plan, JoinParams j, char* room, hipStream_t stream) {
  const int heads = j.heads;
  const auto place = [&](const Shape& s, PartSet* set) {  // the parts of a launch's tiles
    const int64_t rows = part_rows(s, heads);
    float* o = reinterpret_cast<float*>(room);
    room += up16(rows * (D + 2) * 4);
    *set = PartSet{o, o + rows * D, s.rows, s.splits, s.tiles};
  };
  BothParams p = {};
  p.own = base;
  p.own.shared_rows = plan.shared.rows;
  p.own.shared_per = plan.shared.per;
  p.own.shared_splits = plan.shared.splits;
  place(plan.shared, &j.sets[0]);
  p.part_o = j.sets[0].o;
  p.part_ml = j.sets[0].ml;
  p.shared_tiles = static_cast<int32_t>(plan.shared.tiles);
  for (int i = plan.owns - 1; i >= 0; --i) {  // the chunks beside what is shared
    const Shape& own = plan.own[i];
    PartSet& set = j.sets[1 + i];
    place(own, &set);
    p.own.part_o = set.o;
    p.own.part_ml = set.ml;
    p.own.splits = own.splits;
    p.own.per = own.per;
    p.own.rows_from = own.from;
    p.own.rows_to = own.to;
    p.own.launch = i;
    p.own_tiles = static_cast<int32_t>(own.tiles);
    p.own_units = own.tiles * heads * own.splits;
    const bool with = i == plan.owns - 1 && base.g.count > 0;
    p.shared_units = with ? plan.shared.tiles * ((heads * plan.shared.splits + 7) / 8 * 8) : 0;
    launch<F16, D>(with ? plan.shared.rows : own.rows, own.rows, with && plan.owns == 2, p, stream);
  }
  if (plan.owns == 1) j.sets[2] = j.sets[1];
  const int64_t rows = j.tokens * heads * j.group;
  if (rows <= kFewJoins)
    shared_join_kernel<F16, D, 4><<<static_cast<unsigned>(rows), 256, 0, stream>>>(j);
  else
    shared_join_kernel<F16, D, 1><<<static_cast<unsigned>((rows + 3) / 4), 256, 0, stream>>>(j);
}

template <bool F16>
void run(int d, const GroupedParams& p, const Plan& plan, const JoinParams& j, char* room,
         hipStream_t stream) {
  if (d == 64)
    run<F16, 64>(p, plan, j, room, stream);
  else if (d == 128)
    run<F16, 128>(p, plan, j, room, stream);
  else
    run<F16, 256>(p, plan, j, room, stream);
}

}  // namespace

extern "C" int64_t mkv_attend_shared_workspace_size(const mkv_attend_shared_desc_t* d) {
  if (d == nullptr) return -1;
  GroupedParams p;
  Plan plan;
  if (check(*d, &p, &plan) != MKV_OK) return -1;
  return d->attend.tokens == 0 || d->attend.requests == 0 ? 0 : workspace_of(*d, plan);
}

extern "C" int mkv_attend_shared(const mkv_attend_shared_desc_t* d, void* stream) {
  const char* who = "mkv_attend_shared";
  if (d == nullptr) return mkv_fail(MKV_ERR_ARG, "%s: desc is NULL", who);
  const mkv_attend_desc_t& a = d->attend;
  GroupedParams p;
  Plan plan;
  int rc = check(*d, &p, &plan);
  if (rc != MKV_OK) return rc;
  if (a.tokens == 0 || a.requests == 0) return MKV_OK;
  rc = check_attend_rows(who, a, p, workspace_of(*d, plan));
  if (rc != MKV_OK) return rc;
  JoinParams j = {};
  j.starts = a.starts;
  j.requests = a.requests;
  j.tokens = a.tokens;
  j.out = p.out;
  j.out_token = p.out_token;
  j.out_head = p.out_head;
  j.heads = a.cache.heads;
  j.group = p.group;
  char* room = static_cast<char*>(a.workspace);
  p.places = reinterpret_cast<RowPlace*>(room);
  j.places = p.places;
  room += a.tokens * p.group * static_cast<int64_t>(sizeof(RowPlace));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a.dtype == MKV_F16)
    run<true>(a.cache.head_size, p, plan, j, room, s);
  else
    run<false>(a.cache.head_size, p, plan, j, room, s);
  return launched(who);
}
