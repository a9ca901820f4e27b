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

#pragma clang fp contract(off)

namespace {

// Parts of a launch: results of `rows` rows a tile, tiles by KV heads by parts.
struct PartSet {
  const float* o;
  const float* ml;
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

constexpr int kJoinWaves = 4;

// A wave joins a row: 64 parts' m and l at a time, one a lane, then their outputs, D / 4 lanes a
// part.  What the places say is kept within the parts, whatever was changed between launches.
template <bool F16, int D>
__global__ __launch_bounds__(64 * kJoinWaves) void shared_join_kernel(JoinParams p) {
  constexpr int kLanes = D / 4, kGroups = 64 / kLanes;
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const int q_heads = p.heads * p.group;
  const uint32_t unit = blockIdx.x * kJoinWaves + wave;
  const int64_t token = unit / q_heads;
  if (token >= p.tokens) return;
  const int h = unit % q_heads, head = h / p.group;
  RowPlace at = p.places[token * p.group + h % p.group];
  const int32_t* starts = p.starts;
  const int r = last_at_most(p.requests, token, [starts](int i) { return starts[i]; });
  if (r < 0) return;
  const int64_t s0 = starts[r], s1 = starts[r + 1];
  if (s0 < 0 || token < s0 || token >= s1 || s1 > p.tokens) return;  // nobody's
  const PartSet& mine = (at.own_parts >> 16) & 1 ? p.sets[2] : p.sets[1];
  const auto first_of = [&](const PartSet& s, int32_t place) {
    int64_t tile = place / s.rows;
    tile = tile < 0 ? 0 : tile < s.tiles ? tile : s.tiles - 1;
    const int row = place < 0 ? 0 : place % s.rows;
    return (tile * p.heads + head) * s.splits * s.rows + row;
  };
  const int ns = min(max(at.shared_parts, 0), p.sets[0].splits);
  const int no = min(max(at.own_parts & 0xFFFF, 0), mine.splits);
  const int64_t from_s = ns > 0 ? first_of(p.sets[0], at.shared_at) : 0;
  const int64_t from_o = first_of(mine, at.own_at);
  const int d = lane % kLanes, grp = lane / kLanes, n = ns + no;
  f32x4 o = {0, 0, 0, 0};
  float top = -kInf, sum = 0.0f;
  for (int base = 0; base < n; base += 64) {
    const int i = base + lane;
    float m = -kInf, l = 0.0f;
    if (i < n) {
      const PartSet& s = i < ns ? p.sets[0] : mine;
      const int64_t row = i < ns ? from_s + static_cast<int64_t>(i) * s.rows
                                 : from_o + static_cast<int64_t>(i - ns) * s.rows;
      m = s.ml[2 * row];
      l = s.ml[2 * row + 1];
    }
    float now = m;
    for (int x = 32; x > 0; x >>= 1) now = fmaxf(now, __shfl_xor(now, x));
    now = fmaxf(now, top);
    const float b = now == -kInf ? 0.0f : now, old = fast_exp2(top - b), f = fast_exp2(m - b);
    float part = l * f;
    for (int x = 32; x > 0; x >>= 1) part += __shfl_xor(part, x);
    sum = sum * old + part;
    o *= old;
    top = now;
    const int here = min(64, n - base);
    for (int j = grp; j < here; j += kGroups) {
      const int k = base + j;
      const float* x = k < ns ? p.sets[0].o + (from_s + static_cast<int64_t>(k) * p.sets[0].rows) * D
                              : mine.o + (from_o + static_cast<int64_t>(k - ns) * mine.rows) * D;
      o += *reinterpret_cast<const f32x4*>(x + 4 * d) * __shfl(f, j);
    }
  }
#pragma unroll
  for (int x = kLanes; x < 64; x <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], x);
  if (grp != 0) return;
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
  if (each >= 2048 && a.requests > 1 && rest <= 16 * static_cast<int64_t>(a.requests - 1)) {
    plan->own[0] = shape_for(a, 16, 0, 16);
    plan->own[1] = shape_for(a, each, 17, INT32_MAX);
    plan->owns = 2;
  } else {
    plan->own[0] = shape_for(a, each, 0, INT32_MAX);
    plan->owns = 1;
  }
  plan->shared = Shape{};
  if (d.n_groups > 0) {
    mkv_attend_desc_t s = a;  // a group's rows as one request's
    s.requests = d.n_groups;
    s.max_len = d.max_shared;
    const int64_t rows = (a.tokens * p->group + d.n_groups - 1) / d.n_groups;
    plan->shared = shape_for(s, rows, 0, INT32_MAX);
  }
  for (const Shape* s : {&plan->shared, &plan->own[0], &plan->own[1]}) {
    if (s == &plan->own[1] && plan->owns < 2) continue;
    if (s->tiles > (s->rows == kManyRows ? 65535 : UINT32_MAX / (64 * kFewWaves)) ||
        s->tiles * s->rows > INT32_MAX)
      return mkv_fail(MKV_ERR_UNSUPPORTED, "%s: %lld query rows", who,
                      (long long)(a.tokens * p->group));
  }
  if (a.tokens * a.q_heads > UINT32_MAX / 64)
    return mkv_fail(MKV_ERR_UNSUPPORTED, "%s: %lld query rows", who, (long long)(a.tokens * a.q_heads));
  return MKV_OK;
}

// Every launch leaves parts, also where one is all.
int64_t part_rows(const Shape& s, int heads) { return s.tiles * heads * s.splits * s.rows; }

int64_t up16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

int64_t workspace_of(const mkv_attend_shared_desc_t& d, const Plan& plan) {
  const mkv_scaled_cache_t& c = d.attend.cache;
  int64_t rows = 0;
  if (d.n_groups > 0) rows += part_rows(plan.shared, c.heads);
  for (int i = 0; i < plan.owns; ++i) rows += part_rows(plan.own[i], c.heads);
  return d.attend.tokens * (d.attend.q_heads / c.heads) * static_cast<int64_t>(sizeof(RowPlace)) +
         rows * (c.head_size + 2) * 4 + 64;
}

template <int OVER, bool F16, int D>
void launch(const GroupedParams& p, const Shape& s, int heads, hipStream_t stream) {
  const unsigned tiles = static_cast<unsigned>(s.tiles);
  // (few rows: one part more looks through the starts)
  const dim3 few(tiles, heads, s.splits + (OVER == kOwn && p.s.flags != nullptr ? 1 : 0));
  if (s.rows == 16)
    attend_few_kernel<OVER, F16, D, 1><<<few, 64 * kFewWaves, 0, stream>>>(p);
  else if (s.rows == 32)
    attend_few_kernel<OVER, F16, D, 2><<<few, 64 * kFewWaves, 0, stream>>>(p);
  else
    attend_many_kernel<OVER, F16, D><<<dim3(heads, tiles, s.splits), 64 * kManyWaves, 0, stream>>>(p);
}

template <bool F16, int D>
void run(GroupedParams p, const Plan& plan, JoinParams j, char* room, hipStream_t stream) {
  const int heads = j.heads;
  const auto place = [&](const Shape& s, PartSet* set) {
    const int64_t rows = part_rows(s, heads);
    p.part_o = reinterpret_cast<float*>(room);
    p.part_ml = p.part_o + rows * D;
    p.splits = s.splits;
    p.per = s.per;
    p.rows_from = s.from;
    p.rows_to = s.to;
    room += up16(rows * (D + 2) * 4);
    *set = PartSet{p.part_o, p.part_ml, s.rows, s.splits, s.tiles};
  };
  p.shared_rows = 16;
  p.shared_splits = p.shared_per = 1;
  if (p.g.count > 0) {
    p.shared_rows = plan.shared.rows;
    p.shared_per = plan.shared.per;
    p.shared_splits = plan.shared.splits;
    place(plan.shared, &j.sets[0]);
    launch<kShared, F16, D>(p, plan.shared, heads, stream);
  }
  for (int i = 0; i < plan.owns; ++i) {
    p.launch = i;
    place(plan.own[i], &j.sets[1 + i]);
    launch<kOwn, F16, D>(p, plan.own[i], heads, stream);
  }
  if (plan.owns == 1) j.sets[2] = j.sets[1];
  if (p.g.count == 0) j.sets[0] = PartSet{nullptr, nullptr, 16, 0, 1};
  const int64_t rows = j.tokens * heads * j.group;
  shared_join_kernel<F16, D><<<static_cast<unsigned>((rows + kJoinWaves - 1) / kJoinWaves),
                               64 * kJoinWaves, 0, stream>>>(j);
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
