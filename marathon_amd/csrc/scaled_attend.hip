// scaled_attend.hip -- causal attention over the block-scaled 8-bit cache for gfx950.
//
// The kernels and their mathematics are scaled_attend.h's; here their results are joined, and
// the launches chosen.

#include "scaled_attend.h"

#pragma clang fp contract(off)

namespace {

// ------------------------------------------------------------------ over whole histories

template <int RT>
struct Few {
  typedef AttendParams Params;
  static constexpr int kFew = RT;
  static constexpr bool kMany = false, kGrouped = false;
  static __device__ __forceinline__ const Params& params(const Params& p, Over) { return p; }
  static __device__ __forceinline__ Section pick(const Params& p, unsigned& tile, int& head, int& part,
                                                 Over&) {
    head = blockIdx.y;
    part = blockIdx.z;
    // Workgroups go to the eight XCDs in turn: the tiles are turned by the part, so that a long
    // request's parts do not all fall to one (32 ragged requests: 119 -> 112 us).
    tile = (blockIdx.x + blockIdx.z) % gridDim.x;
    if (part == p.splits) {  // (a part of its own: no register is held for it)
      if (blockIdx.x + blockIdx.y == 0) check_starts(p.s, p.tokens, false);
      return kNothing;
    }
    return kFewRows;
  }
};

struct Many {
  typedef AttendParams Params;
  static constexpr int kFew = 0;
  static constexpr bool kMany = true, kGrouped = false, kTwoTerms = false;
  static __device__ __forceinline__ const Params& params(const Params& p, Over) { return p; }
  static __device__ __forceinline__ Section pick(const Params& p, unsigned& tile, int& head, int& part,
                                                 Over&) {
    head = blockIdx.x;
    part = blockIdx.z;
    // the last tiles first: of one request they see the most
    tile = gridDim.y - 1 - blockIdx.y;
    if (blockIdx.x + blockIdx.y + blockIdx.z == 0) check_starts(p.s, p.tokens, false);
    return kManyRowsTile;
  }
};

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
  if (!find_tile<false, BM>(p, blockIdx.x, t) || t.parts <= 1) return;
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

// One launch for all requests, or one for the few rows of most and one for the many of others.
struct Plan {
  Shape shape[2];
  int count;
};

int check(const mkv_attend_desc_t& d, AttendParams* p, Plan* plan) {
  const char* who = "mkv_attend_scaled";
  const int rc = check_attend(who, d, p);
  if (rc != MKV_OK) return rc;

  const int64_t new_most = d.max_new > 0 && d.max_new < d.tokens ? d.max_new : d.tokens;
  const int64_t each = new_most * p->group;
  // A long chunk beside decoding requests: where those behind the largest have 16 rows or
  // fewer on average, the requests of up to 16 rows get a launch of their own, of 16 rows a
  // tile in place of 128. Measured as one launch / two, 4 query heads a KV head: a chunk of
  // 1,024 tokens beside 31 requests at 16,000 tokens 535 / 440 us, 1,000 beside 255 at 4,000
  // 400 / 348, 1,000 beside one at 16,000 314 / 306, 512 beside 3 143 / 145; with a chunk of
  // 129 beside 31 149 / 173, of 13 beside one 41 / 59: there the one launch has room for both.
  const int64_t rest = (d.tokens - new_most) * p->group;
  if (each >= 2048 && d.requests > 1 && rest <= kBesideRows * static_cast<int64_t>(d.requests - 1)) {
    plan->shape[0] = shape_for(d, kBesideRows, 0, kBesideRows);
    plan->shape[1] = shape_for(d, each, kBesideRows + 1, INT32_MAX);
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
  attend_kernel<Few<RT>, F16, D><<<grid, 64 * kFewWaves, 0, stream>>>(p);
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
  attend_kernel<Many, F16, D><<<dim3(heads, tiles, s.splits), 64 * kManyWaves, 0, stream>>>(p);
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
  const int rows = check_attend_rows(who, *d, p, mkv_attend_workspace_size(d));
  if (rows != MKV_OK) return rows;
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
