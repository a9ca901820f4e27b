// scaled_cache.hip -- the block-scaled 8-bit cache's slots, store and shift for gfx950.
//
// None of the three has matrix work; each reads its input once and writes its output once.
//
//   * step_slots: a handful of integers a request and 12 bytes a token.  Bound by latency, so
//     it is one launch: every workgroup makes the prefix sums of all requests for itself in
//     LDS (a few thousand requests at most) instead of waiting for a launch that does.
//   * store and shift: one wave holds 16 rows of one (block, KV head) in registers, 16 values
//     of K and of V a lane, so that a block's largest value is known before its first code is
//     written and nothing is read twice.  A lane's 16 values are 16 bytes of codes: every
//     cache access moves 16 bytes a lane.  Blocks of 32 tokens and more take a wave for each
//     16 rows, which exchange their largest values through LDS.

#include "scaled_cache.h"

#include "fp8_e4m3.h"

#include <cstdlib>
#include <cstring>
#include <type_traits>

#pragma clang fp contract(off)

namespace {

using namespace mkv_scaled;

// ------------------------------------------------------------------------- step slots

constexpr int kSlotThreads = 256;  // (1,024 took 5.1 / 6.6 us where 256 took 3.9 / 5.2)

struct SlotParams {
  const int32_t* held;
  const int32_t* fresh;
  int32_t* tables;
  int64_t table_stride;
  const int32_t* free_blocks;
  const int32_t* free_at;
  int32_t* starts;
  int32_t* lens;
  int64_t* slots;
  int32_t* positions;
  int32_t* free_at_out;
  int32_t* flags;
  int64_t free_len;
  int64_t max_tokens;
  int32_t requests;
  int32_t table_width;
  int32_t block_size;
  int32_t bs_shift;  // -1 where block_size is no power of two
};

// Sizes of at most 2^31 - 1 tokens: 32 bits, unsigned, hold them and what is added.
__device__ __forceinline__ uint32_t block_of(uint32_t pos, const SlotParams& p) {
  return p.bs_shift >= 0 ? pos >> p.bs_shift : pos / static_cast<uint32_t>(p.block_size);
}

__device__ __forceinline__ uint32_t blocks_of(uint32_t tokens, const SlotParams& p) {
  return tokens == 0 ? 0u : block_of(tokens - 1, p) + 1;
}

// The last r in [0, n) with a[r] <= at, by halves in LDS; a[0] = 0 <= at.
__device__ __forceinline__ int owner(const int32_t* a, int n, int at) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a[mid] <= at) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// 32 requests of a token each take 3.6 us, 256 requests and 50,021 tokens 5.0: the lengths, the
// scan's exchanges, a table entry, a slot, each waiting for the one before.
__global__ __launch_bounds__(kSlotThreads) void step_slots_kernel(SlotParams p) {
  __shared__ int32_t s_start[MKV_MAX_REQUESTS + 1];  // new tokens before request r
  __shared__ int32_t s_block[MKV_MAX_REQUESTS + 1];  // fresh blocks before request r
  __shared__ int32_t s_held[MKV_MAX_REQUESTS];
  __shared__ int64_t s_wave[2][kSlotThreads / 64];
  __shared__ int32_t s_bad;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = p.requests;
  const int64_t at = p.free_at[0];  // (here, beside the lengths' loads)
  if (tid == 0) s_bad = 0;
  __syncthreads();
  // prefix sums over the requests, a stretch of kSlotThreads at a time
  int64_t tokens = 0, blocks = 0;
  for (int base = 0; base < n; base += kSlotThreads) {
    const int r = base + tid;
    int64_t held = 0, add = 0, need = 0;
    if (r < n) {
      held = p.held[r];
      add = p.fresh[r];
      s_held[r] = static_cast<int32_t>(held);
      if (held < 0 || add < 0 || held + add > INT32_MAX ||
          blocks_of(static_cast<uint32_t>(held + add), p) > static_cast<uint32_t>(p.table_width)) {
        s_bad = 1;
        held = add = 0;
      }
      need = blocks_of(static_cast<uint32_t>(held + add), p) - blocks_of(static_cast<uint32_t>(held), p);
    }
    int64_t a = add, b = need;  // inclusive within the wave
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t ua = __shfl_up(a, d), ub = __shfl_up(b, d);
      if (lane >= d) {
        a += ua;
        b += ub;
      }
    }
    if (lane == 63) {
      s_wave[0][wave] = a;
      s_wave[1][wave] = b;
    }
    __syncthreads();
    for (int w = 0; w < kSlotThreads / 64; ++w) {
      if (w == wave) {
        a += tokens;
        b += blocks;
      }
      tokens += s_wave[0][w];
      blocks += s_wave[1][w];
    }
    if (r < n) {
      // sums past 32 bits are refused below, before anything reads these
      s_start[r] = static_cast<int32_t>(a - add);
      s_block[r] = static_cast<int32_t>(b - need);
    }
    __syncthreads();
  }
  const bool bad = s_bad != 0 || tokens > p.max_tokens || at < 0 ||
                   at + blocks > p.free_len;
  const int64_t gtid = static_cast<int64_t>(blockIdx.x) * kSlotThreads + tid;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kSlotThreads;
  if (blockIdx.x == 0) {
    if (tid == 0) {
      p.free_at_out[0] = static_cast<int32_t>(bad ? at : at + blocks);
      p.starts[n] = bad ? 0 : static_cast<int32_t>(tokens);
      if (bad) raise(p.flags, MKV_FLAG_DST_RANGE);
    }
    for (int r = tid; r < n; r += kSlotThreads) {
      p.starts[r] = bad ? 0 : s_start[r];
      const int32_t end = r + 1 < n ? s_start[r + 1] : static_cast<int32_t>(tokens);
      p.lens[r] = s_held[r] + (bad ? 0 : end - s_start[r]);
    }
  }
  if (!bad) {  // table entries of the fresh blocks
    for (int64_t j = gtid; j < blocks; j += step) {
      const int r = owner(s_block, n, static_cast<int>(j));
      const int64_t col = blocks_of(static_cast<uint32_t>(s_held[r]), p) + (j - s_block[r]);
      p.tables[r * p.table_stride + col] = p.free_blocks[at + j];
    }
  }
  for (int64_t t = gtid; t < p.max_tokens; t += step) {
    int64_t slot = -1;
    int32_t pos = 0;
    if (!bad && t < tokens) {
      const int r = owner(s_start, n, static_cast<int>(t));
      const int held = s_held[r];
      pos = held + static_cast<int>(t) - s_start[r];
      const uint32_t b = block_of(static_cast<uint32_t>(pos), p);
      const uint32_t before = blocks_of(static_cast<uint32_t>(held), p);
      // a fresh block's id comes from the free list: other workgroups may be writing its entry
      const int64_t id = b < before ? p.tables[r * p.table_stride + b]
                                    : p.free_blocks[at + s_block[r] + (b - before)];
      slot = id < 0 ? -1 : id * p.block_size + (static_cast<uint32_t>(pos) - b * p.block_size);
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
  }
}

// ----------------------------------------------------------------- rows and their scales

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

// Waves of a workgroup: those of two (block, head) pairs, or of one that takes more.  (Four
// pairs: the same with eight heads, and half the waves idle with two: 56 us against 43 for a
// shift of 6,007 tokens x 28 layers of two heads.)
constexpr int kMaxWaves = 8;
int waves_of(int bs_shift, int heads) {
  const int parts = 1 << (bs_shift - 4);
  return parts > 1 || heads == 1 ? parts : 2;
}

// ------------------------------------------------------------------------------- store

struct StoreParams {
  DevCache c;
  DevStep s;
  const char* k;
  const char* v;
  int64_t k_token, k_head, v_token, v_head;  // bytes
  int64_t tokens;
  int32_t group;  // tokens a workgroup looks through for blocks that begin there
};

// 16 values of element type ET at p.
template <int ET>
__device__ __forceinline__ void load16(const char* p, float* x) {
  if constexpr (ET == MKV_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p) + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * i + j] = __uint_as_float(w[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p) + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (ET == MKV_BF16) {
          x[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
          x[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
        } else {
          typedef _Float16 h2 __attribute__((ext_vector_type(2)));
          const uint32_t pair = w[j];  // (a bit cast of w[j] itself takes element 0)
          const h2 h = __builtin_bit_cast(h2, pair);
          x[8 * i + 2 * j] = static_cast<float>(h[0]);
          x[8 * i + 2 * j + 1] = static_cast<float>(h[1]);
        }
      }
    }
  }
}

// A workgroup's waves take the heads of the blocks that begin, for their request and step,
// among `group` consecutive tokens: the first token of a request and those at a block's first
// row lead a block.  A store of 22,141 tokens of 8 heads of 128 (136 MB) takes 29 us, 4.7 TB/s.
template <int ET, int D>
__global__ __launch_bounds__(64 * kMaxWaves) void store_kernel(StoreParams p) {
  using R = Rows<D>;
  constexpr int kBytes = ET == MKV_F32 ? 4 : 2;
  __shared__ uint32_t s_max[kMaxWaves][2];
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const int bs = 1 << p.c.bs_shift, parts = bs >> 4;
  const int heads_here = (blockDim.x >> 6) / parts;
  const int head = blockIdx.y * heads_here + wave / parts, part = wave % parts;
  const bool active = head < p.c.heads;
  const int chunk = lane % R::kChunks, sub = lane / R::kChunks;
  if (blockIdx.x == 0 && blockIdx.y == 0) check_starts(p.s, p.tokens, true);
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
    const int off = static_cast<int>(pos & (bs - 1));
    if (t != s0 && off != 0) {  // a block that an earlier token leads
      t = min(t + bs - off, s1);
      continue;
    }
    const int n = static_cast<int>(min(static_cast<int64_t>(bs - off), s1 - t));
    const int64_t col = pos >> p.c.bs_shift;
    int64_t id = -1;
    if (col < p.s.table_width) id = p.s.tables[r * p.s.table_stride + col];
    if (id < 0 || id >= p.c.num_blocks) {
      if (lane == 0 && wave == 0) raise(p.s.flags, MKV_FLAG_DST_RANGE);
      t += n;
      continue;
    }
    // this wave's rows of the block, and the largest of their new values
    float k[R::kPasses][16], v[R::kPasses][16];
#pragma unroll
    for (int u = 0; u < R::kPasses; ++u) {
      const int row = part * 16 + u * R::kPerPass + sub;
      const bool fresh = active && row >= off && row < off + n;
#pragma unroll
      for (int i = 0; i < 16; ++i) k[u][i] = v[u][i] = 0.0f;
      if (fresh) {
        const int64_t at = t + row - off;
        load16<ET>(p.k + at * p.k_token + head * p.k_head + chunk * 16 * kBytes, k[u]);
        load16<ET>(p.v + at * p.v_token + head * p.v_head + chunk * 16 * kBytes, v[u]);
      }
    }
    const Largest most_k = across(largest<16 * R::kPasses>(k[0]), parts, s_max, wave);
    const Largest most_v = across(largest<16 * R::kPasses>(v[0]), parts, s_max, wave);
    int ek = exponent_for(most_k.bits), ev = exponent_for(most_v.bits);
    if (active) {
      uint8_t* scale = p.c.scales + (id * p.c.heads + head) * 2;
      char* kb = p.c.k + id * p.c.bstride + head * p.c.hstride + chunk * 16;
      char* vb = p.c.v + id * p.c.bstride + head * p.c.hstride + chunk * 16;
      if (off > 0) {  // rows [0, off) stay, under the larger scale
        const int ok = scale_exp(scale[0]), ov = scale_exp(scale[1]);
        const int nk = max(ek, ok), nv = max(ev, ov);
#pragma unroll
        for (int u = 0; u < R::kPasses; ++u) {
          const int row = part * 16 + u * R::kPerPass + sub;
          if (row >= off) continue;
          float x[16];
          if (nk > ok) {
            u32x4* w = reinterpret_cast<u32x4*>(kb + row * p.c.tstride);
            decode16(*w, 1.0f, x);
            *w = encode16(x, min(nk - ok, 100), true);
          }
          if (nv > ov) {
            u32x4* w = reinterpret_cast<u32x4*>(vb + row * p.c.tstride);
            decode16(*w, 1.0f, x);
            *w = encode16(x, min(nv - ov, 100), true);
          }
        }
        ek = nk;
        ev = nv;
      }
#pragma unroll
      for (int u = 0; u < R::kPasses; ++u) {
        const int row = part * 16 + u * R::kPerPass + sub;
        if (row < off || row >= off + n) continue;
        __builtin_nontemporal_store(encode16(k[u], ek, most_k.wild),
                                    reinterpret_cast<u32x4*>(kb + row * p.c.tstride));
        __builtin_nontemporal_store(encode16(v[u], ev, most_v.wild),
                                    reinterpret_cast<u32x4*>(vb + row * p.c.tstride));
      }
    }
    if (parts > 1) __syncthreads();  // every wave has read the old scale
    if (active && part == 0 && lane == 0)
      *reinterpret_cast<uint16_t*>(p.c.scales + (id * p.c.heads + head) * 2) =
          static_cast<uint16_t>((ek + 127) | ((ev + 127) << 8));
    t += n;
  }
}

// ------------------------------------------------------------------------------- shift

struct MoveParams {
  DevCache src;  // geometry; the layers' bases come from the arrays below
  DevCache dst;
  const uint64_t* src_layers;
  const uint64_t* dst_layers;
  const int32_t* units;
  const float* tables;
  int32_t n_spans;
  int32_t rotary;
  int32_t words;    // of a unit, 16 at most
  int32_t sources;  // source blocks in it
};

// Units, and the spans' tables from word `tables_at` on, in the launch's own arguments.  A
// small shift is bound by its latency: 512 tokens x 40 layers of 8 heads take 18.8 us a call,
// where a copy of 2 KB in front of the kernel makes it 28.
constexpr int kHostWords = MKV_SHIFT_HOST_BYTES / 4;
struct MoveWords {
  int32_t tables_at;
  int32_t word[kHostWords];
};
struct NoWords {};
static_assert(sizeof(MoveParams) + sizeof(MoveWords) <= 4096, "a launch's arguments");

// A workgroup makes one destination block of `heads_here` heads in one layer and ends.  What
// it has to know is one record made on the host.  22,141 tokens x 40 layers of 8 heads of 128
// (3.63 GB) take 614 to 652 us, 5.6 to 5.9 TB/s, where a copy of as many rows through shuffled block
// tables takes 653 to 661, through ordered ones 583, and a linear one 542.  Found on the GPU instead
// (span, then tables, then rows), the chain of loads in front of the data made it 818; a loop over
// layers behind one chain, whose loads wait for its stores, 755.
template <int D, typename Words>
__global__ __launch_bounds__(64 * kMaxWaves) void move_kernel(MoveParams p, Words w) {
  constexpr bool kHere = std::is_same_v<Words, MoveWords>;
  using R = Rows<D>;
  constexpr int P = R::kPasses;
  __shared__ uint32_t s_max[kMaxWaves][2];
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const int dbs = 1 << p.dst.bs_shift, parts = dbs >> 4;
  const int heads_here = (blockDim.x >> 6) / parts;
  const int head = blockIdx.y * heads_here + wave / parts, part = wave % parts;
  const bool active = head < p.dst.heads;
  const int piece = lane % R::kChunks, sub = lane / R::kChunks;
  // the record's words, one a lane
  const int64_t word_at = static_cast<int64_t>(blockIdx.x) * p.words + min(lane, p.words - 1);
  int word;
  if constexpr (kHere)
    word = w.word[word_at];
  else
    word = p.units[word_at];
  const int id = __builtin_amdgcn_readlane(word, 0), n = __builtin_amdgcn_readlane(word, 1);
  const int span = __builtin_amdgcn_readlane(word, 2), first = __builtin_amdgcn_readlane(word, 3);
  if (id < 0 || id >= p.dst.num_blocks || span >= p.n_spans || n < 1 || first < 0) return;
  // A block is written with all of its rows or not at all: under the scale of some of them, what
  // the block held in place of the others would be other values.  (Every wave of the workgroup
  // decides alike.)
  const int64_t used = ((static_cast<int64_t>(first) + n - 1) >> p.src.bs_shift) + 1;
  if (used > p.sources || __any(lane >= 4 && lane < 4 + used && (word < 0 || word >= p.src.num_blocks)))
    return;

  // Where each pass's row comes from: a wave's 16 rows lie in two source blocks at most.
  const int start = first + part * 16, block0 = start >> p.src.bs_shift;
  const auto source = [&](int b) {
    return b >= 0 && b < p.sources ? __builtin_amdgcn_readlane(word, 4 + b) : -1;
  };
  const int src0 = source(block0), src1 = source(block0 + 1);
  int64_t from_row[P], from_scale[P];
  bool there[P];
  bool whole = active;  // every row of the wave is the span's: nothing to blank out
#pragma unroll
  for (int u = 0; u < P; ++u) {
    const int row = u * R::kPerPass + sub;
    const int64_t from = (start + row) >> p.src.bs_shift == block0 ? src0 : src1;
    there[u] = active && part * 16 + row < n;
    whole = whole && __all(there[u]);
    from_row[u] = from_scale[u] = 0;
    if (there[u]) {
      from_row[u] = from * p.src.bstride + head * static_cast<int64_t>(p.src.hstride) +
                    ((start + row) & ((1 << p.src.bs_shift) - 1)) * p.src.tstride;
      from_scale[u] = (from * p.src.heads + head) * 2;
    }
  }

  // Rotation mixes dimension d with d + rotary / 2: chunk c of 16 with chunk c + rotary / 32.
  // The two chunks' lanes exchange halves, so that each holds 8 whole pairs: the first lane
  // those of dimensions `at` = 16 c to 16 c + 7, the second those of 16 c + 8 on.
  const bool turn = span >= 0 && p.rotary > 0;
  const int half = p.rotary / 32;
  const bool turned = turn && piece < 2 * half;
  const bool first_half = piece < half;
  const int partner = !turned ? lane : first_half ? lane + half : lane - half;
  const int at = first_half ? 16 * piece : 16 * (piece - half) + 8;

  // the other rows read the cache's first
  const int64_t layer = blockIdx.z;
  const uint64_t* sl = p.src_layers + 3 * layer;
  const char* sk = reinterpret_cast<const char*>(sl[0]);
  const char* sv = reinterpret_cast<const char*>(sl[1]);
  const char* ss = reinterpret_cast<const char*>(sl[2]);
  u32x4 kw[P], vw[P];
  uint32_t scale[P];
#pragma unroll
  for (int u = 0; u < P; ++u) {
    scale[u] = *reinterpret_cast<const uint16_t*>(ss + from_scale[u]);
    kw[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(sk + from_row[u] + 16 * piece));
    vw[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(sv + from_row[u] + 16 * piece));
  }
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) cs[i] = 1.0f, sn[i] = 0.0f;
  if (turned) {
    // (-sin for the first half of a pair, +sin for the second)
    if constexpr (kHere) {
      const int t = w.tables_at + span * 2 * p.rotary + at;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        cs[i] = __builtin_bit_cast(float, w.word[t + i]);
        sn[i] = __builtin_bit_cast(float, w.word[t + p.rotary + i]);
      }
    } else {
      const float* t = p.tables + static_cast<int64_t>(span) * 2 * p.rotary + at;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        cs[i] = t[i];
        sn[i] = t[p.rotary + i];
      }
    }
  }
  if (!whole) {
#pragma unroll
    for (int u = 0; u < P; ++u)
      if (!there[u]) kw[u] = vw[u] = u32x4{0, 0, 0, 0};
  }
  const uint64_t* dl = p.dst_layers + 3 * layer;
  const int64_t to = static_cast<int64_t>(id) * p.dst.bstride + head * static_cast<int64_t>(p.dst.hstride) + 16 * piece;
  char* kb = reinterpret_cast<char*>(dl[0]) + to;
  char* vb = reinterpret_cast<char*>(dl[1]) + to;
  const auto row_of = [&](int u) { return (part * 16 + u * R::kPerPass + sub) * p.dst.tstride; };
  // the half of a chunk that goes to the partner, and the one that it sends
  const auto swap = [&](u32x4& w) {
    const uint32_t g0 = first_half ? w[2] : w[0], g1 = first_half ? w[3] : w[1];
    const uint32_t r0 = __builtin_amdgcn_ds_bpermute(4 * partner, g0);
    const uint32_t r1 = __builtin_amdgcn_ds_bpermute(4 * partner, g1);
    if (first_half)
      w[2] = r0, w[3] = r1;
    else
      w[0] = r0, w[1] = r1;
  };
  float y[P][16];
#pragma unroll
  for (int u = 0; u < P; ++u) {
    if (turn) {  // (lanes that turn nothing are their own partners)
      u32x4 w = kw[u];
      swap(w);
      if (turned) kw[u] = w;
    }
    decode16(kw[u], pow2(scale_exp(scale[u] & 0xFF)), y[u]);
    if (turned) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = y[u][i], b = y[u][8 + i];
        const float a0 = a * cs[i], a1 = b * sn[i], b0 = b * cs[i], b1 = a * -sn[i];
        y[u][i] = a0 + a1;
        y[u][8 + i] = b0 + b1;
      }
    }
  }
  const Largest mk = across(largest<16 * P>(y[0]), parts, s_max, wave);
  const int ek = exponent_for(mk.bits);
#pragma unroll
  for (int u = 0; u < P; ++u) {
    u32x4 w = encode16(y[u], ek, mk.wild);
    if (turn) {
      u32x4 back = w;
      swap(back);
      if (turned) w = back;
    }
    if (there[u]) __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(kb + row_of(u)));
  }
#pragma unroll
  for (int u = 0; u < P; ++u) decode16(vw[u], pow2(scale_exp(scale[u] >> 8)), y[u]);
  const Largest mv = across(largest<16 * P>(y[0]), parts, s_max, wave);
  const int ev = exponent_for(mv.bits);
#pragma unroll
  for (int u = 0; u < P; ++u) {
    const u32x4 w = encode16(y[u], ev, mv.wild);
    if (there[u]) __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(vb + row_of(u)));
  }
  if (active && part == 0 && lane == 0)
    *reinterpret_cast<uint16_t*>(reinterpret_cast<uint8_t*>(dl[2]) +
                                 (static_cast<int64_t>(id) * p.dst.heads + head) * 2) =
        static_cast<uint16_t>((ek + 127) | ((ev + 127) << 8));
}

template <int ET>
void store_launch(int d, dim3 grid, int threads, const StoreParams& p, hipStream_t s) {
  if (d == 64)
    store_kernel<ET, 64><<<grid, threads, 0, s>>>(p);
  else if (d == 128)
    store_kernel<ET, 128><<<grid, threads, 0, s>>>(p);
  else
    store_kernel<ET, 256><<<grid, threads, 0, s>>>(p);
}

}  // namespace

// ------------------------------------------------------------------------- entry points

extern "C" int mkv_step_slots(const int32_t* held, const int32_t* fresh, int32_t requests,
                              int32_t* block_tables, int64_t table_stride, int32_t table_width,
                              const int32_t* free_blocks, int64_t free_len,
                              const int32_t* free_at, int32_t block_size, int32_t* starts,
                              int32_t* lens, int64_t* slots, int32_t* positions,
                              int64_t max_tokens, int32_t* free_at_out, int32_t* error_flags,
                              void* stream) {
  const char* who = "mkv_step_slots";
  if (requests < 0 || requests > MKV_MAX_REQUESTS)
    return mkv_fail(MKV_ERR_ARG, "%s: requests %d outside [0, %d]", who, requests,
                    MKV_MAX_REQUESTS);
  if (block_size <= 0) return mkv_fail(MKV_ERR_ARG, "%s: block_size %d", who, block_size);
  if (table_width < 0 || table_stride < 0 || free_len < 0 || max_tokens < 0 ||
      max_tokens > INT32_MAX || free_len > INT32_MAX)
    return mkv_fail(MKV_ERR_ARG, "%s: a size is negative or past 32 bits", who);
  if (free_at == nullptr || free_at_out == nullptr || starts == nullptr ||
      (requests > 0 && (held == nullptr || fresh == nullptr || lens == nullptr)) ||
      (max_tokens > 0 && (slots == nullptr || positions == nullptr)) ||
      (requests > 0 && table_width > 0 && block_tables == nullptr) ||
      (free_len > 0 && free_blocks == nullptr))
    return mkv_fail(MKV_ERR_ARG, "%s: a pointer is NULL", who);
  if (free_at == free_at_out)
    return mkv_fail(MKV_ERR_ARG, "%s: free_at_out is free_at itself", who);
  const SlotParams p = {held,   fresh,    block_tables, table_stride, free_blocks, free_at,
                        starts, lens,     slots,        positions,    free_at_out, error_flags,
                        free_len, max_tokens, requests, table_width,  block_size,
                        (block_size & (block_size - 1)) == 0 ? __builtin_ctz(block_size) : -1};
  const int64_t want = (max_tokens + kSlotThreads - 1) / kSlotThreads;
  const int grid = static_cast<int>(want < 1 ? 1 : want > 512 ? 512 : want);
  step_slots_kernel<<<grid, kSlotThreads, 0, static_cast<hipStream_t>(stream)>>>(p);
  return launched(who);
}

extern "C" int mkv_store_scaled(const mkv_scaled_cache_t* cache, const void* k,
                                int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                int64_t v_token_stride, int64_t v_head_stride, int64_t tokens,
                                int32_t dtype, const int32_t* block_tables,
                                int64_t table_stride, int32_t table_width,
                                const int32_t* starts, const int32_t* lens, int32_t requests,
                                int32_t* error_flags, void* stream) {
  const char* who = "mkv_store_scaled";
  if (cache == nullptr) return mkv_fail(MKV_ERR_ARG, "%s: cache is NULL", who);
  StoreParams p;
  int rc = check_cache(who, *cache, true, &p.c);
  if (rc == MKV_OK)
    rc = check_step(who, cache->block_size, block_tables, table_stride, table_width, starts, lens, requests,
                    error_flags, &p.s);
  if (rc != MKV_OK) return rc;
  if (dtype != MKV_BF16 && dtype != MKV_F16 && dtype != MKV_F32)
    return mkv_fail(MKV_ERR_DTYPE, "%s: dtype %d is not bf16, fp16 or fp32", who, dtype);
  if (tokens < 0 || tokens > INT32_MAX)
    return mkv_fail(MKV_ERR_ARG, "%s: tokens %lld", who, (long long)tokens);
  if (tokens == 0 || requests == 0) return MKV_OK;
  if (k == nullptr || v == nullptr) return mkv_fail(MKV_ERR_ARG, "%s: k or v is NULL", who);
  const int64_t eb = dtype == MKV_F32 ? 4 : 2;
  const int64_t most = INT64_MAX / 16 / (tokens + cache->heads);
  if (k_token_stride < 0 || k_head_stride < 0 || v_token_stride < 0 || v_head_stride < 0 ||
      k_token_stride > most || k_head_stride > most || v_token_stride > most ||
      v_head_stride > most)
    return mkv_fail(MKV_ERR_ARG, "%s: a stride of k or v is out of range", who);
  p.k = static_cast<const char*>(k);
  p.v = static_cast<const char*>(v);
  p.k_token = k_token_stride * eb;
  p.k_head = k_head_stride * eb;
  p.v_token = v_token_stride * eb;
  p.v_head = v_head_stride * eb;
  if (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | p.k_token | p.k_head |
        p.v_token | p.v_head) & 15) != 0)
    return mkv_fail(MKV_ERR_ALIGN, "%s: k or v is not 16-byte aligned", who);
  p.tokens = tokens;
  const int waves = waves_of(p.c.bs_shift, p.c.heads), parts = cache->block_size / 16;
  const int heads_here = waves / parts;
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
  const int64_t each = tokens * ((cache->heads + heads_here - 1) / heads_here);
  const int64_t ahead = tokens / requests;  // a request's on average
  if (ahead < 16 || (each <= 4096 && ahead < 256))
    p.group = each <= 4096 ? 1 : 4;
  else if (each > 24576)
    p.group = cache->block_size;
  else if (each > 12288)
    p.group = ahead >= 64 ? 16 : 4;
  else
    p.group = cache->block_size >= 64 && ahead >= 64 ? 16 : each > 4096 && ahead >= 1024 ? 8 : 4;
  if ((tokens + p.group - 1) / p.group > UINT32_MAX / (64 * waves))
    return mkv_fail(MKV_ERR_UNSUPPORTED, "%s: %lld tokens", who, (long long)tokens);
  const dim3 grid(static_cast<unsigned>((tokens + p.group - 1) / p.group),
                  static_cast<unsigned>((cache->heads + heads_here - 1) / heads_here));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == MKV_BF16)
    store_launch<MKV_BF16>(cache->head_size, grid, 64 * waves, p, s);
  else if (dtype == MKV_F16)
    store_launch<MKV_F16>(cache->head_size, grid, 64 * waves, p, s);
  else
    store_launch<MKV_F32>(cache->head_size, grid, 64 * waves, p, s);
  return launched(who);
}

extern "C" int mkv_scaled_units(const mkv_span_t* spans, int32_t n_spans, const int32_t* src_table,
                                int64_t src_table_len, const int32_t* dst_table,
                                int64_t dst_table_len, const mkv_scaled_cache_t* src,
                                const mkv_scaled_cache_t* dst, int32_t* units, int64_t max_units,
                                int64_t* n_units, int32_t* flags) {
  const char* who = "mkv_scaled_units";
  if (src == nullptr || dst == nullptr || n_units == nullptr)
    return mkv_fail(MKV_ERR_ARG, "%s: a pointer is NULL", who);
  DevCache s, t;
  int rc = check_cache(who, *src, false, &s);
  if (rc == MKV_OK) rc = check_cache(who, *dst, false, &t);
  if (rc != MKV_OK) return rc;
  if (n_spans < 0 || n_spans > MKV_MAX_SPANS)
    return mkv_fail(MKV_ERR_ARG, "%s: n_spans %d outside [0, %d]", who, n_spans, MKV_MAX_SPANS);
  if (src_table_len < 0 || dst_table_len < 0 || max_units < 0 ||
      (n_spans > 0 && spans == nullptr) || (src_table_len > 0 && src_table == nullptr) ||
      (dst_table_len > 0 && dst_table == nullptr) || (max_units > 0 && units == nullptr))
    return mkv_fail(MKV_ERR_ARG, "%s: a pointer is NULL or a size negative", who);
  int64_t count = 0;
  int32_t raised = 0;
  const int32_t bs = dst->block_size, sbs = src->block_size;
  const int32_t sources = MKV_UNIT_SOURCES(sbs, bs), words = MKV_UNIT_WORDS(sbs, bs);
  // a block number in a table, which positions and indices of any size may leave
  const auto entry = [](const int32_t* table, int64_t len, int64_t index, int64_t block,
                        int64_t blocks) -> int32_t {
    int64_t at;
    if (__builtin_add_overflow(index, block, &at) || at < 0 || at >= len) return -1;
    return table[at] >= 0 && table[at] < blocks ? table[at] : -1;
  };
  for (int32_t i = 0; i < n_spans; ++i) {
    const mkv_span_t& sp = spans[i];
    if (sp.n_tokens < 0 || sp.src_pos < 0 || sp.dst_pos < 0 || sp.dst_pos % bs != 0 ||
        sp.src_pos > INT64_MAX - INT32_MAX || sp.dst_pos > INT64_MAX - INT32_MAX) {
      raised |= MKV_FLAG_SPAN;
      continue;
    }
    for (int64_t at = 0; at < sp.n_tokens; at += bs) {
      const int32_t id = entry(dst_table, dst_table_len, sp.dst_index, (sp.dst_pos + at) / bs,
                               dst->num_blocks);
      if (id < 0) {
        raised |= MKV_FLAG_DST_RANGE;
        continue;
      }
      if (count >= max_units)
        return mkv_fail(MKV_ERR_ARG, "%s: more than %lld units", who, (long long)max_units);
      int32_t* u = units + words * count++;
      const int32_t rows = static_cast<int32_t>(sp.n_tokens - at < bs ? sp.n_tokens - at : bs);
      const int32_t first = static_cast<int32_t>((sp.src_pos + at) % sbs);
      const int64_t block = (sp.src_pos + at) / sbs;
      const int32_t used = (first + rows + sbs - 1) / sbs;
      u[0] = id;
      u[1] = rows;
      u[2] = sp.delta != 0 ? i : -1;
      u[3] = first;
      for (int32_t j = 0; j < words - 4; ++j) {
        u[4 + j] = j >= sources ? 0 : -1;
        if (j < used) {
          u[4 + j] = entry(src_table, src_table_len, sp.src_index, block + j, src->num_blocks);
          if (u[4 + j] < 0) raised |= MKV_FLAG_SRC_RANGE;
        }
      }
    }
  }
  // A block written twice, or read by one unit and written by another, would hold whichever
  // came last: a bit for each destination block says whether one is.
  auto* taken = static_cast<uint8_t*>(count > 0 ? calloc((dst->num_blocks + 7) / 8, 1) : nullptr);
  if (count > 0 && taken == nullptr)
    return mkv_fail(MKV_ERR_ARG, "%s: no memory for %lld blocks", who, (long long)dst->num_blocks);
  int32_t twice = -1, read = -1;
  for (int64_t n = 0; n < count; ++n) {
    const int32_t id = units[words * n];
    if (taken[id >> 3] >> (id & 7) & 1) twice = id;
    taken[id >> 3] |= static_cast<uint8_t>(1 << (id & 7));
  }
  for (int64_t n = 0; src == dst && n < count; ++n)
    for (int32_t j = 0; j < sources; ++j) {
      const int32_t* u = units + words * n;
      const int32_t id = j < (u[3] + u[1] + sbs - 1) / sbs ? u[4 + j] : -1;
      if (id >= 0 && id < dst->num_blocks && taken[id >> 3] >> (id & 7) & 1) read = id;
    }
  free(taken);
  if (twice >= 0)
    return mkv_fail(MKV_ERR_ARG, "%s: block %d is a destination twice", who, twice);
  if (read >= 0)
    return mkv_fail(MKV_ERR_ARG, "%s: block %d is a source and a destination", who, read);
  *n_units = count;
  if (flags != nullptr) *flags = raised;
  return MKV_OK;
}

extern "C" int mkv_shift_scaled(const mkv_scaled_shift_desc_t* d, void* stream) {
  const char* who = "mkv_shift_scaled";
  if (d == nullptr) return mkv_fail(MKV_ERR_ARG, "%s: desc is NULL", who);
  MoveParams p;
  int rc = check_cache(who, d->src, false, &p.src);
  if (rc == MKV_OK) rc = check_cache(who, d->dst, false, &p.dst);
  if (rc != MKV_OK) return rc;
  if (d->src.heads != d->dst.heads || d->src.head_size != d->dst.head_size)
    return mkv_fail(MKV_ERR_ARG, "%s: source and destination differ in heads or head_size", who);
  if (d->rotary < 0 || d->rotary > d->dst.head_size || d->rotary % 32 != 0)
    return mkv_fail(MKV_ERR_UNSUPPORTED, "%s: rotary %d is not a multiple of 32 up to head_size",
                    who, d->rotary);
  if (d->n_spans < 0 || d->n_spans > MKV_MAX_SPANS)
    return mkv_fail(MKV_ERR_ARG, "%s: n_spans %d outside [0, %d]", who, d->n_spans, MKV_MAX_SPANS);
  if (d->layers < 0 || d->layers > 65535)
    return mkv_fail(MKV_ERR_ARG, "%s: layers %d", who, d->layers);
  if (d->n_units < 0 || d->n_units > INT32_MAX)
    return mkv_fail(MKV_ERR_ARG, "%s: n_units %lld", who, (long long)d->n_units);
  if (d->layers == 0 || d->n_units == 0) return MKV_OK;
  if (d->units == nullptr || d->src_layers == nullptr || d->dst_layers == nullptr ||
      (d->rotary > 0 && d->tables == nullptr))
    return mkv_fail(MKV_ERR_ARG, "%s: a pointer is NULL", who);
  if (!d->on_host &&
      ((reinterpret_cast<uintptr_t>(d->tables) | reinterpret_cast<uintptr_t>(d->units)) & 15) != 0)
    return mkv_fail(MKV_ERR_ALIGN, "%s: tables or units are not 16-byte aligned", who);
  p.src_layers = d->src_layers;
  p.dst_layers = d->dst_layers;
  p.units = d->units;
  p.tables = d->tables;
  p.n_spans = d->n_spans;
  p.rotary = d->rotary;
  p.words = MKV_UNIT_WORDS(d->src.block_size, d->dst.block_size);
  p.sources = MKV_UNIT_SOURCES(d->src.block_size, d->dst.block_size);
  const int waves = waves_of(p.dst.bs_shift, p.dst.heads), heads_here = waves / (d->dst.block_size / 16);
  if (d->n_units > UINT32_MAX / (64 * waves))
    return mkv_fail(MKV_ERR_UNSUPPORTED, "%s: %lld units", who, (long long)d->n_units);
  const int64_t head_groups = (d->dst.heads + heads_here - 1) / heads_here;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const auto launch = [&](int64_t units, auto words) {
    using W = decltype(words);
    const dim3 grid(static_cast<unsigned>(units), static_cast<unsigned>(head_groups),
                    static_cast<unsigned>(d->layers));
    if (d->dst.head_size == 64)
      move_kernel<64, W><<<grid, 64 * waves, 0, s>>>(p, words);
    else if (d->dst.head_size == 128)
      move_kernel<128, W><<<grid, 64 * waves, 0, s>>>(p, words);
    else
      move_kernel<256, W><<<grid, 64 * waves, 0, s>>>(p, words);
  };
  if (!d->on_host) {
    launch(d->n_units, NoWords{});
    return launched(who);
  }
  // As many units to a launch as fit with the tables from their lowest span to their highest
  // (one unit and one table always do: 16 words and 512).
  static_assert(16 + 2 * 256 <= kHostWords);
  for (int64_t u = 0; u < d->n_units; ++u) {
    const int32_t span = d->units[u * p.words + 2];
    if (span < -1 || span >= d->n_spans)
      return mkv_fail(MKV_ERR_ARG, "%s: unit %lld is of span %d of %d", who, (long long)u, span,
                      d->n_spans);
  }
  for (int64_t u = 0; u < d->n_units;) {
    MoveWords w;
    memset(&w, 0, sizeof w);
    int32_t lo = 0, hi = -1;
    int n = 0;
    for (; u + n < d->n_units; ++n) {
      const int32_t span = d->units[(u + n) * p.words + 2];
      int32_t l = lo, h = hi;
      if (span >= 0 && d->rotary > 0) {
        l = hi < lo || span < lo ? span : lo;
        h = hi < lo || span > hi ? span : hi;
      }
      const int64_t words = (n + 1) * static_cast<int64_t>(p.words) +
                            (static_cast<int64_t>(h) - l + 1) * 2 * d->rotary;
      if (words > kHostWords) break;
      lo = l;
      hi = h;
    }
    p.n_spans = hi - lo + 1;
    w.tables_at = n * p.words;
    for (int i = 0; i < n; ++i) {
      int32_t* to = w.word + i * p.words;
      memcpy(to, d->units + (u + i) * p.words, 4 * p.words);
      to[2] = to[2] < 0 || d->rotary == 0 ? -1 : to[2] - lo;
    }
    if (p.n_spans > 0)
      memcpy(w.word + w.tables_at, d->tables + static_cast<int64_t>(lo) * 2 * d->rotary,
             static_cast<size_t>(p.n_spans) * 2 * d->rotary * 4);
    launch(n, w);
    u += n;
  }
  return launched(who);
}
