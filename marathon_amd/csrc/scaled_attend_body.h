// scaled_attend_body.h -- the body of scaled_attend.h's kernels, which include it (no header of its own):
// a workgroup's tile, KV head and part, of few rows or of many.  It takes K, F16, D, `params` and `lds`.

  unsigned tile;
  int head, part;
  Over over = kHistory;
  const Section section = K::pick(params, tile, head, part, over);
  if (section == kNothing) return;
  const auto& p = K::params(params, over);

  if constexpr (K::kFew > 0) if (section == kFewRows) {
    constexpr int RT = K::kFew;
    constexpr int BM = 16 * RT, KS = D / 32, DT = D / 16, NQ = D / 64;
    auto& s_o = lds.few.o;
    auto& s_ml = lds.few.ml;
    const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    Tile t;
    t.over = over;
    if (!find_tile<K::kGrouped, BM>(p, tile, t)) return;
    if (part >= t.parts) return;
    if constexpr (K::kGrouped)
      if (t.over == kOwn && head + part == 0) note_places<BM>(p, t, tile);
    const int k0 = t.from + part * t.per, k1 = min(t.keys, k0 + t.per);

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
    if constexpr (K::kGrouped)
      if (t.over == kShared) find_full(p, t);

    // this lane's query rows: operand B of S^T = K Q^T
    u32x4 q[RT][KS];
    int limit[RT];  // tokens the row sees
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int64_t row = t.row0 + rt * 16 + c;
      const bool there = rt * 16 + c < t.rows;
      const int64_t token = row / p.group;
      limit[rt] = there ? row_sees<K::kGrouped>(p, t, token) : 0;
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
    // Beside tiles of many rows the registers are there.
    constexpr int kStride = 32 * kFewWaves;
    for (int base = first; base < k1; base += 64 * kStride) {
      if (base != first) look_up(base);
      const int last = min(64, (k1 - base + kStride - 1) / kStride) - 1;
      if constexpr (K::kMany) {
        FewRaw<D> x, next;
        load(base, 0, x);
        for (int n = 0; n <= last; ++n) {
          if (n < last) load(base + (n + 1) * kStride, n + 1, next);
          step(base + n * kStride, n, x);
          x = next;
        }
      } else {
        for (int n = 0; n <= last; ++n) {
          FewRaw<D> x;
          load(base + n * kStride, n, x);
          step(base + n * kStride, n, x);
        }
      }
    }

    // the four waves' results: their largest, then the sums under it
    // (places found anew: what the queries' addresses took is not kept in registers until here)
    unsigned tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int cc = tid & 15, gg = tid >> 4 & 3;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      l[rt] += __shfl_xor(l[rt], 16);
      l[rt] += __shfl_xor(l[rt], 32);
      if (gg == 0) {
        s_ml[wave][rt * 16 + cc][0] = m[rt];
        s_ml[wave][rt * 16 + cc][1] = l[rt];
      }
    }
    __syncthreads();
    float* part_o = nullptr;
    float* part_ml = nullptr;
    if (K::kGrouped || t.parts > 1) {
      const int64_t at = (static_cast<int64_t>(tile) * p.c.heads + head) * p.splits + part;
      part_o = p.part_o + at * BM * D;
      part_ml = p.part_ml + at * BM * 2;
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      // the largest of a row and the sum under it
      const auto row_sum = [&](int i, float& top) {
        top = -kInf;
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kFewWaves; ++w) top = fmaxf(top, s_ml[w][i][0]);
        const float base = top == -kInf ? 0.0f : top;
#pragma unroll
        for (int w = 0; w < kFewWaves; ++w) sum += s_ml[w][i][1] * fast_exp2(s_ml[w][i][0] - base);
        return sum;
      };
      float top;
      row_sum(rt * 16 + cc, top);
      const float f = fast_exp2(m[rt] - (top == -kInf ? 0.0f : top));
      if (rt > 0) __syncthreads();
      // a row's quarters of a vector exchanged by its number, against bank conflicts
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int dt = 0; dt < DT; dt += 4)
          *reinterpret_cast<f32x4*>(&s_o[wave][cc * D + 4 * (((D / 16) * (4 * gg + r) + dt) / 4 ^ cc)]) =
              f32x4{o[rt][dt][r] * f, o[rt][dt + 1][r] * f, o[rt][dt + 2][r] * f, o[rt][dt + 3][r] * f};
      __syncthreads();
      constexpr int kLanes = D / 4;  // of a row
      const int v = tid % kLanes;
#pragma unroll
      for (int r = tid / kLanes; r < 16; r += 64 * kFewWaves / kLanes) {
        const int i = rt * 16 + r;
        if (i >= t.rows) break;
        f32x4 x[kFewWaves];
#pragma unroll
        for (int w = 0; w < kFewWaves; ++w)
          x[w] = *reinterpret_cast<const f32x4*>(&s_o[w][r * D + 4 * (v ^ r)]);
        const f32x4 all = (x[0] + x[2]) + (x[1] + x[3]);
        const float sum = row_sum(i, top);
        if (part_o != nullptr) {
          *reinterpret_cast<f32x4*>(part_o + i * D + 4 * v) = all;
          if (v == 0) {
            part_ml[2 * i] = top;
            part_ml[2 * i + 1] = sum;
          }
        } else {
          const int64_t row = t.row0 + i;
          char* at = p.out + (t.s0 + row / p.group) * p.out_token +
                     (static_cast<int64_t>(head) * p.group + row % p.group) * p.out_head;
          const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
          *reinterpret_cast<u32x2*>(at + 8 * v) =
              u32x2{out_pair<F16>(all[0] * by, all[1] * by), out_pair<F16>(all[2] * by, all[3] * by)};
        }
      }
    }
    return;
  }

  if constexpr (K::kMany) {
    constexpr int KS = D / 16, MT = D / 32, W = D / 16, KC = D / 16;
    constexpr int kKLoads = 64 * D / 16 / 256;
    constexpr bool kTwoTerms = F16 || K::kTwoTerms;  // of p
    auto& s_k = lds.many.k;
    auto& s_v = lds.many.v;
    auto& s_odd = lds.many.odd;
    const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
    const int c = lane & 31, h = lane >> 5;
    Tile t;
    t.over = over;
    if (!find_tile<K::kGrouped, kManyRows>(p, tile, t)) return;
    if (part >= t.parts) return;
    if constexpr (K::kGrouped)
      if (t.over == kOwn && head + part == 0) note_places<kManyRows>(p, t, tile);
    const int k0 = t.from + part * t.per, k1 = min(t.keys, k0 + t.per);
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

    Groups now = look_up(k0);
    if constexpr (K::kGrouped)
      if (t.over == kShared) find_full(p, t);

    // this wave's rows: operand B of S^T = K Q^T
    const int64_t row = t.row0 + wave * 32 + c;
    const bool there = wave * 32 + c < t.rows;
    u32x4 q[KS];
    int limit = 0;
    {
      const int64_t token = row / p.group;
      if (there) limit = row_sees<K::kGrouped>(p, t, token);
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
      u32x4 ph[4], pl[4];  // P^T: 16 tokens each; and what bf16 leaves of it (kTwoTerms)
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
          if constexpr (kTwoTerms)
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
          if constexpr (kTwoTerms) o[mt] = times(a, pl[g], o[mt]);
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
      Groups next = look_up(k0 + 1024);
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
    if (K::kGrouped || t.parts > 1) {
      const int64_t at = (static_cast<int64_t>(tile) * p.c.heads + head) * p.splits + part;
      if (there && h == 0) {
        p.part_ml[(at * kManyRows + i) * 2] = m;
        p.part_ml[(at * kManyRows + i) * 2 + 1] = l;
      }
      // through LDS, so that rows leave whole, not 16 bytes of each at a time; a row's quarters of
      // a vector are exchanged by its number, as the tiles' were
      float* s_o = reinterpret_cast<float*>(s_k) + wave * 32 * D;
#pragma unroll
      for (int e = 0; e < 8; ++e) {  // dimensions W * d + 0..W-1, two of each mt
        const int d = 8 * (e >> 2) + 4 * h + (e & 3);
#pragma unroll
        for (int mt = 0; mt < MT; mt += 2)
          *reinterpret_cast<f32x4*>(s_o + c * D + 4 * ((W * d + 2 * mt) / 4 ^ (c & 15))) =
              f32x4{o[mt][e], o[mt][e + 8], o[mt + 1][e], o[mt + 1][e + 8]};
      }
      wave_fence();
      constexpr int kLanes = D / 4, kRows = 64 / kLanes;  // of a row; rows a store
      const int v = lane % kLanes, last = min(32, t.rows - wave * 32);
      float* to = p.part_o + (at * kManyRows + wave * 32) * D + 4 * v;
#pragma unroll 8
      for (int r = lane / kLanes; r < last; r += kRows)
        *reinterpret_cast<f32x4*>(to + r * D) =
            *reinterpret_cast<const f32x4*>(s_o + r * D + 4 * (v ^ (r & 15)));
    } else if (there) {
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
