// Attention over a paged KV cache held in 8 bits (kv8.cuh has the layout).
//
// With n query rows of a sequence whose cache holds `len` tokens, row i sees keys
// j < len - n + i + 1 (all `len` of them without causal limits).  With the scales a_u, b_u of
// token j's unit u, and codes k, v,
//   s_j = scale a_u (q . k_j),   o = [ sum_j p_j b_u v_j ] / sum_j p_j,   p_j = exp(s_j - M).
// A row that sees no key returns zeros and lse = -inf.
//
// Codes become fp16 exactly (one conversion for two), the query row is scaled by a power of two so
// that fp16 holds it exactly, products are summed in fp32: scores are as good as fp32's.  The scales
// are powers of two, constant over a matrix fragment of 16 tokens, and go into the softmax's factor
// (keys) and into the weights (values).
//
// The one rounding to fewer bits is that of the weights w = p b_u 2^-k to fp16, 2^-11 relative, an
// eighth of a bf16 output's own; fp16 outputs would lose by it, so for them w is two fp16 parts.  k
// is the row's own: the largest w that it has seen is near 2^7, so a token keeps fp16's
// precision down to 2^-21 of the row's largest contribution, whatever scales its tokens have and
// whatever tokens that it does not see hold.
//
// Work for few query rows is mma.sync's: scores are computed transposed, tokens x rows, so that the
// rows fill the narrow side of the instruction; what tcgen05 would save in products it would cost in
// codes written to shared memory again as 16 bits.  Rows of a tile beyond 16 go to more warps
// of the CTA, which read the same codes from shared memory: HBM delivers them once for up to 64.
//
// Every (sequence, head, tile of rows) lies on one line measured in token steps, of which each team takes
// an equal share; the parts of an item are joined by a second launch in a fixed order.
//
// What bounds it, in a captured graph: one chain of loads and the join for a few tokens (150: 7.4 us;
// 49157, 28/4 heads: 24.4); HBM for many sequences (48 of up to 8192 tokens, 32/8 heads, 412 MB:
// 79 us, 80 % of the copy rate; 24 over encoders, 16 heads: 30 us); the latency of a step with more
// rows (16 x 5 and 4 tokens, 40/8 heads, 25 and 20 rows: fp16 39.6 us, bf16 37.5, of which the
// products are 11 and 7).
#include <type_traits>

#include "attention_kv8.cuh"

namespace kvs {

namespace {

constexpr int kWarps = 4;           // a team
constexpr int kStep = 32;           // tokens a warp takes at a time
constexpr int kStage = 2 * kStep * 128;  // bytes of codes: keys, then values
constexpr int kStages = 8;          // of a team's rings together
constexpr int kOver = 256;          // what starting and ending an item costs, in tokens
// A team's share of the line is no shorter than kLeast tokens, or kFew while that takes no more than
// kSpread teams.
constexpr int kLeast = 512, kFew = 256, kSpread = 148;
// Largest weights are 2^kAbove when their row's units are set, and may come to 2^kMost.
constexpr float kAbove = 7.f, kMost = 15.f;
// Units whose scale is less than 2^-kFar of K's count in the sum of the weights alone: they weigh
// 2^(kLazy - kFar) of K's unit at most, which fp16 rounds to nothing.
constexpr float kFar = 60.f;

struct Work {
  int units;       // a sequence's share of the line
  int tiles, per;  // row tiles a head, units an item
};
template <int UNIT>
KVS_DEV Work work_of(const Attn4Launch& L, const Seq& s, int rows, int group) {
  Work w;
  w.tiles = (s.n * group + rows - 1) / rows;
  w.per = s.len > 0 && !L.whole ? (s.len + UNIT - 1) / UNIT : 1;
  w.units = w.tiles * L.heads * (w.per + kOver / UNIT);
  return w;
}

// A CTA (one an SM) is TEAMS teams of four warps, each with a share of its own, and four more warps
// of which one fetches for each team: it walks through the team's items ahead of it, so that the
// copies of the next item are on their way while this one's results are joined.
// Calls for which a team an SM is enough take CTAs of one team, which start sooner.
template <int NT, bool ONE>
struct Shape {
  static constexpr int TEAMS = ONE ? 1 : NT == 1 ? 3 : 2, THREADS = (TEAMS + 1) * kWarps * 32;
  static constexpr int CH = NT == 1 ? 64 : 128;  // channels that are joined at a time
  // registers of the launch, of the teams and of the other four warps
  static constexpr int REGS = NT == 1 ? 128 : 168, TEAM = NT == 1 ? 152 : 208,
                       OTHER = NT == 1 ? 56 : 88;
  static_assert(ONE || TEAMS * TEAM + OTHER == (TEAMS + 1) * REGS);
  static constexpr int RESULT = kWarps * 8 * NT * CH * 4;  // bytes of a team's results
  static constexpr int SMEM = 1024 + TEAMS * (kStages * kStage + RESULT);
  static_assert(SMEM <= 224 * 1024 && TEAMS * (kStages + 1) < 31);
};

KVS_DEV void team_sync(int team) {
  asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(kWarps * 32) : "memory");
}

// What a team does next: item (sequence r, head h, tile) from unit0 on, `units` of them.
struct Job {
  Seq s;
  Work wk;
  int r, h, tile, unit0, units, nrows, min_seen, limit, stop, item_end;
};
// A team's share [pos, end) of the line; `begin`: of sequence r on it.
template <int UNIT, int ROWS>
struct Share {
  int pos, end, begin, r;
  Seq own;  // sequence r's extents
  KVS_DEV bool next(const Attn4Launch& L, int group, Job& j) {
    constexpr int kOverUnits = kOver / UNIT;
    while (pos < end) {
      j.s = own;
      j.wk = work_of<UNIT>(L, j.s, ROWS, group);
      if (pos >= begin + j.wk.units) {  // on to the next sequence that has work
        begin += j.wk.units;
        own = sequence(L, ++r, false);
        continue;
      }
      const int cost = j.wk.per + kOverUnits;
      const int item = (pos - begin) / cost;
      const int from0 = pos - begin - item * cost;
      const int share = min(end - pos, cost - from0);
      // an item's overhead lies in front of its units
      j.unit0 = max(0, from0 - kOverUnits);
      j.units = max(0, from0 + share - kOverUnits) - j.unit0;
      pos += share;
      if (j.units <= 0) continue;
      j.r = r;
      j.h = item / j.wk.tiles;
      const int ti = item - j.h * j.wk.tiles;
      // low and high tiles in turn: with causal limits, neighbours add up to alike work
      j.tile = (ti & 1) ? j.wk.tiles - 1 - (ti >> 1) : ti >> 1;
      j.nrows = j.s.n * group;
      const int last_row = min(j.nrows, (j.tile + 1) * ROWS) - 1;
      j.min_seen = max(0, seen_by(L, j.s, j.tile * ROWS / group));
      j.limit = max(0, seen_by(L, j.s, last_row / group));
      j.stop = L.whole ? j.limit : min(j.limit, (j.unit0 + j.units) * UNIT);
      j.item_end = begin + (item + 1) * cost - 1;
      return true;
    }
    return false;
  }
};

struct Bars {
  uint64_t full[kStages], empty[kStages];
  uint2 note[kStages];  // the two units' scale bytes; bit 0, 1: the unit is there
};

// Fetches a team's codes: 32 tokens a stage, in turn for its TS rings.
template <int TS, int ROWS>
KVS_DEV void fetch_role(const Attn4Launch& L, const CUtensorMap* map,
                        Share<TS * kStep, ROWS> share, int group, uint32_t stages, Bars* bars) {
  constexpr int ST = kStages / TS;
  const int lane = threadIdx.x & 31;
  const bool wide = L.block_size % kStep == 0;  // the tensor map's boxes are of 32 rows
  uint32_t asked[TS] = {};  // of each ring
  Job job;
  while (share.next(L, group, job)) {
    const int from = job.unit0 * (TS * kStep);
    const int32_t* const table = L.table + job.r * L.table_stride;
    const uint8_t* const head = static_cast<const uint8_t*>(L.cache) + job.h * L.head_stride;
    // Blocks, places and scales of 16 stages' units, a lane each; and of the next 16's.
    int ids = -1, ids2 = -1, offs = 0, offs2 = 0;
    uint32_t scale = 0, scale2 = 0;
    auto look = [&](int k, int& ids, int& offs) {  // from stage k of the item on
      const int tok = from + k * kStep + kUnit8 * lane;
      ids = -1;
      if (tok < job.stop) {
        const int page = tok / L.block_size;
        offs = tok - page * L.block_size;
        ids = table[page];
        if (ids < 0 || ids >= L.num_blocks) {
          record_error(L.err, ERR_BOUNDS);
          ids = -1;
        }
      }
    };
    auto look_scale = [&](int ids, int offs, uint32_t& scale) {
      if (ids >= 0)
        scale = *reinterpret_cast<const uint16_t*>(head + ids * L.block_stride +
                                                   256ll * L.block_size + (offs >> 3));
    };
    const int all = job.stop > from ? (job.stop - from + kStep - 1) / kStep : 0;
    for (int k0 = 0; k0 < all; k0 += TS) {
#pragma unroll
      for (int ring = 0; ring < TS; ++ring) {
        const int k = k0 + ring, step = k & 15;
        if (k >= all) break;
        const uint32_t slot = asked[ring] % ST, at = ring * ST + slot;
        if (k == 0) {
          look(0, ids, offs);
          look_scale(ids, offs, scale);
        } else if (step == 0) {
          ids = ids2;
          offs = offs2;
          scale = scale2;
        } else if (step == 4) {
          look(k + 12, ids2, offs2);
        } else if (step == 10) {
          look_scale(ids2, offs2, scale2);
        }
        if (asked[ring] >= ST && !wait_phase(&bars->empty[at], (asked[ring] / ST - 1) & 1, L.err))
          return;
        ++asked[ring];
        uint64_t* const bar = &bars->full[at];
        const int id0 = __shfl_sync(0xFFFFFFFFu, ids, 2 * step);
        const int id1 = __shfl_sync(0xFFFFFFFFu, ids, 2 * step + 1);
        const int off0 = __shfl_sync(0xFFFFFFFFu, offs, 2 * step);
        const int off1 = __shfl_sync(0xFFFFFFFFu, offs, 2 * step + 1);
        if (elected()) {  // one lane: copies by several are issued one after the other anyway
          const uint32_t to = stages + at * kStage;
          // with wide boxes both units are in one block; a second one behind the end hides itself
          const int halves = wide ? 2 * (id0 >= 0) : (id0 >= 0) + (id1 >= 0);
          mbar_expect_tx(bar, halves * (kStage / 2));
          if (id0 >= 0) {
            load_rows(to, map, off0, job.h, id0, bar);
            load_rows(to + 4096, map, L.block_size + off0, job.h, id0, bar);
          }
          if (id1 >= 0 && !wide) {
            load_rows(to + 2048, map, off1, job.h, id1, bar);
            load_rows(to + 6144, map, L.block_size + off1, job.h, id1, bar);
          }
        }
        __syncwarp();
        // the scales, which an item's first copies need not wait for
        const uint32_t sc0 = __shfl_sync(0xFFFFFFFFu, scale, 2 * step);
        const uint32_t sc1 = __shfl_sync(0xFFFFFFFFu, scale, 2 * step + 1);
        if (elected()) {
          bars->note[at] = make_uint2(sc0 | sc1 << 16, (id0 >= 0 ? 1u : 0u) | (id1 >= 0 ? 2u : 0u));
          mbar_arrive(bar);
        }
        __syncwarp();
      }
    }
  }
}

// A warp takes NT * 8 rows; RG warps side by side the rows of a tile, the TS = 4 / RG such groups of
// a team every TS-th 32 tokens.  Fragments (lane = 4 g + c): K is the A operand, row m = token m,
// lane c's channels 32 c + 4 ks + 0..3 in product ks; the scores' transposed fragments (movmatrix) are
// the B operand of V^T P^T, whose A operand joins the bytes of two tokens: lane g's channels
// 16 g + 0..15, lane c's tokens 2 c, 2 c + 1, 2 c + 8, 2 c + 9.  With the copy engine's swizzle both
// are read in 16-byte pieces without bank conflicts.
template <bool FP16, int NT, int RG>
KVS_DEV void team_role(const Attn4Launch& L, Share<kWarps / RG * kStep, 8 * NT * RG> share, int group,
                       const Deal& deal, const Parts& P, int b, int team, const uint8_t* stages,
                       float* s_o, float2 (*s_ml)[8 * NT * RG], Bars* bars) {
  constexpr int ROWS = 8 * NT * RG, TS = kWarps / RG, ST = kStages / TS, UNIT = TS * kStep;
  const int tid = threadIdx.x & 127, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  const int split = warp / RG, rg = warp % RG, stage0 = split * ST;
  uint32_t taken = 0;  // steps of this ring
  bool lost = false;   // a copy did not come: nothing is waited for any more
  // fragment addresses inside a unit's 16 rows of keys and of values
  uint32_t k_at[2], v_at[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) k_at[i] = g * 128 + (((2 * c + i) ^ g) << 4);
#pragma unroll
  for (int i = 0; i < 2; ++i) v_at[i] = (2 * c + i) * 128 + ((g ^ (2 * c + i)) << 4);
  v_at[2] = v_at[0] + 1024;
  v_at[3] = v_at[1] + 1024;

  Job job;
  while (share.next(L, group, job)) {
    const Seq& s = job.s;
    const int h = job.h, nrows = job.nrows, limit = job.limit;
    const int row0 = job.tile * ROWS + rg * 8 * NT;  // of this warp
    // this warp's steps: tokens first + UNIT k + [0, 32)
    const int first = job.unit0 * UNIT + split * kStep;
    const int steps = first < job.stop ? (job.stop - first + UNIT - 1) / UNIT : 0;

    // ---- query fragments: fp16, each row scaled by a power of two so that its largest
    // element is in [2^14, 2^15); exact unless 2^-31 of the largest
    uint32_t qf[NT][8][2];
    float f[NT][2];  // of this lane's columns 2c, 2c + 1
    int seen[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      uint4 raw[4];
      const int row = row0 + nt * 8 + g;
#pragma unroll
      for (int q = 0; q < 4; ++q) raw[q] = make_uint4(0u, 0u, 0u, 0u);
      if (row < nrows) {
        const uint16_t* qp = static_cast<const uint16_t*>(L.q) +
                             (s.row0 + row / group) * L.q_ts +
                             (h * group + row % group) * L.q_hs + 32 * c;
#pragma unroll
        for (int q = 0; q < 4; ++q) raw[q] = *reinterpret_cast<const uint4*>(qp + 8 * q);
      }
      float x[4][8], top = 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        unpack8<FP16>(raw[q], x[q]);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[q][i]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
      int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
      e = top == 0.f ? 0 : max(kLowestExp, e);
      // an infinite element makes the row what is not a number
      const float up = top < INFINITY ? pow2(14 - e) * (L.scale < 0.f ? -1.f : 1.f)
                                      : __uint_as_float(0x7FC00000u);
      const float fr = fabsf(L.scale) * 1.4426950408889634f * pow2(e - 14);
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float* const y = &x[q][4 * i];
          qf[nt][2 * q + i][0] = half2_bits(y[0] * up, y[1] * up);
          qf[nt][2 * q + i][1] = half2_bits(y[2] * up, y[3] * up);
        }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        f[nt][j] = __shfl_sync(0xFFFFFFFFu, fr, (2 * c + j) * 4);
        const int cr = row0 + nt * 8 + 2 * c + j;
        seen[nt][j] = cr < nrows ? seen_by(L, s, cr / group) : 0x7FFFFFFF;
      }
    }

    float acc[8][NT][4], l[NT][2], M[NT][2], K[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][nt][i] = 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        l[nt][j] = 0.f;
        M[nt][j] = kLowest;
        K[nt][j] = -120.f;  // weights are in units of 2^K, and 2^-K is a normal number
      }
    }

    auto step = [&](auto tag, int t0, const uint8_t* st, uint32_t scales, uint32_t note) {
      constexpr bool MASKED = decltype(tag)::value;
      float sc[2][NT][4], ev[2], top[2][NT][2];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const uint32_t two = scales >> (16 * hf) & 0xFFFFu;
        const float fk = __uint_as_float((two & 0xFFu) << 23);
        ev[hf] = static_cast<float>(static_cast<int>(two >> 8) - 127);
        float a[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) a[nt][i] = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 ka = *reinterpret_cast<const uint4*>(st + 2048 * hf + k_at[i]);
          const uint4 kb = *reinterpret_cast<const uint4*>(st + 2048 * hf + k_at[i] + 1024);
          const uint32_t u[4] = {ka.x, ka.y, ka.z, ka.w}, v[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t a0 = half2_low8(u[q]), a1 = half2_low8(v[q]), a2 = half2_high8(u[q]),
                           a3 = half2_high8(v[q]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816(a[nt], a0, a1, a2, a3, qf[nt][4 * i + q][0], qf[nt][4 * i + q][1]);
          }
        }
        const bool had = note >> hf & 1u;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float fs = f[nt][j] * fk;
#pragma unroll
            for (int i = j; i < 4; i += 2) {
              // rounded before the maximum is taken off: a fused multiply-add would leave the
              // maximum's rounding over, which grows with the score
              float& x = sc[hf][nt][i];
              x = __fmul_rn(a[nt][i], fs);
              if (MASKED) {
                const int tok = t0 + 16 * hf + g + (i < 2 ? 0 : 8);
                if (!had || tok >= seen[nt][j]) x = -INFINITY;
              }
            }
            top[hf][nt][j] = fmaxf(sc[hf][nt][j], sc[hf][nt][j + 2]);
          }
      }
      // ---- a row's running maximum M, passed by up to 2^kLazy before it is moved, and the
      // exponent K of its weights' units
      bool move = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const float d = top[hf][nt][j] - M[nt][j];
            move |= d > kLazy || d + ev[hf] > K[nt][j] + kMost;
          }
      if (__any_sync(0xFFFFFFFFu, move)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float x[2] = {top[0][nt][j], top[1][nt][j]};
#pragma unroll
            for (int o = 4; o < 32; o <<= 1)
#pragma unroll
              for (int hf = 0; hf < 2; ++hf)
                x[hf] = fmaxf(x[hf], __shfl_xor_sync(0xFFFFFFFFu, x[hf], o));
            const float old = M[nt][j], m = fmaxf(old, fmaxf(x[0], x[1])), less = old - m;
            const float k = fmaxf(fmaxf(floorf(K[nt][j] + less), -120.f),
                                  ceilf(fmaxf(x[0] - m + ev[0], x[1] - m + ev[1])) - kAbove);
            const float k1 = ex2(less), k2 = ex2(less + (K[nt][j] - k));
            M[nt][j] = m;
            K[nt][j] = k;
            l[nt][j] *= k1;
#pragma unroll
            for (int d = 0; d < 8; ++d) {
              acc[d][nt][j] *= k2;
              acc[d][nt][j + 2] *= k2;
            }
          }
      }
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        uint4 raw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          raw[i] = *reinterpret_cast<const uint4*>(st + 4096 + 2048 * hf + v_at[i]);
        uint32_t w0[NT], w1[NT], rest0[NT], rest1[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float w[4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            // 2^d in the exponent: it may pass fp32's largest number where p falls below the smallest
            const float d = fmaxf(ev[hf] - K[nt][j], -kFar);
#pragma unroll
            for (int i = j; i < 4; i += 2) w[i] = ex2((sc[hf][nt][i] - M[nt][j]) + d);
            l[nt][j] = fmaf(w[j] + w[j + 2], ex2(-d), l[nt][j]);
          }
          const uint32_t lo = half2_bits(w[0], w[1]), hi = half2_bits(w[2], w[3]);
          w0[nt] = transpose8(lo);
          w1[nt] = transpose8(hi);
          if constexpr (FP16) {  // what the rounding leaves over
            rest0[nt] = transpose8(half2_bits(w[0] - h2f<true>(lo & 0xFFFFu),
                                              w[1] - h2f<true>(lo >> 16)));
            rest1[nt] = transpose8(half2_bits(w[2] - h2f<true>(hi & 0xFFFFu),
                                              w[3] - h2f<true>(hi >> 16)));
          }
        }
        uint32_t v[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[i][0] = raw[i].x, v[i][1] = raw[i].y, v[i][2] = raw[i].z, v[i][3] = raw[i].w;
        if (MASKED) {
          // what no row of the tile sees counts as zeros, whatever its bytes are
          uint32_t nan = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int tok = t0 + 16 * hf + 2 * c + (i & 1) + 8 * (i >> 1);
            const bool keep = (note >> hf & 1u) && tok < limit;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              v[i][q] = keep ? v[i][q] : 0u;
              nan |= (v[i][q] & 0x7F7F7F7Fu) + 0x01010101u;
            }
          }
          if (__any_sync(0xFFFFFFFFu, nan & 0x80808080u)) {
            // Not a number, in tokens that some rows see: zeros in the product, which would
            // carry them to the others, and NaN where a row sees one, by a product of marks.
            uint32_t s0[NT], s1[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              auto mark = [&](int i) { return sc[hf][nt][i] == -INFINITY ? 0.f : 1.f; };
              s0[nt] = transpose8(half2_bits(mark(0), mark(1)));
              s1[nt] = transpose8(half2_bits(mark(2), mark(3)));
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t is[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                is[i] = ((v[i][q] & 0x7F7F7F7Fu) + 0x01010101u) >> 7 & 0x01010101u;
                v[i][q] &= ~(is[i] * 0xFFu);
                is[i] *= 0x38u;  // e4m3's 1
              }
#pragma unroll
              for (int o = 0; o < 2; ++o) {
                const uint32_t pick = o ? 0x7362u : 0x5140u;
                const uint32_t x = __byte_perm(is[0], is[1], pick),
                               y = __byte_perm(is[2], is[3], pick);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  float n[4] = {0.f, 0.f, 0.f, 0.f};
                  mma16816(n, half2_low8(x), half2_high8(x), half2_low8(y), half2_high8(y), s0[nt],
                           s1[nt]);
#pragma unroll
                  for (int i = 0; i < 4; ++i)
                    if (n[i] > 0.f) acc[2 * q + o][nt][i] = __uint_as_float(0x7FC00000u);
                }
              }
            }
          }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int o = 0; o < 2; ++o) {  // channels 16 g + 4 q + 2 o + 0, 1
            const uint32_t pick = o ? 0x7362u : 0x5140u;
            const uint32_t x = __byte_perm(v[0][q], v[1][q], pick),
                           y = __byte_perm(v[2][q], v[3][q], pick);
            const uint32_t a0 = half2_low8(x), a1 = half2_high8(x), a2 = half2_low8(y),
                           a3 = half2_high8(y);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816(acc[2 * q + o][nt], a0, a1, a2, a3, w0[nt], w1[nt]);
            if constexpr (FP16) {
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma16816(acc[2 * q + o][nt], a0, a1, a2, a3, rest0[nt], rest1[nt]);
            }
          }
      }
    };
    for (int k = 0; k < steps; ++k) {
      const uint32_t stage = stage0 + taken % ST;
      if (!lost && !mbar_wait(&bars->full[stage], (taken / ST) & 1, L.err, ERR_MBAR_TIMEOUT))
        lost = true;
      ++taken;
      const int t0 = first + k * UNIT;
      const uint2 note = bars->note[stage];
      if (row0 < nrows) {
        if (note.y != 3u || t0 + kStep > job.min_seen)
          step(std::true_type{}, t0, stages + stage * kStage, note.x, note.y);
        else
          step(std::false_type{}, t0, stages + stage * kStage, note.x, note.y);
      }
      __syncwarp();  // the stage may be overwritten
      if (lane == 0) mbar_arrive(&bars->empty[stage]);
    }

    // ---- join the warps' results, CH channels at a time: s_o is [TS][ROWS][CH]
    constexpr int CH = Shape<NT, false>::CH, ACROSS = CH / 4;  // lanes a row
    const bool whole = job.unit0 == 0 && job.units == job.wk.per;
    const int slot = 2 * b + (job.unit0 == 0 ? 1 : 0);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float ls = l[nt][j];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) ls += __shfl_xor_sync(0xFFFFFFFFu, ls, o);
        if (g == 0) s_ml[split][rg * 8 * NT + nt * 8 + 2 * c + j] = make_float2(M[nt][j], ls);
      }
#pragma unroll 1
    for (int c0 = 0; c0 < 128; c0 += CH) {
      if (16 * g >= c0 && 16 * g < c0 + CH) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int row = rg * 8 * NT + nt * 8 + 2 * c + j;
            const float unit = pow2(static_cast<int>(K[nt][j]));
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *reinterpret_cast<float4*>(s_o + (split * ROWS + row) * CH + 16 * g - c0 + 4 * q) =
                  make_float4(acc[2 * q][nt][j] * unit, acc[2 * q][nt][j + 2] * unit,
                              acc[2 * q + 1][nt][j] * unit, acc[2 * q + 1][nt][j + 2] * unit);
          }
      }
      team_sync(team);
      const int ch = tid % ACROSS * 4;
#pragma unroll 2
      for (int row = tid / ACROSS; row < ROWS; row += kWarps * 32 / ACROSS) {
        const int rr = job.tile * ROWS + row;
        if (rr >= nrows) break;
        float m = kLowest, ls = 0.f;
        float2 ml[TS];
#pragma unroll
        for (int w = 0; w < TS; ++w) {
          ml[w] = s_ml[w][row];
          m = fmaxf(m, ml[w].x);
        }
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < TS; ++w) {
          const float k2 = ex2(ml[w].x - m);
          const float4 x = *reinterpret_cast<const float4*>(s_o + (w * ROWS + row) * CH + ch);
          ls = fmaf(ml[w].y, k2, ls);
          o.x = fmaf(x.x, k2, o.x);
          o.y = fmaf(x.y, k2, o.y);
          o.z = fmaf(x.z, k2, o.z);
          o.w = fmaf(x.w, k2, o.w);
        }
        if (whole) {
          const long long tq = s.row0 + rr / group;
          const int hq = h * group + rr % group;
          const float inv = ls == 0.f ? 0.f : __fdividef(1.f, ls);
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(L.out) + tq * L.o_ts + hq * L.o_hs + c0 +
                                    ch) =
              make_uint2(f2h2<FP16>(o.x * inv, o.y * inv), f2h2<FP16>(o.z * inv, o.w * inv));
          if (L.lse != nullptr && c0 + ch == 0)
            L.lse[tq * L.q_heads + hq] =
                ls == 0.f ? -INFINITY : (m + log2f(ls)) * 0.69314718055994531f;
        } else {
          *reinterpret_cast<float4*>(
              P.o + (static_cast<long long>(slot) * ROWS + row) * 128 + c0 + ch) = o;
          if (c0 + ch == 0) P.ml[slot * ROWS + row] = make_float2(m, ls);
        }
      }
      team_sync(team);  // the next results take their place
    }
    if (!whole && job.unit0 == 0 && tid == 0)  // parts: up to the team that holds the item's end
      P.desc[b] = make_int4(s.row0, h, job.tile, (deal.owner(job.item_end) - b + 1) |
                                                      min(ROWS, nrows - job.tile * ROWS) << 16);
  }
}

template <bool FP16, int NT, int RG, bool ONE>
__global__ void __launch_bounds__(Shape<NT, ONE>::THREADS, 1)
    k_attn8(const __grid_constant__ Attn4Launch L, const __grid_constant__ CUtensorMap map) {
  using S = Shape<NT, ONE>;
  constexpr int ROWS = 8 * NT * RG, TS = kWarps / RG, UNIT = TS * kStep, TEAMS = S::TEAMS;
  constexpr int WARPS = S::THREADS / 32;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  __shared__ Bars s_bars[TEAMS];
  __shared__ int s_scan[WARPS], s_begin[TEAMS], s_seq[TEAMS];
  __shared__ Seq s_own[TEAMS];
  __shared__ float2 s_ml[TEAMS][TS][ROWS];
  __shared__ int2 s_named[WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = L.q_heads / L.heads;
  // Teams are numbered across the SMs first: few of them get an SM each.
  const int B = gridDim.x * TEAMS;
  const Parts P = parts(L.scratch, B, ROWS);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- the teams' shares [pos, end) and the sequences that they begin in
  if (warp == WARPS - 1) {
    if (lane < TEAMS * kStages) {
      mbar_init(&s_bars[lane / kStages].full[lane % kStages], 1);
      mbar_init(&s_bars[lane / kStages].empty[lane % kStages], RG);
      fence_mbar_init();
    } else if (lane < TEAMS * (kStages + 1)) {
      P.desc[(lane - TEAMS * kStages) * gridDim.x + blockIdx.x] = make_int4(-1, 0, 0, 0);
    } else if (lane == 31) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map)));
    }
  }
  int U = 0, mine = 0;
  Seq own = {};
  Named named;
  for (int r = tid; r < L.seqs; r += S::THREADS) {
    own = sequence(L, r, blockIdx.x == 0);
    named.take(L, own, r);
    mine = work_of<UNIT>(L, own, ROWS, group).units;
    U += mine;
  }
  auto scan = [&](int x) {  // the sum of the warp's up to this lane
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xFFFFFFFFu, x, o);
      if (lane >= o) x += y;
    }
    return x;
  };
  int inc = scan(U);
  if (lane == 31) s_scan[warp] = inc;
  named.leave(L, s_named);
  __syncthreads();
  named.clear<WARPS>(L, s_named);
  U = 0;
  int before = inc;  // of the line up to this thread's sequence (if there are no more than threads)
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += s_scan[w];
    U += s_scan[w];
  }
  constexpr int kLeastUnits = kLeast / UNIT, kFewUnits = kFew / UNIT, kOverUnits = kOver / UNIT;
  const int used = min(B, L.whole ? U / (1 + kOverUnits)  // an item a team
                                  : max((U + kLeastUnits - 1) / kLeastUnits,
                                        min(kSpread, (U + kFewUnits - 1) / kFewUnits)));
  const Deal deal{U / max(used, 1), U % max(used, 1)};
  auto found = [&](int r, int from, int to) {  // sequence r has [from, to) of the line
#pragma unroll
    for (int t = 0; t < TEAMS; ++t) {
      const int b = t * gridDim.x + blockIdx.x, pos = deal.begin(b);
      if (b < used && from <= pos && pos < to) {
        s_seq[t] = r;
        s_begin[t] = from;
        s_own[t] = own;
      }
    }
  };
  if (L.seqs <= S::THREADS) {
    found(tid, before - mine, before);
  } else {
    int base = 0;
    for (int r0 = 0; r0 < L.seqs; r0 += S::THREADS) {
      const int r = r0 + tid;
      own = {};
      if (r < L.seqs) own = sequence(L, r, false);
      mine = r < L.seqs ? work_of<UNIT>(L, own, ROWS, group).units : 0;
      inc = scan(mine);
      __syncthreads();
      if (lane == 31) s_scan[warp] = inc;
      __syncthreads();
      before = base + inc;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        if (w < warp) before += s_scan[w];
        base += s_scan[w];
      }
      found(r, before - mine, before);
    }
  }
  __syncthreads();
  const bool fetches = warp >= TEAMS * kWarps;
  const int team = fetches ? warp - TEAMS * kWarps : warp / kWarps;
  const int b = team * gridDim.x + blockIdx.x;
  Share<UNIT, ROWS> share{};
  if (team < TEAMS && b < used)
    share = {deal.begin(b), deal.begin(b + 1), s_begin[team], s_seq[team], s_own[team]};
  uint8_t* const stages = smem + min(team, TEAMS - 1) * (kStages * kStage);
  if (!fetches) {
    if constexpr (!ONE) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::TEAM));
    team_role<FP16, NT, RG>(L, share, group, deal, P, b, team, stages,
                            reinterpret_cast<float*>(smem + TEAMS * kStages * kStage +
                                                     team * S::RESULT),
                            s_ml[team], &s_bars[team]);
  } else {
    if constexpr (!ONE) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::OTHER));
    fetch_role<TS, ROWS>(L, &map, share, group, smem_u32(stages), &s_bars[min(team, TEAMS - 1)]);
  }
}

struct Grid {
  int ctas, teams, rows;
  long long items;
  bool fits;   // the line's length is an int
  bool split;  // whether items may be split
  bool one;    // a team a CTA
};

// Tables of at most so many tokens are not split: the launch that joins the parts takes longer
// than a second step.
constexpr int kWholeTokens = 256;

Grid grid_of(const Attn4Launch* L) {
  Grid g;
  const int group = L->q_heads / L->heads;
  const long long rows = static_cast<long long>(L->max_q) * group;
  g.rows = rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
  const int unit = g.rows <= 16 ? 128 : g.rows == 32 ? 64 : 32;
  const long long room = static_cast<long long>(L->table_cols) * L->block_size;
  const long long per = (room + unit - 1) / unit;
  const long long items = static_cast<long long>(L->seqs) * L->heads *
                          ((rows + g.rows - 1) / g.rows);
  g.split = room > kWholeTokens;
  const long long units = items * (g.split ? per : 1);
  g.items = items;
  g.fits = items < (1ll << 31) && items * (per + 1 + kOver / unit) < (1ll << 31);
  g.ctas = static_cast<int>(units < 148 ? units : 148);
  g.one = units <= 148;
  g.teams = g.ctas * (g.one ? 1 : g.rows == 8 ? Shape<1, false>::TEAMS : Shape<2, false>::TEAMS);
  return g;
}

// Whether a call goes to attention_kv8_tile.cu: many rows a kv head, and enough of them by what the
// host knows (max_query_len, and the tokens that the table has room for).  Measured, us here / there
// (bf16; fp16 is 10 to 16 % more here, 8 there): 32 sequences of 2000 tokens, 8 heads: 48 rows
// 99 / 101, 64 rows 101 / 102 (fp16 115 / 111), 96 rows 141 / 103; 16 of 2000: 64 rows 59 / 60, 96 rows
// 80 / 61; 8 of 8000, 4 heads: 56 rows 55 / 51, 84 rows 74 / 51; 64 of 1000, 4 heads: 84 rows 84 / 75.
// With little to do (Mi rows times tokens times heads): one of 1024 tokens, 4 heads: 448 rows (1.8 Mi)
// 22 / 26; one of 4000, 8 heads: 128 rows (3.9 Mi) 33 / 28, 512 rows 56 / 37; one of 16000, 4 heads:
// 112 rows (6.8 Mi) 40 / 31.
constexpr int kManyRows = 64;
constexpr long long kMuchWork = 3ll << 20;
bool many_rows(const Attn4Launch* L) {
  const long long rows = static_cast<long long>(L->max_q) * (L->q_heads / L->heads);
  const double work = static_cast<double>(rows) * L->seqs * L->heads * L->table_cols *
                      L->block_size;
  return rows > kManyRows && work > static_cast<double>(kMuchWork);
}

template <bool FP16, int NT, int RG, bool ONE>
cudaError_t launch_shape(const Attn4Launch& L, const Grid& g, const CUtensorMap& map, cudaStream_t s) {
  using S = Shape<NT, ONE>;
  const cudaError_t e = cudaFuncSetAttribute(
      k_attn8<FP16, NT, RG, ONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
  if (e != cudaSuccess) return e;
  k_attn8<FP16, NT, RG, ONE><<<g.ctas, S::THREADS, S::SMEM, s>>>(L, map);
  return cudaGetLastError();
}
template <bool FP16, int NT, int RG>
cudaError_t launch(const Attn4Launch& L, const Grid& g, const CUtensorMap& map, cudaStream_t s) {
  const cudaError_t e = g.one ? launch_shape<FP16, NT, RG, true>(L, g, map, s)
                              : launch_shape<FP16, NT, RG, false>(L, g, map, s);
  if (e != cudaSuccess || !g.split) return e;
  constexpr int ROWS = 8 * NT * RG;
  return launch_join<FP16, ROWS>(L, g.teams, g.items, s);
}
template <bool FP16>
cudaError_t launch_rows(const Attn4Launch& L, const Grid& g, const CUtensorMap& map,
                        cudaStream_t s) {
  return g.rows == 8    ? launch<FP16, 1, 1>(L, g, map, s)
         : g.rows == 16 ? launch<FP16, 2, 1>(L, g, map, s)
         : g.rows == 32 ? launch<FP16, 2, 2>(L, g, map, s)
                        : launch<FP16, 2, 4>(L, g, map, s);
}

}  // namespace
}  // namespace kvs

using namespace kvs;

extern "C" {

long long kvs_attn8_scratch_bytes(const Attn4Launch* L) {
  if (many_rows(L)) return attn8_tile_scratch(*L);
  const Grid g = grid_of(L);
  return 16ll * g.teams + 2ll * g.teams * g.rows * (8 + 512);
}

int kvs_attention_kv8(const Attn4Launch* L, void* stream) {
  if (L->seqs <= 0 || L->max_q <= 0 || L->tokens <= 0 || L->heads <= 0) return 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  CUtensorMap map;
  if (many_rows(L)) {
    if (!record_map(*L, kUnit8, &map)) return -3;
    return attn8_tile_launch(*L, map, s) == cudaSuccess ? 0 : -1;
  }
  const Grid g = grid_of(L);
  if (!g.fits) return -2;
  Attn4Launch A = *L;
  A.whole = !g.split;
  if (!record_map(A, A.block_size % kStep == 0 ? kStep : kUnit8, &map)) return -3;
  const cudaError_t e = L->fp16 ? launch_rows<true>(A, g, map, s) : launch_rows<false>(A, g, map, s);
  return e == cudaSuccess ? 0 : -1;
}

}  // extern "C"
