// Attention over a paged 4-bit cache for many query rows (prefill chunks).
//
// The mathematics is attention_kv4.cu's; here 2 x 128 query rows (several
// tokens times the query heads of one kv head) share each key, so the keys
// are worth turning into 16-bit tiles once, for tcgen05:
//   S = Q K^T, O += P V, fp16 products of 128 rows and 64 tokens into tensor memory.
// K and V become fp16 with one power of two for each 32 tokens, chosen from
// the largest step and mid among them; the power goes into the softmax's factor (K) and, where it
// is not the largest that the row has seen, into the exponentials (V), a row's O being kept in units
// of that one.  Where 32 tokens' scales are more than 2^8 apart, each takes its own power: else
// a large token would take the small ones' bits from the rows that do not see it.  K's tile
// holds step (code - 8) alone; mid times the sum of the group's query elements is 16 more columns
// of the product: that sum in three fp16 parts against mid three times.
//
// Roundings to fewer bits than fp32's:
//   K, bf16 caches: none, step (code - 8) has 8 + 3 bits and fp16 holds 11.
//   K and V, fp16 caches: none to speak of.  A step has 11 bits, so a second tile holds what the
//     first one's rounding leaves over, and each product is taken with both.  Without it scores
//     were off by 2^-11 of |q| |k| (errors of outputs and lse four times those of fp32 arithmetic;
//     2 x 700 rows over 3000 tokens, 28/4 heads, 100 us); with it 135 us.
//   V, bf16 caches: to fp16, 2^-11 of |v| at most, an eighth of the output's own rounding.
//   Weights: to fp16, 2^-11, as the matrix instructions' A operand has to be of V's type; their
//     sum is taken before that.  An fp16 output's error grows by a third (2.1e-4 to 2.8e-4 of the
//     norm), a bf16 output's does not change; three parts of fp32 weights would need twice the
//     products and tensor memory, of which none is left.
//
// Roles of a CTA (one an SM, 16 warps whose registers are dealt out anew):
//   warps 0-3, 4-7   softmax of query tile 0, 1: a thread a row, which it reads
//                    from tensor memory and writes back as fp16 exponentials,
//                    the A operand of O += P V
//   warps 8-11       packed rows to fp16 tiles in shared memory, a thread a token
//   warps 12-15      issue the matrix instructions: S of tile 0, 1, O of tile 0, 1
// The softmax warps take 64 tokens' scores at a time into registers, so that the next ones are
// computed while they work.  O stays in tensor memory; it is rescaled by the
// softmax warps when 64 weights of a row sum up to more than kMostSum, which
// after the first tiles is rare.
//
// What bounds it: the softmax warps' chain of barriers, tensor memory and exponentials, about
// 2400 clocks for 64 tokens of both tiles, of which the exponentials' rate (16 a clock and SM)
// is 1024 and the products take 1320 (fp16 caches: 2560, and twice the conversion).  2 x 2048
// tokens over up to 8193, 28/4 heads (361 GFLOP), bf16: 472 us in a captured graph, 489 in calls
// of their own, 738 TFLOP/s; on mma.sync, a warp 16 rows, it was 2000 us.
//
// The work is dealt out as in attention_kv4.cu, here by the number of visible
// keys a tile has, so that causal tiles of a long chunk load all SMs alike.
#include "attention_tile.cuh"

namespace kvs {

namespace {

constexpr int kOverTile = 2;  // an item's own cost, in steps
// Tokens (of 32) with scales less than kApart of the largest take a scale each: a row may see only
// the small ones, or need their bits.
constexpr float kApart = 0x1p-8f;
constexpr uint32_t kHides = 1, kWideK = 2, kWideV = 4;
constexpr int kFar = 60;
// A score is a factor times 128 products of less than 2^15 and 2^11.  Where the factor lets it pass
// 2^27, or tokens have a scale each, the product is rounded before the maximum is taken off: the
// fused multiply-add leaves the maximum's own rounding over, up to 2^-25 of it, and weights are 2 to
// that from where they should be (the same for all of a row's, so that 2^4 does no harm).
constexpr float kHuge = 0x1p-6f;

struct Ctrl {
  uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[2], s_free[2], p_full[2][2], pv_done[2][2], e_full[4];  // [tile][buffer]
  uint32_t tmem;
  // What the converting warps say of a step (ring of four), by 32 tokens:
  float k_up[4][4];        // K in shared memory times this is K
  int v_exp[4][4];         // V in shared memory times 2^this is V
  uint32_t gone[4][4];     // tokens whose block does not exist
  uint32_t bad[4][4][4];   // [..][group] tokens with a step or mid of V that is not finite
  uint32_t flags[4][4];    // kHides: any of the two is set; kWideK, kWideV: a scale each token,
  float k_tok[4][kTile];   //   in the place of k_up,
  float v_tok[4][kTile];   //   and 2^v_exp
  long long scan[kThreads / 32];
  int2 named[kThreads / 32];
  long long begin;
  int seq;
};

// Behind the tiles: [128 rows][16] fp16, two for the queries, two for the keys' stages.
constexpr int kMidTile = 4096;
constexpr int kMidAt = 12 * kHalfTile, kCtrlAt = kMidAt + 4 * kMidTile;
constexpr int kSmem = 1024 + kCtrlAt + static_cast<int>(sizeof(Ctrl));
static_assert(kSmem <= 227 * 1024);

// The 16 extra columns: no swizzle, cores of 8 rows by 16 bytes, the two of a row 128 bytes
// apart (leading offset), groups of 8 rows 256 bytes (stride offset).
constexpr uint32_t kMidHigh = (256u >> 4) | (1u << 14);
KVS_DEV uint32_t mid_desc(uint32_t saddr) { return (saddr >> 4) | ((128u >> 4) << 16); }
KVS_DEV uint32_t mid_at(int row) { return (row >> 3) * 256 + (row & 7) * 16; }
// Column 3 g + 0..2 of the extra ones belongs to group g: `part(g, i)` packed into a row's two
// 16-byte chunks.
template <int NG, class F>
KVS_DEV void store_mids(uint8_t* tile, int row, F part) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int a = 2 * i, b = 2 * i + 1;
    const uint32_t lo = a < 3 * NG ? part(a / 3, a % 3) : 0u;
    const uint32_t hi = b < 3 * NG ? part(b / 3, b % 3) : 0u;
    w[i] = lo | (hi << 16);
  }
  *reinterpret_cast<uint4*>(tile + mid_at(row)) = make_uint4(w[0], w[1], w[2], w[3]);
  *reinterpret_cast<uint4*>(tile + mid_at(row) + 128) = make_uint4(w[4], w[5], w[6], w[7]);
}
constexpr float kMidUp = 128.f;  // mids times this, query sums by it: both inside fp16's range
// ---------------------------------------------------- packed rows to tiles
// Where a step's tiles lie.  bf16 caches: two slots of 128 tokens, a step in each in turn.  fp16
// caches: tokens 0..63 of every step are slot 0, 64..127 slot 1; the first 32 KB hold the tile
// rounded to fp16, the next 32 KB, kRestAt on, what that leaves over.
template <bool FP16>
KVS_DEV uint32_t slot_of(uint32_t step, uint32_t half) {
  return FP16 ? half : step & 1;
}
template <bool FP16>
KVS_DEV uint32_t phase_of(uint32_t step) {  // of its slot's barriers
  return (FP16 ? step : step >> 1) & 1;
}
constexpr int kRestAt = 2 * kHalfTile;

template <bool FP16, int NG>
KVS_DEV void convert_role(const Attn4Launch& L, Walk<kOverTile, false> walk, int group, uint8_t* q_tile,
                          uint8_t* k_tile, uint8_t* v_tile, Ctrl* C) {
  const int lane = threadIdx.x & 31, seg = (threadIdx.x >> 5) & 3, row = seg * 32 + lane;
  constexpr uint32_t kInf = FP16 ? 0x7C00u : 0x7F80u;
  constexpr uint32_t k1024 = 0x64006400u;
  uint32_t step_no = 0;
  Piece p;
  while (walk.next(L, group, p)) {
    const uint8_t* const head = static_cast<const uint8_t*>(L.cache) + p.h * L.head_stride;
    const int32_t* const table = L.table + p.r * L.table_stride;
    const Kv4Record R{NG, L.block_size};
    // A step's row of this thread: nothing behind `stop`, nor in a block that is not there.
    const uint8_t* rec = nullptr;
    int off = 0;
    bool gone = false;
    auto locate = [&](int j) {
      const int tok = p.start + j * kTile + row;
      rec = nullptr;
      gone = false;
      if (tok < p.stop) {
        const int page = tok / L.block_size;
        off = tok - page * L.block_size;
        const int id = table[page];
        gone = id < 0 || id >= L.num_blocks;
        if (gone) record_error(L.err, ERR_BOUNDS);
        else rec = head + id * L.block_stride;
      }
    };
    uint4 code[2][4];
    uint32_t meta[2][NG], coming[2][NG];
    auto load_codes = [&](int v) {
      const uint4* src = reinterpret_cast<const uint4*>(rec + R.codes(v, off));
#pragma unroll
      for (int i = 0; i < 4; ++i) code[v][i] = rec ? src[i] : make_uint4(0u, 0u, 0u, 0u);
    };
    auto load_meta = [&]() {
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const uint32_t* src = reinterpret_cast<const uint32_t*>(rec + R.meta(v, off));
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) coming[v][gr] = rec ? src[gr] : 0u;
      }
    };
    if (p.steps > 0) {
      locate(0);
      load_meta();
      load_codes(0);
      load_codes(1);
    }
    for (int j = 0; j < p.steps; ++j, ++step_no) {
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) meta[v][gr] = coming[v][gr];
      const uint32_t lost = __ballot_sync(0xFFFFFFFFu, gone);
      if (j + 1 < p.steps) locate(j + 1);  // its loads go out as registers become free
      // exponent of the largest finite step or mid of the warp's 32 tokens, or of each one's
      float up[2], down[2];
      int exps[2];
      uint32_t bad[NG], wide = 0;
      const int ring = step_no & 3;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) bad[gr] = 0;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        uint32_t top = 0;
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          const uint32_t a = meta[v][gr] & 0x7FFFu, z = (meta[v][gr] >> 16) & 0x7FFFu;
          const bool fine = a < kInf && z < kInf;
          if (fine) top = max(top, max(a, z));
          if (v == 1) {
            bad[gr] = __ballot_sync(0xFFFFFFFFu, !fine);
            if (!fine) meta[v][gr] = 0;  // rows that see it are marked instead
          }
        }
        const float own = h2f<FP16>(top);
        float most = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(own)));
        if (__any_sync(0xFFFFFFFFu, own < most * kApart && own != 0.f)) {
          wide |= v ? kWideV : kWideK;
          most = own;
        }
        // in steps of 16, so that V's powers seldom differ; K of zeros gets any
        int e = max(static_cast<int>(__float_as_uint(most) >> 23) - 127, kLowestExp);
        e = (v == 0 && most == 0.f ? 0 : (e + 3) & ~3) - 7;
        up[v] = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        down[v] = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
        exps[v] = e;
      }
      if (wide) {
        C->k_tok[ring][row] = down[0];
        C->v_tok[ring][row] = down[1];
        __syncwarp();
      }
      if (lane == 0) {
        uint32_t any = lost;
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          C->bad[ring][seg][gr] = bad[gr];
          any |= bad[gr];
        }
        C->k_up[ring][seg] = down[0];  // where they are apart, nobody takes these two
        C->v_exp[ring][seg] = exps[1];
        C->gone[ring][seg] = lost;
        C->flags[ring][seg] = (any ? kHides : 0u) | wide;
        mbar_arrive(&C->e_full[ring]);
      }
      const uint32_t slot = slot_of<FP16>(step_no, seg >> 1);
      const uint32_t again = phase_of<FP16>(step_no) ^ 1;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        uint64_t* const empty = v ? &C->v_empty[slot] : &C->k_empty[slot];
        if (!KVS_WAIT(empty, again)) return;
        uint8_t* const dst = (v ? v_tile : k_tile) + (FP16 ? 0 : slot * 2 * kHalfTile);
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[4 * i] = code[v][i].x;
          w[4 * i + 1] = code[v][i].y;
          w[4 * i + 2] = code[v][i].z;
          w[4 * i + 3] = code[v][i].w;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t m = meta[v][q * NG / 4];
          const __half2 step = __float2half2_rn(h2f<FP16>(m & 0xFFFFu) * up[v]);
          const __half2 mid = __float2half2_rn(h2f<FP16>(m >> 16) * up[v]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            // the eight codes of channels 32 q + 8 c + 0..7, pairs (i, i + 4)
            const uint32_t x = v == 0 ? w[4 * c + q]
                                      : __byte_perm(w[4 * c + (q >> 1)], w[4 * c + 2 + (q >> 1)],
                                                    (q & 1) ? 0x7632 : 0x5410);
            uint32_t u[4], low[4];
            codes4(x, k1024, u);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const __half2 code2 = *reinterpret_cast<const __half2*>(&u[i]);
              __half2 y, rest;
              if constexpr (FP16) {
                y = __hmul2(code2, step);
                rest = __hfma2(code2, step, __hneg2(y));  // exact
                if (v == 1) {  // what y + mid leaves over, by the two-sum of its terms
                  const __half2 z = __hadd2_rn(y, mid), w = __hsub2_rn(z, y);
                  rest = __hadd2_rn(rest, __hadd2_rn(__hsub2_rn(y, __hsub2_rn(z, w)),
                                                     __hsub2_rn(mid, w)));
                  y = z;
                }
              } else {
                y = v == 0 ? __hmul2(code2, step) : __hfma2(code2, step, mid);
                rest = y;
              }
              u[i] = *reinterpret_cast<const uint32_t*>(&y);
              low[i] = *reinterpret_cast<const uint32_t*>(&rest);
            }
            uint8_t* const at = dst + chunk_at(row, 4 * q + c);
            *reinterpret_cast<uint4*>(at) = make_uint4(u[0], u[1], u[2], u[3]);
            if constexpr (FP16)
              *reinterpret_cast<uint4*>(at + kRestAt) = make_uint4(low[0], low[1], low[2], low[3]);
          }
        }
        if (v == 0)
          store_mids<NG>(q_tile + kMidAt + (FP16 ? 2 : 2 + slot) * kMidTile, row, [&](int gr, int) {
            return f2h<true>(h2f<FP16>(meta[0][gr] >> 16) * (up[0] * kMidUp));
          });
        if (j + 1 < p.steps) {
          if (v == 0) load_meta();
          load_codes(v);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(v ? &C->v_full[slot] : &C->k_full[slot]);
      }
    }
  }
}

// ------------------------------------------------------ matrix instructions
// Four warps issue them, one a query tile x and product, each on a scheduler of its own: all
// from one warp, its scheduler's two softmax warps were a third slower than the others.
//
// Scores of half i + 1 are asked for as soon as the softmax warps have those of half i in their
// registers, so they find them ready when they are through; the weights have two buffers of
// their own.  A stage is free when both tiles' products with it are done; without a second tile
// its warps only say so.
template <bool FP16, bool QK>
KVS_DEV void mma_role(const Attn4Launch& L, Walk<kOverTile, false> walk, int group, int x, uint32_t q_tile,
                      uint32_t kv_tile, uint32_t tmem, Ctrl* C) {
  uint32_t step_no = 0, piece_no = 0, half_no = 0;
  Piece p;
  const uint32_t qd = uniform(k_desc(q_tile) + x * (2 * kHalfTile >> 4)),
                 qm = uniform(mid_desc(q_tile + kMidAt) + x * (kMidTile >> 4)),
                 km = uniform(mid_desc(q_tile + kMidAt + 2 * kMidTile)),
                 kvd = uniform(QK ? k_desc(kv_tile) : mn_desc(kv_tile)),
                 scores = uniform(tmem + 64 * x), weights = uniform(tmem + kWeightsAt + 64 * x),
                 result = uniform(tmem + kOutAt + 128 * x);
  while (walk.next(L, group, p)) {
    if (p.steps == 0) continue;
    const int H = static_cast<int>(uniform(p.halves));
    const bool idle = x == 1 && !p.two;
    if (QK && !idle && !KVS_WAIT(&C->q_full[x], piece_no++ & 1)) return;
    uint64_t *const fulls = QK ? C->k_full : C->v_full, *const empties = QK ? C->k_empty : C->v_empty;
    for (int i = 0; i < H; ++i) {
      const uint32_t no = step_no + (i >> 1), slot = slot_of<FP16>(no, i & 1);
      const bool last = FP16 || (i & 1) || i == H - 1;  // half of the slot
      if ((FP16 || !(i & 1)) && !KVS_WAIT(&fulls[slot], phase_of<FP16>(no))) return;
      uint64_t* const empty = &empties[slot];
      if (idle) {
        if (last && (threadIdx.x & 31) == 0) mbar_arrive(empty);
        continue;
      }
      const uint32_t b = kvd + (FP16 ? 0 : slot * (2 * kHalfTile >> 4)) + (i & 1) * (8192 >> 4);
      if constexpr (QK) {
        if (i > 0 && !KVS_WAIT(&C->s_free[x], (half_no - 1) & 1)) return;
        tc_fence_after();
        const uint32_t bm = km + (FP16 ? 0 : slot * (kMidTile >> 4)) + (i & 1) * (2048 >> 4);
        if (elected()) {
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            const uint32_t off = ((ks >> 2) * kHalfTile + (ks & 3) * 32) >> 4;
            mma_qk<kDescHigh>(scores, qd + off, b + off, ks > 0 ? 1u : 0u);
            if constexpr (FP16) mma_qk<kDescHigh>(scores, qd + off, b + (kRestAt >> 4) + off, 1u);
          }
          mma_qk<kMidHigh>(scores, qm, bm, 1u);
          umma_commit(&C->s_full[x]);
          if (last) umma_commit(empty);
        }
      } else {
        const uint32_t buf = half_no & 1;
        if (!KVS_WAIT(&C->p_full[x][buf], (half_no >> 1) & 1)) return;
        tc_fence_after();
        if (elected()) {
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {  // 16 tokens: two groups of eight rows, 8 columns of P
            const uint32_t p = weights + 32 * buf + 8 * ks, at = b + ks * (2048 >> 4);
            mma_pv(result, p, at, ks > 0 || i > 0 ? 1u : 0u);
            if constexpr (FP16) mma_pv(result, p, at + (kRestAt >> 4), 1u);
          }
          umma_commit(&C->pv_done[x][buf]);
          if (last) umma_commit(empty);
        }
      }
      __syncwarp();
      ++half_no;
    }
    if (FP16 && (H & 1)) {  // the step's second half, which nothing needs
      if (!KVS_WAIT(&fulls[1], phase_of<FP16>(step_no + (H >> 1)))) return;
      if ((threadIdx.x & 31) == 0) mbar_arrive(&empties[1]);
    }
    // the last half's scores were taken, too: one phase of s_free a half
    if (QK && !idle && !KVS_WAIT(&C->s_free[x], (half_no - 1) & 1)) return;
    step_no += p.steps;
  }
  // The last products' commits arrive on their own: not after the CTA has gone.
  for (uint32_t back = 1; back < 3 && step_no >= (FP16 ? 1 : back); ++back) {
    const uint32_t no = step_no - (FP16 ? 1 : back), slot = slot_of<FP16>(no, back & 1);
    if (!KVS_WAIT(QK ? &C->k_empty[slot] : &C->v_empty[slot], phase_of<FP16>(no))) return;
  }
}

// ------------------------------------------------------------------ softmax
template <bool FP16, int NG>
KVS_DEV void softmax_role(const Attn4Launch& L, Walk<kOverTile, false> walk, int group, uint8_t* q_tile,
                          uint32_t tmem, const Parts& P, Ctrl* C) {
  const int x = threadIdx.x >> 7, row = threadIdx.x & 127;
  const uint32_t lanes = static_cast<uint32_t>((threadIdx.x >> 5) & 3) << 21;  // a warp's 32
  const uint32_t S = tmem + 64 * x + lanes, O = tmem + kOutAt + 128 * x + lanes;
  uint8_t* const qt = q_tile + x * 2 * kHalfTile;
  uint32_t step_no = 0, half_no = 0;
  Piece p;
  while (walk.next(L, group, p)) {
    if (x == 1 && !p.two) {
      step_no += p.steps;
      continue;
    }
    const int rr = p.tile * kRows + x * 128 + row;
    const bool mine = rr < p.nrows;
    const long long tq = p.s.row0 + rr / group;
    const int hq = p.h * group + rr % group;
    const int seen = mine ? p.s.len - p.s.n + rr / group + 1 : 0;
    float m = kLowest, l = 0.f, f = 0.f;
    int E = kLowestExp;  // of this row's units
    uint32_t poison = 0;
    if (p.steps > 0) {
      // ---- the row as fp16, scaled by a power of two: largest element in [2^14, 2^15)
      uint4 raw[16] = {};
      if (mine) {
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(L.q) +
                                                          tq * L.q_ts + hq * L.q_hs);
#pragma unroll
        for (int i = 0; i < 16; ++i) raw[i] = src[i];
      }
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float y[8];
        unpack8<FP16>(raw[i], y);
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(y[k]));
      }
      int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
      e = top == 0.f ? 0 : max(kLowestExp, e);
      const float up = __uint_as_float(static_cast<uint32_t>(127 + 14 - e) << 23) *
                       (L.scale < 0.f ? -1.f : 1.f);
      f = fabsf(L.scale) * 1.4426950408889634f *
          __uint_as_float(static_cast<uint32_t>(127 - 14 + e) << 23);
      float sums[NG];
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) sums[gr] = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float y[8];
        unpack8<FP16>(raw[i], y);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          y[k] *= up;
          sums[i * NG / 16] += y[k];
        }
        *reinterpret_cast<uint4*>(qt + chunk_at(row, i)) =
            make_uint4(half2_bits(y[0], y[4]), half2_bits(y[1], y[5]), half2_bits(y[2], y[6]),
                       half2_bits(y[3], y[7]));
      }
      store_mids<NG>(q_tile + kMidAt + x * kMidTile, row, [&](int gr, int i) {
        float rest = sums[gr] * (1.f / kMidUp);
        uint32_t part = f2h<true>(rest);
        for (; i > 0; --i) {  // what the parts before leave over
          rest -= h2f<true>(part);
          part = f2h<true>(rest);
        }
        return part;
      });
      fence_proxy_async_smem();
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(&C->q_full[x]);
      // of the keys' scale, for scores that the exponentials take as they are
      const float up_most =
          kHuge / __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(f)));
      // tokens that every row of this warp sees
      const int all_see = __reduce_min_sync(0xFFFFFFFFu, mine ? max(seen, 0) : 0x7FFFFFFF);
      const int plain_to = min(all_see, p.stop);
      // what the converting warps say of half i's tokens, read a half ahead
      struct {
        uint32_t flag;
        int v_exp[2];
        float k_up[2];
      } said;
      auto listen = [&](int i) {
        const uint32_t ring = (step_no + (i >> 1)) & 3, seg0 = 2 * (i & 1);
        said.flag = C->flags[ring][seg0] | C->flags[ring][seg0 + 1];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          said.v_exp[k] = C->v_exp[ring][seg0 + k];
          said.k_up[k] = C->k_up[ring][seg0 + k];
        }
      };
      // The first scores' barrier before the converting warps' one: tile 1 walks past pieces
      // without a second tile and waits for nothing there, so it can be many steps ahead, and a
      // parity cannot tell the phase wanted from the one two before it.  Once the scores are there,
      // e_full is past this step and cannot be a phase further.
      if (!KVS_WAIT(&C->s_full[x], half_no & 1)) return;
      if (!KVS_WAIT(&C->e_full[step_no & 3], (step_no >> 2) & 1)) return;
      listen(0);
      uint32_t s_ready = 1;
      for (int i = 0; i < p.halves; ++i, ++half_no) {
        const int ring = (step_no + (i >> 1)) & 3, seg0 = 2 * (i & 1), t0 = p.start + 64 * i;
        const uint32_t buf = half_no & 1, W = tmem + kWeightsAt + 64 * x + 32 * buf + lanes;
        const uint32_t flag = said.flag;
        int v_exp[2] = {said.v_exp[0], said.v_exp[1]};
        // not zero: a hidden score is -inf times it
        const float said_up[2] = {said.k_up[0], said.k_up[1]};
        float fs[2] = {fmaxf(f * said_up[0], 1.17549435e-38f),
                       fmaxf(f * said_up[1], 1.17549435e-38f)};
        if (!__all_sync(0xFFFFFFFFu, s_ready) && !KVS_WAIT(&C->s_full[x], half_no & 1)) return;
        tc_fence_after();
        uint32_t v[2][32];
        tmem_ld32_start(S, v[0]);
        tmem_ld32_start(S + 32, v[1]);
        // Asked long before the answers are needed: a wait costs 140 clocks even when it is over
        // (asking saves 30 us of 500 at 2 x 2048 tokens).
        const bool next = i + 1 < p.halves;
        const uint32_t no = step_no + ((i + 1) >> 1);  // of the next half
        const uint32_t ahead =
            peek_phase(&C->pv_done[x][buf], ((half_no >> 1) & 1) ^ 1) &
            ((i & 1) && next ? peek_phase(&C->e_full[no & 3], (no >> 2) & 1) : 1u);
        tmem_arrived(v[0]);
        tmem_arrived(v[1]);
        tc_fence_before();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(&C->s_free[x]);
        // columns of a segment of 32 that this row sees
        auto visible = [&](int sg) {
          const int n = min(seen, p.stop) - t0 - 32 * sg;
          const uint32_t v = n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u;
          return v & ~C->gone[ring][seg0 + sg];
        };
        const bool huge = fmaxf(said_up[0], said_up[1]) > up_most || (flag & kWideK) != 0;
        if (t0 + 64 > plain_to || flag != 0 || huge) {  // hidden scores become -inf
          if (huge) {
#pragma unroll
            for (int sg = 0; sg < 2; ++sg) {
              const float* const up = C->k_tok[ring] + 32 * (seg0 + sg);
              if (C->flags[ring][seg0 + sg] & kWideK) {
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  v[sg][k] = __float_as_uint(__uint_as_float(v[sg][k]) * (f * up[k]));
                fs[sg] = 1.f;
              } else {
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  v[sg][k] = __float_as_uint(__fmul_rn(__uint_as_float(v[sg][k]), fs[sg]));
                fs[sg] = 1.f;
              }
            }
          }
#pragma unroll
          for (int sg = 0; sg < 2; ++sg) {
            const uint32_t vis = visible(sg);
#pragma unroll
            for (int k = 0; k < 32; ++k) v[sg][k] = vis >> k & 1u ? v[sg][k] : 0xFF800000u;
            // values that the row does not see have no say in its units
            if (vis == 0) v_exp[sg] = kLowestExp;
            if (flag) {
#pragma unroll
              for (int gr = 0; gr < NG; ++gr)
                if (C->bad[ring][seg0 + sg][gr] & vis) poison |= 1u << gr;
              if (C->flags[ring][seg0 + sg] & kWideV) {
                float most = 0.f;
#pragma unroll 4
                for (int k = 0; k < 32; ++k)
                  if (vis >> k & 1u) most = fmaxf(most, C->v_tok[ring][32 * (seg0 + sg) + k]);
                v_exp[sg] = max(static_cast<int>(__float_as_uint(most) >> 23) - 127, kLowestExp);
              }
            }
          }
        }
        const bool raise = __any_sync(0xFFFFFFFFu, max(v_exp[0], v_exp[1]) > E);
        // Against the reference that there is, the scores only pass through once; a row
        // whose weights' sum has passed kMostSum, or larger values, make the warp find the maximum,
        // rescale and take the scores again (the first half always does).
        uint32_t h[2][16];
        float sum;
        bool ready = false;
        for (bool fresh = i == 0 || raise;; fresh = true) {
          if (fresh) {
            const int e_new = max(E, max(v_exp[0], v_exp[1]));
            float part[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              part[0] = fmaxf(part[0], __uint_as_float(v[0][k]));
              part[1] = fmaxf(part[1], __uint_as_float(v[1][k]));
            }
            const float mx = fmaxf(part[0] * fs[0], part[1] * fs[1]) - kAbove;
            const float m_new = fmaxf(m, mx), k2 = ex2(m - m_new);
            l *= k2;
            if (i > 0) {
              if (!KVS_WAIT(&C->pv_done[x][buf ^ 1], ((half_no - 1) >> 1) & 1)) return;
              tc_fence_after();
              const float ko = k2 * ex2(static_cast<float>(E - e_new));
#pragma unroll 1
              for (int cg = 0; cg < 4; ++cg) {
                float v[32];
                tmem_ld32(O + 32 * cg, v);
                uint32_t a[16], b[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                  a[k] = __float_as_uint(v[k] * ko);
                  b[k] = __float_as_uint(v[k + 16] * ko);
                }
                tmem_st16(O + 32 * cg, a);
                tmem_st16(O + 32 * cg + 16, b);
              }
            }
            m = m_new;
            E = e_new;
          }
          // Tokens whose V is in units smaller by 2^d than O's weigh less by that, which their sum
          // gets back; more than kFar is nothing beside O.
          const int d[2] = {huge ? 0 : min(E - v_exp[0], kFar),  // lost beside a huge m
                            huge ? 0 : min(E - v_exp[1], kFar)};
          // four sums: one would be a chain as long as the row
          f32x2_t s2[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) s2[k] = f2_pack(0.f, 0.f);
          float refs[2] = {-m, -m};
          if ((d[0] | d[1]) != 0) {
            refs[0] -= static_cast<float>(d[0]);
            refs[1] -= static_cast<float>(d[1]);
          }
#pragma unroll
          for (int sg = 0; sg < 2; ++sg) {
            const f32x2_t fs2 = f2_pack(fs[sg], fs[sg]), ref2 = f2_pack(refs[sg], refs[sg]);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float u0, u1;
              f2_unpack(f2_fma(f2_pack(__uint_as_float(v[sg][2 * k]),
                                       __uint_as_float(v[sg][2 * k + 1])), fs2, ref2), u0, u1);
              const float p0 = ex2(u0), p1 = ex2(u1);
              f32x2_t& part = s2[2 * sg + (k & 1)];
              part = f2_add(part, f2_pack(p0, p1));
              h[sg][k] = half2_bits(p0, p1);
            }
          }
          float s0, s1, s2a, s2b;
          f2_unpack(f2_add(s2[0], s2[1]), s0, s1);
          f2_unpack(f2_add(s2[2], s2[3]), s2a, s2b);
          s0 += s1;
          s2a += s2b;
          if ((d[0] | d[1]) != 0) {
            s0 *= __uint_as_float(static_cast<uint32_t>(127 + d[0]) << 23);
            s2a *= __uint_as_float(static_cast<uint32_t>(127 + d[1]) << 23);
          }
          sum = s0 + s2a;
          if (fresh) break;
          ready = __all_sync(0xFFFFFFFFu, ahead != 0 && !(sum > kMostSum));
          if (ready || !__any_sync(0xFFFFFFFFu, sum > kMostSum)) break;
        }
        l += sum;
        if (!ready) {
          // the products with the weights two halves ago; what is said of the next half
          if (!KVS_WAIT(&C->pv_done[x][buf], ((half_no >> 1) & 1) ^ 1)) return;
          if ((i & 1) && next && !KVS_WAIT(&C->e_full[no & 3], (no >> 2) & 1)) return;
        }
        tc_fence_after();
        if (next) listen(i + 1);
        s_ready = next ? peek_phase(&C->s_full[x], (half_no + 1) & 1) : 0u;
        if (flag & kWideV || huge) {
#pragma unroll
          for (int sg = 0; sg < 2; ++sg) {
            const bool each = flag & kWideV && C->flags[ring][seg0 + sg] & kWideV;
            const int from = huge ? E : v_exp[sg];  // what the exponentials did not do
            const float unit = __uint_as_float(static_cast<uint32_t>(127 - from) << 23),
                        one = ex2(static_cast<float>(v_exp[sg] - from));
            const float* const tok = C->v_tok[ring] + 32 * (seg0 + sg);
#pragma unroll
            for (int k = 0; k < 16; ++k) {  // those that the row does not see weigh nothing
              const __half2 g = __floats2half2_rn(each ? fminf(tok[2 * k] * unit, 1.f) : one,
                                                  each ? fminf(tok[2 * k + 1] * unit, 1.f) : one);
              const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&h[sg][k]), g);
              h[sg][k] = *reinterpret_cast<const uint32_t*>(&y);
            }
          }
        }
        tmem_st16(W, h[0]);
        tmem_st16(W + 16, h[1]);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(&C->p_full[x][half_no & 1]);
      }
      step_no += p.steps;
      for (int back = p.halves > 1 ? 2 : 1; back > 0; --back) {  // both buffers' last products
        const uint32_t no = half_no - back;
        if (!KVS_WAIT(&C->pv_done[x][no & 1], (no >> 1) & 1)) return;
      }
      tc_fence_after();
    }
    // ---- the result, or this part of it
    const float scale_o = p.steps > 0 ? ex2(static_cast<float>(E)) : 0.f;
    const float inv = l == 0.f ? 0.f : __fdividef(scale_o, l);
    const int slot = 2 * static_cast<int>(blockIdx.x) + (p.begins ? 1 : 0);
    uint16_t* const out = static_cast<uint16_t*>(L.out) + tq * L.o_ts + hq * L.o_hs;
    float* const part = P.o + (static_cast<long long>(slot) * kRows + x * 128 + row) * 128;
#pragma unroll
    for (int cg = 0; cg < 4; ++cg) {  // 32 channels: one group or part of one
      float v[32];
      if (p.steps > 0) {
        tmem_ld32(O + 32 * cg, v);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0.f;
      }
      if (poison >> (cg * NG / 4) & 1u) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(0x7FC00000u);
      }
      if (!mine) continue;
      const float k = p.whole ? inv : scale_o;
#pragma unroll
      for (int ch = 0; ch < 4; ++ch) {  // columns hold channels 0, 4, 1, 5, 2, 6, 3, 7 of eight
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[(i >> 1) + 4 * (i & 1)] = v[8 * ch + i] * k;
        if (p.whole) {
          *reinterpret_cast<uint4*>(out + 32 * cg + 8 * ch) = pack8<FP16>(y);
        } else {
          float4* d = reinterpret_cast<float4*>(part + 32 * cg + 8 * ch);
          d[0] = make_float4(y[0], y[1], y[2], y[3]);
          d[1] = make_float4(y[4], y[5], y[6], y[7]);
        }
      }
    }
    if (mine) {
      if (!p.whole)
        P.ml[slot * kRows + x * 128 + row] = make_float2(m, l);
      else if (L.lse != nullptr)
        L.lse[tq * L.q_heads + hq] =
            l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
    }
    if (!p.whole && p.begins && threadIdx.x == 0)
      P.desc[blockIdx.x] = make_int4(p.r, p.h, p.tile, p.parts);
    tc_fence_before();
    __syncwarp();
  }
}

template <bool FP16, int NG>
__global__ void __launch_bounds__(kThreads, 1) k_attn4_tile(const __grid_constant__ Attn4Launch L) {
  extern __shared__ uint8_t raw_smem[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t *const q_tile = smem, *const k_tile = smem + 4 * kHalfTile,
                 *const v_tile = smem + 8 * kHalfTile;
  Ctrl* const C = reinterpret_cast<Ctrl*>(smem + kCtrlAt);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = L.q_heads / L.heads, B = gridDim.x, b = blockIdx.x;
  const Parts P = parts(L.scratch, B, kRows);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    P.desc[b] = make_int4(-1, 0, 0, 0);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&C->q_full[i], 4);
      mbar_init(&C->k_full[i], FP16 ? 2 : 4);
      mbar_init(&C->k_empty[i], 2);
      mbar_init(&C->v_full[i], FP16 ? 2 : 4);
      mbar_init(&C->v_empty[i], 2);
      mbar_init(&C->s_full[i], 1);
      mbar_init(&C->s_free[i], 4);
      for (int k = 0; k < 2; ++k) {
        mbar_init(&C->p_full[i][k], 4);
        mbar_init(&C->pv_done[i][k], 1);
      }
    }
    for (int i = 0; i < 4; ++i) mbar_init(&C->e_full[i], 4);
    fence_mbar_init();
  }
  if (warp == 12) tmem_alloc(&C->tmem, 512);
  tc_fence_before();

  // ---- this CTA's share of the line
  long long total = 0, mine = 0;
  Named named;
  for (int r = tid; r < L.seqs; r += kThreads) {
    const Seq s = sequence(L, r, b == 0);
    named.take(L, s, r);
    mine = tile_work<kOverTile>(L, s, group).head * L.heads;
    total += mine;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
  if (lane == 0) C->scan[warp] = total;
  named.leave(L, C->named);
  __syncthreads();
  named.clear<kThreads / 32>(L, C->named);
  tc_fence_after();
  const uint32_t tmem = C->tmem;
  total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) total += C->scan[w];
  const long long least = static_cast<long long>(kLeastTile) * kTile * group;
  Walk<kOverTile, false> walk;
  walk.U = total;
  walk.b = b;
  walk.used = static_cast<int>(min(static_cast<long long>(B), (total + least - 1) / least));
  if (b < walk.used) {
    walk.pos = walk.share(b);
    walk.end = walk.share(b + 1);
    long long base = 0;
    for (int r0 = 0; r0 < L.seqs; r0 += kThreads) {
      const int r = r0 + tid;
      if (L.seqs > kThreads)  // else `mine` is it
        mine = r < L.seqs ? tile_work<kOverTile>(L, sequence(L, r, false), group).head * L.heads : 0;
      long long inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += y;
      }
      __syncthreads();
      if (lane == 31) C->scan[warp] = inc;
      __syncthreads();
      long long before = base;
      for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) before += C->scan[w];
        base += C->scan[w];
      }
      if (before + inc - mine <= walk.pos && walk.pos < before + inc) {
        C->seq = r;
        C->begin = before + inc - mine;
      }
      if (walk.pos < base) break;  // the same for every thread
    }
    __syncthreads();
    walk.r = C->seq;
    walk.begin = C->begin;
    // 256 x 168 + 128 x 104 + 128 x 72 = the 512 x 128 registers of the launch
    if (warp < 8) {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
      softmax_role<FP16, NG>(L, walk, group, q_tile, tmem, P, C);
    } else if (warp < 12) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
      convert_role<FP16, NG>(L, walk, group, q_tile, k_tile, v_tile, C);
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
      if (warp < 14)
        mma_role<FP16, true>(L, walk, group, warp & 1, smem_u32(q_tile), smem_u32(k_tile), tmem, C);
      else
        mma_role<FP16, false>(L, walk, group, warp & 1, smem_u32(q_tile), smem_u32(v_tile), tmem, C);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(tmem, 512);
}

template <bool FP16, int NG>
cudaError_t launch(const Attn4Launch& L, cudaStream_t s) {
  cudaError_t e = cudaFuncSetAttribute(k_attn4_tile<FP16, NG>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  const int ctas = tile_ctas<kOverTile>(L);
  k_attn4_tile<FP16, NG><<<ctas, kThreads, kSmem, s>>>(L);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  return launch_combine<FP16, kRows / 8, 1>(L, ctas, s);
}

}  // namespace

cudaError_t attn4_tile_launch(const Attn4Launch& L, cudaStream_t s) {
  if (L.fp16)
    return L.groups == 1 ? launch<true, 1>(L, s) : L.groups == 2 ? launch<true, 2>(L, s)
                                                                 : launch<true, 4>(L, s);
  return L.groups == 1 ? launch<false, 1>(L, s) : L.groups == 2 ? launch<false, 2>(L, s)
                                                                : launch<false, 4>(L, s);
}

long long attn4_tile_scratch(const Attn4Launch& L) {
  return 16ll * tile_ctas<kOverTile>(L) + 2ll * tile_ctas<kOverTile>(L) * kRows * (8 + 512);
}

}  // namespace kvs
