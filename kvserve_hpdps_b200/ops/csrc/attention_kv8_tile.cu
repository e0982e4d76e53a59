// Attention over a paged 8-bit cache for many query rows (prefill chunks, prompts' cross attention).
//
// The mathematics is attention_kv8.cu's; here 2 x 128 query rows (several tokens times the query
// heads of one kv head) share each key, so the codes are turned into fp16 tiles once, for tcgen05:
//   S = Q K^T, O += P V, fp16 products of 128 rows and 64 tokens into tensor memory.
// fp16 holds every code exactly, so the tiles lose nothing whatever the scales of their tokens: a
// unit's key scale goes into the softmax's factor, its value scale b = 2^e into the weights,
//   w = 2^(s - M + e - K),  l += 2^(K - e) w,  o = 2^K O / l,
// M near the row's running maximum of s and K such that the largest w was 2^kAbove when it was set.
//
// The one rounding to fewer bits than fp32's is that of the weights to fp16, 2^-11, as the matrix
// instructions' A operand has to be of V's type; their sum is taken before that.  An fp16 output's
// error grows by a third, a bf16 output's does not change; two parts of the weights would need
// half as many products again and tensor memory, of which none is left.
//
// Roles of a CTA (one an SM, 16 warps whose registers are dealt out anew):
//   warps 0-3, 4-7   softmax of query tile 0, 1: a thread a row, which it reads from tensor memory
//                    and writes back as fp16 weights, the A operand of O += P V
//   warps 8-11       codes to fp16 tiles in shared memory, a warp two units, eight lanes a row
//   warps 12-15      issue the matrix instructions: S of tile 0, 1, O of tile 0, 1
// The softmax warps take 64 tokens' scores at a time into registers, so that the next ones are
// computed while they work.  O stays in tensor memory; it is rescaled by the softmax warps when 64
// weights of a row sum up to more than kMostSum, which after the first tiles is rare.
#include "attention_kv8.cuh"
#include "attention_tile.cuh"

namespace kvs {

namespace {

constexpr uint32_t kHides = 1;
// Units whose scale is less than 2^-kFar of K's weigh nothing beside it in fp16, but count in the sum.
constexpr float kFar = 60.f;
// A score is a factor times 128 products of less than 2^15 and 2^9.  Where the factor lets it pass
// 2^27, the product is rounded before the maximum is taken off: the fused multiply-add leaves the
// maximum's own rounding over, up to 2^-25 of it, and weights are 2 to that from where they should
// be (the same for all of a row's, so that 2^4 does no harm).
constexpr float kHuge = 0x1p-4f;

struct Ctrl {
  uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[2], s_free[2], p_full[2][2], pv_done[2][2], e_full[4];  // [tile][buffer]
  uint32_t tmem;
  // What the converting warps say of a step (ring of four):
  float4 k_up[4][2];       // by halves, its four units: the keys' scale
  float4 v_exp[4][2];      // and the exponent of the values'
  uint32_t gone[4][4];     // by 32 tokens: those whose block does not exist
  uint32_t bad[4][4];      // those with a value that is not a number
  uint32_t flags[4][4];    // kHides: any of the two is set
  uint4 poison[kRows];     // channels of a row that are not numbers
  long long scan[kThreads / 32];
  int2 named[kThreads / 32];
  long long begin;
  int seq;
};

constexpr int kCtrlAt = 12 * kHalfTile;
constexpr int kSmem = 1024 + kCtrlAt + static_cast<int>(sizeof(Ctrl));
static_assert(kSmem <= 227 * 1024);

// ------------------------------------------------------------ codes to tiles
// Tiles have two slots of 128 tokens, a step in each in turn.  A warp takes the 32 tokens of its
// segment, four rows at a time: lane 8 i + c the 16 codes of chunk c, which become two chunks of fp16.
KVS_DEV void convert_role(const Attn4Launch& L, Walk walk, int group, uint8_t* k_tile,
                          uint8_t* v_tile, Ctrl* C) {
  const int lane = threadIdx.x & 31, seg = (threadIdx.x >> 5) & 3, sub = lane >> 3, c = lane & 7;
  uint32_t step_no = 0;
  Piece p;
  // of the two fp16 chunks 2 c and 2 c + 1 the one whose place leaves no bank conflict goes first
  const int swap = c >> 2;
  while (walk.next(L, group, p)) {
    const uint8_t* const head = static_cast<const uint8_t*>(L.cache) + p.h * L.head_stride;
    const int32_t* const table = L.table + p.r * L.table_stride;
    const uint8_t* rec[2] = {nullptr, nullptr};  // of a unit's first row; none: not there
    uint32_t scale[2] = {0x7F7Fu, 0x7F7Fu};
    uint32_t gone = 0;
    int left = 0;  // tokens of the segment up to `stop`
    auto locate = [&](int j) {
      const int tok = p.start + j * kTile + 32 * seg;
      left = p.stop - tok;
      gone = 0;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        rec[u] = nullptr;
        scale[u] = 0x7F7Fu;
        if (left <= 16 * u) continue;
        const int page = (tok + 16 * u) / L.block_size;
        const int off = tok + 16 * u - page * L.block_size;
        const int id = table[page];
        if (id < 0 || id >= L.num_blocks) {
          if (lane == 0) record_error(L.err, ERR_BOUNDS);
          gone |= 0xFFFFu << (16 * u);
        } else {
          const uint8_t* const at = head + id * L.block_stride;
          scale[u] = *reinterpret_cast<const uint16_t*>(at + 256ll * L.block_size + (off >> 3));
          rec[u] = at + off * 128;
        }
      }
    };
    uint4 code[2][8];
    auto load_codes = [&](int v) {
      const long long plane = v ? 128ll * L.block_size : 0;
#pragma unroll
      for (int it = 0; it < 8; ++it) {
        const int row = 4 * it + sub;
        code[v][it] = make_uint4(0u, 0u, 0u, 0u);
        if (rec[it >> 2] != nullptr && row < left)
          code[v][it] = *reinterpret_cast<const uint4*>(rec[it >> 2] + plane +
                                                        (row & 15) * 128 + 16 * c);
      }
    };
    if (p.steps > 0) {
      locate(0);
      load_codes(0);
      load_codes(1);
    }
    for (int j = 0; j < p.steps; ++j, ++step_no) {
      // ---- values that are not numbers: zeros in the tile; rows that see them are marked
      uint32_t nan = 0, bad = 0;
#pragma unroll
      for (int it = 0; it < 8; ++it) {
        const uint4& w = code[1][it];
        nan |= (w.x & 0x7F7F7F7Fu) + 0x01010101u;
        nan |= (w.y & 0x7F7F7F7Fu) + 0x01010101u;
        nan |= (w.z & 0x7F7F7F7Fu) + 0x01010101u;
        nan |= (w.w & 0x7F7F7F7Fu) + 0x01010101u;
      }
      if (__any_sync(0xFFFFFFFFu, nan & 0x80808080u)) {
#pragma unroll
        for (int it = 0; it < 8; ++it) {
          uint32_t w[4] = {code[1][it].x, code[1][it].y, code[1][it].z, code[1][it].w}, any = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t is = ((w[i] & 0x7F7F7F7Fu) + 0x01010101u) >> 7 & 0x01010101u;
            any |= is;
            w[i] &= ~(is * 0xFFu);
          }
          code[1][it] = make_uint4(w[0], w[1], w[2], w[3]);
          const uint32_t rows = __ballot_sync(0xFFFFFFFFu, any != 0);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (rows >> (8 * i) & 0xFFu) bad |= 1u << (4 * it + i);
        }
      }
      const int ring = step_no & 3;
      if (lane == 0) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          reinterpret_cast<float*>(C->k_up[ring])[2 * seg + u] =
              __uint_as_float((scale[u] & 0xFFu) << 23);
          reinterpret_cast<float*>(C->v_exp[ring])[2 * seg + u] =
              static_cast<float>(static_cast<int>(scale[u] >> 8) - 127);
        }
        C->gone[ring][seg] = gone;
        C->bad[ring][seg] = bad;
        C->flags[ring][seg] = gone | bad ? kHides : 0u;
        mbar_arrive(&C->e_full[ring]);
      }
      if (j + 1 < p.steps) locate(j + 1);  // its loads go out as registers become free
      const uint32_t slot = step_no & 1, again = (step_no >> 1 & 1) ^ 1;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        uint64_t* const empty = v ? &C->v_empty[slot] : &C->k_empty[slot];
        if (!wait_phase(empty, again, L.err)) return;
        uint8_t* const dst = (v ? v_tile : k_tile) + slot * 2 * kHalfTile;
#pragma unroll
        for (int it = 0; it < 8; ++it) {
          const uint4 w = code[v][it];
          const uint4 lo = make_uint4(half2_low8(w.x), half2_high8(w.x), half2_low8(w.y),
                                      half2_high8(w.y)),
                      hi = make_uint4(half2_low8(w.z), half2_high8(w.z), half2_low8(w.w),
                                      half2_high8(w.w));
          const int row = 32 * seg + 4 * it + sub;
          *reinterpret_cast<uint4*>(dst + chunk_at(row, 2 * c + swap)) = swap ? hi : lo;
          *reinterpret_cast<uint4*>(dst + chunk_at(row, 2 * c + 1 - swap)) = swap ? lo : hi;
        }
        if (j + 1 < p.steps) load_codes(v);
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
template <bool QK>
KVS_DEV void mma_role(const Attn4Launch& L, Walk walk, int group, int x, uint32_t q_tile,
                      uint32_t kv_tile, uint32_t tmem, Ctrl* C) {
  uint32_t step_no = 0, piece_no = 0, half_no = 0;
  Piece p;
  const uint32_t qd = uniform(k_desc(q_tile) + x * (2 * kHalfTile >> 4)),
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
      const uint32_t no = step_no + (i >> 1), slot = no & 1;
      const bool last = (i & 1) || i == H - 1;  // half of the slot
      if (!(i & 1) && !KVS_WAIT(&fulls[slot], (no >> 1) & 1)) return;
      uint64_t* const empty = &empties[slot];
      if (idle) {
        if (last && (threadIdx.x & 31) == 0) mbar_arrive(empty);
        continue;
      }
      const uint32_t b = kvd + slot * (2 * kHalfTile >> 4) + (i & 1) * (8192 >> 4);
      if constexpr (QK) {
        if (i > 0 && !KVS_WAIT(&C->s_free[x], (half_no - 1) & 1)) return;
        tc_fence_after();
        if (elected()) {
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            const uint32_t off = ((ks >> 2) * kHalfTile + (ks & 3) * 32) >> 4;
            mma_qk<kDescHigh>(scores, qd + off, b + off, ks > 0 ? 1u : 0u);
          }
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
            mma_pv(result, weights + 32 * buf + 8 * ks, b + ks * (2048 >> 4),
                   ks > 0 || i > 0 ? 1u : 0u);
          }
          umma_commit(&C->pv_done[x][buf]);
          if (last) umma_commit(empty);
        }
      }
      __syncwarp();
      ++half_no;
    }
    // the last half's scores were taken, too: one phase of s_free a half
    if (QK && !idle && !KVS_WAIT(&C->s_free[x], (half_no - 1) & 1)) return;
    step_no += p.steps;
  }
  // The last products' commits arrive on their own: not after the CTA has gone.
  for (uint32_t back = 1; back < 3 && step_no >= back; ++back) {
    const uint32_t no = step_no - back, slot = no & 1;
    if (!KVS_WAIT(QK ? &C->k_empty[slot] : &C->v_empty[slot], (no >> 1) & 1)) return;
  }
}

// ------------------------------------------------------------------ softmax
template <bool FP16>
KVS_DEV void softmax_role(const Attn4Launch& L, Walk walk, int group, uint8_t* q_tile,
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
    const int seen = mine ? seen_by(L, p.s, rr / group) : 0;
    float m = kLowest, l = 0.f, f = 0.f, K = -120.f;
    bool poisoned = false;
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
      e = top == 0.f ? 0 : max(kLowestExp, min(e, 100));
      const float up = pow2(14 - e) * (L.scale < 0.f ? -1.f : 1.f);
      f = fabsf(L.scale) * 1.4426950408889634f * pow2(e - 14);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float y[8];
        unpack8<FP16>(raw[i], y);
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] *= up;
        *reinterpret_cast<uint4*>(qt + chunk_at(row, i)) =
            make_uint4(half2_bits(y[0], y[1]), half2_bits(y[2], y[3]), half2_bits(y[4], y[5]),
                       half2_bits(y[6], y[7]));
      }
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
        float4 v_exp, k_up;
      } said;
      auto listen = [&](int i) {
        const uint32_t ring = (step_no + (i >> 1)) & 3, half = i & 1;
        said.flag = C->flags[ring][2 * half] | C->flags[ring][2 * half + 1];
        said.v_exp = C->v_exp[ring][half];
        said.k_up = C->k_up[ring][half];
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
        const float ev[4] = {said.v_exp.x, said.v_exp.y, said.v_exp.z, said.v_exp.w};
        const float up4[4] = {said.k_up.x, said.k_up.y, said.k_up.z, said.k_up.w};
        float fs[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)  // not zero: a hidden score is -inf times it
          fs[u] = fmaxf(f * up4[u], 1.17549435e-38f);
        if (!__all_sync(0xFFFFFFFFu, s_ready) && !KVS_WAIT(&C->s_full[x], half_no & 1)) return;
        tc_fence_after();
        uint32_t v[2][32];
        tmem_ld32_start(S, v[0]);
        tmem_ld32_start(S + 32, v[1]);
        // Asked long before the answers are needed: a wait costs 140 clocks even when it is over.
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
        const bool huge = fmaxf(fmaxf(up4[0], up4[1]), fmaxf(up4[2], up4[3])) > up_most;
        if (t0 + 64 > plain_to || flag != 0 || huge) {  // hidden scores become -inf
          if (huge) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                uint32_t& y = v[u >> 1][16 * (u & 1) + k];
                y = __float_as_uint(__fmul_rn(__uint_as_float(y), fs[u]));
              }
              fs[u] = 1.f;
            }
          }
#pragma unroll
          for (int sg = 0; sg < 2; ++sg) {
            const int n = min(seen, p.stop) - t0 - 32 * sg;
            uint32_t vis = n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u;
            vis &= ~C->gone[ring][seg0 + sg];
#pragma unroll
            for (int k = 0; k < 32; ++k) v[sg][k] = vis >> k & 1u ? v[sg][k] : 0xFF800000u;
            if (flag) {
              for (uint32_t b = C->bad[ring][seg0 + sg] & vis; b != 0; b &= b - 1) {
                // the row sees a token with values that are not numbers: which, from its codes
                const int tok = t0 + 32 * sg + __ffs(b) - 1, page = tok / L.block_size;
                const uint4* const codes = reinterpret_cast<const uint4*>(
                    static_cast<const uint8_t*>(L.cache) +
                    L.table[p.r * L.table_stride + page] * L.block_stride + p.h * L.head_stride +
                    (L.block_size + tok - page * L.block_size) * 128ll);
                uint32_t* const to = reinterpret_cast<uint32_t*>(&C->poison[x * 128 + row]);
#pragma unroll 1
                for (int w = 0; w < 4; ++w) {
                  uint32_t bits = poisoned ? to[w] : 0u;
#pragma unroll 1
                  for (int k = 0; k < 8; ++k) {
                    const uint32_t four = reinterpret_cast<const uint32_t*>(codes)[8 * w + k];
                    const uint32_t is = ((four & 0x7F7F7F7Fu) + 0x01010101u) >> 7 & 0x01010101u;
                    bits |= ((is * 0x01020408u) >> 24 & 15u) << (4 * k);
                  }
                  to[w] = bits;
                }
                poisoned = true;
              }
            }
          }
        }
        // Against the reference that there is, the scores only pass through once; a row whose
        // weights' sum has passed kMostSum makes the warp find the maximum, rescale and take the
        // scores again (the first half always does).
        uint32_t h[2][16];
        float sum;
        bool ready = false;
        for (bool fresh = i == 0;; fresh = true) {
          if (fresh) {
            float part[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              part[u] = -INFINITY;
#pragma unroll
              for (int k = 0; k < 16; ++k)
                part[u] = fmaxf(part[u], __uint_as_float(v[u >> 1][16 * (u & 1) + k]));
              part[u] *= fs[u];
            }
            const float m_new =
                fmaxf(m, fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
            const float less = m - m_new;
            float most = part[0] - m_new + ev[0];
#pragma unroll
            for (int u = 1; u < 4; ++u) most = fmaxf(most, part[u] - m_new + ev[u]);
            const float k_new =
                fmaxf(fmaxf(floorf(K + less), -120.f), ceilf(most) - kAbove);
            l *= ex2(less);
            if (i > 0) {
              if (!KVS_WAIT(&C->pv_done[x][buf ^ 1], ((half_no - 1) >> 1) & 1)) return;
              tc_fence_after();
              const float ko = ex2(less + (K - k_new));
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
            K = k_new;
          }
          f32x2_t s2[4];
          float d[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            d[u] = fmaxf(ev[u] - K, -kFar);
            s2[u] = f2_pack(0.f, 0.f);
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float ref = d[u] - m;
            const f32x2_t fs2 = f2_pack(fs[u], fs[u]), ref2 = f2_pack(ref, ref);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int at = 16 * (u & 1) + 2 * k;
              float u0, u1;
              f2_unpack(f2_fma(f2_pack(__uint_as_float(v[u >> 1][at]),
                                       __uint_as_float(v[u >> 1][at + 1])), fs2, ref2), u0, u1);
              const float p0 = ex2(u0), p1 = ex2(u1);
              s2[u] = f2_add(s2[u], f2_pack(p0, p1));
              h[u >> 1][8 * (u & 1) + k] = half2_bits(p0, p1);
            }
          }
          float all = 0.f;
          sum = 0.f;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            float s0, s1;
            f2_unpack(s2[u], s0, s1);
            s0 += s1;
            all += s0;
            sum = fmaf(s0, ex2(-d[u]), sum);
          }
          if (fresh) break;
          ready = __all_sync(0xFFFFFFFFu, ahead != 0 && !(all > kMostSum));
          if (ready || !__any_sync(0xFFFFFFFFu, all > kMostSum)) break;
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
    const float unit = p.steps > 0 ? pow2(static_cast<int>(K)) : 0.f;
    const float inv = l == 0.f ? 0.f : __fdividef(1.f, l);
    const int slot = 2 * static_cast<int>(blockIdx.x) + (p.begins ? 1 : 0);
    uint16_t* const out = static_cast<uint16_t*>(L.out) + tq * L.o_ts + hq * L.o_hs;
    float* const part = P.o + (static_cast<long long>(slot) * kRows + x * 128 + row) * 128;
#pragma unroll
    for (int cg = 0; cg < 4; ++cg) {
      float v[32];
      if (p.steps > 0) {
        tmem_ld32(O + 32 * cg, v);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0.f;
      }
      if (poisoned) {
        const uint32_t bits = reinterpret_cast<const uint32_t*>(&C->poison[x * 128 + row])[cg];
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (bits >> i & 1u) v[i] = __uint_as_float(0x7FC00000u);
      }
      if (!mine) continue;
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] *= unit;
      if (p.whole) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] *= inv;
      }
#pragma unroll
      for (int ch = 0; ch < 4; ++ch) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = v[8 * ch + i];
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

template <bool FP16>
__global__ void __launch_bounds__(kThreads, 1) k_attn8_tile(const __grid_constant__ Attn4Launch L) {
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
      mbar_init(&C->k_full[i], 4);
      mbar_init(&C->k_empty[i], 2);
      mbar_init(&C->v_full[i], 4);
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
    mine = tile_work(L, s, group).head * L.heads;
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
  Walk walk;
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
        mine = r < L.seqs ? tile_work(L, sequence(L, r, false), group).head * L.heads : 0;
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
      softmax_role<FP16>(L, walk, group, q_tile, tmem, P, C);
    } else if (warp < 12) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
      convert_role(L, walk, group, k_tile, v_tile, C);
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
      if (warp < 14)
        mma_role<true>(L, walk, group, warp & 1, smem_u32(q_tile), smem_u32(k_tile), tmem, C);
      else
        mma_role<false>(L, walk, group, warp & 1, smem_u32(q_tile), smem_u32(v_tile), tmem, C);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(tmem, 512);
}

template <bool FP16>
cudaError_t launch(const Attn4Launch& L, cudaStream_t s) {
  cudaError_t e = cudaFuncSetAttribute(k_attn8_tile<FP16>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  const int ctas = tile_ctas(L);
  k_attn8_tile<FP16><<<ctas, kThreads, kSmem, s>>>(L);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  return launch_combine<FP16, kRows / 8, 1>(L, ctas, s);
}

}  // namespace

cudaError_t attn8_tile_launch(const Attn4Launch& L, cudaStream_t s) {
  return L.fp16 ? launch<true>(L, s) : launch<false>(L, s);
}

long long attn8_tile_scratch(const Attn4Launch& L) {
  return 16ll * tile_ctas(L) + 2ll * tile_ctas(L) * kRows * (8 + 512);
}

}  // namespace kvs
