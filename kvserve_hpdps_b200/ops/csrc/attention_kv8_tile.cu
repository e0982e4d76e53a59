// Attention over a paged 8-bit cache for many query rows (prefill chunks, prompts' cross attention).
//
// The mathematics is attention_kv8.cu's; here 2 x 128 query rows (several tokens times the query
// heads of one kv head) share each key, on tcgen05:
//   S = Q K^T, O += P V, products of 128 rows and 64 tokens into tensor memory.
// K's codes are matrix operands as they are (kind::f8f6f4, fp32 sums: measured off by at most 2^-21.9 of
// the sum of magnitudes).  A query row, scaled by a power of two to at most 448, is taken in 8-bit
// parts that add up to it: one in e4m3 (4 bits) and one for bf16, two for fp16, in e5m2 (3 bits and a
// sign each, down to 2^-16).  That is exact for elements down to 2^-6, which is less than 2^-13 of the
// row's largest; those below are off by at most 2^-14 (bf16) and 2^-17 (fp16), 2^-21 and 2^-24 of it.  A
// channel that a bias has made 1000 times the others leaves these as good as exact (parts in e4m3
// alone end at 2^-10: the logarithms of the sums were off by 1e-2 then).
// V's codes become fp16 tiles, which hold every code exactly.  The scales stay out of the products: a
// unit's key scale goes into the softmax's factor, its value scale b = 2^e into the weights,
//   w = 2^(s - M + e - K),  l += 2^(K - e) w,  o = 2^K O / l,
// M a whole number near the row's running maximum of s, K such that the largest w was about 2^kAbove
// when it was set.
//
// The other rounding to fewer bits than fp32's is that of the weights to fp16, 2^-11, as the matrix
// instructions' A operand has to be of V's type; their sum is taken before that.  An fp16 output's
// error grows by a third, a bf16 output's does not change; two parts of the weights would need
// half as many products again and tensor memory, of which none is left.
//
// Roles of a CTA (one an SM, 16 warps whose registers are dealt out anew):
//   warps 0-3, 4-7   softmax of query tile 0, 1: a thread a row, which it reads from tensor memory
//                    and writes back as fp16 weights, the A operand of O += P V
//   warps 8-11       turn the values' codes into fp16 tiles in shared memory, a warp a unit of each half
//   warps 12, 13, 14 issue the matrix instructions: S of tile 0, 1, O of both
//   warp 15          deals out the pieces of the CTA's share and asks the copy engine for codes, ahead
// All go by halves of 64 tokens.  The softmax warps take a half's scores into registers, so that the
// next ones are computed while they work.  O stays in tensor memory; it is rescaled by the softmax
// warps when 64 weights of a row sum up to more than kMostSum, which after the first tiles is rare.
//
// What bounds it: the softmax warps' chain, 2300 clocks for 64 tokens of both tiles, of which the
// exponentials' rate (16 a clock and SM) is 1024 and the products take 1050 (fp16: 1320).
// 2048 tokens over 8193 and 1366 over 6144, 28/4 heads (317 GFLOP), in a captured graph: bf16 375 us
// (846 TFLOP/s), fp16 398; 6 prompts of 389 and 260 tokens over up to 1501, 16 heads: 72 us (fp16 77), a
// third of it what pieces cost beside their steps.  With K as fp16 tiles it was 633 us and 107.
//
// The work is dealt out as in attention_kv8.cu, here by the number of visible keys a tile has.
#include "attention_kv8.cuh"
#include "attention_tile.cuh"

namespace kvs {

namespace {

// Units whose scale is less than 2^-kFar of K's weigh nothing beside it in fp16, but count in the sum.
// Their weights, of 2^-kFar as it were, have to stay below fp16's 2^-25: a row's maximum moves on when
// the sum of 64 passes 2^20 without their units, too (times kSumBefore that is kMostSum).
constexpr float kFar = 60.f;
constexpr float kSumBefore = kMostSum * 0x1p-20f;
// Equal scores have to weigh alike whatever their values' scales are.  The reference is a whole
// number, so that it and a unit's exponent add up without a rounding below 2^24, and one fused
// multiply-add takes a score against both.  A score is a factor times 128 products of at most
// 448^2: where the factor lets it pass 2^22.7, every half is taken against its own maximum first
// (the score rounded before, if that is above 2^23: what the maximum's rounding leaves over would
// be an exponent of its own), and the units' exponents are added to the differences.
constexpr float kHuge = 0x1p-2f;

// An item's own cost in steps of 128 tokens: the share is what a CTA's pieces take, 18000 clocks each
// and 4600 a step (2048 and 1366 tokens: 379 us with 2, 374.6 with 3, 373 with 4, 374 with 6; 6 prompts
// 72.6, 71.4, 71.6, 71.8).
constexpr int kOverTile = 3;
constexpr int kHalf = 64;                  // tokens
constexpr int kCodes = kHalf * 128;        // bytes of a half's key or value codes
constexpr int kValues = 2 * kHalf * 128;   // of its values as fp16
constexpr int kPart = 128 * 128;           // of a part of a query tile
constexpr int kNotes = 16;                 // halves that something is known of
constexpr int kPieces = 4;                 // pieces that are dealt out ahead
constexpr int kReaders = 15;               // warps that take them

// RING halves' key codes and value codes are there or on their way, four halves' values as fp16.
template <bool FP16>
struct Room {
  static constexpr int PARTS = FP16 ? 3 : 2, RING = FP16 ? 3 : 4;
};
constexpr int kTiles = 4;

struct Ctrl {
  uint64_t q_full[2], k_full[4], k_empty[4], v_came[4], v_taken[4], v_full[kTiles], v_empty[kTiles];
  uint64_t s_full[2], s_free[2], p_full[2][2], pv_done[2][2], done[2];
  uint64_t piece_full[kPieces], piece_empty[kPieces];
  Piece piece[kPieces];
  uint32_t tmem;
  uint32_t any_bad;         // some half of this CTA had values that are not numbers
  // What is known of a half, by units:
  float4 k_up[kNotes];      // the keys' scale
  float4 v_exp[kNotes];     // the exponent of the values'
  uint32_t gone[kNotes];    // a byte a unit: 1 if its block does not exist
  uint16_t bad[kNotes][4];  // tokens with a value that is not a number
  uint4 poison[kRows];      // channels of a row that are not numbers
  long long scan[kThreads / 32];
  int2 named[kThreads / 32];
  long long begin;
  int seq;
};

template <bool FP16>
struct Layout {
  static constexpr int keys = 2 * Room<FP16>::PARTS * kPart, codes = keys + Room<FP16>::RING * kCodes,
                       values = codes + Room<FP16>::RING * kCodes, ctrl = values + kTiles * kValues,
                       bytes = 1024 + ctrl + static_cast<int>(sizeof(Ctrl));
  static_assert(bytes <= 227 * 1024);
};

// A slot of a ring and the phase of its barriers.
template <int N>
struct Turn {
  uint32_t slot = 0, phase = 0;
  KVS_DEV void next() {
    if (++slot == N) {
      slot = 0;
      phase ^= 1;
    }
  }
};

// [rows][128 bytes], 16-byte chunks swizzled by the row.
KVS_DEV uint32_t at128(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

// Bytes of a word that are not numbers: 1 in each.
KVS_DEV uint32_t not_numbers(uint32_t w) {
  return ((w & 0x7F7F7F7Fu) + 0x01010101u) >> 7 & 0x01010101u;
}

// ---------------------------------------------------------- pieces and codes
// The next piece, as the fetching warp left it; false behind the last one.
KVS_DEV bool take_piece(const Attn4Launch& L, Ctrl* C, Turn<kPieces>& at, Piece& p) {
  if (!wait_phase(&C->piece_full[at.slot], at.phase, L.err)) return false;
  p = C->piece[at.slot];
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(&C->piece_empty[at.slot]);
  at.next();
  return p.r >= 0;
}

// One warp walks through the CTA's share, ahead of all others, and asks the copy engine for codes.
template <bool FP16>
KVS_DEV void fetch_role(const Attn4Launch& L, const CUtensorMap* map, Walk<kOverTile, true> walk, int group,
                        uint32_t smem, Ctrl* C) {
  constexpr int RING = Room<FP16>::RING;
  const int lane = threadIdx.x & 31;
  Turn<RING> asks;
  Turn<kPieces> to;
  uint32_t asked = 0, told = 0;
  for (bool more = true; more;) {
    Piece p;
    more = walk.next(L, group, p);
    if (told >= kPieces && !wait_phase(&C->piece_empty[to.slot], to.phase ^ 1, L.err)) return;
    if (elected()) {
      if (!more) p.r = -1;
      C->piece[to.slot] = p;
      mbar_arrive(&C->piece_full[to.slot]);
    }
    __syncwarp();
    to.next();
    ++told;
    if (!more) return;
    const uint8_t* const head = static_cast<const uint8_t*>(L.cache) + p.h * L.head_stride;
    const int32_t* const table = L.table + p.r * L.table_stride;
    // Blocks, places and scales of 8 halves' units, a lane each; and of the next 8's.
    int id = -1, off = 0, id2 = -1, off2 = 0;
    uint32_t scale = 0x7F7Fu, scale2 = 0x7F7Fu;
    auto look = [&](int i, int& id, int& off) {  // from half i on
      const int tok = p.start + i * kHalf + kUnit8 * lane;
      id = -1;
      if (tok < p.stop) {
        const int page = tok / L.block_size;
        off = tok - page * L.block_size;
        id = table[page];
        if (id < 0 || id >= L.num_blocks) {
          record_error(L.err, ERR_BOUNDS);
          id = -2;
        }
      }
    };
    auto look_scale = [&](int id, int off, uint32_t& scale) {
      scale = 0x7F7Fu;
      if (id >= 0)
        scale = *reinterpret_cast<const uint16_t*>(head + id * L.block_stride +
                                                   256ll * L.block_size + (off >> 3));
    };
    for (int i = 0; i < p.halves; ++i, ++asked) {
      const int at = i & 7;
      if (i == 0) {
        look(0, id, off);
        look_scale(id, off, scale);
      } else if (at == 0) {
        id = id2;
        off = off2;
        scale = scale2;
      } else if (at == 2) {
        look(i + 6, id2, off2);
      } else if (at == 5) {
        look_scale(id2, off2, scale2);
      }
      if (asked >= RING && (!wait_phase(&C->k_empty[asks.slot], asks.phase ^ 1, L.err) ||
                            !wait_phase(&C->v_taken[asks.slot], asks.phase ^ 1, L.err)))
        return;
      uint64_t *const k_bar = &C->k_full[asks.slot], *const v_bar = &C->v_came[asks.slot];
      int block[4], place[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        block[u] = __shfl_sync(0xFFFFFFFFu, id, 4 * at + u);
        place[u] = __shfl_sync(0xFFFFFFFFu, off, 4 * at + u);
      }
      if (elected()) {  // one lane: copies by several are issued one after the other anyway
        const uint32_t bytes = kUnit8 * 128 * ((block[0] >= 0) + (block[1] >= 0) +
                                               (block[2] >= 0) + (block[3] >= 0));
        mbar_expect_tx(k_bar, bytes);
        mbar_expect_tx(v_bar, bytes);
        const uint32_t dst = smem + asks.slot * kCodes;
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (block[u] >= 0)
            load_rows(dst + Layout<FP16>::keys + u * (kUnit8 * 128), map, place[u], p.h, block[u],
                      k_bar);
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (block[u] >= 0)
            load_rows(dst + Layout<FP16>::codes + u * (kUnit8 * 128), map, L.block_size + place[u],
                      p.h, block[u], v_bar);
      }
      __syncwarp();
      // the scales, which a piece's first copies need not wait for
      const int mine = __shfl_sync(0xFFFFFFFFu, id, 4 * at + (lane & 3));
      const uint32_t sc = __shfl_sync(0xFFFFFFFFu, scale, 4 * at + (lane & 3));
      const uint32_t note = asked % kNotes;
      if (lane < 4) {
        reinterpret_cast<float*>(&C->k_up[note])[lane] = __uint_as_float((sc & 0xFFu) << 23);
        reinterpret_cast<float*>(&C->v_exp[note])[lane] =
            static_cast<float>(static_cast<int>(sc >> 8) - 127);
        reinterpret_cast<uint8_t*>(&C->gone[note])[lane] = mine == -2 ? 1 : 0;
        C->bad[note][lane] = 0;
      }
      __syncwarp();
      if (elected()) {
        mbar_arrive(k_bar);
        mbar_arrive(v_bar);
      }
      __syncwarp();
      asks.next();
    }
  }
}

// Values' codes to fp16 tiles, a warp a unit of each half.
template <bool FP16>
KVS_DEV void convert_role(const Attn4Launch& L, uint8_t* smem, Ctrl* C) {
  constexpr int RING = Room<FP16>::RING;
  const int lane = threadIdx.x & 31, unit = (threadIdx.x >> 5) & 3, sub = lane >> 3, c = lane & 7;
  Turn<RING> comes;
  Turn<kTiles> fills;
  Turn<kPieces> pieces;
  uint32_t half_no = 0;
  Piece p;
  // of the two fp16 chunks 2 c and 2 c + 1 the one whose place leaves no bank conflict goes first
  const bool swap = c >= 4;
  while (take_piece(L, C, pieces, p)) {
    for (int i = 0; i < p.halves; ++i, ++half_no) {
      if (!wait_phase(&C->v_came[comes.slot], comes.phase, L.err)) return;
      // rows of the unit that are there
      const int left = C->gone[half_no % kNotes] >> (8 * unit) & 1u
                           ? 0
                           : p.stop - (p.start + i * kHalf + kUnit8 * unit);
      uint4 w[4];
      uint32_t nan = 0;
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        const int row = 4 * it + sub;
        w[it] = make_uint4(0u, 0u, 0u, 0u);
        if (row < left)
          w[it] = *reinterpret_cast<const uint4*>(smem + Layout<FP16>::codes + comes.slot * kCodes +
                                                  at128(kUnit8 * unit + row, c));
        nan |= (w[it].x & 0x7F7F7F7Fu) + 0x01010101u;
        nan |= (w[it].y & 0x7F7F7F7Fu) + 0x01010101u;
        nan |= (w[it].z & 0x7F7F7F7Fu) + 0x01010101u;
        nan |= (w[it].w & 0x7F7F7F7Fu) + 0x01010101u;
      }
      if (__any_sync(0xFFFFFFFFu, nan & 0x80808080u)) {
        // values that are not numbers: zeros in the tile; rows that see them are marked
        uint32_t bad = 0;
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          uint32_t y[4] = {w[it].x, w[it].y, w[it].z, w[it].w}, any = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t is = not_numbers(y[k]);
            any |= is;
            y[k] &= ~(is * 0xFFu);
          }
          w[it] = make_uint4(y[0], y[1], y[2], y[3]);
          const uint32_t rows = __ballot_sync(0xFFFFFFFFu, any != 0);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (rows >> (8 * k) & 0xFFu) bad |= 1u << (4 * it + k);
        }
        if (lane == 0) {
          C->bad[half_no % kNotes][unit] = static_cast<uint16_t>(bad);
          C->any_bad = 1;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&C->v_taken[comes.slot]);
      comes.next();
      if (half_no >= kTiles && !wait_phase(&C->v_empty[fills.slot], fills.phase ^ 1, L.err)) return;
      uint8_t* const dst = smem + Layout<FP16>::values + fills.slot * kValues;
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        const uint32_t a0 = swap ? w[it].z : w[it].x, a1 = swap ? w[it].w : w[it].y,
                       b0 = swap ? w[it].x : w[it].z, b1 = swap ? w[it].y : w[it].w;
        // channels 64 (c / 4) + ...: two blocks of 64 channels, rows of 128 bytes
        uint8_t* const block = dst + (c >> 2) * (kHalf * 128);
        const int row = kUnit8 * unit + 4 * it + sub, chunk = 2 * (c & 3);
        *reinterpret_cast<uint4*>(block + at128(row, chunk + swap)) =
            make_uint4(half2_low8(a0), half2_high8(a0), half2_low8(a1), half2_high8(a1));
        *reinterpret_cast<uint4*>(block + at128(row, chunk + 1 - swap)) =
            make_uint4(half2_low8(b0), half2_high8(b0), half2_low8(b1), half2_high8(b1));
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&C->v_full[fills.slot]);
      fills.next();
    }
  }
}

// ------------------------------------------------------ matrix instructions
// A: a part of the queries, e4m3 (number 0, which is also fp16's) or e5m2 (number 1).
template <bool E5M2>
KVS_DEV void mma_codes(uint32_t d, uint32_t a, uint32_t b, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\t"
      "mov.b64 x, {%1, %4};\n\tmov.b64 y, {%2, %4};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], x, y, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(kIdescQK | (E5M2 ? 1u << 7 : 0u)), "n"(kDescHigh), "r"(accumulate)
      : "memory");
}
// Values: 64 channels a block, blocks 8 KB apart (leading offset).
KVS_DEV uint32_t values_desc(uint32_t saddr) {
  return (saddr >> 4) | (static_cast<uint32_t>(kHalf * 128 >> 4) << 16);
}

// Three warps issue them, on schedulers of their own: the scores of query tile 0, of tile 1, and both
// tiles' output.
//
// Scores of half i + 1 are asked for as soon as the softmax warps have those of half i in their
// registers, so they find them ready when they are through; the weights have two buffers of
// their own, and their products time to wait for the other tile's.  A slot is free when both tiles'
// products with it are done; without a second tile its warp only says so.
//
// The last products' commits arrive on their own: not after the CTA has gone.
template <int N>
KVS_DEV void last_commits(const Attn4Launch& L, uint64_t* empties, Turn<N> turn, uint32_t all) {
  for (int back = 0; back < N && all > 0; ++back, --all) {
    turn.slot = turn.slot == 0 ? N - 1 : turn.slot - 1;
    if (turn.slot == N - 1) turn.phase ^= 1;
    if (!KVS_WAIT(&empties[turn.slot], turn.phase)) return;
  }
}

template <bool FP16>
KVS_DEV void qk_role(const Attn4Launch& L, int x, uint32_t smem, uint32_t tmem, Ctrl* C) {
  constexpr int PARTS = Room<FP16>::PARTS, RING = Room<FP16>::RING;
  uint32_t piece_no = 0, half_no = 0, all = 0;
  Turn<RING> turn;
  Turn<kPieces> pieces;
  Piece p;
  const uint32_t qd = uniform(k_desc(smem + x * PARTS * kPart)),
                 kd = uniform(k_desc(smem + Layout<FP16>::keys)), scores = uniform(tmem + 64 * x);
  while (take_piece(L, C, pieces, p)) {
    const int H = static_cast<int>(uniform(p.halves));
    if (H == 0) continue;
    const bool idle = x == 1 && !p.two;
    if (!idle && !KVS_WAIT(&C->q_full[x], piece_no++ & 1)) return;
    for (int i = 0; i < H; ++i, ++all) {
      if (!KVS_WAIT(&C->k_full[turn.slot], turn.phase)) return;
      uint64_t* const empty = &C->k_empty[turn.slot];
      const uint32_t b = kd + turn.slot * (kCodes >> 4);
      turn.next();
      if (idle) {
        if ((threadIdx.x & 31) == 0) mbar_arrive(empty);
        continue;
      }
      if (i > 0 && !KVS_WAIT(&C->s_free[x], (half_no - 1) & 1)) return;
      tc_fence_after();
      if (elected()) {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          mma_codes<false>(scores, qd + (ks * 32 >> 4), b + (ks * 32 >> 4), ks > 0 ? 1u : 0u);
#pragma unroll
        for (int part = 1; part < PARTS; ++part)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            mma_codes<true>(scores, qd + ((part * kPart + ks * 32) >> 4), b + (ks * 32 >> 4), 1u);
        umma_commit(&C->s_full[x]);
        umma_commit(empty);
      }
      __syncwarp();
      ++half_no;
    }
    // The last half's scores were taken, too: one phase of s_free a half.  And not on to pieces without
    // this tile, which free slots as they come, before its softmax has read what is known of this one's.
    if (!idle && (!KVS_WAIT(&C->s_free[x], (half_no - 1) & 1) ||
                  !KVS_WAIT(&C->done[x], (piece_no - 1) & 1)))
      return;
  }
  last_commits(L, C->k_empty, turn, all);
}

template <bool FP16>
KVS_DEV void pv_role(const Attn4Launch& L, uint32_t smem, uint32_t tmem, Ctrl* C) {
  uint32_t halves_of[2] = {0, 0}, all = 0;  // of a tile, so far
  Turn<kTiles> turn;
  Turn<kPieces> pieces;
  Piece p;
  const uint32_t vd = uniform(values_desc(smem + Layout<FP16>::values)),
                 weights = uniform(tmem + kWeightsAt), result = uniform(tmem + kOutAt);
  while (take_piece(L, C, pieces, p)) {
    const int H = static_cast<int>(uniform(p.halves));
    const bool two = uniform(p.two) != 0;
    for (int i = 0; i < H; ++i, ++all) {
      if (!KVS_WAIT(&C->v_full[turn.slot], turn.phase)) return;
      const uint32_t b = vd + turn.slot * (kValues >> 4);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (x == 1 && !two) continue;
        const uint32_t buf = halves_of[x] & 1;
        if (!KVS_WAIT(&C->p_full[x][buf], (halves_of[x] >> 1) & 1)) return;
        tc_fence_after();
        if (elected()) {
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)  // 16 tokens: two groups of eight rows, 8 columns of P
            mma_pv(result + 128 * x, weights + 64 * x + 32 * buf + 8 * ks, b + ks * (2048 >> 4),
                   ks > 0 || i > 0 ? 1u : 0u);
          umma_commit(&C->pv_done[x][buf]);
          if (x == 1 || !two) umma_commit(&C->v_empty[turn.slot]);
        }
        __syncwarp();
        ++halves_of[x];
      }
      turn.next();
    }
  }
  last_commits(L, C->v_empty, turn, all);
}

// ------------------------------------------------------------------ softmax
// A pointer that another lane has.
KVS_DEV const uint8_t* of_lane(const uint8_t* p, int lane) {
  return reinterpret_cast<const uint8_t*>(
      __shfl_sync(0xFFFFFFFFu, reinterpret_cast<unsigned long long>(p), lane));
}

template <bool FP16>
KVS_DEV void softmax_role(const Attn4Launch& L, int group, uint8_t* smem, uint32_t tmem,
                          const Parts& P, Ctrl* C) {
  const int x = threadIdx.x >> 7, row = threadIdx.x & 127;
  const uint32_t lanes = static_cast<uint32_t>((threadIdx.x >> 5) & 3) << 21;  // a warp's 32
  const uint32_t S = tmem + 64 * x + lanes, O = tmem + kOutAt + 128 * x + lanes;
  constexpr int PARTS = Room<FP16>::PARTS;
  uint8_t* const qt = smem + x * PARTS * kPart;
  // Two places of 32 rows of 128 bytes, 16 KB apart: the warp's own queries', where rows and results
  // change from a thread a row to whole lines.
  const int lane = threadIdx.x & 31;
  uint8_t* const area = qt + (row - lane) * 128;
  uint32_t notes = 0, half_no = 0;  // halves before this piece; this tile's
  Turn<kPieces> pieces;
  Piece p;
  while (take_piece(L, C, pieces, p)) {
    if (x == 1 && !p.two) {
      notes += p.halves;
      continue;
    }
    const int rr = p.tile * kRows + x * 128 + row;
    const bool mine = rr < p.nrows;
    const uint32_t has = __ballot_sync(0xFFFFFFFFu, mine);
    const long long tq = p.s.row0 + rr / group;
    const int hq = p.h * group + rr % group;
    const int seen = mine ? seen_by(L, p.s, rr / group) : 0;
    float m = kLowest, l = 0.f, f = 0.f, K = -120.f;
    bool poisoned = false;
    if (p.steps > 0) {
      // ---- the row scaled by a power of two, its largest element in (224, 448], in parts
      uint4 raw[16];
      // a row that is not there is read from the first one: with a load each behind a condition of
      // its own the 16 came one after the other (11000 clocks a piece against 3800)
      const uint8_t* const src = reinterpret_cast<const uint8_t*>(
          static_cast<const uint16_t*>(L.q) + (mine ? tq * L.q_ts + hq * L.q_hs : 0));
#pragma unroll
      for (int i = 0; i < 16; ++i) {  // half a warp a row: whole lines, where a thread's own row is 16
        const int r = 2 * i + (lane >> 4);
        const uint8_t* const from = of_lane(src, r);
        raw[i] = *reinterpret_cast<const uint4*>(from + 16 * (lane & 15));
        if (!(has >> r & 1u)) raw[i] = make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        *reinterpret_cast<uint4*>(area + (lane >> 3 & 1) * kPart +
                                  at128(2 * i + (lane >> 4), lane & 7)) = raw[i];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 16; ++i)
        raw[i] = *reinterpret_cast<const uint4*>(area + (i >> 3) * kPart + at128(lane, i & 7));
      __syncwarp();  // the parts take their place
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float y[8];
        unpack8<FP16>(raw[i], y);
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(y[k]));
      }
      const int e = min(scale_exponent(__float_as_uint(top)), 120);
      // an infinite element makes the row what is not a number
      const float up = top < INFINITY ? pow2(-e) * (L.scale < 0.f ? -1.f : 1.f)
                                      : __uint_as_float(0x7FC00000u);
      f = fabsf(L.scale) * 1.4426950408889634f * pow2(e);
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // 16 channels
        float y[16];
        unpack8<FP16>(raw[2 * i], *reinterpret_cast<float(*)[8]>(y));
        unpack8<FP16>(raw[2 * i + 1], *reinterpret_cast<float(*)[8]>(y + 8));
#pragma unroll
        for (int k = 0; k < 16; ++k) y[k] *= up;
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          uint32_t four[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float z[4];
            if (part == 0) {
              four[k] = codes8x4(y + 4 * k);
              values8x4(four[k], z);
            } else {
              four[k] = codes52x4(y + 4 * k);
              values52x4(four[k], z);
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) y[4 * k + n] -= z[n];  // what the part leaves over, exactly
          }
          *reinterpret_cast<uint4*>(qt + part * kPart + at128(row, i)) =
              make_uint4(four[0], four[1], four[2], four[3]);
        }
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
      auto visible = [&](int i, int u, uint32_t gone) {  // of a unit's tokens, by this row
        const int n = min(seen, p.stop) - p.start - kHalf * i - kUnit8 * u;
        return n <= 0 || (gone >> (8 * u) & 1u) ? 0u : n >= 16 ? 0xFFFFu : (1u << n) - 1u;
      };
      // The row sees tokens of half i with values that are not numbers: which, from their codes.
      auto mark = [&](int i) {
        const uint32_t note = (notes + i) % kNotes;
#pragma unroll 1
        for (int u = 0; u < 4; ++u) {
#pragma unroll 1
          for (uint32_t b = C->bad[note][u] & visible(i, u, C->gone[note]); b != 0; b &= b - 1) {
            const int tok = p.start + kHalf * i + kUnit8 * u + __ffs(b) - 1;
            const int page = tok / L.block_size;
            const uint32_t* const codes = reinterpret_cast<const uint32_t*>(
                static_cast<const uint8_t*>(L.cache) +
                L.table[p.r * L.table_stride + page] * L.block_stride + p.h * L.head_stride +
                (L.block_size + tok - page * L.block_size) * 128ll);
            uint32_t* const to = reinterpret_cast<uint32_t*>(&C->poison[x * 128 + row]);
#pragma unroll 1
            for (int w = 0; w < 4; ++w) {
              uint32_t bits = poisoned ? to[w] : 0u;
#pragma unroll 1
              for (int k = 0; k < 8; ++k)
                bits |= (not_numbers(codes[8 * w + k]) * 0x01020408u >> 24 & 15u) << (4 * k);
              to[w] = bits;
            }
            poisoned = true;
          }
        }
      };
      if (!KVS_WAIT(&C->s_full[x], half_no & 1)) return;
      uint32_t s_ready = 1;
      for (int i = 0; i < p.halves; ++i, ++half_no) {
        const int t0 = p.start + kHalf * i;
        const uint32_t buf = half_no & 1, W = tmem + kWeightsAt + 64 * x + 32 * buf + lanes;
        if (!__all_sync(0xFFFFFFFFu, s_ready) && !KVS_WAIT(&C->s_full[x], half_no & 1)) return;
        tc_fence_after();
        uint32_t v[2][32];
        tmem_ld32_start(S, v[0]);
        tmem_ld32_start(S + 32, v[1]);
        // what is known of the half was written before its codes were asked for
        const uint32_t note = (notes + i) % kNotes, gone = C->gone[note], any_bad = C->any_bad;
        const float4 v_exp = C->v_exp[note], k_up = C->k_up[note];
        const float ev[4] = {v_exp.x, v_exp.y, v_exp.z, v_exp.w};
        const float up4[4] = {k_up.x, k_up.y, k_up.z, k_up.w};
        float fs[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)  // not zero: a maximum of -inf is taken times it
          fs[u] = fmaxf(f * up4[u], 1.17549435e-38f);
        // Asked long before the answer is needed: a wait costs 140 clocks even when it is over.
        const bool next = i + 1 < p.halves;
        const uint32_t ahead = peek_phase(&C->pv_done[x][buf], ((half_no >> 1) & 1) ^ 1);
        tmem_arrived(v[0]);
        tmem_arrived(v[1]);
        tc_fence_before();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(&C->s_free[x]);
        const bool huge = fmaxf(fmaxf(up4[0], up4[1]), fmaxf(up4[2], up4[3])) > up_most;
        if (t0 + kHalf > plain_to || gone != 0) {  // hidden scores become -inf
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const uint32_t vis = visible(i, u, gone);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              uint32_t& y = v[u >> 1][16 * (u & 1) + k];
              y = vis >> k & 1u ? y : 0xFF800000u;
            }
          }
        }
        // Against the reference that there is, the scores only pass through once; a row whose
        // weights' sum has passed kMostSum (or 2^20 before the values' scales) makes the warp find the
        // maximum, rescale and take the scores again (the first half always does, and one whose scores
        // may be huge).
        uint32_t h[2][16];
        float sum;
        bool ready = false;
        for (bool fresh = i == 0 || huge;; fresh = true) {
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
                fmaxf(m, ceilf(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]))));
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
            if (huge) {
              const bool rounded = fabsf(m) > 0x1p23f;
#pragma unroll
              for (int u = 0; u < 4; ++u) {
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                  uint32_t& y = v[u >> 1][16 * (u & 1) + k];
                  const float s = __uint_as_float(y);
                  y = __float_as_uint(rounded ? __fsub_rn(__fmul_rn(s, fs[u]), m)
                                              : fmaf(s, fs[u], -m));
                }
                fs[u] = 1.f;
              }
            }
          }
          const float off = huge ? 0.f : m;
          f32x2_t s2[4];
          float d[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            d[u] = fmaxf(ev[u] - K, -kFar);
            s2[u] = f2_pack(0.f, 0.f);
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float ref = d[u] - off;
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
          const bool past = fmaxf(all, sum * kSumBefore) > kMostSum;
          ready = __all_sync(0xFFFFFFFFu, ahead != 0 && !past);
          if (ready || !__any_sync(0xFFFFFFFFu, past)) break;
        }
        l += sum;
        // the products with the weights two halves ago
        if (!ready && !KVS_WAIT(&C->pv_done[x][buf], ((half_no >> 1) & 1) ^ 1)) return;
        tc_fence_after();
        if (any_bad && i >= 3) mark(i - 3);  // whose values were converted when any_bad was read
        s_ready = next ? peek_phase(&C->s_full[x], (half_no + 1) & 1) : 0u;
        tmem_st16(W, h[0]);
        tmem_st16(W + 16, h[1]);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(&C->p_full[x][half_no & 1]);
      }
      for (int back = p.halves > 1 ? 2 : 1; back > 0; --back) {  // both buffers' last products
        const uint32_t no = half_no - back;
        if (!KVS_WAIT(&C->pv_done[x][no & 1], (no >> 1) & 1)) return;
      }
      tc_fence_after();
      if (C->any_bad)
        for (int i = max(0, p.halves - 3); i < p.halves; ++i) mark(i);
      notes += p.halves;
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(&C->done[x]);
    }
    // ---- the result, or this part of it
    const float unit = p.steps > 0 ? pow2(static_cast<int>(K)) : 0.f;
    const float inv = l == 0.f ? 0.f : __fdividef(1.f, l);
    const int slot = 2 * static_cast<int>(blockIdx.x) + (p.begins ? 1 : 0);
    uint8_t* const out = reinterpret_cast<uint8_t*>(static_cast<uint16_t*>(L.out) + tq * L.o_ts +
                                                    hq * L.o_hs);
    uint8_t* const part = reinterpret_cast<uint8_t*>(
        P.o + (static_cast<long long>(slot) * kRows + x * 128 + row) * 128);
    // 128 bytes of each row, from a thread a row
    auto flush = [&](const uint4 (&w)[8], uint8_t* at, uint8_t* to) {
#pragma unroll
      for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(at + at128(lane, i)) = w[i];
      __syncwarp();
      uint4 y[8];
      uint8_t* dst[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + (lane >> 3);
        y[i] = *reinterpret_cast<const uint4*>(at + at128(r, lane & 7));
        dst[i] = const_cast<uint8_t*>(of_lane(to, r)) + 16 * (lane & 7);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (has >> (4 * i + (lane >> 3)) & 1u) *reinterpret_cast<uint4*>(dst[i]) = y[i];
    };
    // 32 channels of the output, in loops: what runs once a piece is not in the instruction cache
    auto channels = [&](int cg, float (&v)[32]) {
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
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] *= unit;
    };
    if (p.whole) {
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        uint4 w[8];
#pragma unroll
        for (int cg = 0; cg < 2; ++cg) {
          float v[32];
          channels(2 * half + cg, v);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] *= inv;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[4 * cg + i] = pack8<FP16>(*reinterpret_cast<const float(*)[8]>(v + 8 * i));
        }
        flush(w, area + half * kPart, out + 128 * half);
      }
    } else {
#pragma unroll 1
      for (int cg = 0; cg < 4; ++cg) {
        float v[32];
        channels(cg, v);
        uint4 w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          w[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]),
                            __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
        flush(w, area + (cg & 1) * kPart, part + 128 * cg);
        __syncwarp();
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
      P.desc[blockIdx.x] = make_int4(p.s.row0, p.h, p.tile,
                                     p.parts | min(kRows, p.nrows - p.tile * kRows) << 16);
    tc_fence_before();
    __syncwarp();
  }
}

template <bool FP16>
__global__ void __launch_bounds__(kThreads, 1)
    k_attn8_tile(const __grid_constant__ Attn4Launch L, const __grid_constant__ CUtensorMap map) {
  extern __shared__ uint8_t raw_smem[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  Ctrl* const C = reinterpret_cast<Ctrl*>(smem + Layout<FP16>::ctrl);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = L.q_heads / L.heads, B = gridDim.x, b = blockIdx.x;
  const Parts P = parts(L.scratch, B, kRows);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    P.desc[b] = make_int4(-1, 0, 0, 0);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&C->q_full[i], 4);
      mbar_init(&C->s_full[i], 1);
      mbar_init(&C->s_free[i], 4);
      mbar_init(&C->done[i], 4);
      for (int k = 0; k < 2; ++k) {
        mbar_init(&C->p_full[i][k], 4);
        mbar_init(&C->pv_done[i][k], 1);
      }
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&C->k_full[i], 1);
      mbar_init(&C->k_empty[i], 2);
      mbar_init(&C->v_came[i], 1);
      mbar_init(&C->v_taken[i], 4);
      mbar_init(&C->v_full[i], 4);
      mbar_init(&C->v_empty[i], 1);
    }
    for (int i = 0; i < kPieces; ++i) {
      mbar_init(&C->piece_full[i], 1);
      mbar_init(&C->piece_empty[i], kReaders);
    }
    C->any_bad = 0;
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
  Walk<kOverTile, true> walk;
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
    // 256 x 168 + 256 x 88 = the 512 x 128 registers of the launch
    if (warp < 8) {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
      softmax_role<FP16>(L, group, smem, tmem, P, C);
    } else if (warp < 12) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
      convert_role<FP16>(L, smem, C);
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
      if (warp < 14)
        qk_role<FP16>(L, warp & 1, smem_u32(smem), tmem, C);
      else if (warp == 14)
        pv_role<FP16>(L, smem_u32(smem), tmem, C);
      else
        fetch_role<FP16>(L, &map, walk, group, smem_u32(smem), C);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(tmem, 512);
}

template <bool FP16>
cudaError_t launch(const Attn4Launch& L, const CUtensorMap& map, cudaStream_t s) {
  cudaError_t e = cudaFuncSetAttribute(k_attn8_tile<FP16>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<FP16>::bytes);
  if (e != cudaSuccess) return e;
  const int ctas = tile_ctas<kOverTile>(L);
  k_attn8_tile<FP16><<<ctas, kThreads, Layout<FP16>::bytes, s>>>(L, map);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  const long long rows = static_cast<long long>(L.max_q) * (L.q_heads / L.heads);
  return launch_join<FP16, kRows>(L, ctas, static_cast<long long>(L.seqs) * L.heads *
                                               ((rows + kRows - 1) / kRows), s);
}

}  // namespace

cudaError_t attn8_tile_launch(const Attn4Launch& L, const CUtensorMap& map, cudaStream_t s) {
  return L.fp16 ? launch<true>(L, map, s) : launch<false>(L, map, s);
}

long long attn8_tile_scratch(const Attn4Launch& L) {
  return 16ll * tile_ctas<kOverTile>(L) + 2ll * tile_ctas<kOverTile>(L) * kRows * (8 + 512);
}

}  // namespace kvs
