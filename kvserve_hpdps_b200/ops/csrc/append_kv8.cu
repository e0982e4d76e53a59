// New tokens into a paged KV cache held in 8 bits (kv8.cuh has the layout), the position rotation
// applied on the way (append_kv.cu has its formulas), and its rows back as 16-bit values.
//
// For a unit of 16 tokens and one head, keys and values apart, N being the call's tokens in it:
//   need = scale_exponent(max over N of |x|),  e = need when N has the token at offset 0
//                                                  max(need, the unit's e) else
//   code = e4m3(x 2^-e) for N; the unit's other codes become e4m3(code 2^(its e - e)).
// x is the rotated fp32 value, not rounded to 16 bits in between.  A token at offset 0 begins its
// unit anew: what the unit held is a former sequence's, whose scale must not stay.
//
// A unit's scale needs all of the call's tokens in it, wherever they stand in slot_mapping.  The
// first of them (the leader) takes all 16 slots: so no two CTAs write one unit, there is no second
// launch and no atomic on the cache, and results do not depend on timing.  A CTA looks for leaders
// among a window of tokens.  Tokens of a unit mostly stand next to each other: every warp looks at
// the 15 tokens before and behind by itself, and a unit that it finds there whole, and not begun
// before, is settled without another word.  Only for the others (both ends of a sequence's
// new tokens, a decode step's) all slots of the call are looked through, by 256 threads.  In any
// order at all that is quadratic: 16384 tokens of 8 heads take 45 us in order, 219 shuffled.
//
// What bounds it: for many tokens the instructions of rotating and encoding between the loads and the
// stores (16379 tokens of 32+8 heads, 378 MB: 74 us, 78 % of the copy rate), for few the chain
// slots, rows, codes (in a captured graph of several states in turn: one token 2.9 us, 48 of as many
// sequences 4.3).
#include <type_traits>

#include "append_kv.cuh"
#include "kv8.cuh"

namespace kvs {

namespace {

constexpr int kWarps8 = kThreads / 32, kJobs = kWarps8 / 2;  // heads' keys or values at once
// A CTA takes one token up to kFewTokens (decode steps: every token has a unit of its own), else 16.
// Measured, 32+8 heads, one a CTA / 16: 300 tokens of as many sequences 12.3 / 27.7 us, of one 9.6 /
// 7.9; 500 tokens 15.4 / 30.7 and 12.3 / 7.9; 700 tokens 22.5 / 31.4 and 16.4 / 7.9.
constexpr int kFewTokens = 512;

// Rows of queries, eight lanes each, as k_append_kv deals them out.
template <bool FP16, int MODE, int EACH>
KVS_DEV void rotate_queries(const AppendLaunch& L, const Spread& S, int x, int y) {
  const int l = threadIdx.x & 7, gi = threadIdx.x >> 3;
  const uint32_t mask = 0xFFu << (threadIdx.x & 24);
  const int t = x * (kGroups / S.across) + gi / S.across;
  if (t >= L.tokens) return;
  const int first = y * S.across * EACH + (gi & (S.across - 1));
  if (first >= L.q_heads) return;
  const long long pos = load_index(L.pos, t, L.pos64);
  const bool turn = pos >= 0 && pos < L.max_pos;
  if (!turn && l == 0) record_error(L.err, ERR_BOUNDS);
  float co[2][8], si[2][8];
  if (turn) load_angles<FP16, MODE>(L, pos, l, co, si);
  uint4 raw[EACH][2], partner[EACH][2];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int h = first + S.across * e;
    if (h >= L.q_heads) break;
    const uint16_t* src = static_cast<const uint16_t*>(L.query) + t * L.q_ts + h * L.q_hs;
    raw[e][0] = *reinterpret_cast<const uint4*>(src + 8 * l);
    raw[e][1] = *reinterpret_cast<const uint4*>(src + 8 * l + 64);
    if (MODE == kPart) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int ch = 8 * (l + 8 * k);
        if (ch < L.rotary)
          partner[e][k] = *reinterpret_cast<const uint4*>(src + partner_of(ch, L.rotary));
      }
    }
  }
  if (MODE == kPart) __syncwarp(mask);  // rotated in place: all read before any writes
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int h = first + S.across * e;
    if (h >= L.q_heads) break;
    float v[2][8];
    unpack8<FP16>(raw[e][0], v[0]);
    unpack8<FP16>(raw[e][1], v[1]);
    if (turn) rotate<FP16, MODE>(L.rotary, l, partner[e], co, si, v);
    uint16_t* dst = static_cast<uint16_t*>(L.query_out) + t * L.qo_ts + h * L.qo_hs;
    *reinterpret_cast<uint4*>(dst + 8 * l) = pack8<FP16>(v[0]);
    *reinterpret_cast<uint4*>(dst + 8 * l + 64) = pack8<FP16>(v[1]);
  }
}

struct Units {
  int id[kUnit8];               // units to be looked for, or -1
  int member[kUnit8][kUnit8];   // [unit][offset] the call's last token there, or -1
  int first[kUnit8];            // the call's first token in the unit
};

// One unit's keys or values of one head, two warps, eight rows each (16 in one warp's registers do
// not fit beside a rotation's angles): four at a time, eight lanes a row.  This warp's row
// 4 it + sub is token tok<it> at position pos<it>, or is not the call's (-1).
template <bool FP16, int MODE>
KVS_DEV void append_unit(const AppendLaunch& L, int tok0, int tok1, long long pos0, long long pos1,
                         bool begins, bool whole, int unit, int h, int value, uint32_t* s_top) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane & 7, sub = lane >> 3;
  const int tok[2] = {tok0, tok1};
  const long long pos[2] = {pos0, pos1};
  // the largest of both warps'
  auto both = [&](uint32_t top) {
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if (lane == 0) s_top[warp] = top;
    asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp >> 1)) : "memory");
    top = max(top, s_top[warp ^ 1]);
    asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp >> 1)) : "memory");
    return top;
  };
  const uint32_t per = static_cast<uint32_t>(L.block_size) / kUnit8;
  const uint32_t blk = static_cast<uint32_t>(unit) / per;
  const int u = static_cast<int>(static_cast<uint32_t>(unit) - blk * per);
  uint8_t* const rec = static_cast<uint8_t*>(L.cache) +
                       static_cast<long long>(blk) * L.block_stride + h * L.head_stride;
  uint8_t* const rows = rec + (value * L.block_size + u * kUnit8 + 8 * (warp & 1)) * 128ll;
  uint8_t* const byte = rec + 256ll * L.block_size + 2 * u + value;
  const int was = whole ? 0 : *byte;
  float y[2][2][8];
  uint32_t top = 0;
  uint4 raw[2][2], partner[2][2];
#pragma unroll
  for (int it = 0; it < 2; ++it) {
    raw[it][0] = raw[it][1] = make_uint4(0u, 0u, 0u, 0u);
    if (tok[it] < 0) continue;
    const uint16_t* src =
        value ? static_cast<const uint16_t*>(L.value) + tok[it] * L.val_ts + h * L.val_hs
              : static_cast<const uint16_t*>(L.key) + tok[it] * L.key_ts + h * L.key_hs;
    raw[it][0] = *reinterpret_cast<const uint4*>(src + 8 * l);
    raw[it][1] = *reinterpret_cast<const uint4*>(src + 8 * l + 64);
    if (MODE == kPart && !value && L.pos != nullptr) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int ch = 8 * (l + 8 * k);
        if (ch < L.rotary)
          partner[it][k] = *reinterpret_cast<const uint4*>(src + partner_of(ch, L.rotary));
      }
    }
  }
#pragma unroll
  for (int it = 0; it < 2; ++it) {
    unpack8<FP16>(raw[it][0], y[it][0]);
    unpack8<FP16>(raw[it][1], y[it][1]);
    if (!value && L.pos != nullptr && tok[it] >= 0) {
      float co[2][8], si[2][8];
      load_angles<FP16, MODE>(L, pos[it], l, co, si);
      rotate<FP16, MODE>(L.rotary, l, partner[it], co, si, y[it]);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      top = max(top, __float_as_uint(y[it][i >> 3][i & 7]) & 0x7FFFFFFFu);
  }
  top = both(top);
  constexpr uint32_t kInf = 0x7F800000u;
  if (top >= kInf) {  // the largest that is finite; infinities become what is not a number
    top = 0;
#pragma unroll
    for (int it = 0; it < 2; ++it)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float& x = y[it][i >> 3][i & 7];
        const uint32_t bits = __float_as_uint(x) & 0x7FFFFFFFu;
        if (bits < kInf)
          top = max(top, bits);
        else
          x = __uint_as_float(0x7FC00000u);
      }
    top = both(top);
  }
  // a byte that no append writes is a cache's that was never cleared: it has no say
  const int old = was > kTopByte ? kLowScale : max(was - 127, kLowScale);
  const int need = scale_exponent(top), e = begins ? need : max(need, old);
  const float down = pow2(-e);
#pragma unroll
  for (int it = 0; it < 2; ++it) {
    uint8_t* const row = rows + (4 * it + sub) * 128;
    if (tok[it] >= 0) {
#pragma unroll
      for (int i = 0; i < 16; ++i) y[it][i >> 3][i & 7] *= down;
#pragma unroll
      for (int k = 0; k < 2; ++k)
        *reinterpret_cast<uint2*>(row + 64 * k + 8 * l) =
            make_uint2(codes8x4(y[it][k]), codes8x4(y[it][k] + 4));
    } else if (!begins && e > old) {  // the scale has grown past a row that was there
      const float f = pow2(max(old - e, -127));
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint2* const at = reinterpret_cast<uint2*>(row + 64 * k + 8 * l);
        float x[8];
        values8x4(at->x, x);
        values8x4(at->y, x + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= f;
        *at = make_uint2(codes8x4(x), codes8x4(x + 4));
      }
    }
  }
  if (lane == 0 && !(warp & 1)) *byte = static_cast<uint8_t>(e + 127);
}

// Blocks [0, kv): of window x / parts the heads of part x % parts.  Behind them the queries.
template <bool FP16, int MODE, int WINDOW, int EACH, int CTAS>
__global__ void __launch_bounds__(kThreads, CTAS)
    k_append_kv8(const __grid_constant__ AppendLaunch L, const __grid_constant__ Spread S, int kv,
                 int parts) {
  if (static_cast<int>(blockIdx.x) >= kv) {
    const unsigned q = blockIdx.x - kv;
    rotate_queries<FP16, MODE, EACH>(L, S, static_cast<int>(q % S.x), static_cast<int>(q / S.x));
    return;
  }
  __shared__ Units U;
  __shared__ int s_from[kWarps8][kUnit8];
  __shared__ uint32_t s_top[kWarps8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sub = lane >> 3;
  const int x = static_cast<int>(blockIdx.x), part = x % parts, i0 = x / parts * WINDOW;
  // This pair of warps' heads' keys or values, keys and values in turn.
  const int jobs = 2 * L.heads;
  auto each = [&](auto f) {
#pragma unroll 1
    for (int n = part, j; (j = n * kJobs + (warp >> 1)) < jobs; n += parts) f(j >> 1, (j + n) & 1);
  };
  const int row0 = 8 * (warp & 1) + sub;  // of this lane in a unit; 4 further on the second
  auto fine = [&](long long slot, long long pos) {
    return slot >= 0 && slot < L.num_slots && (L.pos == nullptr || (pos >= 0 && pos < L.max_pos));
  };
  auto position = [&](int i) { return L.pos != nullptr ? load_index(L.pos, i, L.pos64) : 0; };
  if constexpr (WINDOW == 1) {
    // ---- few tokens: every warp looks through all slots, which it asks for with its own token's
    long long at[kFewTokens / 32];
#pragma unroll
    for (int n = 0; n < kFewTokens / 32; ++n) {
      if (32 * n >= L.tokens) break;
      at[n] = lane + 32 * n < L.tokens ? load_index(L.slots, lane + 32 * n, L.slots64) : -1;
    }
    const long long slot = load_index(L.slots, i0, L.slots64), pos = position(i0);
    if (!fine(slot, pos)) {
      if (slot >= 0 && part + tid == 0) record_error(L.err, ERR_BOUNDS);
      return;
    }
    if (lane < kUnit8) s_from[warp][lane] = -1;
    __syncwarp();
    int first = i0;
#pragma unroll
    for (int n = 0; n < kFewTokens / 32; ++n) {
      if (32 * n >= L.tokens) break;
      const int i = lane + 32 * n;
      if (at[n] / kUnit8 == slot / kUnit8 && at[n] >= 0 && (i == i0 || fine(at[n], position(i)))) {
        atomicMax(&s_from[warp][at[n] % kUnit8], i);
        first = min(first, i);
      }
    }
    __syncwarp();
    if (__reduce_min_sync(0xFFFFFFFFu, first) < i0) return;
    const uint32_t has = __ballot_sync(0xFFFFFFFFu, lane < kUnit8 && s_from[warp][lane & 15] >= 0);
    int tok[2];
    long long where[2];
#pragma unroll
    for (int it = 0; it < 2; ++it) {
      tok[it] = s_from[warp][row0 + 4 * it];
      where[it] = tok[it] < 0 || tok[it] == i0 ? pos : position(tok[it]);
    }
    each([&](int h, int value) {
      append_unit<FP16, MODE>(L, tok[0], tok[1], where[0], where[1], has & 1u, has == 0xFFFFu,
                              static_cast<int>(slot / kUnit8), h, value, s_top);
    });
    return;
  }
  // ---- the window's tokens, the 15 behind them and the 15 before
  long long slot = -1, slot_b = -1, pos = 0, pos_b = 0;
  const int ia = i0 + lane, ib = i0 - 15 + lane;
  const bool in = lane < WINDOW + 15 && ia < L.tokens, in_b = lane < 15 && ib >= 0;
  if (in) slot = load_index(L.slots, ia, L.slots64);
  if (in_b) slot_b = load_index(L.slots, ib, L.slots64);
  if (L.pos != nullptr) {
    if (in) pos = load_index(L.pos, ia, L.pos64);
    if (in_b) pos_b = load_index(L.pos, ib, L.pos64);
  }
  if (lane < WINDOW && slot >= 0 && !fine(slot, pos) && part + warp == 0)
    record_error(L.err, ERR_BOUNDS);
  const int unit = fine(slot, pos) ? static_cast<int>(slot / kUnit8) : -1;
  const int unit_b = fine(slot_b, pos_b) ? static_cast<int>(slot_b / kUnit8) : -2;
  const int off = static_cast<int>(slot) & (kUnit8 - 1);
  const uint32_t same = __match_any_sync(0xFFFFFFFFu, unit);
  uint32_t todo = __ballot_sync(0xFFFFFFFFu, lane < WINDOW && unit >= 0 && __ffs(same) - 1 == lane);
  uint32_t open = 0;  // window tokens whose units have to be looked for everywhere
  for (; todo != 0; todo &= todo - 1) {
    const int k = __ffs(todo) - 1;
    const int u = __shfl_sync(0xFFFFFFFFu, unit, k);
    if (__any_sync(0xFFFFFFFFu, unit_b == u)) continue;  // begun before: another window's
    const bool is = unit == u;
    const uint32_t found = __ballot_sync(0xFFFFFFFFu, is);
    const uint32_t offs = __reduce_or_sync(0xFFFFFFFFu, is ? 1u << off : 0u);
    if (__popc(found) != kUnit8 || offs != 0xFFFFu) {
      open |= 1u << k;
      continue;
    }
    if (is) s_from[warp][off] = lane;
    __syncwarp();
    int tok[2];
    long long at[2];
#pragma unroll
    for (int it = 0; it < 2; ++it) {
      const int from = s_from[warp][row0 + 4 * it];
      tok[it] = i0 + from;
      at[it] = __shfl_sync(0xFFFFFFFFu, pos, from);
    }
    each([&](int h, int value) {
      append_unit<FP16, MODE>(L, tok[0], tok[1], at[0], at[1], true, true, u, h, value, s_top);
    });
    __syncwarp();
  }
  if (open == 0) return;  // the same for all warps
  // ---- the others: the tokens of the call that are in them, wherever they stand
  if (warp == 0 && lane < WINDOW) {
    U.id[lane] = open >> lane & 1u ? unit : -1;
    U.first[lane] = 0x7FFFFFFF;
  }
  for (int i = tid; i < WINDOW * kUnit8; i += kThreads) U.member[i / kUnit8][i % kUnit8] = -1;
  __syncthreads();
  // Eight slots a thread at a time, whose loads are in flight together: one after the other they
  // took 40 us for 16384.
  const bool wanted = lane < WINDOW && (open >> lane & 1u);
  const int low = __reduce_min_sync(0xFFFFFFFFu, wanted ? unit : 0x7FFFFFFF),
            high = __reduce_max_sync(0xFFFFFFFFu, wanted ? unit : -1);
  for (int from = tid; from < L.tokens; from += 8 * kThreads) {
    long long at[8];
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const int i = from + n * kThreads;
      at[n] = i < L.tokens ? load_index(L.slots, i, L.slots64) : -1;
    }
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      if (at[n] < 0 || at[n] >= L.num_slots) continue;
      const int in_unit = static_cast<int>(at[n] / kUnit8), i = from + n * kThreads;
      if (in_unit < low || in_unit > high) continue;
#pragma unroll 1
      for (int k = 0; k < WINDOW; ++k) {
        if (U.id[k] != in_unit) continue;
        if (fine(at[n], position(i))) {
          atomicMax(&U.member[k][at[n] % kUnit8], i);
          atomicMin(&U.first[k], i);
        }
        break;
      }
    }
  }
  __syncthreads();
#pragma unroll 1
  for (; open != 0; open &= open - 1) {
    const int k = __ffs(open) - 1;
    if (U.first[k] < i0) continue;
    int tok[2];
    long long at[2];
#pragma unroll
    for (int it = 0; it < 2; ++it) {
      tok[it] = U.member[k][row0 + 4 * it];
      at[it] = tok[it] >= 0 ? position(tok[it]) : 0;
    }
    each([&](int h, int value) {
      append_unit<FP16, MODE>(L, tok[0], tok[1], at[0], at[1], U.member[k][0] >= 0, false,
                              U.id[k], h, value, s_top);
    });
  }
}

// Eight lanes read one row: key rows of a token, then value rows; slot < 0 reads zeros.
template <bool FP16, int EACH>
__global__ void __launch_bounds__(kThreads, 3)
    k_read_kv8(const __grid_constant__ Read4Launch L, const __grid_constant__ Spread S) {
  const int l = threadIdx.x & 7, gi = threadIdx.x >> 3;
  const int t = static_cast<int>(blockIdx.x) * (kGroups / S.across) + gi / S.across;
  if (t >= L.tokens) return;
  const int first = static_cast<int>(blockIdx.y) * S.across * EACH + (gi & (S.across - 1));
  const int rows = 2 * L.heads;
  if (first >= rows) return;
  long long slot = load_index(L.slots, t, L.slots64);
  if (slot >= L.num_slots) {
    if (l == 0) record_error(L.err, ERR_BOUNDS);
    slot = -1;
  }
  const long long blk = slot < 0 ? 0
                        : L.num_slots < (1ll << 31)
                            ? static_cast<long long>(static_cast<uint32_t>(slot) /
                                                     static_cast<uint32_t>(L.block_size))
                            : slot / L.block_size;
  const int off = slot < 0 ? 0 : static_cast<int>(slot - blk * L.block_size);
  uint2 w[EACH][2];
  uint32_t b[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int r = first + S.across * e;
    w[e][0] = w[e][1] = make_uint2(0u, 0u);
    b[e] = 0;
    if (r >= rows || slot < 0) continue;
    const int value = r >= L.heads, h = r - value * L.heads;
    const uint8_t* rec =
        static_cast<const uint8_t*>(L.cache) + blk * L.block_stride + h * L.head_stride;
    const uint8_t* row = rec + (value * L.block_size + off) * 128ll + 8 * l;
    w[e][0] = *reinterpret_cast<const uint2*>(row);
    w[e][1] = *reinterpret_cast<const uint2*>(row + 64);
    b[e] = rec[256ll * L.block_size + 2 * (off / kUnit8) + value];
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int r = first + S.across * e;
    if (r >= rows) break;
    const int value = r >= L.heads, h = r - value * L.heads;
    uint16_t* out = static_cast<uint16_t*>(L.out) +
                    ((static_cast<long long>(value) * L.tokens + t) * L.heads + h) * 128 + 8 * l;
    const float f = __uint_as_float(b[e] << 23);
    constexpr float kMost = FP16 ? 65504.f : 0x1.FEp127f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float y[8];
      values8x4(w[e][k].x, y);
      values8x4(w[e][k].y, y + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i)  // a code may round up past the type's largest number
        y[i] = min_nan(max_nan(y[i] * f, -kMost), kMost);
      *reinterpret_cast<uint4*>(out + 64 * k) = pack8<FP16>(y);
    }
  }
}

template <bool FP16, int MODE, int WINDOW>
int append(const AppendLaunch& L, cudaStream_t s) {
  const Spread S = spread_of(L.tokens, L.q_heads);
  const long long windows = (L.tokens + WINDOW - 1) / WINDOW;
  // All heads in one CTA when the windows fill the SMs: finding its units takes as long as a job.
  // Measured, 32+8 heads, apart / in one CTA: one token a window, 64 tokens 4.1 / 6.2 us, 128 6.8 /
  // 6.5, 256 13.3 / 8.5; 16 tokens a window, 2000 tokens 12.7 / 14.3, 3000 17.7 / 15.5, 4000 24.6 /
  // 19.5.
  const int most = (2 * L.heads + kJobs - 1) / kJobs;
  const int parts = windows > 148 ? (most > 0) : most;
  const long long kv = windows * parts;
  const long long q = L.q_heads > 0 ? static_cast<long long>(S.x) * S.y : 0;
  if (kv + q >= (1ll << 31) || L.num_slots / kUnit8 >= (1ll << 31)) return -2;
  const unsigned grid = static_cast<unsigned>(kv + q);
  const int kv_ctas = static_cast<int>(kv);
  // Registers for two CTAs an SM, or for three whose windows are many: their loads cover one
  // another's, and spilled registers cost less than that.  Measured, 32+8 heads, two / three: 700
  // tokens 7.5 / 9.2 us, 4096 20.1 / 26.3, 6000 30.7 / 32.1, 8192 41.3 / 41.0, 16379 83 / 74; rotated in
  // part 16379 92 / 163.
  auto start = [&](auto each, auto ctas) {
    k_append_kv8<FP16, MODE, WINDOW, each.value, ctas.value>
        <<<grid, kThreads, 0, s>>>(L, S, kv_ctas, parts);
  };
  using One = std::integral_constant<int, 1>;
  using Four = std::integral_constant<int, 4>;
  using Two = std::integral_constant<int, 2>;
  if constexpr (WINDOW > 1 && MODE != kPart) {
    if (windows > 400) {
      using Three = std::integral_constant<int, 3>;
      S.each == 4 ? start(Four{}, Three{}) : start(One{}, Three{});
      return cudaGetLastError() == cudaSuccess ? 0 : -1;
    }
  }
  S.each == 4 ? start(Four{}, Two{}) : start(One{}, Two{});
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}
template <bool FP16, int MODE>
int append_window(const AppendLaunch& L, cudaStream_t s) {
  return L.tokens <= kFewTokens ? append<FP16, MODE, 1>(L, s) : append<FP16, MODE, kUnit8>(L, s);
}
template <bool FP16>
int append_mode(const AppendLaunch& L, cudaStream_t s) {
  if (L.pos == nullptr || (!L.interleaved && L.rotary == 128))
    return append_window<FP16, kHalves>(L, s);
  return L.interleaved ? append_window<FP16, kPairs>(L, s) : append_window<FP16, kPart>(L, s);
}
template <bool FP16>
void read(const Read4Launch& L, const Spread& S, cudaStream_t s) {
  if (S.each == 4)
    k_read_kv8<FP16, 4><<<dim3(S.x, S.y), kThreads, 0, s>>>(L, S);
  else
    k_read_kv8<FP16, 1><<<dim3(S.x, S.y), kThreads, 0, s>>>(L, S);
}

}  // namespace
}  // namespace kvs

using namespace kvs;

extern "C" {

int kvs_append_kv8(const AppendLaunch* L, void* stream) {
  if (L->tokens <= 0 || L->q_heads + L->heads <= 0) return 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return L->fp16 ? append_mode<true>(*L, s) : append_mode<false>(*L, s);
}

int kvs_read_kv8(const Read4Launch* L, void* stream) {
  if (L->tokens <= 0 || L->heads <= 0) return 0;
  const Spread S = spread_of(L->tokens, 2 * L->heads);
  if (S.y > 65535u) return -2;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (L->fp16)
    read<true>(*L, S, s);
  else
    read<false>(*L, S, s);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}

}  // extern "C"
