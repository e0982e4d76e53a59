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
// launch and no atomic, and results do not depend on timing.  A CTA looks for leaders among
// a window of tokens.  Tokens of a unit mostly stand next to each other, so it first looks at the 15
// tokens around; a unit that it finds there whole is settled.  Only for the others (both ends of
// a sequence's new tokens, a decode step's) all slots of the call are looked through, by
// 256 threads: 2 us for 16384.  In any order at all that is quadratic, and still 60 us for 16384.
#include "append_kv.cuh"
#include "kv8.cuh"

namespace kvs {

namespace {

constexpr int kWarps8 = kThreads / 32;
constexpr int kManyTokens = 4096;  // from here on a CTA takes 16 tokens instead of one

// Where a token goes; false: nowhere.
KVS_DEV bool place(const AppendLaunch& L, int i, bool report, long long& slot) {
  slot = load_index(L.slots, i, L.slots64);
  if (slot < 0) return false;
  bool ok = slot < L.num_slots;
  if (ok && L.pos != nullptr) {
    const long long pos = load_index(L.pos, i, L.pos64);
    ok = pos >= 0 && pos < L.max_pos;
  }
  if (!ok && report) record_error(L.err, ERR_BOUNDS);
  return ok;
}

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
  long long id[kUnit8];         // of a window token that is the first of its unit there; else -1
  int member[kUnit8][kUnit8];   // [window token][offset] the call's last token there, or -1
  int first[kUnit8];            // the call's first token in the unit
  int count[kUnit8];            // tokens found around the window
  int open;                     // some unit has to be looked for everywhere
};

// One unit's keys or values of one head, a warp: four rows at a time, eight lanes each.
template <bool FP16, int MODE>
KVS_DEV void append_unit(const AppendLaunch& L, const int (&member)[kUnit8], long long unit, int h,
                         int value) {
  const int lane = threadIdx.x & 31, l = lane & 7, sub = lane >> 3;
  const int per = L.block_size / kUnit8;
  const long long blk = L.num_slots < (1ll << 31)
                            ? static_cast<long long>(static_cast<uint32_t>(unit) /
                                                     static_cast<uint32_t>(per))
                            : unit / per;
  const int u = static_cast<int>(unit - blk * per);
  uint8_t* const rec = static_cast<uint8_t*>(L.cache) + blk * L.block_stride + h * L.head_stride;
  uint8_t* const rows = rec + (value * L.block_size + u * kUnit8) * 128ll;
  uint8_t* const byte = rec + 256ll * L.block_size + 2 * u + value;
  const int was = *byte;
  const bool begins = member[0] >= 0;
  int tok[4];
  float y[4][2][8];
  uint32_t top = 0;
  uint4 raw[4][2], partner[4][2];
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    tok[it] = member[4 * it + sub];
    raw[it][0] = raw[it][1] = make_uint4(0u, 0u, 0u, 0u);
    if (tok[it] < 0) continue;
    const uint16_t* src = value ? static_cast<const uint16_t*>(L.value) + tok[it] * L.val_ts + h * L.val_hs
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
  for (int it = 0; it < 4; ++it) {
    unpack8<FP16>(raw[it][0], y[it][0]);
    unpack8<FP16>(raw[it][1], y[it][1]);
    if (!value && L.pos != nullptr && tok[it] >= 0) {
      float co[2][8], si[2][8];
      load_angles<FP16, MODE>(L, load_index(L.pos, tok[it], L.pos64), l, co, si);
      rotate<FP16, MODE>(L.rotary, l, partner[it], co, si, y[it]);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      top = max(top, __float_as_uint(y[it][i >> 3][i & 7]) & 0x7FFFFFFFu);
  }
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  constexpr uint32_t kInf = 0x7F800000u;
  if (top >= kInf) {  // the largest that is finite; infinities become what is not a number
    top = 0;
#pragma unroll
    for (int it = 0; it < 4; ++it)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float& x = y[it][i >> 3][i & 7];
        const uint32_t bits = __float_as_uint(x) & 0x7FFFFFFFu;
        if (bits < kInf)
          top = max(top, bits);
        else
          x = __uint_as_float(0x7FC00000u);
      }
    top = __reduce_max_sync(0xFFFFFFFFu, top);
  }
  // a byte that no append writes is a cache's that was never cleared: it has no say
  const int old = was > kTopByte ? kLowScale : max(was - 127, kLowScale);
  const int need = scale_exponent(top), e = begins ? need : max(need, old);
  const float down = pow2(-e);
#pragma unroll
  for (int it = 0; it < 4; ++it) {
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
  __syncwarp();
  if (lane == 0) *byte = static_cast<uint8_t>(e + 127);
}

// Blocks [0, kv): window x / parts, heads of part x % parts.  Behind them the queries.
template <bool FP16, int MODE, int WINDOW, int EACH>
__global__ void __launch_bounds__(kThreads, 2)
    k_append_kv8(const __grid_constant__ AppendLaunch L, const __grid_constant__ Spread S, int kv,
                 int parts) {
  if (static_cast<int>(blockIdx.x) >= kv) {
    const unsigned q = blockIdx.x - kv;
    rotate_queries<FP16, MODE, EACH>(L, S, static_cast<int>(q % S.x), static_cast<int>(q / S.x));
    return;
  }
  __shared__ Units U;
  const int tid = threadIdx.x, warp = tid >> 5;
  const int part = static_cast<int>(blockIdx.x) % parts;
  const int i0 = static_cast<int>(blockIdx.x) / parts * WINDOW;
  const int lo = max(0, i0 - 15), hi = min(L.tokens, i0 + WINDOW + 15);
  // ---- the window's units
  if (tid < 32) {
    long long unit = -1;
    if (tid < WINDOW && i0 + tid < L.tokens) {
      long long slot;
      if (place(L, i0 + tid, part == 0, slot)) unit = slot / kUnit8;
    }
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, unit);
    if (unit >= 0 && __ffs(same) - 1 != tid) unit = -1;
    if (tid < WINDOW) {
      U.id[tid] = unit;
      U.first[tid] = 0x7FFFFFFF;
      U.count[tid] = 0;
    }
    if (tid == 0) U.open = 0;
  }
  for (int i = tid; i < WINDOW * kUnit8; i += kThreads) U.member[i / kUnit8][i % kUnit8] = -1;
  __syncthreads();
  auto take = [&](int i) {
    const long long slot = load_index(L.slots, i, L.slots64);
    if (slot < 0 || slot >= L.num_slots) return;
#pragma unroll
    for (int k = 0; k < WINDOW; ++k) {
      if (U.id[k] == slot / kUnit8) {
        long long again;
        if (!place(L, i, false, again)) return;
        atomicMax(&U.member[k][slot % kUnit8], i);
        atomicMin(&U.first[k], i);
        atomicAdd(&U.count[k], 1);
      }
    }
  };
  // ---- the tokens around it, then all others where a unit is not found whole
  if (lo + tid < hi) take(lo + tid);
  __syncthreads();
  if (tid < WINDOW && U.id[tid] >= 0 && (lo > 0 || hi < L.tokens)) {
    bool whole = U.count[tid] == kUnit8;
#pragma unroll
    for (int k = 0; k < kUnit8; ++k) whole &= U.member[tid][k] >= 0;
    if (!whole && U.first[tid] >= i0) U.open = 1;
  }
  __syncthreads();
  if (U.open) {
    for (int i = tid; i < lo; i += kThreads) take(i);
    for (int i = hi + tid; i < L.tokens; i += kThreads) take(i);
    __syncthreads();
  }
  // ---- a warp a head's keys or values
  const int job = part * kWarps8 + warp;
  if (job >= 2 * L.heads) return;
#pragma unroll 1
  for (int k = 0; k < WINDOW; ++k)
    if (U.id[k] >= 0 && U.first[k] >= i0)
      append_unit<FP16, MODE>(L, U.member[k], U.id[k], job >> 1, job & 1);
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
  const int parts = (2 * L.heads + kWarps8 - 1) / kWarps8;
  const long long kv = windows * parts, q = L.q_heads > 0 ? static_cast<long long>(S.x) * S.y : 0;
  if (kv + q >= (1ll << 31)) return -2;
  const unsigned grid = static_cast<unsigned>(kv + q);
  if (S.each == 4)
    k_append_kv8<FP16, MODE, WINDOW, 4><<<grid, kThreads, 0, s>>>(L, S, static_cast<int>(kv), parts);
  else
    k_append_kv8<FP16, MODE, WINDOW, 1><<<grid, kThreads, 0, s>>>(L, S, static_cast<int>(kv), parts);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}
template <bool FP16, int MODE>
int append_window(const AppendLaunch& L, cudaStream_t s) {
  return L.tokens <= kManyTokens ? append<FP16, MODE, 1>(L, s) : append<FP16, MODE, kUnit8>(L, s);
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
