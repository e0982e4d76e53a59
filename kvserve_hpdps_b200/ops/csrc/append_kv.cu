// New tokens into a paged KV cache, the position rotation applied on the way,
// and rows of a 4-bit cache back out as 16-bit values.
//
// Rotation of a head row x by the token's table row (c, s), rotary size rd:
//   halves:       y[i] = x[i] c[i] - x[i + rd/2] s[i],
//                 y[i + rd/2] = x[i + rd/2] c[i] + x[i] s[i]
//   interleaved:  the same on the pairs (x[2i], x[2i + 1]).
// Everything is computed in fp32 with each operation rounded once (no fused
// multiply-add), so codes equal those of the same formula in plain fp32.
// A 16-bit cache takes the result rounded once; a 4-bit cache (kv4.cuh) takes
// it quantised per group of g channels, without a 16-bit rounding in between:
//   step = T((max - min) (1 / 15)), mid = T(min + 8 step),
//   code = clamp(floor((x - mid) * (1 / step) + 8.5), 0, 15),
// T being the 16-bit type.  Codes are taken against the rounded (step, mid):
// the pair that readers use.  The product with the rounded 1 / 15 is within
// 2^-23 of the quotient, where a division is within 2^-24; T's own half step is
// 2^-11 (fp16) or 2^-8 (bf16) of it, and a division by the number 15 in torch on
// the device is that product too, so that the bytes are those of the formula there.
//
// Eight lanes hold one row: lane l the 16-byte chunks l and l + 8, so a row
// is read with two 16-byte loads a lane, the two halves of a full rotation
// are in the same lane, and a group's extremes are two or three shuffles.
// The table row is read once for all rows that a lane takes.
#include "append_kv.cuh"

namespace kvs {

namespace {

// Extremes of a lane's chunk over the lanes of its group.
KVS_DEV void group_extremes(uint32_t mask, int lanes, float& lo, float& hi) {
  for (int o = 1; o < lanes; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(mask, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(mask, hi, o));
  }
}

// (step, mid) of a group, packed, and the numbers its codes are taken with.
template <bool FP16>
KVS_DEV uint32_t group_meta(float lo, float hi, float& mid, float& inv) {
  uint32_t sb = f2h<FP16>(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f));
  float step = h2f<FP16>(sb);
  if (step < 1.17549435e-38f) {  // 1 / step would overflow: the group is its mid
    sb = 0;
    step = 0.f;
  }
  const uint32_t mb = f2h<FP16>(__fadd_rn(lo, __fmul_rn(8.f, step)));
  mid = h2f<FP16>(mb);
  inv = step == 0.f ? 0.f : __frcp_rn(step);  // 0: every code is 8, the mid
  return sb | (mb << 16);
}

KVS_DEV uint32_t group_codes(const float (&y)[8], float mid, float inv) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float t = __fadd_rn(__fmul_rn(__fsub_rn(y[i], mid), inv), 8.5f);
    t = fminf(fmaxf(t, 0.f), 15.f);  // not a number -> 0; clamped first, the floor is a cut
    w |= static_cast<uint32_t>(t) << (4 * i);
  }
  return w;
}

// Eight lanes store one 4-bit row: y0 / y1 are chunks l and l + 8.
template <bool FP16>
KVS_DEV void store_row4(const AppendLaunch& L, uint8_t* rec, int value, int off, int l,
                        uint32_t mask, const float (&y0)[8], const float (&y1)[8]) {
  const Kv4Record R{L.groups, L.block_size};
  float lo0 = y0[0], hi0 = y0[0], lo1 = y1[0], hi1 = y1[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo0 = min_nan(lo0, y0[i]);
    hi0 = max_nan(hi0, y0[i]);
    lo1 = min_nan(lo1, y1[i]);
    hi1 = max_nan(hi1, y1[i]);
  }
  if (L.groups == 1) {
    lo0 = lo1 = min_nan(lo0, lo1);
    hi0 = hi1 = max_nan(hi0, hi1);
  }
  const int lanes = L.groups == 4 ? 4 : 8;
  group_extremes(mask, lanes, lo0, hi0);
  group_extremes(mask, lanes, lo1, hi1);
  float mid0, inv0, mid1, inv1;
  const uint32_t m0 = group_meta<FP16>(lo0, hi0, mid0, inv0);
  const uint32_t m1 = group_meta<FP16>(lo1, hi1, mid1, inv1);
  const uint32_t w0 = group_codes(y0, mid0, inv0), w1 = group_codes(y1, mid1, inv1);
  // chunk l = 4 q + c is in w0 with q = l / 4, chunk 4 (q + 2) + c in w1; lanes l and l ^ 4 swap
  // one each, so that lanes below 4 hold q = 0, 1 and the others 2, 3: neighbours in the row
  const int c = l & 3, q = l >> 2;
  const uint32_t got = __shfl_xor_sync(mask, q ? w0 : w1, 4);
  const uint32_t a = q ? got : w0, b = q ? w1 : got;
  uint8_t* row = rec + R.codes(value, off) + 16 * c;
  if (!value) {
    *reinterpret_cast<uint2*>(row + 8 * q) = make_uint2(a, b);
  } else {
    *reinterpret_cast<uint32_t*>(row + 4 * q) = __byte_perm(a, b, 0x5410);
    *reinterpret_cast<uint32_t*>(row + 8 + 4 * q) = __byte_perm(a, b, 0x7632);
  }
  uint32_t* meta = reinterpret_cast<uint32_t*>(rec + R.meta(value, off));
  if (L.groups == 4) {
    if (c == 0) {
      meta[q] = m0;
      meta[q + 2] = m1;
    }
  } else if (l == 0) {
    meta[0] = m0;
    if (L.groups == 2) meta[1] = m1;
  }
}

// Rows of a token: q_heads query rows, then key rows, then value rows.
// 16-bit caches: bound by memory, 16384 tokens of 32 + 8 heads in 71 us, 5.7 TB/s or 87% of the
// copy rate.  4-bit caches: by the quantisation's instructions and the loads in front of them, about
// 780 a warp for four rows in 59% of the issue slots (4097 tokens of 28 + 4 heads 20 us, three CTAs
// an SM; 24 us with two).  A decode step of either is one launch, 4.3 us.
template <bool FP16, int MODE, bool FOUR, int EACH>
__global__ void __launch_bounds__(kThreads, 3)
    k_append_kv(const __grid_constant__ AppendLaunch L, const __grid_constant__ Spread S) {
  const int l = threadIdx.x & 7, gi = threadIdx.x >> 3;
  const uint32_t mask = 0xFFu << (threadIdx.x & 24);
  const int t = static_cast<int>(blockIdx.x) * (kGroups / S.across) + gi / S.across;
  if (t >= L.tokens) return;
  const int first = static_cast<int>(blockIdx.y) * S.across * EACH + (gi & (S.across - 1));
  const int rows = L.q_heads + 2 * L.heads;
  if (first >= rows) return;
  bool ok = true, turn = L.pos != nullptr;
  long long pos = 0;
  if (turn) {
    pos = load_index(L.pos, t, L.pos64);
    if (pos < 0 || pos >= L.max_pos) {
      if (l == 0) record_error(L.err, ERR_BOUNDS);
      ok = turn = false;
    }
  }
  long long slot = -1, blk = 0;
  int off = 0;
  if (first + S.across * (EACH - 1) >= L.q_heads) {  // some row is a key or a value
    slot = load_index(L.slots, t, L.slots64);
    if (slot >= L.num_slots) {
      if (l == 0) record_error(L.err, ERR_BOUNDS);
      slot = -1;
    }
    if (!ok) slot = -1;
    if (slot >= 0) {
      blk = L.num_slots < (1ll << 31) ? static_cast<long long>(static_cast<uint32_t>(slot) /
                                                               static_cast<uint32_t>(L.block_size))
                                      : slot / L.block_size;
      off = static_cast<int>(slot - blk * L.block_size);
    }
  }
  const int rd = L.rotary;
  float co[2][8], si[2][8];  // of chunks l and l + 8
  if (turn) load_angles<FP16, MODE>(L, pos, l, co, si);
  uint4 x[EACH][2];
  uint4 partner[MODE == kPart ? EACH : 1][2];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int r = first + S.across * e;
    if (r >= rows) break;
    const int kind = r < L.q_heads ? 0 : r < L.q_heads + L.heads ? 1 : 2;  // query, key, value
    const int h = r - (kind == 0 ? 0 : L.q_heads + (kind - 1) * L.heads);
    if (kind && slot < 0) continue;
    const uint16_t* src =
        static_cast<const uint16_t*>(kind == 0 ? L.query : kind == 1 ? L.key : L.value) +
        t * (kind == 0 ? L.q_ts : kind == 1 ? L.key_ts : L.val_ts) +
        h * (kind == 0 ? L.q_hs : kind == 1 ? L.key_hs : L.val_hs);
    x[e][0] = *reinterpret_cast<const uint4*>(src + 8 * l);
    x[e][1] = *reinterpret_cast<const uint4*>(src + 8 * l + 64);
    if (MODE == kPart && turn && kind < 2) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int ch = 8 * (l + 8 * k);
        if (ch < rd) partner[e][k] = *reinterpret_cast<const uint4*>(src + partner_of(ch, rd));
      }
    }
  }
  if (MODE == kPart) __syncwarp(mask);  // a query rotated in place: all read before any writes
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int r = first + S.across * e;
    if (r >= rows) break;
    const int kind = r < L.q_heads ? 0 : r < L.q_heads + L.heads ? 1 : 2;
    const int h = r - (kind == 0 ? 0 : L.q_heads + (kind - 1) * L.heads);
    if (kind && slot < 0) continue;
    float y[2][8];
    unpack8<FP16>(x[e][0], y[0]);
    unpack8<FP16>(x[e][1], y[1]);
    if (kind < 2 && turn) rotate<FP16, MODE>(rd, l, partner[MODE == kPart ? e : 0], co, si, y);
    uint16_t* dst;
    if (kind == 0) {
      dst = static_cast<uint16_t*>(L.query_out) + t * L.qo_ts + h * L.qo_hs;
    } else if (FOUR) {
      store_row4<FP16>(L, static_cast<uint8_t*>(L.cache) + blk * L.block_stride +
                              h * L.head_stride,
                       kind - 1, off, l, mask, y[0], y[1]);
      continue;
    } else {
      dst = static_cast<uint16_t*>(L.cache) + blk * L.block_stride + (kind - 1) * L.kv_stride +
            off * L.slot_stride + h * L.head_stride;
    }
    *reinterpret_cast<uint4*>(dst + 8 * l) = pack8<FP16>(y[0]);
    *reinterpret_cast<uint4*>(dst + 8 * l + 64) = pack8<FP16>(y[1]);
  }
}

// Eight lanes read one row: key rows of a token, then value rows; slot < 0 reads zeros.  Lane
// 4 hi + c holds the codes of q = 2 hi and 2 hi + 1, i.e. the chunks 8 hi + c and 8 hi + 4 + c.
template <bool FP16, int EACH>
__global__ void __launch_bounds__(kThreads, 3)
    k_read_kv4(const __grid_constant__ Read4Launch L, const __grid_constant__ Spread S) {
  const int l = threadIdx.x & 7, gi = threadIdx.x >> 3, c = l & 3, hi = l >> 2;
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
  const Kv4Record R{L.groups, L.block_size};
  const long long blk = slot < 0 ? 0
                        : L.num_slots < (1ll << 31)
                            ? static_cast<long long>(static_cast<uint32_t>(slot) /
                                                     static_cast<uint32_t>(L.block_size))
                            : slot / L.block_size;
  const int off = slot < 0 ? 0 : static_cast<int>(slot - blk * L.block_size);
  uint2 w[EACH];
  uint32_t m[EACH][2];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int r = first + S.across * e;
    w[e] = make_uint2(0u, 0u);
    m[e][0] = m[e][1] = 0u;
    if (r >= rows || slot < 0) continue;
    const int value = r >= L.heads, h = r - value * L.heads;
    const uint8_t* rec =
        static_cast<const uint8_t*>(L.cache) + blk * L.block_stride + h * L.head_stride;
    const uint8_t* row = rec + R.codes(value, off) + 16 * c;
    const uint32_t* meta = reinterpret_cast<const uint32_t*>(rec + R.meta(value, off));
    if (!value) {
      w[e] = *reinterpret_cast<const uint2*>(row + 8 * hi);
    } else {
      const uint32_t a = *reinterpret_cast<const uint32_t*>(row + 4 * hi);
      const uint32_t b = *reinterpret_cast<const uint32_t*>(row + 8 + 4 * hi);
      w[e] = make_uint2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
    }
    m[e][0] = meta[L.groups == 4 ? 2 * hi : L.groups == 2 ? hi : 0];
    m[e][1] = L.groups == 4 ? meta[2 * hi + 1] : m[e][0];
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int r = first + S.across * e;
    if (r >= rows) break;
    const int value = r >= L.heads, h = r - value * L.heads;
    uint16_t* out = static_cast<uint16_t*>(L.out) +
                    ((static_cast<long long>(value) * L.tokens + t) * L.heads + h) * 128 +
                    64 * hi + 8 * c;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t x = k ? w[e].y : w[e].x;
      const float step = h2f<FP16>(m[e][k] & 0xFFFFu), mid = h2f<FP16>(m[e][k] >> 16);
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float code = static_cast<float>(static_cast<int>((x >> (4 * i)) & 15u) - 8);
        y[i] = __fadd_rn(mid, __fmul_rn(code, step));
      }
      *reinterpret_cast<uint4*>(out + 32 * k) = pack8<FP16>(y);
    }
  }
}

template <bool FP16, int MODE, bool FOUR>
void append(const AppendLaunch& L, const Spread& S, cudaStream_t s) {
  if (S.each == 4)
    k_append_kv<FP16, MODE, FOUR, 4><<<dim3(S.x, S.y), kThreads, 0, s>>>(L, S);
  else
    k_append_kv<FP16, MODE, FOUR, 1><<<dim3(S.x, S.y), kThreads, 0, s>>>(L, S);
}
template <bool FP16, bool FOUR>
void append_mode(const AppendLaunch& L, const Spread& S, cudaStream_t s) {
  if (L.pos == nullptr || (!L.interleaved && L.rotary == 128))
    append<FP16, kHalves, FOUR>(L, S, s);
  else if (L.interleaved)
    append<FP16, kPairs, FOUR>(L, S, s);
  else
    append<FP16, kPart, FOUR>(L, S, s);
}
template <bool FP16>
void append_cache(const AppendLaunch& L, const Spread& S, cudaStream_t s) {
  if (L.groups)
    append_mode<FP16, true>(L, S, s);
  else
    append_mode<FP16, false>(L, S, s);
}
template <bool FP16>
void read(const Read4Launch& L, const Spread& S, cudaStream_t s) {
  if (S.each == 4)
    k_read_kv4<FP16, 4><<<dim3(S.x, S.y), kThreads, 0, s>>>(L, S);
  else
    k_read_kv4<FP16, 1><<<dim3(S.x, S.y), kThreads, 0, s>>>(L, S);
}

}  // namespace
}  // namespace kvs

using namespace kvs;

extern "C" {

int kvs_append_kv(const AppendLaunch* L, void* stream) {
  if (L->tokens <= 0 || L->q_heads + L->heads <= 0) return 0;
  const Spread S = spread_of(L->tokens, L->q_heads + 2 * L->heads);
  if (S.y > 65535u) return -2;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (L->fp16)
    append_cache<true>(*L, S, s);
  else
    append_cache<false>(*L, S, s);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}

int kvs_read_kv4(const Read4Launch* L, void* stream) {
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
