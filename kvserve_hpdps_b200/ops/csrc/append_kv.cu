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
//   step = T((max - min) / 15), mid = T(min + 8 step),
//   code = clamp(floor((x - mid) * (1 / step) + 8.5), 0, 15),
// T being the 16-bit type.  Codes are taken against the rounded (step, mid):
// the pair that readers use.
//
// Eight lanes hold one row: lane l the 16-byte chunks l and l + 8, so a row
// is read with two 16-byte loads a lane, the two halves of a full rotation
// are in the same lane, and a group's extremes are two or three shuffles.
#include "kv4.cuh"

namespace kvs {

namespace {

constexpr int kAppendThreads = 256;

// cos / sin of the 8 (halves) or 4 (interleaved) table columns from `col` on.
template <bool FP16>
KVS_DEV void load_table(const AppendLaunch& L, long long row, int col, int n, float (&x)[8]) {
  const long long at = row * L.table_stride + col;
  for (int i = 0; i < 8; ++i) x[i] = 0.f;
  if (L.table32) {
    const float* t = static_cast<const float*>(L.table) + at;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) x[i] = t[i];
  } else {
    const uint16_t* t = static_cast<const uint16_t*>(L.table) + at;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) x[i] = h2f<FP16>(t[i]);
  }
}

// Chunk `c` (channels 8c..8c+7) of a row at `src`, rotated.
template <bool FP16>
KVS_DEV void rotated_chunk(const AppendLaunch& L, const uint16_t* src, long long row, int c,
                           float (&y)[8]) {
  float x[8];
  unpack8<FP16>(*reinterpret_cast<const uint4*>(src + 8 * c), x);
  const int rd = L.rotary, half = rd >> 1;
  if (8 * c >= rd) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i];
    return;
  }
  float co[8], si[8];
  if (L.interleaved) {
    load_table<FP16>(L, row, 4 * c, 4, co);
    load_table<FP16>(L, row, half + 4 * c, 4, si);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = x[2 * i], b = x[2 * i + 1];
      y[2 * i] = __fsub_rn(__fmul_rn(a, co[i]), __fmul_rn(b, si[i]));
      y[2 * i + 1] = __fadd_rn(__fmul_rn(b, co[i]), __fmul_rn(a, si[i]));
    }
    return;
  }
  const bool first = 8 * c < half;
  const int col = first ? 8 * c : 8 * c - half;
  float p[8];
  unpack8<FP16>(*reinterpret_cast<const uint4*>(src + (first ? 8 * c + half : 8 * c - half)), p);
  load_table<FP16>(L, row, col, 8, co);
  load_table<FP16>(L, row, half + col, 8, si);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float u = __fmul_rn(x[i], co[i]), v = __fmul_rn(p[i], si[i]);
    y[i] = first ? __fsub_rn(u, v) : __fadd_rn(u, v);
  }
}

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
  uint32_t sb = f2h<FP16>(__fdiv_rn(__fsub_rn(hi, lo), 15.f));
  float step = h2f<FP16>(sb);
  if (step < 1.17549435e-38f) {  // 1 / step would overflow: the group is its mid
    sb = 0;
    step = 0.f;
  }
  const uint32_t mb = f2h<FP16>(__fadd_rn(lo, __fmul_rn(8.f, step)));
  mid = h2f<FP16>(mb);
  inv = step == 0.f ? 0.f : __fdiv_rn(1.f, step);  // 0: every code is 8, the mid
  return sb | (mb << 16);
}

KVS_DEV uint32_t group_codes(const float (&y)[8], float mid, float inv) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float t = floorf(__fadd_rn(__fmul_rn(__fsub_rn(y[i], mid), inv), 8.5f));
    t = fminf(fmaxf(t, 0.f), 15.f);  // not a number -> 0
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
  uint8_t* row = rec + R.codes(value, off);
  const int c = l & 3, q = l >> 2;  // chunk l = 4 q + c, chunk l + 8 = 4 (q + 2) + c
  if (!value) {
    *reinterpret_cast<uint32_t*>(row + 16 * c + 4 * q) = w0;
    *reinterpret_cast<uint32_t*>(row + 16 * c + 4 * q + 8) = w1;
  } else {
    *reinterpret_cast<uint16_t*>(row + 16 * c + 2 * q) = static_cast<uint16_t>(w0);
    *reinterpret_cast<uint16_t*>(row + 16 * c + 8 + 2 * q) = static_cast<uint16_t>(w0 >> 16);
    *reinterpret_cast<uint16_t*>(row + 16 * c + 2 * q + 4) = static_cast<uint16_t>(w1);
    *reinterpret_cast<uint16_t*>(row + 16 * c + 8 + 2 * q + 4) = static_cast<uint16_t>(w1 >> 16);
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

// Rows of token t: q_heads query rows, then key rows, then value rows.
template <bool FP16>
__global__ void __launch_bounds__(kAppendThreads) k_append_kv(const __grid_constant__ AppendLaunch L) {
  const int l = threadIdx.x & 7;
  const uint32_t mask = 0xFFu << (threadIdx.x & 24);
  const int rows = L.q_heads + 2 * L.heads;
  const long long item =
      (static_cast<long long>(blockIdx.x) * kAppendThreads + threadIdx.x) >> 3;
  if (item >= static_cast<long long>(L.tokens) * rows) return;
  const int t = static_cast<int>(item / rows);
  int r = static_cast<int>(item - static_cast<long long>(t) * rows);
  long long pos = 0;
  bool ok = true, turn = L.pos != nullptr;
  if (turn) {
    pos = load_index(L.pos, t, L.pos64);
    if (pos < 0 || pos >= L.max_pos) {
      if (l == 0) record_error(L.err, ERR_BOUNDS);
      ok = turn = false;
    }
  }
  const bool query = r < L.q_heads;
  const int kind = query ? 0 : (r - L.q_heads) / L.heads + 1;  // 0 query, 1 key, 2 value
  const int h = query ? r : (r - L.q_heads) % L.heads;
  const uint16_t* src =
      static_cast<const uint16_t*>(kind == 0 ? L.query : kind == 1 ? L.key : L.value) +
      t * (kind == 0 ? L.q_ts : kind == 1 ? L.key_ts : L.val_ts) +
      h * (kind == 0 ? L.q_hs : kind == 1 ? L.key_hs : L.val_hs);
  long long slot = 0;
  if (kind) {
    slot = load_index(L.slots, t, L.slots64);
    if (slot >= L.num_slots) {
      if (l == 0) record_error(L.err, ERR_BOUNDS);
      return;
    }
    if (slot < 0 || !ok) return;
  }
  float y0[8], y1[8];
  if (kind < 2 && turn) {
    rotated_chunk<FP16>(L, src, pos, l, y0);
    rotated_chunk<FP16>(L, src, pos, l + 8, y1);
  } else {
    unpack8<FP16>(*reinterpret_cast<const uint4*>(src + 8 * l), y0);
    unpack8<FP16>(*reinterpret_cast<const uint4*>(src + 8 * l + 64), y1);
  }
  __syncwarp(mask);  // a query rotated in place: every lane has read before any writes
  uint16_t* dst;
  if (kind == 0) {
    dst = static_cast<uint16_t*>(L.query_out) + t * L.qo_ts + h * L.qo_hs;
  } else {
    const long long blk = slot / L.block_size;
    const int off = static_cast<int>(slot - blk * L.block_size);
    if (L.groups) {
      store_row4<FP16>(L, static_cast<uint8_t*>(L.cache) + blk * L.block_stride +
                              h * L.head_stride,
                       kind - 1, off, l, mask, y0, y1);
      return;
    }
    dst = static_cast<uint16_t*>(L.cache) + blk * L.block_stride + (kind - 1) * L.kv_stride +
          off * L.slot_stride + h * L.head_stride;
  }
  *reinterpret_cast<uint4*>(dst + 8 * l) = pack8<FP16>(y0);
  *reinterpret_cast<uint4*>(dst + 8 * l + 64) = pack8<FP16>(y1);
}

// Eight lanes read one row (plane, token, head); slot < 0 reads zeros.
template <bool FP16>
__global__ void __launch_bounds__(kAppendThreads) k_read_kv4(const __grid_constant__ Read4Launch L) {
  const int l = threadIdx.x & 7;
  const long long item =
      (static_cast<long long>(blockIdx.x) * kAppendThreads + threadIdx.x) >> 3;
  const long long plane = static_cast<long long>(L.tokens) * L.heads;
  if (item >= 2 * plane) return;
  const int value = item >= plane;
  const long long th = item - value * plane;
  const int t = static_cast<int>(th / L.heads), h = static_cast<int>(th % L.heads);
  const long long slot = load_index(L.slots, t, L.slots64);
  uint16_t* out = static_cast<uint16_t*>(L.out) + item * 128;
  float y0[8], y1[8];
  if (slot < 0 || slot >= L.num_slots) {
    if (l == 0 && slot >= 0) record_error(L.err, ERR_BOUNDS);
#pragma unroll
    for (int i = 0; i < 8; ++i) y0[i] = y1[i] = 0.f;
  } else {
    const Kv4Record R{L.groups, L.block_size};
    const long long blk = slot / L.block_size;
    const int off = static_cast<int>(slot - blk * L.block_size);
    const uint8_t* rec =
        static_cast<const uint8_t*>(L.cache) + blk * L.block_stride + h * L.head_stride;
    const uint8_t* row = rec + R.codes(value, off);
    const uint32_t* meta = reinterpret_cast<const uint32_t*>(rec + R.meta(value, off));
    const int c = l & 3, q = l >> 2;
    uint32_t w0, w1;
    if (!value) {
      w0 = *reinterpret_cast<const uint32_t*>(row + 16 * c + 4 * q);
      w1 = *reinterpret_cast<const uint32_t*>(row + 16 * c + 4 * q + 8);
    } else {
      const uint16_t* p = reinterpret_cast<const uint16_t*>(row + 16 * c + 2 * q);
      w0 = p[0] | (static_cast<uint32_t>(p[4]) << 16);
      w1 = p[2] | (static_cast<uint32_t>(p[6]) << 16);
    }
    const uint32_t m0 = meta[L.groups == 4 ? q : 0];
    const uint32_t m1 = meta[L.groups == 4 ? q + 2 : L.groups - 1];
    const float s0 = h2f<FP16>(m0 & 0xFFFFu), mid0 = h2f<FP16>(m0 >> 16);
    const float s1 = h2f<FP16>(m1 & 0xFFFFu), mid1 = h2f<FP16>(m1 >> 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c0 = static_cast<float>(static_cast<int>((w0 >> (4 * i)) & 15u) - 8);
      const float c1 = static_cast<float>(static_cast<int>((w1 >> (4 * i)) & 15u) - 8);
      y0[i] = __fadd_rn(mid0, __fmul_rn(c0, s0));
      y1[i] = __fadd_rn(mid1, __fmul_rn(c1, s1));
    }
  }
  *reinterpret_cast<uint4*>(out + 8 * l) = pack8<FP16>(y0);
  *reinterpret_cast<uint4*>(out + 8 * l + 64) = pack8<FP16>(y1);
}

}  // namespace
}  // namespace kvs

using namespace kvs;

extern "C" {

int kvs_append_kv(const AppendLaunch* L, void* stream) {
  const long long items = static_cast<long long>(L->tokens) * (L->q_heads + 2 * L->heads);
  if (items <= 0) return 0;
  const long long blocks = (items * 8 + kAppendThreads - 1) / kAppendThreads;
  if (blocks > 0x7FFFFFFFll) return -2;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (L->fp16)
    k_append_kv<true><<<static_cast<unsigned>(blocks), kAppendThreads, 0, s>>>(*L);
  else
    k_append_kv<false><<<static_cast<unsigned>(blocks), kAppendThreads, 0, s>>>(*L);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}

int kvs_read_kv4(const Read4Launch* L, void* stream) {
  const long long items = 2ll * L->tokens * L->heads;
  if (items <= 0) return 0;
  const long long blocks = (items * 8 + kAppendThreads - 1) / kAppendThreads;
  if (blocks > 0x7FFFFFFFll) return -2;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (L->fp16)
    k_read_kv4<true><<<static_cast<unsigned>(blocks), kAppendThreads, 0, s>>>(*L);
  else
    k_read_kv4<false><<<static_cast<unsigned>(blocks), kAppendThreads, 0, s>>>(*L);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}

}  // extern "C"
