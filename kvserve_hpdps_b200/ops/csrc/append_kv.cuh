// Rows of a step's new tokens, read and rotated: shared by the kernels that append them to
// 16-bit and 4-bit caches (append_kv.cu) and to 8-bit ones (append_kv8.cu).
//
// Eight lanes hold one row: lane l the 16-byte chunks l and l + 8.
#pragma once

#include "kv4.cuh"

namespace kvs {

namespace {

constexpr int kThreads = 256;
constexpr int kGroups = kThreads / 8;  // rows that a CTA has in hand at once

// How the rows of a launch are dealt out: `across` groups of eight lanes side
// by side on one token, each taking rows across, 2 across, ... further on, `each` in all.
struct Spread {
  int across, each;
  unsigned x, y;  // grid: tokens, row blocks
};
// Few rows: one a group, so that all SMs take part.  Many: four a group,
// whose loads are in flight together and which share the table row.
Spread spread_of(int tokens, int rows) {
  Spread s;
  const bool many = static_cast<long long>(tokens) * rows >= 148ll * 8 * kGroups;
  s.each = many ? 4 : 1;
  s.across = 1;
  while (s.across < kGroups && s.across * s.each < rows) s.across *= 2;
  if (many && s.across > 4) s.across = 4;
  const int per_cta = kGroups / s.across;
  s.x = static_cast<unsigned>((tokens + per_cta - 1) / per_cta);
  s.y = static_cast<unsigned>((rows + s.across * s.each - 1) / (s.across * s.each));
  return s;
}

// kHalves: full rotation of halves, both in one lane.  kPart: halves of fewer
// channels, whose partners are loaded too.  kPairs: adjacent channels.
enum Mode { kHalves, kPart, kPairs };

// Eight (halves) or four (pairs) table values from column `col` on; both are
// 16-byte multiples because rd is a multiple of 16.
template <bool FP16>
KVS_DEV void load_table(const AppendLaunch& L, long long at, int n, float (&x)[8]) {
  if (L.table32) {
    const float4* t = reinterpret_cast<const float4*>(static_cast<const float*>(L.table) + at);
    const float4 a = t[0], b = n > 4 ? t[1] : a;
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
    x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint2* t = reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(L.table) + at);
    const uint2 a = t[0], b = n > 4 ? t[1] : a;
    unpack8<FP16>(make_uint4(a.x, a.y, b.x, b.y), x);
  }
}

// A token's cosines and sines for chunks l and l + 8.
template <bool FP16, int MODE>
KVS_DEV void load_angles(const AppendLaunch& L, long long pos, int l, float (&co)[2][8],
                         float (&si)[2][8]) {
  const int rd = L.rotary, half = rd >> 1;
  const long long row = pos * L.table_stride;
  if (MODE == kHalves) {
    load_table<FP16>(L, row + 8 * l, 8, co[0]);
    load_table<FP16>(L, row + 64 + 8 * l, 8, si[0]);
  } else {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int ch = 8 * (l + 8 * k);
      if (ch < rd) {
        const int col = MODE == kPairs ? ch / 2 : ch < half ? ch : ch - half;
        load_table<FP16>(L, row + col, MODE == kPairs ? 4 : 8, co[k]);
        load_table<FP16>(L, row + half + col, MODE == kPairs ? 4 : 8, si[k]);
      }
    }
  }
}

// Where a chunk's partners lie when halves of fewer than 128 channels are rotated.
KVS_DEV int partner_of(int ch, int rd) { return ch < rd >> 1 ? ch + (rd >> 1) : ch - (rd >> 1); }

// Chunks l and l + 8 of a row, rotated; `partner` is for kPart alone.
template <bool FP16, int MODE>
KVS_DEV void rotate(int rd, int l, const uint4 (&partner)[2], const float (&co)[2][8],
                    const float (&si)[2][8], float (&y)[2][8]) {
  if (MODE == kHalves) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = y[0][i], b = y[1][i];
      y[0][i] = __fsub_rn(__fmul_rn(a, co[0][i]), __fmul_rn(b, si[0][i]));
      y[1][i] = __fadd_rn(__fmul_rn(b, co[0][i]), __fmul_rn(a, si[0][i]));
    }
  } else {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int ch = 8 * (l + 8 * k);
      if (ch >= rd) continue;
      if (MODE == kPairs) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a = y[k][2 * i], b = y[k][2 * i + 1];
          y[k][2 * i] = __fsub_rn(__fmul_rn(a, co[k][i]), __fmul_rn(b, si[k][i]));
          y[k][2 * i + 1] = __fadd_rn(__fmul_rn(b, co[k][i]), __fmul_rn(a, si[k][i]));
        }
      } else {
        float p[8];
        unpack8<FP16>(partner[k], p);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float u = __fmul_rn(y[k][i], co[k][i]), v = __fmul_rn(p[i], si[k][i]);
          y[k][i] = ch < (rd >> 1) ? __fsub_rn(u, v) : __fadd_rn(u, v);
        }
      }
    }
  }
}

}  // namespace
}  // namespace kvs
