// Rows of a paged KV cache held in 4 bits: layout and arithmetic shared by the
// kernels that write, read and attend over them.
//
// A (block, head) record of a cache with block size bs and ng = 128 / g
// channel groups holds, in this order,
//   K codes  [bs][64 B]      V codes  [bs][64 B]
//   K meta   [bs][ng][4 B]   V meta   [bs][ng][4 B]
// so one record is contiguous, and 16 consecutive tokens of each part are
// contiguous 16-byte multiples.  A group's metadata is (step, mid), two
// floats of the cache's 16-bit type; a channel reads
//   value = mid + (code - 8) * step,  code in [0, 15].
//
// Code order.  The attention kernels make matrix operands from these bytes
// pair by pair with one AND-OR and one fused multiply-add (and a shift for
// every second pair), so channels are placed where their fragments want
// them.  With channel d = 32 q + r:
//   K: r = 8 c + i: nibble i of the 32-bit word at byte 16 c + 4 q;
//   V: r = 4 j + i: nibble i of the 16-bit word at byte 8 j + 2 q.
#pragma once

#include "common.cuh"
#include "kvs_types.h"

namespace kvs {

struct Kv4Record {
  int ng, bs;
  KVS_DEV long long codes(int value, int off) const {
    return static_cast<long long>(value * bs + off) * 64;
  }
  KVS_DEV long long meta(int value, int off) const {
    return 128ll * bs + static_cast<long long>(value * bs + off) * ng * 4;
  }
};

// 16-bit types.
template <bool FP16>
KVS_DEV float h2f(uint32_t bits) {
  if constexpr (FP16) return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
  return __uint_as_float(bits << 16);
}
template <bool FP16>
KVS_DEV uint32_t f2h(float x) {
  if constexpr (FP16) return __half_as_ushort(__float2half_rn(x));
  return __bfloat16_as_ushort(__float2bfloat16_rn(x));
}
template <bool FP16>
KVS_DEV uint32_t f2h2(float lo, float hi) {
  if constexpr (FP16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  return cvt_bf16x2(lo, hi);
}
template <bool FP16>
KVS_DEV void unpack8(const uint4& u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = h2f<FP16>(w[i] & 0xFFFFu);
    x[2 * i + 1] = h2f<FP16>(w[i] >> 16);
  }
}
template <bool FP16>
KVS_DEV uint4 pack8(const float (&x)[8]) {
  return make_uint4(f2h2<FP16>(x[0], x[1]), f2h2<FP16>(x[2], x[3]), f2h2<FP16>(x[4], x[5]),
                    f2h2<FP16>(x[6], x[7]));
}

// min / max that return NaN when either operand is NaN, so that a group that
// holds one reads back as NaN instead of hiding it.
KVS_DEV float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
KVS_DEV float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

KVS_DEV long long load_index(const void* p, int i, int wide) {
  return wide ? static_cast<const long long*>(p)[i]
              : static_cast<long long>(static_cast<const int*>(p)[i]);
}

}  // namespace kvs
