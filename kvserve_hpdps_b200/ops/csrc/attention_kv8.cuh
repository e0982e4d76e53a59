// What the attention kernels over an 8-bit cache share.
#pragma once

#include "attention_kv4.cuh"
#include "kv8.cuh"
#include "tensor_map.h"

namespace kvs {

namespace {

// Rows of records as the copy engine sees them: 128 bytes, 2 bs + 1 rows, heads, blocks; boxes of
// `rows` rows, 16-byte chunks swizzled by the row.
inline bool record_map(const Attn4Launch& L, unsigned rows, CUtensorMap* map) {
  const EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t record = 128ull * (2 * L.block_size + 1);
  // A cache without blocks has no address; the encoder wants one and a block, which no id names.
  const bool none = L.num_blocks == 0;
  const cuuint64_t dims[4] = {128, 2ull * L.block_size + 1, static_cast<cuuint64_t>(L.heads),
                              none ? 1 : static_cast<cuuint64_t>(L.num_blocks)};
  // a stride that nothing is multiplied by may be anything in torch
  const cuuint64_t strides[3] = {128,
                                 L.heads > 1 ? static_cast<cuuint64_t>(L.head_stride) : record,
                                 L.num_blocks > 1 ? static_cast<cuuint64_t>(L.block_stride) : record};
  const cuuint32_t box[4] = {128, rows, 1, 1}, step[4] = {1, 1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, none ? L.out : const_cast<void*>(L.cache), dims,
            strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Bytes that a phase waits for, beside its arrivals.
KVS_DEV void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)),
               "r"(bytes)
               : "memory");
}
KVS_DEV void load_rows(uint32_t dst, const CUtensorMap* map, int row, int head, int block,
                       uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row), "r"(head), "r"(block),
      "r"(smem_u32(bar))
      : "memory");
}

// Joins the parts of the items that several CTAs (or teams of one) share.  A part's weights are
// relative to its own maximum; they are added up in order, so results do not depend on timing.
//
// Few parts an item (many items): CTA b takes the item that begins with team b and goes on, if one
// does, a warp a row.  Many parts (DEEP; few items, which the host knows): the CTAs of column i look for
// the i-th of them and take a row each, 16 warps every 16th part.  One sequence of 49157 tokens, 4
// heads, 97 parts each: 17 us with four warps a row and a CTA a team, of which most found nothing.
template <bool FP16, int ROWS, bool DEEP>
__global__ void __launch_bounds__(DEEP ? 512 : 256)
    k_attn8_join(const __grid_constant__ Attn4Launch L, int B) {
  constexpr int WARPS = DEEP ? 16 : 8;
  __shared__ int s_count[WARPS], s_b;
  __shared__ float2 s_ml[DEEP ? WARPS : 1];
  __shared__ float4 s_o[DEEP ? WARPS : 1][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Parts P = parts(L.scratch, B, ROWS);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int b = blockIdx.x;
  if constexpr (DEEP) {
    int base = 0;  // items found
    for (int b0 = 0; b0 < B; b0 += 32 * WARPS) {
      const bool is = b0 + tid < B && P.desc[b0 + tid].x >= 0;
      const uint32_t mask = __ballot_sync(0xFFFFFFFFu, is);
      if (tid == 0) s_b = -1;
      if (lane == 0) s_count[warp] = __popc(mask);
      __syncthreads();
      int before = base;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        if (w < warp) before += s_count[w];
        base += s_count[w];
      }
      if (is && before + __popc(mask & ((1u << lane) - 1)) == static_cast<int>(blockIdx.x))
        s_b = b0 + tid;
      __syncthreads();
      b = s_b;
      if (b >= 0) break;
      __syncthreads();
    }
    if (b < 0) return;
  }
  const int row = DEEP ? static_cast<int>(blockIdx.y) : static_cast<int>(blockIdx.y) * 8 + warp;
  // part 0 is in team b's second slot, the others in the first ones of the next teams
  auto slot = [&](int i) { return (i == 0 ? 2 * b + 1 : 2 * (b + i)) * ROWS + row; };
  float2 ml[4];
  float4 x[4];
  auto load = [&](int u, int i, bool is) {
    ml[u] = make_float2(kLowest, 0.f);
    x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (is) {
      ml[u] = P.ml[slot(i)];
      x[u] = *reinterpret_cast<const float4*>(P.o + slot(i) * 128ll + lane * 4);
    }
  };
  // most items have two parts: theirs come together with what says so
  if constexpr (!DEEP) {
    load(0, 0, true);
    load(1, 1, b + 1 < B);
  }
  const int4 d = P.desc[b];
  if (d.x < 0) return;
  const int group = L.q_heads / L.heads, np = d.w & 0xFFFF;
  if (row >= d.w >> 16) return;
  float m = kLowest, ls = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float m2, float l2, const float4& x) {
    const float top = fmaxf(m, m2), k1 = ex2(m - top), k2 = ex2(m2 - top);
    m = top;
    ls = fmaf(ls, k1, l2 * k2);
    a.x = fmaf(a.x, k1, x.x * k2);
    a.y = fmaf(a.y, k1, x.y * k2);
    a.z = fmaf(a.z, k1, x.z * k2);
    a.w = fmaf(a.w, k1, x.w * k2);
  };
  if constexpr (!DEEP) {
#pragma unroll
    for (int u = 0; u < 2; ++u) add(ml[u].x, ml[u].y, x[u]);
  }
  for (int i0 = DEEP ? warp : 2; i0 < np; i0 += DEEP ? 4 * WARPS : 4) {  // four loads together
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + (DEEP ? WARPS : 1) * u;
      load(u, i, i < np);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) add(ml[u].x, ml[u].y, x[u]);
  }
  if constexpr (DEEP) {
    s_o[warp][lane] = a;
    if (lane == 0) s_ml[warp] = make_float2(m, ls);
    __syncthreads();
    if (warp != 0) return;
#pragma unroll 4
    for (int w = 1; w < WARPS; ++w) add(s_ml[w].x, s_ml[w].y, s_o[w][lane]);
  }
  const int rr = d.z * ROWS + row;
  const long long tq = d.x + rr / group;
  const int hq = d.y * group + rr % group;
  const float inv = ls == 0.f ? 0.f : __fdividef(1.f, ls);
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(L.out) + tq * L.o_ts + hq * L.o_hs + lane * 4) =
      make_uint2(f2h2<FP16>(a.x * inv, a.y * inv), f2h2<FP16>(a.z * inv, a.w * inv));
  if (L.lse != nullptr && lane == 0)
    L.lse[tq * L.q_heads + hq] = ls == 0.f ? -INFINITY : (m + log2f(ls)) * 0.69314718055994531f;
}

template <bool FP16, int ROWS>
cudaError_t launch_join(const Attn4Launch& L, int teams, long long items, cudaStream_t s) {
  // a row a CTA pays while there are two rounds of them at most (16 items of 256 rows, 9 parts each:
  // 61 us a call against 44)
  const bool deep = 8 * items <= teams && items * ROWS <= 1184;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = deep ? dim3(static_cast<unsigned>(items), ROWS) : dim3(teams, ROWS / 8);
  cfg.blockDim = dim3(deep ? 512 : 256);
  cfg.stream = s;
  cudaLaunchAttribute attr = {};  // it may start while the attention kernel ends
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return deep ? cudaLaunchKernelEx(&cfg, k_attn8_join<FP16, ROWS, true>, L, teams)
              : cudaLaunchKernelEx(&cfg, k_attn8_join<FP16, ROWS, false>, L, teams);
}

}  // namespace

// attention_kv8_tile.cu: many query rows a sequence.
cudaError_t attn8_tile_launch(const Attn4Launch& L, const CUtensorMap& map, cudaStream_t s);
long long attn8_tile_scratch(const Attn4Launch& L);

}  // namespace kvs
