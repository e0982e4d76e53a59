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
  const cuuint64_t dims[4] = {128, 2ull * L.block_size + 1, static_cast<cuuint64_t>(L.heads),
                              static_cast<cuuint64_t>(L.num_blocks)};
  // a stride that nothing is multiplied by may be anything in torch
  const cuuint64_t strides[3] = {128,
                                 L.heads > 1 ? static_cast<cuuint64_t>(L.head_stride) : record,
                                 L.num_blocks > 1 ? static_cast<cuuint64_t>(L.block_stride) : record};
  const cuuint32_t box[4] = {128, rows, 1, 1}, step[4] = {1, 1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(L.cache), dims, strides, box,
            step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
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

}  // namespace

// attention_kv8_tile.cu: many query rows a sequence.
cudaError_t attn8_tile_launch(const Attn4Launch& L, const CUtensorMap& map, cudaStream_t s);
long long attn8_tile_scratch(const Attn4Launch& L);

}  // namespace kvs
