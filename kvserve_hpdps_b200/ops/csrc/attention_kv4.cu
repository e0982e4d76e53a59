// Attention over a paged KV cache held in 4 bits (kv4.cuh has the layout).
//
// With n query rows of a sequence whose cache holds `len` tokens, row i sees
// keys j < len - n + i + 1.  Over a group g of channels,
//   q . k_j = sum_g [ step_jg * (sum_d q_d code_jd - 8 Q_g) + mid_jg * Q_g ],
// Q_g = sum of q over the group; likewise the output is
//   o_d = (sum_j p_j (mid_jg + (code_jd - 8) step_jg)) / sum_j p_j.
// A row that sees no key returns zeros and lse = -inf.
//
// k_attn4_simple: one warp a (row, head), four channels a lane, one pass over
// the keys with the running maximum and sum.
#include "kv4.cuh"

namespace kvs {

namespace {

struct Seq {
  int row0, n, len;  // first query row, query rows, cached tokens
};

// The sequence's extents, held to what the launch's arrays cover.
KVS_DEV Seq sequence(const Attn4Launch& L, int r, bool report) {
  Seq s;
  int end;
  if (L.start != nullptr) {
    s.row0 = L.start[r];
    end = L.start[r + 1];
  } else {
    s.row0 = r;
    end = r + 1;
  }
  s.n = end - s.row0;
  s.len = L.lens[r];
  const long long cap = static_cast<long long>(L.table_cols) * L.block_size;
  const bool bad = s.row0 < 0 || end < s.row0 || end > L.tokens || s.n > L.max_q || s.len < 0 ||
                   s.len > cap;
  if (bad) {
    if (report) record_error(L.err, ERR_BOUNDS);
    s.n = 0;
  }
  return s;
}

template <bool FP16>
__global__ void __launch_bounds__(128) k_attn4_simple(const __grid_constant__ Attn4Launch L) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = blockIdx.y, i = blockIdx.x / L.q_heads, hq = blockIdx.x % L.q_heads;
  const int group = L.q_heads / L.heads, h = hq / group;
  const Seq s = sequence(L, r, threadIdx.x == 0);
  if (i >= s.n) return;
  const long long t = s.row0 + i;
  const Kv4Record R{L.groups, L.block_size};
  const int q = lane >> 3, j = lane & 7, ch = 32 * q + 4 * j;  // the lane's four channels
  const int grp = ch / (128 / L.groups);
  const uint16_t* qp = static_cast<const uint16_t*>(L.q) + t * L.q_ts + hq * L.q_hs + ch;
  float qv[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, sum = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) qv[k] = h2f<FP16>(qp[k]) * L.scale;
  const int seen = s.len - s.n + i + 1;
  for (int tok = warp; tok < seen; tok += 4) {
    const int blk = L.table[r * L.table_stride + tok / L.block_size];
    if (blk < 0 || blk >= L.num_blocks) {
      if (lane == 0) record_error(L.err, ERR_BOUNDS);
      continue;
    }
    const int off = tok % L.block_size;
    const uint8_t* rec = static_cast<const uint8_t*>(L.cache) + blk * L.block_stride +
                         h * L.head_stride;
    const uint32_t kc = *reinterpret_cast<const uint16_t*>(rec + R.codes(0, off) + 16 * (j >> 1) +
                                                           4 * q + 2 * (j & 1));
    const uint32_t vc = *reinterpret_cast<const uint16_t*>(rec + R.codes(1, off) + 8 * j + 2 * q);
    const uint32_t km = reinterpret_cast<const uint32_t*>(rec + R.meta(0, off))[grp];
    const uint32_t vm = reinterpret_cast<const uint32_t*>(rec + R.meta(1, off))[grp];
    float dot = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      dot += qv[k] * (h2f<FP16>(km >> 16) +
                      (static_cast<float>((kc >> (4 * k)) & 15u) - 8.f) * h2f<FP16>(km & 0xFFFFu));
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, x);
    const float mn = fmaxf(m, dot), p = __expf(dot - mn), f = __expf(m - mn);
    m = mn;
    sum = sum * f + p;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      o[k] = o[k] * f +
             p * (h2f<FP16>(vm >> 16) +
                  (static_cast<float>((vc >> (4 * k)) & 15u) - 8.f) * h2f<FP16>(vm & 0xFFFFu));
  }
  __shared__ float sm[4], ss[4], so[4][128];
  if (lane == 0) {
    sm[warp] = m;
    ss[warp] = sum;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) so[warp][ch + k] = o[k];
  __syncthreads();
  const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float total = 0.f, acc = 0.f;
  if (!(top == -INFINITY)) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = sm[w] == -INFINITY ? 0.f : __expf(sm[w] - top);
      total += ss[w] * f;
      acc += so[w][threadIdx.x] * f;
    }
    acc /= total;
  }
  static_cast<uint16_t*>(L.out)[t * L.o_ts + hq * L.o_hs + threadIdx.x] =
      static_cast<uint16_t>(f2h<FP16>(acc));
  if (L.lse != nullptr && threadIdx.x == 0)
    L.lse[t * L.q_heads + hq] = top == -INFINITY ? -INFINITY : top + logf(total);
}

}  // namespace
}  // namespace kvs

using namespace kvs;

extern "C" {

int kvs_attn4_launch_size(void) { return static_cast<int>(sizeof(Attn4Launch)); }

long long kvs_attn4_scratch_bytes(const Attn4Launch*) { return 0; }

int kvs_attention_kv4(const Attn4Launch* L, void* stream) {
  if (L->seqs <= 0 || L->max_q <= 0 || L->tokens <= 0) return 0;
  if (L->seqs > 65535) return -2;
  const dim3 grid(static_cast<unsigned>(L->max_q) * L->q_heads, L->seqs);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (L->fp16)
    k_attn4_simple<true><<<grid, 128, 0, s>>>(*L);
  else
    k_attn4_simple<false><<<grid, 128, 0, s>>>(*L);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}

}  // extern "C"
