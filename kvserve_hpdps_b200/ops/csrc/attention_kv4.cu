// Attention over a paged KV cache held in 4 bits (kv4.cuh has the layout).
//
// With n query rows of a sequence whose cache holds `len` tokens, row i sees
// keys j < len - n + i + 1.  Over a group g of channels,
//   q . k_j = sum_g [ step_jg * sum_d q_d (code_jd - 8) + mid_jg * Q_g ],
// Q_g = sum of q over the group, and the output is
//   o_d = [ sum_j w_jg (code_jd - 8) + sum_j p_j mid_jg ] / sum_j p_j,
// w_jg = p_j step_jg.  A row that sees no key returns zeros and lse = -inf.
//
// A code is turned into the fp16 code - 8 by one AND-OR that puts it into the
// mantissa of 1024 and one exact fused multiply-add, for two codes at a time
// (and a shift for every second pair): the integer pipe, which has half the
// rate, shares the work with the floating-point one.  Products with the
// power-of-two scaled query are then exact and sums are fp32, so scores are
// as good as fp32's.  (Codes taken as fp16 subnormals by the AND alone cost one
// instruction less, but sums are aligned to the operands' exponent fields, so
// they lose the bits that a subnormal has in front of its first one.)
//
// The one rounding to fewer bits is that of w to fp16, the matrix
// instructions' type: 2^-11 relative, an eighth of a bf16 output's own.  An fp16
// output would lose by it (errors 1.1 to 1.55 times those of fp32 arithmetic), so for fp16
// caches w is two fp16 parts and V's product is taken with both (16 x 5 rows
// 54 -> 61 us, 48 ragged sequences 67 -> 74).  Weights share a row's exponent: a
// channel group whose steps are 2^-14 of the largest step or mid that the row
// has seen is in fp16's subnormals and keeps 2^-25 of that one.
//
// Why mma.sync and not tcgen05 for few query rows: tcgen05 reads its operands
// from shared or tensor memory, so every code would be written there as 16
// bits and read again, 4 + 4 bytes for each byte that HBM delivers.  At HBM's
// rate (23 bytes a clock and SM) that is above what shared memory moves.
// mma.sync takes the operands from the registers that unpack them.
//
// What bounds it: instructions and their latency.  32 tokens of one head and up to 8 rows take a
// warp about 780, 304 of them to unpack 8192 codes; 12 warps an SM fill 63% of the issue slots
// and half of the integer pipe.  48 ragged sequences of up to 8192 tokens, 32/8 heads, groups of
// 64 (230 MB): 69 to 72 us, 3.2 TB/s, where HBM would allow 35.  Not faster there: 16 warps with
// 128 registers (71 us against 69), 64 tokens a step (70), 16 tokens a step (87).
#include <type_traits>

#include "attention_kv4.cuh"

namespace kvs {

namespace {

constexpr int kWarps = 4;             // a CTA
constexpr int kStep = 32;             // tokens a warp takes at a time
constexpr int kUnit = kWarps * kStep; // tokens a CTA takes at a time: the unit of work
constexpr int kOver = 2;              // what starting and ending an item costs, in units
// A CTA's share of the line is no shorter than kLeast, or kFew while that takes no more than
// kSpread CTAs: short chains against few parts to join (kFew and kLeast alone: one sequence of
// 2000 tokens, 8 heads, 11.5 and 12.5 us; of 32768, 4 heads, 22.8 and 20.7).
constexpr int kLeast = 4, kFew = 2, kSpread = 148;
KVS_DEV void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
KVS_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
KVS_DEV void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
KVS_DEV uint4 lds128(const uint8_t* a) { return *reinterpret_cast<const uint4*>(a); }
KVS_DEV uint2 lds64(const uint8_t* a) { return *reinterpret_cast<const uint2*>(a); }
KVS_DEV uint32_t lds32(const uint8_t* a) { return *reinterpret_cast<const uint32_t*>(a); }
template <int NG>
KVS_DEV void lds_meta(const uint8_t* a, uint32_t (&m)[NG]) {
  if constexpr (NG == 4) {
    const uint4 v = lds128(a);
    m[0] = v.x;
    m[1] = v.y;
    m[2] = v.z;
    m[3] = v.w;
  } else if constexpr (NG == 2) {
    const uint2 v = lds64(a);
    m[0] = v.x;
    m[1] = v.y;
  } else {
    m[0] = lds32(a);
  }
}

// ------------------------------------------------------------- work split
// The work is cut at the granularity of kUnit tokens and dealt out evenly:
// item (sequence, kv head, row tile) has ceil(len / kUnit) units (at least
// one, so that rows that see nothing are written) and costs kOver more for
// its queries and its result.  The items' costs form one line of length U,
// and CTA b of B takes U / B of it, the first U % B CTAs one more, B being
// what is resident at once or, for little work, less.
// Ragged batches load every CTA alike and one long sequence is spread over
// all of them (U < 2^31: the host refuses more).  A CTA that holds
// an item whole writes its output; else it leaves a partial result (at most
// two: one for an item that began before its share, one for an item that
// goes on behind it) and k_attn4_combine joins an item's parts in order, so
// results do not depend on timing.
struct Work {
  int units;       // a sequence's share of the line
  int tiles, per;  // row tiles a head, units an item
};
KVS_DEV Work work_of(const Attn4Launch& L, const Seq& s, int rows, int group) {
  Work w;
  w.tiles = (s.n * group + rows - 1) / rows;
  w.per = s.len > 0 && !L.whole ? (s.len + kUnit - 1) / kUnit : 1;
  w.units = w.tiles * L.heads * (w.per + kOver);
  return w;
}

template <int NG>
constexpr int half_bytes() {  // 16 tokens in shared memory: K, V codes, K, V meta
  return 2048 + 128 * NG;
}

// NT * 8 query rows a tile.  Fragments (lane = 4 g + c): scores are computed
// transposed, tokens x rows, so that the 8 rows of a kv head's group fill the
// narrow side of the instruction and none of the 16 is padding; K is the A
// operand as loaded.  Their transposed fragments (movmatrix) are the B
// operand of V^T P^T, whose A operand is V with two tokens' words joined.
// Row m of a 16-token tile is token (m / 2) + 4 (m % 2) (+ 8): with the
// swizzle below both kinds of fragment loads are free of bank conflicts.
template <bool FP16, int NG, int NT>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 3 : 2)
    k_attn4(const __grid_constant__ Attn4Launch L) {
  constexpr int ROWS = 8 * NT;
  constexpr int HALF = half_bytes<NG>();
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_scan[kWarps], s_begin, s_seq;
  __shared__ float2 s_ml[kWarps][ROWS];
  __shared__ int2 s_named[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  const int group = L.q_heads / L.heads;
  const int B = gridDim.x, b = blockIdx.x;
  const Parts P = parts(L.scratch, B, ROWS);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- this CTA's share [pos, end) and the sequence that it begins in
  if (tid == 0) P.desc[b] = make_int4(-1, 0, 0, 0);
  int U = 0, mine = 0;
  Named named;
  for (int r = tid; r < L.seqs; r += kWarps * 32) {
    const Seq s = sequence(L, r, b == 0);
    named.take(L, s, r);
    mine = work_of(L, s, ROWS, group).units;
    U += mine;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) U += __shfl_xor_sync(0xFFFFFFFFu, U, o);
  if (lane == 0) s_scan[warp] = U;
  named.leave(L, s_named);
  __syncthreads();
  named.clear<kWarps>(L, s_named);
  U = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) U += s_scan[w];
  const int used =
      min(B, L.whole ? U / (1 + kOver)  // an item a CTA
                     : max((U + kLeast - 1) / kLeast, min(kSpread, (U + kFew - 1) / kFew)));
  if (b >= used) return;
  const Deal deal{U / used, U % used};
  int pos = deal.begin(b), base = 0;
  const int end = deal.begin(b + 1);
  for (int r0 = 0; r0 < L.seqs; r0 += kWarps * 32) {
    const int r = r0 + tid;
    if (L.seqs > kWarps * 32)  // else `mine` is it
      mine = r < L.seqs ? work_of(L, sequence(L, r, false), ROWS, group).units : 0;
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xFFFFFFFFu, inc, o);
      if (lane >= o) inc += x;
    }
    __syncthreads();
    if (lane == 31) s_scan[warp] = inc;
    __syncthreads();
    int before = base;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += s_scan[w];
      base += s_scan[w];
    }
    if (before + inc - mine <= pos && pos < before + inc) {
      s_seq = r;
      s_begin = before + inc - mine;
    }
    if (pos < base) break;  // the same for every thread
  }
  __syncthreads();
  int r = s_seq;
  int begin = s_begin;  // of sequence r on the line

  const uint32_t ring = smem_u32(smem) + warp * (4 * HALF);  // two stages of two halves
  float* const s_o = reinterpret_cast<float*>(smem + warp * (4 * HALF));  // later: [ROWS][128]
  uint32_t k1024;  // fp16 1024 twice, kept in a register: and_or's third operand
  asm volatile("mov.b32 %0, 0x64006400;" : "=r"(k1024));
  const int granules = L.block_size / 16;
  const int sg = (g >> 1) + 4 * (g & 1);  // the token of fragment row g
  // fragment addresses inside a half
  const uint32_t k_at = (sg >> 1) * 128 + (((((sg & 1) << 2) | c) ^ (sg & 4)) << 4);
  const uint32_t v_at = 1024 + (c >> 1) * 128 + (c & 1) * 64 +
                        ((((g >> 1) ^ (c & 2)) << 4) | ((g & 1) << 3));
  const uint32_t m_at = 2048 + sg * 4 * NG;
  // copy addresses inside a half: chunk `lane` of K, of V (chunk lane + 32 is
  // 512 bytes on in both places: eight rows further, the same swizzle)
  const int v_src = L.block_size * 64;
  const int m_src = lane < 4 * NG ? L.block_size * 128 + lane * 16
                                  : L.block_size * (128 + 4 * NG) + (lane - 4 * NG) * 16;
  const int crow = lane >> 2, cc = lane & 3;
  const uint32_t ck_dst = (crow >> 1) * 128 + (((((crow & 1) << 2) | cc) ^ (crow & 4)) << 4);
  const uint32_t cv_dst = 1024 + (crow >> 1) * 128 + (crow & 1) * 64 + ((cc ^ (crow & 2)) << 4);

  while (pos < end) {
    const Seq s = sequence(L, r, false);
    const Work wk = work_of(L, s, ROWS, group);
    if (pos >= begin + wk.units) {  // on to the next sequence that has work
      begin += wk.units;
      ++r;
      continue;
    }
    const int cost = wk.per + kOver;
    const int item = (pos - begin) / cost;
    const int from0 = pos - begin - item * cost;
    const int share = min(end - pos, cost - from0);
    // an item's overhead lies in front of its units
    const int unit0 = max(0, from0 - kOver), units = max(0, from0 + share - kOver) - unit0;
    pos += share;
    if (units <= 0) continue;
    const int h = item / wk.tiles, ti = item - h * wk.tiles;
    // low and high tiles in turn: with causal limits, neighbours add up to alike work
    const int tile = (ti & 1) ? wk.tiles - 1 - (ti >> 1) : ti >> 1;
    const int nrows = s.n * group;
    const int last_row = min(nrows, (tile + 1) * ROWS) - 1;
    const int min_seen = max(0, s.len - s.n + tile * ROWS / group + 1);
    const int limit = max(0, s.len - s.n + last_row / group + 1);

    // ---- this warp's steps: tokens first + kUnit k + [0, 32)
    const int first = unit0 * kUnit + warp * kStep;
    const int stop = L.whole ? limit : min(limit, (unit0 + units) * kUnit);
    const int steps = first < stop ? (stop - first + kUnit - 1) / kUnit : 0;
    const uint8_t* const head = static_cast<const uint8_t*>(L.cache) + h * L.head_stride;
    const int32_t* const table = L.table + r * L.table_stride;
    int ids = -1, offs = 0;      // of step k % 16 = lane / 2, half lane % 2
    uint32_t have = 0;           // bit 2 (k % 2) + half: that half was copied
    auto copy_step = [&](int k) {
      if ((k & 15) == 0) {
        const int tok = first + (k + (lane >> 1)) * kUnit + 16 * (lane & 1);
        ids = -1;
        if (tok < stop) {
          const int page = tok / 16 / granules;
          offs = tok - page * L.block_size;
          ids = table[page];
          if (ids < 0 || ids >= L.num_blocks) {
            record_error(L.err, ERR_BOUNDS);
            ids = -1;
          }
        }
      }
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int from = 2 * (k & 15) + hf;
        const int id = __shfl_sync(0xFFFFFFFFu, ids, from);
        const int off = __shfl_sync(0xFFFFFFFFu, offs, from);
        const uint32_t bit = 1u << (2 * (k & 1) + hf);
        have &= ~bit;
        if (id >= 0) {
          have |= bit;
          const uint8_t* rec = head + static_cast<uint64_t>(static_cast<uint32_t>(id)) *
                                          static_cast<uint32_t>(L.block_stride);
          const uint8_t* kc = rec + (off * 64 + lane * 16);
          const uint8_t* vc = kc + v_src;
          const uint32_t dst = ring + ((k & 1) * 2 + hf) * HALF;
          cp_async16(dst + ck_dst, kc);
          cp_async16(dst + ck_dst + 512, kc + 512);
          cp_async16(dst + cv_dst, vc);
          cp_async16(dst + cv_dst + 512, vc + 512);
          if (lane < 8 * NG) cp_async16(dst + 2048 + lane * 16, rec + (off * (4 * NG) + m_src));
        }
      }
      cp_async_commit();
    };
    uint4 raw[NT][4] = {};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = tile * ROWS + nt * 8 + g;
      if (row < nrows) {
        const uint16_t* qp = static_cast<const uint16_t*>(L.q) +
                             (s.row0 + row / group) * L.q_ts +
                             (h * group + row % group) * L.q_hs + 8 * c;
#pragma unroll
        for (int q = 0; q < 4; ++q) raw[nt][q] = *reinterpret_cast<const uint4*>(qp + 32 * q);
      }
    }
    if (steps > 0) copy_step(0);

    // ---- query fragments: fp16, each row scaled by a power of two so that its largest
    // element is in [2^14, 2^15); exact unless 2^-31 of the largest
    uint32_t qf[NT][4][2][2];
    float f[NT][2], qs[NG][NT][2];  // of this lane's columns 2c, 2c + 1
    int seen[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x[4][8], top = 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        unpack8<FP16>(raw[nt][q], x[q]);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[q][i]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
      int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
      e = top == 0.f ? 0 : max(kLowestExp, e);
      // an infinite element makes the row what is not a number
      const float up = __uint_as_float(top < INFINITY ? static_cast<uint32_t>(127 + 14 - e) << 23
                                                      : 0x7FC00000u) *
                       (L.scale < 0.f ? -1.f : 1.f);
      // not zero: a hidden score is -inf times it
      const float fr = fmaxf(fabsf(L.scale) * 1.4426950408889634f *
                                 __uint_as_float(static_cast<uint32_t>(127 - 14 + e) << 23),
                             1.17549435e-38f);
      float sum[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        sum[q] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[q][i] *= up;
          sum[q] += x[q][i];
        }
        sum[q] += __shfl_xor_sync(0xFFFFFFFFu, sum[q], 1);
        sum[q] += __shfl_xor_sync(0xFFFFFFFFu, sum[q], 2);
        qf[nt][q][0][0] = half2_bits(x[q][0], x[q][4]);
        qf[nt][q][0][1] = half2_bits(x[q][2], x[q][6]);
        qf[nt][q][1][0] = half2_bits(x[q][1], x[q][5]);
        qf[nt][q][1][1] = half2_bits(x[q][3], x[q][7]);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int from = (2 * c + j) * 4;
        f[nt][j] = __shfl_sync(0xFFFFFFFFu, fr, from);
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) qs[gr][nt][j] = 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          qs[q * NG / 4][nt][j] += __shfl_sync(0xFFFFFFFFu, sum[q], from);
        const int cr = tile * ROWS + nt * 8 + 2 * c + j;
        seen[nt][j] = cr < nrows ? s.len - s.n + cr / group + 1 : 0x7FFFFFFF;
      }
    }

    float acc[8][NT][4], msum[NG][NT][2], l[NT][2], M[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][nt][i] = 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        l[nt][j] = 0.f;
        M[nt][j] = kLowest;
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) msum[gr][nt][j] = 0.f;
      }
    }
    float E[NT][2], most_in = __uint_as_float(static_cast<uint32_t>(127 + 4 + kLowestExp) << 23);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) E[nt][0] = E[nt][1] = kLowestExp;

    auto step = [&](auto tag, int t0, const uint8_t* st, uint32_t had) {
      constexpr bool MASKED = decltype(tag)::value;
      float sc[2][NT][4];
      uint32_t vm[2][2][NG];  // [half][row g, g + 8] (step, mid) of the values
      uint32_t big = 0;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const uint8_t* const at = st + hf * HALF;
        const uint4 ka = lds128(at + k_at), kb = lds128(at + k_at + 512);
        const uint32_t kw0[4] = {ka.x, ka.y, ka.z, ka.w}, kw1[4] = {kb.x, kb.y, kb.z, kb.w};
        uint32_t km0[NG], km1[NG];
        lds_meta<NG>(at + m_at, km0);
        lds_meta<NG>(at + m_at + 32 * NG, km1);
        lds_meta<NG>(at + m_at + 64 * NG, vm[hf][0]);
        lds_meta<NG>(at + m_at + 96 * NG, vm[hf][1]);
        if (MASKED) {  // what no row of the tile sees counts as zeros, whatever its bytes are
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (!(had >> hf & 1u) || t0 + 16 * hf + sg + 8 * i >= limit) {
#pragma unroll
              for (int gr = 0; gr < NG; ++gr) vm[hf][i][gr] = 0;
            }
        }
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          float a[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) a[nt][i] = 0.f;
#pragma unroll
          for (int q = gr * 4 / NG; q < (gr + 1) * 4 / NG; ++q) {
            uint32_t u[4], v[4];
            codes4(kw0[q], k1024, u);
            codes4(kw1[q], k1024, v);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816(a[nt], u[0], v[0], u[2], v[2], qf[nt][q][0][0], qf[nt][q][0][1]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816(a[nt], u[1], v[1], u[3], v[3], qf[nt][q][1][0], qf[nt][q][1][1]);
          }
          const float s0 = h2f<FP16>(km0[gr] & 0xFFFFu), s1 = h2f<FP16>(km1[gr] & 0xFFFFu);
          const float z0 = h2f<FP16>(km0[gr] >> 16), z1 = h2f<FP16>(km1[gr] >> 16);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float z = i < 2 ? z0 : z1, y = qs[gr][nt][i & 1];
              sc[hf][nt][i] = fmaf(i < 2 ? s0 : s1, a[nt][i],
                                   gr == 0 ? z * y : fmaf(z, y, sc[hf][nt][i]));
            }
          big = max_u16x2(big, max_u16x2(vm[hf][0][gr] & 0x7FFF7FFFu, vm[hf][1][gr] & 0x7FFF7FFFu));
        }
        if (MASKED) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int tok = t0 + 16 * hf + sg + (i < 2 ? 0 : 8);
              if (!(had >> hf & 1u) || tok >= seen[nt][i & 1]) sc[hf][nt][i] = -INFINITY;
            }
        }
      }
      // ---- reference M + E of the exponentials: a row's running maximum, passed by up to
      // 2^kLazy before it is moved, and the exponent of the largest step or
      // mid that the row has seen (moved when passed by 2^4, `most_in`): w then stays inside
      // fp16's range whatever the values' scale, and sums keep one scale.
      const float most = fmaxf(h2f<FP16>(big & 0xFFFFu), h2f<FP16>(big >> 16));
      bool move = most > most_in;
      float top[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          top[nt][j] = fmaxf(fmaxf(sc[0][nt][j], sc[0][nt][j + 2]),
                             fmaxf(sc[1][nt][j], sc[1][nt][j + 2])) * f[nt][j];
          move |= top[nt][j] - M[nt][j] > kLazy;
        }
      if (__any_sync(0xFFFFFFFFu, move)) {
        // the largest that is finite: an infinite step or mid makes its own channels NaN and
        // must not put the other channels' weights out of range; nor must a token that the row
        // does not see
        constexpr uint32_t kInf = FP16 ? 0x7C00u : 0x7F80u;
        uint32_t fine[2][2];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
          for (int r2 = 0; r2 < 2; ++r2) {
            fine[hf][r2] = 0;
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
              const uint32_t a = vm[hf][r2][gr] & 0x7FFFu, z = vm[hf][r2][gr] >> 16 & 0x7FFFu;
              fine[hf][r2] = max(fine[hf][r2], max(a < kInf ? a : 0u, z < kInf ? z : 0u));
            }
          }
        float low = 100.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float x = top[nt][j];
            uint32_t all = 0;
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
#pragma unroll
              for (int r2 = 0; r2 < 2; ++r2)
                if (!MASKED || sc[hf][nt][2 * r2 + j] != -INFINITY) all = max(all, fine[hf][r2]);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
              x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, o));
              if (MASKED) all = max(all, __shfl_xor_sync(0xFFFFFFFFu, all, o));
            }
            if (!MASKED) all = __reduce_max_sync(0xFFFFFFFFu, all);
            const int bits = static_cast<int>(__float_as_uint(h2f<FP16>(all)) >> 23) - 127;
            const float old = M[nt][j], e = fminf(fmaxf(static_cast<float>(bits), E[nt][j]), 100.f);
            const float m = fmaxf(old, x), less = (old - m) + (E[nt][j] - e);
            M[nt][j] = m;
            E[nt][j] = e;
            low = fminf(low, e);
            // in two factors: E alone may move by more than the range of one (tokens whose
            // values are zero, then large ones), and their part of the sum has to stay
            const float k1 = ex2(0.5f * less), k2 = k1 * k1;
            l[nt][j] = l[nt][j] * k1 * k1;
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) msum[gr][nt][j] *= k2;
#pragma unroll
            for (int d = 0; d < 8; ++d) {
              acc[d][nt][j] *= k2;
              acc[d][nt][j + 2] *= k2;
            }
          }
        most_in = __uint_as_float(static_cast<uint32_t>(127 + 4 + static_cast<int>(low)) << 23);
      }
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const uint8_t* const at = st + hf * HALF;
        float p[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // rounded as the maximum was, and that taken off first: a fused multiply-add would
            // leave the maximum's rounding over, which grows with the score
            p[nt][i] = ex2(__fmul_rn(sc[hf][nt][i], f[nt][i & 1]) - M[nt][i & 1] - E[nt][i & 1]);
            l[nt][i & 1] += p[nt][i];
          }
        const uint2 v0 = lds64(at + v_at), v1 = lds64(at + v_at + 256),
                    v2 = lds64(at + v_at + 512), v3 = lds64(at + v_at + 768);
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          const float s0 = h2f<FP16>(vm[hf][0][gr] & 0xFFFFu), z0 = h2f<FP16>(vm[hf][0][gr] >> 16);
          const float s1 = h2f<FP16>(vm[hf][1][gr] & 0xFFFFu), z1 = h2f<FP16>(vm[hf][1][gr] >> 16);
          uint32_t b0[NT], b1[NT], rest0[NT], rest1[NT];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              w[i] = p[nt][i] * (i < 2 ? s0 : s1);
              float& ms = msum[gr][nt][i & 1];
              if (MASKED) {  // a row takes nothing of a token it does not see, NaN or not
                const bool hid = sc[hf][nt][i] == -INFINITY;
                if (hid) w[i] = 0.f;
                ms += hid ? 0.f : p[nt][i] * (i < 2 ? z0 : z1);
              } else {
                ms = fmaf(p[nt][i], i < 2 ? z0 : z1, ms);
              }
            }
            const uint32_t lo = half2_bits(w[0], w[1]), hi = half2_bits(w[2], w[3]);
            b0[nt] = transpose8(lo);
            b1[nt] = transpose8(hi);
            if constexpr (FP16) {  // what the rounding leaves over
              rest0[nt] = transpose8(half2_bits(w[0] - h2f<true>(lo & 0xFFFFu),
                                                w[1] - h2f<true>(lo >> 16)));
              rest1[nt] = transpose8(half2_bits(w[2] - h2f<true>(hi & 0xFFFFu),
                                                w[3] - h2f<true>(hi >> 16)));
            }
          }
#pragma unroll
          for (int q = gr * 4 / NG; q < (gr + 1) * 4 / NG; ++q) {
            const uint32_t pick = (q & 1) ? 0x7632u : 0x5410u;
            const uint32_t x01 = __byte_perm(q < 2 ? v0.x : v0.y, q < 2 ? v1.x : v1.y, pick);
            const uint32_t x23 = __byte_perm(q < 2 ? v2.x : v2.y, q < 2 ? v3.x : v3.y, pick);
            uint32_t u[4], v[4];
            codes4(x01, k1024, u);
            codes4(x23, k1024, v);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816(acc[2 * q][nt], u[0], u[2], v[0], v[2], b0[nt], b1[nt]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816(acc[2 * q + 1][nt], u[1], u[3], v[1], v[3], b0[nt], b1[nt]);
            if constexpr (FP16) {
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma16816(acc[2 * q][nt], u[0], u[2], v[0], v[2], rest0[nt], rest1[nt]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma16816(acc[2 * q + 1][nt], u[1], u[3], v[1], v[3], rest0[nt], rest1[nt]);
            }
          }
        }
      }
    };
    for (int k = 0; k < steps; ++k) {
      const uint32_t had = have >> (2 * (k & 1));
      if (k + 1 < steps) {
        copy_step(k + 1);
        cp_async_wait<1>();
      } else {
        cp_async_wait<0>();
      }
      __syncwarp();
      const int t0 = first + k * kUnit;
      const uint8_t* const st = smem + warp * (4 * HALF) + (k & 1) * 2 * HALF;
      if ((had & 3u) != 3u || t0 + kStep > min_seen)
        step(std::true_type{}, t0, st, had);
      else
        step(std::false_type{}, t0, st, had);
      __syncwarp();  // the stage may be overwritten
    }

    // ---- join the warps' results
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = nt * 8 + 2 * c + j;
        float ls = l[nt][j], corr[NG];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) ls += __shfl_xor_sync(0xFFFFFFFFu, ls, o);
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          float ms = msum[gr][nt][j];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) ms += __shfl_xor_sync(0xFFFFFFFFu, ms, o);
          corr[gr] = ms;
        }
        // out of the units of this warp's E, which the others need not share
        const float unit =
            __uint_as_float(static_cast<uint32_t>(127 + static_cast<int>(E[nt][j])) << 23);
        if (g == 0) s_ml[warp][row] = make_float2(M[nt][j], ls * unit);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float z = corr[q * NG / 4];
          float4 o4;  // channels 32 q + 4 g + 0..3
          o4.x = (acc[2 * q][nt][j] + z) * unit;
          o4.y = (acc[2 * q + 1][nt][j] + z) * unit;
          o4.z = (acc[2 * q][nt][j + 2] + z) * unit;
          o4.w = (acc[2 * q + 1][nt][j + 2] + z) * unit;
          *reinterpret_cast<float4*>(s_o + row * 128 + 32 * q + 4 * g) = o4;
        }
      }
    __syncthreads();
    const bool whole = unit0 == 0 && units == wk.per;
    const int slot = 2 * b + (unit0 == 0 ? 1 : 0);
#pragma unroll
    for (int it = 0; it < ROWS / kWarps; ++it) {  // a warp a row, four channels a lane
      const int row = it * kWarps + warp, rr = tile * ROWS + row;
      if (rr >= nrows) break;
      float m = kLowest, ls = 0.f;
      float2 ml[kWarps];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        ml[w] = s_ml[w][row];
        m = fmaxf(m, ml[w].x);
      }
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float k2 = ex2(ml[w].x - m);
        const float4 x =
            *reinterpret_cast<const float4*>(smem + w * (4 * HALF) + row * 512 + lane * 16);
        ls = fmaf(ml[w].y, k2, ls);
        o.x = fmaf(x.x, k2, o.x);
        o.y = fmaf(x.y, k2, o.y);
        o.z = fmaf(x.z, k2, o.z);
        o.w = fmaf(x.w, k2, o.w);
      }
      if (whole) {
        const long long tq = s.row0 + rr / group;
        const int hq = h * group + rr % group;
        const float inv = ls == 0.f ? 0.f : __fdividef(1.f, ls);
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(L.out) + tq * L.o_ts + hq * L.o_hs +
                                  lane * 4) =
            make_uint2(f2h2<FP16>(o.x * inv, o.y * inv), f2h2<FP16>(o.z * inv, o.w * inv));
        if (L.lse != nullptr && lane == 0)
          L.lse[tq * L.q_heads + hq] =
              ls == 0.f ? -INFINITY : (m + log2f(ls)) * 0.69314718055994531f;
      } else {
        *reinterpret_cast<float4*>(
            P.o + (static_cast<long long>(slot) * ROWS + row) * 128 + lane * 4) = o;
        if (lane == 0) P.ml[slot * ROWS + row] = make_float2(m, ls);
      }
    }
    if (!whole && unit0 == 0 && tid == 0)  // parts: up to the CTA that holds the item's end
      P.desc[b] = make_int4(r, h, tile, deal.owner(begin + (item + 1) * cost - 1) - b + 1);
    __syncthreads();
  }
}

struct Grid {
  int ctas, rows;
  bool fits;   // the line's length is an int
  bool split;  // whether items may be split
};

// Tables of at most so many units are not split: the launch that joins the parts takes longer
// than a second step (150 tokens, one sequence: 9.5 us in a table of 32768 tokens, 7.4 in one of
// 160; the host knows the table's width and not the lengths).
constexpr int kWholeUnits = 2;

// Rows a tile: 8 hold a decode step's query heads of one kv head (up to 8);
// more rows take 16, which unpack each code once for twice the rows.
Grid grid_of(const Attn4Launch* L) {
  Grid g;
  const int group = L->q_heads / L->heads;
  const long long rows = static_cast<long long>(L->max_q) * group;
  g.rows = rows <= 8 ? 8 : 16;
  const long long per = (static_cast<long long>(L->table_cols) * L->block_size + kUnit - 1) / kUnit;
  const long long items = static_cast<long long>(L->seqs) * L->heads *
                          ((rows + g.rows - 1) / g.rows);
  const long long units = items * (per > kWholeUnits ? per : 1);
  // block offsets are 32 x 32 -> 64 bit products
  g.fits = L->block_stride >= 0 && L->block_stride < (1ll << 32) && items < (1ll << 31) &&
           items * (per + 1 + kOver) < (1ll << 31);
  const long long most = 148ll * (g.rows == 8 ? 3 : 2);  // resident at once
  g.ctas = static_cast<int>(units < most ? units : most);
  g.split = per > kWholeUnits;
  return g;
}

// Whether a call goes to attention_kv4_tile.cu: many rows a kv head, and enough of them by what the
// host knows (max_query_len, and the tokens that the table has room for; tables as wide as the
// sequences below).  fp16 caches, whose tiles take twice the conversion there, from more rows on.
// Measured, us here / there for bf16 and for fp16, groups of 64: 32 sequences of 2000 tokens,
// 8 heads: 48 rows 99 / 97 and 114 / 174, 80 rows 153 / 103 and 179 / 178; 16 of 2000: 64 rows
// 72 / 58 and 81 / 93, 96 rows 99 / 62 and 113 / 96; 8 of 8000, 4 heads: 56 rows 61 / 51 and
// 71 / 80, 84 rows 86 / 55 and 100 / 82; 64 of 1000, 4 heads: 84 rows 122 / 78 and 143 / 114.
// With little to do the tiles' fixed cost decides (Mi rows times tokens times heads): one of
// 1024 tokens, 4 heads: 1792 rows (7 Mi) 43 / 37 and 49 / 40; 8 of 2000, 8 heads: 52 rows (6.3 Mi)
// 43 / 37; 4 of 2000: 96 rows (5.9 Mi) 36 / 32 and 39 / 40.  One long sequence on many heads
// loses there: one of 4000, 8 heads: 192 rows (5.9 Mi) 32 / 40 and 36 / 44.  A call goes there as
// a whole: one of 512 rows over 4096 tokens beside 48 sequences of one row, 32/8 heads, takes
// 327 us, the two kinds in calls of their own 149.
constexpr int kManyRows = 48, kManyRowsFp16 = 80;
constexpr long long kMuchWork = 5ll << 20;
bool many_rows(const Attn4Launch* L) {
  const long long rows = static_cast<long long>(L->max_q) * (L->q_heads / L->heads);
  const double work = static_cast<double>(rows) * L->seqs * L->heads * L->table_cols *
                      L->block_size;
  return rows > (L->fp16 ? kManyRowsFp16 : kManyRows) && work > static_cast<double>(kMuchWork);
}

template <bool FP16, int NG, int NT>
cudaError_t launch(const Attn4Launch& L, const Grid& g, cudaStream_t s) {
  const int smem = kWarps * 4 * half_bytes<NG>();  // at most 40 KB: no opt-in needed
  static_assert(kWarps * 4 * half_bytes<NG>() <= 46 * 1024);
  k_attn4<FP16, NG, NT><<<g.ctas, kWarps * 32, smem, s>>>(L);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !g.split) return e;
  return launch_combine<FP16, NT, 4>(L, g.ctas, s);
}

template <bool FP16, int NG>
cudaError_t launch_rows(const Attn4Launch& L, const Grid& g, cudaStream_t s) {
  return g.rows == 8 ? launch<FP16, NG, 1>(L, g, s) : launch<FP16, NG, 2>(L, g, s);
}
template <bool FP16>
cudaError_t launch_groups(const Attn4Launch& L, const Grid& g, cudaStream_t s) {
  return L.groups == 1   ? launch_rows<FP16, 1>(L, g, s)
         : L.groups == 2 ? launch_rows<FP16, 2>(L, g, s)
                         : launch_rows<FP16, 4>(L, g, s);
}

}  // namespace
}  // namespace kvs

using namespace kvs;

extern "C" {

long long kvs_attn4_scratch_bytes(const Attn4Launch* L) {
  if (many_rows(L)) return attn4_tile_scratch(*L);
  const Grid g = grid_of(L);
  return 16ll * g.ctas + 2ll * g.ctas * g.rows * (8 + 512);
}

int kvs_attention_kv4(const Attn4Launch* L, void* stream) {
  if (L->seqs <= 0 || L->max_q <= 0 || L->tokens <= 0 || L->heads <= 0) return 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (many_rows(L)) return attn4_tile_launch(*L, s) == cudaSuccess ? 0 : -1;
  const Grid g = grid_of(L);
  if (!g.fits) return -2;
  Attn4Launch A = *L;
  A.whole = !g.split;
  const cudaError_t e = L->fp16 ? launch_groups<true>(A, g, s) : launch_groups<false>(A, g, s);
  return e == cudaSuccess ? 0 : -1;
}

}  // extern "C"
