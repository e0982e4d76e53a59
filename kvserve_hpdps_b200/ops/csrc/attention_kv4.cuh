// What the attention kernels over 4-bit and 8-bit caches share: the sequences' extents, 4-bit codes
// as fp16, the running softmax's constants, how work is dealt out and the join of partial results.
#pragma once

#include "kv4.cuh"

namespace kvs {

namespace {

// Running maximum of a row that has seen nothing: finite, so that differences of two are numbers,
// and below any score that fp32 holds in comfort.
constexpr float kLowest = -3e38f;
constexpr int kLowestExp = -100;      // smallest exponent that values are scaled by
constexpr float kLazy = 8.f;          // log2 by which a score may pass its running maximum

struct Seq {
  int row0, n, len;  // first query row, query rows, cached tokens
  bool bad;          // left out
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
  // what the table has room for, and tokens whose number plus a few steps is an int
  const long long cap = min(static_cast<long long>(L.table_cols) * L.block_size, 0x7FFF0000ll);
  s.bad = s.row0 < 0 || end < s.row0 || end > L.tokens || s.n > L.max_q || s.len < 0 ||
          s.len > cap;
  if (s.bad) {
    if (report) record_error(L.err, ERR_BOUNDS);
    s.n = 0;
  }
  return s;
}

// Tokens that row i of a sequence's query rows sees.
KVS_DEV int seen_by(const Attn4Launch& L, const Seq& s, int i) {
  return L.causal ? s.len - s.n + i + 1 : s.len;
}

// Rows [from, to) have no result: 16 bytes `at`, at + by, ... of them.  Called, not inlined: inside
// the kernels it costs the registers of calls that clear nothing (drafts 55.7 us against 54.1).
__device__ __noinline__ void clear_rows(const Attn4Launch& L, long long from, long long to, long long at,
                        long long by) {
  for (long long i = at; i < (to - from) * L.q_heads * 16; i += by) {
    const long long row = i >> 4, t = from + row / L.q_heads;
    const int h = static_cast<int>(row % L.q_heads);
    if (L.clear)
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(L.out) + t * L.o_ts + h * L.o_hs +
                                (i & 15) * 8) = make_uint4(0u, 0u, 0u, 0u);
    if (L.lse != nullptr && (i & 15) == 0) L.lse[t * L.q_heads + h] = -INFINITY;
  }
}
// The rows of a sequence that is left out, by one thread a CTA (few calls have any); not those
// that another sequence names too and has results for.
KVS_DEV void clear_sequence(const Attn4Launch& L, int r) {
  const int from = max(0, L.start ? L.start[r] : r), to = min(L.tokens, L.start ? L.start[r + 1] : r + 1);
  for (int t = from + static_cast<int>(blockIdx.x); t < to; t += gridDim.x) {
    bool named = false;
    for (int i = 0; L.start && i < L.seqs && !named; ++i) {
      const Seq s = sequence(L, i, false);
      named = !s.bad && t >= s.row0 && t - s.row0 < s.n;
    }
    if (!named) clear_rows(L, t, t + 1, 0, 1);
  }
}
// Keeps the book of the rows that sequences have, for those in front of the first and behind the
// last, which are dealt out to all threads.
struct Named {
  int lo, hi;
  KVS_DEV Named() : lo(0x7FFFFFFF), hi(0) {}
  KVS_DEV void take(const Attn4Launch& L, const Seq& s, int r) {
    if (!L.clear && L.lse == nullptr) return;
    if (s.bad) {
      clear_sequence(L, r);
    } else {
      lo = min(lo, s.row0);
      hi = max(hi, s.row0 + s.n);
    }
  }
  // Between the two a __syncthreads.
  KVS_DEV void leave(const Attn4Launch& L, int2* smem) {
    if ((!L.clear && L.lse == nullptr) || L.start == nullptr) return;
    const int a = __reduce_min_sync(0xFFFFFFFFu, lo), z = __reduce_max_sync(0xFFFFFFFFu, hi);
    if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = make_int2(a, z);
  }
  template <int WARPS>
  KVS_DEV void clear(const Attn4Launch& L, const int2* smem) {
    if (!L.clear && L.lse == nullptr) return;
    int a = 0, z = L.seqs;
    if (L.start != nullptr) {
      a = L.tokens;
      z = 0;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        a = min(a, smem[w].x);
        z = max(z, smem[w].y);
      }
    }
    if (a == 0 && z == L.tokens) return;
    const long long at = static_cast<long long>(blockIdx.x) * (32 * WARPS) + threadIdx.x,
                    by = static_cast<long long>(gridDim.x) * (32 * WARPS);
    clear_rows(L, 0, a, at, by);
    clear_rows(L, z, L.tokens, at, by);
  }
};

KVS_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The codes in nibbles 0..3 of both halves of a word, each less 8, as fp16 pairs.
KVS_DEV uint32_t and_or(uint32_t a, uint32_t mask, uint32_t with) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(mask), "r"(with));
  return d;
}
KVS_DEV void codes4(uint32_t w, uint32_t k1024, uint32_t (&r)[4]) {
  const uint32_t v = w >> 8;
  const __half2 low = __float2half2_rn(-1032.f), part = __float2half2_rn(0.0625f),
                high = __float2half2_rn(-72.f);
  auto as_half2 = [](uint32_t x) { return *reinterpret_cast<const __half2*>(&x); };
  auto bits = [](__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); };
  r[0] = bits(__hadd2(as_half2(and_or(w, 0x000F000Fu, k1024)), low));
  r[1] = bits(__hfma2(as_half2(and_or(w, 0x00F000F0u, k1024)), part, high));
  r[2] = bits(__hadd2(as_half2(and_or(v, 0x000F000Fu, k1024)), low));
  r[3] = bits(__hfma2(as_half2(and_or(v, 0x00F000F0u, k1024)), part, high));
}
KVS_DEV uint32_t half2_bits(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
KVS_DEV uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
KVS_DEV void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                      uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transposes an 8x8 matrix of 16-bit elements held two to a lane.
KVS_DEV uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// Whether all lanes saw the phase end.
KVS_DEV bool wait_phase(uint64_t* bar, uint32_t parity, uint32_t* err) {
  return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, err, ERR_MBAR_TIMEOUT));
}
// One lane of a whole warp.
KVS_DEV bool elected() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xFFFFFFFF;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(p));
  return p != 0;
}
// CTA b's share of a line of length U dealt to B: [begin(b), begin(b + 1)).
struct Deal {
  int each, more;  // U / B, U % B
  KVS_DEV int begin(int b) const { return each * b + min(b, more); }
  KVS_DEV int owner(int x) const {
    const int wide = more * (each + 1);
    return x < wide ? x / (each + 1) : more + (x - wide) / each;
  }
};

// Partial results of items that several CTAs share.  A CTA leaves at most two: one for an item
// that began before its share, one for an item that goes on behind it.
struct Parts {
  int4* desc;   // [B] item that begins in CTA b and goes on: (r, h, tile, parts) or r < 0
  float2* ml;   // [2 B][rows] running maximum and sum
  float* o;     // [2 B][rows][128]
};
KVS_DEV Parts parts(void* scratch, int B, int rows) {
  Parts p;
  p.desc = static_cast<int4*>(scratch);
  p.ml = reinterpret_cast<float2*>(p.desc + B);
  p.o = reinterpret_cast<float*>(p.ml + 2ll * B * rows);
  return p;
}

// Joins the parts of the item that begins in CTA blockIdx.x and goes on in
// the next ones: eight rows at a time, WARPS warps a row, each every WARPS-th part.  Few rows an
// item come with many parts (one long sequence on all SMs): four warps.  Tiles of 256 rows
// come with few parts: one warp, and eight small CTAs an item, most of which have nothing to
// do (32 of them, a CTA for eight rows, cost 5 to 10 us more a call).
template <bool FP16, int NT, int WARPS>
__global__ void __launch_bounds__(256 * WARPS)
    k_attn4_combine(const __grid_constant__ Attn4Launch L) {
  constexpr int ROWS = 8 * NT;
  __shared__ float s_m[WARPS][8], s_l[WARPS][8];
  __shared__ float4 s_acc[WARPS][8][32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int B = gridDim.x, b = blockIdx.x;
  const Parts P = parts(L.scratch, B, ROWS);
  const int4 d = P.desc[b];
  if (d.x < 0) return;
  const int group = L.q_heads / L.heads, np = d.w;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r8 = warp & 7, quarter = warp >> 3;
  const Seq s = sequence(L, d.x, false);
  const int rows = min(ROWS, s.n * group - d.z * ROWS);  // of this tile
  for (int r0 = blockIdx.y * 8; r0 < rows; r0 += gridDim.y * 8) {
    const int row = r0 + r8;
    // part 0 is in CTA b's second slot, the others in the first ones of the next CTAs
    auto slot = [&](int i) { return (i == 0 ? 2 * b + 1 : 2 * (b + i)) * ROWS + row; };
    float m = kLowest, ls = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = quarter; i0 < np; i0 += 4 * WARPS) {  // four parts at a time, loads together
      float2 ml[4];
      float4 x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + WARPS * u;
        ml[u] = make_float2(kLowest, 0.f);
        x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < np && row < rows) {
          ml[u] = P.ml[slot(i)];
          x[u] = *reinterpret_cast<const float4*>(P.o + slot(i) * 128ll + lane * 4);
        }
      }
      const float top = fmaxf(fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), m);
      const float k0 = ex2(m - top);
      m = top;
      ls *= k0;
      a.x *= k0;
      a.y *= k0;
      a.z *= k0;
      a.w *= k0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float k2 = ex2(ml[u].x - top);
        ls = fmaf(ml[u].y, k2, ls);
        a.x = fmaf(x[u].x, k2, a.x);
        a.y = fmaf(x[u].y, k2, a.y);
        a.z = fmaf(x[u].z, k2, a.z);
        a.w = fmaf(x[u].w, k2, a.w);
      }
    }
    if constexpr (WARPS > 1) {
      s_acc[quarter][r8][lane] = a;
      if (lane == 0) {
        s_m[quarter][r8] = m;
        s_l[quarter][r8] = ls;
      }
      __syncthreads();
      if (quarter == 0) {
        m = kLowest;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) m = fmaxf(m, s_m[w][r8]);
        ls = 0.f;
        a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float k2 = ex2(s_m[w][r8] - m);
          const float4 x = s_acc[w][r8][lane];
          ls = fmaf(s_l[w][r8], k2, ls);
          a.x = fmaf(x.x, k2, a.x);
          a.y = fmaf(x.y, k2, a.y);
          a.z = fmaf(x.z, k2, a.z);
          a.w = fmaf(x.w, k2, a.w);
        }
      }
    }
    if (quarter == 0 && row < rows) {
      const int rr = d.z * ROWS + row;
      const long long tq = s.row0 + rr / group;
      const int hq = d.y * group + rr % group;
      const float inv = ls == 0.f ? 0.f : __fdividef(1.f, ls);
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(L.out) + tq * L.o_ts + hq * L.o_hs +
                                lane * 4) =
          make_uint2(f2h2<FP16>(a.x * inv, a.y * inv), f2h2<FP16>(a.z * inv, a.w * inv));
      if (L.lse != nullptr && lane == 0)
        L.lse[tq * L.q_heads + hq] =
            ls == 0.f ? -INFINITY : (m + log2f(ls)) * 0.69314718055994531f;
    }
    if constexpr (WARPS > 1) __syncthreads();  // the next rows' sums take their place
  }
}

// Launches the join behind the attention kernel, allowed to start while that ends.
template <bool FP16, int NT, int WARPS>
cudaError_t launch_combine(const Attn4Launch& L, int ctas, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, NT < 8 ? NT : 8);
  cfg.blockDim = dim3(256 * WARPS);
  cfg.stream = s;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_attn4_combine<FP16, NT, WARPS>, L);
}

}  // namespace

// attention_kv4_tile.cu: many query rows a sequence.
cudaError_t attn4_tile_launch(const Attn4Launch& L, cudaStream_t s);
long long attn4_tile_scratch(const Attn4Launch& L);

}  // namespace kvs
