// What the attention kernels for many query rows (4-bit and 8-bit caches) share: tiles in shared
// and tensor memory, matrix instructions, and how the work is dealt out.
#pragma once

#include "attention_kv4.cuh"

namespace kvs {

namespace {

constexpr int kRows = 256;       // an item's query rows, two tiles
constexpr int kTile = 128;       // tokens a step
constexpr int kThreads = 16 * 32;
constexpr int kLeastTile = 2;    // steps a CTA takes at least
// The largest weight is 2^kAbove at its maximum's time, so that those down to 2^-21 of it are normal
// fp16 numbers (a first token often takes nearly all of the weight and has a small value).
constexpr float kAbove = 7.f;
constexpr float kMostSum = 32768.f;  // of 64 weights, without a new maximum (fp16 ends at 65504)
constexpr int kHalfTile = 16384; // 128 rows x 64 channels of fp16

// Instruction descriptors: fp16 x fp16 -> fp32, M = 128; N = 64 tokens with B K-major, N = 128
// channels with B MN-major.
constexpr uint32_t kIdescQK = (1u << 4) | ((64u >> 3) << 17) | ((128u >> 4) << 24);
constexpr uint32_t kIdescPV = (1u << 4) | (1u << 16) | ((128u >> 3) << 17) | ((128u >> 4) << 24);

// Tensor memory: scores of query tile x at 64 x, its weights in buffer b at 128 + 64 x + 32 b
// (fp16 pairs), its output at 256 + 128 x.
constexpr uint32_t kWeightsAt = 128, kOutAt = 256;

// Tile [128 rows][128 channels] in shared memory: two halves of 64 channels, rows of 128
// bytes, 16-byte chunks swizzled by the row.  As K (rows: N, channels: K) it is K-major;
// as V (rows: K, channels: N) it is MN-major: 64 channels a block, blocks 16 KB apart
// (leading offset), groups of 8 tokens 1 KB apart (stride offset).  Descriptors: the lower
// word is start address / 16 and leading offset / 16, the upper one stride offset / 16,
// version and 128-byte swizzle; moving along the tile adds to the lower word.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
KVS_DEV uint32_t k_desc(uint32_t saddr) { return (saddr >> 4) | (1u << 16); }
KVS_DEV uint32_t mn_desc(uint32_t saddr) {
  return (saddr >> 4) | (static_cast<uint32_t>(kHalfTile >> 4) << 16);
}
// A value that all lanes of the warp share, as a reduction over it: the compiler then keeps it where
// the matrix instructions want their operands (536 us at 2 x 2048 tokens against 736 without, when
// one warp issued them all).
KVS_DEV uint32_t uniform(uint32_t v) { return __reduce_max_sync(0xFFFFFFFFu, v); }
KVS_DEV uint32_t chunk_at(int row, int chunk) {
  return (chunk >> 3) * kHalfTile + (row >> 3) * 1024 + (row & 7) * 128 +
         (((chunk & 7) ^ (row & 7)) << 4);
}
template <uint32_t HIGH>
KVS_DEV void mma_qk(uint32_t d, uint32_t a, uint32_t b, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\t"
      "mov.b64 x, {%1, %4};\n\tmov.b64 y, {%2, %4};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(kIdescQK), "n"(HIGH), "r"(accumulate)
      : "memory");
}
KVS_DEV void mma_pv(uint32_t d, uint32_t a_tmem, uint32_t b, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\t"
      "mov.b64 y, {%2, %4};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}\n" ::"r"(d),
      "r"(a_tmem), "r"(b), "r"(kIdescPV), "n"(kDescHigh), "r"(accumulate)
      : "memory");
}
// A load of 32 columns that is waited for later: tmem_arrived() orders the uses behind it.
KVS_DEV void tmem_ld32_start(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(taddr));
}
KVS_DEV void tmem_arrived(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
  asm volatile(""
               : "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                 "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
                 "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
KVS_DEV void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}
KVS_DEV void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ------------------------------------------------------------- work split
// A tile's cost is linear in its number: with n rows' worth of queries and `len` tokens,
// tile t's last row sees about len - n + (256 t + 255) / group + 1 of them (all without causal
// limits).  In units of 1 / group tokens: cost(t) = first + more t, which sums up in closed form.
// a / b.  SHORT: of numbers that mostly have 32 bits, in a form of its own beside the long one's some
// 150 instructions.  That pays where one warp walks (8 bits); where each role does, its code costs
// more than it saves (4 bits, 2 x 2048 rows: 476 us without, 495 with it).
template <bool SHORT>
KVS_DEV long long div64(long long a, long long b) {
  if (SHORT && ((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}
struct TileWork {
  int tiles, more;        // what each tile costs more than the one before it
  long long first, head;  // cost of tile 0; of a head's tiles together
  KVS_DEV long long before(long long t) const { return t * first + more * (t * (t - 1) / 2); }
};
template <int OVER>  // an item's own cost, in steps
KVS_DEV TileWork tile_work(const Attn4Launch& L, const Seq& s, int group) {
  TileWork w;
  w.tiles = static_cast<int>((static_cast<long long>(s.n) * group + kRows - 1) / kRows);
  w.more = L.causal ? kRows : 0;
  w.first = static_cast<long long>(group) * (OVER * kTile + 1 +
                                             (L.causal ? max(s.len - s.n, 0) : s.len)) +
            kRows - 1;
  w.head = w.before(w.tiles);
  return w;
}

struct Piece {
  Seq s;
  int r, h, tile, nrows;     // nrows: the sequence's query rows times heads of the group
  int start, stop;           // tokens [start, stop), in
  int steps, halves;         // tiles and halves of 64
  bool two, whole, begins;   // second query tile in use; not shared; the item's first part
  int parts;                 // begins and not whole: CTAs that share it
};

// Walks the pieces of a CTA's share; every thread does the same.
template <int OVER, bool SHORT>
struct Walk {
  long long U, pos, end, begin;
  int r, used, b;
  KVS_DEV long long share(int i) const { return div64<SHORT>(U * i, used); }
  KVS_DEV bool next(const Attn4Launch& L, int group, Piece& p) {
    const long long unit = static_cast<long long>(kTile) * group;
    while (pos < end) {
      p.s = sequence(L, r, false);
      const TileWork w = tile_work<OVER>(L, p.s, group);
      if (pos >= begin + w.head * L.heads) {
        begin += w.head * L.heads;
        ++r;
        continue;
      }
      long long off = pos - begin;
      const int h = static_cast<int>(div64<SHORT>(off, w.head));
      off -= h * w.head;
      int lo = 0, hi = w.tiles - 1;  // the last tile that begins at or before off
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (w.before(mid) <= off) lo = mid;
        else hi = mid - 1;
      }
      const long long item = begin + h * w.head + w.before(lo);
      const long long cost = w.first + static_cast<long long>(w.more) * lo;
      const long long body = item + OVER * unit;  // the steps lie behind the item's own cost
      const long long to = min(end, item + cost);
      p.nrows = p.s.n * group;
      const int last_row = min(p.nrows, (lo + 1) * kRows) - 1;
      const int limit = max(0, seen_by(L, p.s, last_row / group));
      const int all = max(1, (limit + kTile - 1) / kTile);
      auto step_of = [&](long long x) {
        if (x >= item + cost) return all;
        if (x <= body) return 0;
        const long long k = div64<SHORT>(x - body, unit);
        return static_cast<int>(k < all ? k : all);
      };
      const int u0 = step_of(pos), u1 = step_of(to);
      pos = to;
      if (u0 >= u1) continue;
      p.r = r;
      p.h = h;
      p.tile = lo;
      p.start = u0 * kTile;
      p.stop = min(limit, u1 * kTile);
      p.halves = p.stop > p.start ? (p.stop - p.start + 63) / 64 : 0;
      p.steps = (p.halves + 1) / 2;
      p.two = p.nrows - lo * kRows > 128;
      p.begins = u0 == 0;
      p.whole = u0 == 0 && u1 == all;
      if (p.begins && !p.whole) {  // the last part is the CTA's whose share reaches the last step
        const long long x = min(item + cost, body + all * unit) - 1;
        p.parts = static_cast<int>(div64<SHORT>((x + 1) * used + U - 1, U) - 1) - b + 1;
      }
      return true;
    }
    return false;
  }
};

#define KVS_WAIT(bar, parity) wait_phase(bar, parity, L.err)
// Whether the phase is over; nothing waits for the answer before it is used.
KVS_DEV uint32_t peek_phase(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done;
}

template <int OVER>
int tile_ctas(const Attn4Launch& L) {
  const int group = L.q_heads / L.heads;
  const long long tiles = (static_cast<long long>(L.max_q) * group + kRows - 1) / kRows;
  const long long steps =
      (static_cast<long long>(L.table_cols) * L.block_size + kTile - 1) / kTile;
  const long long most = static_cast<long long>(L.seqs) * L.heads * tiles * (steps + OVER + 1);
  return static_cast<int>(most < 148 ? (most > 0 ? most : 1) : 148);
}

}  // namespace

}  // namespace kvs
