// What the kernels of shared_prefix.hip share: the line of tiles of all prefixes
// and all sequences' own slots, a workgroup's pieces of it, and who sees what.
#pragma once

#include "tree_attention.h"

namespace mi355 {

// How a stretch of slots is worked on.  Up to 16 SM query rows: every wave takes
// tiles of 32 slots for itself.  More: the waves take 16 MT rows each and share
// tiles of 16 slots per wave through LDS.
constexpr int kWaveSlots = 32;

// What the line counts for a tile and, the first `pad` of it, for a piece's other
// work: queries, first loads, sums to write and join.
struct SharedCost {
  int tile, pad;
};

struct SharedArgs {
  TreeArgs t;             // lens, queries, mask, page numbers; partial and stats of the pieces that are cut
  const int32_t* prefix;  // [groups]
  const int32_t* bounds;  // [groups + 1], ascending: where groups begin; null: every `even` sequences
  const int32_t* shared;  // [batch]: a sequence's shared slots, with bounds
  float* whole;           // [2][rows][d]: what one workgroup has of a prefix, of own slots
  float2* whole_stats;    // [2][rows]
  int2* pieces;           // [2][rows]: where a row's first piece is, and how many there are
  int groups, even;
  int rows;               // of all sequences: batch tokens q_heads
  int mt_rows;            // tokens group: rows of a sequence and key/value head
  int block_log;          // log2 of the rows of a block
  int few;                // rows that every wave takes for itself
  SharedCost many_cost, few_cost;
  int least;              // a share has at least this
  uint32_t seq_mul, seq_shift, group_mul, group_shift;  // n / mt_rows = n * seq_mul >> seq_shift, likewise group
  uint32_t even_mul, even_shift;
};

__device__ __forceinline__ int divide(int n, uint32_t mul, uint32_t shift) {
  return static_cast<int>((static_cast<uint64_t>(n) * mul) >> shift);
}

// A sequence's length, new tokens and end, within the table.
struct Lengths {
  int len, fresh, end;
  __device__ __forceinline__ Lengths(const TreeArgs& a, int len_, int fresh_) {
    const int cap = a.c.capacity();
    len = max(0, min(len_, cap));
    fresh = max(0, min(fresh_, a.tokens));
    end = min(len + fresh, cap);
  }
};

// A stretch of slots that some rows attend to: the prefix of group v, or the own
// slots of sequence v - groups.
struct Stretch {
  int first, begin, end, rows;  // first: the sequence of row 0, whose page table counts
  int base, slots;              // tiles of `slots` slots from `base` on, a multiple of 16
  int tiles, blocks;            // per head and row block
  SharedCost cost;
  __device__ __forceinline__ int piece() const { return cost.pad + tiles * cost.tile; }
  __device__ __forceinline__ int size(const TreeArgs& a) const { return tiles ? a.c.heads * blocks * piece() : 0; }
};

// Reads stretch v with LOAD(pointer, index): vector loads of a lane's, all on
// their way at once, or scalar ones.
template <typename LOAD> __device__ __forceinline__ Stretch stretch_of(const SharedArgs& s, int v, const LOAD& load) {
  const TreeArgs& a = s.t;
  const bool group = v < s.groups;
  const int b = group ? 0 : v - s.groups;
  const int g = group ? v : s.groups && !s.bounds ? divide(b, s.even_mul, s.even_shift) : 0;
  const int len = load(a.lens, b), fresh = a.new_lens ? load(a.new_lens, b) : a.tokens;
  const int prefix = s.groups ? load(s.prefix, g) : 0;
  int g0 = g * s.even, g1 = g0 + s.even, shared = prefix;
  if (s.bounds) {
    g0 = load(s.bounds, g);
    g1 = load(s.bounds, g + 1);
    shared = load(s.shared, b);
  }
  const Lengths n(a, len, fresh);
  Stretch r;
  r.first = group ? g0 : b;
  r.begin = group ? 0 : max(0, min(shared, n.len));
  r.end = group ? max(0, min(prefix, a.c.capacity())) : n.end;
  r.rows = group ? (g1 - g0) * s.mt_rows : s.mt_rows;
  const bool few = r.rows <= s.few;
  const int log = few ? 7 : 6;  // of the slots of a tile
  static_assert(kWaves * kWaveSlots == 128 && kWaves * 16 == 64, "");
  r.cost = few ? s.few_cost : s.many_cost;
  r.base = r.begin & ~15;
  r.slots = 1 << log;
  const bool any = (group ? r.rows > 0 : n.fresh > 0) && r.end > r.begin;
  r.tiles = any ? (r.end - r.base + r.slots - 1) >> log : 0;
  r.blocks = few ? 1 : (r.rows + (1 << s.block_log) - 1) >> s.block_log;
  return r;
}
__device__ __forceinline__ Stretch lane_stretch(const SharedArgs& s, int v) {
  return stretch_of(s, v, [](const int32_t* p, int i) { return p[i]; });
}

// A workgroup's share [at, last) of the line, piece by piece, in scalar
// registers.  A tile is in the share that its first unit is in.
struct SharedShare {
  int at, last, first, size, place, count;
  int v, start;  // the stretch at hand and where it begins
  // one piece: tiles of slots [from, stop) for rows row0 .. row0 + rows - 1
  Stretch w;
  int h, row0, rows, from, stop, tiles, width;
  int pieces;  // of the rows of a piece that begins here
  bool prefix, few, cut, begins;
  const int32_t* table;

  // Chunks of 64 stretches whose sizes stay in registers; those of more are read again,
  // one after the other.  28 / 4 heads, prefix 2000, 200 own slots, int8: 256 sequences
  // 61 us, 257 64, 512 101, 1024 179.
  static constexpr int kHeld = 4;

  __device__ __forceinline__ explicit SharedShare(const SharedArgs& s) {
    const TreeArgs& a = s.t;
    const int lane = threadIdx.x & 63;
    count = s.groups + a.batch;
    int total = 0, held[kHeld];
    const auto chunk = [&](int v0) {  // the running sum of 64 sizes
      const int size = lane_stretch(s, min(v0 + lane, count - 1)).size(a);
      return wave_scan(v0 + lane < count ? size : 0);
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      held[i] = 0;
      if (64 * i < count) held[i] = chunk(64 * i);
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i) total += __builtin_amdgcn_readlane(held[i], 63);
    for (int v0 = 64 * kHeld; v0 < count; v0 += 64) total += __builtin_amdgcn_readlane(chunk(v0), 63);
    size = uniform(max(s.least, (total + a.grid - 1) / a.grid));
    place = uniform(line_place(a, blockIdx.x));
    at = first = uniform(min(place * size, total));
    last = uniform(min(at + size, total));
    v = count;
    start = total;
    if (at == last) return;
    int before = 0;
    const auto look = [&](int v0, int sum) {
      const uint64_t past = __builtin_amdgcn_ballot_w64(before + sum > at);
      if (past) {
        const int i = uniform(__builtin_ctzll(past));
        start = uniform(before + (i ? __builtin_amdgcn_readlane(sum, i - 1) : 0));
        v = uniform(v0 + i);
      }
      before += __builtin_amdgcn_readlane(sum, 63);
      return past != 0;
    };
    bool found = false;
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (!found) found = look(64 * i, held[i]);
    for (int v0 = 64 * kHeld; !found && v0 < count; v0 += 64) found = look(v0, chunk(v0));
    w = scalar_stretch(s, v);
  }
  static __device__ __forceinline__ Stretch scalar_stretch(const SharedArgs& s, int v) {
    Stretch r = stretch_of(s, v, [](const int32_t* p, int i) { return scalar_load(p, i); });
    r.first = uniform(r.first);
    r.begin = uniform(r.begin);
    r.end = uniform(r.end);
    r.rows = uniform(r.rows);
    r.base = uniform(r.base);
    r.slots = uniform(r.slots);
    r.cost.tile = uniform(r.cost.tile);
    r.cost.pad = uniform(r.cost.pad);
    r.tiles = uniform(r.tiles);
    r.blocks = uniform(r.blocks);
    return r;
  }
  __device__ __forceinline__ bool next(const SharedArgs& s) {
    const TreeArgs& a = s.t;
    while (v < count && at < last) {
      const int piece = w.piece();
      const int hm = w.tiles ? uniform((at - start) / piece) : 0;
      if (w.tiles == 0 || hm >= a.c.heads * w.blocks) {
        start = uniform(start + w.size(a));
        v = uniform(v + 1);
        if (v < count) w = scalar_stretch(s, v);
        continue;
      }
      const int v0 = uniform(at - start - hm * piece), v1 = uniform(min(piece, v0 + last - at));
      width = v1 - v0;
      const int c = w.cost.tile;
      const int t0 = uniform(max(0, v0 - w.cost.pad + c - 1) / c), t1 = uniform(max(0, v1 - w.cost.pad + c - 1) / c);
      if (t1 <= t0) {  // no tile begins in this part
        done();
        continue;
      }
      cut = t0 > 0 || t1 < w.tiles;
      begins = t0 == 0;
      pieces = cut ? uniform((start + (hm + 1) * piece - c) / size) - place + 1 : 1;
      h = uniform(hm / w.blocks);
      row0 = uniform((hm - h * w.blocks) << s.block_log);
      few = w.rows <= s.few;
      rows = uniform(few ? w.rows : min(1 << s.block_log, w.rows - row0));
      prefix = v < s.groups;
      tiles = t1 - t0;
      from = uniform(w.base + t0 * w.slots);
      stop = uniform(min(w.end, w.base + t1 * w.slots));
      table = a.c.table + static_cast<int64_t>(w.first) * a.c.table_stride;
      return true;
    }
    return false;
  }
  // where a piece that is cut goes in the workspace; the pieces behind a row's
  // first are the first of the workgroups that follow
  __device__ __forceinline__ int slot() const { return 2 * place + (at == first ? 0 : 1); }
  __device__ __forceinline__ void done() { at = uniform(at + width); }
};

// The slots that sequence b shares, by lane.
__device__ __forceinline__ int shared_of(const SharedArgs& s, int b, int len) {
  if (s.bounds) return s.shared[b];
  return s.groups ? max(0, min(s.prefix[divide(b, s.even_mul, s.even_shift)], len)) : 0;
}

// A query row of a piece, by lane.
struct SharedRow {
  int b, t, hq;    // which
  int len, fresh;  // of its sequence
  int limit;       // it sees the slots of the piece below this; kAll: all of them
  static constexpr int kAll = 0x7fffffff;
  __device__ __forceinline__ SharedRow() = default;
  __device__ __forceinline__ SharedRow(const SharedArgs& s, const SharedShare& p, int r) {
    const TreeArgs& a = s.t;
    const int row = p.row0 + min(r, p.rows - 1);
    const int member = divide(row, s.seq_mul, s.seq_shift);
    const int rest = row - member * s.mt_rows;
    t = divide(rest, s.group_mul, s.group_shift);
    hq = p.h * a.group + rest - t * a.group;
    b = p.w.first + member;
    const Lengths n(a, a.lens[b], a.new_lens ? a.new_lens[b] : a.tokens);
    len = n.len;
    fresh = r < p.rows ? n.fresh : 0;
    limit = !p.prefix ? n.len : t < fresh ? shared_of(s, b, n.len) : kAll;
  }
  __device__ __forceinline__ int64_t out_row(const TreeArgs& a) const {
    return (static_cast<int64_t>(b) * a.tokens + t) * a.q_heads + hq;
  }
  // whether it sees a slot of the piece
  __device__ __forceinline__ bool sees(const TreeArgs& a, const SharedShare& p, int slot) const {
    if (p.prefix) return slot < limit;
    const int i = slot - len;
    if (slot < p.w.begin) return false;
    if (i < 0) return true;
    return t < fresh && i < fresh && (a.mask ? a.mask[b * a.mask_b + t * a.mask_t + i] != 0 : i <= t);
  }
};

// Which of the 8 slots (bit 4 u + j: slot first + 16 u + 4 quad + j) a row sees.
__device__ __forceinline__ uint32_t shared_seen(const TreeArgs& a, const SharedShare& p, const SharedRow& row, int first,
                                                uint32_t units) {
  const int quad = (threadIdx.x & 63) >> 4;
  const int s0 = first + 4 * quad;  // 16 u + j further
  const uint32_t there = (units & 1 ? 0xfu : 0u) | (units & 2 ? 0xf0u : 0u);
  uint32_t below = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) below |= s0 + 16 * (e >> 2) + (e & 3) < row.limit ? 1u << e : 0u;
  if (p.prefix) return below & there;
  const int i0 = s0 - row.len;  // the new token in slot s0
  uint32_t edge = 0, fresh = 0, own = 0;
  if (a.mask) {
    const uint8_t* m = a.mask + row.b * a.mask_b + min(row.t, a.tokens - 1) * a.mask_t;
    uint8_t byte[8];  // all on their way at once
#pragma unroll
    for (int e = 0; e < 8; ++e) byte[e] = m[max(0, min(i0 + 16 * (e >> 2) + (e & 3), a.tokens - 1))];
#pragma unroll
    for (int e = 0; e < 8; ++e) edge |= byte[e] ? 1u << e : 0u;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) edge |= i0 + 16 * (e >> 2) + (e & 3) <= row.t ? 1u << e : 0u;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int at = 16 * (e >> 2) + (e & 3);
    fresh |= i0 + at >= 0 && i0 + at < row.fresh ? 1u << e : 0u;
    own |= s0 + at >= p.w.begin ? 1u << e : 0u;
  }
  return (below | (row.t < row.fresh ? fresh & edge : 0u)) & own & there;
}

// Q^T operands of a lane's row.  AHEAD: loaded before the row's length is here,
// which takes registers.
template <typename T, int FMT, bool AHEAD, int NQ>
__device__ __forceinline__ void shared_queries(const TreeArgs& a, const SharedRow& row, u32x4 (&q)[NQ]) {
  typedef typename T::bits bits;
  const int quad = (threadIdx.x & 63) >> 4;
  const bits* from = static_cast<const bits*>(a.q) + row.b * a.qb + row.t * a.qt + row.hq * a.qh;
  const auto is = [&](int n) { return row.t < row.fresh && key_element<FMT>(n, quad) < a.c.d; };
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int e = key_element<FMT>(n, quad);
    if constexpr (AHEAD) q[n] = *reinterpret_cast<const u32x4*>(from + (e < a.c.d ? e : 0));
    else q[n] = is(n) ? *reinterpret_cast<const u32x4*>(from + e) : u32x4{0, 0, 0, 0};
  }
  if constexpr (AHEAD) {
#pragma unroll
    for (int n = 0; n < NQ; ++n)
      if (!is(n)) q[n] = u32x4{0, 0, 0, 0};
  }
}

// Sets the elements of the output rows [r0, r1) of a piece that see a NaN or an
// infinity among its values to the sum of those (the second product cannot, as
// set_non_finite of the tree's attention has it); acc row 0 is row r0.  Rare.
template <typename T, int FMT, int PITCH>
__device__ __forceinline__ void set_shared_non_finite(const SharedArgs& s, const SharedShare& p, float (*acc)[PITCH], int r0,
                                                      int r1, int first, int step, int slots) {  // slots first .. + slots - 1, first + step .., ..
  const TreeArgs& a = s.t;
#pragma unroll 1
  for (int e = threadIdx.x & 63; e < a.c.d; e += 64) {
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {  // what the product left goes first
#pragma unroll 1
      for (int tile = first; tile < p.stop; tile += step) {
#pragma unroll 1
        for (int slot = tile; slot < min(tile + slots, p.stop); ++slot) {
          const int64_t at = a.c.row(p.w.first, slot, p.h);
          if (at < 0) continue;
          float v;
          if constexpr (FMT == KV_16BIT) {
            v = load_elem<T>(a.c.v, at * a.c.d + e);
          } else {
            float four[4];
            decode4<FMT>(static_cast<const uint8_t*>(a.c.v)[at * a.c.d + e], four);
            v = four[0];
          }
          if (v - v == 0.f) continue;
#pragma unroll 1
          for (int r = r0; r < r1; ++r) {
            const SharedRow row(s, p, r);
            if (row.t >= row.fresh || !row.sees(a, p, slot)) continue;
            float* sum = &acc[r - r0][e];
            *sum = pass ? *sum + v : 0.f;
          }
        }
      }
    }
  }
}

}  // namespace mi355
