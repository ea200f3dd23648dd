// What the kernels of shared_prefix.hip share: the line of tiles of all prefixes
// and all sequences' own slots, a workgroup's pieces of it, and who sees what.
#pragma once

#include "tree_attention.h"

namespace mi355 {

struct SharedArgs {
  TreeArgs t;             // lens, queries, mask, page numbers; partial, stats, starts of the pieces that are cut
  const int32_t* prefix;  // [groups]
  const int32_t* bounds;  // [groups + 1], ascending: where groups begin; null: every `even` sequences
  const int32_t* first;   // [batch]: the first sequence of a sequence's group, with bounds
  const int32_t* shared;  // [batch]: its shared slots, with bounds
  float* whole;           // [2][rows][d]: what one workgroup has of a prefix, of own slots
  float2* whole_stats;    // [2][rows]
  int groups, even;
  int rows;               // of all sequences: batch tokens q_heads
  int mt_rows;            // tokens group: rows of a sequence and key/value head
  uint32_t seq_mul, seq_shift, group_mul, group_shift;  // n / mt_rows = n * seq_mul >> seq_shift, likewise group
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

// Slots that sequence b shares, and with whom, by lane.
__device__ __forceinline__ int shared_of(const SharedArgs& a, int b, int len, int* first) {
  *first = b;
  if (a.bounds) {
    *first = a.first[b];
    return a.shared[b];
  }
  if (a.groups == 0) return 0;
  const int g = b / a.even;
  *first = g * a.even;
  return max(0, min(a.prefix[g], len));
}

// A stretch of slots that some rows attend to: the prefix of group v, or the own
// slots of sequence v - groups.  `tiles` per head and row block.
struct Stretch {
  int first, begin, end, rows, tiles, blocks;  // first: the sequence of row 0, whose page table counts
  __device__ __forceinline__ int size(const TreeArgs& a) const { return tiles ? a.c.heads * blocks * (tiles + a.pad) : 0; }
};
__device__ __forceinline__ Stretch stretch_of(const SharedArgs& s, int v) {
  const TreeArgs& a = s.t;
  Stretch r;
  if (v < s.groups) {
    const int g0 = s.bounds ? s.bounds[v] : v * s.even;
    const int g1 = s.bounds ? s.bounds[v + 1] : g0 + s.even;
    r.first = g0;
    r.begin = 0;
    r.end = max(0, min(s.prefix[v], a.c.capacity()));
    r.rows = (g1 - g0) * s.mt_rows;
    r.tiles = r.rows ? (r.end + a.tile - 1) / a.tile : 0;
  } else {
    const int b = v - s.groups;
    const Lengths n(a, a.lens[b], a.new_lens ? a.new_lens[b] : a.tokens);
    int first;
    r.first = b;
    r.begin = shared_of(s, b, n.len, &first);
    r.end = n.end;
    r.rows = s.mt_rows;
    r.tiles = n.fresh && r.end > r.begin ? (r.end + a.tile - 1) / a.tile - r.begin / a.tile : 0;
  }
  r.blocks = (r.rows + a.block_rows - 1) / a.block_rows;
  return r;
}

// A workgroup's share [at, last) of the line, piece by piece, in scalar
// registers.  The first `pad` tiles of a piece stand for what it costs beside
// its tiles.
struct SharedShare {
  int at, last, first, size, place, count;
  int v, start;  // the stretch at hand and where it begins
  // one piece: tiles [t0, t1) of rows row0 .. row0 + rows - 1
  Stretch w;
  int h, row0, rows, t0, t1, stop, width;
  bool prefix, cut;
  const int32_t* table;

  __device__ __forceinline__ explicit SharedShare(const SharedArgs& s) {
    const TreeArgs& a = s.t;
    const int lane = threadIdx.x & 63;
    count = s.groups + a.batch;
    int total = 0;
    int mine = 0;  // of the first 64 stretches, up to this lane's
    for (int v0 = 0; v0 < count; v0 += 64) {
      const int upto = wave_scan(v0 + lane < count ? stretch_of(s, v0 + lane).size(a) : 0);
      if (v0 == 0) mine = upto;
      total += __builtin_amdgcn_readlane(upto, 63);
    }
    size = uniform(max(1, (total + a.grid - 1) / a.grid));
    place = uniform(line_place(a, blockIdx.x));
    at = first = uniform(min(place * size, total));
    last = uniform(min(at + size, total));
    v = count;
    start = total;
    int before = 0;
    for (int v0 = 0; v0 < count; v0 += 64) {
      const int upto = before + (v0 ? wave_scan(v0 + lane < count ? stretch_of(s, v0 + lane).size(a) : 0) : mine);
      if (blockIdx.x == 0 && threadIdx.x < 64 && v0 + lane < count) a.starts[1 + v0 + lane + 1] = upto;
      const uint64_t past = __builtin_amdgcn_ballot_w64(upto > at);
      if (past && v == count) {
        const int i = uniform(__builtin_ctzll(past));
        start = uniform(i ? __builtin_amdgcn_readlane(upto, i - 1) : before);
        v = uniform(v0 + i);
        if (blockIdx.x != 0) break;
      }
      before = __builtin_amdgcn_readlane(upto, 63);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      a.starts[0] = size;
      a.starts[1] = 0;
    }
    if (v < count) w = scalar_stretch(s, v);
  }
  static __device__ __forceinline__ Stretch scalar_stretch(const SharedArgs& s, int v) {
    Stretch r = stretch_of(s, v);
    r.first = uniform(r.first);
    r.begin = uniform(r.begin);
    r.end = uniform(r.end);
    r.rows = uniform(r.rows);
    r.tiles = uniform(r.tiles);
    r.blocks = uniform(r.blocks);
    return r;
  }
  __device__ __forceinline__ bool next(const SharedArgs& s) {
    const TreeArgs& a = s.t;
    while (v < count && at < last) {
      const int piece = w.tiles + a.pad;
      const int hm = w.tiles ? uniform((at - start) / piece) : 0;
      if (w.tiles == 0 || hm >= a.c.heads * w.blocks) {
        start = uniform(start + w.size(a));
        v = uniform(v + 1);
        if (v < count) w = scalar_stretch(s, v);
        continue;
      }
      const int v0 = uniform(at - start - hm * piece), v1 = uniform(min(piece, v0 + last - at));
      width = v1 - v0;
      t0 = max(0, v0 - a.pad);
      t1 = v1 - a.pad;
      if (t1 <= t0) {  // the share ends before the piece's first tile
        done();
        continue;
      }
      cut = t0 > 0 || t1 < w.tiles;
      h = uniform(hm / w.blocks);
      row0 = uniform((hm - h * w.blocks) * a.block_rows);
      rows = uniform(min(a.block_rows, w.rows - row0));
      prefix = v < s.groups;
      const int base = w.begin / a.tile;  // own tiles begin where the prefix ends
      t0 = uniform(t0 + base);
      t1 = uniform(t1 + base);
      stop = uniform(min(w.end, t1 * a.tile));
      table = a.c.table + static_cast<int64_t>(w.first) * a.c.table_stride;
      return true;
    }
    return false;
  }
  // where a piece that is cut goes in the workspace
  __device__ __forceinline__ int64_t slot() const { return 2 * static_cast<int64_t>(place) + (at == first ? 0 : 1); }
  __device__ __forceinline__ void done() { at = uniform(at + width); }
};

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
    int first;
    limit = !p.prefix ? n.len : t < fresh ? shared_of(s, b, n.len, &first) : kAll;
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

// Q^T operands of a lane's row.
template <typename T, int FMT, int NQ>
__device__ __forceinline__ void shared_queries(const TreeArgs& a, const SharedRow& row, u32x4 (&q)[NQ]) {
  typedef typename T::bits bits;
  const int quad = (threadIdx.x & 63) >> 4;
  const bits* from = static_cast<const bits*>(a.q) + row.b * a.qb + row.t * a.qt + row.hq * a.qh;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int e = key_element<FMT>(n, quad);
    q[n] = row.t < row.fresh && e < a.c.d ? *reinterpret_cast<const u32x4*>(from + e) : u32x4{0, 0, 0, 0};
  }
}

// Sets the elements of the output rows [r0, r1) of a piece that see a NaN or an
// infinity among its values to the sum of those (the second product cannot, as
// set_non_finite of the tree's attention has it); acc row 0 is row r0.  Rare.
template <typename T, int FMT, int PITCH>
__device__ __forceinline__ void set_shared_non_finite(const SharedArgs& s, const SharedShare& p, float (*acc)[PITCH], int r0,
                                                      int r1, int first, int step, int slots) {
  const TreeArgs& a = s.t;
#pragma unroll 1
  for (int e = threadIdx.x & 63; e < a.c.d; e += 64) {
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {  // what the product left goes first
#pragma unroll 1
      for (int tile = first; tile * slots < p.stop; tile += step) {
#pragma unroll 1
        for (int slot = tile * slots; slot < min((tile + 1) * slots, p.stop); ++slot) {
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
