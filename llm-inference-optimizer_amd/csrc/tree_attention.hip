// Attention of a few new tokens per sequence (one, a chain or a tree of drafted
// ones) over a paged cache of 16-bit values or one-byte codes, for gfx950.
//
//   S[s] = scale q . K[s],   out = sum_s exp(S[s] - m) V[s] / sum_s exp(S[s] - m)
//
// over the slots s that a token sees: one pass over the cache with a running
// maximum m and sum.  A decode step reads every key and value once for a few
// rows of q, so it is bound by HBM: the T q_heads / kv_heads rows that share a
// key/value head are taken together.
//
// Products on MFMA (v_mfma_f32_16x16x32).  Up to 32 rows a wave makes its operands
// in registers, without LDS (tree_attention_stream); for more rows the waves share
// them through LDS (tree_attention_wide).  Of tiles of 32 slots a wave computes
//   S^T = K Q^T   A = K: lane (r = l % 16, quad = l / 16) holds 8 elements of
//                 the key in slot r of a 16-slot unit; B = Q^T: the lane's
//                 column is query row l % 16.  A lane gets S of its query row
//                 for the slots 4 quad .. 4 quad + 3 of both units -- which is
//                 what the next product wants from it:
//   O^T = V^T P^T B = P^T: its 8 weights; A = V^T: 8 slots of one element d.
// The order of the summed index is free as long as A and B agree, and so is the
// order of rows: row r of V^T tile x is element d = NV r + x (NV = DP / 16), so
// that a lane loads NV consecutive elements of each of its 8 values, whole
// cache lines per row, and an output row lies in consecutive registers.
// Softmax statistics of a query row stay in its lane's column; they meet other
// lanes only where the maximum moves, and at the end.
//
// Precision: codes are exact in 16 bits, so S is an fp32 sum of exact products
// times the key's scale.  Weights times the value's scale go to the second
// product as two bf16 parts (fp16 for an fp16 cache), high and rest: 16
// significant bits where one part would have 8.  It costs a second MFMA, of
// which a decode step has plenty to spare.  What exponents are relative to moves
// rarely, so most tiles do not rescale O (`Rows` has the rules, and what fp16's
// short exponents ask for).
//
// Split: the tiles of all sequences, heads and row blocks form one line, of
// which every workgroup takes an equal share, whatever the contexts' lengths;
// the four waves take its tiles in turn and join in LDS.  A (sequence, head,
// row block) that one workgroup holds whole is written at once; the pieces of
// the others go to the workspace and tree_attention_join adds them in order.
//
// What may not be read: the buffer descriptor of each 16-slot unit ends with
// the last slot in use (and is empty for a page that is not there), so that
// loads beyond return zeros in hardware.  Slots that some rows see and others
// do not (drafted tokens) keep NaN and infinities out of the second product,
// which would spread them to every row; the elements that see them are set at
// the end, as are those that 16-bit values made NaN or infinite.  (Codes have no
// infinities; a scale that is not finite makes NaN of both parts, so of its row.)
#include <type_traits>

#include "tree_attention.h"

namespace mi355 {
namespace {

constexpr int kStreamTile = 32;  // slots of a wave's tile
constexpr int kWideTile = 64;    // slots of a workgroup's tile

// Waves that a SIMD holds at the registers of tree_attention_stream.
constexpr int stream_waves(int dp, int mt) {
  return mt == 1 && dp <= 64 ? 4 : mt == 1 && dp <= 128 ? 3 : dp * mt <= 256 ? 2 : 1;
}

// Up to 16 MT = 32 query rows per key/value head: a wave for itself, tile by
// tile, loads straight to MFMA operands.  The next tile's keys are loaded as soon
// as this one's scores are taken, its values after the second product: the
// registers hold one tile, and the other waves of the SIMD cover the rest.
// Bound by HBM where contexts are long: a call (with its join) over growing
// contexts of 2 sequences (28 / 4 heads of 128) is a line of 5.9 TB/s for int8,
// 6.0 for e4m3 and 6.6 for 16 bits that begins at 12 - 14 us: two launches, the
// line of tiles, the first loads' trip and the join.  This kernel alone: 2 of
// 120011 slots (e4m3, 253 MB) 49.8 us, 32 ragged ones to 6000 (int8, 114 MB)
// 28.6, one of 777 7.0, all of it latency.  28 rows (4 tokens) over 8 contexts of
// 4096 20.0 (int8, 35 MB) and 22.7 us (16 bits, 67 MB): short shares again, the
// vector unit 39% and 29% busy, the matrix unit 9% and 8%.
// Loads are non-temporal.  Against loads that stay in the caches, calls in a
// graph over three caches in turn: 55.3 / 59.3 us for the 253 MB, 48.6 / 53.2 for
// 225 MB of 16 bits; 35.0 / 34.6 for 116 MB of int8 and 30.2 / 28.3 for 67 MB, of
// which some is still there from three calls before.
template <typename T, int FMT, int DP, int MT>
__global__ __launch_bounds__(64 * kWaves, stream_waves(DP, MT)) void tree_attention_stream(TreeArgs a) {
  typedef UnitRegs<T, FMT, DP, kStreamAux> Regs;  // the cache is read once
  constexpr int NV = Regs::NV, NQ = DP / 32, ROWS = 16 * MT, PITCH = DP + 4, TILE = kStreamTile;
  // the weights' type in the second product: codes and bf16 values are exact in bf16
  typedef typename std::conditional<FMT == KV_16BIT, T, BF16>::type VT;
  constexpr bool SCALED = FMT != KV_16BIT;
  __shared__ float joined[kWaves][ROWS][PITCH];
  __shared__ float wave_max[kWaves][ROWS], wave_sum[kWaves][ROWS];
  const int col = threadIdx.x & 15, quad = (threadIdx.x & 63) >> 4;
  const int wave = uniform(threadIdx.x >> 6);
  const int d = a.c.d;

  Share share(a, kWaves);
  while (share.next(a)) {
    const Piece& p = share.p;
    const int t1 = share.t1;
    int tile = share.t0 + wave;
    const auto page = [&](int at) { return page_of(a, share.table, at, p.stop); };
    const auto there = [&](int n) { return n >= 0 && n < a.c.pages; };
    int p0 = page(tile * TILE), p1 = page(tile * TILE + 16);
    int next0 = page((tile + kWaves) * TILE), next1 = page((tile + kWaves) * TILE + 16);

    u32x4 q[MT][NQ];
    int token[MT];
    Rows<NV, VT> rows[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      load_queries<T, FMT>(a, p, m, q[m], token[m]);
      rows[m].clear();
    }

    Regs kv[2];
    bool left_out = false, whole;
    {
      const Unit<FMT> u0(a, p.h, tile * TILE, p.stop, p0), u1(a, p.h, tile * TILE + 16, p.stop, p1);
      whole = u0.whole && u1.whole;
      kv[0].load_keys(u0, d);
      kv[1].load_keys(u1, d);
      kv[0].load_values(u0, d);
      kv[1].load_values(u1, d);
    }

    for (; tile < t1; tile += kWaves) {
      f32x4 sc[MT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m) sc[m][0] = sc[m][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const u32x4 k0 = kv[0].keys(n), k1 = kv[1].keys(n);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          sc[m][0] = mfma16<T>(k0, q[m][n], sc[m][0]);
          sc[m][1] = mfma16<T>(k1, q[m][n], sc[m][1]);
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float f = SCALED ? a.scale * kv[u].ks[j] : a.scale;
#pragma unroll
          for (int m = 0; m < MT; ++m) sc[m][u][j] *= f;
        }

      const bool masked = !whole || (tile + 1) * TILE > p.len;
      uint32_t seen[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) seen[m] = 0xff;
      if (masked) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          seen[m] = seen_slots(a, p, tile * TILE, token[m], there(p0), there(p1));
#pragma unroll
          for (int e = 0; e < 8; ++e) sc[m][e >> 2][e & 3] = (seen[m] >> e) & 1 ? sc[m][e >> 2][e & 3] : -INFINITY;
        }
        left_out |= kv[0].take_out_non_finite();
        left_out |= kv[1].take_out_non_finite();
      }

      // the next tile's keys, while this one's weights are computed; nothing
      // is loaded beyond the share, whose units are empty
      const int at = (tile + kWaves) * TILE;
      const Unit<FMT> n0(a, p.h, at, p.stop, next0), n1(a, p.h, at + 16, p.stop, next1);
      kv[0].load_keys(n0, d);
      kv[1].load_keys(n1, d);

      u32x4 hi[MT], lo[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const float most = Rows<NV, VT>::largest(sc[m]);
        if (rows[m].moves(most)) rows[m].move(most);
        rows[m].template weights<SCALED>(sc[m], kv[0].vs, kv[1].vs, masked, seen[m], hi[m], lo[m]);
      }
#pragma unroll
      for (int x = 0; x < NV; x += 2) {
        u32x2 e0, o0, e1, o1;
        kv[0].values2(x, e0, o0);
        kv[1].values2(x, e1, o1);
        const u32x4 even = {e0[0], e0[1], e1[0], e1[1]}, odd = {o0[0], o0[1], o1[0], o1[1]};
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          rows[m].o[x] = mfma16<VT>(even, hi[m], rows[m].o[x]);
          rows[m].o[x + 1] = mfma16<VT>(odd, hi[m], rows[m].o[x + 1]);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          rows[m].o[x] = mfma16<VT>(even, lo[m], rows[m].o[x]);
          rows[m].o[x + 1] = mfma16<VT>(odd, lo[m], rows[m].o[x + 1]);
        }
      }
      kv[0].load_values(n0, d);
      kv[1].load_values(n1, d);
      whole = n0.whole && n1.whole;
      p0 = next0;
      p1 = next1;
      next0 = page(at + kWaves * TILE);
      next1 = page(at + kWaves * TILE + 16);
    }

    // join the waves: common maximum, scaled sums
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const float sum = sum_quads(rows[m].sum);
      if (quad == 0) {
        wave_max[wave][16 * m + col] = rows[m].top;
        wave_sum[wave][16 * m + col] = sum;
      }
    }
    __syncthreads();
    const auto common = [&](int r) {
      return fmaxf(fmaxf(wave_max[0][r], wave_max[1][r]), fmaxf(wave_max[2][r], wave_max[3][r]));
    };
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = 16 * m + col;
      rows[m].put(joined[wave][r], __builtin_amdgcn_exp2f(rows[m].top - common(r)));
      if constexpr (!SCALED) left_out |= rows[m].non_finite();
    }
    if (__builtin_expect(left_out, false)) {
      wave_sync();
      set_non_finite<T, FMT>(a, p, joined[wave], 0, p.rows, (share.t0 + wave) * TILE, kWaves * TILE, TILE);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.rows * (d / 4); e += 64 * kWaves) {
      const int r = e / (d / 4), c = 4 * (e - r * (d / 4));
      const float most = common(r);
      float total = 0.f;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        total += wave_sum[w][r] * __builtin_amdgcn_exp2f(wave_max[w][r] - most);
        v += *reinterpret_cast<const f32x4*>(&joined[w][r][c]);
      }
      store_result<T>(a, p, share.cut(), share.slot(), r, c, v, most, total);
    }
    __syncthreads();
    share.done();
  }
  share.finish(a);
}

// More rows: the four waves of a workgroup take 16 MT rows each and share the
// cache's tiles.  Each wave loads one of a tile's four units, makes its MFMA
// operands -- the conversion of codes and the transposition of values, which
// cost more than the products of 16 rows -- and puts them into LDS, one 16-byte
// packet per lane as the operand is read back, so that neither side meets a
// bank twice.  Two tiles in LDS: while one is used, the next is written and the
// one after it is on its way to registers; one barrier per tile.
// 8 trees of 48 tokens over ragged contexts to 4100 (28 / 4 heads of 128, 16-bit,
// 45 MB): 49.6 us (fp16 52.2) for 13.2 GFLOP, 20 with the low parts of the weights:
// per SIMD the matrix unit is busy 26% of the time and the vector unit 47%
// (exponentials, the split of the weights, masks), with two waves to overlap them.
constexpr int wide_groups(int dp, int mt) { return dp <= 64 && mt == 1 ? 3 : dp <= 128 ? 2 : 1; }  // of a CU

template <typename T, int FMT, int DP, int MT>
__global__ __launch_bounds__(64 * kWaves, wide_groups(DP, MT)) void tree_attention_wide(TreeArgs a) {
  typedef UnitRegs<T, FMT, DP, 0> Regs;  // row blocks of a head meet its cache in the L2
  constexpr int NV = Regs::NV, NQ = DP / 32, PITCH = DP + 4, TILE = kWideTile;
  typedef typename std::conditional<FMT == KV_16BIT, T, BF16>::type VT;
  constexpr bool SCALED = FMT != KV_16BIT;
  struct Stage {
    u32x4 k[4][NQ][64];      // unit, k-step, lane
    u32x2 v[2][NV][64][2];   // pair of units, element, lane, unit of the pair
    float ks[TILE], vs[TILE];
  };
  constexpr int kFix = kWaves * 16 * MT * PITCH * 4;
  __shared__ __align__(16) uint8_t lds[2 * sizeof(Stage) > kFix ? 2 * sizeof(Stage) : kFix];
  __shared__ int non_finite[kWaves];
  __shared__ int64_t out_row[kWaves][16 * MT];  // where a row's result goes, in elements
  __shared__ float inverse[kWaves][16 * MT];    // of its sum; -1: nothing to divide
  Stage* stage = reinterpret_cast<Stage*>(lds);
  const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
  const int wave = uniform(threadIdx.x >> 6);
  const int d = a.c.d;

  Share share(a, 1);
  while (share.next(a)) {
    const Piece& p = share.p;
    const int t1 = share.t1;
    // the page of this wave's unit of a tile, and which of the tile's four units
    // are there: scalar loads, the same for all waves
    const bool one_page = a.c.page_size % TILE == 0;  // of a tile
    const auto page = [&](int tile, uint32_t& units) {
      const auto there = [&](int n) { return n >= 0 && n < a.c.pages; };
      const int last = (p.stop - tile * TILE + 15) / 16;  // units in use
      const uint32_t used = last >= 4 ? 0xfu : last <= 0 ? 0u : (1u << last) - 1;
      if (one_page) {
        const int n = page_of(a, share.table, tile * TILE, p.stop);
        units = there(n) ? used : 0;
        return n;
      }
      int mine = -1;
      units = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int n = page_of(a, share.table, tile * TILE + 16 * u, p.stop);
        units |= there(n) ? 1u << u : 0u;
        mine = u == wave ? n : mine;
      }
      units &= used;
      return mine;
    };
    // a tile that not every row sees whole
    const auto edge = [&](int tile, uint32_t units) { return units != 0xf || (tile + 1) * TILE > p.len; };
    bool left_out = false;

    // this wave's unit of a tile: registers -> LDS
    Regs kv;
    uint32_t units, units_ahead;  // of the tile in registers, of the next
    const int first_page = page(share.t0, units);
    int ahead = page(share.t0 + 1, units_ahead);
    const auto load = [&](int tile, int n) {
      const Unit<FMT> u(a, p.h, tile * TILE + 16 * wave, p.stop, n);
      kv.load_keys(u, d);
      kv.load_values(u, d);
    };
    load(share.t0, first_page);

    u32x4 q[MT][NQ];
    int token[MT];
    Rows<NV, VT> rows[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      load_queries<T, FMT>(a, p, MT * wave + m, q[m], token[m]);
      rows[m].clear();
    }

    const auto put = [&](int tile) {
      Stage& s = stage[tile & 1];
      if (edge(tile, units)) left_out |= kv.take_out_non_finite();
#pragma unroll
      for (int n = 0; n < NQ; ++n) s.k[wave][n][lane] = kv.keys(n);
#pragma unroll
      for (int x = 0; x < NV; x += 2) {
        u32x2 even, odd;
        kv.values2(x, even, odd);
        s.v[wave >> 1][x][lane][wave & 1] = even;
        s.v[wave >> 1][x + 1][lane][wave & 1] = odd;
      }
      if constexpr (SCALED) {
        if (col == 0) {
          *reinterpret_cast<f32x4*>(&s.ks[16 * wave + 4 * quad]) = kv.ks;
          *reinterpret_cast<f32x4*>(&s.vs[16 * wave + 4 * quad]) = kv.vs;
        }
      }
    };
    __syncthreads();  // the last piece is read
    put(share.t0);
    uint32_t units_now = units;  // of the tile in LDS
    load(share.t0 + 1, ahead);
    units = units_ahead;
    ahead = page(share.t0 + 2, units_ahead);

    for (int tile = share.t0; tile < t1; ++tile) {
      __syncthreads();
      const Stage& s = stage[tile & 1];
      const bool masked = edge(tile, units_now);
      uint32_t seen[MT];  // both pairs of units
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        seen[m] = 0xffff;
        if (masked)
          seen[m] = seen_slots(a, p, tile * TILE, token[m], units_now & 1, units_now & 2) |
                    seen_slots(a, p, tile * TILE + 32, token[m], units_now & 4, units_now & 8) << 8;
      }
      if (tile + 1 < t1) {
        put(tile + 1);
        units_now = units;
        load(tile + 2, ahead);
        units = units_ahead;
        ahead = page(tile + 3, units_ahead);
      }
      // scores of both pairs of units, then one look at the maximum
      f32x4 sc[2][MT][2];
#pragma unroll
      for (int pair = 0; pair < 2; ++pair) {
#pragma unroll
        for (int m = 0; m < MT; ++m) sc[pair][m][0] = sc[pair][m][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          const u32x4 k0 = s.k[2 * pair][n][lane], k1 = s.k[2 * pair + 1][n][lane];
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            sc[pair][m][0] = mfma16<T>(k0, q[m][n], sc[pair][m][0]);
            sc[pair][m][1] = mfma16<T>(k1, q[m][n], sc[pair][m][1]);
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          f32x4 f = {a.scale, a.scale, a.scale, a.scale};
          if constexpr (SCALED) f *= *reinterpret_cast<const f32x4*>(&s.ks[32 * pair + 16 * u + 4 * quad]);
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int m = 0; m < MT; ++m) sc[pair][m][u][j] *= f[j];
        }
        if (masked) {
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int e = 0; e < 8; ++e)
              sc[pair][m][e >> 2][e & 3] = (seen[m] >> (8 * pair + e)) & 1 ? sc[pair][m][e >> 2][e & 3] : -INFINITY;
        }
      }
      float most[MT];
      bool moves = false;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        most[m] = fmaxf(Rows<NV, VT>::largest(sc[0][m]), Rows<NV, VT>::largest(sc[1][m]));
        moves |= rows[m].moves(most[m]);
      }
      if (moves) {
#pragma unroll
        for (int m = 0; m < MT; ++m) rows[m].move(most[m]);
      }
      u32x4 hi[2][MT], lo[2][MT];
#pragma unroll
      for (int pair = 0; pair < 2; ++pair) {
        f32x4 vs0 = {1.f, 1.f, 1.f, 1.f}, vs1 = vs0;
        if constexpr (SCALED) {
          vs0 = *reinterpret_cast<const f32x4*>(&s.vs[32 * pair + 4 * quad]);
          vs1 = *reinterpret_cast<const f32x4*>(&s.vs[32 * pair + 16 + 4 * quad]);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
          rows[m].template weights<SCALED>(sc[pair][m], vs0, vs1, masked, seen[m] >> (8 * pair), hi[pair][m],
                                           lo[pair][m]);
      }
#pragma unroll
      for (int x = 0; x < NV; ++x) {
        const u32x4 v0 = *reinterpret_cast<const u32x4*>(&s.v[0][x][lane][0]);
        const u32x4 v1 = *reinterpret_cast<const u32x4*>(&s.v[1][x][lane][0]);
#pragma unroll
        for (int m = 0; m < MT; ++m) rows[m].o[x] = mfma16<VT>(v0, hi[0][m], rows[m].o[x]);
#pragma unroll
        for (int m = 0; m < MT; ++m) rows[m].o[x] = mfma16<VT>(v0, lo[0][m], rows[m].o[x]);
#pragma unroll
        for (int m = 0; m < MT; ++m) rows[m].o[x] = mfma16<VT>(v1, hi[1][m], rows[m].o[x]);
#pragma unroll
        for (int m = 0; m < MT; ++m) rows[m].o[x] = mfma16<VT>(v1, lo[1][m], rows[m].o[x]);
      }
    }

    // every wave has its rows to itself; through LDS for whole lines of stores
    if constexpr (!SCALED) {
#pragma unroll
      for (int m = 0; m < MT; ++m) left_out |= rows[m].non_finite();
    }
    if (lane == 0) non_finite[wave] = left_out;
    const int64_t slot = share.slot();
    const bool cut = share.cut();
    const int r0 = 16 * MT * wave, r1 = min(p.rows, r0 + 16 * MT);
    __syncthreads();
    float (*mine)[PITCH] = reinterpret_cast<float (*)[PITCH]>(lds) + r0;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const float total = sum_quads(rows[m].sum);
      const int r = 16 * m + col;
      rows[m].put(mine[r], 1.0f);
      if (quad == 0 && r0 + r < r1) {
        if (cut) {
          a.stats[slot * a.block_rows + r0 + r] = float2{rows[m].top, total};
        } else {
          const int g = p.row0 + r0 + r - token[m] * a.group;
          const int64_t at = (static_cast<int64_t>(p.b) * a.tokens + token[m]) * a.q_heads + p.h * a.group + g;
          out_row[wave][r] = at * d;
          inverse[wave][r] = token[m] >= p.fresh || total == 0.f ? -1.0f : 1.0f / total;  // -1: zeros
        }
      }
    }
    wave_sync();
    if (__builtin_expect(uniform(non_finite[0] | non_finite[1] | non_finite[2] | non_finite[3]), 0)) {
      set_non_finite<T, FMT>(a, p, mine, r0, r1, share.t0 * TILE, TILE, TILE);
      wave_sync();
    }
    constexpr int LINE = DP / 4;  // lanes of a row
    const int c = 4 * (lane % LINE);
    float* partial = a.partial + (slot * a.block_rows + r0) * d + c;
    for (int r = lane / LINE; r < 16 * MT; r += 64 / LINE) {
      if (r0 + r >= r1 || c >= d) continue;
      const f32x4 v = *reinterpret_cast<const f32x4*>(&mine[r][c]);
      if (cut) {
        *reinterpret_cast<f32x4*>(partial + static_cast<int64_t>(r) * d) = v;
      } else {
        const float f = inverse[wave][r];
        const u32x2 o = {narrow2<T>(f32x2{v[0] * f, v[1] * f}), narrow2<T>(f32x2{v[2] * f, v[3] * f})};
        *reinterpret_cast<u32x2*>(static_cast<typename T::bits*>(a.out) + out_row[wave][r] + c) =
            f < 0.f ? u32x2{0, 0} : o;
      }
    }
    share.done();
  }
  share.finish(a);
}

// Adds the pieces of one query row that was cut, in order: lanes 0 - 31 and
// 32 - 63 of each of WAVES waves take every 2 WAVES-th piece with a running
// maximum, 4 (and, beyond 128, 4 more) elements per lane.  Latency is all there
// is to it: the more waves a row has, the more of its pieces are in flight at
// once.  A workgroup holds one row, or with one wave per row eight of them.
constexpr int kJoinRows = 8;

template <typename T, int WAVES>
__global__ __launch_bounds__(64 * (WAVES == 1 ? kJoinRows : WAVES)) void tree_attention_join(TreeArgs a) {
  typedef typename T::bits bits;
  constexpr int PARTS = 2 * WAVES;
  const int lane = threadIdx.x & 63, w_id = uniform(threadIdx.x >> 6);
  const int wave = WAVES == 1 ? 0 : w_id;  // of the row's
  const int qrow = WAVES == 1 ? static_cast<int>(blockIdx.x) * kJoinRows + w_id : static_cast<int>(blockIdx.x);
  const int row_count = a.batch * a.tokens * a.q_heads;
  const int hq = qrow % a.q_heads, bt = qrow / a.q_heads;
  const int t = bt % a.tokens, b = min(bt / a.tokens, a.batch - 1);
  const int share = scalar_load(a.starts, 0), start = scalar_load(a.starts, 1 + b);
  const Seq s = Seq::of(a, b);
  const int block_rows = a.block_rows;
  const int h = hq / a.group, r = t * a.group + hq - h * a.group;
  const int block = r / block_rows, rr = r - block * block_rows;
  const int first = start + (h * a.blocks + block) * s.tiles;
  const int w0 = (first + a.pad) / share, w1 = (first + s.tiles - 1) / share;
  const bool mine = qrow < row_count && w0 != w1;  // else written by the first kernel
  if (WAVES > 1 && !mine) return;

  const int part = 2 * wave + lane / 32;
  const int c0 = 4 * (lane % 32);
  const bool in0 = c0 < a.c.d, in1 = c0 + 128 < a.c.d;
  f32x4 v0 = {0.f, 0.f, 0.f, 0.f}, v1 = v0;
  float most = kLow, total = 0.f;
#pragma unroll 4
  for (int w = w0 + part; w <= w1; w += PARTS) {
    // where workgroup w left its piece: the first of its tiles, or the last
    const int64_t at = (2 * static_cast<int64_t>(w) + (w * share >= first ? 0 : 1)) * block_rows + rr;
    if (!mine) break;
    const float2 st = a.stats[at];
    const float* p = a.partial + at * a.c.d + c0;
    const f32x4 p0 = in0 ? *reinterpret_cast<const f32x4*>(p) : f32x4{0.f, 0.f, 0.f, 0.f};
    const f32x4 p1 = in1 ? *reinterpret_cast<const f32x4*>(p + 128) : f32x4{0.f, 0.f, 0.f, 0.f};
    const float now = fmaxf(most, st.x);
    const float was = __builtin_amdgcn_exp2f(most - now), f = __builtin_amdgcn_exp2f(st.x - now);
    most = now;
    total = total * was + st.y * f;
    v0 = v0 * was + p0 * f;
    v1 = v1 * was + p1 * f;
  }
  // lanes l and l + 32
  {
    const float other = __shfl_xor(most, 32), now = fmaxf(most, other);
    const float f = __builtin_amdgcn_exp2f(most - now);
    most = now;
    total *= f;
    total += __shfl_xor(total, 32);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v0[e] *= f;
      v1[e] *= f;
      v0[e] += __shfl_xor(v0[e], 32);
      v1[e] += __shfl_xor(v1[e], 32);
    }
  }
  if constexpr (WAVES > 1) {
    __shared__ f32x4 acc[WAVES][64];
    __shared__ float2 sums[WAVES];
    acc[wave][lane] = lane < 32 ? v0 : v1;
    if (lane == 0) sums[wave] = float2{most, total};
    __syncthreads();
    if (wave) return;
    for (int w = 1; w < WAVES; ++w) most = fmaxf(most, sums[w].x);
    v0 = f32x4{0.f, 0.f, 0.f, 0.f};
    total = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float f = __builtin_amdgcn_exp2f(sums[w].x - most);
      v0 += acc[w][lane] * f;
      total += sums[w].y * f;
    }
    v1 = v0;
  }
  if (!mine) return;
  const float inv = 1.0f / total;
  const bool none = t >= s.fresh || total == 0.f;
  const int c = c0 + 128 * (lane / 32);  // lanes 32 - 63 write the second half
  if (c >= a.c.d) return;
  f32x4 o = lane < 32 ? v0 : v1;
  const f32x4 zero = o - o;
  if (__builtin_expect(zero[0] + zero[1] + zero[2] + zero[3] != 0.f, false)) {
    // a piece has a NaN or an infinity, which stays whatever the piece's factor:
    // one that is 0 in 32 bits makes NaN of an infinity
    f32x4 bad = {0.f, 0.f, 0.f, 0.f};
    for (int w = w0; w <= w1; ++w) {
      const int64_t at = (2 * static_cast<int64_t>(w) + (w * share >= first ? 0 : 1)) * block_rows + rr;
      const f32x4 part = *reinterpret_cast<const f32x4*>(a.partial + at * a.c.d + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) bad[e] += part[e] - part[e] == 0.f ? 0.f : part[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = bad[e] == 0.f ? o[e] : bad[e];
  }
  *reinterpret_cast<u32x2*>(static_cast<bits*>(a.out) + static_cast<int64_t>(qrow) * a.c.d + c) =
      none ? u32x2{0, 0} : u32x2{narrow2<T>(f32x2{o[0] * inv, o[1] * inv}), narrow2<T>(f32x2{o[2] * inv, o[3] * inv})};
}

// Kernel, row blocks and grid of a call.
struct Plan {
  bool wide;
  int mt, block_rows, blocks, tile, pad, step, grid;
  int64_t partial_bytes, stats_bytes, bytes;  // of the workspace; 0: no split
};

Plan plan(const mi355_kv_cache& c, int64_t batch, int64_t tokens, int64_t q_heads, int cus) {
  Plan p{};
  const int dp = c.head_dim <= 64 ? 64 : c.head_dim <= 128 ? 128 : 256;
  const int64_t rows = tokens * (q_heads / c.kv_heads);
  // The stream kernel to 32 rows: calls in a graph, stream / wide in us, over 8
  // contexts of 4096 (over 24 of 700 the same order):
  //              28 rows, D 64   D 128         32 rows, D 256
  //   int8       15.9 / 20.4     26.6 / 30.5   23.6 / 25.6
  //   16 bits    16.6 / 18.9     29.6 / 29.4   28.2 / 25.4
  //              56 rows, D 64   D 128         64 rows, D 256
  //   int8       21.5 / 23.8     33.3 / 31.2   30.8 / 28.9
  //   16 bits    22.3 / 22.5     38.5 / 30.3   35.6 / 28.0
  // (e4m3 as int8): heads of 64 would take the stream kernel further, 16 bits of
  // 256 the wide one earlier, by up to a tenth.  Wide: 16 rows per wave while one
  // block holds them all, then 32 (336 rows of D 128, blocks of 128 / 64: 81 / 90
  // us for 8 contexts of 4096 of int8, 64.6 / 66.2 us for ragged ones of 16 bits);
  // 256-wide heads have the registers for 16.
  p.wide = rows > 32;
  p.mt = p.wide ? (rows <= 64 || dp == 256 ? 1 : 2) : (rows <= 16 ? 1 : 2);
  p.block_rows = 16 * p.mt * (p.wide ? kWaves : 1);
  p.blocks = static_cast<int>((rows + p.block_rows - 1) / p.block_rows);
  p.tile = p.wide ? kWideTile : kStreamTile;
  p.step = p.wide ? 1 : kWaves;  // tiles of a workgroup's step
  // What a piece costs beside its tiles, in tiles.  Stream, 0 / 4 / 8 / 16: 32
  // ragged contexts to 6000, D 128 37.6 / 35.3 / 35.0 / 35.7 us (int8) and 50.7 /
  // 48.6 / 48.9 / 49.8 (16 bits), D 64 21.5 / 20.4 / 18.4 / 18.5 and 24.1 / 22.4 /
  // 21.0 / 21.3, D 256 28.9 / 25.4 / 23.7 / 24.1 and 47.6 / 42.9 / 42.6 / 44.9; one
  // of 777 slots 13.4 / 10.1 / 10.2 / 10.2.  Wide, 0 / 2 / 4 / 6: 8 trees of 48
  // 64.4 / 60.0 / 59.1 / 59.9, 24 of 9 with D 64 25.6 / 24.6 / 24.8 / 24.5 (int8)
  // and 25.0 / 23.5 / 23.5 / 23.4 (16 bits), 8 of 16 with D 256 36.6 / 32.2 / 31.9 /
  // 32.2 and 36.8 / 32.1 / 31.8 / 32.7.
  p.pad = p.wide ? 4 : 8;
  const int64_t pieces = batch * c.kv_heads * p.blocks;
  const int64_t tiles = (c.table_width * c.page_size + p.tile - 1) / p.tile + p.pad;  // of the longest possible context
  p.grid = static_cast<int>(pieces);
  if (tiles - p.pad <= 2 * p.step || pieces * tiles > 0x7fffffff - 65536 * p.step) return p;
  const int64_t wanted = (pieces * tiles + p.step - 1) / p.step;
  const int64_t most = static_cast<int64_t>(cus) * (p.wide ? wide_groups(dp, p.mt) : stream_waves(dp, p.mt));
  p.grid = static_cast<int>(wanted < most ? wanted : most);
  p.partial_bytes = 2 * int64_t{p.grid} * p.block_rows * c.head_dim * 4;
  p.stats_bytes = 2 * int64_t{p.grid} * p.block_rows * 8;
  p.bytes = p.partial_bytes + p.stats_bytes + 4 * (batch + 1);
  return p;
}

template <typename T, int FMT> int tree_typed(const TreeArgs& a, const Plan& p, hipStream_t s) {
  static const char* what = "tree_attention launch";
  const dim3 grid(static_cast<unsigned>(p.grid));
#define MI355_TREE(KERNEL, DP, MT) return launch(KERNEL<T, FMT, DP, MT>, grid, 64 * kWaves, 0, a, s, what)
  if (p.wide) {
    if (a.c.d > 128) MI355_TREE(tree_attention_wide, 256, 1);
    if (a.c.d > 64 && p.mt == 1) MI355_TREE(tree_attention_wide, 128, 1);
    if (a.c.d > 64) MI355_TREE(tree_attention_wide, 128, 2);
    if (p.mt == 1) MI355_TREE(tree_attention_wide, 64, 1);
    MI355_TREE(tree_attention_wide, 64, 2);
  }
  if (a.c.d > 128 && p.mt == 1) MI355_TREE(tree_attention_stream, 256, 1);
  if (a.c.d > 128) MI355_TREE(tree_attention_stream, 256, 2);
  if (a.c.d > 64 && p.mt == 1) MI355_TREE(tree_attention_stream, 128, 1);
  if (a.c.d > 64) MI355_TREE(tree_attention_stream, 128, 2);
  if (p.mt == 1) MI355_TREE(tree_attention_stream, 64, 1);
  MI355_TREE(tree_attention_stream, 64, 2);
#undef MI355_TREE
}

template <typename T> int tree_join(const TreeArgs& a, const Plan& p, hipStream_t s) {
  static const char* what = "tree_attention join launch";
  const int64_t rows = int64_t{a.batch} * a.tokens * a.q_heads;
  const int64_t pieces = p.grid / (int64_t{a.batch} * a.c.heads * a.blocks);  // of a row, on average
  // Twice as many waves per row while half a wave has more than one piece and
  // the chip (8192 waves) holds them.  Against one wave per row: 56 rows of 96
  // pieces 55.9 / 73.5 us with the first kernel; 896 rows of 6 3.96 / 4.84 us
  // (4 waves / 1); 3024 rows of 16 7.2 / 7.9 (2 / 1; 8.7 with 4, 13.1 with 8);
  // 10752 rows of 5 13.5 / 9.9 (2 / 1).  Whole calls with 1 / 2 / 4 / 8 waves, of
  // which the rule takes 8: 28 rows of 256 pieces with D 64 70.5 / 29.7 / 24.7 / 23.2
  // us, 16 with D 256 71.5 / 32.8 / 27.8 / 26.3; 896 rows of 16 26.3 / 24.9 / 25.2 /
  // 26.4, 1024 rows of 16 with D 256 32.3 / 30.1 / 29.9 / 31.8: there it is off by 6%.
  const auto fits = [&](int waves) { return pieces > 2 * waves && 2 * rows * waves <= 8192; };
  const auto grid = [&](int64_t groups) { return dim3(static_cast<unsigned>(groups)); };
  if (fits(4)) return launch(tree_attention_join<T, 8>, grid(rows), 512, 0, a, s, what);
  if (fits(2)) return launch(tree_attention_join<T, 4>, grid(rows), 256, 0, a, s, what);
  if (fits(1)) return launch(tree_attention_join<T, 2>, grid(rows), 128, 0, a, s, what);
  return launch(tree_attention_join<T, 1>, grid((rows + kJoinRows - 1) / kJoinRows), 64 * kJoinRows, 0, a, s, what);
}

}  // namespace

int64_t tree_attention_workspace(const mi355_kv_cache& cache, int64_t batch, int64_t tokens, int64_t q_heads) {
  int cus = 0;
  if (compute_units(&cus) != MI355_OK) return 0;
  return plan(cache, batch, tokens, q_heads, cus).bytes;
}

int tree_attention_launch(const mi355_kv_cache& cache, const void* q, void* out, const int32_t* lens,
                          const int32_t* new_lens, const uint8_t* mask, int64_t mask_b, int64_t mask_t, int64_t batch,
                          int tokens, int q_heads, const int64_t* q_strides, float scale, int dtype, void* work,
                          int64_t work_bytes, hipStream_t stream) {
  int cus = 0;
  const int st = compute_units(&cus);
  if (st != MI355_OK) return st;
  Plan p = plan(cache, batch, tokens, q_heads, cus);
  TreeArgs a{kv_cache_args(cache), q, out, lens, new_lens, mask, mask_b, mask_t, q_strides[0], q_strides[1],
             q_strides[2], nullptr, nullptr, nullptr, static_cast<int>(batch), tokens, q_heads,
             q_heads / static_cast<int>(cache.kv_heads), p.block_rows, p.blocks, p.tile, 0, 0, 0, 0, scale * kLog2e};
  if (p.bytes > 0 && work != nullptr && work_bytes >= p.bytes) {
    a.partial = static_cast<float*>(work);
    a.pad = p.pad;
    a.stats = reinterpret_cast<float2*>(static_cast<uint8_t*>(work) + p.partial_bytes);
    a.starts = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(work) + p.partial_bytes + p.stats_bytes);
  } else {
    p.grid = static_cast<int>(batch * cache.kv_heads * p.blocks);
  }
  a.grid = p.grid;
  // unit / units_per_page for unit < 2^27: ceil(2^(31 + L) / u) with L = ceil(log2 u) fits 32 bits, and the product
  // is off by less than 2^L in 2^(31 + L), too little to reach the next integer
  const uint32_t upp = static_cast<uint32_t>(cache.page_size / 16);
  uint32_t log = 0;
  while ((uint64_t{1} << log) < upp) ++log;
  a.page_mul = static_cast<uint32_t>(((uint64_t{1} << (31 + log)) + upp - 1) / upp);
  a.page_shift = 31 + log;
  int r;
  if (dtype == MI355_F16) {
    r = cache.format == KV_INT8   ? tree_typed<F16, KV_INT8>(a, p, stream)
        : cache.format == KV_E4M3 ? tree_typed<F16, KV_E4M3>(a, p, stream)
                                  : tree_typed<F16, KV_16BIT>(a, p, stream);
  } else {
    r = cache.format == KV_INT8   ? tree_typed<BF16, KV_INT8>(a, p, stream)
        : cache.format == KV_E4M3 ? tree_typed<BF16, KV_E4M3>(a, p, stream)
                                  : tree_typed<BF16, KV_16BIT>(a, p, stream);
  }
  if (r != MI355_OK || a.partial == nullptr) return r;
  return dtype == MI355_F16 ? tree_join<F16>(a, p, stream) : tree_join<BF16>(a, p, stream);
}

}  // namespace mi355
