// The kernels of attention under shared prefixes; shared_prefix.hip has the host
// side and the instantiations for fp16, shared_prefix_bf16.hip those for bf16.
#pragma once

#include <type_traits>

#include "shared_prefix.h"

namespace mi355 {

// Row blocks and grid of a call, and its workspace.
struct SharedPlan {
  int mt, sm, grid;
  int64_t partial, stats, whole, whole_stats, pieces, bounds, shared, bytes;  // offsets
};

// Workgroups of a CU: two tiles in LDS of each.
constexpr int shared_groups(int dp) { return dp > 128 ? 1 : 2; }

// Pages of the 64 units of 16 slots from a slot on, by lane; -1 where there is none.
__device__ __forceinline__ int load_pages(const TreeArgs& a, const SharedShare& p, int slot0) {
  const int slot = slot0 + 16 * static_cast<int>(threadIdx.x & 63);
  const int page = p.table[divide(max(0, min(slot, p.stop - 1)) / 16, a.page_mul, a.page_shift)];
  return slot < p.stop && page < a.c.pages ? page : -1;
}

// Whether the largest weights of 16 rows, each the largest of four lanes', ask for
// another maximum (as Rows::moves).
template <typename VT> __device__ __forceinline__ bool weights_move(float most) {
  typedef Rows<2, VT> R;
  static_assert(R::kMost == (R::FOLLOW ? 15.0f : 8.0f) && R::kLeast == 7.0f, "the powers of 2 below");
  const bool over = __builtin_amdgcn_ballot_w64(!(most <= (R::FOLLOW ? 32768.0f : 256.0f))) != 0;
  if constexpr (!R::FOLLOW) return over;
  uint64_t near = __builtin_amdgcn_ballot_w64(most >= 128.0f);
  near |= near >> 32;
  near |= near >> 16;
  return over || (near & 0xffff) != 0xffff;
}

// 8 weights as the two parts of a P^T operand.
template <typename VT>
__device__ __forceinline__ void split_weights(const f32x4 (&w)[2], u32x4& hi, u32x4& lo) {
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const float a = w[p >> 1][2 * (p & 1)], b = w[p >> 1][2 * (p & 1) + 1];
    hi[p] = narrow2<VT>(f32x2{a, b});
    const f32x2 back = widen2<VT>(hi[p]);
    lo[p] = narrow2<VT>(f32x2{a - back.x, b - back.y});
  }
}

// Weights of 32 slots for 16 rows from their scores (q . k, without the scale; f:
// the scores' factors), relative to the maximum so far; the largest of a lane's.
// Where all rows see all slots, and none of the weights asks for another maximum,
// they are the weights.
template <int NV, typename VT>
__device__ __forceinline__ float weights_at_once(const Rows<NV, VT>& rows, const f32x4 (&sc)[2], const f32x4 (&f)[2],
                                                 f32x4 (&w)[2]) {
  float most = 0.f;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[u][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][j], f[u][j], -rows.top));
      most = fmaxf(most, w[u][j]);
    }
  return most;
}
// Adds them to the rows' sums; times the values' scales they are the two parts of
// a P^T operand.
template <int NV, typename VT, bool SCALED>
__device__ __forceinline__ void take_weights(Rows<NV, VT>& rows, f32x4 (&w)[2], const f32x4 (&vs)[2], u32x4& hi, u32x4& lo) {
  rows.sum += ((w[0][0] + w[0][1]) + (w[0][2] + w[0][3])) + ((w[1][0] + w[1][1]) + (w[1][2] + w[1][3]));
  if constexpr (SCALED) {
    w[0] *= vs[0];
    w[1] *= vs[1];
  }
  split_weights<VT>(w, hi, lo);
}
// The same with masks and another maximum where it is asked for.
template <int NV, typename VT, bool SCALED>
__device__ __forceinline__ void weights_by_maximum(Rows<NV, VT>& rows, f32x4 (&sc)[2], const f32x4 (&f)[2],
                                                   const f32x4 (&vs)[2], bool masked, uint32_t seen, u32x4& hi,
                                                   u32x4& lo) {
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      sc[u][j] = (seen >> (4 * u + j)) & 1 ? fp32_value(sc[u][j] * f[u][j]) : -INFINITY;
  const float most = Rows<NV, VT>::largest(sc);
  if (rows.moves(most)) rows.move(most);
  rows.template weights<SCALED>(sc, vs[0], vs[1], masked, seen, hi, lo);
}

// One pass over this workgroup's pieces of the line.  Products on MFMA with the
// layouts of tree_attention.hip; weights in two parts of 16 bits, so that they are
// off by 2^-17 and not by 2^-9, which takes half as many products again.
//
// Many rows are bound by the vector units (an exponential and a dozen further
// operations per score), the loads of operands from LDS and the matrix units, which
// overlap little: 28 query heads' 128 sequences under 32768 slots of bf16 take 149
// us, of which the products alone are 60 and the fixed work about 35.  Few rows, and
// short prefixes, are bound by that fixed work: a piece waits for its page numbers,
// then for its first tiles, 4 to 10 us, whatever its length.  32 sequences under
// 8011 slots of int8 and 700 of their own: 29 us; 40 with drafts of 6 tokens under 5
// prefixes of up to 3003 slots of e4m3: 65; 4 under 700: 12.
template <typename T, int FMT, int DP, int MT, int SM> struct SharedTiles {
  typedef UnitRegs<T, FMT, DP, 0> Regs;  // row blocks of a head meet its cache in the L2
  static constexpr int WAVES = kWaves, NV = Regs::NV, NQ = DP / 32, PITCH = DP + 4;
  // the weights' type in the second product: codes and bf16 values are exact in bf16
  typedef typename std::conditional<FMT == KV_16BIT, T, BF16>::type VT;
  static constexpr bool SCALED = FMT != KV_16BIT;
  static constexpr int TILE = 16 * WAVES, PAIRS = WAVES / 2;

  struct Stage {
    u32x4 k[PAIRS][2][NQ][64];   // pair of units, unit, k-step, lane
    u32x2 v[PAIRS][NV][64][2];   // pair, element, lane, unit
    float ks[TILE], vs[TILE];
  };
  union Lds {
    Stage stage[2];
    float many[WAVES][16 * MT][PITCH];  // output rows: a wave's own
    float few[WAVES][16 * SM][PITCH];   // every wave's part of the same
  };

  // Where the sums of a piece go, and what the join needs to find them.
  struct To {
    float* sums;
    float2* stats;
    int64_t kind;  // of the rows, in s.whole and s.pieces
    __device__ __forceinline__ To(const SharedArgs& s, const SharedShare& p)
        : sums(p.cut ? s.t.partial : s.whole), stats(p.cut ? s.t.stats : s.whole_stats), kind(p.prefix ? 0 : s.rows) {}
    // row r of the piece
    __device__ __forceinline__ int64_t row(const SharedArgs& s, const SharedShare& p, const SharedRow& at, int r) const {
      const int64_t out = kind + at.out_row(s.t);
      const int slot = (p.slot() << s.block_log) + r;
      if (p.begins) s.pieces[out] = int2{p.cut ? slot : -1, p.pieces};
      return p.cut ? slot : out;
    }
  };

  // Tiles of 16 slots per wave for 16 MT rows per wave.  Each wave loads one unit
  // of 16 slots, makes its operands and puts them into LDS; two tiles there, and
  // one more on its way to registers.
  static __device__ void many(const SharedArgs& s, const SharedShare& p, Lds& lds, float (&note)[2][WAVES],
                              int64_t (&out_row)[WAVES][16 * (MT > SM ? MT : SM)]) {
    const TreeArgs& a = s.t;
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const int wave = uniform(threadIdx.x >> 6);
    const int d = a.c.d;
    int pages = load_pages(a, p, p.from), pages_ahead = -1, held = 0;
    // page of this wave's unit of tile i; there: a bit for each unit of the tile that is there
    constexpr int HELD = 64 / WAVES;  // tiles whose pages 64 lanes hold
    constexpr uint32_t UNITS = (1u << WAVES) - 1;
    const auto page = [&](int i, uint32_t& there) {
      if (i - held >= HELD) {
        pages = pages_ahead;
        held += HELD;
      }
      if (i - held == HELD - 2) pages_ahead = load_pages(a, p, p.from + (held + HELD) * TILE);
      const int at = WAVES * (i - held);
      there = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(pages >= 0) >> at) & UNITS;
      return __builtin_amdgcn_readlane(pages, at + wave);
    };
    Regs kv;
    const auto load = [&](int i, int n) {
      const Unit<FMT> u(a, p.h, p.from + i * TILE + 16 * wave, p.stop, n);
      kv.load_keys(u, d);
      kv.load_values(u, d);
    };
    bool left_out = false;
    uint32_t there, there_ahead;
    const int page0 = page(0, there);
    load(0, page0);
    int page_ahead = page(1, there_ahead);

    u32x4 q[MT][NQ];
    SharedRow row[MT];
    Rows<NV, VT> rows[MT];
    int below = SharedRow::kAll;  // slots that all rows see
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      row[m] = SharedRow(s, p, 16 * (MT * wave + m) + col);
      shared_queries<T, FMT, MT == 1>(a, row[m], q[m]);
      rows[m].clear();
      below = min(below, row[m].limit);
    }
    for (int m = 8; m; m >>= 1) below = min(below, __shfl_xor(below, m));
    if (lane == 0) note[0][wave] = __builtin_bit_cast(float, below);
    __syncthreads();  // the last piece is read
#pragma unroll
    for (int w = 0; w < WAVES; ++w) below = min(below, __builtin_bit_cast(int, note[0][w]));
    below = uniform(below);
    // a tile that not every row sees whole
    const auto edge = [&](int i, uint32_t units) {
      return units != UNITS || p.from + (i + 1) * TILE > min(below, p.stop) || p.from + i * TILE < p.w.begin;
    };
    const auto put = [&](int i, uint32_t units) {
      Stage& st = lds.stage[i & 1];
      if (edge(i, units)) left_out |= kv.take_out_non_finite();
#pragma unroll
      for (int n = 0; n < NQ; ++n) st.k[wave >> 1][wave & 1][n][lane] = kv.keys(n);
#pragma unroll
      for (int x = 0; x < NV; x += 2) {
        u32x2 even, odd;
        kv.values2(x, even, odd);
        st.v[wave >> 1][x][lane][wave & 1] = even;
        st.v[wave >> 1][x + 1][lane][wave & 1] = odd;
      }
      if constexpr (SCALED) {
        if (col == 0) {
          *reinterpret_cast<f32x4*>(&st.ks[16 * wave + 4 * quad]) = kv.ks;
          *reinterpret_cast<f32x4*>(&st.vs[16 * wave + 4 * quad]) = kv.vs;
        }
      }
    };
    put(0, there);
    uint32_t there_next = there;  // of the tile in LDS
    load(1, page_ahead);
    there = there_ahead;
    page_ahead = page(2, there_ahead);
    const bool work = 16 * MT * wave < p.rows;  // else this wave only loads

#pragma unroll 1
    for (int i = 0; i < p.tiles; ++i) {
      __syncthreads();
      const Stage& st = lds.stage[i & 1];
      const uint32_t there_now = there_next;
      const bool masked = edge(i, there_now);
      if (i + 1 < p.tiles) {
        put(i + 1, there);
        there_next = there;
        load(i + 2, page_ahead);
        there = there_ahead;
        page_ahead = page(i + 3, there_ahead);
      }
      if (!work) continue;
      // Two pairs of units: the weights of one, on the vector units, may be computed
      // between the products of the other, on the matrix units.
      static_assert(PAIRS == 2, "the order of the steps below");
      f32x4 sc[PAIRS][MT][2], w[MT][2], f[2], vs[2];
      float most[MT];
      const auto scores = [&](int pair) {
#pragma unroll
        for (int m = 0; m < MT; ++m) sc[pair][m][0] = sc[pair][m][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          const u32x4 k0 = st.k[pair][0][n][lane], k1 = st.k[pair][1][n][lane];
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            sc[pair][m][0] = mfma16<T>(k0, q[m][n], sc[pair][m][0]);
            sc[pair][m][1] = mfma16<T>(k1, q[m][n], sc[pair][m][1]);
          }
        }
      };
      const auto weights = [&](int pair) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          f[u] = f32x4{a.scale, a.scale, a.scale, a.scale};
          vs[u] = f32x4{1.f, 1.f, 1.f, 1.f};
          if constexpr (SCALED) {
            f[u] *= *reinterpret_cast<const f32x4*>(&st.ks[32 * pair + 16 * u + 4 * quad]);
            vs[u] = *reinterpret_cast<const f32x4*>(&st.vs[32 * pair + 16 * u + 4 * quad]);
          }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) most[m] = weights_at_once(rows[m], sc[pair][m], f, w[m]);
      };
      u32x4 hi[MT], lo[MT];
      // masks, or another maximum
      const auto look = [&](int pair) {
        bool move = masked;
#pragma unroll
        for (int m = 0; m < MT; ++m) move |= weights_move<VT>(most[m]);
        if (!move) {
#pragma unroll
          for (int m = 0; m < MT; ++m) take_weights<NV, VT, SCALED>(rows[m], w[m], vs, hi[m], lo[m]);
          return;
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          uint32_t seen = 0xff;
          if (masked) {
            const int slot = p.from + i * TILE + 32 * pair;
            seen = shared_seen(a, p, row[m], slot, there_now >> (2 * pair) & 3);
          }
          weights_by_maximum<NV, VT, SCALED>(rows[m], sc[pair][m], f, vs, masked, seen, hi[m], lo[m]);
        }
      };
      const auto sums = [&](int pair) {
#pragma unroll
        for (int x = 0; x < NV; ++x) {
          const u32x4 v = *reinterpret_cast<const u32x4*>(&st.v[pair][x][lane][0]);
#pragma unroll
          for (int m = 0; m < MT; ++m) rows[m].o[x] = mfma16<VT>(v, hi[m], rows[m].o[x]);
#pragma unroll
          for (int m = 0; m < MT; ++m) rows[m].o[x] = mfma16<VT>(v, lo[m], rows[m].o[x]);
        }
      };
      // Both pairs' scores first where registers allow it (codes' scales take more of
      // them): 128 rows under 32768 slots of bf16 149 us instead of 156, but 40
      // sequences of e4m3 70 instead of 64.
      scores(0);
      if constexpr (!SCALED) scores(1);
      weights(0);
      look(0);
      sums(0);
      if constexpr (SCALED) scores(1);
      weights(1);
      look(1);
      sums(1);
    }

    // every wave has its rows to itself; through LDS for whole lines of stores
    if constexpr (!SCALED) {
#pragma unroll
      for (int m = 0; m < MT; ++m) left_out |= rows[m].non_finite();
    }
    if (lane == 0) note[1][wave] = left_out ? 1.f : 0.f;
    const int r0 = 16 * MT * wave, r1 = min(p.rows, r0 + 16 * MT);
    __syncthreads();
    const To to(s, p);
    float (*mine)[PITCH] = lds.many[wave];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const float total = sum_quads(rows[m].sum);
      const int r = 16 * m + col;
      rows[m].put(mine[r], 1.0f);
      if (quad == 0 && r0 + r < r1) {
        const int64_t at = to.row(s, p, row[m], r0 + r);
        to.stats[at] = float2{rows[m].top, total};
        out_row[wave][r] = at;
      }
    }
    wave_sync();
    float any = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) any += note[1][w];
    if (__builtin_expect(uniform(any != 0.f), 0)) {
      set_shared_non_finite<T, FMT>(s, p, mine, r0, r1, p.from, TILE, TILE);
      wave_sync();
    }
    constexpr int LINE = DP / 4;  // lanes of a row
    const int c = 4 * (lane % LINE);
    for (int r = lane / LINE; r < 16 * MT; r += 64 / LINE) {
      if (r0 + r >= r1 || c >= d) continue;
      *reinterpret_cast<f32x4*>(to.sums + out_row[wave][r] * d + c) = *reinterpret_cast<const f32x4*>(&mine[r][c]);
    }
  }

  // Tiles of 32 slots for up to 16 SM rows: a wave for itself, loads straight to
  // operands, as tree_attention_stream does; the waves join in LDS.
  static __device__ void few(const SharedArgs& s, const SharedShare& p, Lds& lds,
                             float (&tops)[WAVES][16 * SM], float (&sums)[WAVES][16 * SM],
                             int64_t (&out_row)[WAVES][16 * (MT > SM ? MT : SM)]) {
    const TreeArgs& a = s.t;
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const int wave = uniform(threadIdx.x >> 6);
    const int d = a.c.d;
    constexpr int STEP = kWaveSlots * WAVES;
    const auto page = [&](int slot) { return page_of(a, p.table, slot, p.stop); };
    const auto there = [&](int n) { return n >= 0 && n < a.c.pages; };
    int slot = p.from + kWaveSlots * wave;
    int p0 = page(slot), p1 = page(slot + 16);
    Regs kv[2];
    bool left_out = false, whole;
    {
      const Unit<FMT> u0(a, p.h, slot, p.stop, p0), u1(a, p.h, slot + 16, p.stop, p1);
      whole = u0.whole && u1.whole;
      kv[0].load_keys(u0, d);
      kv[1].load_keys(u1, d);
      kv[0].load_values(u0, d);
      kv[1].load_values(u1, d);
    }
    int next0 = page(slot + STEP), next1 = page(slot + STEP + 16);
    u32x4 q[SM][NQ];
    SharedRow row[SM];
    Rows<NV, VT> rows[SM];
    int below = SharedRow::kAll;
#pragma unroll
    for (int m = 0; m < SM; ++m) {
      row[m] = SharedRow(s, p, 16 * m + col);
      shared_queries<T, FMT, MT == 1>(a, row[m], q[m]);
      rows[m].clear();
      below = min(below, row[m].limit);
    }
    for (int m = 8; m; m >>= 1) below = min(below, __shfl_xor(below, m));
    below = uniform(below);

#pragma unroll 1
    for (; slot < p.stop; slot += STEP) {
      f32x4 sc[SM][2];
#pragma unroll
      for (int m = 0; m < SM; ++m) sc[m][0] = sc[m][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const u32x4 k0 = kv[0].keys(n), k1 = kv[1].keys(n);
#pragma unroll
        for (int m = 0; m < SM; ++m) {
          sc[m][0] = mfma16<T>(k0, q[m][n], sc[m][0]);
          sc[m][1] = mfma16<T>(k1, q[m][n], sc[m][1]);
        }
      }
      f32x4 f[2] = {{a.scale, a.scale, a.scale, a.scale}, {a.scale, a.scale, a.scale, a.scale}};
      if constexpr (SCALED) {
        f[0] *= kv[0].ks;
        f[1] *= kv[1].ks;
      }
      const bool masked = !whole || slot + kWaveSlots > below || slot < p.w.begin;
      if (masked) {
        left_out |= kv[0].take_out_non_finite();
        left_out |= kv[1].take_out_non_finite();
      }
      const Unit<FMT> n0(a, p.h, slot + STEP, p.stop, next0), n1(a, p.h, slot + STEP + 16, p.stop, next1);
      kv[0].load_keys(n0, d);  // while this tile's weights are computed
      kv[1].load_keys(n1, d);
      u32x4 hi[SM], lo[SM];
#pragma unroll
      for (int m = 0; m < SM; ++m) {
        uint32_t seen = 0xff;
        if (masked) seen = shared_seen(a, p, row[m], slot, (there(p0) ? 1u : 0u) | (there(p1) ? 2u : 0u));
        const f32x4 vs[2] = {kv[0].vs, kv[1].vs};
        weights_by_maximum<NV, VT, SCALED>(rows[m], sc[m], f, vs, masked, seen, hi[m], lo[m]);
      }
#pragma unroll
      for (int x = 0; x < NV; x += 2) {
        u32x2 e0, o0, e1, o1;
        kv[0].values2(x, e0, o0);
        kv[1].values2(x, e1, o1);
        const u32x4 even = {e0[0], e0[1], e1[0], e1[1]}, odd = {o0[0], o0[1], o1[0], o1[1]};
#pragma unroll
        for (int m = 0; m < SM; ++m) {
          rows[m].o[x] = mfma16<VT>(even, hi[m], rows[m].o[x]);
          rows[m].o[x + 1] = mfma16<VT>(odd, hi[m], rows[m].o[x + 1]);
        }
#pragma unroll
        for (int m = 0; m < SM; ++m) {
          rows[m].o[x] = mfma16<VT>(even, lo[m], rows[m].o[x]);
          rows[m].o[x + 1] = mfma16<VT>(odd, lo[m], rows[m].o[x + 1]);
        }
      }
      kv[0].load_values(n0, d);
      kv[1].load_values(n1, d);
      whole = n0.whole && n1.whole;
      p0 = next0;
      p1 = next1;
      next0 = page(slot + 2 * STEP);
      next1 = page(slot + 2 * STEP + 16);
    }

    // join the waves: common maximum, scaled sums
    __syncthreads();  // the last piece is read
#pragma unroll
    for (int m = 0; m < SM; ++m) {
      const float sum = sum_quads(rows[m].sum);
      if (quad == 0) {
        tops[wave][16 * m + col] = rows[m].top;
        sums[wave][16 * m + col] = sum;
      }
    }
    const To to(s, p);
    if (wave == 0) {
#pragma unroll
      for (int m = 0; m < SM; ++m) {
        const int r = 16 * m + col;
        if (quad == 0 && r < p.rows) out_row[0][r] = to.row(s, p, row[m], r);
      }
    }
    __syncthreads();
    const auto common = [&](int r) {
      float most = tops[0][r];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) most = fmaxf(most, tops[w][r]);
      return most;
    };
#pragma unroll
    for (int m = 0; m < SM; ++m) {
      const int r = 16 * m + col;
      rows[m].put(lds.few[wave][r], __builtin_amdgcn_exp2f(rows[m].top - common(r)));
      if constexpr (!SCALED) left_out |= rows[m].non_finite();
    }
    if (__builtin_expect(left_out, false)) {
      wave_sync();
      set_shared_non_finite<T, FMT>(s, p, lds.few[wave], 0, p.rows, p.from + kWaveSlots * wave, STEP, kWaveSlots);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.rows * (d / 4); e += 64 * WAVES) {
      const int r = e / (d / 4), c = 4 * (e - r * (d / 4));
      const float most = common(r);
      float total = 0.f;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        total += sums[w][r] * __builtin_amdgcn_exp2f(tops[w][r] - most);
        v += *reinterpret_cast<const f32x4*>(&lds.few[w][r][c]);
      }
      *reinterpret_cast<f32x4*>(to.sums + out_row[0][r] * d + c) = v;
      if (c == 0) to.stats[out_row[0][r]] = float2{most, total};
    }
  }
};

template <typename T, int FMT, int DP, int MT, int SM>
__global__ __launch_bounds__(64 * kWaves, shared_groups(DP)) void shared_prefix_tiles(SharedArgs s) {
  typedef SharedTiles<T, FMT, DP, MT, SM> K;
  __shared__ __align__(16) typename K::Lds lds;
  __shared__ float note[2][K::WAVES], tops[K::WAVES][16 * SM], sums[K::WAVES][16 * SM];
  __shared__ int64_t out_row[K::WAVES][16 * (MT > SM ? MT : SM)];  // where a row's sums go, in rows
  SharedShare p(s);
  while (p.next(s)) {
    if (p.few) K::few(s, p, lds, tops, sums, out_row);
    else K::many(s, p, lds, note, out_row);
    p.done();
  }
}

// Bound by three trips of loads that wait for each other (where the pieces are,
// their sums, the row's end): 48 rows 4 us, 896 rows of some 30 pieces 6, 9600 rows 10.
//
// Adds the pieces of one query row, those of the prefix and its own, in order:
// lanes 0 - 31 and 32 - 63 of each of WAVES waves take every 2 WAVES-th piece with
// a running maximum, 4 (and, beyond 128, 4 more) elements per lane.
constexpr int kSharedJoinRows = 8;

template <typename T, int WAVES>
__global__ __launch_bounds__(64 * (WAVES == 1 ? kSharedJoinRows : WAVES)) void shared_prefix_join(SharedArgs s) {
  typedef typename T::bits bits;
  constexpr int PARTS = 2 * WAVES;
  const TreeArgs& a = s.t;
  const int lane = threadIdx.x & 63, w_id = uniform(threadIdx.x >> 6);
  const int wave = WAVES == 1 ? 0 : w_id;
  const int qrow = WAVES == 1 ? static_cast<int>(blockIdx.x) * kSharedJoinRows + w_id : static_cast<int>(blockIdx.x);
  const bool mine = qrow < s.rows;
  const int at_row = min(qrow, s.rows - 1);
  const int bt = at_row / a.q_heads;
  const int b = bt / a.tokens, t = bt - b * a.tokens;
  // where the pieces are: all that is needed for it on its way at once
  int2 of_prefix = s.pieces[at_row], own = s.pieces[s.rows + at_row];
  const Lengths n(a, a.lens[b], a.new_lens ? a.new_lens[b] : a.tokens);
  const int shared = shared_of(s, b, n.len);
  if (t >= n.fresh || shared == 0) of_prefix.y = 0;
  if (t >= n.fresh || n.end <= shared) own.y = 0;
  const int count = of_prefix.y + own.y;
  // piece j's sums and statistics
  const auto piece = [&](int j, const float*& sums, float2& st) {
    const bool is_own = j >= of_prefix.y;
    const int2 p = is_own ? own : of_prefix;
    const int i = is_own ? j - of_prefix.y : j;
    if (p.x < 0) {
      const int64_t at = static_cast<int64_t>(is_own ? s.rows : 0) + at_row;
      sums = s.whole + at * a.c.d;
      st = s.whole_stats[at];
    } else {
      // the first, or the first of the i-th workgroup behind its own
      const int slot = p.x >> s.block_log, rr = p.x - (slot << s.block_log);
      const int64_t at = (static_cast<int64_t>(i ? (slot & ~1) + 2 * i : slot) << s.block_log) + rr;
      sums = a.partial + at * a.c.d;
      st = a.stats[at];
    }
  };

  const int part = 2 * wave + lane / 32;
  const int c0 = 4 * (lane % 32);
  const bool in0 = c0 < a.c.d, in1 = c0 + 128 < a.c.d;
  f32x4 v0 = {0.f, 0.f, 0.f, 0.f}, v1 = v0;
  float most = kLow, total = 0.f;
#pragma unroll 2
  for (int j = part; j < count; j += PARTS) {
    const float* p;
    float2 st;
    piece(j, p, st);
    const f32x4 p0 = in0 ? *reinterpret_cast<const f32x4*>(p + c0) : f32x4{0.f, 0.f, 0.f, 0.f};
    const f32x4 p1 = in1 ? *reinterpret_cast<const f32x4*>(p + c0 + 128) : f32x4{0.f, 0.f, 0.f, 0.f};
    const float now = fmaxf(most, st.x);
    const float was = __builtin_amdgcn_exp2f(most - now), f = __builtin_amdgcn_exp2f(st.x - now);
    most = now;
    total = total * was + st.y * f;
    v0 = v0 * was + p0 * f;
    v1 = v1 * was + p1 * f;
  }
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
  const int c = c0 + 128 * (lane / 32);  // lanes 32 - 63 write the second half
  if (!mine || c >= a.c.d) return;
  const float inv = 1.0f / total;
  const bool none = t >= n.fresh || total == 0.f;
  f32x4 o = lane < 32 ? v0 : v1;
  const f32x4 zero = o - o;
  if (__builtin_expect(zero[0] + zero[1] + zero[2] + zero[3] != 0.f, false)) {
    // a piece has a NaN or an infinity, which stays whatever the piece's factor:
    // one that is 0 in 32 bits makes NaN of an infinity
    f32x4 bad = {0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < count; ++j) {
      const float* p;
      float2 st;
      piece(j, p, st);
      const f32x4 sums = *reinterpret_cast<const f32x4*>(p + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) bad[e] += sums[e] - sums[e] == 0.f ? 0.f : sums[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = bad[e] == 0.f ? o[e] : bad[e];
  }
  *reinterpret_cast<u32x2*>(static_cast<bits*>(a.out) + static_cast<int64_t>(qrow) * a.c.d + c) =
      none ? u32x2{0, 0} : u32x2{narrow2<T>(f32x2{o[0] * inv, o[1] * inv}), narrow2<T>(f32x2{o[2] * inv, o[3] * inv})};
}

template <typename T, int FMT> int shared_tiles_typed(const SharedArgs& a, const SharedPlan& p, hipStream_t s) {
  static const char* what = "shared_prefix_attention launch";
  const dim3 grid(static_cast<unsigned>(p.grid));
#define MI355_SHARED(DP, MT, SM) \
  return launch(shared_prefix_tiles<T, FMT, DP, MT, SM>, grid, 64 * kWaves, 0, a, s, what)
  if (a.t.c.d > 128 && p.sm == 1) MI355_SHARED(256, 1, 1);
  if (a.t.c.d > 128) MI355_SHARED(256, 1, 2);
  if (a.t.c.d > 64) {
    if (p.mt == 1 && p.sm == 1) MI355_SHARED(128, 1, 1);
    if (p.mt == 1) MI355_SHARED(128, 1, 2);
    if (p.sm == 1) MI355_SHARED(128, 2, 1);
    MI355_SHARED(128, 2, 2);
  }
  if (p.mt == 1 && p.sm == 1) MI355_SHARED(64, 1, 1);
  if (p.mt == 1) MI355_SHARED(64, 1, 2);
  if (p.sm == 1) MI355_SHARED(64, 2, 1);
  MI355_SHARED(64, 2, 2);
#undef MI355_SHARED
}

// The kernels of a call: tiles, then the join.
template <typename T> int shared_prefix_run(const SharedArgs& a, const SharedPlan& p, int format, hipStream_t s) {
  const int st = format == KV_INT8   ? shared_tiles_typed<T, KV_INT8>(a, p, s)
                 : format == KV_E4M3 ? shared_tiles_typed<T, KV_E4M3>(a, p, s)
                                     : shared_tiles_typed<T, KV_16BIT>(a, p, s);
  if (st != MI355_OK) return st;
  static const char* what = "shared_prefix_attention join launch";
  const auto grid = [&](int64_t groups) { return dim3(static_cast<unsigned>(groups)); };
  const int64_t rows = a.rows;
  // as many waves a row as the card has room for at once
  if (8 * rows <= 8192) return launch(shared_prefix_join<T, 8>, grid(rows), 512, 0, a, s, what);
  if (2 * rows <= 8192) return launch(shared_prefix_join<T, 2>, grid(rows), 128, 0, a, s, what);
  return launch(shared_prefix_join<T, 1>, grid((rows + kSharedJoinRows - 1) / kSharedJoinRows), 64 * kSharedJoinRows, 0, a,
                s, what);
}

}  // namespace mi355
