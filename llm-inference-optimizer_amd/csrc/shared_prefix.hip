// Attention of a batch whose sequences share prefixes, over a paged cache, for
// gfx950: tree attention in which the slots below a sequence's shared length are
// those of its group's first sequence.
#include <type_traits>

#include "shared_prefix.h"

namespace mi355 {
namespace {

constexpr int kTile = 64;       // slots of a workgroup's tile
constexpr int kJoinRows = 8;

struct RowsArgs {
  KvCache c;
  const void* q;
  void* out;
  const int32_t *lens, *new_lens, *prefix_lens, *groups;
  const uint8_t* mask;
  int64_t mask_b, mask_t;
  int64_t qb, qt, qh;
  int batch, tokens, q_heads, group, group_count;
  float scale;
};

// A wave per query row.
template <typename T, int FMT> __global__ __launch_bounds__(64) void shared_prefix_rows(RowsArgs a) {
  typedef typename T::bits bits;
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int hq = static_cast<int>(row % a.q_heads), t = static_cast<int>(row / a.q_heads % a.tokens);
  const int b = static_cast<int>(row / a.q_heads / a.tokens), h = hq / a.group, d = a.c.d;
  const int cap = a.c.capacity();
  const int len = max(0, min(a.lens[b], cap)), fresh = max(0, min(a.new_lens ? a.new_lens[b] : a.tokens, a.tokens));
  const int end = min(len + fresh, cap);
  int first = b, shared = 0;
  if (a.groups) {
    int g0 = 0, g1 = 0;  // a boundary below an earlier one counts as that
    for (int g = 0; g < a.group_count; ++g) {
      g0 = max(g1, min(a.groups[g], a.batch));
      g1 = max(g0, min(a.groups[g + 1], a.batch));
      if (b >= g0 && b < g1) {
        first = g0;
        shared = max(0, min(a.prefix_lens[g], len));
        break;
      }
    }
  } else if (a.group_count) {
    const int even = a.batch / a.group_count;
    first = b / even * even;
    shared = max(0, min(a.prefix_lens[b / even], len));
  }
  __shared__ float q[256], weight[64];
  __shared__ int64_t rows[64];
  const bits* from = static_cast<const bits*>(a.q) + b * a.qb + t * a.qt + hq * a.qh;
  for (int e = lane; e < d; e += 64) q[e] = load_elem<T>(from, e);
  __syncthreads();
  float o[4] = {0, 0, 0, 0}, bad[4] = {0, 0, 0, 0}, most = kLow, sum = 0;
  for (int s0 = 0; s0 < (t < fresh ? end : 0); s0 += 64) {
    const int s = s0 + lane;
    int64_t at = s < end ? a.c.row(s < shared ? first : b, s, h) : -1;
    if (s >= len && at >= 0) {
      const int j = s - len;
      if (!(a.mask ? a.mask[b * a.mask_b + t * a.mask_t + j] != 0 : j <= t)) at = -1;
    }
    float score = -INFINITY;
    if (at >= 0) {
      float acc = 0;
      for (int e = 0; e < d; e += 4) {
        float k[4];
        if constexpr (FMT == KV_16BIT) {
          for (int i = 0; i < 4; ++i) k[i] = load_elem<T>(a.c.k, at * d + e + i);
        } else {
          decode4<FMT>(*reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.c.k) + at * d + e), k);
        }
        for (int i = 0; i < 4; ++i) acc += k[i] * q[e + i];
      }
      if constexpr (FMT != KV_16BIT) acc *= a.c.k_scale[at];
      score = acc * a.scale;
    }
    float top = score;
    for (int m = 32; m; m >>= 1) top = fmaxf(top, __shfl_xor(top, m));
    const float now = fmaxf(most, top), was = __builtin_amdgcn_exp2f(most - now);
    const float w = at >= 0 ? __builtin_amdgcn_exp2f(score - now) : 0.f;
    most = now;
    float part = w;
    for (int m = 32; m; m >>= 1) part += __shfl_xor(part, m);
    sum = sum * was + part;
    weight[lane] = w;
    rows[lane] = at;
    __syncthreads();
    for (int i = 0; i < 4; ++i) o[i] *= was;
    for (int j = 0; j < 64; ++j) {
      const int64_t r = rows[j];
      if (r < 0) continue;
      float vs = FMT != KV_16BIT ? a.c.v_scale[r] : 1.f;
      if (vs - vs != 0.f) vs = NAN;  // a scale that is not finite makes its row NaN
      for (int i = 0; 64 * i + lane < d; ++i) {
        const int e = 64 * i + lane;
        float v;
        if constexpr (FMT == KV_16BIT) {
          v = load_elem<T>(a.c.v, r * d + e);
        } else {
          float four[4];
          decode4<FMT>(static_cast<const uint8_t*>(a.c.v)[r * d + e], four);
          v = fp32_value(four[0] * vs);  // rounded: not fused into the test below
        }
        if (v - v == 0.f) o[i] += weight[j] * v;
        else bad[i] += v;
      }
    }
    __syncthreads();
  }
  for (int i = 0; 64 * i + lane < d; ++i) {
    const float v = bad[i] != 0.f || bad[i] != bad[i] ? bad[i] : sum == 0.f ? 0.f : o[i] / sum;
    store_elem<T>(a.out, row * d + 64 * i + lane, v);
  }
}

// What groups given by their boundaries mean for each sequence: one workgroup.
struct SetupArgs {
  const int32_t *lens, *prefix, *groups;
  int32_t *bounds, *first, *shared;
  int batch, count, cap;
};
__global__ __launch_bounds__(1024) void shared_prefix_setup(SetupArgs a) {
  __shared__ int scan[1024];
  int most = 0;
  for (int i0 = 0; i0 <= a.count; i0 += 1024) {  // a boundary below an earlier one counts as that
    const int i = i0 + threadIdx.x;
    scan[threadIdx.x] = i <= a.count ? max(0, min(a.groups[i], a.batch)) : 0;
    __syncthreads();
    for (int step = 1; step < 1024; step *= 2) {
      const int other = static_cast<int>(threadIdx.x) >= step ? scan[threadIdx.x - step] : 0;
      __syncthreads();
      scan[threadIdx.x] = max(scan[threadIdx.x], other);
      __syncthreads();
    }
    if (i <= a.count) a.bounds[i] = max(most, scan[threadIdx.x]);
    most = max(most, scan[1023]);
    __syncthreads();
  }
  __threadfence_block();
  __syncthreads();
  for (int b = threadIdx.x; b < a.batch; b += 1024) {
    int lo = 0, hi = a.count + 1;  // the first boundary beyond b
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (a.bounds[mid] > b) hi = mid;
      else lo = mid + 1;
    }
    const int g = lo - 1;
    const bool in = g >= 0 && g < a.count;
    a.first[b] = in ? a.bounds[g] : b;
    a.shared[b] = in ? max(0, min(a.prefix[g], min(a.lens[b], a.cap))) : 0;
  }
}

// Tiles of 64 slots for 64 MT rows: the four waves take 16 MT rows each and share
// a tile's MFMA operands through LDS, as tree_attention_wide does.
constexpr int shared_groups(int dp, int mt) { return dp <= 64 && mt == 1 ? 3 : dp <= 128 ? 2 : 1; }  // of a CU

template <typename T, int FMT, int DP, int MT>
__global__ __launch_bounds__(64 * kWaves, shared_groups(DP, MT)) void shared_prefix_tiles(SharedArgs s) {
  typedef UnitRegs<T, FMT, DP, 0> Regs;
  constexpr int NV = Regs::NV, NQ = DP / 32, PITCH = DP + 4, TILE = kTile;
  typedef typename std::conditional<FMT == KV_16BIT, T, BF16>::type VT;
  constexpr bool SCALED = FMT != KV_16BIT;
  struct Stage {
    u32x4 k[4][NQ][64];      // unit, k-step, lane
    u32x2 v[2][NV][64][2];   // pair of units, element, lane, unit of the pair
    float ks[TILE], vs[TILE];
  };
  constexpr int kFix = kWaves * 16 * MT * PITCH * 4;
  __shared__ __align__(16) uint8_t lds[2 * sizeof(Stage) > kFix ? 2 * sizeof(Stage) : kFix];
  __shared__ int non_finite[kWaves], limits[kWaves];
  __shared__ int64_t out_row[kWaves][16 * MT];  // where a row's sums go, in rows
  Stage* stage = reinterpret_cast<Stage*>(lds);
  const TreeArgs& a = s.t;
  const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
  const int wave = uniform(threadIdx.x >> 6);
  const int d = a.c.d;

  SharedShare p(s);
  while (p.next(s)) {
    const int t1 = p.t1;
    const auto there = [&](int n) { return n >= 0 && n < a.c.pages; };
    // the page of this wave's unit of a tile, and which of the tile's four units are there
    const auto page = [&](int tile, uint32_t& units) {
      const int last = (p.stop - tile * TILE + 15) / 16;  // units in use
      const uint32_t used = last >= 4 ? 0xfu : last <= 0 ? 0u : (1u << last) - 1;
      int mine = -1;
      units = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int n = page_of(a, p.table, tile * TILE + 16 * u, p.stop);
        units |= there(n) ? 1u << u : 0u;
        mine = u == wave ? n : mine;
      }
      units &= used;
      return mine;
    };
    bool left_out = false;
    Regs kv;
    uint32_t units, units_ahead;  // of the tile in registers, of the next
    const int first_page = page(p.t0, units);
    int ahead = page(p.t0 + 1, units_ahead);
    const auto load = [&](int tile, int n) {
      const Unit<FMT> u(a, p.h, tile * TILE + 16 * wave, p.stop, n);
      kv.load_keys(u, d);
      kv.load_values(u, d);
    };
    load(p.t0, first_page);

    u32x4 q[MT][NQ];
    SharedRow row[MT];
    Rows<NV, VT> rows[MT];
    int below = SharedRow::kAll;  // slots that all rows see
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      row[m] = SharedRow(s, p, 16 * (MT * wave + m) + col);
      shared_queries<T, FMT>(a, row[m], q[m]);
      rows[m].clear();
      below = min(below, row[m].limit);
    }
    for (int m = 8; m; m >>= 1) below = min(below, __shfl_xor(below, m));
    if (lane == 0) limits[wave] = below;
    __syncthreads();  // the last piece is read
    const int all_see = uniform(min(min(limits[0], limits[1]), min(limits[2], limits[3])));
    // a tile that not every row sees whole
    const auto edge = [&](int tile, uint32_t units) {
      return units != 0xf || (tile + 1) * TILE > all_see || tile * TILE < p.w.begin;
    };
    // this wave's unit of a tile: registers -> LDS
    const auto put = [&](int tile) {
      Stage& st = stage[tile & 1];
      if (edge(tile, units)) left_out |= kv.take_out_non_finite();
#pragma unroll
      for (int n = 0; n < NQ; ++n) st.k[wave][n][lane] = kv.keys(n);
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
    put(p.t0);
    uint32_t units_now = units;  // of the tile in LDS
    load(p.t0 + 1, ahead);
    units = units_ahead;
    ahead = page(p.t0 + 2, units_ahead);

    for (int tile = p.t0; tile < t1; ++tile) {
      __syncthreads();
      const Stage& st = stage[tile & 1];
      const bool masked = edge(tile, units_now);
      uint32_t seen[MT];  // both pairs of units
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        seen[m] = 0xffff;
        if (masked)
          seen[m] = shared_seen(a, p, row[m], tile * TILE, units_now) |
                    shared_seen(a, p, row[m], tile * TILE + 32, units_now >> 2) << 8;
      }
      if (tile + 1 < t1) {
        put(tile + 1);
        units_now = units;
        load(tile + 2, ahead);
        units = units_ahead;
        ahead = page(tile + 3, units_ahead);
      }
      f32x4 sc[2][MT][2];
#pragma unroll
      for (int pair = 0; pair < 2; ++pair) {
#pragma unroll
        for (int m = 0; m < MT; ++m) sc[pair][m][0] = sc[pair][m][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          const u32x4 k0 = st.k[2 * pair][n][lane], k1 = st.k[2 * pair + 1][n][lane];
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            sc[pair][m][0] = mfma16<T>(k0, q[m][n], sc[pair][m][0]);
            sc[pair][m][1] = mfma16<T>(k1, q[m][n], sc[pair][m][1]);
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          f32x4 f = {a.scale, a.scale, a.scale, a.scale};
          if constexpr (SCALED) f *= *reinterpret_cast<const f32x4*>(&st.ks[32 * pair + 16 * u + 4 * quad]);
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
          vs0 = *reinterpret_cast<const f32x4*>(&st.vs[32 * pair + 4 * quad]);
          vs1 = *reinterpret_cast<const f32x4*>(&st.vs[32 * pair + 16 + 4 * quad]);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
          rows[m].template weights<SCALED>(sc[pair][m], vs0, vs1, masked, seen[m] >> (8 * pair), hi[pair][m],
                                           lo[pair][m]);
      }
#pragma unroll
      for (int x = 0; x < NV; ++x) {
        const u32x4 v0 = *reinterpret_cast<const u32x4*>(&st.v[0][x][lane][0]);
        const u32x4 v1 = *reinterpret_cast<const u32x4*>(&st.v[1][x][lane][0]);
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
    const int r0 = 16 * MT * wave, r1 = min(p.rows, r0 + 16 * MT);
    __syncthreads();
    float (*mine)[PITCH] = reinterpret_cast<float (*)[PITCH]>(lds) + r0;
    const int64_t slot = p.slot();
    float* to = p.cut ? a.partial : s.whole + (p.prefix ? 0 : static_cast<int64_t>(s.rows) * d);
    float2* to_stats = p.cut ? a.stats : s.whole_stats + (p.prefix ? 0 : s.rows);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const float total = sum_quads(rows[m].sum);
      const int r = 16 * m + col;
      rows[m].put(mine[r], 1.0f);
      if (quad == 0 && r0 + r < r1) {
        const int64_t at = p.cut ? slot * a.block_rows + r0 + r : row[m].out_row(a);
        to_stats[at] = float2{rows[m].top, total};
        out_row[wave][r] = at;
      }
    }
    wave_sync();
    if (__builtin_expect(uniform(non_finite[0] | non_finite[1] | non_finite[2] | non_finite[3]), 0)) {
      set_shared_non_finite<T, FMT>(s, p, mine, r0, r1, p.t0, 1, TILE);
      wave_sync();
    }
    constexpr int LINE = DP / 4;  // lanes of a row
    const int c = 4 * (lane % LINE);
    for (int r = lane / LINE; r < 16 * MT; r += 64 / LINE) {
      if (r0 + r >= r1 || c >= d) continue;
      *reinterpret_cast<f32x4*>(to + out_row[wave][r] * d + c) = *reinterpret_cast<const f32x4*>(&mine[r][c]);
    }
    p.done();
  }
}

// The pieces of a row in one stretch: workgroups [w0, w1], or a whole one.
struct Pieces {
  int64_t base;   // of the whole piece, in rows
  int w0, n;      // n pieces
  int start, rr;  // of the stretch's line for this head and block; the row's place in its block
  __device__ __forceinline__ Pieces() : base(0), w0(0), n(0), start(0), rr(0) {}
  __device__ __forceinline__ Pieces(const SharedArgs& s, int v, int r, int h, int share, int64_t whole) {
    const TreeArgs& a = s.t;
    const Stretch w = stretch_of(s, v);
    base = whole;
    n = w0 = start = rr = 0;
    if (w.tiles == 0) return;
    const int block = r / a.block_rows;
    rr = r - block * a.block_rows;
    const int piece = w.tiles + a.pad;
    start = a.starts[1 + v] + (h * w.blocks + block) * piece;
    w0 = (start + a.pad) / share;
    n = (start + piece - 1) / share - w0 + 1;
  }
};

// Adds the pieces of one query row, those of the prefix and its own, in order:
// lanes 0 - 31 and 32 - 63 of each of WAVES waves take every 2 WAVES-th piece with
// a running maximum, 4 (and, beyond 128, 4 more) elements per lane.
template <typename T, int WAVES>
__global__ __launch_bounds__(64 * (WAVES == 1 ? kJoinRows : WAVES)) void shared_prefix_join(SharedArgs s) {
  typedef typename T::bits bits;
  constexpr int PARTS = 2 * WAVES;
  const TreeArgs& a = s.t;
  const int lane = threadIdx.x & 63, w_id = uniform(threadIdx.x >> 6);
  const int wave = WAVES == 1 ? 0 : w_id;
  const int qrow = WAVES == 1 ? static_cast<int>(blockIdx.x) * kJoinRows + w_id : static_cast<int>(blockIdx.x);
  const bool mine = qrow < s.rows;
  const int at_row = min(qrow, s.rows - 1);
  const int hq = at_row % a.q_heads, bt = at_row / a.q_heads;
  const int t = bt % a.tokens, b = bt / a.tokens;
  const int h = hq / a.group, gq = hq - h * a.group;
  const Lengths len(a, a.lens[b], a.new_lens ? a.new_lens[b] : a.tokens);
  const int share = a.starts[0];
  int first = b;
  const int shared = shared_of(s, b, len.len, &first);
  Pieces of_prefix, own;
  if (t < len.fresh) {
    if (shared > 0) {
      int g = 0;
      if (s.bounds) {
        int lo = 0, hi = s.groups + 1;  // the first boundary beyond b
        while (lo < hi) {
          const int mid = (lo + hi) / 2;
          if (s.bounds[mid] > b) hi = mid;
          else lo = mid + 1;
        }
        g = lo - 1;
      } else {
        g = b / s.even;
      }
      of_prefix = Pieces(s, g, (b - first) * s.mt_rows + t * a.group + gq, h, share, at_row);
    }
    own = Pieces(s, s.groups + b, t * a.group + gq, h, share, static_cast<int64_t>(s.rows) + at_row);
  }
  const int count = of_prefix.n + own.n;
  // piece j's sums and statistics
  const auto piece = [&](int j, const float*& sums, float2& st) {
    const bool is_own = j >= of_prefix.n;
    const Pieces& p = is_own ? own : of_prefix;
    if (p.n == 1) {
      sums = s.whole + p.base * a.c.d;
      st = s.whole_stats[p.base];
    } else {
      const int w = p.w0 + (is_own ? j - of_prefix.n : j);
      const int64_t at = (2 * static_cast<int64_t>(w) + (w * share >= p.start ? 0 : 1)) * a.block_rows + p.rr;
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
  const bool none = t >= len.fresh || total == 0.f;
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

int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }

// Row blocks and grid of a call, and its workspace.
struct Plan {
  int mt, block_rows, pad, grid;
  int64_t partial, stats, whole, whole_stats, starts, bounds, first, shared, bytes;  // offsets
};

// False where the line of tiles could pass 2^31.
bool plan(const mi355_kv_cache& c, int64_t batch, int64_t tokens, int64_t q_heads, int64_t groups, int cus, Plan* to) {
  Plan& p = *to;
  const int dp = c.head_dim <= 64 ? 64 : c.head_dim <= 128 ? 128 : 256;
  const int64_t mt_rows = tokens * (q_heads / c.kv_heads);
  const int64_t group_rows = groups ? (batch + groups - 1) / groups * mt_rows : mt_rows;  // on average
  p.mt = group_rows <= 64 || dp == 256 ? 1 : 2;
  p.block_rows = 16 * p.mt * kWaves;
  p.pad = 4;
  p.grid = cus * shared_groups(dp, p.mt);
  const int64_t tiles = (c.table_width * c.page_size + kTile - 1) / kTile + p.pad + 1;  // of a piece at most
  // row blocks of all prefixes and of all sequences
  const int64_t blocks = (batch * mt_rows / p.block_rows + groups) + batch * ((mt_rows + p.block_rows - 1) / p.block_rows);
  if (c.kv_heads * blocks > (0x7fffffff - 65536 * int64_t{64}) / tiles) return false;
  const int64_t rows = batch * tokens * q_heads;
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t was = at;
    at += up16(bytes);
    return was;
  };
  p.partial = take(2 * int64_t{p.grid} * p.block_rows * c.head_dim * 4);
  p.stats = take(2 * int64_t{p.grid} * p.block_rows * 8);
  p.whole = take(2 * rows * c.head_dim * 4);
  p.whole_stats = take(2 * rows * 8);
  p.starts = take(4 * (groups + batch + 2));
  p.bounds = take(4 * (groups + 1));
  p.first = take(4 * batch);
  p.shared = take(4 * batch);
  p.bytes = at;
  return true;
}

template <typename T, int FMT> int tiles_typed(const SharedArgs& a, const Plan& p, hipStream_t s) {
  static const char* what = "shared_prefix_attention launch";
  const dim3 grid(static_cast<unsigned>(p.grid));
#define MI355_SHARED(DP, MT) return launch(shared_prefix_tiles<T, FMT, DP, MT>, grid, 64 * kWaves, 0, a, s, what)
  if (a.t.c.d > 128) MI355_SHARED(256, 1);
  if (a.t.c.d > 64 && p.mt == 1) MI355_SHARED(128, 1);
  if (a.t.c.d > 64) MI355_SHARED(128, 2);
  if (p.mt == 1) MI355_SHARED(64, 1);
  MI355_SHARED(64, 2);
#undef MI355_SHARED
}

template <typename T> int join_typed(const SharedArgs& a, const Plan& p, hipStream_t s) {
  static const char* what = "shared_prefix_attention join launch";
  const auto grid = [&](int64_t groups) { return dim3(static_cast<unsigned>(groups)); };
  const int64_t rows = a.rows;
  if (8 * rows <= 8192) return launch(shared_prefix_join<T, 8>, grid(rows), 512, 0, a, s, what);
  if (2 * rows <= 8192) return launch(shared_prefix_join<T, 2>, grid(rows), 128, 0, a, s, what);
  return launch(shared_prefix_join<T, 1>, grid((rows + kJoinRows - 1) / kJoinRows), 64 * kJoinRows, 0, a, s, what);
}

// n / u for n < 2^27 as n * mul >> shift: ceil(2^(31 + L) / u) with L = ceil(log2 u) fits 32 bits, and the product is
// off by less than 2^L in 2^(31 + L), too little to reach the next integer
void reciprocal(uint32_t u, uint32_t* mul, uint32_t* shift) {
  uint32_t log = 0;
  while ((uint64_t{1} << log) < u) ++log;
  *mul = static_cast<uint32_t>(((uint64_t{1} << (31 + log)) + u - 1) / u);
  *shift = 31 + log;
}

}  // namespace

int64_t shared_prefix_workspace(const mi355_kv_cache& cache, int64_t batch, int64_t tokens, int64_t q_heads,
                                int64_t group_count) {
  int cus = 0;
  Plan p;
  if (compute_units(&cus) != MI355_OK || !plan(cache, batch, tokens, q_heads, group_count, cus, &p)) return 0;
  return p.bytes;
}

int shared_prefix_launch(const mi355_kv_cache& cache, const void* q, void* out, const int32_t* lens,
                         const int32_t* new_lens, const int32_t* prefix_lens, const int32_t* groups, int group_count,
                         const uint8_t* mask, int64_t mask_b, int64_t mask_t, int64_t batch, int tokens, int q_heads,
                         const int64_t* q_strides, float scale, int dtype, void* work, int64_t work_bytes,
                         hipStream_t stream) {
  int cus = 0;
  int st = compute_units(&cus);
  if (st != MI355_OK) return st;
  const int group = q_heads / static_cast<int>(cache.kv_heads);
  Plan p;
  if (!plan(cache, batch, tokens, q_heads, group_count, cus, &p) || work == nullptr || work_bytes < p.bytes) {
    const RowsArgs a{kv_cache_args(cache), q, out, lens, new_lens, prefix_lens, groups, mask, mask_b, mask_t,
                     q_strides[0], q_strides[1], q_strides[2], static_cast<int>(batch), tokens, q_heads, group,
                     group_count, scale * kLog2e};
    const dim3 grid(static_cast<unsigned>(batch * tokens * q_heads));
    const auto run = [&](auto* kernel) { return launch(kernel, grid, 64, 0, a, stream, "shared_prefix_attention launch"); };
    if (dtype == MI355_F16)
      return cache.format == KV_INT8   ? run(shared_prefix_rows<F16, KV_INT8>)
             : cache.format == KV_E4M3 ? run(shared_prefix_rows<F16, KV_E4M3>)
                                       : run(shared_prefix_rows<F16, KV_16BIT>);
    return cache.format == KV_INT8   ? run(shared_prefix_rows<BF16, KV_INT8>)
           : cache.format == KV_E4M3 ? run(shared_prefix_rows<BF16, KV_E4M3>)
                                     : run(shared_prefix_rows<BF16, KV_16BIT>);
  }
  uint8_t* base = static_cast<uint8_t*>(work);
  SharedArgs a{};
  a.t = TreeArgs{kv_cache_args(cache), q, out, lens, new_lens, mask, mask_b, mask_t, q_strides[0], q_strides[1],
                 q_strides[2], reinterpret_cast<float*>(base + p.partial), reinterpret_cast<float2*>(base + p.stats),
                 reinterpret_cast<int32_t*>(base + p.starts), static_cast<int>(batch), tokens, q_heads, group,
                 p.block_rows, 2, kTile, p.pad, p.grid, 0, 0, scale * kLog2e};
  reciprocal(static_cast<uint32_t>(cache.page_size / 16), &a.t.page_mul, &a.t.page_shift);
  a.prefix = prefix_lens;
  a.whole = reinterpret_cast<float*>(base + p.whole);
  a.whole_stats = reinterpret_cast<float2*>(base + p.whole_stats);
  a.groups = group_count;
  a.even = group_count ? static_cast<int>(batch / group_count) : 0;
  a.rows = static_cast<int>(batch * tokens * q_heads);
  a.mt_rows = tokens * group;
  reciprocal(static_cast<uint32_t>(a.mt_rows), &a.seq_mul, &a.seq_shift);
  reciprocal(static_cast<uint32_t>(group), &a.group_mul, &a.group_shift);
  if (groups != nullptr && group_count > 0) {
    int32_t *bounds = reinterpret_cast<int32_t*>(base + p.bounds), *first = reinterpret_cast<int32_t*>(base + p.first),
            *shared = reinterpret_cast<int32_t*>(base + p.shared);
    const SetupArgs setup{lens, prefix_lens, groups, bounds, first, shared, static_cast<int>(batch), group_count,
                          static_cast<int>(cache.table_width * cache.page_size)};
    st = launch(shared_prefix_setup, dim3(1), 1024, 0, setup, stream, "shared_prefix_attention setup launch");
    if (st != MI355_OK) return st;
    a.bounds = bounds;
    a.first = first;
    a.shared = shared;
  }
  if (dtype == MI355_F16) {
    st = cache.format == KV_INT8   ? tiles_typed<F16, KV_INT8>(a, p, stream)
         : cache.format == KV_E4M3 ? tiles_typed<F16, KV_E4M3>(a, p, stream)
                                   : tiles_typed<F16, KV_16BIT>(a, p, stream);
    return st != MI355_OK ? st : join_typed<F16>(a, p, stream);
  }
  st = cache.format == KV_INT8   ? tiles_typed<BF16, KV_INT8>(a, p, stream)
       : cache.format == KV_E4M3 ? tiles_typed<BF16, KV_E4M3>(a, p, stream)
                                 : tiles_typed<BF16, KV_16BIT>(a, p, stream);
  return st != MI355_OK ? st : join_typed<BF16>(a, p, stream);
}

}  // namespace mi355
