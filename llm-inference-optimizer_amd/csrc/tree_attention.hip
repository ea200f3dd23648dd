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
// Products on MFMA (v_mfma_f32_16x16x32), without LDS: a wave takes tiles of
// 32 slots and computes
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
// which a decode step has plenty to spare.  The maximum moves only when a score
// passes it by 2^8, so most tiles do not rescale O; weights then are at most 2^8.
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
// which would spread them to every row; the rows that see them get them added
// at the end.
#include <type_traits>

#include "kv_cache.h"

namespace mi355 {
namespace {

constexpr int kTile = 32;            // slots of a tile: two units of 16

constexpr int kWaves = 4;            // of a workgroup

// Waves that a SIMD holds at the registers of a kernel.
constexpr int simd_waves(int dp, int mt) { return mt == 1 && dp <= 64 ? 4 : mt == 1 && dp <= 128 ? 3 : dp * mt <= 256 ? 2 : 1; }
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLow = -1e30f;       // the running maximum before any score
constexpr float kSlack = 8.0f;       // log2 of how far scores may pass it

struct TreeArgs {
  KvCache c;
  const void* q;
  void* out;  // [batch, tokens, q_heads, d]
  const int32_t *lens, *new_lens;
  const uint8_t* mask;  // [batch, tokens, tokens] by strides, or null: a chain
  int64_t mask_b, mask_t;
  int64_t qb, qt, qh;
  float* partial;       // [2 workgroups][rows of a block][d]; null: no split
  float2* stats;        // [2 workgroups][rows of a block]: maximum and sum
  int32_t* starts;      // [1 + batch]: the workgroups' share of tiles, the first tile of each sequence
  int batch, tokens, q_heads, group;  // group = q_heads / kv_heads
  int mt, blocks;                     // row blocks of 16 mt rows
  int grid;                           // workgroups of the first kernel
  uint32_t page_mul, page_shift;      // unit / units per page = unit * page_mul >> page_shift
  float scale;                        // times log2 e
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Scalar load of read-only memory at a uniform index: counted apart from the
// vector loads in flight, which a vector load of a page number would wait for.
__device__ __forceinline__ int32_t scalar_load(const int32_t* p, int64_t i) {
  typedef const __attribute__((address_space(4))) int32_t* constant_ptr;
  return reinterpret_cast<constant_ptr>(reinterpret_cast<uintptr_t>(p))[i];
}

// One sequence: its context, new tokens, slots in use, and tiles per head and
// row block.
struct Seq {
  int len, fresh, end, tiles;
  __device__ __forceinline__ Seq(const TreeArgs& a, int len_, int fresh_) {
    const int cap = a.c.capacity();
    len = max(0, min(len_, cap));
    fresh = max(0, min(fresh_, a.tokens));
    end = min(len + fresh, cap);
    tiles = max(1, (end + kTile - 1) / kTile);
  }
  // by a scalar b
  static __device__ __forceinline__ Seq of(const TreeArgs& a, int b) {
    return Seq(a, scalar_load(a.lens, b), a.new_lens ? scalar_load(a.new_lens, b) : a.tokens);
  }
  // the tiles of sequence b0 + lane, 0 beyond the last
  static __device__ __forceinline__ int of_lane(const TreeArgs& a, int b0) {
    const int b = b0 + static_cast<int>(threadIdx.x & 63);
    return b < a.batch ? Seq(a, a.lens[b], a.new_lens ? a.new_lens[b] : a.tokens).tiles : 0;
  }
};

template <int CTRL, int ROWS> __device__ __forceinline__ int dpp_add(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
// Sum of v over this lane and those before it.
__device__ __forceinline__ int wave_scan(int v) {
  v = dpp_add<0x111, 0xf>(v);  // row_shr:1
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
  v = dpp_add<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
  return v;
}

// The line of tiles: sequence b has Seq::tiles of them for each of its heads
// and row blocks, head and block outermost.
struct Line {
  int len, fresh;  // of this lane's sequence among the first 64
  int first;       // tiles per head and block, of it and those before
  int total;       // of all sequences
  Line() = default;
  __device__ __forceinline__ explicit Line(const TreeArgs& a) {
    const int b = min(static_cast<int>(threadIdx.x & 63), a.batch - 1);
    len = a.lens[b];
    fresh = a.new_lens ? a.new_lens[b] : a.tokens;
    first = wave_scan(static_cast<int>(threadIdx.x & 63) < a.batch ? Seq(a, len, fresh).tiles : 0);
    total = __builtin_amdgcn_readlane(first, 63);
    for (int b0 = 64; b0 < a.batch; b0 += 64) total += __builtin_amdgcn_readlane(wave_scan(Seq::of_lane(a, b0)), 63);
    total *= a.c.heads * a.blocks;
  }
  // Sequence b < 64.
  __device__ __forceinline__ Seq seq(const TreeArgs& a, int b) const {
    return Seq(a, __builtin_amdgcn_readlane(len, b), __builtin_amdgcn_readlane(fresh, b));
  }
  // The sequence that tile `at` belongs to (batch: none) and its first tile.
  __device__ __forceinline__ int find(const TreeArgs& a, int at, int* start) const {
    const int hm = a.c.heads * a.blocks;
    int before = 0, upto = first;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
      if (b0) upto = wave_scan(Seq::of_lane(a, b0));
      const uint64_t past = __builtin_amdgcn_ballot_w64((before + upto) * hm > at);
      if (past) {
        const int i = uniform(__builtin_ctzll(past));
        *start = (before + (i ? __builtin_amdgcn_readlane(upto, i - 1) : 0)) * hm;
        return b0 + i;
      }
      before += __builtin_amdgcn_readlane(upto, 63);
    }
    *start = before * hm;
    return a.batch;
  }
  // For the join: the share, then the first tile of every sequence.
  __device__ __forceinline__ void write(const TreeArgs& a, int share, int32_t* to) const {
    const int lane = threadIdx.x & 63;
    if (lane == 0) to[0] = share;
    int before = 0, upto = first;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
      if (b0) upto = wave_scan(Seq::of_lane(a, b0));
      const int b = b0 + lane + 1;
      if (b < a.batch) to[1 + b] = (before + upto) * a.c.heads * a.blocks;
      before += __builtin_amdgcn_readlane(upto, 63);
    }
    if (lane == 0) to[1] = 0;
  }
};

// Tiles per workgroup: equal shares, a whole number of tiles for each wave.
__device__ __forceinline__ int line_share(int total, int grid) {
  return ((total + grid - 1) / grid + kWaves - 1) / kWaves * kWaves;
}

template <int FMT> __device__ __forceinline__ constexpr int elem_bytes() { return FMT == KV_16BIT ? 2 : 1; }

// The 16 slots of a unit: descriptors that end with its last slot in use.
template <int FMT> struct Unit {
  rsrc_t k, v, ks, vs;
  bool whole;  // 16 slots, all there
  __device__ __forceinline__ Unit(const TreeArgs& a, int h, int slot, int end, int page) {
    const int upp = a.c.page_size / 16;
    const int u = slot / 16;
    const int in_page = u - static_cast<int>((static_cast<uint64_t>(u) * a.page_mul) >> a.page_shift) * upp;
    int n = max(0, min(end - slot, 16));
    if (page < 0 || page >= a.c.pages) n = 0;
    whole = n == 16;
    const int64_t row = n ? (static_cast<int64_t>(page) * a.c.heads + h) * a.c.page_size + 16 * in_page : 0;
    const uint32_t bytes = static_cast<uint32_t>(n * a.c.d * elem_bytes<FMT>());
    k = make_rsrc(static_cast<const uint8_t*>(a.c.k) + row * a.c.d * elem_bytes<FMT>(), bytes);
    v = make_rsrc(static_cast<const uint8_t*>(a.c.v) + row * a.c.d * elem_bytes<FMT>(), bytes);
    if constexpr (FMT != KV_16BIT) {
      ks = make_rsrc(a.c.k_scale + row, static_cast<uint32_t>(4 * n));
      vs = make_rsrc(a.c.v_scale + row, static_cast<uint32_t>(4 * n));
    }
  }
};

// Page of a unit, or -1.  In a scalar register, as the descriptors made from
// it have to be (a vector one would make each load a loop over the lanes).
__device__ __forceinline__ int page_of(const TreeArgs& a, const int32_t* table, int slot, int end) {
  const int u = max(0, min(slot, end - 1)) / 16;  // without a branch: a table has a page at least
  const int page = scalar_load(table, static_cast<int64_t>((static_cast<uint64_t>(u) * a.page_mul) >> a.page_shift));
  return slot < end ? page : -1;
}

// Four codes of a dword, as MFMA operands of T: two dwords.
template <typename T, int FMT> __device__ __forceinline__ u32x2 widen_codes(uint32_t d) {
  if constexpr (FMT == KV_INT8) {
    return widen_i8x4<T>(d);
  } else if constexpr (T::code == MI355_F16) {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d, 1.0f, true))};
  } else {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d, 1.0f, true))};
  }
}

__device__ __forceinline__ float max_quads(float v) {  // over the 4 lanes of a column
  {
    const uint32_t b = as_u32(v);
    auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    const uint32_t lo = r[0], hi = r[1];
    v = fmaxf(as_f32(lo), as_f32(hi));
  }
  {
    const uint32_t b = as_u32(v);
    auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    const uint32_t lo = r[0], hi = r[1];
    v = fmaxf(as_f32(lo), as_f32(hi));
  }
  return v;
}
__device__ __forceinline__ float sum_quads(float v) {
  {
    const uint32_t b = as_u32(v);
    auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    const uint32_t lo = r[0], hi = r[1];
    v = as_f32(lo) + as_f32(hi);
  }
  {
    const uint32_t b = as_u32(v);
    auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    const uint32_t lo = r[0], hi = r[1];
    v = as_f32(lo) + as_f32(hi);
  }
  return v;
}

// The keys, values and scales of a tile in a lane's registers.
//   keys    unit u, load i: slot l % 16, elements (8-bit) 64 i + 16 quad .. + 15
//           or (16-bit) 32 i + 8 quad .. + 7
//   values  unit u, slot 4 quad + j, elements NV (l % 16) .. + NV - 1
//   scales  unit u, slots 4 quad .. 4 quad + 3
template <typename T, int FMT, int DP, int AUX> struct Tile {
  static constexpr int ES = FMT == KV_16BIT ? 2 : 1;
  static constexpr int NV = DP / 16;
  static constexpr int KL = DP * ES / 64;     // 16-byte key loads per unit
  static constexpr int VD = NV * ES / 4;      // dwords of a value per lane
  u32x4 k[2][KL];
  uint32_t v[2][4][VD];
  f32x4 ks[2], vs[2];

  __device__ __forceinline__ void load_keys(const Unit<FMT>& u0, const Unit<FMT>& u1, int d) {
    const int lane = threadIdx.x & 63, r = lane & 15, quad = lane >> 4;
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      const int byte = 64 * i + 16 * quad;
      const uint32_t off = byte < d * ES ? static_cast<uint32_t>(r * d * ES + byte) : kOob;
      k[0][i] = __builtin_amdgcn_raw_buffer_load_b128(u0.k, off, 0, AUX);
      k[1][i] = __builtin_amdgcn_raw_buffer_load_b128(u1.k, off, 0, AUX);
    }
    if constexpr (FMT != KV_16BIT) {
      ks[0] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(u0.ks, 16u * quad, 0, AUX));
      ks[1] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(u1.ks, 16u * quad, 0, AUX));
    }
  }

  __device__ __forceinline__ void load_values(const Unit<FMT>& u0, const Unit<FMT>& u1, int d) {
    const int lane = threadIdx.x & 63, r = lane & 15, quad = lane >> 4;
    if constexpr (FMT != KV_16BIT) {
      vs[0] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(u0.vs, 16u * quad, 0, AUX));
      vs[1] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(u1.vs, 16u * quad, 0, AUX));
    }
    const uint32_t first = NV * r < d ? static_cast<uint32_t>((4 * quad * d + NV * r) * ES) : kOob;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const rsrc_t rsrc = u ? u1.v : u0.v;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = j * d * ES;  // uniform: the scalar offset of the load
        if constexpr (VD == 1) {
          v[u][j][0] = __builtin_amdgcn_raw_buffer_load_b32(rsrc, first, at, AUX);
        } else if constexpr (VD == 2) {
          const u32x2 t = __builtin_amdgcn_raw_buffer_load_b64(rsrc, first, at, AUX);
          v[u][j][0] = t[0];
          v[u][j][1] = t[1];
        } else {
#pragma unroll
          for (int w = 0; w < VD / 4; ++w) {
            const u32x4 t = __builtin_amdgcn_raw_buffer_load_b128(rsrc, first + 16 * w, at, AUX);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[u][j][4 * w + e] = t[e];
          }
        }
      }
    }
  }

  // MFMA k-step n (32 of the DP elements) of unit u's keys.
  __device__ __forceinline__ u32x4 keys(int u, int n) const {
    if constexpr (FMT == KV_16BIT) {
      return k[u][n];
    } else {
      const u32x2 lo = widen_codes<T, FMT>(k[u][n / 2][2 * (n & 1)]), hi = widen_codes<T, FMT>(k[u][n / 2][2 * (n & 1) + 1]);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
  }

  // Elements x (even) and x + 1 of the 8 values: two V^T operands.
  __device__ __forceinline__ void values2(int x, u32x4& even, u32x4& odd) const {
#pragma unroll
    for (int p = 0; p < 4; ++p) {  // the slot pairs of a k-step
      const int u = p >> 1, j = 2 * (p & 1);
      if constexpr (FMT == KV_16BIT) {
        const uint32_t a = v[u][j][x / 2], b = v[u][j + 1][x / 2];
        even[p] = __builtin_amdgcn_perm(b, a, 0x05040100u);
        odd[p] = __builtin_amdgcn_perm(b, a, 0x07060302u);
      } else if constexpr (FMT == KV_E4M3) {
        const uint32_t a8 = v[u][j][x / 4], b8 = v[u][j + 1][x / 4];
        uint32_t a, b;
        if (x & 2) {
          a = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a8, 1.0f, true));
          b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b8, 1.0f, true));
        } else {
          a = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a8, 1.0f, false));
          b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b8, 1.0f, false));
        }
        even[p] = __builtin_amdgcn_perm(b, a, 0x05040100u);
        odd[p] = __builtin_amdgcn_perm(b, a, 0x07060302u);
      } else {
        // the upper half of an fp32 integer below 2^8 is its bf16 pattern
        const uint32_t a8 = v[u][j][x / 4] >> (8 * (x & 3)), b8 = v[u][j + 1][x / 4] >> (8 * (x & 3));
        even[p] = __builtin_amdgcn_perm(as_u32(static_cast<float>(static_cast<int8_t>(b8 & 0xff))),
                                        as_u32(static_cast<float>(static_cast<int8_t>(a8 & 0xff))), 0x07060302u);
        odd[p] = __builtin_amdgcn_perm(as_u32(static_cast<float>(static_cast<int8_t>((b8 >> 8) & 0xff))),
                                       as_u32(static_cast<float>(static_cast<int8_t>((a8 >> 8) & 0xff))), 0x07060302u);
      }
    }
  }

  // Zeroes the elements of the values that are NaN or infinite; whether any
  // lane had one.
  __device__ __forceinline__ bool take_out_non_finite() {
    if constexpr (FMT == KV_INT8) return false;
    bool hit = false;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int w = 0; w < VD; ++w) {
          const uint32_t e = v[u][j][w];
          uint32_t drop = 0;
          if constexpr (FMT == KV_E4M3) {
            // a byte of 0x7f behind its sign: adding 1 carries into the sign bit
            const uint32_t full = ((e & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
            drop = (full >> 7) * 0xffu;
          } else {
            constexpr uint32_t ex = T::code == MI355_F16 ? 0x7c00u : 0x7f80u;
            if ((e & ex) == ex) drop = 0xffffu;
            if ((e >> 16 & ex) == ex) drop |= 0xffff0000u;
          }
          hit |= drop != 0;
          v[u][j][w] = e & ~drop;
        }
    return __builtin_amdgcn_ballot_w64(hit) != 0;
  }
};

// Adds the NaN and infinities that take_out_non_finite left out of one wave's
// tiles to the output rows that see them: rare, and slow.  In LDS, where rows
// and elements can be indexed.  Weights do not matter to them.
template <typename T, int FMT, int PITCH>
__device__ __forceinline__ void add_non_finite(const TreeArgs& a, float (*acc)[PITCH], int b, int h, int row0, int rows,
                                               int len, int fresh, int first, int last) {
  const int lane = threadIdx.x & 63;
  for (int tile = first; tile < last; tile += kWaves) {
#pragma unroll 1
    for (int slot = tile * kTile; slot < (tile + 1) * kTile; ++slot) {
      const int64_t at = slot < len + fresh ? a.c.row(b, slot, h) : -1;
      if (at < 0) continue;
#pragma unroll 1
      for (int e = lane; e < a.c.d; e += 64) {
        float v;
        if constexpr (FMT == KV_16BIT) {
          v = load_elem<T>(a.c.v, at * a.c.d + e);
        } else {
          float f[4];
          decode4<FMT>(static_cast<const uint8_t*>(a.c.v)[at * a.c.d + e], f);
          v = f[0];
        }
        if (v - v == 0.f) continue;
#pragma unroll 1
        for (int r = 0; r < rows; ++r) {
          const int t = (row0 + r) / a.group, i = slot - len;
          const bool see = i < 0 || (t < fresh && (a.mask ? a.mask[b * a.mask_b + t * a.mask_t + i] != 0 : i <= t));
          if (see) acc[r][e] += v;
        }
      }
    }
  }
}

template <typename T, int FMT, int DP, int MT>
__global__ __launch_bounds__(64 * kWaves, simd_waves(DP, MT)) void tree_attention_split(TreeArgs a) {
  typedef typename T::bits bits;
  // rows that fit one block read the cache once; more blocks meet it in the L2
  typedef Tile<T, FMT, DP, MT == 4 ? 0 : kStreamAux> KvTile;
  constexpr int NV = KvTile::NV, NQ = DP / 32, ROWS = 16 * MT, PITCH = DP + 4;
  // the weights' type in the second product: codes and bf16 values are exact in bf16
  typedef typename std::conditional<FMT == KV_16BIT, T, BF16>::type VT;
  __shared__ float joined[kWaves][ROWS][PITCH];
  __shared__ float wave_max[kWaves][ROWS], wave_sum[kWaves][ROWS];

  const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
  const int wave = uniform(threadIdx.x >> 6);
  const int d = a.c.d, hm_count = a.c.heads * a.blocks;

  // this workgroup's tiles [at, last) of the line, or one (head, block) of one sequence
  int at, last, b, start;
  Line line;
  if (a.partial) {
    line = Line(a);
    const int share = line_share(line.total, a.grid);
    at = static_cast<int>(blockIdx.x) * share;
    last = at + share;
    b = line.find(a, at, &start);
    if (blockIdx.x == 0 && wave == 0) line.write(a, share, a.starts);
  } else {
    b = blockIdx.x / hm_count;
    start = 0;
    at = (blockIdx.x % hm_count) * Seq::of(a, b).tiles;
    last = at + 1;  // the first tile; widened to the whole below
  }
  const int line_first = at;

  while (b < a.batch && at < last) {
    const Seq s = a.partial && b < 64 ? line.seq(a, b) : Seq::of(a, b);
    const int len = s.len, fresh = s.fresh, tiles = s.tiles, end = s.end;
    const int hm = (at - start) / tiles, t0 = at - start - hm * tiles;
    if (hm >= hm_count) {
      start += tiles * hm_count;
      ++b;
      continue;
    }
    if (!a.partial) last = at + tiles;
    const int t1 = min(tiles, t0 + last - at);
    const int h = hm / a.blocks, row0 = (hm % a.blocks) * ROWS;
    const int rows = min(ROWS, a.tokens * a.group - row0);
    const int32_t* table = a.c.table + static_cast<int64_t>(b) * a.c.table_stride;
    int tile = t0 + wave;
    // nothing is loaded for tiles from t1 on: their units are empty
    const int stop = min(end, t1 * kTile);
    const int p0_first = page_of(a, table, tile * kTile, stop), p1_first = page_of(a, table, tile * kTile + 16, stop);
    int p0 = page_of(a, table, (tile + kWaves) * kTile, stop), p1 = page_of(a, table, (tile + kWaves) * kTile + 16, stop);

    // Q^T operands: 16-byte packets of this lane's query rows, elements as the keys'
    u32x4 q[MT][NQ];
    int token[MT];  // of the lane's query row; fresh or more: none
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = row0 + 16 * m + col;
      const int t = r / a.group, g = r - t * a.group;
      token[m] = t;
      const bool in = 16 * m + col < rows && t < fresh;
      const bits* qr = static_cast<const bits*>(a.q) + b * a.qb + t * a.qt + (static_cast<int64_t>(h) * a.group + g) * a.qh;
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const int e = FMT == KV_16BIT ? 32 * n + 8 * quad : 64 * (n / 2) + 16 * quad + 8 * (n & 1);
        q[m][n] = in && e < d ? *reinterpret_cast<const u32x4*>(qr + e) : u32x4{0, 0, 0, 0};
      }
    }

    f32x4 o[MT][NV];
    float top[MT], sum[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      top[m] = kLow;
      sum[m] = 0.f;
#pragma unroll
      for (int x = 0; x < NV; ++x) o[m][x] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    KvTile kv;
    bool left_out = false;
    bool whole;
    {
      const Unit<FMT> u0(a, h, tile * kTile, stop, p0_first), u1(a, h, tile * kTile + 16, stop, p1_first);
      whole = u0.whole && u1.whole;
      kv.load_keys(u0, u1, d);
      kv.load_values(u0, u1, d);
    }
    bool there0 = p0_first >= 0 && p0_first < a.c.pages, there1 = p1_first >= 0 && p1_first < a.c.pages;

    for (; tile < t1; tile += kWaves) {
      f32x4 sc[MT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m) sc[m][0] = sc[m][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const u32x4 k0 = kv.keys(0, n), k1 = kv.keys(1, n);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          sc[m][0] = mfma16<T>(k0, q[m][n], sc[m][0]);
          sc[m][1] = mfma16<T>(k1, q[m][n], sc[m][1]);
        }
      }
      float kscale[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) kscale[u][j] = FMT == KV_16BIT ? a.scale : a.scale * kv.ks[u][j];

      // the next tile's keys, while this one's weights are computed
      const Unit<FMT> n0(a, h, (tile + kWaves) * kTile, stop, p0), n1(a, h, (tile + kWaves) * kTile + 16, stop, p1);
      kv.load_keys(n0, n1, d);

      const bool masked = !whole || (tile + 1) * kTile > len;
      uint32_t seen[MT];  // bit 4 u + j
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        seen[m] = 0xff;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[m][u][j] *= kscale[u][j];
      }
      if (masked) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const int t = min(token[m], a.tokens - 1);
          uint32_t bits8 = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int i = tile * kTile + 16 * (e >> 2) + 4 * quad + (e & 3) - len;  // the new token in this slot
            const bool edge = a.mask ? a.mask[b * a.mask_b + t * a.mask_t + max(0, min(i, a.tokens - 1))] != 0 : i <= t;
            const bool see = (e < 4 ? there0 : there1) & ((i < 0) | ((i < fresh) & (token[m] < fresh) & edge));
            bits8 |= static_cast<uint32_t>(see) << e;
            sc[m][e >> 2][e & 3] = see ? sc[m][e >> 2][e & 3] : -INFINITY;
          }
          seen[m] = bits8;
        }
        left_out |= kv.take_out_non_finite();
      }

      u32x4 hi[MT], lo[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float most = fmaxf(fmaxf(fmaxf(sc[m][0][0], sc[m][0][1]), fmaxf(sc[m][0][2], sc[m][0][3])),
                           fmaxf(fmaxf(sc[m][1][0], sc[m][1][1]), fmaxf(sc[m][1][2], sc[m][1][3])));
        if (__builtin_amdgcn_ballot_w64(most > top[m] + kSlack)) {
          const float now = fmaxf(top[m], max_quads(most));
          const float f = __builtin_amdgcn_exp2f(top[m] - now);
          top[m] = now;
          sum[m] *= f;
#pragma unroll
          for (int x = 0; x < NV; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[m][x][i] *= f;
        }
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          w[e] = __builtin_amdgcn_exp2f(sc[m][e >> 2][e & 3] - top[m]);
          sum[m] += w[e];
          if constexpr (FMT != KV_16BIT) w[e] *= kv.vs[e >> 2][e & 3];
        }
        if (masked) {  // a scale that nobody sees may be anything
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = (seen[m] >> e) & 1 ? w[e] : 0.f;
        }
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          hi[m][p] = narrow2<VT>(f32x2{w[2 * p], w[2 * p + 1]});
          const f32x2 back = widen2<VT>(hi[m][p]);
          lo[m][p] = narrow2<VT>(f32x2{w[2 * p] - back.x, w[2 * p + 1] - back.y});
        }
      }

#pragma unroll
      for (int x = 0; x < NV; x += 2) {
        u32x4 even, odd;
        kv.values2(x, even, odd);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          o[m][x] = mfma16<VT>(even, hi[m], o[m][x]);
          o[m][x] = mfma16<VT>(even, lo[m], o[m][x]);
          o[m][x + 1] = mfma16<VT>(odd, hi[m], o[m][x + 1]);
          o[m][x + 1] = mfma16<VT>(odd, lo[m], o[m][x + 1]);
        }
      }
      kv.load_values(n0, n1, d);
      whole = n0.whole && n1.whole;
      there0 = p0 >= 0 && p0 < a.c.pages;
      there1 = p1 >= 0 && p1 < a.c.pages;
      p0 = page_of(a, table, (tile + 2 * kWaves) * kTile, stop);
      p1 = page_of(a, table, (tile + 2 * kWaves) * kTile + 16, stop);
    }

    // join the waves: common maximum, scaled sums
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      sum[m] = sum_quads(sum[m]);
      if (quad == 0) {
        wave_max[wave][16 * m + col] = top[m];
        wave_sum[wave][16 * m + col] = sum[m];
      }
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = 16 * m + col;
      float most = wave_max[0][r];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) most = fmaxf(most, wave_max[w][r]);
      const float f = __builtin_amdgcn_exp2f(top[m] - most);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x = 0; x < NV; x += 4)
          *reinterpret_cast<f32x4*>(&joined[wave][r][NV * (4 * quad + i) + x]) =
              f32x4{o[m][x][i] * f, o[m][x + 1][i] * f, o[m][x + 2][i] * f, o[m][x + 3][i] * f};
    }
    if (left_out) add_non_finite<T, FMT>(a, joined[wave], b, h, row0, rows, len, fresh, t0 + wave, t1);
    __syncthreads();
    const bool cut = t0 > 0 || t1 < tiles;
    const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (at == line_first ? 0 : 1);
    for (int e = threadIdx.x; e < rows * (d / 4); e += 64 * kWaves) {
      const int r = e / (d / 4), c = 4 * (e - r * (d / 4));
      float most = wave_max[0][r];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) most = fmaxf(most, wave_max[w][r]);
      float total = 0.f;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        total += wave_sum[w][r] * __builtin_amdgcn_exp2f(wave_max[w][r] - most);
        v += *reinterpret_cast<const f32x4*>(&joined[w][r][c]);
      }
      if (cut) {
        *reinterpret_cast<f32x4*>(a.partial + (slot * ROWS + r) * d + c) = v;
        if (c == 0) a.stats[slot * ROWS + r] = float2{most, total};
      } else {
        const int t = (row0 + r) / a.group, g = row0 + r - t * a.group;
        const float inv = 1.0f / total;
        const bool none = t >= fresh || total == 0.f;
        bits* out = static_cast<bits*>(a.out) +
                    ((static_cast<int64_t>(b) * a.tokens + t) * a.q_heads + h * a.group + g) * d + c;
        *reinterpret_cast<u32x2*>(out) = none ? u32x2{0, 0} : u32x2{narrow2<T>(f32x2{v[0] * inv, v[1] * inv}),
                                                                     narrow2<T>(f32x2{v[2] * inv, v[3] * inv})};
      }
    }
    __syncthreads();
    at += t1 - t0;
  }
}

// Adds the pieces of one query row that was cut, in order: lanes 0 - 31 and
// 32 - 63 of each of WAVES waves take every 2 WAVES-th piece with a running
// maximum, 4 (and, beyond 128, 4 more) elements per lane.  Latency is all there
// is to it: one wave per row, or eight where pieces per row are many, so that
// most pieces are in flight at once.
constexpr int kJoinWaves = 8;

template <typename T, int WAVES>
__global__ __launch_bounds__(64 * kJoinWaves) void tree_attention_join(TreeArgs a) {
  typedef typename T::bits bits;
  constexpr int PARTS = 2 * WAVES, PER = kJoinWaves / WAVES;  // rows of a workgroup
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int qrow = static_cast<int>(blockIdx.x) * PER + wave / WAVES;
  const int row_count = a.batch * a.tokens * a.q_heads;
  const int hq = qrow % a.q_heads, bt = qrow / a.q_heads;
  const int t = bt % a.tokens, b = min(bt / a.tokens, a.batch - 1);
  const int share = scalar_load(a.starts, 0), start = scalar_load(a.starts, 1 + b);
  const Seq s = Seq::of(a, b);
  const int block_rows = 16 * a.mt;
  const int h = hq / a.group, r = t * a.group + hq - h * a.group;
  const int block = r / block_rows, rr = r - block * block_rows;
  const int first = start + (h * a.blocks + block) * s.tiles;
  const int w0 = first / share, w1 = (first + s.tiles - 1) / share;
  const bool mine = qrow < row_count && w0 != w1;  // else written by the first kernel
  if (WAVES > 1 && !mine) return;

  const int part = 2 * (wave % WAVES) + lane / 32;
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
  const f32x4 o = lane < 32 ? v0 : v1;
  *reinterpret_cast<u32x2*>(static_cast<bits*>(a.out) + static_cast<int64_t>(qrow) * a.c.d + c) =
      none ? u32x2{0, 0} : u32x2{narrow2<T>(f32x2{o[0] * inv, o[1] * inv}), narrow2<T>(f32x2{o[2] * inv, o[3] * inv})};
}

// Row blocks and grid of a call.
struct Plan {
  int mt, blocks, grid;
  int64_t partial_bytes, stats_bytes, bytes;  // of the workspace; 0: no split
};

Plan plan(const mi355_kv_cache& c, int64_t batch, int64_t tokens, int64_t q_heads, int cus) {
  Plan p{};
  const int64_t rows = tokens * (q_heads / c.kv_heads);
  p.mt = rows <= 16 ? 1 : rows <= 32 || c.head_dim > 128 ? 2 : 4;
  p.blocks = static_cast<int>((rows + 16 * p.mt - 1) / (16 * p.mt));
  const int64_t pieces = batch * c.kv_heads * p.blocks;
  const int64_t tiles = (c.table_width * c.page_size + kTile - 1) / kTile;  // of the longest possible context
  p.grid = static_cast<int>(pieces);
  const int dp = c.head_dim <= 64 ? 64 : c.head_dim <= 128 ? 128 : 256;
  if (tiles <= 2 * kWaves || pieces * tiles > 0x7fffffff - 65536 * kWaves) return p;
  const int64_t wanted = (pieces * tiles + kWaves - 1) / kWaves;
  const int64_t most = static_cast<int64_t>(cus) * simd_waves(dp, p.mt);
  p.grid = static_cast<int>(wanted < most ? wanted : most);
  p.partial_bytes = 2 * int64_t{p.grid} * 16 * p.mt * c.head_dim * 4;
  p.stats_bytes = 2 * int64_t{p.grid} * 16 * p.mt * 8;
  p.bytes = p.partial_bytes + p.stats_bytes + 4 * (batch + 1);
  return p;
}

template <typename T, int FMT> int tree_typed(const TreeArgs& a, const Plan& p, hipStream_t s) {
  static const char* what = "tree_attention launch";
  const dim3 grid(static_cast<unsigned>(p.grid));
#define MI355_TREE(DP, MT) return launch(tree_attention_split<T, FMT, DP, MT>, grid, 64 * kWaves, 0, a, s, what)
  if (a.c.d <= 64) {
    if (p.mt == 1) MI355_TREE(64, 1);
    if (p.mt == 2) MI355_TREE(64, 2);
    MI355_TREE(64, 4);
  }
  if (a.c.d <= 128) {
    if (p.mt == 1) MI355_TREE(128, 1);
    if (p.mt == 2) MI355_TREE(128, 2);
    MI355_TREE(128, 4);
  }
  if (p.mt == 1) MI355_TREE(256, 1);
  MI355_TREE(256, 2);
#undef MI355_TREE
}

template <typename T> int tree_join(const TreeArgs& a, const Plan& p, hipStream_t s) {
  static const char* what = "tree_attention join launch";
  const int64_t rows = int64_t{a.batch} * a.tokens * a.q_heads;
  if (p.grid > 8 * int64_t{a.batch} * a.c.heads * a.blocks)  // most rows have more than 8 pieces
    return launch(tree_attention_join<T, kJoinWaves>, dim3(static_cast<unsigned>(rows)), 64 * kJoinWaves, 0, a, s, what);
  return launch(tree_attention_join<T, 1>, dim3(static_cast<unsigned>((rows + kJoinWaves - 1) / kJoinWaves)),
                64 * kJoinWaves, 0, a, s, what);
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
             q_heads / static_cast<int>(cache.kv_heads), p.mt, p.blocks, 0, 0, 0, scale * kLog2e};
  if (p.bytes > 0 && work != nullptr && work_bytes >= p.bytes) {
    a.partial = static_cast<float*>(work);
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
