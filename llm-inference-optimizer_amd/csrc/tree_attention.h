// What the kernels of tree_attention.hip share: the line of tiles that
// workgroups divide, the loads of a 16-slot unit of the cache and its MFMA
// operands, who sees what, and the running softmax of 16 query rows.
#pragma once

#include "kv_cache.h"

namespace mi355 {

constexpr int kWaves = 4;            // of a workgroup
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLow = -3.4028235e38f;  // the running maximum before any score: the lowest number

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
  int block_rows, blocks;             // row blocks
  int tile, pad;                      // slots of a tile on the line, tiles that a piece costs beside its own
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
// row block.  `pad` of those, the first, stand for what a piece costs besides
// its tiles (queries to load, sums to join and write): a share that holds the
// beginning of more pieces holds fewer tiles.
struct Seq {
  int len, fresh, end, tiles;
  __device__ __forceinline__ Seq(const TreeArgs& a, int len_, int fresh_) {
    const int cap = a.c.capacity();
    len = max(0, min(len_, cap));
    fresh = max(0, min(fresh_, a.tokens));
    end = min(len + fresh, cap);
    tiles = a.pad + max(1, (end + a.tile - 1) / a.tile);
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

// Tiles per workgroup: equal shares of whole `step`s.
__device__ __forceinline__ int line_share(int total, int grid, int step) {
  return ((total + grid - 1) / grid + step - 1) / step * step;
}

// The share that workgroup i takes.  Workgroups go around the chip's 8 dies;
// with more than one row block, neighbours on the line read the same part of the
// cache and belong on one die, behind one L2 (8 trees of 48 tokens, 3 blocks:
// 50.5 -> 46.6 us; with one block 17.2 against 16.7 us for 24 trees of 9).
__device__ __forceinline__ int line_place(const TreeArgs& a, int i) {
  constexpr int kDies = 8;
  const int die = i % kDies;
  return a.blocks == 1 ? i : die * (a.grid / kDies) + min(die, a.grid % kDies) + i / kDies;
}

template <int FMT> __device__ __forceinline__ constexpr int elem_bytes() { return FMT == KV_16BIT ? 2 : 1; }

// The 16 slots of a unit: descriptors that end with its last slot in use.
template <int FMT> struct Unit {
  rsrc_t k, v, ks, vs;
  bool whole;  // 16 slots, all there
  __device__ __forceinline__ Unit(const TreeArgs& a, int h_, int slot_, int end_, int page_) {
    // uniform all, which the compiler does not always see
    const int h = uniform(h_), slot = uniform(slot_), end = uniform(end_), page = uniform(page_);
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

// The 16 slots of a unit in a lane's registers (r = l % 16, quad = l / 16):
//   keys    slot r, elements (8-bit) 64 i + 16 quad .. + 15 or (16-bit)
//           32 i + 8 quad .. + 7 in load i
//   values  slot 4 quad + j, elements NV r .. + NV - 1
//   scales  slots 4 quad .. 4 quad + 3
// Elements from d on are zero.  AUX: cache policy of the loads.
template <typename T, int FMT, int DP, int AUX> struct UnitRegs {
  static constexpr int ES = FMT == KV_16BIT ? 2 : 1;
  static constexpr int NV = DP / 16;
  static constexpr int KL = DP * ES / 64;     // 16-byte key loads
  static constexpr int VD = NV * ES / 4;      // dwords of a value per lane
  u32x4 k[KL];
  uint32_t v[4][VD];
  f32x4 ks, vs;

  __device__ __forceinline__ void load_keys(const Unit<FMT>& u, int d) {
    const int lane = threadIdx.x & 63, r = lane & 15, quad = lane >> 4;
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      const int byte = 64 * i + 16 * quad;
      k[i] = __builtin_amdgcn_raw_buffer_load_b128(
          u.k, byte < d * ES ? static_cast<uint32_t>(r * d * ES + byte) : kOob, 0, AUX);
    }
    if constexpr (FMT != KV_16BIT)
      ks = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(u.ks, 16u * quad, 0, AUX));
  }

  __device__ __forceinline__ void load_values(const Unit<FMT>& u, int d) {
    const int lane = threadIdx.x & 63, r = lane & 15, quad = lane >> 4;
    if constexpr (FMT != KV_16BIT)
      vs = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(u.vs, 16u * quad, 0, AUX));
    // beyond the unit in the last packet too: kOob and a packet would be 0
    constexpr uint32_t kBeyond = VD > 4 ? kOob - 16 * (VD / 4 - 1) : kOob;
    const uint32_t first = NV * r < d ? static_cast<uint32_t>((4 * quad * d + NV * r) * ES) : kBeyond;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = j * d * ES;  // uniform: the scalar offset of the load
      if constexpr (VD == 1) {
        v[j][0] = __builtin_amdgcn_raw_buffer_load_b32(u.v, first, at, AUX);
      } else if constexpr (VD == 2) {
        const u32x2 t = __builtin_amdgcn_raw_buffer_load_b64(u.v, first, at, AUX);
        v[j][0] = t[0];
        v[j][1] = t[1];
      } else {
#pragma unroll
        for (int w = 0; w < VD / 4; ++w) {
          const u32x4 t = __builtin_amdgcn_raw_buffer_load_b128(u.v, first + 16 * w, at, AUX);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j][4 * w + e] = t[e];
        }
      }
    }
  }

  // The K operand of MFMA k-step n (32 of the DP elements).
  __device__ __forceinline__ u32x4 keys(int n) const {
    if constexpr (FMT == KV_16BIT) {
      return k[n];
    } else {
      const u32x2 lo = widen_codes<T, FMT>(k[n / 2][2 * (n & 1)]), hi = widen_codes<T, FMT>(k[n / 2][2 * (n & 1) + 1]);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
  }

  // Elements x (even) and x + 1 of the 4 values: halves of two V^T operands,
  // which two units make up.
  __device__ __forceinline__ void values2(int x, u32x2& even, u32x2& odd) const {
#pragma unroll
    for (int p = 0; p < 2; ++p) {  // slots 2 p and 2 p + 1
      const uint32_t a = v[2 * p][x * ES / 4], b = v[2 * p + 1][x * ES / 4];
      if constexpr (FMT == KV_INT8) {
        // the upper half of an fp32 integer below 2^8 is its bf16 pattern
        const int sh = 8 * (x & 3);
        even[p] = __builtin_amdgcn_perm(as_u32(static_cast<float>(static_cast<int8_t>(b >> sh & 0xff))),
                                        as_u32(static_cast<float>(static_cast<int8_t>(a >> sh & 0xff))), 0x07060302u);
        odd[p] = __builtin_amdgcn_perm(as_u32(static_cast<float>(static_cast<int8_t>(b >> (sh + 8) & 0xff))),
                                       as_u32(static_cast<float>(static_cast<int8_t>(a >> (sh + 8) & 0xff))),
                                       0x07060302u);
      } else {
        uint32_t a2 = a, b2 = b;  // elements x and x + 1
        if constexpr (FMT == KV_E4M3) {
          const u32x2 a4 = widen_codes<BF16, FMT>(a), b4 = widen_codes<BF16, FMT>(b);
          a2 = x & 2 ? a4[1] : a4[0];
          b2 = x & 2 ? b4[1] : b4[0];
        }
        even[p] = __builtin_amdgcn_perm(b2, a2, 0x05040100u);
        odd[p] = __builtin_amdgcn_perm(b2, a2, 0x07060302u);
      }
    }
  }

  // Zeroes the elements of the values that are NaN or infinite; whether any
  // lane had one.
  __device__ __forceinline__ bool take_out_non_finite() {
    if constexpr (FMT == KV_INT8) return false;
    bool hit = false;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int w = 0; w < VD; ++w) {
        const uint32_t e = v[j][w];
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
        v[j][w] = e & ~drop;
      }
    return __builtin_amdgcn_ballot_w64(hit) != 0;
  }
};

// Element e of the B operand's k-step n, quad `quad`: the order of d in keys().
template <int FMT> __device__ __forceinline__ int key_element(int n, int quad) {
  return FMT == KV_16BIT ? 32 * n + 8 * quad : 64 * (n / 2) + 16 * quad + 8 * (n & 1);
}

// One workgroup's piece: tiles of one sequence, head and row block.
struct Piece {
  int b, h, row0, rows, len, fresh, stop;  // stop: the slots that it may load end there
};

// Which of the 8 slots (bit 4 u + j: slot first + 16 u + 4 quad + j) token t of
// the piece sees; there[u]: the unit's page is.
__device__ __forceinline__ uint32_t seen_slots(const TreeArgs& a, const Piece& p, int first, int t, bool there0,
                                               bool there1) {
  const int quad = (threadIdx.x & 63) >> 4;
  const int row = min(t, a.tokens - 1);
  const int i0 = first + 4 * quad - p.len;  // the new token in slot 0; 16 + j, j: + 16 u + j
  uint32_t edge = 0;                        // of the tree, to tokens 0 .. tokens - 1
  if (a.mask) {
    const uint8_t* m = a.mask + p.b * a.mask_b + row * a.mask_t;
    uint8_t byte[8];  // all on their way at once
#pragma unroll
    for (int e = 0; e < 8; ++e) byte[e] = m[max(0, min(i0 + 16 * (e >> 2) + (e & 3), a.tokens - 1))];
#pragma unroll
    for (int e = 0; e < 8; ++e) edge |= byte[e] ? 1u << e : 0u;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) edge |= i0 + 16 * (e >> 2) + (e & 3) <= row ? 1u << e : 0u;
  }
  uint32_t before = 0, fresh = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int i = i0 + 16 * (e >> 2) + (e & 3);
    before |= i < 0 ? 1u << e : 0u;
    fresh |= i >= 0 && i < p.fresh ? 1u << e : 0u;
  }
  return (before | (t < p.fresh ? fresh & edge : 0u)) & ((there0 ? 0xfu : 0u) | (there1 ? 0xf0u : 0u));
}

// 16 query rows, one per column of the MFMA tiles: O^T in NV tiles, what the
// exponents are relative to (log2; the same in a column's four lanes) and this
// lane's part of the sum.  VT: the type of the weights' two parts.
//
// bf16 parts have fp32's exponents: `top` is the running maximum, which moves
// only when a score passes it by 2^8.  fp16 parts end at 2^-24: relative to the
// maximum, 17 nats down nothing would be left of a weight that the sum still
// counts, and a slot that outweighs all others but has a small value (often the
// first) makes such weights the result.  So there `top` follows the tiles, up
// and down: it moves where a tile's largest weight would lie outside 2^7 ..
// 2^15 (half the type's largest), to a whole number that puts it between 2^11
// and 2^12.  Weights from 2^-8 on keep 16 bits, those below are off by 2^-25 at
// most, that is 2^-32 of the tile's largest; o and sum are multiplied by powers
// of 2, exactly.  The way down ends where the sum is 2^64 of a weight: o, of
// values below 2^16, stays in range, and what is 2^-64 of the result is nothing
// to 16-bit outputs.
template <int NV, typename VT> struct Rows {
  static constexpr bool FOLLOW = VT::code == MI355_F16;
  static constexpr float kMost = FOLLOW ? 15.0f : 8.0f;  // log2 of the largest weight
  static constexpr float kLeast = 7.0f, kRest = 12.0f, kMostSum = 64.0f;
  f32x4 o[NV];
  float top, sum;

  __device__ __forceinline__ void clear() {
    top = kLow;
    sum = 0.f;
#pragma unroll
    for (int x = 0; x < NV; ++x) o[x] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // The largest of 8 scores.
  static __device__ __forceinline__ float largest(const f32x4 (&sc)[2]) {
    return fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                 fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
  }
  // Whether a column's largest score, the largest of its lanes', asks for
  // another `top`.  (A column that sees nothing of a tile asks, and keeps its own.)
  __device__ __forceinline__ bool moves(float most) const {
    const bool above = __builtin_amdgcn_ballot_w64(most > top + kMost) != 0;
    if constexpr (!FOLLOW) return above;
    uint64_t near = __builtin_amdgcn_ballot_w64(most >= top + kLeast);
    near |= near >> 32;
    near |= near >> 16;
    return above || (near & 0xffff) != 0xffff;
  }
  // Moves `top` by the column's largest score.
  __device__ __forceinline__ void move(float most) {
    const float column = max_quads(most);
    float now = fmaxf(top, column);
    if constexpr (FOLLOW) {
      const float least = top + __builtin_amdgcn_logf(sum_quads(sum)) - kMostSum;  // log2; -infinity without a sum
      now = column >= kLow ? ceilf(fmaxf(column - kRest, least)) : top;
    }
    const float f = __builtin_amdgcn_exp2f(top - now);
    top = now;
    sum *= f;
#pragma unroll
    for (int x = 0; x < NV; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[x][i] *= f;
  }

  // Scores of 8 slots (log2; -infinity where not seen) -> weights times the
  // values' scales, as the two parts of a P^T operand.
  template <bool SCALED>
  __device__ __forceinline__ void weights(const f32x4 (&sc)[2], const f32x4& vs0, const f32x4& vs1, bool masked,
                                          uint32_t seen, u32x4& hi, u32x4& lo) {
    // The score has been multiplied by the scale and rounded, as the maximum has:
    // fused into the subtraction, the unrounded product of a large score would
    // differ from the maximum made of it by more than the exponential holds.
#pragma clang fp contract(off)
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[e] = __builtin_amdgcn_exp2f(sc[e >> 2][e & 3] - top);
      sum += w[e];
      if constexpr (SCALED) w[e] *= e < 4 ? vs0[e & 3] : vs1[e & 3];
    }
    if (SCALED && masked) {  // a scale that nobody sees may be anything
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = (seen >> e) & 1 ? w[e] : 0.f;
    }
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      hi[p] = narrow2<VT>(f32x2{w[2 * p], w[2 * p + 1]});
      const f32x2 back = widen2<VT>(hi[p]);
      lo[p] = narrow2<VT>(f32x2{w[2 * p] - back.x, w[2 * p + 1] - back.y});
    }
  }

  // Whether a lane holds a NaN or an infinity of O.
  __device__ __forceinline__ bool non_finite() const {
    float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < NV; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) zero[i] = __builtin_fmaf(o[x][i], 0.f, zero[i]);
    return __builtin_amdgcn_ballot_w64(zero[0] + zero[1] + zero[2] + zero[3] != 0.f) != 0;
  }

  // O of this lane's row to LDS or from it: row[NV (4 quad + i) + x].
  __device__ __forceinline__ void put(float* row, float f) const {
    const int quad = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int x = 0; x < NV; x += 4)
        *reinterpret_cast<f32x4*>(row + NV * (4 * quad + i) + x) =
            f32x4{o[x][i] * f, o[x + 1][i] * f, o[x + 2][i] * f, o[x + 3][i] * f};
  }
};

// Q^T operands of 16 rows from row0 + 16 m on; token: of this lane's row.
template <typename T, int FMT, int NQ>
__device__ __forceinline__ void load_queries(const TreeArgs& a, const Piece& p, int m, u32x4 (&q)[NQ], int& token) {
  typedef typename T::bits bits;
  const int col = threadIdx.x & 15, quad = (threadIdx.x & 63) >> 4;
  const int r = p.row0 + 16 * m + col;
  const int t = r / a.group, g = r - t * a.group;
  token = t;
  const bool in = 16 * m + col < p.rows && t < p.fresh;
  const bits* row =
      static_cast<const bits*>(a.q) + p.b * a.qb + t * a.qt + (static_cast<int64_t>(p.h) * a.group + g) * a.qh;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int e = key_element<FMT>(n, quad);
    q[n] = in && e < a.c.d ? *reinterpret_cast<const u32x4*>(row + e) : u32x4{0, 0, 0, 0};
  }
}

// Sets the elements of the output rows [r0, r1) that see a NaN or an infinity
// among the values of the tiles (of `slots` slots) first, first + step, .. to
// the sum of those.  The second product cannot do it: it spreads a value to rows
// that do not see it (take_out_non_finite), and an infinity times a weight's low
// part, or a weight that is 0 in 32 bits, is NaN.  Weights do not matter to
// them.  Rare; a lane for two elements, one look at the page per 16 slots, whose
// loads go out together.  In LDS, where rows and elements can be indexed; acc
// row 0 is row r0.
template <typename T, int FMT, int PITCH>
__device__ __forceinline__ void set_non_finite(const TreeArgs& a, const Piece& p, float (*acc)[PITCH], int r0, int r1,
                                               int first, int step, int slots) {
  // f(slot, which, value) of every NaN and infinity of elements e and e + 1 in
  // slots [from, to)
  const auto each = [&](int e, int from, int to, const auto& f) {
#pragma unroll 1
    for (int tile = first; tile < to; tile += step) {
#pragma unroll 1
      for (int unit = max(tile, from & ~15); unit < min(tile + slots, to); unit += 16) {
        const int64_t at = a.c.row(p.b, unit, p.h);
        if (at < 0) continue;
        uint32_t two[16];  // a page has whole units
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int64_t i = (at + j) * a.c.d + e;
          if constexpr (FMT == KV_16BIT) two[j] = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(a.c.v) + i);
          else two[j] = *reinterpret_cast<const uint16_t*>(static_cast<const uint8_t*>(a.c.v) + i);
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          float v[4];
          if constexpr (FMT == KV_16BIT) {
            const f32x2 w = widen2<T>(two[j]);
            v[0] = w.x;
            v[1] = w.y;
          } else {
            decode4<FMT>(two[j], v);
          }
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if (v[k] - v[k] != 0.f && unit + j >= from && unit + j < to) f(unit + j, k, v[k]);
        }
      }
    }
  };
#pragma unroll 1
  for (int e = 2 * (threadIdx.x & 63); e < a.c.d; e += 128) {
    float context[2] = {0.f, 0.f};  // which every row sees
    each(e, 0, min(p.len, p.stop), [&](int, int k, float v) { context[k] += v; });
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (context[k] != 0.f)
        for (int r = r0; r < r1; ++r) acc[r - r0][e + k] = context[k];
    if (p.stop <= p.len) continue;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {  // what the product left goes first
      each(e, p.len, p.stop, [&](int slot, int k, float v) {
#pragma unroll 1
        for (int r = r0; r < r1; ++r) {
          const int t = (p.row0 + r) / a.group, i = slot - p.len;
          float* sum = &acc[r - r0][e + k];
          if (t < p.fresh && (a.mask ? a.mask[p.b * a.mask_b + t * a.mask_t + i] != 0 : i <= t))
            *sum = pass ? *sum + v : context[k] != 0.f ? *sum : 0.f;
        }
      });
    }
  }
}

// Four elements (from c on) of one row's result: its sums divided, or, of a
// row that other workgroups hold parts of, as they are.
template <typename T>
__device__ __forceinline__ void store_result(const TreeArgs& a, const Piece& p, bool cut, int64_t slot, int r, int c,
                                             f32x4 v, float most, float total) {
  typedef typename T::bits bits;
  if (cut) {
    *reinterpret_cast<f32x4*>(a.partial + (slot * a.block_rows + r) * a.c.d + c) = v;
    if (c == 0) a.stats[slot * a.block_rows + r] = float2{most, total};
    return;
  }
  const int t = (p.row0 + r) / a.group, g = p.row0 + r - t * a.group;
  const float inv = 1.0f / total;
  const bool none = t >= p.fresh || total == 0.f;
  bits* out = static_cast<bits*>(a.out) +
              ((static_cast<int64_t>(p.b) * a.tokens + t) * a.q_heads + p.h * a.group + g) * a.c.d + c;
  *reinterpret_cast<u32x2*>(out) =
      none ? u32x2{0, 0} : u32x2{narrow2<T>(f32x2{v[0] * inv, v[1] * inv}), narrow2<T>(f32x2{v[2] * inv, v[3] * inv})};
}

// This workgroup's tiles [at, last) of the line, piece by piece.  All of it is
// the same in every lane, and kept in scalar registers: descriptors made from
// vector registers would make each load a loop over the lanes.
struct Share {
  Line line;
  int at, last, b, start, first, size;
  int alone;  // without a split: head and block
  int place;  // with one: which share of the line
  // one piece
  Piece p;
  int t0, t1, tiles;  // tiles [t0, t1) of `tiles`
  int width;          // on the line
  const int32_t* table;

  __device__ __forceinline__ Share(const TreeArgs& a, int step) {
    if (a.partial) {
      line = Line(a);
      size = line_share(line.total, a.grid, step);
      place = line_place(a, blockIdx.x);
      at = place * size;
      last = at + size;
      b = line.find(a, at, &start);
    } else {  // one (head, block) of one sequence
      const int hm_count = a.c.heads * a.blocks;
      b = blockIdx.x / hm_count;
      alone = blockIdx.x - b * hm_count;
      start = at = 0;
      last = Seq::of(a, b).tiles;
    }
    first = at;
  }
  __device__ __forceinline__ bool next(const TreeArgs& a) {
    const int hm_count = a.c.heads * a.blocks;
    while (b < a.batch && at < last) {
      const Seq s = a.partial && b < 64 ? line.seq(a, b) : Seq::of(a, b);
      const int hm = a.partial ? uniform((at - start) / s.tiles) : alone;
      if (hm >= hm_count) {
        start = uniform(start + s.tiles * hm_count);
        b = uniform(b + 1);
        continue;
      }
      const int v0 = a.partial ? uniform(at - start - hm * s.tiles) : 0;
      const int v1 = uniform(min(s.tiles, v0 + last - at));
      tiles = uniform(s.tiles - a.pad);
      t0 = max(0, v0 - a.pad);
      t1 = v1 - a.pad;
      width = v1 - v0;
      if (t1 <= t0) {  // the share ends before the piece's first tile
        done();
        continue;
      }
      const int h = uniform(hm / a.blocks), row0 = uniform((hm - h * a.blocks) * a.block_rows);
      p = Piece{b, h, row0, uniform(min(a.block_rows, a.tokens * a.group - row0)), uniform(s.len), uniform(s.fresh),
                uniform(min(s.end, t1 * a.tile))};
      table = a.c.table + static_cast<int64_t>(b) * a.c.table_stride;
      return true;
    }
    return false;
  }
  // For the join; last, since loads wait for the stores before them.
  __device__ __forceinline__ void finish(const TreeArgs& a) const {
    if (a.partial && blockIdx.x == 0 && uniform(threadIdx.x >> 6) == 0) line.write(a, size, a.starts);
  }
  __device__ __forceinline__ bool cut() const { return t0 > 0 || t1 < tiles; }
  // where the piece goes in the workspace: the first of the share, or the last
  __device__ __forceinline__ int64_t slot() const { return 2 * static_cast<int64_t>(place) + (at == first ? 0 : 1); }
  __device__ __forceinline__ void done() { at = uniform(at + width); }
};

}  // namespace mi355
