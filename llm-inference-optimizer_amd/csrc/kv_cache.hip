// Writing a key/value cache (with the rotary of queries and keys fused in),
// reading it back, and moving the kept tokens of a draft together.
//
// All three are bound by HBM on long inputs and by launch and load latency on
// a decode step's few rows.  A row (one token and head, head_dim elements) is
// held by 4 to 32 lanes of one 8-element packet each; a wave of the append
// takes a token, or with few tokens a pass over some of its rows.
//
//   append  per row of new keys (rotated, in fp32) and values:
//             amax = max |x|,  scale = max(amax / top, 1e-8),  top = 127 | 448
//             code = round(x / scale)    (int8: ties to even; e4m3: its grid)
//           The rotated key is not rounded to 16 bits in between.  The row's
//           maximum is taken on the magnitudes' bit patterns, which order like
//           the values and put NaN on top: a row that holds an infinity or a
//           NaN gets that as its scale and codes of zero, so that all of it
//           reads back as NaN instead of as numbers.
//   read    code * scale, rounded once.
//   keep    slot len + i <- slot len + kept[i]: a workgroup takes one sequence,
//           head, pool and 128 bytes of the rows, loads those of every kept
//           row into LDS and then writes, so that any order and any overlap of
//           slots is right.
//
// Measured: append of 3001 tokens of 4 sequences, half of them padding (28 + 2 x
// 4 heads of 128, bf16 to e4m3, queries and keys rotated, 194 MB) 33.7 us, 5.8
// TB/s; of 16 single tokens 4.7 us: a launch, the position and slot, the page and
// the row's store are trips that wait for each other.  Read of the former (32 MB)
// 7.8 us, 4.1 TB/s: a lane's one packet waits for lengths, the page and the codes;
// of one token 2.4.  Keep of up to 9 of 64 tokens of 128 sequences (8 heads of
// 16-bit values, 5 MB) 6.9 us, of 4 sequences 3.6: five such trips, as it is
// written -- kept_lens bounds the loop that loads `kept`, and the destination's
// page is looked up behind the barrier.
#include "kv_cache.h"
#include "rotary.h"

namespace mi355 {
namespace {

// Largest v among the `lanes` (4 .. 32, a power of two) that share a row.
template <int CTRL> __device__ __forceinline__ uint32_t dpp_umax(uint32_t v) {
  return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, false)));
}
__device__ __forceinline__ uint32_t row_max(uint32_t v, int lanes) {
  v = dpp_umax<0xb1>(v);                     // quad_perm [1,0,3,2]
  v = dpp_umax<0x4e>(v);                     // quad_perm [2,3,0,1]
  if (lanes >= 8) v = dpp_umax<0x141>(v);    // row_half_mirror
  if (lanes >= 16) v = dpp_umax<0x140>(v);   // row_mirror
  if (lanes >= 32) {
    auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(static_cast<uint32_t>(r[0]), static_cast<uint32_t>(r[1]));
  }
  return v;
}

struct Strides {
  int64_t b, t, h;
};

struct AppendArgs {
  KvCache c;
  RotaryArgs rot;
  const void *k, *v, *q;
  void* q_out;
  const int32_t *lens, *new_lens;
  Strides ks, vs, qs;
  int rows, tokens, q_heads, lanes;  // rows = batch * tokens
  // heads per wave; from which blockIdx.y on it takes keys and values
  int q_per_wave, kv_per_wave, kv_from;
};

constexpr int kAhead = 2;  // query rows of a lane in flight
constexpr int kWaves = 4;  // of a workgroup, each for itself

template <typename T, int FMT, int MODE> __global__ __launch_bounds__(64 * kWaves) void append_rows(AppendArgs a) {
  typedef typename T::bits bits;
  __shared__ float angles[kWaves][2 * kMaxPairs];
  const int index = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int token = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(wave);
  if (token >= a.rows) return;
  float* cs = angles[wave];
  const int b = token / a.tokens, t = token - b * a.tokens;
  const int64_t position = MODE == ROTARY_NONE ? 0 : a.rot.positions[b * a.rot.pos_stride_b + t * a.rot.pos_stride_t];
  const int64_t slot = static_cast<int64_t>(a.lens[b]) + t;
  const bool stored = a.new_lens == nullptr || t < a.new_lens[b];
  RotaryLane<T, MODE> lane(a.rot, (index % a.lanes) * 8);
  const bool in = lane.d0 < a.c.d;
  const int step = 64 / a.lanes, mine = index / a.lanes;

  // Rows of a token: its query heads, then its keys' and values'.  The grid's
  // y takes passes of `step` rows: query passes first.
  const int q_last = in ? min(a.q_heads, (static_cast<int>(blockIdx.y) + 1) * a.q_per_wave) : 0;
  int h = blockIdx.y * a.q_per_wave + mine;
  const bits* q = static_cast<const bits*>(a.q) + b * a.qs.b + t * a.qs.t + h * a.qs.h;
  bits* q_out = static_cast<bits*>(a.q_out) + (static_cast<int64_t>(token) * a.q_heads + h) * a.c.d + lane.d0;
  RotaryPacket<T, MODE> p[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u)
    if (h + u * step < q_last) p[u].load(q + u * step * a.qs.h, lane, a.rot);

  const int kv_rows = 2 * a.c.heads;
  const int kv_first = (static_cast<int>(blockIdx.y) - a.kv_from) * a.kv_per_wave;
  // a wave of queries, and one of padding, has no rows of keys and values
  const int kv_last = kv_first < 0 || !stored ? 0 : min(kv_rows, kv_first + a.kv_per_wave);
  int r = max(kv_first, 0) + mine;
  const auto kv_row = [&](int i) {
    return i < a.c.heads ? static_cast<const bits*>(a.k) + b * a.ks.b + t * a.ks.t + i * a.ks.h
                         : static_cast<const bits*>(a.v) + b * a.vs.b + t * a.vs.t + (i - a.c.heads) * a.vs.h;
  };
  RotaryPacket<T, MODE> kv;
  if (in && r < kv_last) kv.load(kv_row(r), lane, a.rot);
  const int64_t first = kv_last > 0 ? a.c.row(b, slot, 0) : -1;  // of head 0

  if constexpr (MODE != ROTARY_NONE) {
    rotary_angles(cs, a.rot, position, index, 64);  // while the rows are on their way
    wave_sync();
    lane.angles(a.rot, cs);
  }

  while (h < q_last) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (h >= q_last) break;
      float y[8];
      p[u].turn(y, lane);
      Packet<T> o;
      o.pack(y);
      if (h + kAhead * step < q_last) p[u].load(q + kAhead * step * a.qs.h, lane, a.rot);
      *reinterpret_cast<u32x4*>(q_out) = o.raw;
      h += step;
      q += step * a.qs.h;
      q_out += step * a.c.d;
    }
  }

  if (first < 0) return;  // padding, or a slot without a place
  for (; r < kv_last; r += step) {
    const bool key = r < a.c.heads;
    const int64_t at = first + static_cast<int64_t>(key ? r : r - a.c.heads) * a.c.page_size;
    void* pool = key ? a.c.k : a.c.v;
    float y[8];
    if (in) {
      if (key) kv.turn(y, lane);
      else kv.own.unpack(y);
      if (r + step < kv_last) kv.load(kv_row(r + step), lane, a.rot);
    }
    if constexpr (FMT == KV_16BIT) {
      Packet<T> o;
      o.pack(y);
      if (in) *reinterpret_cast<u32x4*>(static_cast<bits*>(pool) + at * a.c.d + lane.d0) = o.raw;
    } else {
      uint32_t top = 0;
      if (in) {
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, as_u32(y[e]) & 0x7fffffffu);
      }
      top = row_max(top, a.lanes);
      const bool finite = top < 0x7f800000u;
      const float scale = finite ? fmaxf(as_f32(top) / kv_top<FMT>(), 1e-8f) : as_f32(top);
      if (in) {
        const float rc = 1.0f / scale;
        float lo[4], hi[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          lo[e] = quotient(y[e], scale, rc);
          hi[e] = quotient(y[4 + e], scale, rc);
        }
        const u32x2 code = {encode4<FMT>(lo), encode4<FMT>(hi)};
        *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(pool) + at * a.c.d + lane.d0) = finite ? code : u32x2{0, 0};
      }
      if (lane.d0 == 0) (key ? a.c.k_scale : a.c.v_scale)[at] = scale;
    }
  }
}

struct ReadArgs {
  KvCache c;
  void *k_out, *v_out;  // [batch, heads, tokens, d]
  const int32_t *start, *end;
  int64_t rows;  // batch * heads * tokens
  uint32_t tokens;
  int lanes;
};

// A lane's packet of a row's keys and values; every load of a row is issued
// before any of its stores.
template <typename T, int FMT> __global__ __launch_bounds__(256) void read_rows(ReadArgs a) {
  typedef typename T::bits bits;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * (256 / a.lanes) + threadIdx.x / a.lanes;
  const int d0 = (threadIdx.x % a.lanes) * 8;
  if (r >= a.rows || d0 >= a.c.d) return;
  // 32 bits hold a row: fewer than 2^26 of them
  const uint32_t bh = static_cast<uint32_t>(r) / a.tokens, i = static_cast<uint32_t>(r) - bh * a.tokens;
  const uint32_t b = bh / a.c.heads, h = bh - b * a.c.heads;
  const int64_t slot = static_cast<int64_t>(a.start ? a.start[b] : 0) + i;
  const int64_t at = slot < a.end[b] ? a.c.row(b, slot, static_cast<int>(h)) : -1;
  Packet<T> o[2];
  o[0].raw = o[1].raw = u32x4{0, 0, 0, 0};
  if (at >= 0) {
    if constexpr (FMT == KV_16BIT) {
      o[0].raw = *reinterpret_cast<const u32x4*>(static_cast<const bits*>(a.c.k) + at * a.c.d + d0);
      o[1].raw = *reinterpret_cast<const u32x4*>(static_cast<const bits*>(a.c.v) + at * a.c.d + d0);
    } else {
      u32x2 code[2];
      code[0] = *reinterpret_cast<const u32x2*>(static_cast<const uint8_t*>(a.c.k) + at * a.c.d + d0);
      code[1] = *reinterpret_cast<const u32x2*>(static_cast<const uint8_t*>(a.c.v) + at * a.c.d + d0);
      const float scale[2] = {a.c.k_scale[at], a.c.v_scale[at]};
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        float lo[4], hi[4], f[8];
        decode4<FMT>(code[side][0], lo);
        decode4<FMT>(code[side][1], hi);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[j] = lo[j] * scale[side];
          f[4 + j] = hi[j] * scale[side];
        }
        o[side].pack(f);
      }
    }
  }
  *reinterpret_cast<u32x4*>(static_cast<bits*>(a.k_out) + r * a.c.d + d0) = o[0].raw;
  *reinterpret_cast<u32x4*>(static_cast<bits*>(a.v_out) + r * a.c.d + d0) = o[1].raw;
}

struct KeepArgs {
  KvCache c;
  const int32_t *lens, *kept, *kept_lens;
  int64_t kept_stride;
  int most, row_bytes;
};

constexpr int kSlice = 128;    // bytes of a row per workgroup
constexpr int kMostKept = 128;

// Grid: (sequence, head, 2 slice + keys | values).
__global__ __launch_bounds__(256) void keep_rows(KeepArgs a) {
  __shared__ u32x4 held[kMostKept * (kSlice / 16)];
  __shared__ float held_scale[kMostKept];
  const int64_t b = blockIdx.x;
  const int h = blockIdx.y, first = (blockIdx.z >> 1) * kSlice;
  const bool values = (blockIdx.z & 1) != 0;
  uint8_t* pool = static_cast<uint8_t*>(values ? a.c.v : a.c.k) + first;
  float* scales = first != 0 ? nullptr : values ? a.c.v_scale : a.c.k_scale;
  const int packets = min(kSlice, a.row_bytes - first) / 16;
  const int n = min(a.kept_lens ? a.kept_lens[b] : a.most, a.most);
  const int64_t len = a.lens[b];
  const int32_t* kept = a.kept + b * a.kept_stride;
  for (int e = threadIdx.x; e < n * packets; e += 256) {
    const int i = e / packets, p = e % packets;
    const int64_t from = kept[i] < 0 ? -1 : a.c.row(b, len + kept[i], h);
    if (from < 0) continue;
    held[e] = *reinterpret_cast<const u32x4*>(pool + from * a.row_bytes + 16 * p);
    if (p == 0 && scales) held_scale[i] = scales[from];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < n * packets; e += 256) {
    const int i = e / packets, p = e % packets;
    const int64_t from = kept[i] < 0 ? -1 : a.c.row(b, len + kept[i], h), to = a.c.row(b, len + i, h);
    if (from < 0 || to < 0) continue;
    *reinterpret_cast<u32x4*>(pool + to * a.row_bytes + 16 * p) = held[e];
    if (p == 0 && scales) scales[to] = held_scale[i];
  }
}

template <typename T, int FMT> int append_format(const AppendArgs& a, dim3 grid, hipStream_t s) {
  static const char* what = "kv_cache_append launch";
  switch (rotary_mode(a.rot, 8)) {
    case ROTARY_NONE: return launch(append_rows<T, FMT, ROTARY_NONE>, grid, 256, 0, a, s, what);
    case ROTARY_HALF: return launch(append_rows<T, FMT, ROTARY_HALF>, grid, 256, 0, a, s, what);
    case ROTARY_PAIRS: return launch(append_rows<T, FMT, ROTARY_PAIRS>, grid, 256, 0, a, s, what);
    default: return launch(append_rows<T, FMT, ROTARY_ODD>, grid, 256, 0, a, s, what);
  }
}

template <typename T> int append_typed(const AppendArgs& a, int fmt, dim3 grid, hipStream_t s) {
  if (fmt == KV_INT8) return append_format<T, KV_INT8>(a, grid, s);
  if (fmt == KV_E4M3) return append_format<T, KV_E4M3>(a, grid, s);
  return append_format<T, KV_16BIT>(a, grid, s);
}

template <typename T> int read_typed(const ReadArgs& a, int fmt, dim3 grid, hipStream_t s) {
  static const char* what = "kv_cache_read launch";
  if (fmt == KV_INT8) return launch(read_rows<T, KV_INT8>, grid, 256, 0, a, s, what);
  if (fmt == KV_E4M3) return launch(read_rows<T, KV_E4M3>, grid, 256, 0, a, s, what);
  return launch(read_rows<T, KV_16BIT>, grid, 256, 0, a, s, what);
}

}  // namespace

int kv_append_launch(const mi355_kv_cache& cache, const RotaryArgs& rot, const void* k, const void* v, const void* q,
                     void* q_out, const int32_t* lens, const int32_t* new_lens, const int64_t* strides, int64_t batch,
                     int64_t tokens, int q_heads, int dtype, hipStream_t stream) {
  AppendArgs a{kv_cache_args(cache), rot, k, v, q, q_out, lens, new_lens,
               {strides[0], strides[1], strides[2]}, {strides[3], strides[4], strides[5]},
               {strides[6], strides[7], strides[8]}, static_cast<int>(batch * tokens),
               static_cast<int>(tokens), q_heads, row_lanes(cache.head_dim / 8),
               0, 0, 0};
  const int step = 64 / a.lanes, kv_rows = 2 * a.c.heads;
  const int q_passes = (q_heads + step - 1) / step, kv_passes = (kv_rows + step - 1) / step;
  dim3 grid(static_cast<unsigned>((batch * tokens + kWaves - 1) / kWaves));
  // a pass per wave until the tokens alone fill the chip (a pass against a token
  // per wave: 8.7 / 9.55 us for 512 tokens of 28 + 2 x 4 heads, 18.0 / 14.2 us
  // for 2048)
  if (batch * tokens < 1024) {
    a.q_per_wave = a.kv_per_wave = step;
    a.kv_from = q_passes;
    grid.y = static_cast<unsigned>(q_passes + kv_passes);
  } else {
    a.q_per_wave = q_heads;
    a.kv_per_wave = kv_rows;
  }
  return dtype == MI355_F16 ? append_typed<F16>(a, cache.format, grid, stream)
                            : append_typed<BF16>(a, cache.format, grid, stream);
}

int kv_read_launch(const mi355_kv_cache& cache, void* k_out, void* v_out, const int32_t* start, const int32_t* end,
                   int64_t batch, int64_t tokens, int dtype, hipStream_t stream) {
  ReadArgs a{kv_cache_args(cache), k_out, v_out, start, end, batch * cache.kv_heads * tokens,
             static_cast<uint32_t>(tokens), 0};
  a.lanes = row_lanes(a.c.d / 8);
  const int per = 256 / a.lanes;
  const dim3 grid(static_cast<unsigned>((a.rows + per - 1) / per));
  return dtype == MI355_F16 ? read_typed<F16>(a, cache.format, grid, stream)
                            : read_typed<BF16>(a, cache.format, grid, stream);
}

int kv_keep_launch(const mi355_kv_cache& cache, const int32_t* lens, const int32_t* kept, const int32_t* kept_lens,
                   int64_t kept_stride, int64_t batch, int most, hipStream_t stream) {
  KeepArgs a{kv_cache_args(cache), lens, kept, kept_lens, kept_stride, most, 0};
  a.row_bytes = a.c.d * (cache.format == KV_16BIT ? 2 : 1);
  const dim3 grid(static_cast<unsigned>(batch), static_cast<unsigned>(a.c.heads),
                  static_cast<unsigned>(2 * ((a.row_bytes + kSlice - 1) / kSlice)));
  return launch(keep_rows, grid, 256, 0, a, stream, "kv_cache_keep launch");
}

}  // namespace mi355
