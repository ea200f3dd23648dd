// Writing a key/value cache (with the rotary of queries and keys fused in),
// reading it back, and moving the kept tokens of a draft together.
//
// All three are bound by HBM on long inputs and by launch and load latency on
// a decode step's few rows.  A row (one token and head, head_dim elements) is
// held by 4 to 32 lanes of one 8-element packet each.
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
  int64_t tokens;
  int q_heads, lanes, rows_per_wg;
};

template <typename T, int FMT> __global__ __launch_bounds__(256) void append_rows(AppendArgs a) {
  typedef typename T::bits bits;
  __shared__ float cs[2 * kMaxPairs];
  const int64_t b = blockIdx.x / a.tokens, t = blockIdx.x % a.tokens;
  if (a.rot.rotary) {
    rotary_angles(cs, a.rot, a.rot.positions[b * a.rot.pos_stride_b + t * a.rot.pos_stride_t]);
    __syncthreads();
  }
  const int64_t slot = a.lens[b] + t;
  const bool stored = a.new_lens == nullptr || t < a.new_lens[b];
  const int d0 = (threadIdx.x % a.lanes) * 8;
  const bool in = d0 < a.c.d;
  // rows of a token: its query heads, then its keys', then its values'
  const int rows = a.q_heads + 2 * a.c.heads;
  const int first = blockIdx.y * a.rows_per_wg;
  for (int r = first + threadIdx.x / a.lanes; r < min(rows, first + a.rows_per_wg); r += 256 / a.lanes) {
    RotaryPacket<T> p;
    float y[8];
    if (r < a.q_heads) {
      if (in) {
        const bits* row = static_cast<const bits*>(a.q) + b * a.qs.b + t * a.qs.t + r * a.qs.h;
        p.load(row, d0, a.rot);
        p.rotate(y, row, d0, a.rot, cs);
        Packet<T> o;
        o.pack(y);
        bits* out = static_cast<bits*>(a.q_out) + (static_cast<int64_t>(blockIdx.x) * a.q_heads + r) * a.c.d;
        *reinterpret_cast<u32x4*>(out + d0) = o.raw;
      }
      continue;
    }
    const bool key = r < a.q_heads + a.c.heads;
    const int h = r - a.q_heads - (key ? 0 : a.c.heads);
    const int64_t at = stored ? a.c.row(b, slot, h) : -1;
    if (at < 0) continue;  // the same for all lanes of a row
    uint32_t top = 0;
    if (in) {
      const bits* row = key ? static_cast<const bits*>(a.k) + b * a.ks.b + t * a.ks.t + h * a.ks.h
                            : static_cast<const bits*>(a.v) + b * a.vs.b + t * a.vs.t + h * a.vs.h;
      RotaryArgs rot = a.rot;
      if (!key) rot.rotary = 0;
      p.load(row, d0, rot);
      p.rotate(y, row, d0, rot, cs);
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, as_u32(y[i]) & 0x7fffffffu);
    }
    void* pool = key ? a.c.k : a.c.v;
    if constexpr (FMT == KV_16BIT) {
      if (in) {
        Packet<T> o;
        o.pack(y);
        *reinterpret_cast<u32x4*>(static_cast<bits*>(pool) + at * a.c.d + d0) = o.raw;
      }
    } else {
      top = row_max(top, a.lanes);
      const bool finite = top < 0x7f800000u;
      const float scale = finite ? fmaxf(as_f32(top) / kv_top<FMT>(), 1e-8f) : as_f32(top);
      if (in) {
        u32x2 code = {0, 0};
        if (finite) {
          float lo[4], hi[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            lo[i] = y[i] / scale;
            hi[i] = y[4 + i] / scale;
          }
          code = u32x2{encode4<FMT>(lo), encode4<FMT>(hi)};
        }
        *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(pool) + at * a.c.d + d0) = code;
      }
      if (d0 == 0) (key ? a.c.k_scale : a.c.v_scale)[at] = scale;
    }
  }
}

struct ReadArgs {
  KvCache c;
  void *k_out, *v_out;  // [batch, heads, tokens, d]
  const int32_t *start, *end;
  int64_t tokens, rows;  // rows = batch * heads * tokens
  int lanes;
};

template <typename T, int FMT> __global__ __launch_bounds__(256) void read_rows(ReadArgs a) {
  typedef typename T::bits bits;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * (256 / a.lanes) + threadIdx.x / a.lanes;
  const int d0 = (threadIdx.x % a.lanes) * 8;
  if (r >= a.rows || d0 >= a.c.d) return;
  const int64_t bh = r / a.tokens, i = r % a.tokens, b = bh / a.c.heads;
  const int64_t slot = (a.start ? a.start[b] : 0) + i;
  const int64_t at = slot < a.end[b] ? a.c.row(b, slot, static_cast<int>(bh % a.c.heads)) : -1;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    Packet<T> o;
    o.raw = u32x4{0, 0, 0, 0};
    const void* pool = side ? a.c.v : a.c.k;
    if (at >= 0) {
      if constexpr (FMT == KV_16BIT) {
        o.raw = *reinterpret_cast<const u32x4*>(static_cast<const bits*>(pool) + at * a.c.d + d0);
      } else {
        const u32x2 code = *reinterpret_cast<const u32x2*>(static_cast<const uint8_t*>(pool) + at * a.c.d + d0);
        const float scale = (side ? a.c.v_scale : a.c.k_scale)[at];
        float lo[4], hi[4], f[8];
        decode4<FMT>(code[0], lo);
        decode4<FMT>(code[1], hi);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[j] = lo[j] * scale;
          f[4 + j] = hi[j] * scale;
        }
        o.pack(f);
      }
    }
    *reinterpret_cast<u32x4*>(static_cast<bits*>(side ? a.v_out : a.k_out) + r * a.c.d + d0) = o.raw;
  }
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

template <typename T> int append_typed(const AppendArgs& a, int fmt, dim3 grid, hipStream_t s) {
  static const char* what = "kv_cache_append launch";
  if (fmt == KV_INT8) return launch(append_rows<T, KV_INT8>, grid, 256, 0, a, s, what);
  if (fmt == KV_E4M3) return launch(append_rows<T, KV_E4M3>, grid, 256, 0, a, s, what);
  return launch(append_rows<T, KV_16BIT>, grid, 256, 0, a, s, what);
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
               {strides[6], strides[7], strides[8]}, tokens, q_heads, 0, 0};
  const int rows = q_heads + 2 * a.c.heads;
  a.lanes = row_lanes(a.c.d / 8);
  // one pass over rows per workgroup until the tokens alone fill the chip
  a.rows_per_wg = batch * tokens < 1024 ? 256 / a.lanes : rows;
  const dim3 grid(static_cast<unsigned>(batch * tokens),
                  static_cast<unsigned>((rows + a.rows_per_wg - 1) / a.rows_per_wg));
  return dtype == MI355_F16 ? append_typed<F16>(a, cache.format, grid, stream)
                            : append_typed<BF16>(a, cache.format, grid, stream);
}

int kv_read_launch(const mi355_kv_cache& cache, void* k_out, void* v_out, const int32_t* start, const int32_t* end,
                   int64_t batch, int64_t tokens, int dtype, hipStream_t stream) {
  ReadArgs a{kv_cache_args(cache), k_out, v_out, start, end, tokens, batch * cache.kv_heads * tokens, 0};
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
