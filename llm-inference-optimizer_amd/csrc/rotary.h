// Rotary positions, shared by the rotation alone (rotary.hip) and the cache
// append that rotates queries and keys on their way (kv_cache.hip).
//
// With R = 2 len(inv_freq) <= D rotated elements per head, position p and
// frequency f_j:   a = p f_j,  c = scale cos a,  s = scale sin a
//   y0 = x0 c - x1 s,   y1 = x1 c + x0 s      (fp32, rounded once)
// for the pairs (x_j, x_{j + R/2}) of the half layout or (x_2j, x_2j+1) of the
// interleaved one; the other D - R elements pass unchanged.
//
// Angles: p f_j reaches 10^6 radians, where one fp32 rounding of the product
// is off by 0.03.  A 64-bit product of an int64 position (below 2^29) and an
// fp32 frequency is exact; it is reduced to a fraction of a turn in 64 bits,
// and only that fraction (|t| <= 1/2) goes to 32 bits for the sine and cosine:
// at most 2^-26 turns, 10^-7 radians.  64-bit operations run at half the
// 32-bit rate on this chip, and a wave computes a token's R/2 angles once for
// all of its heads (through LDS).
#pragma once

#include "common.h"

namespace mi355 {

constexpr int kMaxPairs = 128;  // R / 2 of heads up to 256 wide

struct RotaryArgs {
  const int64_t* positions;  // [batch, tokens] by the two strides
  const float* inv_freq;     // [rotary / 2]
  int64_t pos_stride_b, pos_stride_t;
  float scale;
  int rotary;       // R
  int interleaved;  // 0: half layout
};

// Fills cs[j] = scale cos(p f_j), cs[kMaxPairs + j] = scale sin(p f_j) with
// `count` threads, this one the `index`-th; a barrier among them follows.
__device__ __forceinline__ void rotary_angles(float* cs, const RotaryArgs& a, int64_t p, int index, int count) {
  for (int j = index; j < a.rotary / 2; j += count) {
    const double turns = static_cast<double>(p) * static_cast<double>(a.inv_freq[j]) * 0.15915494309189533577;
    const float t = static_cast<float>(turns - __builtin_rint(turns));
    float s, c;
    sincospif(2.0f * t, &s, &c);
    cs[j] = a.scale * c;
    cs[kMaxPairs + j] = a.scale * s;
  }
}

// How a lane's packet of elements meets its pairs.
enum RotaryMode {
  ROTARY_NONE,   // nothing is rotated
  ROTARY_HALF,   // half layout, whole packets of partners
  ROTARY_PAIRS,  // interleaved
  ROTARY_ODD     // half layout, R / 2 no multiple of a packet: partners one by one
};
inline RotaryMode rotary_mode(const RotaryArgs& a, int width) {
  if (a.rotary == 0) return ROTARY_NONE;
  if (a.interleaved) return ROTARY_PAIRS;
  return a.rotary / 2 % width == 0 ? ROTARY_HALF : ROTARY_ODD;
}

// A lane's elements d0 .. d0 + W - 1 of every head turn by the same angles:
//   y[i] = x[i] c[i] + (partner of x[i]) s[i]     for i < turned, x[i] beyond
// with the sine's sign in s.  Held in registers over the heads of a token.
template <typename T, int MODE> struct RotaryLane {
  static constexpr int W = pack_width<T>::value;
  float c[W], s[W];
  int d0, turned;

  __device__ __forceinline__ RotaryLane(const RotaryArgs& a, int d0_) : d0(d0_) {
    turned = MODE == ROTARY_NONE ? 0 : max(0, min(a.rotary - d0, W));
  }
  // The element that rotates into element d of a half layout.
  static __device__ __forceinline__ int partner(const RotaryArgs& a, int d) {
    const int half = a.rotary / 2;
    return d < half ? d + half : d - half;
  }
  __device__ __forceinline__ void angles(const RotaryArgs& a, const float* cs) {
    const int half = a.rotary / 2;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if (i >= turned) break;
      const int d = d0 + i;
      const bool first = MODE == ROTARY_PAIRS ? (i & 1) == 0 : d < half;
      const int j = MODE == ROTARY_PAIRS ? d / 2 : first ? d : d - half;
      c[i] = cs[j];
      s[i] = first ? -cs[kMaxPairs + j] : cs[kMaxPairs + j];
    }
  }
};

// A head's packet and what rotates into it, on their way.
template <typename T, int MODE> struct RotaryPacket {
  static constexpr int W = pack_width<T>::value;
  typedef typename T::bits bits;
  Packet<T> own, other;
  bits single[MODE == ROTARY_ODD ? W : 1];

  __device__ __forceinline__ void load(const void* row, const RotaryLane<T, MODE>& lane, const RotaryArgs& a) {
    const bits* r = static_cast<const bits*>(row);
    own.raw = *reinterpret_cast<const u32x4*>(r + lane.d0);
    if constexpr (MODE == ROTARY_HALF)
      other.raw = *reinterpret_cast<const u32x4*>(r + (lane.turned ? lane.partner(a, lane.d0) : lane.d0));
    if constexpr (MODE == ROTARY_ODD) {
#pragma unroll
      for (int i = 0; i < W; ++i) single[i] = r[i < lane.turned ? lane.partner(a, lane.d0 + i) : lane.d0];
    }
  }
  __device__ __forceinline__ void turn(float (&y)[W], const RotaryLane<T, MODE>& lane) const {
    own.unpack(y);
    if constexpr (MODE == ROTARY_NONE) return;
    float o[W];
    if constexpr (MODE == ROTARY_HALF) other.unpack(o);
    if constexpr (MODE == ROTARY_PAIRS) own.unpack(o);
    if constexpr (MODE == ROTARY_ODD) {
#pragma unroll
      for (int i = 0; i < W; ++i) o[i] = load_elem<T>(&single[i], 0);
    }
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float v = y[i] * lane.c[i] + o[MODE == ROTARY_PAIRS ? i ^ 1 : i] * lane.s[i];
      y[i] = i < lane.turned ? v : y[i];
    }
  }
};

// Lanes that share a head's row, one 16-byte packet each: the power of two
// that holds them, so that rows do not straddle waves.
inline int row_lanes(int64_t packets) {
  int n = 4;
  while (n < packets) n *= 2;
  return n;
}

}  // namespace mi355
