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
// For one wave: LDS operations of a wave are done in order.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// How a lane's packet of elements meets its pairs.
enum RotaryMode {
  ROTARY_NONE,    // nothing is rotated
  ROTARY_HALF,    // half layout, whole packets of partners
  ROTARY_PAIRS,   // interleaved, whole packets of pairs
  ROTARY_SINGLE   // element by element: R / 2 (or, interleaved, R) is no multiple of a packet
};
inline RotaryMode rotary_mode(const RotaryArgs& a, int width) {
  if (a.rotary == 0) return ROTARY_NONE;
  if (a.interleaved) return a.rotary % width == 0 ? ROTARY_PAIRS : ROTARY_SINGLE;
  return a.rotary / 2 % width == 0 ? ROTARY_HALF : ROTARY_SINGLE;
}

// A lane's elements d0 .. d0 + W - 1 of every head turn by the same angles:
//   y[i] = x[i] c[i] + (partner of x[i]) s[i]
// with the sine's sign in s.  Held in registers over the heads of a token.
template <typename T, int MODE> struct RotaryLane {
  static constexpr int W = pack_width<T>::value;
  float c[W], s[W];
  int d0, partner;  // first element of the packet that holds the partners
  bool turned;

  __device__ __forceinline__ RotaryLane(const RotaryArgs& a, int d0_) : d0(d0_) {
    const int half = a.rotary / 2;
    turned = MODE != ROTARY_NONE && d0 < a.rotary;
    partner = MODE != ROTARY_HALF || !turned ? d0 : d0 < half ? d0 + half : d0 - half;
  }
  __device__ __forceinline__ void angles(const RotaryArgs& a, const float* cs) {
    if constexpr (MODE == ROTARY_HALF || MODE == ROTARY_PAIRS) {
      if (!turned) return;
      const int half = a.rotary / 2;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const int j = MODE == ROTARY_PAIRS ? (d0 + i) / 2 : (d0 < half ? d0 : d0 - half) + i;
        const bool first = MODE == ROTARY_PAIRS ? (i & 1) == 0 : d0 < half;
        c[i] = cs[j];
        s[i] = first ? -cs[kMaxPairs + j] : cs[kMaxPairs + j];
      }
    }
  }
  // The packet `own` of a head and, in the half layout, its partners'.
  __device__ __forceinline__ void turn(float (&y)[W], const Packet<T>& own, const Packet<T>& other, const void* row,
                                       const RotaryArgs& a, const float* cs) const {
    own.unpack(y);
    if (!turned) return;
    if constexpr (MODE == ROTARY_HALF) {
      float o[W];
      other.unpack(o);
#pragma unroll
      for (int i = 0; i < W; ++i) y[i] = y[i] * c[i] + o[i] * s[i];
    } else if constexpr (MODE == ROTARY_PAIRS) {
#pragma unroll
      for (int i = 0; i < W; i += 2) {
        const float x0 = y[i], x1 = y[i + 1];
        y[i] = x0 * c[i] + x1 * s[i];
        y[i + 1] = x1 * c[i + 1] + x0 * s[i + 1];
      }
    } else if constexpr (MODE == ROTARY_SINGLE) {
      const float* sn = cs + kMaxPairs;
      const int half = a.rotary / 2;
#pragma unroll 1
      for (int i = 0; i < W; ++i) {
        const int d = d0 + i;
        if (d >= a.rotary) break;
        const bool first = a.interleaved ? (d & 1) == 0 : d < half;
        const int j = a.interleaved ? d / 2 : first ? d : d - half;
        const float x = load_elem<T>(row, d);
        const float o = load_elem<T>(row, a.interleaved ? d ^ 1 : first ? d + half : d - half);
        const float v = x * cs[j] + (first ? -(o * sn[j]) : o * sn[j]);
#pragma unroll
        for (int e = 0; e < W; ++e) y[e] = e == i ? v : y[e];
      }
    }
  }
};

// A head's packet and its partners', on their way.
template <typename T, int MODE> struct RotaryPacket {
  Packet<T> own, other;
  __device__ __forceinline__ void load(const void* row, const RotaryLane<T, MODE>& lane) {
    const typename T::bits* r = static_cast<const typename T::bits*>(row);
    own.raw = *reinterpret_cast<const u32x4*>(r + lane.d0);
    if constexpr (MODE == ROTARY_HALF) other.raw = *reinterpret_cast<const u32x4*>(r + lane.partner);
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
