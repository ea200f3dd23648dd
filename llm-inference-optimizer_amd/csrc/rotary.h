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
// 32-bit rate on this chip, and a workgroup computes a token's R/2 angles once
// for all of its heads (through LDS).
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

// Fills cs[j] = scale cos(p f_j), cs[kMaxPairs + j] = scale sin(p f_j); every
// thread of the workgroup calls it, then a barrier.
__device__ __forceinline__ void rotary_angles(float* cs, const RotaryArgs& a, int64_t p) {
  for (int j = threadIdx.x; j < a.rotary / 2; j += blockDim.x) {
    const double turns = static_cast<double>(p) * static_cast<double>(a.inv_freq[j]) * 0.15915494309189533577;
    const float t = static_cast<float>(turns - __builtin_rint(turns));
    float s, c;
    sincospif(2.0f * t, &s, &c);
    cs[j] = a.scale * c;
    cs[kMaxPairs + j] = a.scale * s;
  }
}

// Elements d0 .. d0 + W - 1 of one head, loaded with what rotates into them.
// `row` is the head's first element, 16-byte aligned; d0 a multiple of W.
template <typename T> struct RotaryPacket {
  static constexpr int W = pack_width<T>::value;
  Packet<T> own, other;

  __device__ __forceinline__ void load(const void* row, int d0, const RotaryArgs& a) {
    const typename T::bits* r = static_cast<const typename T::bits*>(row);
    own.raw = *reinterpret_cast<const u32x4*>(r + d0);
    const int half = a.rotary / 2;
    // half layout with whole packets of partners; single elements otherwise
    if (!a.interleaved && half % W == 0 && d0 < a.rotary)
      other.raw = *reinterpret_cast<const u32x4*>(r + (d0 < half ? d0 + half : d0 - half));
  }

  __device__ __forceinline__ void rotate(float (&y)[W], const void* row, int d0, const RotaryArgs& a,
                                         const float* cs) const {
    const float* sn = cs + kMaxPairs;
    const int half = a.rotary / 2;
    own.unpack(y);
    if (d0 >= a.rotary) return;
    if (a.interleaved) {
#pragma unroll
      for (int i = 0; i < W; i += 2) {
        if (d0 + i >= a.rotary) break;
        const int j = (d0 + i) / 2;
        const float x0 = y[i], x1 = y[i + 1];
        y[i] = x0 * cs[j] - x1 * sn[j];
        y[i + 1] = x1 * cs[j] + x0 * sn[j];
      }
    } else if (half % W == 0) {
      float o[W];
      other.unpack(o);
      const int j = d0 < half ? d0 : d0 - half;
      const float sign = d0 < half ? -1.0f : 1.0f;
#pragma unroll
      for (int i = 0; i < W; ++i) y[i] = y[i] * cs[j + i] + sign * (o[i] * sn[j + i]);
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const int d = d0 + i;
        if (d >= a.rotary) break;
        const bool lo = d < half;
        const float o = load_elem<T>(row, lo ? d + half : d - half);
        const int j = lo ? d : d - half;
        y[i] = y[i] * cs[j] + (lo ? -(o * sn[j]) : o * sn[j]);
      }
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
