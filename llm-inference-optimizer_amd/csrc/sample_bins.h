// The bins of weights that sample.hip counts a row's logits in, a quarter of a
// power of 2 wide.  Host and device code.
#pragma once

#include <math.h>
#include <stdint.h>

namespace mi355 {

constexpr int kBins = 256;  // the last holds all that is further down

// Bins per unit of the logits, c = log2 e / temperature: 0 for an infinite
// temperature, infinity for those below 2^-126.
__host__ __device__ inline float bins_per_unit(double c) { return 4.f * static_cast<float>(c); }

// The bin of a logit: a monotone function of it alone, for every scale.  Infinity
// is in the highest bin also where its product with a scale of 0 is NaN; 0 times
// an infinite scale is, as logits below it, in the lowest.
__host__ __device__ inline int bin_of(float x, float scale) {
  const float q = fminf(fmaxf(floorf(x * scale), -1e9f), 1e9f);
  return static_cast<int>(x == INFINITY ? 1e9f : q);
}
// Where a part whose largest logit has bin `top` counts one of bin q <= top.
__host__ __device__ inline int bin_in_part(int top, int q) {
  const int below = top - q > 0 ? top - q : 0;
  return below < kBins - 1 ? below : kBins - 1;
}
// The row's bin g is the part's bin g - this, `q_top` and q <= q_top being the largest
// logits' bins: in [0, kBins], as indexes are made of it.
__host__ __device__ inline int shift_of_part(int q_top, int q) {
  const int below = q_top - q > 0 ? q_top - q : 0;
  return below < kBins ? below : kBins;
}

}  // namespace mi355
