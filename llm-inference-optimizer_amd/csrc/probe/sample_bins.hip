// For checks on the CPU, not part of the kernel ABI: the bins of sample.hip
// (sample_bins.h), computed by the host.
#include <hip/hip_runtime.h>

#include "../sample_bins.h"

// out3 = {bin of logit x, where a part whose largest logit is `part` counts x,
// the shift of such a part in a row whose largest logit is `row`}.
extern "C" __attribute__((visibility("default"))) void mi355_probe_sample_bins(float temperature, float x, float part,
                                                                                float row, int* out3) {
  const float scale = mi355::bins_per_unit(1.4426950408889634074 / static_cast<double>(temperature));
  const int bin = mi355::bin_of(x, scale), top = mi355::bin_of(part, scale);
  out3[0] = bin;
  out3[1] = mi355::bin_in_part(top, bin);
  out3[2] = mi355::shift_of_part(mi355::bin_of(row, scale), top);
}
