// Attention under shared prefixes: the kernels for bf16.
#include "shared_prefix_kernels.h"

namespace mi355 {

int shared_prefix_run_bf16(const SharedArgs& a, const SharedPlan& p, int format, hipStream_t s) {
  return shared_prefix_run<BF16>(a, p, format, s);
}

}  // namespace mi355
