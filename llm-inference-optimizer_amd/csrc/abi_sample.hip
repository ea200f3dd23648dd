// C ABI entry point of drawing tokens (include/mi355_fused.h): argument
// validation.  Kernels and their launcher live in sample.hip.
#include "common.h"

namespace mi355 {

int64_t sample_workspace(int64_t rows, int64_t vocab);
int sample_launch(const void* logits, const float* uniform, int64_t* tokens, float* logprobs, const float* temperature,
                  const int32_t* top_k, const float* top_p, const float* min_p, float temperature_all, int32_t top_k_all,
                  float top_p_all, float min_p_all, int64_t rows, int vocab, int64_t stride, int dtype, void* work,
                  hipStream_t stream);

}  // namespace mi355

using mi355::set_error;

namespace {
constexpr int64_t kMaxRows = int64_t{1} << 20, kMaxVocab = int64_t{1} << 20;
}

MI355_EXPORT int64_t mi355_sample_tokens_workspace(int64_t rows, int64_t vocab) {
  mi355::clear_error();
  if (rows < 1 || rows >= kMaxRows || vocab < 1 || vocab >= kMaxVocab) return 0;
  return mi355::sample_workspace(rows, vocab);
}

MI355_EXPORT int mi355_sample_tokens_fwd(const void* logits, const float* uniform, int64_t* tokens, float* logprobs,
                                         const float* temperature, const int32_t* top_k, const float* top_p,
                                         const float* min_p, float temperature_all, int32_t top_k_all, float top_p_all,
                                         float min_p_all, int64_t rows, int64_t vocab, int64_t row_stride, int dtype,
                                         void* workspace, int64_t workspace_bytes, void* stream) {
  static const char* fn = "mi355_sample_tokens_fwd";
  mi355::clear_error();
  if (!mi355::valid_dtype(dtype)) {
    set_error("%s: unknown dtype code %d", fn, dtype);
    return MI355_ERR_INVALID;
  }
  if (rows < 0 || vocab < 1 || row_stride < vocab) {
    set_error("%s: sizes out of range (rows >= 0, vocab >= 1, row_stride >= vocab)", fn);
    return MI355_ERR_INVALID;
  }
  if (rows == 0) return MI355_OK;
  if (rows >= kMaxRows || vocab >= kMaxVocab) {
    set_error("%s: size beyond the kernel's limits (rows < 2^20, vocab < 2^20)", fn);
    return MI355_ERR_UNSUPPORTED;
  }
  if (logits == nullptr || uniform == nullptr || tokens == nullptr) {
    set_error("%s: null pointer", fn);
    return MI355_ERR_INVALID;
  }
  const int64_t needs = mi355::sample_workspace(rows, vocab);
  if (needs > 0 && (workspace == nullptr || !mi355::aligned16(workspace) || workspace_bytes < needs)) {
    set_error("%s: the workspace must be 16-byte aligned and of %lld bytes", fn, static_cast<long long>(needs));
    return MI355_ERR_INVALID;
  }
  return mi355::sample_launch(logits, uniform, tokens, logprobs, temperature, top_k, top_p, min_p, temperature_all,
                              top_k_all, top_p_all, min_p_all, rows, static_cast<int>(vocab), row_stride, dtype,
                              workspace, static_cast<hipStream_t>(stream));
}
