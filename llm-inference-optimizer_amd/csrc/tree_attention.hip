// Attention of a few new tokens per sequence over a paged cache (simple form:
// a wave per query row, one cache slot after the other).
#include "kv_cache.h"

namespace mi355 {
namespace {

struct TreeArgs {
  KvCache c;
  const void* q;
  void* out;  // [batch, tokens, q_heads, d]
  const int32_t *lens, *new_lens;
  const uint8_t* mask;  // [batch, tokens, tokens] by strides, or null: a chain
  int64_t mask_b, mask_t;
  int64_t qb, qt, qh;
  int64_t rows;
  int tokens, q_heads;
  float scale;
};

template <typename T, int FMT> __device__ __forceinline__ float cache_elem(const void* pool, const float* scales, int64_t row, int d, int i) {
  if constexpr (FMT == KV_16BIT) return load_elem<T>(pool, row * d + i);
  else {
    const uint32_t code = static_cast<const uint8_t*>(pool)[row * d + i];
    float f[4];
    decode4<FMT>(code, f);
    return f[0] * scales[row];
  }
}

template <typename T, int FMT> __global__ __launch_bounds__(64) void tree_attention_rows(TreeArgs a) {
  const int64_t r = blockIdx.x;
  const int lane = threadIdx.x;
  const int h = r % a.q_heads, kvh = h / (a.q_heads / a.c.heads);
  const int64_t bt = r / a.q_heads, b = bt / a.tokens;
  const int t = bt % a.tokens;
  const int cap = a.c.capacity();
  const int len = max(0, min(a.lens[b], cap));
  const int fresh = max(0, min(a.new_lens ? a.new_lens[b] : a.tokens, a.tokens));
  const int last = t < fresh ? min(len + fresh, cap) : 0;
  float q[4], o[4] = {0, 0, 0, 0}, m = -INFINITY, sum = 0;
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    q[i] = d < a.c.d ? load_elem<T>(a.q, b * a.qb + t * a.qt + h * a.qh + d) : 0.f;
  }
  for (int s = 0; s < last; ++s) {
    if (s >= len) {
      const int j = s - len;
      if (a.mask ? a.mask[b * a.mask_b + t * a.mask_t + j] == 0 : j > t) continue;
    }
    const int64_t row = a.c.row(b, s, kvh);
    if (row < 0) continue;
    float dot = 0;
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      if (d < a.c.d) dot += q[i] * cache_elem<T, FMT>(a.c.k, a.c.k_scale, row, a.c.d, d);
    }
    const float score = wave_allreduce_sum(dot) * a.scale;
    if (score == -INFINITY) continue;
    const float top = fmaxf(m, score);
    const float was = expf(m - top), p = expf(score - top);
    m = top;
    sum = sum * was + p;
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      if (d < a.c.d) o[i] = o[i] * was + p * cache_elem<T, FMT>(a.c.v, a.c.v_scale, row, a.c.d, d);
    }
  }
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    if (d < a.c.d) store_elem<T>(a.out, r * a.c.d + d, sum == 0.f ? 0.f : o[i] / sum);
  }
}

template <typename T> int tree_typed(const TreeArgs& a, int fmt, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.rows));
  static const char* what = "tree_attention launch";
  if (fmt == KV_INT8) return launch(tree_attention_rows<T, KV_INT8>, grid, 64, 0, a, s, what);
  if (fmt == KV_E4M3) return launch(tree_attention_rows<T, KV_E4M3>, grid, 64, 0, a, s, what);
  return launch(tree_attention_rows<T, KV_16BIT>, grid, 64, 0, a, s, what);
}

}  // namespace

int64_t tree_attention_workspace(const mi355_kv_cache&, int64_t, int64_t, int64_t) { return 0; }

int tree_attention_launch(const mi355_kv_cache& cache, const void* q, void* out, const int32_t* lens,
                          const int32_t* new_lens, const uint8_t* mask, int64_t mask_b, int64_t mask_t, int64_t batch,
                          int tokens, int q_heads, const int64_t* q_strides, float scale, int dtype, void*, int64_t,
                          hipStream_t stream) {
  const TreeArgs a{kv_cache_args(cache), q, out, lens, new_lens, mask, mask_b, mask_t, q_strides[0], q_strides[1],
                   q_strides[2], batch * tokens * q_heads, tokens, q_heads, scale};
  return dtype == MI355_F16 ? tree_typed<F16>(a, cache.format, stream) : tree_typed<BF16>(a, cache.format, stream);
}

}  // namespace mi355
