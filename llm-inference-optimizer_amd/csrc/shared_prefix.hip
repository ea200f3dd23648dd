// Attention of a batch whose sequences share prefixes, over a paged cache, for
// gfx950: tree attention in which the slots below a sequence's shared length are
// those of its group's first sequence.
#include "tree_attention.h"

namespace mi355 {
namespace {

struct SharedArgs {
  KvCache c;
  const void* q;
  void* out;
  const int32_t *lens, *new_lens, *prefix_lens, *groups;
  const uint8_t* mask;
  int64_t mask_b, mask_t;
  int64_t qb, qt, qh;
  int batch, tokens, q_heads, group, group_count;
  float scale;
};

// A wave per query row.
template <typename T, int FMT> __global__ __launch_bounds__(64) void shared_prefix_rows(SharedArgs a) {
  typedef typename T::bits bits;
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int hq = static_cast<int>(row % a.q_heads), t = static_cast<int>(row / a.q_heads % a.tokens);
  const int b = static_cast<int>(row / a.q_heads / a.tokens), h = hq / a.group, d = a.c.d;
  const int cap = a.c.capacity();
  const int len = max(0, min(a.lens[b], cap)), fresh = max(0, min(a.new_lens ? a.new_lens[b] : a.tokens, a.tokens));
  const int end = min(len + fresh, cap);
  int first = b, shared = 0;
  for (int g = 0; g < a.group_count; ++g) {
    const int even = a.batch / a.group_count;
    const int g0 = a.groups ? max(0, min(a.groups[g], a.batch)) : g * even;
    const int g1 = a.groups ? max(0, min(a.groups[g + 1], a.batch)) : (g + 1) * even;
    if (b >= g0 && b < g1) {
      first = g0;
      shared = max(0, min(a.prefix_lens[g], len));
      break;
    }
  }
  __shared__ float q[256], weight[64];
  __shared__ int64_t rows[64];
  const bits* from = static_cast<const bits*>(a.q) + b * a.qb + t * a.qt + hq * a.qh;
  for (int e = lane; e < d; e += 64) q[e] = load_elem<T>(from, e);
  __syncthreads();
  float o[4] = {0, 0, 0, 0}, bad[4] = {0, 0, 0, 0}, most = kLow, sum = 0;
  for (int s0 = 0; s0 < (t < fresh ? end : 0); s0 += 64) {
    const int s = s0 + lane;
    int64_t at = s < end ? a.c.row(s < shared ? first : b, s, h) : -1;
    if (s >= len && at >= 0) {
      const int j = s - len;
      if (!(a.mask ? a.mask[b * a.mask_b + t * a.mask_t + j] != 0 : j <= t)) at = -1;
    }
    float score = -INFINITY;
    if (at >= 0) {
      float acc = 0;
      for (int e = 0; e < d; e += 4) {
        float k[4];
        if constexpr (FMT == KV_16BIT) {
          for (int i = 0; i < 4; ++i) k[i] = load_elem<T>(a.c.k, at * d + e + i);
        } else {
          decode4<FMT>(*reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.c.k) + at * d + e), k);
        }
        for (int i = 0; i < 4; ++i) acc += k[i] * q[e + i];
      }
      if constexpr (FMT != KV_16BIT) acc *= a.c.k_scale[at];
      score = acc * a.scale;
    }
    float top = score;
    for (int m = 32; m; m >>= 1) top = fmaxf(top, __shfl_xor(top, m));
    const float now = fmaxf(most, top), was = __builtin_amdgcn_exp2f(most - now);
    const float w = at >= 0 ? __builtin_amdgcn_exp2f(score - now) : 0.f;
    most = now;
    float part = w;
    for (int m = 32; m; m >>= 1) part += __shfl_xor(part, m);
    sum = sum * was + part;
    weight[lane] = w;
    rows[lane] = at;
    __syncthreads();
    for (int i = 0; i < 4; ++i) o[i] *= was;
    for (int j = 0; j < 64; ++j) {
      const int64_t r = rows[j];
      if (r < 0) continue;
      float vs = FMT != KV_16BIT ? a.c.v_scale[r] : 1.f;
      if (vs - vs != 0.f) vs = NAN;  // a scale that is not finite makes its row NaN
      for (int i = 0; 64 * i + lane < d; ++i) {
        const int e = 64 * i + lane;
        float v;
        if constexpr (FMT == KV_16BIT) {
          v = load_elem<T>(a.c.v, r * d + e);
        } else {
          float four[4];
          decode4<FMT>(static_cast<const uint8_t*>(a.c.v)[r * d + e], four);
          v = fp32_value(four[0] * vs);  // rounded: not fused into the test below
        }
        if (v - v == 0.f) o[i] += weight[j] * v;
        else bad[i] += v;
      }
    }
    __syncthreads();
  }
  for (int i = 0; 64 * i + lane < d; ++i) {
    const float v = bad[i] != 0.f || bad[i] != bad[i] ? bad[i] : sum == 0.f ? 0.f : o[i] / sum;
    store_elem<T>(a.out, row * d + 64 * i + lane, v);
  }
}

}  // namespace

int64_t shared_prefix_workspace(const mi355_kv_cache&, int64_t, int64_t, int64_t, int64_t) { return 0; }

int shared_prefix_launch(const mi355_kv_cache& cache, const void* q, void* out, const int32_t* lens,
                         const int32_t* new_lens, const int32_t* prefix_lens, const int32_t* groups, int group_count,
                         const uint8_t* mask, int64_t mask_b, int64_t mask_t, int64_t batch, int tokens, int q_heads,
                         const int64_t* q_strides, float scale, int dtype, void*, int64_t, hipStream_t stream) {
  const SharedArgs a{kv_cache_args(cache), q, out, lens, new_lens, prefix_lens, groups, mask, mask_b, mask_t,
                     q_strides[0], q_strides[1], q_strides[2], static_cast<int>(batch), tokens, q_heads,
                     q_heads / static_cast<int>(cache.kv_heads), group_count, scale * kLog2e};
  const dim3 grid(static_cast<unsigned>(batch * tokens * q_heads));
  const auto run = [&](auto* kernel) { return launch(kernel, grid, 64, 0, a, stream, "shared_prefix_attention launch"); };
  if (dtype == MI355_F16)
    return cache.format == KV_INT8   ? run(shared_prefix_rows<F16, KV_INT8>)
           : cache.format == KV_E4M3 ? run(shared_prefix_rows<F16, KV_E4M3>)
                                     : run(shared_prefix_rows<F16, KV_16BIT>);
  return cache.format == KV_INT8   ? run(shared_prefix_rows<BF16, KV_INT8>)
         : cache.format == KV_E4M3 ? run(shared_prefix_rows<BF16, KV_E4M3>)
                                   : run(shared_prefix_rows<BF16, KV_16BIT>);
}

}  // namespace mi355
