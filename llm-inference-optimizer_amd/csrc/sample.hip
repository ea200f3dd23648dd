// Drawing a token per row of logits with temperature, top-k, top-p and min-p from
// one given uniform number, for gfx950.
//
// Tokens are ranked by their logit, equal ones by index; what the filters keep is
// a beginning of that order: all above a threshold and the first few equal to
// it.  The threshold is found digit by digit from histograms of the logits as
// ordered integers -- of counts for top-k, of weights for top-p, these as integer
// multiples of 2^-43, whose sums do not depend on the order of the atomics.
#include "common.h"

namespace mi355 {
namespace {

constexpr int kBlock = 1024, kBlockWaves = kBlock / 64;
constexpr double kUnit = 8796093022208.0;  // 2^43: sums of 2^20 weights fit 64 bits

struct SampleArgs {
  const void* logits;
  const float* uniform;
  int64_t* tokens;
  float* logprobs;
  const float* temperature;
  const int32_t* top_k;
  const float *top_p, *min_p;
  float temperature_all;
  int32_t top_k_all;
  float top_p_all, min_p_all;
  int64_t rows, stride;
  int vocab;
};

// Logits as integers in their order; those that are never drawn are 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > -INFINITY)) return 0;
  const uint32_t b = as_u32(x + 0.f);  // -0 counts as 0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return as_f32(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

template <typename V> __device__ __forceinline__ V block_sum(V v, V* part) {
  for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  V sum = part[0];
  for (int w = 1; w < kBlockWaves; ++w) sum += part[w];
  __syncthreads();
  return sum;
}

template <typename T> struct Row {
  const SampleArgs& a;
  int64_t base;
  uint32_t top;      // key of the largest logit
  double peak, heat; // its value, the temperature
  __device__ __forceinline__ uint32_t key(int i) const { return key_of(load_elem<T>(a.logits, base + i)); }
  __device__ __forceinline__ double weight(uint32_t k) const {
    if (k == 0) return 0.;
    if (top == key_of(INFINITY)) return k == top ? 1. : 0.;
    return exp((static_cast<double>(value_of(k)) - peak) / heat);
  }
};

// The key at which the count (WEIGHTS: the weights) of the ranked tokens reaches
// `want`: f(key) of all above it is below want.  *above: theirs.
template <bool WEIGHTS, typename T>
__device__ uint32_t cross(const Row<T>& r, uint64_t want, uint64_t* above, uint64_t* bins) {
  uint32_t prefix = 0, mask = 0;
  uint64_t before = 0;
  __shared__ uint32_t digit;
  __shared__ uint64_t upto;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kBlock) bins[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < r.a.vocab; i += kBlock) {
      const uint32_t k = r.key(i);
      if (k == 0 || (k & mask) != prefix) continue;
      const uint64_t v = WEIGHTS ? static_cast<uint64_t>(r.weight(k) * kUnit + 0.5) : 1;
      atomicAdd(reinterpret_cast<unsigned long long*>(&bins[k >> shift & 255]), static_cast<unsigned long long>(v));
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      uint64_t s = before;
      int found = 0, lowest = 0;
      for (int i = 255; i >= 0; --i) {
        if (bins[i] == 0) continue;
        lowest = i;
        if (s + bins[i] >= want) {
          found = 1;
          break;
        }
        s += bins[i];
      }
      if (!found) s -= bins[lowest];  // fewer than wanted: the last
      digit = lowest;
      upto = s;
    }
    __syncthreads();
    prefix |= digit << shift;
    mask |= 255u << shift;
    before = upto;
    __syncthreads();
  }
  *above = before;
  return prefix;
}

template <typename T> __global__ __launch_bounds__(kBlock) void sample_rows(SampleArgs a) {
  __shared__ uint64_t bins[256];
  __shared__ double parts[kBlockWaves];
  __shared__ int ints[kBlockWaves];
  __shared__ double scan[kBlock];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Row<T> r{a, row * a.stride, 0, 0, 0};
  const float heat = a.temperature ? a.temperature[row] : a.temperature_all;
  const int top_k = a.top_k ? a.top_k[row] : a.top_k_all;
  const float top_p = a.top_p ? a.top_p[row] : a.top_p_all, min_p = a.min_p ? a.min_p[row] : a.min_p_all;
  const float u = fminf(fmaxf(a.uniform[row], 0.f), 0.99999994f);

  uint32_t top = 0;
  for (int i = threadIdx.x; i < a.vocab; i += kBlock) top = max(top, r.key(i));
  for (int m = 32; m; m >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), m)));
  if (lane == 0) bins[wave] = top;
  __syncthreads();
  for (int w = 0; w < kBlockWaves; ++w) top = max(top, static_cast<uint32_t>(bins[w]));
  __syncthreads();
  if (top == 0) {
    if (threadIdx.x == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    return;
  }
  r.top = top;
  r.peak = value_of(top);
  r.heat = heat;
  const bool greedy = !(heat > 0.f);

  // what is kept: keys above `edge`, the first `ties` tokens of that key, weights from `least` on
  uint32_t edge = 0;
  int64_t ties = 0;
  if (greedy) {
    edge = top;
    ties = 1;
  } else {
    double total = 0;
    if (top_k > 0 && top_k < a.vocab) {
      uint64_t above;
      edge = cross<false>(r, top_k, &above, bins);
      ties = top_k - static_cast<int64_t>(above);
    }
    if (top_p < 1.f) {
      for (int i = threadIdx.x; i < a.vocab; i += kBlock) {
        const uint32_t k = r.key(i);
        if (k > edge) total += r.weight(k);
      }
      total = block_sum(total, parts) + static_cast<double>(ties) * r.weight(edge);
      const double need = static_cast<double>(top_p) * total;
      uint64_t above;
      const uint32_t at = cross<true>(r, max(uint64_t{1}, static_cast<uint64_t>(ceil(need * kUnit))), &above, bins);
      const double before = static_cast<double>(above) / kUnit, w = r.weight(at);
      int64_t m = w > 0 ? static_cast<int64_t>(fmin(ceil((need - before) / w), 1e9)) : 1;
      m = max(m, int64_t{1});
      if (at == edge) ties = min(ties, m);
      else if (at > edge) edge = at, ties = m;
    }
  }
  const double least = !greedy && min_p > 0.f ? min_p : 0.;

  // the order of the vocabulary, twice: the kept weights' total, then the first token beyond u of it
  double total = 0, goal = 0;
  int last = -1;  // the last kept token so far
  for (int pass = 0; pass < 2; ++pass) {
    int64_t equal = 0;  // tokens of key `edge` so far
    double before = 0;
    for (int i0 = 0; i0 < a.vocab; i0 += kBlock) {
      const int i = i0 + threadIdx.x;
      const uint32_t k = i < a.vocab ? r.key(i) : 0;
      const bool tie = k != 0 && k == edge;
      const uint64_t all = __builtin_amdgcn_ballot_w64(tie);
      if (lane == 0) ints[wave] = __popcll(all);
      __syncthreads();
      int64_t rank = equal + __popcll(all & ((uint64_t{1} << lane) - 1));
      for (int w = 0; w < kBlockWaves; ++w) {
        if (w < wave) rank += ints[w];
        equal += ints[w];
      }
      double v = k > edge || (tie && rank < ties) ? r.weight(k) : 0.;
      if (v < least && k != top) v = 0;
      if (k == top && (k > edge || rank < ties)) v = 1;
      scan[threadIdx.x] = v;
      __syncthreads();
      for (int step = 1; step < kBlock; step *= 2) {
        const double add = static_cast<int>(threadIdx.x) >= step ? scan[threadIdx.x - step] : 0.;
        __syncthreads();
        scan[threadIdx.x] += add;
        __syncthreads();
      }
      const double upto = before + scan[threadIdx.x];
      if (pass == 1) {
        const bool hit = v > 0 && upto > goal;
        const bool other = v > 0;
        const uint64_t hits = __builtin_amdgcn_ballot_w64(hit), others = __builtin_amdgcn_ballot_w64(other);
        if (lane == 0) {
          ints[wave] = hits ? i0 + 64 * wave + __builtin_ctzll(hits) : -1;
          bins[wave] = others ? i0 + 64 * wave + 63 - __builtin_clzll(others) : 0xffffffffu;
        }
        __syncthreads();
        int found = -1;
        for (int w = kBlockWaves - 1; w >= 0; --w) {
          if (ints[w] >= 0) found = ints[w];
        }
        for (int w = 0; w < kBlockWaves; ++w)
          if (bins[w] != 0xffffffffu) last = static_cast<int>(bins[w]);
        if (found >= 0) {
          last = found;
          break;
        }
      }
      before += scan[kBlock - 1];
      __syncthreads();
    }
    __syncthreads();
    if (pass == 0) {
      total = before;
      goal = static_cast<double>(u) * total;
    }
  }
  if (threadIdx.x == 0) {
    a.tokens[row] = last;
    if (a.logprobs) a.logprobs[row] = static_cast<float>(log((greedy ? 1. : r.weight(r.key(last))) / total));
  }
}

}  // namespace

int64_t sample_workspace(int64_t, int64_t) { return 0; }

int sample_launch(const void* logits, const float* uniform, int64_t* tokens, float* logprobs, const float* temperature,
                  const int32_t* top_k, const float* top_p, const float* min_p, float temperature_all, int32_t top_k_all,
                  float top_p_all, float min_p_all, int64_t rows, int vocab, int64_t stride, int dtype, void*,
                  hipStream_t stream) {
  const SampleArgs a{logits, uniform, tokens, logprobs, temperature, top_k, top_p, min_p, temperature_all, top_k_all,
                     top_p_all, min_p_all, rows, stride, vocab};
  const dim3 grid(static_cast<unsigned>(rows));
  static const char* what = "sample_tokens launch";
  if (dtype == MI355_F32) return launch(sample_rows<F32>, grid, kBlock, 0, a, stream, what);
  if (dtype == MI355_F16) return launch(sample_rows<F16>, grid, kBlock, 0, a, stream, what);
  return launch(sample_rows<BF16>, grid, kBlock, 0, a, stream, what);
}

}  // namespace mi355
