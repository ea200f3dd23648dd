// Drawing a token per row of logits with temperature, top-k, top-p and min-p from
// one given uniform number, for gfx950.
//
// Tokens are ranked by their logit, equal ones by index; what the filters keep is
// a beginning of that order, told by its last token: a threshold of logits and,
// among those equal to it, of indexes.
//
//   w_i = 2^((x_i - M) log2 e / T),   M the largest logit
//
// Weights and sums have 64 bits: a token next to the border of the cumulated
// weights has to fall on the right side of it, whatever the order of the sums; in
// 32 bits one draw in a hundred from 150000 tokens would not.
//
// sample_parts reads the logits once, in parts of 4096 on all compute units: each
// part's largest logit and sum of weights, the largest logit of each block of
// 512, and, for rows with filters, how much weight (and for top-k, how many
// tokens) a part has in bins a quarter of a power of 2 wide.  Then a workgroup per
// row draws: without filters (sample_plain) from the part that the number falls
// into.  With them (sample_rows) a threshold's bin is known from the bins; that
// bin's tokens are sorted, which is the one other time that a row is read, and
// only blocks that reach up to it; and what is kept of a part is the sum of its
// bins above and of the sorted tokens before the threshold.
//
// sample_parts is bound by HBM without filters (512 rows of 151936 fp32, 311 MB: 79
// us, 3.9 TB/s) and by the weights' 64-bit arithmetic and the bins' atomics with them
// (64 rows of bf16: 20 us).  A row's workgroup is bound by trips of loads that wait
// for each other, some 1.5 us each: settings and parts 2 us, bins 4, the list 4 for
// a sharp row and 17 for a flat one, narrowing it 5 to 7 a step, kept parts 5, the
// drawing 3: 25 us for one row of 151936 with top-k and top-p, 60 for 64 rows of a
// nucleus, sharp and flat, 39 for 256 rows of 32000 with settings of their own, 18
// for 512 without filters.
//
// Not every threshold is in a bin that is short enough to list: at low temperatures,
// and where a mask leaves fewer tokens than top-k, the last one kept is in the last
// bin; flat rows have more than 8192 tokens in one.  Then the row's workgroup goes
// over the row for every digit of the threshold (by_digits) and a wave over it for
// the equal logits, which is slower than all else here by a factor of 10 to 40.
// One row of 151936 bf16, and 64 of them, us: top-k 50 at temperature 0.1 654, 870
// (with top-p 937, 1420); top-p 0.9 at temperature 2 902, 1117; 5 tokens left and
// top-k 20 640, 903.
#include "common.h"
#include "sample_bins.h"

namespace mi355 {
namespace {

constexpr int kPart = 4096, kBlock = 512, kPartBlocks = kPart / kBlock;
constexpr int kPartThreads = 256, kRowThreads = 512, kRowWaves = kRowThreads / 64;
constexpr int kListed = 8192, kPicked = 256;  // tokens that a row's workgroup lists, and sorts of them
constexpr int64_t kChunkParts = 32768;  // parts that the workspace holds, of whole rows: 100 MB
// Weights in whole numbers, whose sums do not depend on the atomics' order: 4096 of a
// part's, 2^20 of a row's fit 64 bits.  The row's are in two words, of 2^-43 and 2^-86
// (Fixed): a light token's weight may be little next to the first word's unit, but
// thousands of them are not, and with a small random number one of them is drawn.
constexpr double kBinUnit = 0x1p51, kUnit = 0x1p43;
constexpr float kHottest = 1e30f;   // temperatures beyond (infinity) have no weight range to clamp to

struct Part {
  float top;   // largest logit; -infinity: nothing to draw
  int32_t q;   // its bin
  double sum;  // of weights relative to it
};

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
  int64_t row0, rows, stride;  // of a chunk
  int vocab, parts;
  Part* part;                  // [rows][parts]
  float* block_top;            // [rows][parts * kPartBlocks]
  uint64_t* bins;              // [rows][parts][kBins]: weights relative to the part's largest, of kBinUnit
  uint32_t* counts;            // [rows][parts][kBins], of rows with top-k
};

struct Settings {
  float heat, top_p, min_p;
  int top_k;
  double c;  // log2 e / T
  bool greedy, by_count, by_weight, by_least;
  __device__ __forceinline__ Settings(const SampleArgs& a, int64_t row) {
    heat = a.temperature ? a.temperature[row] : a.temperature_all;
    top_k = a.top_k ? a.top_k[row] : a.top_k_all;
    top_p = a.top_p ? a.top_p[row] : a.top_p_all;
    min_p = a.min_p ? a.min_p[row] : a.min_p_all;
    if (min_p > 1.f) {  // no token weighs that much: the first of rank 0 alone
      top_k = 1;
      min_p = 0.f;
    }
    greedy = !(heat > 0.f);
    c = 1.4426950408889634074 / static_cast<double>(heat);
    by_count = !greedy && top_k > 0 && top_k < a.vocab;
    by_weight = !greedy && top_p < 1.f;
    by_least = !greedy && min_p > 0.f;
  }
  __device__ __forceinline__ bool filters() const { return by_count || by_weight || by_least; }
  __device__ __forceinline__ int bin(float x) const { return bin_of(x, bins_per_unit(c)); }
};

// 2^t for -1000 <= t <= 1/2: 1 + f g(f), with the polynomial g of degree 8 that meets
// (2^f - 1) / f at the Chebyshev nodes of [-1/2, 1/2], off by 3.7e-14 of it at most;
// exactly 1 for 0, so that equal largest logits weigh the same whole number in every sum.
__device__ __forceinline__ double exp2_64(double t) {
  const double magic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are t, rounded
  const double s = t + magic;
  const double f = t - (s - magic);
  double p = 1.0203121063391729e-07;
  p = __builtin_fma(p, f, 1.3255224878668817e-06);
  p = __builtin_fma(p, f, 1.525268684626772e-05);
  p = __builtin_fma(p, f, 0.00015403455852453838);
  p = __builtin_fma(p, f, 0.0013333558179043112);
  p = __builtin_fma(p, f, 0.009618129159402558);
  p = __builtin_fma(p, f, 0.055504108664760424);
  p = __builtin_fma(p, f, 0.2402265069581299);
  p = __builtin_fma(p, f, 0.6931471805599453);
  p = __builtin_fma(p, f, 1.0);
  const uint64_t n = __builtin_bit_cast(uint64_t, s) << 52;
  return __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, p) + n);
}

// Weights relative to a largest logit.  A weight below 2^-1000 counts as that: next
// to the largest, 1, it is nothing in 64 bits.  Only `exact` says whether there is
// a weight at all.
struct Weights {
  double top, c, least;  // least: of x - top
  float top32;
  bool plain;
  __device__ __forceinline__ Weights(const Settings& s, float top_) {
    top32 = top_;
    top = top_;
    c = s.c;
    least = -1000.0 / c;
    plain = top_ < INFINITY && s.heat <= kHottest;
  }
  __device__ __forceinline__ double fast(float x) const {
    return exp2_64(fmax(static_cast<double>(x) - top, least) * c);
  }
  __device__ __forceinline__ double exact(float x) const {
    if (!(x > -INFINITY)) return 0.;
    if (top32 == INFINITY) return x == INFINITY ? 1. : 0.;
    const double t = (static_cast<double>(x) - top) * c;
    return t < -1000. ? 0. : exp2_64(t);
  }
};

// A weight from 0 to 1 in two words, and what sums of them are.
struct Fixed {
  unsigned long long high, low;  // low: with a sign
  __device__ __forceinline__ explicit Fixed(double v) {
    const double a = __builtin_fma(v, kUnit, 0x1p52);  // rounded to whole numbers, which its low bits hold
    const double b = __builtin_fma(__builtin_fma(v, kUnit, -(a - 0x1p52)), kUnit, 0x1.8p52);
    high = __builtin_bit_cast(uint64_t, a) - __builtin_bit_cast(uint64_t, 0x1p52);
    low = __builtin_bit_cast(uint64_t, b) - __builtin_bit_cast(uint64_t, 0x1.8p52);
  }
  static __device__ __forceinline__ double value(unsigned long long high, unsigned long long low) {
    return (static_cast<double>(high) + static_cast<double>(static_cast<int64_t>(low)) / kUnit) / kUnit;
  }
};

__device__ __forceinline__ uint32_t key_of(float x) {  // in the logits' order; -0 counts as 0
  const uint32_t b = as_u32(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return as_f32(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// Logits of block `block` of a row: 8 per lane, -infinity beyond the vocabulary.
// PACKETS: rows start on 16 bytes and hold whole packets of 16.
template <typename T, bool PACKETS> struct Block {
  static constexpr int W = PACKETS ? pack_width<T>::value : 1;  // consecutive
  int first;
  u32x4 raw[PACKETS ? 8 / W : 1];
  float elem[PACKETS ? 1 : 8];
  static __device__ __forceinline__ int place(int e) {  // of element e, from the block's beginning
    const int lane = threadIdx.x & 63;
    return e / W * 64 * W + lane * W + e % W;
  }
  __device__ __forceinline__ void load(const SampleArgs& a, int64_t row, int block) {
    first = block * kBlock;
    const typename T::bits* p = static_cast<const typename T::bits*>(a.logits) + row * a.stride;
    if constexpr (PACKETS) {
      const rsrc_t r = make_rsrc(p, static_cast<uint32_t>(a.vocab) * sizeof(typename T::bits));
#pragma unroll
      for (int i = 0; i < 8 / W; ++i)
        raw[i] = buf_load16_cached(r, static_cast<uint32_t>((first + place(W * i)) * sizeof(typename T::bits)));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) elem[e] = load_elem<T>(p, min(first + place(e), a.vocab - 1));
    }
  }
  __device__ __forceinline__ void take(const SampleArgs& a, float (&x)[8]) const {
    if constexpr (PACKETS) {
#pragma unroll
      for (int i = 0; i < 8 / W; ++i) {
        Packet<T> k{raw[i]};
        float f[W];
        k.unpack(f);
#pragma unroll
        for (int e = 0; e < W; ++e) x[W * i + e] = f[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = elem[e];
    }
    if (first + kBlock > a.vocab) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = first + place(e) < a.vocab ? x[e] : -INFINITY;
    }
  }
  __device__ __forceinline__ int index(int e) const { return first + place(e); }
};

__device__ __forceinline__ float wave_max(float v) {
  for (int m = 32; m; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
  return v;
}
__device__ __forceinline__ double wave_sum(double v) {
  for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

template <typename T, bool PACKETS> __global__ __launch_bounds__(kPartThreads) void sample_parts(SampleArgs a) {
  constexpr int WAVES = kPartThreads / 64, OWN = kPartBlocks / WAVES;  // blocks of a wave
  __shared__ unsigned long long bins[kBins];
  __shared__ uint32_t counts[kBins];
  __shared__ float tops[WAVES];
  __shared__ double sums[WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  {
    const int64_t item = blockIdx.x, r = item / a.parts, row = a.row0 + r;
    const int part = static_cast<int>(item - r * a.parts);
    Block<T, PACKETS> b[OWN];
    float x[OWN][8];
#pragma unroll
    for (int i = 0; i < OWN; ++i) b[i].load(a, row, part * kPartBlocks + wave * OWN + i);
    const Settings s(a, row);
    const bool filters = s.filters();
    if (filters) bins[threadIdx.x] = counts[threadIdx.x] = 0;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      b[i].take(a, x[i]);
      float most = -INFINITY;  // NaN is no largest
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, x[i][e]);
      most = wave_max(most);
      if (lane == 0) a.block_top[(r * a.parts + part) * kPartBlocks + wave * OWN + i] = most;
      top = fmaxf(top, most);
    }
    if (lane == 0) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, tops[w]);
    const int q = s.bin(top);
    double sum = 0.;
    if (!s.greedy && top > -INFINITY) {
      const Weights w(s, top);
      const auto each = [&](const auto& weight) {
#pragma unroll
        for (int i = 0; i < OWN; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) sum += weight(x[i][e]);
      };
      const auto binned = [&](float x, double v) {
        if (x > -INFINITY) {
          const int l = bin_in_part(q, s.bin(x));
          // v times the unit, rounded, in the low 52 bits
          static_assert(kBinUnit <= 0x1p51, "2^52 more has the same exponent");
          const uint64_t fixed = __builtin_bit_cast(uint64_t, __builtin_fma(v, kBinUnit, 0x1p52)) & 0xfffffffffffffull;
          atomicAdd(&bins[l], static_cast<unsigned long long>(fixed));
          if (s.by_count) atomicAdd(&counts[l], 1u);
        }
        return v;
      };
      if (w.plain && !filters) each([&](float x) { return w.fast(x); });
      else if (w.plain) each([&](float x) { return binned(x, w.fast(x)); });
      else each([&](float x) { const double v = w.exact(x); return filters ? binned(x, v) : v; });
      sum = wave_sum(sum);
    }
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      double all = sums[0];
      for (int w = 1; w < WAVES; ++w) all += sums[w];
      a.part[r * a.parts + part] = Part{top, q, top > -INFINITY ? all : 0.};
    }
    if (filters) a.bins[(r * a.parts + part) * kBins + threadIdx.x] = bins[threadIdx.x];
    if (s.by_count) a.counts[(r * a.parts + part) * kBins + threadIdx.x] = counts[threadIdx.x];
    __syncthreads();
  }
}

// ------------------------------------------------------------------ a row

struct RowShared {
  uint64_t list[kListed + 64]; // tokens of some bins: key inverted, token
  double weight[2048];         // of blocks: these hold 2^20 tokens
  double parts[kRowWaves + 1];
  double bin_weight[kBins], bin_ranks[kBins];  // the row's
  double steps[kBins], ranks[kBins];           // of a part of the list
  unsigned long long radix[kBins], radix_low[kBins];  // Fixed sums; of counts the first alone
  uint32_t step_count[kBins];
  double part_unit[256];       // weight of a part's bins' unit
  int part_shift[256];         // the row's bin g is the part's bin g - shift
  alignas(16) uint64_t picked[kPicked];
  uint64_t sorted[kPicked];  // of the list, the tokens that a threshold is among
  int place[kPicked];
  int count, found, last, picked_count;
  float above;                 // the least logit above the list's bins
  unsigned long long low, high;
  uint32_t digit;
  uint64_t upto;
  double chosen;
};

// Sums of v over the threads before this one and it; *all: over all threads.
__device__ __forceinline__ double block_scan(double v, double* parts, double* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int step = 1; step < 64; step *= 2) {
    const double add = __shfl_up(v, step);
    if (lane >= step) v += add;
  }
  if (lane == 63) parts[wave] = v;
  __syncthreads();
  double before = 0., total = 0.;
  for (int w = 0; w < kRowWaves; ++w) {
    if (w == wave) before = total;
    total += parts[w];
  }
  __syncthreads();
  *all = total;
  return before + v;
}

// What a row's workgroup begins with: thread t's part and the row's largest logit.
struct RowStart {
  Part mine;
  float top;
  __device__ __forceinline__ RowStart(const SampleArgs& a, int64_t r, double* parts) {
    mine = static_cast<int>(threadIdx.x) < a.parts ? a.part[r * a.parts + threadIdx.x] : Part{-INFINITY, 0, 0.};
    top = wave_max(mine.top);
    if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = top;
    __syncthreads();
    for (int w = 0; w < kRowWaves; ++w) top = fmaxf(top, static_cast<float>(parts[w]));
    __syncthreads();
  }
};

__device__ __forceinline__ void write(const SampleArgs& a, int64_t row, int token, double p) {
  a.tokens[row] = token;
  // sums of rounded weights may be a last bit below one of them
  if (a.logprobs) a.logprobs[row] = p > 0. ? static_cast<float>(log(fmin(p, 1.))) : -INFINITY;
}

// The first of `n` threads' tokens (thread t's is first + t) that goes beyond
// `goal`, `before` being what the tokens before them weigh; without one, by
// rounding at the end, the last that weighs anything.
__device__ __forceinline__ void draw_from(const SampleArgs& a, int64_t row, double v, int token, double goal, double before,
                                          double total, int* found, double* parts) {
  if (threadIdx.x == 0) found[0] = 0x7fffffff, found[1] = -1;
  double sum;
  const double upto = before + block_scan(v, parts, &sum);
  if (v > 0. && upto > goal) atomicMin(&found[0], token);
  if (v > 0.) atomicMax(&found[1], token);
  __syncthreads();
  if (v > 0. && token == (found[0] == 0x7fffffff ? found[1] : found[0])) write(a, row, token, v / total);
}

// Draws from the tokens of a part that keeps(logit, token) holds for; *chosen: what
// the parts before it weigh.
template <typename T, typename KEEPS>
__device__ __forceinline__ void draw_part(const SampleArgs& a, int64_t row, int part, double goal, double total,
                                          const Weights& w, const KEEPS& keeps, int (&found)[2], double* parts,
                                          double* chosen) {
  // some tokens per thread, then one of them; part < 0 (nothing weighs anything) cannot be
  part = max(part, 0);
  constexpr int OWN = kPart / kRowThreads;
  float x[OWN];
  double v[OWN], sum = 0.;
  const int first = part * kPart + OWN * static_cast<int>(threadIdx.x);
#pragma unroll
  for (int e = 0; e < OWN; ++e)
    x[e] = fmaxf(load_elem<T>(a.logits, row * a.stride + min(first + e, a.vocab - 1)), -INFINITY);
#pragma unroll
  for (int e = 0; e < OWN; ++e) sum += v[e] = first + e < a.vocab && keeps(x[e], first + e) ? w.exact(x[e]) : 0.;
  __syncthreads();
  double before = *chosen, all;
  if (threadIdx.x == 0) found[0] = 0x7fffffff, found[1] = -1;
  before += block_scan(sum, parts, &all) - sum;
  int token = -1, last = -1;
  double of_token = 0., of_last = 0.;
#pragma unroll
  for (int e = 0; e < OWN; ++e) {
    before += v[e];
    if (v[e] > 0.) {
      last = first + e;
      of_last = v[e];
      if (before > goal && token < 0) {
        token = first + e;
        of_token = v[e];
      }
    }
  }
  if (token >= 0) atomicMin(&found[0], token);
  if (last >= 0) atomicMax(&found[1], last);
  __syncthreads();
  const bool end = found[0] == 0x7fffffff;  // by rounding: the last that weighs anything
  if (end ? last >= 0 && last == found[1] : token >= 0 && token == found[0])
    write(a, row, end ? last : token, (end ? of_last : of_token) / total);
}

// Rows without filters, and greedy ones: true if this was one.
template <typename T>
__device__ __forceinline__ bool draw_plain(const SampleArgs& a, const Settings& s, const RowStart& start, const Weights& w,
                                           int64_t r, int64_t row, double u, int (&found)[2], double* parts,
                                           double* chosen, double* total) {
  const int blocks = (a.vocab + kBlock - 1) / kBlock;
  const float* block_top = a.block_top + r * a.parts * kPartBlocks;
  if (!(start.top > -INFINITY)) {
    if (threadIdx.x == 0) write(a, row, -1, 0.);
    return true;
  }
  if (threadIdx.x == 0) found[0] = 0x7fffffff, found[1] = -1;
  if (s.greedy) {  // the first token of the first block that has the largest logit
    __syncthreads();
    for (int b = threadIdx.x; b < blocks; b += kRowThreads)
      if (block_top[b] == start.top) atomicMin(&found[0], b);
    __syncthreads();
    const int i = found[0] * kBlock + threadIdx.x;
    __syncthreads();
    const bool hit = threadIdx.x < kBlock && i < a.vocab && load_elem<T>(a.logits, row * a.stride + i) == start.top;
    draw_from(a, row, hit ? 1. : 0., i, 0., 0., 1., found, parts);
    return true;
  }
  // weights of the parts relative to the row's largest logit
  const double weight = start.mine.sum > 0. ? start.mine.sum * w.exact(start.mine.top) : 0.;
  const double upto = block_scan(weight, parts, total);
  if (s.filters()) return false;
  const double goal = u * *total;
  if (weight > 0.) {
    if (upto > goal) atomicMin(&found[0], static_cast<int>(threadIdx.x));
    atomicMax(&found[1], static_cast<int>(threadIdx.x));
  }
  __syncthreads();
  const int at = found[0] == 0x7fffffff ? found[1] : found[0];
  if (static_cast<int>(threadIdx.x) == at) *chosen = upto - weight;
  draw_part<T>(a, row, at, goal, *total, w, [](float, int) { return true; }, found, parts, chosen);
  return true;
}

template <typename T> __global__ __launch_bounds__(kRowThreads) void sample_plain(SampleArgs a) {
  __shared__ double parts[kRowWaves + 1], chosen;
  __shared__ int found[2];
  const int64_t r = blockIdx.x, row = a.row0 + r;
  const Settings s(a, row);
  const double u = static_cast<double>(fminf(fmaxf(a.uniform[row], 0.f), 0.99999994f));
  const RowStart start(a, r, parts);
  const Weights w(s, start.top);
  double total;
  draw_plain<T>(a, s, start, w, r, row, u, found, parts, &chosen, &total);
}

// Kept are logits above `edge`, and of those equal to it the tokens up to `last`.
struct Kept {
  uint32_t edge;  // key
  int last;
  __device__ __forceinline__ bool has(float x, int i) const {
    const uint32_t k = key_of(x);
    return x > -INFINITY && (k > edge || (k == edge && i <= last));
  }
};

template <typename T, bool PACKETS> struct RowWork {
  const SampleArgs& a;
  RowShared& l;
  const Settings& s;
  const Weights& w;
  int64_t row;
  const float* block_top;
  int blocks, q_top;

  // f(blocks, how many), a wave per block, for the blocks of whose largest logit
  // wanted(it) holds, in groups of which the next is on its way (without branches
  // between a group's loads, so that each waits for its own).
  template <int GROUP, typename WANTED, typename F>
  __device__ __forceinline__ void each_group(const WANTED& wanted, const F& f) const {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int b0 = wave; b0 < blocks; b0 += 64 * kRowWaves) {
      const int mine = b0 + kRowWaves * lane;
      const float top = mine < blocks ? block_top[mine] : -INFINITY;
      uint64_t todo = __builtin_amdgcn_ballot_w64(top > -INFINITY && wanted(top));
      Block<T, PACKETS> b[GROUP], next[GROUP];
      const auto load = [&](Block<T, PACKETS> (&to)[GROUP]) {
        int number = 0, n = 0;
#pragma unroll
        for (int i = 0; i < GROUP; ++i) {  // the last one again where there are fewer
          number = todo ? b0 + kRowWaves * __builtin_ctzll(todo) : number;
          n += todo ? 1 : 0;
          todo &= todo - 1;
          to[i].load(a, row, number);
        }
        return n;
      };
      if (!todo) continue;
      int n = load(b);
#pragma unroll 1
      for (;;) {
        int more = 0;
        if (todo) more = load(next);
        f(b, n);
        if (!more) break;
        n = more;
#pragma unroll
        for (int i = 0; i < GROUP; ++i) b[i] = next[i];
      }
    }
  }
  // f(block, its logits, its number), one by one.
  template <typename WANTED, typename F>
  __device__ __forceinline__ void each_block(const WANTED& wanted, const F& f) const {
    each_group<1>(wanted, [&](const auto& b, int) {
      float x[8];
      b[0].take(a, x);
      f(b[0], x, b[0].first / kBlock);
    });
  }

  // The least logit of bin q or a higher one: its neighbours are looked at by 64
  // lanes.  False where it is not near q's quotient (bins at the ends of all).
  __device__ __forceinline__ bool least_of(int q, float* x) const {
    const float about = static_cast<float>(static_cast<double>(q) / (4. * s.c));
    if (!(fabsf(about) < 1e37f)) return false;
    const int lane = threadIdx.x & 63;
    const float mine = value_of(key_of(about) + static_cast<uint32_t>(lane - 32));
    const uint64_t from = __builtin_amdgcn_ballot_w64(s.bin(mine) >= q);
    if (from == 0 || (from & 1)) return false;
    *x = __shfl(mine, __builtin_ctzll(from));
    return true;
  }

  // Lists the tokens of the row's bins [low, high]; false if there are too many.
  __device__ __forceinline__ bool look(int low, int high) {
    const int q_low = q_top - high, q_high = q_top - low;
    const bool open = low == 0;
    float from, to = INFINITY;  // as logits
    if (!least_of(q_low, &from)) return false;
    if (!open) {
      if (!least_of(q_high + 1, &to)) return false;
      if (threadIdx.x == 0) l.above = to;
    }
    if (threadIdx.x == 0) l.count = 0;
    __syncthreads();
    const int lane = threadIdx.x & 63;
    constexpr int GROUP = PACKETS && sizeof(typename T::bits) == 2 ? 6 : 4;  // and the next: more take registers that are not there
    each_group<GROUP>([&](float top) { return top >= from; }, [&](const auto& b, int n) {
      uint64_t in = 0;  // bit 8 i + e: block i's element e
#pragma unroll
      for (int i = 0; i < GROUP; ++i) {
        float x[8];
        b[i].take(a, x);
        uint32_t of = 0;
#pragma unroll
        for (int e = 7; e >= 0; --e) of = 2 * of + ((x[e] >= from) & ((x[e] < to) | open) ? 1 : 0);
        in |= static_cast<uint64_t>(i < n ? of : 0) << 8 * i;
      }
      if (!__builtin_amdgcn_ballot_w64(in != 0)) return;
      const int own = __popcll(in), upto = wave_scan(own);
      int at = 0;
      if (lane == 63) at = atomicAdd(&l.count, upto);
      at = __builtin_amdgcn_readlane(at, 63) + upto - own;
      // few lanes have more than one or two: their numbers, and the logits afterwards
      while (in) {
        const int e = __builtin_ctzll(in);
        int first = b[0].first;
#pragma unroll
        for (int i = 1; i < GROUP; ++i) first = e >> 3 == i ? b[i].first : first;
        if (at < kListed) l.list[at] = static_cast<uint32_t>(first + b[0].place(e & 7));
        ++at;
        in &= in - 1;
      }
    });
    __syncthreads();
    const int count = l.count;
    if (count > kListed) return false;
    constexpr int OWN = 8;  // on their way at once
#pragma unroll 1
    for (int i0 = threadIdx.x; i0 < count; i0 += OWN * kRowThreads) {
      uint32_t token[OWN];
      float x[OWN];
#pragma unroll
      for (int e = 0; e < OWN; ++e) token[e] = static_cast<uint32_t>(l.list[min(i0 + e * kRowThreads, count - 1)]);
#pragma unroll
      for (int e = 0; e < OWN; ++e) x[e] = load_elem<T>(a.logits, row * a.stride + token[e]);
#pragma unroll
      for (int e = 0; e < OWN; ++e)
        if (i0 + e * kRowThreads < count) l.list[i0 + e * kRowThreads] = static_cast<uint64_t>(~key_of(x[e])) << 32 | token[e];
    }
    __syncthreads();
    return true;
  }
  // to one of l.radix
  __device__ __forceinline__ void add(int at, double v) const {
    const Fixed f(v);
    atomicAdd(&l.radix[at], f.high);
    atomicAdd(&l.radix_low[at], f.low);
  }
  __device__ __forceinline__ float logit(uint64_t entry) const { return value_of(~static_cast<uint32_t>(entry >> 32)); }
  // The `count` entries at l.picked in order, at l.sorted: each one's place is how
  // many are before it, which the threads of an entry count a share each of.
  __device__ __forceinline__ void sort_picked(int count) {
    constexpr int SHARES = kRowThreads / kPicked;
    const int e = threadIdx.x % kPicked, share = threadIdx.x / kPicked;
    if (share == 0) {
      l.place[e] = 0;
      if (e >= count) l.picked[e] = ~uint64_t{0};
    }
    __syncthreads();
    const uint64_t mine = l.picked[e];
    int before = 0;
    constexpr int AT_ONCE = 4;  // pairs
#pragma unroll 1
    for (int i0 = 2 * share; i0 < count; i0 += 2 * SHARES * AT_ONCE) {
      ulonglong2 other[AT_ONCE];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i)
        other[i] = *reinterpret_cast<const ulonglong2*>(&l.picked[(i0 + 2 * SHARES * i) % kPicked]);
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const int more = (other[i].x < mine ? 1 : 0) + (other[i].y < mine ? 1 : 0);
        before += i0 + 2 * SHARES * i < kPicked ? more : 0;
      }
    }
    atomicAdd(&l.place[e], before);
    __syncthreads();
    if (share == 0 && e < count) l.sorted[l.place[e]] = mine;
    __syncthreads();
  }

  // The first of 256 at which the sum up to it reaches `want`; the last without one.
  // *upto: the sum before it.
  __device__ __forceinline__ int reaches(double want, const double* sums, double* upto) {
    const int lane = threadIdx.x & 63;
    if (threadIdx.x < 64) {
      double own[4], sum = 0.;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sum += own[i] = sums[4 * lane + i];
      double at = -sum;
      for (int step = 1; step < 64; step *= 2) {
        const double add = __shfl_up(sum, step);
        if (lane >= step) sum += add;
      }
      at += sum;
      const uint64_t past = __builtin_amdgcn_ballot_w64(sum >= want);
      if (lane == (past ? __builtin_ctzll(past) : 63)) {
        int bin = 4 * lane;
#pragma unroll
        for (int i = 0; i < 3; ++i)
          if (bin == 4 * lane + i && at + own[i] < want) {
            at += own[i];
            ++bin;
          }
        l.found = past ? bin : kBins - 1;
        l.chosen = at;
      }
    }
    __syncthreads();
    const int bin = l.found;
    *upto = l.chosen;
    __syncthreads();
    return bin;
  }
  __device__ __forceinline__ double weight_before(int bin) {  // of the bins
    const int lane = threadIdx.x & 63;
    double sum = 0.;
    for (int i = lane; i < bin; i += 64) sum += l.bin_weight[i];
    return wave_sum(sum);
  }

  enum Rule { COUNT, WEIGHT, LEAST };
  // The last ranked token that a rule keeps, and the kept weight up to it: the rank
  // below `want`; less than `want` before it; a weight of `want`.  bins: the first and
  // last bin that the list holds, its own among them.  False if that
  // does not say it.
  __device__ __forceinline__ bool threshold(Rule rule, double want, Kept* kept, double* weight, int (&bins)[2]) {
    double ahead = 0.;
    int low, high;
    if (rule == LEAST) {  // its logit in 32 bits may be in a bin next to its own
      const int q = s.bin(static_cast<float>(w.top + log2(want) / s.c));
      low = max(0, q_top - q - 1);
      high = q_top - q + 1;
    } else {
      low = high = reaches(want, rule == COUNT ? l.bin_ranks : l.bin_weight, &ahead);
      // few: all up to it, among which the other rules find theirs
      if (rule == COUNT && ahead + l.bin_ranks[high] <= kPicked) {
        low = 0;
        ahead = 0.;
      }
    }
    if (high < 0 || high >= kBins - 1) return false;
    if (low < bins[0] || high > bins[1]) {
      bins[0] = low;
      bins[1] = high;
      if (!look(low, high)) {
        bins[0] = kBins;
        return false;
      }
    }
    low = bins[0];
    const int count = l.count;
    double above = weight_before(low);
    if (rule == LEAST) {  // how many of them is what is wanted
      if (threadIdx.x == 0) l.found = 0;
      __syncthreads();
      int some = 0;
#pragma unroll 1
      for (int i = threadIdx.x; i < count; i += kRowThreads) some += w.exact(logit(l.list[i])) >= want ? 1 : 0;
      some = __builtin_amdgcn_readlane(wave_scan(some), 63);
      if ((threadIdx.x & 63) == 0) atomicAdd(&l.found, some);
      __syncthreads();
      some = l.found;
      __syncthreads();
      if (some == 0) {  // all that are above them
        *weight = above;
        *kept = Kept{key_of(l.above), 0x7fffffff};
        if (low == 0) return false;  // not: the largest weighs 1
        return true;
      }
      want = some;
      ahead = 0.;
    }
    // the 256th of the entries' range that it is in, again and again
    unsigned long long from = 0, to = ~0ull;
    int picked = count;
#pragma unroll 1
    while (picked > kPicked) {
      if (threadIdx.x < kBins) {
        l.radix[threadIdx.x] = l.radix_low[threadIdx.x] = 0;
        l.step_count[threadIdx.x] = 0;
      }
      if (threadIdx.x == 0) {
        l.low = ~0ull;
        l.high = 0;
      }
      __syncthreads();
      unsigned long long least = ~0ull, most = 0;
#pragma unroll 1
      for (int i = threadIdx.x; i < count; i += kRowThreads) {
        const unsigned long long e = l.list[i];
        if (e < from || e > to) continue;
        least = min(least, e);
        most = max(most, e);
      }
      for (int m = 32; m; m >>= 1) {
        least = min(least, __shfl_xor(least, m));
        most = max(most, __shfl_xor(most, m));
      }
      if ((threadIdx.x & 63) == 0) {
        atomicMin(&l.low, least);
        atomicMax(&l.high, most);
      }
      __syncthreads();
      from = l.low;
      to = l.high;
      const int shift = max(0, 56 - __builtin_clzll(to - from));
#pragma unroll 1
      for (int i = threadIdx.x; i < count; i += kRowThreads) {
        const unsigned long long e = l.list[i];
        if (e < from || e > to) continue;
        const int step = static_cast<int>((e - from) >> shift);
        add(step, w.exact(logit(e)));
        atomicAdd(&l.step_count[step], 1u);
      }
      __syncthreads();
      if (threadIdx.x < kBins) {
        l.steps[threadIdx.x] = Fixed::value(l.radix[threadIdx.x], l.radix_low[threadIdx.x]);
        l.ranks[threadIdx.x] = l.step_count[threadIdx.x];
      }
      __syncthreads();
      double before;
      const int step = reaches(rule == WEIGHT ? want - above : want - ahead, rule == WEIGHT ? l.steps : l.ranks, &before);
      if (l.step_count[step] == 0) return false;
      double ranks = 0., weights = 0.;  // of the steps before it
      for (int i = threadIdx.x & 63; i < step; i += 64) {
        ranks += l.ranks[i];
        weights += l.steps[i];
      }
      ahead += wave_sum(ranks);
      above += wave_sum(weights);
      picked = static_cast<int>(l.step_count[step]);
      from += static_cast<unsigned long long>(step) << shift;
      to = min(to, from + ((1ull << shift) - 1));
      __syncthreads();
    }
    if (threadIdx.x == 0) l.picked_count = 0;
    __syncthreads();
#pragma unroll 1
    for (int i = threadIdx.x; i < count; i += kRowThreads) {
      const unsigned long long e = l.list[i];
      if (e >= from && e <= to) l.picked[atomicAdd(&l.picked_count, 1)] = e;
    }
    __syncthreads();
    sort_picked(picked);
    if (threadIdx.x == 0) l.found = -1;
    __syncthreads();
    {
      const int i = threadIdx.x;
      const double v = i < picked ? w.exact(logit(l.sorted[i])) : 0.;
      double all;
      const double upto = above + block_scan(v, l.parts, &all);
      bool is = false;  // the last that is kept
      if (i < picked) {
        is = rule == WEIGHT ? upto - v < want && (upto >= want || i == picked - 1) : ahead + i + 1 == want;
      }
      if (is) {
        l.found = i;
        l.chosen = upto;
        l.upto = l.sorted[i];
      }
      __syncthreads();
    }
    if (l.found < 0) return false;
    *weight = l.chosen;
    *kept = Kept{~static_cast<uint32_t>(l.upto >> 32), static_cast<int>(l.upto)};
    __syncthreads();
    return true;
  }

  // As threshold, digit by digit over all tokens that are kept so far.
  __device__ __forceinline__ Kept by_digits(double need, bool by_count, const Kept& within) {
    uint32_t prefix = 0, mask = 0;
    double before = 0.;
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (threadIdx.x < 256) l.radix[threadIdx.x] = l.radix_low[threadIdx.x] = 0;
      __syncthreads();
      each_block([&](float top) { return key_of(top) >= max(within.edge, prefix); }, [&](const auto& b, const float (&x)[8], int) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t k = key_of(x[e]);
          if (!within.has(x[e], b.index(e)) || (k & mask) != prefix) continue;
          if (by_count) atomicAdd(&l.radix[k >> shift & 255], 1ull);
          else add(k >> shift & 255, w.exact(x[e]));
        }
      });
      __syncthreads();
      if (threadIdx.x == 0) {
        double sum = before, ahead = before;  // ahead: of the digits above the lowest so far
        int lowest = 0;
#pragma unroll 1
        for (int i = 255; i >= 0; --i) {
          if (l.radix[i] == 0 && l.radix_low[i] == 0) continue;
          lowest = i;
          ahead = sum;
          sum += by_count ? static_cast<double>(l.radix[i]) : Fixed::value(l.radix[i], l.radix_low[i]);
          if (sum >= need) break;  // without one, the last
        }
        l.digit = lowest;
        l.chosen = ahead;
      }
      __syncthreads();
      prefix |= l.digit << shift;
      mask |= 255u << shift;
      before = l.chosen;
      __syncthreads();
    }
    // of the tokens equal to it, in order, as many as are needed
    const double each = by_count ? 1. : w.exact(value_of(prefix));
    const double left = need - before;
    const int ties = each > 0. ? max(1, static_cast<int>(fmin(ceil(left / each), 1e9))) : 1;
    if (threadIdx.x == 0) l.last = -1;
    __syncthreads();
    if (threadIdx.x < 64) {
      int seen = 0;
#pragma unroll 1
      for (int i0 = 0; i0 < a.vocab && seen < ties; i0 += 64) {
        const int i = i0 + threadIdx.x;
        const float x = i < a.vocab ? load_elem<T>(a.logits, row * a.stride + i) : -INFINITY;
        const bool tie = x > -INFINITY && key_of(x) == prefix && within.has(x, i);
        const uint64_t all = __builtin_amdgcn_ballot_w64(tie);
        const int rank = seen + __popcll(all & ((uint64_t{1} << threadIdx.x) - 1));
        if (tie && rank < ties) atomicMax(&l.last, i);
        seen += __popcll(all);
      }
    }
    __syncthreads();
    return Kept{prefix, l.last};
  }

  // Weights of the blocks' kept tokens, in l.weight; their sum.
  __device__ __forceinline__ double weigh(const Kept& kept, double least) {
    for (int b = threadIdx.x; b < 2048; b += kRowThreads) l.weight[b] = 0.;
    __syncthreads();
    each_block([&](float top) { return key_of(top) >= kept.edge; }, [&](const auto& b, const float (&x)[8], int number) {
      double sum = 0.;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (!kept.has(x[e], b.index(e))) continue;
        const double v = w.exact(x[e]);
        if (v >= least) sum += v;
      }
      sum = wave_sum(sum);
      if ((threadIdx.x & 63) == 0) l.weight[number] = sum;
    });
    __syncthreads();
    double all, sum = 0.;
    constexpr int OWN = 2048 / kRowThreads;
    const int first = OWN * threadIdx.x;
#pragma unroll 1
    for (int e = 0; e < OWN; ++e) sum += l.weight[first + e];
    double upto = block_scan(sum, l.parts, &all) - sum;
#pragma unroll 1
    for (int e = 0; e < OWN; ++e) l.weight[first + e] = upto += l.weight[first + e];  // up to a block, and it
    __syncthreads();
    return all;
  }
};

template <typename T, bool PACKETS> __global__ __launch_bounds__(kRowThreads) void sample_rows(SampleArgs a) {
  __shared__ RowShared l;
  __shared__ int found[2];
  const int64_t r = blockIdx.x, row = a.row0 + r;
  const Settings s(a, row);
  const double u = static_cast<double>(fminf(fmaxf(a.uniform[row], 0.f), 0.99999994f));
  const RowStart start(a, r, l.parts);
  const Weights w(s, start.top);
  double total;
  if (draw_plain<T>(a, s, start, w, r, row, u, found, l.parts, &l.chosen, &total)) return;
  const int blocks = (a.vocab + kBlock - 1) / kBlock;
  RowWork<T, PACKETS> work{a, l, s, w, row, a.block_top + r * a.parts * kPartBlocks, blocks, s.bin(start.top)};

  if (start.mine.sum > 0.) {
    l.part_unit[threadIdx.x] = w.exact(start.mine.top) / kBinUnit;
    // beyond all bins where the part has nothing in them
    l.part_shift[threadIdx.x] = shift_of_part(work.q_top, start.mine.q);
  } else if (static_cast<int>(threadIdx.x) < a.parts) {
    l.part_unit[threadIdx.x] = 0.;
    l.part_shift[threadIdx.x] = kBins;
  }
  __syncthreads();
  const uint64_t* bins = a.bins + r * a.parts * kBins;
  const uint32_t* counts = a.counts + r * a.parts * kBins;
  {
    // the row's bins, by two groups of threads; the last is nobody's
    const int g = threadIdx.x & (kBins - 1), group = threadIdx.x / kBins;
    constexpr int AT_ONCE = 8;
    uint32_t count = 0;
    double weight = 0.;
    for (int p0 = group; p0 < a.parts; p0 += AT_ONCE * (kRowThreads / kBins)) {
      uint64_t v[AT_ONCE];
      uint32_t n[AT_ONCE];
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) {  // all on their way at once, without branches
        const int p = min(p0 + e * (kRowThreads / kBins), a.parts - 1);
        v[e] = bins[p * kBins + max(g - l.part_shift[p], 0)];
      }
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) {
        const int p = min(p0 + e * (kRowThreads / kBins), a.parts - 1);
        n[e] = s.by_count ? counts[p * kBins + max(g - l.part_shift[p], 0)] : 0;
      }
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) {
        const int p = p0 + e * (kRowThreads / kBins), last = min(p, a.parts - 1);
        const bool in = p < a.parts && g >= l.part_shift[last] && g != kBins - 1;
        count += in ? n[e] : 0;
        weight += in ? static_cast<double>(v[e]) * l.part_unit[last] : 0.;
      }
    }
    l.weight[threadIdx.x] = weight;
    l.weight[kRowThreads + threadIdx.x] = count;
    __syncthreads();
    static_assert(kRowThreads == 2 * kBins, "groups of threads");
    if (threadIdx.x < kBins) {
      l.bin_weight[g] = weight + l.weight[g + kBins];
      l.bin_ranks[g] = count + l.weight[kRowThreads + g + kBins];
    }
    __syncthreads();
  }
  const double least = s.by_least ? static_cast<double>(s.min_p) : 0.;
  Kept kept{0, 0x7fffffff};
  int at_bin[2] = {-1, -1};  // of `kept`: the list's bins when it was found
  int listed[2] = {kBins, -1};
  double base = total;
  bool known = true;  // that is what is kept
  typedef RowWork<T, PACKETS> Work;
#pragma unroll 1
  for (int i = 0; i < 3; ++i) {
    const typename Work::Rule rule = i == 0 ? Work::COUNT : i == 1 ? Work::WEIGHT : Work::LEAST;
    if (!(i == 0 ? s.by_count : i == 1 ? s.by_weight : s.by_least)) continue;
    const double want = i == 0 ? static_cast<double>(s.top_k) : i == 1 ? static_cast<double>(s.top_p) * base : least;
    Kept k;
    double weight;
    if (known && work.threshold(rule, want, &k, &weight, listed)) {
      if (k.edge > kept.edge || (k.edge == kept.edge && k.last < kept.last)) {
        kept = k;
        base = weight;
        at_bin[0] = listed[0];
        at_bin[1] = listed[1];
      }
    } else if (i < 2) {
      known = false;
      kept = work.by_digits(want, i == 0, kept);
      if (i == 0 && s.by_weight) base = work.weigh(kept, 0.);
    } else {
      known = false;
    }
    __syncthreads();
  }
  if (known) {
    if (listed[0] != at_bin[0] || listed[1] != at_bin[1]) work.look(at_bin[0], at_bin[1]);  // it held them
    // what is kept of each part: its bins above the list's, and of the list
    if (threadIdx.x < 256) l.radix[threadIdx.x] = l.radix_low[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < l.count; i += kRowThreads) {
      const int token = static_cast<int>(l.list[i]);
      const uint32_t key = ~static_cast<uint32_t>(l.list[i] >> 32);
      if (key > kept.edge || (key == kept.edge && token <= kept.last))
        work.add(token / kPart, w.exact(work.logit(l.list[i])));
    }
    constexpr int AT_ONCE = 4;
#pragma unroll 1
    for (int p0 = threadIdx.x >> 6; p0 < a.parts; p0 += AT_ONCE * kRowWaves) {
      unsigned long long sum[AT_ONCE] = {};  // exactly
      const int lane = threadIdx.x & 63;
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) {
        const int p = min(p0 + e * kRowWaves, a.parts - 1), end = at_bin[0] - l.part_shift[p];
#pragma unroll
        for (int i = 0; i < kBins; i += 64) {
          const uint64_t v = bins[p * kBins + i + lane];
          sum[e] += i + lane < end ? v : 0;
        }
      }
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) {
        const int p = p0 + e * kRowWaves;
        for (int m = 32; m; m >>= 1) sum[e] += __shfl_xor(sum[e], m);
        if (lane == 0 && p < a.parts) l.weight[p] = static_cast<double>(sum[e]) * l.part_unit[p];
      }
    }
    __syncthreads();
    const double v = static_cast<int>(threadIdx.x) < a.parts
                         ? l.weight[threadIdx.x] + Fixed::value(l.radix[threadIdx.x], l.radix_low[threadIdx.x]) : 0.;
    double all;
    const double upto = block_scan(v, l.parts, &all), goal = u * all;
    if (threadIdx.x == 0) found[0] = 0x7fffffff, found[1] = -1;
    __syncthreads();
    if (v > 0.) {
      if (upto > goal) atomicMin(&found[0], static_cast<int>(threadIdx.x));
      atomicMax(&found[1], static_cast<int>(threadIdx.x));
    }
    __syncthreads();
    const int at = found[0] == 0x7fffffff ? found[1] : found[0];
    if (static_cast<int>(threadIdx.x) == at) l.chosen = upto - v;
    draw_part<T>(a, row, at, goal, all, w, [&](float x, int i) { return kept.has(x, i); }, found, l.parts, &l.chosen);
    return;
  }

  // Too many tokens in one bin (equal ones, or weights that hardly differ): the
  // kept weights block by block
  const double all = work.weigh(kept, least), goal = u * all;
  // the first block beyond the goal; without one, by rounding, the last that weighs anything
  if (threadIdx.x == 0) found[0] = 0x7fffffff, found[1] = -1;
  __syncthreads();
  for (int b = threadIdx.x; b < blocks; b += kRowThreads) {
    const double upto = l.weight[b], before = b ? l.weight[b - 1] : 0.;
    if (upto > before) {
      if (upto > goal) atomicMin(&found[0], b);
      atomicMax(&found[1], b);
    }
  }
  __syncthreads();
  const int block = found[0] == 0x7fffffff ? found[1] : found[0];
  const int i = block * kBlock + threadIdx.x;  // a thread per token
  double v = 0.;
  if (threadIdx.x < kBlock && i < a.vocab) {
    const float x = fmaxf(load_elem<T>(a.logits, row * a.stride + i), -INFINITY);
    if (kept.has(x, i)) {
      v = w.exact(x);
      if (v < least) v = 0.;
    }
  }
  __syncthreads();
  draw_from(a, row, v, i, goal, block ? l.weight[block - 1] : 0., all, found, l.parts);
}

int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
int64_t part_count(int64_t vocab) { return (vocab + kPart - 1) / kPart; }
int64_t chunk_rows(int64_t rows, int64_t vocab) {
  const int64_t most = kChunkParts / part_count(vocab);
  return rows < most ? rows : most;
}

}  // namespace

int64_t sample_workspace(int64_t rows, int64_t vocab) {
  const int64_t n = chunk_rows(rows, vocab) * part_count(vocab);
  return up16(n * sizeof(Part)) + up16(n * kPartBlocks * 4) + n * kBins * 12;
}

int sample_launch(const void* logits, const float* uniform, int64_t* tokens, float* logprobs, const float* temperature,
                  const int32_t* top_k, const float* top_p, const float* min_p, float temperature_all, int32_t top_k_all,
                  float top_p_all, float min_p_all, int64_t rows, int vocab, int64_t stride, int dtype, void* work,
                  hipStream_t stream) {
  SampleArgs a{logits, uniform, tokens, logprobs, temperature, top_k, top_p, min_p, temperature_all, top_k_all,
               top_p_all, min_p_all, 0, 0, stride, vocab, static_cast<int>(part_count(vocab)), nullptr, nullptr,
               nullptr, nullptr};
  const int64_t es = dtype == MI355_F32 ? 4 : 2;
  const bool packets = aligned16(logits) && vocab * es % 16 == 0 && (rows == 1 || stride * es % 16 == 0);
  const int64_t chunk = chunk_rows(rows, vocab), n = chunk * a.parts;
  uint8_t* at = static_cast<uint8_t*>(work);
  a.part = reinterpret_cast<Part*>(at);
  at += up16(n * sizeof(Part));
  a.block_top = reinterpret_cast<float*>(at);
  at += up16(n * kPartBlocks * 4);
  a.bins = reinterpret_cast<uint64_t*>(at);
  a.counts = reinterpret_cast<uint32_t*>(at + n * kBins * 8);
  static const char* what = "sample_tokens launch";
  // known here: no row has filters
  const bool plain = top_k == nullptr && top_p == nullptr && min_p == nullptr && temperature == nullptr &&
                     (!(temperature_all > 0.f) ||
                      ((top_k_all <= 0 || top_k_all >= vocab) && !(top_p_all < 1.f) && !(min_p_all > 0.f)));
  const auto run = [&](auto* parts, auto* draw) {
    const int st = launch(parts, dim3(static_cast<unsigned>(a.rows * a.parts)), kPartThreads, 0, a, stream, what);
    return st != MI355_OK ? st : launch(draw, dim3(static_cast<unsigned>(a.rows)), kRowThreads, 0, a, stream, what);
  };
  for (a.row0 = 0; a.row0 < rows; a.row0 += chunk) {
    a.rows = rows - a.row0 < chunk ? rows - a.row0 : chunk;
    int st;
    const auto typed = [&](auto t) {
      typedef decltype(t) T;
      if (packets) return run(sample_parts<T, true>, plain ? sample_plain<T> : sample_rows<T, true>);
      return run(sample_parts<T, false>, plain ? sample_plain<T> : sample_rows<T, false>);
    };
    if (dtype == MI355_F32) st = typed(F32{});
    else if (dtype == MI355_F16) st = typed(F16{});
    else st = typed(BF16{});
    if (st != MI355_OK) return st;
  }
  return MI355_OK;
}

}  // namespace mi355
