// Attention of a batch whose sequences share prefixes, over a paged cache, for
// gfx950: tree attention in which the slots below a sequence's shared length are
// those of its group's first sequence.
#include "shared_prefix_kernels.h"

namespace mi355 {

int shared_prefix_run_bf16(const SharedArgs& a, const SharedPlan& p, int format, hipStream_t s);

namespace {

struct RowsArgs {
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

// A wave per query row, for callers without a workspace: right for every case, and
// 25 to 200 times slower (4 sequences under 700 slots 395 us, 128 under 32768 30 ms).
template <typename T, int FMT> __global__ __launch_bounds__(64) void shared_prefix_rows(RowsArgs a) {
  typedef typename T::bits bits;
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int hq = static_cast<int>(row % a.q_heads), t = static_cast<int>(row / a.q_heads % a.tokens);
  const int b = static_cast<int>(row / a.q_heads / a.tokens), h = hq / a.group, d = a.c.d;
  const int cap = a.c.capacity();
  const int len = max(0, min(a.lens[b], cap)), fresh = max(0, min(a.new_lens ? a.new_lens[b] : a.tokens, a.tokens));
  const int end = min(len + fresh, cap);
  int first = b, shared = 0;
  if (a.groups) {
    int g0 = 0, g1 = 0;  // a boundary below an earlier one counts as that
    for (int g = 0; g < a.group_count; ++g) {
      g0 = max(g1, min(a.groups[g], a.batch));
      g1 = max(g0, min(a.groups[g + 1], a.batch));
      if (b >= g0 && b < g1) {
        first = g0;
        shared = max(0, min(a.prefix_lens[g], len));
        break;
      }
    }
  } else if (a.group_count) {
    const int even = a.batch / a.group_count;
    first = b / even * even;
    shared = max(0, min(a.prefix_lens[b / even], len));
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

// What groups given by their boundaries mean for each sequence: one workgroup, 5 us,
// so that no other has to look through the boundaries for its rows.
struct SetupArgs {
  const int32_t *lens, *prefix, *groups;
  int32_t *bounds, *shared;
  int batch, count, cap;
};
__global__ __launch_bounds__(1024) void shared_prefix_setup(SetupArgs a) {
  __shared__ int scan[1024];
  int most = 0;
  for (int i0 = 0; i0 <= a.count; i0 += 1024) {  // a boundary below an earlier one counts as that
    const int i = i0 + threadIdx.x;
    scan[threadIdx.x] = i <= a.count ? max(0, min(a.groups[i], a.batch)) : 0;
    __syncthreads();
    for (int step = 1; step < 1024; step *= 2) {
      const int other = static_cast<int>(threadIdx.x) >= step ? scan[threadIdx.x - step] : 0;
      __syncthreads();
      scan[threadIdx.x] = max(scan[threadIdx.x], other);
      __syncthreads();
    }
    if (i <= a.count) a.bounds[i] = max(most, scan[threadIdx.x]);
    most = max(most, scan[1023]);
    __syncthreads();
  }
  __threadfence_block();
  __syncthreads();
  const int32_t* bounds = a.count < 1024 ? scan : a.bounds;  // one pass: still in LDS
  for (int b = threadIdx.x; b < a.batch; b += 1024) {
    int lo = 0, hi = a.count + 1;  // the first boundary beyond b
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (bounds[mid] > b) hi = mid;
      else lo = mid + 1;
    }
    const int g = lo - 1;
    const bool in = g >= 0 && g < a.count;
    a.shared[b] = in ? max(0, min(a.prefix[g], min(a.lens[b], a.cap))) : 0;
  }
}

int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }

// False where the line of tiles could pass 2^31.
bool plan(const mi355_kv_cache& c, int64_t batch, int64_t tokens, int64_t q_heads, int64_t groups, int cus, SharedArgs* args,
          SharedPlan* to) {
  SharedPlan& p = *to;
  SharedArgs& a = *args;
  const int dp = c.head_dim <= 64 ? 64 : c.head_dim <= 128 ? 128 : 256;
  const int64_t rows = tokens * (q_heads / c.kv_heads);                         // of a sequence
  const int64_t group_rows = groups ? (batch + groups - 1) / groups * rows : rows;  // on average
  p.sm = rows <= 16 ? 1 : 2;
  p.grid = cus * shared_groups(dp);
  // Blocks of 128 rows, which read a tile half as often as those of 64, unless a
  // workgroup has few tiles: then the sums to write and join, 64 KB a piece, count.
  // 32 sequences under 8011 slots (2 of 128 a workgroup): 64 rows 28.8 + 6.2 us, 128
  // rows 30.0 + 7.4; 40 under 3003, drafts (9): 92.9 + 8.5, 66.8 + 10.3; 128 under
  // 32768 (28): 217 + 7.6, 148 + 9.5.
  const int64_t of_128 = groups * ((group_rows + 127) / 128) + (rows > 32 ? batch * ((rows + 127) / 128) : 0);
  const int64_t all_tiles = c.kv_heads * of_128 * (c.table_width * c.page_size / 64);
  p.mt = group_rows <= 16 * kWaves || dp == 256 || all_tiles < 4 * p.grid ? 1 : 2;
  a.few = 16 * p.sm;
  a.block_log = 0;
  while ((1 << a.block_log) < 16 * p.mt * kWaves) ++a.block_log;
  // What a tile and a piece cost, many tile, pad, few tile, pad, and the least
  // share, in us: 4 samples of 700 slots, 32 sequences of 8011 + 700, 40 of 3003 +
  // 500 with trees of 6, 128 of 32768 + 400:
  //   4 16 4 12 24   28.0  49.1  77.2  170.3      4  8 4  8 4   16.1  39.1  72.7  154.6
  //   4 16 4 12  4   16.1  39.2  73.8  160.8      4 24 2 10 4   16.9  38.3  75.2  147.1
  //   4 12 2  6  4   16.0  36.5  81.4  150.3      4  8 2  8 4   16.1  36.5  76.3  148.0
  a.many_cost = {4, 8};
  a.few_cost = {2, 8};
  a.least = 4;
  // pieces of all prefixes and of all sequences, and what one costs at most
  const int64_t blocks = (batch * rows >> a.block_log) + groups + batch * ((rows >> a.block_log) + 1);
  const int64_t tiles = c.table_width * c.page_size / (16 * kWaves) + 2;
  if (c.kv_heads * blocks > (int64_t{1} << 30) / (4 * tiles + 16)) return false;
  const int64_t all = batch * tokens * q_heads;
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t was = at;
    at += up16(bytes);
    return was;
  };
  const int64_t slots = 2 * int64_t{p.grid} << a.block_log;
  p.partial = take(slots * c.head_dim * 4);
  p.stats = take(slots * 8);
  p.whole = take(2 * all * c.head_dim * 4);
  p.whole_stats = take(2 * all * 8);
  p.pieces = take(2 * all * 8);
  p.bounds = take(4 * (groups + 1));
  p.shared = take(4 * batch);
  p.bytes = at;
  return true;
}

// n / u for n < 2^27 as n * mul >> shift: ceil(2^(31 + L) / u) with L = ceil(log2 u) fits 32 bits, and the product is
// off by less than 2^L in 2^(31 + L), too little to reach the next integer
void reciprocal(uint32_t u, uint32_t* mul, uint32_t* shift) {
  uint32_t log = 0;
  while ((uint64_t{1} << log) < u) ++log;
  *mul = static_cast<uint32_t>(((uint64_t{1} << (31 + log)) + u - 1) / u);
  *shift = 31 + log;
}

}  // namespace

int64_t shared_prefix_workspace(const mi355_kv_cache& cache, int64_t batch, int64_t tokens, int64_t q_heads,
                                int64_t group_count) {
  int cus = 0;
  SharedArgs a{};
  SharedPlan p;
  if (compute_units(&cus) != MI355_OK || !plan(cache, batch, tokens, q_heads, group_count, cus, &a, &p)) return 0;
  return p.bytes;
}

int shared_prefix_launch(const mi355_kv_cache& cache, const void* q, void* out, const int32_t* lens,
                         const int32_t* new_lens, const int32_t* prefix_lens, const int32_t* groups, int group_count,
                         const uint8_t* mask, int64_t mask_b, int64_t mask_t, int64_t batch, int tokens, int q_heads,
                         const int64_t* q_strides, float scale, int dtype, void* work, int64_t work_bytes,
                         hipStream_t stream) {
  int cus = 0;
  int st = compute_units(&cus);
  if (st != MI355_OK) return st;
  const int group = q_heads / static_cast<int>(cache.kv_heads);
  SharedArgs a{};
  SharedPlan p;
  if (!plan(cache, batch, tokens, q_heads, group_count, cus, &a, &p) || work == nullptr || work_bytes < p.bytes) {
    const RowsArgs r{kv_cache_args(cache), q, out, lens, new_lens, prefix_lens, groups, mask, mask_b, mask_t,
                     q_strides[0], q_strides[1], q_strides[2], static_cast<int>(batch), tokens, q_heads, group,
                     group_count, scale * kLog2e};
    const dim3 grid(static_cast<unsigned>(batch * tokens * q_heads));
    const auto run = [&](auto* kernel) { return launch(kernel, grid, 64, 0, r, stream, "shared_prefix_attention launch"); };
    if (dtype == MI355_F16)
      return cache.format == KV_INT8   ? run(shared_prefix_rows<F16, KV_INT8>)
             : cache.format == KV_E4M3 ? run(shared_prefix_rows<F16, KV_E4M3>)
                                       : run(shared_prefix_rows<F16, KV_16BIT>);
    return cache.format == KV_INT8   ? run(shared_prefix_rows<BF16, KV_INT8>)
           : cache.format == KV_E4M3 ? run(shared_prefix_rows<BF16, KV_E4M3>)
                                     : run(shared_prefix_rows<BF16, KV_16BIT>);
  }
  uint8_t* base = static_cast<uint8_t*>(work);
  a.t = TreeArgs{kv_cache_args(cache), q, out, lens, new_lens, mask, mask_b, mask_t, q_strides[0], q_strides[1],
                 q_strides[2], reinterpret_cast<float*>(base + p.partial), reinterpret_cast<float2*>(base + p.stats),
                 nullptr, static_cast<int>(batch), tokens, q_heads, group,
                 1 << a.block_log, 2, 0, 0, p.grid, 0, 0, scale * kLog2e};
  reciprocal(static_cast<uint32_t>(cache.page_size / 16), &a.t.page_mul, &a.t.page_shift);
  a.prefix = prefix_lens;
  a.whole = reinterpret_cast<float*>(base + p.whole);
  a.whole_stats = reinterpret_cast<float2*>(base + p.whole_stats);
  a.pieces = reinterpret_cast<int2*>(base + p.pieces);
  a.groups = group_count;
  a.even = group_count ? static_cast<int>(batch / group_count) : 0;
  a.rows = static_cast<int>(batch * tokens * q_heads);
  a.mt_rows = tokens * group;
  if (a.even) reciprocal(static_cast<uint32_t>(a.even), &a.even_mul, &a.even_shift);
  reciprocal(static_cast<uint32_t>(a.mt_rows), &a.seq_mul, &a.seq_shift);
  reciprocal(static_cast<uint32_t>(group), &a.group_mul, &a.group_shift);
  if (groups != nullptr && group_count > 0) {
    int32_t *bounds = reinterpret_cast<int32_t*>(base + p.bounds), *shared = reinterpret_cast<int32_t*>(base + p.shared);
    const SetupArgs setup{lens, prefix_lens, groups, bounds, shared, static_cast<int>(batch), group_count,
                          static_cast<int>(cache.table_width * cache.page_size)};
    st = launch(shared_prefix_setup, dim3(1), 1024, 0, setup, stream, "shared_prefix_attention setup launch");
    if (st != MI355_OK) return st;
    a.bounds = bounds;
    a.shared = shared;
  }
  return dtype == MI355_F16 ? shared_prefix_run<F16>(a, p, cache.format, stream)
                            : shared_prefix_run_bf16(a, p, cache.format, stream);
}

}  // namespace mi355
