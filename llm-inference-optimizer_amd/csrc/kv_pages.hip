// Page tables and slot maps from the lengths of requests, for gfx950.
//
// kv_reserve: entry (b, c) of the new table is the old one where sequence b needs
// column c and has a page there, else a free page, the k-th such entry (b first)
// taking the k-th page that nobody keeps.  Bound by launches: a table is read and
// written once, 8 bytes per entry.
#include "kv_cache.h"

namespace mi355 {
namespace {

constexpr int kBlock = 256, kBlockWaves = kBlock / 64;
constexpr int kSpan = 4096;  // pages whose free ones one workgroup lists

struct PagesArgs {
  KvCache c;
  const int32_t *lens, *new_lens;
  int32_t* out;
  int64_t out_stride;
  int32_t* missing;
  int batch, spans;
  uint8_t* used;          // [pages]: whether an entry keeps the page
  int32_t* lacks;         // [batch]: pages that a sequence lacks, within the table
  int32_t* group_lacks;   // [ceil(batch / kBlockWaves)]
  int32_t* span_free;     // [spans]
  int32_t* listed;        // [spans * kSpan]: the free pages of a span, in order
};

__device__ __forceinline__ int64_t slots_of(const PagesArgs& a, int b) {
  return static_cast<int64_t>(max(0, a.lens[b])) + (a.new_lens ? max(0, a.new_lens[b]) : 0);
}
__device__ __forceinline__ int64_t pages_of(const PagesArgs& a, int b) {
  return (slots_of(a, b) + a.c.page_size - 1) / a.c.page_size;
}

__global__ __launch_bounds__(kBlock) void kv_reserve_clear(PagesArgs a) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
  if (i < a.c.pages) a.used[i] = 0;
}

// A wave per sequence: marks the pages that it keeps, counts those it lacks.
__global__ __launch_bounds__(kBlock) void kv_reserve_mark(PagesArgs a) {
  __shared__ int counts[kBlockWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = blockIdx.x * kBlockWaves + wave;
  int lacks = 0;
  if (b < a.batch) {
    const int need = static_cast<int>(min(pages_of(a, b), static_cast<int64_t>(a.c.table_width)));
    const int32_t* row = a.c.table + b * a.c.table_stride;
    for (int c = lane; c < need; c += 64) {
      const int32_t page = row[c];
      const bool has = page >= 0 && page < a.c.pages;
      if (has) a.used[page] = 1;
      lacks += !has;
    }
    for (int m = 32; m; m >>= 1) lacks += __shfl_xor(lacks, m);
    if (lane == 0) a.lacks[b] = lacks;
  }
  if (lane == 0) counts[wave] = lacks;
  __syncthreads();
  if (threadIdx.x == 0) {
    int sum = 0;
    for (int w = 0; w < kBlockWaves; ++w) sum += counts[w];
    a.group_lacks[blockIdx.x] = sum;
  }
}

// A wave per span of pages: lists its free ones.
__global__ __launch_bounds__(64) void kv_reserve_list(PagesArgs a) {
  const int lane = threadIdx.x;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kSpan;
  int count = 0;
  for (int i = 0; i < kSpan; i += 64) {
    const int64_t page = first + i + lane;
    const bool is_free = page < a.c.pages && !a.used[page];
    const uint64_t all = __builtin_amdgcn_ballot_w64(is_free);
    if (is_free) a.listed[first + count + __popcll(all & ((uint64_t{1} << lane) - 1))] = static_cast<int32_t>(page);
    count += __popcll(all);
  }
  if (lane == 0) a.span_free[blockIdx.x] = count;
}

// A wave per sequence: writes its row, the free pages from the rank on that the
// sequences before it leave.
__global__ __launch_bounds__(kBlock) void kv_reserve_assign(PagesArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = blockIdx.x * kBlockWaves + wave;
  if (b >= a.batch) return;
  int64_t rank = 0;  // pages that sequences before this one lack
  for (int i = lane; i < static_cast<int>(blockIdx.x); i += 64) rank += a.group_lacks[i];
  for (int m = 32; m; m >>= 1) rank += __shfl_xor(rank, m);
  for (int w = 0; w < wave; ++w) rank += a.lacks[blockIdx.x * kBlockWaves + w];
  const int64_t wanted = pages_of(a, b);
  const int need = static_cast<int>(min(wanted, static_cast<int64_t>(a.c.table_width)));
  const int32_t* row = a.c.table + b * a.c.table_stride;
  int32_t* out = a.out + b * a.out_stride;
  int span = 0, have = 0;
  int64_t before = 0;  // free pages of the spans before `span`
  for (int c0 = 0; c0 < a.c.table_width; c0 += 64) {
    const int c = c0 + lane;
    int32_t page = c < need ? row[c] : -1;
    bool has = page >= 0 && page < a.c.pages;
    const bool lacks = c < need && !has;
    const uint64_t all = __builtin_amdgcn_ballot_w64(lacks);
    if (!has) page = -1;
    if (lacks) {
      const int64_t k = rank + __popcll(all & ((uint64_t{1} << lane) - 1));
      while (span < a.spans && before + a.span_free[span] <= k) before += a.span_free[span++];
      if (span < a.spans) page = a.listed[static_cast<int64_t>(span) * kSpan + (k - before)];
      has = page >= 0;
    }
    rank += __popcll(all);
    have += __popcll(__builtin_amdgcn_ballot_w64(has));
    if (c < a.c.table_width) out[c] = page;
  }
  if (lane == 0) a.missing[b] = static_cast<int32_t>(wanted - have);
}

struct SlotsArgs {
  KvCache c;
  const int32_t *lens, *new_lens;
  int64_t* slots;
  int32_t* sequences;
  int64_t* positions;
  int64_t* ends;  // [batch]: tokens of the sequences up to this one
  int batch;
  int64_t tokens;
};

// One workgroup: the running sum of the new lengths.
__global__ __launch_bounds__(kBlock) void kv_slot_ends(SlotsArgs a) {
  __shared__ int64_t sums[kBlock];
  int64_t before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kBlock) {
    const int b = b0 + threadIdx.x;
    sums[threadIdx.x] = b < a.batch ? max(0, a.new_lens[b]) : 0;
    __syncthreads();
    for (int step = 1; step < kBlock; step *= 2) {
      const int64_t add = static_cast<int>(threadIdx.x) >= step ? sums[threadIdx.x - step] : 0;
      __syncthreads();
      sums[threadIdx.x] += add;
      __syncthreads();
    }
    if (b < a.batch) a.ends[b] = before + sums[threadIdx.x];
    before += sums[kBlock - 1];
    __syncthreads();
  }
}

__global__ __launch_bounds__(kBlock) void kv_slot_fill(SlotsArgs a) {
  const int64_t j = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
  if (j >= a.tokens) return;
  int lo = 0, hi = a.batch;  // the first sequence whose tokens end beyond j
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (a.ends[mid] > j) hi = mid;
    else lo = mid + 1;
  }
  int64_t slot = -1, position = 0;
  if (lo < a.batch) {
    position = static_cast<int64_t>(max(0, a.lens[lo])) + (j - (lo ? a.ends[lo - 1] : 0));
    if (position < a.c.capacity()) {
      const int p = static_cast<int>(position);
      const int32_t page = a.c.table[lo * a.c.table_stride + p / a.c.page_size];
      if (page >= 0 && page < a.c.pages) slot = static_cast<int64_t>(page) * a.c.page_size + p % a.c.page_size;
    }
  }
  a.slots[j] = slot;
  a.sequences[j] = lo < a.batch ? lo : -1;
  a.positions[j] = position;
}

int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
int64_t span_count(int64_t pages) { return (pages + kSpan - 1) / kSpan; }
int64_t group_count(int64_t batch) { return (batch + kBlockWaves - 1) / kBlockWaves; }

}  // namespace

int64_t kv_reserve_workspace(const mi355_kv_cache& c, int64_t batch) {
  const int64_t spans = span_count(c.pages);
  return up16(c.pages) + up16(4 * batch) + up16(4 * group_count(batch)) + up16(4 * spans) + 4 * spans * kSpan;
}

int kv_reserve_launch(const mi355_kv_cache& cache, const int32_t* lens, const int32_t* new_lens, int32_t* out,
                      int64_t out_stride, int32_t* missing, int64_t batch, void* work, hipStream_t stream) {
  static const char* what = "kv_cache_reserve launch";
  PagesArgs a{kv_cache_args(cache), lens, new_lens, out, out_stride, missing, static_cast<int>(batch),
              static_cast<int>(span_count(cache.pages)), static_cast<uint8_t*>(work), nullptr, nullptr, nullptr, nullptr};
  uint8_t* at = a.used + up16(cache.pages);
  a.lacks = reinterpret_cast<int32_t*>(at);
  at += up16(4 * batch);
  a.group_lacks = reinterpret_cast<int32_t*>(at);
  at += up16(4 * group_count(batch));
  a.span_free = reinterpret_cast<int32_t*>(at);
  a.listed = reinterpret_cast<int32_t*>(at + up16(4 * int64_t{a.spans}));
  const dim3 rows(static_cast<unsigned>(group_count(batch)));
  int st = launch(kv_reserve_clear, dim3(static_cast<unsigned>((cache.pages + kBlock - 1) / kBlock)), kBlock, 0, a, stream, what);
  if (st == MI355_OK) st = launch(kv_reserve_mark, rows, kBlock, 0, a, stream, what);
  if (st == MI355_OK) st = launch(kv_reserve_list, dim3(static_cast<unsigned>(a.spans)), 64, 0, a, stream, what);
  return st != MI355_OK ? st : launch(kv_reserve_assign, rows, kBlock, 0, a, stream, what);
}

int64_t kv_slot_map_workspace(int64_t batch) { return 8 * batch; }

int kv_slot_map_launch(const mi355_kv_cache& cache, const int32_t* lens, const int32_t* new_lens, int64_t* slots,
                       int32_t* sequences, int64_t* positions, int64_t batch, int64_t tokens, void* work,
                       hipStream_t stream) {
  static const char* what = "kv_slot_map launch";
  const SlotsArgs a{kv_cache_args(cache), lens, new_lens, slots, sequences, positions, static_cast<int64_t*>(work),
                    static_cast<int>(batch), tokens};
  const int st = launch(kv_slot_ends, dim3(1), kBlock, 0, a, stream, what);
  if (st != MI355_OK) return st;
  return launch(kv_slot_fill, dim3(static_cast<unsigned>((tokens + kBlock - 1) / kBlock)), kBlock, 0, a, stream, what);
}

}  // namespace mi355
