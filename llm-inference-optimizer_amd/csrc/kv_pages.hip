// Page tables and slot maps from the lengths of requests, for gfx950.
//
// kv_reserve: entry (b, c) of the new table is the old one where sequence b needs
// column c and has a page there, else a free page, the k-th such entry (b first)
// taking the k-th page that nobody keeps.  Bound by launches and by the trips of
// loads that wait for each other: a table is read and written once, 8 bytes per
// entry.  Tables of a decode step are one workgroup's work (kv_reserve_one), its
// pages a bit each in LDS; larger ones take four launches.  32 sequences of up to
// 4001 tokens, 64 a page: 4.1 us, 8.5 with the launch, where the four launches take
// 17.  4096 sequences of up to 8300 tokens, 16 a page: 30 us, of which clear 2,
// mark 9, list 3 and assign 16; its 9.6 MB would take 2 us at a copy's rate.
#include "kv_cache.h"

namespace mi355 {
namespace {

constexpr int kBlock = 256, kBlockWaves = kBlock / 64;
constexpr int kSpans = 2048;  // of pages at most, whose free ones a wave lists each
constexpr int kOneThreads = 1024, kOneWaves = kOneThreads / 64;
constexpr int kOneWords = 16384;  // 2^19 pages
constexpr int kOneEntries = 32768, kOneRows = 1024;

struct PagesArgs {
  KvCache c;
  const int32_t *lens, *new_lens;
  int32_t* out;
  int64_t out_stride;
  int32_t* missing;
  int batch, spans, span;
  uint8_t* used;          // [spans * span]: whether an entry keeps the page
  int32_t* lacks;         // [batch]: pages that a sequence lacks, within the table
  int32_t* group_lacks;   // [ceil(batch / kBlockWaves)]
  int32_t* span_free;     // [spans]
  int32_t* listed;        // [spans * span]: the free pages of a span, in order
};

__device__ __forceinline__ int64_t slots_of(const PagesArgs& a, int b) {
  return static_cast<int64_t>(max(0, a.lens[b])) + (a.new_lens ? max(0, a.new_lens[b]) : 0);
}
__device__ __forceinline__ int64_t pages_of(const PagesArgs& a, int b) {
  return (slots_of(a, b) + a.c.page_size - 1) / a.c.page_size;
}

// One workgroup.  Its waves take as many sequences each, in order.
__global__ __launch_bounds__(kOneThreads) void kv_reserve_one(PagesArgs a) {
  __shared__ uint32_t kept[kOneWords];       // a bit per page
  __shared__ int32_t before[kOneThreads];    // free pages before a thread's words
  __shared__ int32_t lacks[kOneWaves], frees[kOneWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int words = (a.c.pages + 31) / 32, own = (words + kOneThreads - 1) / kOneThreads;
  const int rows = (a.batch + kOneWaves - 1) / kOneWaves, first = wave * rows, last = min(first + rows, a.batch);
  const int64_t mine = first + lane < last ? pages_of(a, first + lane) : 0;  // at most 64 rows
  const int cut = static_cast<int>(min(mine, static_cast<int64_t>(a.c.table_width)));
  for (int i = threadIdx.x; i < words; i += kOneThreads) kept[i] = 0;
  __syncthreads();
  int lack = 0;
  for (int b = first; b < last; ++b) {
    const int need = __builtin_amdgcn_readlane(cut, b - first);
    const int32_t* row = a.c.table + b * a.c.table_stride;
    for (int c = lane; c < need; c += 64) {
      const int32_t page = row[c];
      const bool has = page >= 0 && page < a.c.pages;
      if (has) atomicOr(&kept[page >> 5], 1u << (page & 31));
      lack += !has;
    }
  }
  lack = wave_scan(lack);
  if (lane == 63) lacks[wave] = lack;
  __syncthreads();
  // free pages before each thread's words
  int count = 0;
  for (int i = threadIdx.x * own; i < min((static_cast<int>(threadIdx.x) + 1) * own, words); ++i)
    count += min(32, a.c.pages - 32 * i) - __popc(kept[i]);
  const int upto = wave_scan(count);
  if (lane == 63) frees[wave] = upto;
  __syncthreads();
  int rank = 0, base = 0, all = 0;
  for (int w = 0; w < kOneWaves; ++w) {
    rank += w < wave ? lacks[w] : 0;
    base += w < wave ? frees[w] : 0;
    all += frees[w];
  }
  before[threadIdx.x] = base + upto - count;
  __syncthreads();
  for (int b = first; b < last; ++b) {
    const int need = __builtin_amdgcn_readlane(cut, b - first);
    const int32_t* row = a.c.table + b * a.c.table_stride;
    int32_t* out = a.out + b * a.out_stride;
    int have = 0;
    for (int c0 = 0; c0 < a.c.table_width; c0 += 64) {
      const int c = c0 + lane;
      int32_t page = c < need ? row[c] : -1;
      if (page >= a.c.pages) page = -1;
      const bool lacks_it = c < need && page < 0;
      const uint64_t some = __builtin_amdgcn_ballot_w64(lacks_it);
      if (some) {
        const int k = rank + __popcll(some & ((uint64_t{1} << lane) - 1));
        page = lacks_it ? -1 : page;
        if (lacks_it && k < all) {
          int lo = 0, hi = kOneThreads - 1;  // the last thread before whose words at most k are free
          while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (before[mid] <= k) lo = mid;
            else hi = mid - 1;
          }
          int left = k - before[lo], i = lo * own;
          for (;; ++i) {
            const int n = min(32, a.c.pages - 32 * i) - __popc(kept[i]);
            if (left < n) break;
            left -= n;
          }
          uint32_t open = ~kept[i];
          for (; left; --left) open &= open - 1;
          page = 32 * i + __builtin_ctz(open);
        }
        rank += __popcll(some);
      }
      have += __popcll(__builtin_amdgcn_ballot_w64(page >= 0));
      if (c < a.c.table_width) out[c] = page;
    }
    if (lane == b - first) a.missing[b] = static_cast<int32_t>(mine - have);
  }
}

__global__ __launch_bounds__(kBlock) void kv_reserve_clear(PagesArgs a) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
  if (16 * i < static_cast<int64_t>(a.spans) * a.span) reinterpret_cast<u32x4*>(a.used)[i] = u32x4{0, 0, 0, 0};
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
    for (int c0 = lane; c0 < need; c0 += 4 * 64) {
      int32_t page[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) page[i] = row[min(c0 + 64 * i, need - 1)];  // all on their way
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = c0 + 64 * i < need, has = page[i] >= 0 && page[i] < a.c.pages;
        if (in && has) a.used[page[i]] = 1;
        lacks += in && !has;
      }
    }
    lacks = __builtin_amdgcn_readlane(wave_scan(lacks), 63);
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

// A wave per span of pages, 1024 at a time: lists its free ones.
__global__ __launch_bounds__(64) void kv_reserve_list(PagesArgs a) {
  const int lane = threadIdx.x;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * a.span;
  int count = 0;
  for (int i0 = 0; i0 < a.span; i0 += 4096) {
    u32x4 used[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t page = first + min(i0 + 1024 * j, a.span - 1024) + 16 * lane;
      used[j] = *reinterpret_cast<const u32x4*>(a.used + page);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (i0 + 1024 * j >= a.span) break;
      const int64_t page = first + i0 + 1024 * j + 16 * lane;
      uint32_t open = 0;  // a bit per page
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const uint32_t four = used[j][k / 4];
        open |= ((four >> (8 * (k % 4)) & 0xff) == 0 && page + k < a.c.pages) ? 1u << k : 0u;
      }
      const int own = __popc(open), upto = wave_scan(own);
      int64_t at = first + count + upto - own;
      for (; open; open &= open - 1) a.listed[at++] = static_cast<int32_t>(page + __builtin_ctz(open));
      count += __builtin_amdgcn_readlane(upto, 63);
    }
  }
  if (lane == 0) a.span_free[blockIdx.x] = count;
}

// A wave per sequence: writes its row, the free pages from the rank on that the
// sequences before it leave.
__global__ __launch_bounds__(kBlock) void kv_reserve_assign(PagesArgs a) {
  __shared__ int32_t before[kSpans];  // free pages of the spans before one
  __shared__ int32_t sums[kBlockWaves], ranks[kBlockWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = blockIdx.x * kBlockWaves + wave;
  constexpr int OWN = kSpans / kBlock;
  int count[OWN], own = 0, earlier = 0;
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    const int span = threadIdx.x * OWN + i;
    count[i] = span < a.spans ? a.span_free[span] : 0;
  }
  for (int i = threadIdx.x; i < static_cast<int>(blockIdx.x); i += kBlock) earlier += a.group_lacks[i];
#pragma unroll
  for (int i = 0; i < OWN; ++i) own += count[i];
  const int upto = wave_scan(own);
  earlier = wave_scan(earlier);
  if (lane == 63) {
    sums[wave] = upto;
    ranks[wave] = earlier;
  }
  __syncthreads();
  int at = upto - own, all = 0, rank = 0;
  for (int w = 0; w < kBlockWaves; ++w) {
    at += w < wave ? sums[w] : 0;
    all += sums[w];
    rank += ranks[w];
  }
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    before[threadIdx.x * OWN + i] = at;
    at += count[i];
  }
  __syncthreads();
  if (b >= a.batch) return;
  for (int w = 0; w < wave; ++w) rank += a.lacks[blockIdx.x * kBlockWaves + w];
  const int64_t wanted = pages_of(a, b);
  const int need = static_cast<int>(min(wanted, static_cast<int64_t>(a.c.table_width)));
  const int32_t* row = a.c.table + b * a.c.table_stride;
  int32_t* out = a.out + b * a.out_stride;
  int have = 0;
  for (int c0 = lane; c0 - lane < a.c.table_width; c0 += 4 * 64) {
    int32_t page[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) page[i] = c0 + 64 * i < need ? row[c0 + 64 * i] : -1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = c0 + 64 * i;
      if (page[i] >= a.c.pages || page[i] < 0) page[i] = -1;
      const bool lacks = c < need && page[i] < 0;
      const uint64_t some = __builtin_amdgcn_ballot_w64(lacks);
      if (lacks) {
        const int k = rank + __popcll(some & ((uint64_t{1} << lane) - 1));
        if (k < all) {
          int lo = 0, hi = a.spans - 1;  // the last span before which at most k are free
          while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (before[mid] <= k) lo = mid;
            else hi = mid - 1;
          }
          page[i] = a.listed[static_cast<int64_t>(lo) * a.span + (k - before[lo])];
        }
      }
      rank += __popcll(some);
      have += __popcll(__builtin_amdgcn_ballot_w64(page[i] >= 0));
      if (c < a.c.table_width) out[c] = page[i];
    }
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
  bool pairs;     // two rows are stored at once
  int64_t tokens;
};

// The row of a token of sequence `b`, `before` it the packed batch's.
struct SlotRow {
  int64_t slot, position;
  __device__ __forceinline__ SlotRow(const SlotsArgs& a, int b, int64_t j, int64_t before) : slot(-1), position(0) {
    if (b >= a.batch) return;
    position = static_cast<int64_t>(max(0, a.lens[b])) + (j - before);
    if (position >= a.c.capacity()) return;
    const int p = static_cast<int>(position), c = p / a.c.page_size;
    const int32_t page = a.c.table[b * a.c.table_stride + c];
    if (page >= 0 && page < a.c.pages) slot = static_cast<int64_t>(page) * a.c.page_size + (p - c * a.c.page_size);
  }
};

// The first sequence whose tokens end beyond j.
template <typename E> __device__ __forceinline__ int sequence_of(const E* ends, int batch, int64_t j) {
  int lo = 0, hi = batch;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (ends[mid] > j) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// Up to 4096 sequences: every workgroup sums their lengths for itself, for 2048
// tokens, two neighbours per thread and store.  16 sequences of 8 tokens: 3.1 us, 8.5
// with the launch; 300 prompts of 2.3 million tokens: 19 us, 2.4 TB/s written, where
// a launch for the sums and one for the rows take 23.
constexpr int kSlotBatch = 4096, kSlotTokens = 2048;

__global__ __launch_bounds__(kBlock) void kv_slot_rows(SlotsArgs a) {
  __shared__ int64_t ends[kSlotBatch];
  __shared__ int64_t sums[kBlockWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int own = (a.batch + kBlock - 1) / kBlock, first = threadIdx.x * own;
  int64_t sum = 0;
  for (int i = first; i < min(first + own, a.batch); ++i) sum += max(0, a.new_lens[i]);
  int64_t upto = sum;
  for (int step = 1; step < 64; step *= 2) {
    const int64_t add = __shfl_up(upto, step);
    if (lane >= step) upto += add;
  }
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  upto -= sum;
  for (int w = 0; w < wave; ++w) upto += sums[w];
  for (int i = first; i < min(first + own, a.batch); ++i) ends[i] = upto += max(0, a.new_lens[i]);
  __syncthreads();
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kSlotTokens;
  typedef int64_t i64x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int k = 0; k < kSlotTokens / (2 * kBlock); ++k) {
    const int64_t j = base + 2 * (k * kBlock + static_cast<int>(threadIdx.x));
    if (j >= a.tokens) break;
    const int b0 = sequence_of(ends, a.batch, j);
    const int b1 = b0 < a.batch && ends[b0] > j + 1 ? b0 : sequence_of(ends, a.batch, j + 1);
    const SlotRow r0(a, b0, j, b0 ? ends[b0 - 1] : 0), r1(a, b1, j + 1, b1 ? ends[b1 - 1] : 0);
    const int32_t s0 = b0 < a.batch ? b0 : -1, s1 = b1 < a.batch ? b1 : -1;
    if (a.pairs && j + 1 < a.tokens) {
      *reinterpret_cast<i64x2*>(a.slots + j) = i64x2{r0.slot, r1.slot};
      *reinterpret_cast<i64x2*>(a.positions + j) = i64x2{r0.position, r1.position};
      *reinterpret_cast<int2*>(a.sequences + j) = int2{s0, s1};
    } else {
      a.slots[j] = r0.slot;
      a.positions[j] = r0.position;
      a.sequences[j] = s0;
      if (j + 1 < a.tokens) {
        a.slots[j + 1] = r1.slot;
        a.positions[j + 1] = r1.position;
        a.sequences[j + 1] = s1;
      }
    }
  }
}

// More: one workgroup makes the running sum of the new lengths, 256 at a time: 23 us
// for 4097 sequences of up to 8 tokens (16 for 4096), 83 for 20000.
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
  const int b = sequence_of(a.ends, a.batch, j);
  const SlotRow r(a, b, j, b ? a.ends[b - 1] : 0);
  a.slots[j] = r.slot;
  a.sequences[j] = b < a.batch ? b : -1;
  a.positions[j] = r.position;
}

int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
// Pages of a span, whole 1024, so that there are at most kSpans of them.
int64_t span_of(int64_t pages) {
  int64_t span = 1024;
  while (pages > span * kSpans) span *= 2;
  return span;
}
int64_t span_count(int64_t pages) { return (pages + span_of(pages) - 1) / span_of(pages); }
bool one_workgroup(const mi355_kv_cache& c, int64_t batch) {
  return batch <= kOneRows && batch * c.table_width <= kOneEntries && c.pages <= 32 * kOneWords;
}
int64_t group_count(int64_t batch) { return (batch + kBlockWaves - 1) / kBlockWaves; }

}  // namespace

int64_t kv_reserve_workspace(const mi355_kv_cache& c, int64_t batch) {
  if (one_workgroup(c, batch)) return 0;
  const int64_t spans = span_count(c.pages), pages = spans * span_of(c.pages);
  return up16(pages) + up16(4 * batch) + up16(4 * group_count(batch)) + up16(4 * spans) + 4 * pages;
}

int kv_reserve_launch(const mi355_kv_cache& cache, const int32_t* lens, const int32_t* new_lens, int32_t* out,
                      int64_t out_stride, int32_t* missing, int64_t batch, void* work, hipStream_t stream) {
  static const char* what = "kv_cache_reserve launch";
  PagesArgs a{kv_cache_args(cache), lens, new_lens, out, out_stride, missing, static_cast<int>(batch),
              static_cast<int>(span_count(cache.pages)), static_cast<int>(span_of(cache.pages)),
              static_cast<uint8_t*>(work), nullptr, nullptr, nullptr, nullptr};
  if (one_workgroup(cache, batch)) return launch(kv_reserve_one, dim3(1), kOneThreads, 0, a, stream, what);
  const int64_t pages = int64_t{a.spans} * a.span;
  uint8_t* at = a.used + up16(pages);
  a.lacks = reinterpret_cast<int32_t*>(at);
  at += up16(4 * batch);
  a.group_lacks = reinterpret_cast<int32_t*>(at);
  at += up16(4 * group_count(batch));
  a.span_free = reinterpret_cast<int32_t*>(at);
  a.listed = reinterpret_cast<int32_t*>(at + up16(4 * int64_t{a.spans}));
  const dim3 rows(static_cast<unsigned>(group_count(batch)));
  int st = launch(kv_reserve_clear, dim3(static_cast<unsigned>((pages / 16 + kBlock - 1) / kBlock)), kBlock, 0, a, stream, what);
  if (st == MI355_OK) st = launch(kv_reserve_mark, rows, kBlock, 0, a, stream, what);
  if (st == MI355_OK) st = launch(kv_reserve_list, dim3(static_cast<unsigned>(a.spans)), 64, 0, a, stream, what);
  return st != MI355_OK ? st : launch(kv_reserve_assign, rows, kBlock, 0, a, stream, what);
}

int64_t kv_slot_map_workspace(int64_t batch) { return batch <= kSlotBatch ? 0 : 8 * batch; }

int kv_slot_map_launch(const mi355_kv_cache& cache, const int32_t* lens, const int32_t* new_lens, int64_t* slots,
                       int32_t* sequences, int64_t* positions, int64_t batch, int64_t tokens, void* work,
                       hipStream_t stream) {
  static const char* what = "kv_slot_map launch";
  const bool pairs = aligned16(slots) && aligned16(positions) && aligned16(sequences);
  const SlotsArgs a{kv_cache_args(cache), lens, new_lens, slots, sequences, positions, static_cast<int64_t*>(work),
                    static_cast<int>(batch), pairs, tokens};
  if (batch <= kSlotBatch)
    return launch(kv_slot_rows, dim3(static_cast<unsigned>((tokens + kSlotTokens - 1) / kSlotTokens)), kBlock, 0, a, stream, what);
  const int st = launch(kv_slot_ends, dim3(1), kBlock, 0, a, stream, what);
  if (st != MI355_OK) return st;
  return launch(kv_slot_fill, dim3(static_cast<unsigned>((tokens + kBlock - 1) / kBlock)), kBlock, 0, a, stream, what);
}

}  // namespace mi355
