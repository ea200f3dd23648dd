// C ABI entry points of rotary positions, the key/value cache and attention
// over it (include/mi355_fused.h): argument validation.  Kernels and their
// launchers live in rotary.hip, kv_cache.hip, kv_pages.hip, tree_attention.hip
// and shared_prefix.hip.
#include "kv_cache.h"
#include "rotary.h"

namespace mi355 {

int rotary_launch(const void* x, void* y, const RotaryArgs& rot, int64_t batch, int64_t tokens, int heads, int d,
                  int64_t sb, int64_t st, int64_t sh, int dtype, hipStream_t stream);
int kv_append_launch(const mi355_kv_cache& cache, const RotaryArgs& rot, const void* k, const void* v, const void* q,
                     void* q_out, const int32_t* lens, const int32_t* new_lens, const int64_t* strides, int64_t batch,
                     int64_t tokens, int q_heads, int dtype, hipStream_t stream);
int kv_read_launch(const mi355_kv_cache& cache, void* k_out, void* v_out, const int32_t* start, const int32_t* end,
                   int64_t batch, int64_t tokens, int dtype, hipStream_t stream);
int kv_keep_launch(const mi355_kv_cache& cache, const int32_t* lens, const int32_t* kept, const int32_t* kept_lens,
                   int64_t kept_stride, int64_t batch, int most, hipStream_t stream);
int64_t tree_attention_workspace(const mi355_kv_cache& cache, int64_t batch, int64_t tokens, int64_t q_heads);
int tree_attention_launch(const mi355_kv_cache& cache, const void* q, void* out, const int32_t* lens,
                          const int32_t* new_lens, const uint8_t* mask, int64_t mask_b, int64_t mask_t, int64_t batch,
                          int tokens, int q_heads, const int64_t* q_strides, float scale, int dtype, void* work,
                          int64_t work_bytes, hipStream_t stream);
int64_t shared_prefix_workspace(const mi355_kv_cache& cache, int64_t batch, int64_t tokens, int64_t q_heads,
                                int64_t group_count);
int shared_prefix_launch(const mi355_kv_cache& cache, const void* q, void* out, const int32_t* lens,
                         const int32_t* new_lens, const int32_t* prefix_lens, const int32_t* groups, int group_count,
                         const uint8_t* mask, int64_t mask_b, int64_t mask_t, int64_t batch, int tokens, int q_heads,
                         const int64_t* q_strides, float scale, int dtype, void* work, int64_t work_bytes,
                         hipStream_t stream);
int64_t kv_reserve_workspace(const mi355_kv_cache& cache, int64_t batch);
int kv_reserve_launch(const mi355_kv_cache& cache, const int32_t* lens, const int32_t* new_lens, int32_t* out,
                      int64_t out_stride, int32_t* missing, int64_t batch, void* work, hipStream_t stream);
int64_t kv_slot_map_workspace(int64_t batch);
int kv_slot_map_launch(const mi355_kv_cache& cache, const int32_t* lens, const int32_t* new_lens, int64_t* slots,
                       int32_t* sequences, int64_t* positions, int64_t batch, int64_t tokens, void* work,
                       hipStream_t stream);

}  // namespace mi355

using mi355::aligned16;
using mi355::set_error;

namespace {

typedef long long ll;
constexpr int64_t kMaxRows = int64_t{1} << 24;  // workgroups of 256 threads in a launch's 2^32

int bad(const char* fn, const char* what) {
  set_error("%s: %s", fn, what);
  return MI355_ERR_INVALID;
}
int beyond(const char* fn, const char* what) {
  set_error("%s: %s", fn, what);
  return MI355_ERR_UNSUPPORTED;
}

// a * b < limit for a, b >= 0, without overflow.
bool product_below(int64_t a, int64_t b, int64_t limit) { return a == 0 || b <= (limit - 1) / a; }

int check_cache(const char* fn, const mi355_kv_cache* c) {
  if (c == nullptr) return bad(fn, "null cache");
  if (c->format != MI355_KV_16BIT && c->format != MI355_KV_INT8 && c->format != MI355_KV_E4M3) {
    set_error("%s: unknown cache format %d", fn, c->format);
    return MI355_ERR_INVALID;
  }
  if (c->pages < 0 || c->kv_heads < 1 || c->page_size < 1 || c->head_dim < 1 || c->table_width < 0 ||
      c->table_stride < c->table_width) {
    set_error("%s: cache sizes out of range (pages %lld, kv_heads %lld, page_size %lld, head_dim %lld, table %lld of "
              "stride %lld)", fn, static_cast<ll>(c->pages), static_cast<ll>(c->kv_heads),
              static_cast<ll>(c->page_size), static_cast<ll>(c->head_dim), static_cast<ll>(c->table_width),
              static_cast<ll>(c->table_stride));
    return MI355_ERR_INVALID;
  }
  if (c->head_dim % 16 != 0 || c->head_dim > 256) return beyond(fn, "head_dim must be a multiple of 16, at most 256");
  if (c->page_size % 16 != 0) return beyond(fn, "page_size must be a multiple of 16");
  if (c->kv_heads > 65535 || c->pages > 0x7fffffff || !product_below(c->table_width, c->page_size, int64_t{1} << 30))
    return beyond(fn, "cache beyond the kernels' limits (kv_heads <= 65535, pages < 2^31, table slots < 2^30)");
  return MI355_OK;
}

// The pointers of a cache that a call is about to use.
int check_pools(const char* fn, const mi355_kv_cache* c) {
  if (c->k == nullptr || c->v == nullptr || c->page_table == nullptr) return bad(fn, "null pointer in the cache");
  if (c->pages < 1 || c->table_width < 1) return bad(fn, "a cache without pages");
  if (!aligned16(c->k) || !aligned16(c->v)) return bad(fn, "the cache's pools must be 16-byte aligned");
  if (c->format != MI355_KV_16BIT) {
    if (c->k_scale == nullptr || c->v_scale == nullptr) return bad(fn, "a quantised cache needs its scales");
    if (!aligned16(c->k_scale) || !aligned16(c->v_scale)) return bad(fn, "the scales must be 16-byte aligned");
  }
  return MI355_OK;
}

int check_dtype16(const char* fn, int dtype) {
  if (!mi355::valid_dtype(dtype)) {
    set_error("%s: unknown dtype code %d", fn, dtype);
    return MI355_ERR_INVALID;
  }
  return dtype == MI355_F32 ? beyond(fn, "dtype must be fp16 or bf16") : MI355_OK;
}

int check_rotary(const char* fn, int64_t rotary_dim, int64_t head_dim, const void* positions, const void* inv_freq) {
  if (rotary_dim < 0 || rotary_dim % 2 != 0 || rotary_dim > head_dim) {
    set_error("%s: rotary_dim must be even and in [0, head_dim] (got %lld of %lld)", fn, static_cast<ll>(rotary_dim),
              static_cast<ll>(head_dim));
    return MI355_ERR_INVALID;
  }
  if (rotary_dim > 2 * mi355::kMaxPairs) return beyond(fn, "rotary_dim must be at most 256");
  if (rotary_dim > 0 && (positions == nullptr || inv_freq == nullptr))
    return bad(fn, "rotation needs positions and inv_freq");
  return MI355_OK;
}

// Rows of 16-bit elements that a kernel loads in 16-byte packets.
bool packet_rows(const void* p, const int64_t* strides) {
  return aligned16(p) && ((strides[0] | strides[1] | strides[2]) & 7) == 0;
}
bool negative(const int64_t* strides) { return strides[0] < 0 || strides[1] < 0 || strides[2] < 0; }

}  // namespace

MI355_EXPORT int mi355_rotary_fwd(const void* x, void* y, const int64_t* positions, const float* inv_freq,
                                  int64_t batch, int64_t tokens, int64_t heads, int64_t head_dim, int64_t rotary_dim,
                                  int64_t x_stride_b, int64_t x_stride_t, int64_t x_stride_h, int64_t pos_stride_b,
                                  int64_t pos_stride_t, float scale, int interleaved, int dtype, void* stream) {
  static const char* fn = "mi355_rotary_fwd";
  mi355::clear_error();
  if (!mi355::valid_dtype(dtype)) {
    set_error("%s: unknown dtype code %d", fn, dtype);
    return MI355_ERR_INVALID;
  }
  if (batch < 0 || tokens < 0 || heads < 0 || head_dim < 1) return bad(fn, "sizes out of range");
  if (x_stride_b < 0 || x_stride_t < 0 || x_stride_h < 0) return bad(fn, "strides of x must be >= 0");
  int st = check_rotary(fn, rotary_dim, head_dim, positions, inv_freq);
  if (st != MI355_OK) return st;
  if (batch == 0 || tokens == 0 || heads == 0) return MI355_OK;
  if (!product_below(batch, tokens, kMaxRows) || heads > 65535 || head_dim >= (1 << 20))
    return beyond(fn, "size beyond the kernel's limits (batch * tokens < 2^24, heads <= 65535, head_dim < 2^20)");
  if (x == nullptr || y == nullptr) return bad(fn, "null pointer");
  const mi355::RotaryArgs rot{positions, inv_freq, pos_stride_b, pos_stride_t, scale, static_cast<int>(rotary_dim),
                              interleaved != 0};
  return mi355::rotary_launch(x, y, rot, batch, tokens, static_cast<int>(heads), static_cast<int>(head_dim),
                              x_stride_b, x_stride_t, x_stride_h, dtype, static_cast<hipStream_t>(stream));
}

MI355_EXPORT int mi355_kv_cache_append_fwd(const mi355_kv_cache* cache, const void* k, const void* v, const void* q,
                                           void* q_out, const int32_t* seq_lens, const int32_t* new_lens,
                                           const int64_t* positions, const float* inv_freq, int64_t batch,
                                           int64_t tokens, int64_t q_heads, int64_t rotary_dim,
                                           const int64_t* strides, int64_t pos_stride_b, int64_t pos_stride_t,
                                           float scale, int interleaved, int dtype, void* stream) {
  static const char* fn = "mi355_kv_cache_append_fwd";
  mi355::clear_error();
  int st = check_cache(fn, cache);
  if (st == MI355_OK) st = check_dtype16(fn, dtype);
  if (st != MI355_OK) return st;
  if (batch < 0 || tokens < 0 || q_heads < 0) return bad(fn, "sizes out of range");
  st = check_rotary(fn, rotary_dim, cache->head_dim, positions, inv_freq);
  if (st != MI355_OK) return st;
  if (batch == 0 || tokens == 0) return MI355_OK;
  if (!product_below(batch, tokens, kMaxRows) || q_heads > 65535 || q_heads + 2 * cache->kv_heads > 65535)
    return beyond(fn, "size beyond the kernel's limits (batch * tokens < 2^24, q_heads + 2 kv_heads <= 65535)");
  if (k == nullptr || v == nullptr || seq_lens == nullptr || strides == nullptr ||
      (q_heads > 0 && (q == nullptr || q_out == nullptr)))
    return bad(fn, "null pointer");
  if (negative(strides) || negative(strides + 3) || (q_heads > 0 && negative(strides + 6)))
    return bad(fn, "strides must be >= 0");
  if (!packet_rows(k, strides) || !packet_rows(v, strides + 3) ||
      (q_heads > 0 && (!packet_rows(q, strides + 6) || !aligned16(q_out))))
    return beyond(fn, "k, v and q must be 16-byte aligned, their strides multiples of 8");
  st = check_pools(fn, cache);
  if (st != MI355_OK) return st;
  const mi355::RotaryArgs rot{positions, inv_freq, pos_stride_b, pos_stride_t, scale, static_cast<int>(rotary_dim),
                              interleaved != 0};
  int64_t all[9] = {strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], 0, 0, 0};
  if (q_heads > 0)
    for (int i = 6; i < 9; ++i) all[i] = strides[i];
  return mi355::kv_append_launch(*cache, rot, k, v, q, q_out, seq_lens, new_lens, all, batch, tokens,
                                 static_cast<int>(q_heads), dtype, static_cast<hipStream_t>(stream));
}

MI355_EXPORT int mi355_kv_cache_read_fwd(const mi355_kv_cache* cache, void* k_out, void* v_out, const int32_t* start,
                                         const int32_t* end, int64_t batch, int64_t tokens, int dtype, void* stream) {
  static const char* fn = "mi355_kv_cache_read_fwd";
  mi355::clear_error();
  int st = check_cache(fn, cache);
  if (st == MI355_OK) st = check_dtype16(fn, dtype);
  if (st != MI355_OK) return st;
  if (batch < 0 || tokens < 0) return bad(fn, "sizes out of range");
  if (batch == 0 || tokens == 0) return MI355_OK;
  // a workgroup of 256 threads holds 8 rows at least
  if (!product_below(batch, tokens, (4 * kMaxRows) / cache->kv_heads))
    return beyond(fn, "size beyond the kernel's limits (batch * tokens * kv_heads < 2^26)");
  if (k_out == nullptr || v_out == nullptr || end == nullptr) return bad(fn, "null pointer");
  if (!aligned16(k_out) || !aligned16(v_out)) return bad(fn, "k_out and v_out must be 16-byte aligned");
  st = check_pools(fn, cache);
  if (st != MI355_OK) return st;
  return mi355::kv_read_launch(*cache, k_out, v_out, start, end, batch, tokens, dtype,
                               static_cast<hipStream_t>(stream));
}

MI355_EXPORT int mi355_kv_cache_keep_fwd(const mi355_kv_cache* cache, const int32_t* seq_lens, const int32_t* kept,
                                         const int32_t* kept_lens, int64_t batch, int64_t max_kept,
                                         int64_t kept_stride, void* stream) {
  static const char* fn = "mi355_kv_cache_keep_fwd";
  mi355::clear_error();
  int st = check_cache(fn, cache);
  if (st != MI355_OK) return st;
  if (batch < 0 || max_kept < 0 || kept_stride < 0) return bad(fn, "sizes out of range");
  if (batch == 0 || max_kept == 0) return MI355_OK;
  if (max_kept > 128 || batch >= kMaxRows)
    return beyond(fn, "size beyond the kernel's limits (max_kept <= 128, batch < 2^24)");
  if (seq_lens == nullptr || kept == nullptr) return bad(fn, "null pointer");
  st = check_pools(fn, cache);
  if (st != MI355_OK) return st;
  return mi355::kv_keep_launch(*cache, seq_lens, kept, kept_lens, kept_stride, batch, static_cast<int>(max_kept),
                               static_cast<hipStream_t>(stream));
}

MI355_EXPORT int64_t mi355_tree_attention_workspace(const mi355_kv_cache* cache, int64_t batch, int64_t tokens,
                                                    int64_t q_heads) {
  static const char* fn = "mi355_tree_attention_workspace";
  mi355::clear_error();
  if (check_cache(fn, cache) != MI355_OK || batch < 1 || tokens < 1 || tokens > 128 || q_heads < 1 ||
      q_heads > 65535 || q_heads % cache->kv_heads != 0 || !product_below(batch, tokens * q_heads, kMaxRows))
    return 0;
  return mi355::tree_attention_workspace(*cache, batch, tokens, q_heads);
}

namespace {

// What both attentions check.  *empty: nothing to do.
int check_attention(const char* fn, const mi355_kv_cache* cache, const void* q, const void* out, const int32_t* seq_lens,
                    const void* tree_mask, int64_t mask_stride_b, int64_t mask_stride_t, int64_t batch, int64_t tokens,
                    int64_t q_heads, const int64_t* q_strides, int dtype, const void* workspace,
                    int64_t workspace_bytes, bool* empty) {
  *empty = false;
  int st = check_cache(fn, cache);
  if (st == MI355_OK) st = check_dtype16(fn, dtype);
  if (st != MI355_OK) return st;
  if (batch < 0 || tokens < 0 || q_heads < 0) return bad(fn, "sizes out of range");
  if (q_heads % cache->kv_heads != 0) return bad(fn, "q_heads must be a multiple of kv_heads");
  *empty = batch == 0 || tokens == 0 || q_heads == 0;
  if (*empty) return MI355_OK;
  if (tokens > 128 || q_heads > 65535 || !product_below(batch, tokens * q_heads, kMaxRows))
    return beyond(fn, "size beyond the kernel's limits (tokens <= 128, q_heads <= 65535, "
                      "batch * tokens * q_heads < 2^24)");
  if (q == nullptr || out == nullptr || seq_lens == nullptr || q_strides == nullptr) return bad(fn, "null pointer");
  if (negative(q_strides) || (tree_mask != nullptr && (mask_stride_b < 0 || mask_stride_t < 0)))
    return bad(fn, "strides must be >= 0");
  if (!packet_rows(q, q_strides) || !aligned16(out))
    return beyond(fn, "q and out must be 16-byte aligned, the strides of q multiples of 8");
  if (workspace != nullptr && (!aligned16(workspace) || workspace_bytes < 0))
    return bad(fn, "the workspace must be 16-byte aligned and its size >= 0");
  return check_pools(fn, cache);
}

// The page table alone, and a workspace that the call cannot do without.
int check_pages(const char* fn, const mi355_kv_cache* cache, const void* workspace, int64_t workspace_bytes,
                int64_t needs) {
  if (cache->page_table == nullptr) return bad(fn, "null pointer in the cache");
  if (cache->pages < 1 || cache->table_width < 1) return bad(fn, "a cache without pages");
  if (needs > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < needs)) {
    set_error("%s: the workspace must be 16-byte aligned and of %lld bytes", fn, static_cast<ll>(needs));
    return MI355_ERR_INVALID;
  }
  return MI355_OK;
}

}  // namespace

MI355_EXPORT int mi355_tree_attention_fwd(const mi355_kv_cache* cache, const void* q, void* out,
                                          const int32_t* seq_lens, const int32_t* new_lens, const uint8_t* tree_mask,
                                          int64_t mask_stride_b, int64_t mask_stride_t, int64_t batch, int64_t tokens,
                                          int64_t q_heads, const int64_t* q_strides, float scale, int dtype,
                                          void* workspace, int64_t workspace_bytes, void* stream) {
  static const char* fn = "mi355_tree_attention_fwd";
  mi355::clear_error();
  bool empty;
  const int st = check_attention(fn, cache, q, out, seq_lens, tree_mask, mask_stride_b, mask_stride_t, batch, tokens,
                                 q_heads, q_strides, dtype, workspace, workspace_bytes, &empty);
  if (st != MI355_OK || empty) return st;
  return mi355::tree_attention_launch(*cache, q, out, seq_lens, new_lens, tree_mask, mask_stride_b, mask_stride_t,
                                      batch, static_cast<int>(tokens), static_cast<int>(q_heads), q_strides, scale,
                                      dtype, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

MI355_EXPORT int64_t mi355_shared_prefix_attention_workspace(const mi355_kv_cache* cache, int64_t batch,
                                                             int64_t tokens, int64_t q_heads, int64_t group_count) {
  static const char* fn = "mi355_shared_prefix_attention_workspace";
  mi355::clear_error();
  if (check_cache(fn, cache) != MI355_OK || batch < 1 || tokens < 1 || tokens > 128 || q_heads < 1 ||
      q_heads > 65535 || q_heads % cache->kv_heads != 0 || !product_below(batch, tokens * q_heads, kMaxRows) ||
      group_count < 0 || group_count > batch)
    return 0;
  return mi355::shared_prefix_workspace(*cache, batch, tokens, q_heads, group_count);
}

MI355_EXPORT int mi355_shared_prefix_attention_fwd(
    const mi355_kv_cache* cache, const void* q, void* out, const int32_t* seq_lens, const int32_t* new_lens,
    const int32_t* prefix_lens, const int32_t* groups, int64_t group_count, const uint8_t* tree_mask,
    int64_t mask_stride_b, int64_t mask_stride_t, int64_t batch, int64_t tokens, int64_t q_heads,
    const int64_t* q_strides, float scale, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  static const char* fn = "mi355_shared_prefix_attention_fwd";
  mi355::clear_error();
  bool empty;
  const int st = check_attention(fn, cache, q, out, seq_lens, tree_mask, mask_stride_b, mask_stride_t, batch, tokens,
                                 q_heads, q_strides, dtype, workspace, workspace_bytes, &empty);
  if (st != MI355_OK) return st;
  if (group_count < 0 || group_count > batch) return bad(fn, "group_count must be in [0, batch]");
  if (empty) return MI355_OK;
  if (group_count > 0 && prefix_lens == nullptr) return bad(fn, "null pointer");
  if (group_count > 0 && groups == nullptr && batch % group_count != 0)
    return bad(fn, "without groups, batch must be a multiple of group_count");
  return mi355::shared_prefix_launch(*cache, q, out, seq_lens, new_lens, prefix_lens, groups,
                                     static_cast<int>(group_count), tree_mask, mask_stride_b, mask_stride_t, batch,
                                     static_cast<int>(tokens), static_cast<int>(q_heads), q_strides, scale, dtype,
                                     workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

namespace {
bool reserve_fits(const mi355_kv_cache* c, int64_t batch) {
  return batch < kMaxRows && c->pages < (int64_t{1} << 30) && product_below(batch, c->table_width, int64_t{1} << 31);
}
}  // namespace

MI355_EXPORT int64_t mi355_kv_cache_reserve_workspace(const mi355_kv_cache* cache, int64_t batch) {
  mi355::clear_error();
  if (check_cache("mi355_kv_cache_reserve_workspace", cache) != MI355_OK || batch < 1 || !reserve_fits(cache, batch))
    return 0;
  return mi355::kv_reserve_workspace(*cache, batch);
}

MI355_EXPORT int mi355_kv_cache_reserve_fwd(const mi355_kv_cache* cache, const int32_t* seq_lens,
                                            const int32_t* new_lens, int32_t* table_out, int64_t out_stride,
                                            int32_t* missing, int64_t batch, void* workspace, int64_t workspace_bytes,
                                            void* stream) {
  static const char* fn = "mi355_kv_cache_reserve_fwd";
  mi355::clear_error();
  int st = check_cache(fn, cache);
  if (st != MI355_OK) return st;
  if (batch < 0 || out_stride < cache->table_width) return bad(fn, "sizes out of range (out_stride >= table_width)");
  if (batch == 0) return MI355_OK;
  if (!reserve_fits(cache, batch))
    return beyond(fn, "size beyond the kernel's limits (batch < 2^24, batch * table_width < 2^31, pages < 2^30)");
  if (seq_lens == nullptr || table_out == nullptr || missing == nullptr) return bad(fn, "null pointer");
  if (table_out == cache->page_table && batch > 1 && out_stride != cache->table_stride)
    return bad(fn, "in place, out_stride must be the table's");
  st = check_pages(fn, cache, workspace, workspace_bytes, mi355::kv_reserve_workspace(*cache, batch));
  if (st != MI355_OK) return st;
  return mi355::kv_reserve_launch(*cache, seq_lens, new_lens, table_out, out_stride, missing, batch, workspace,
                                  static_cast<hipStream_t>(stream));
}

MI355_EXPORT int64_t mi355_kv_slot_map_workspace(int64_t batch) {
  mi355::clear_error();
  return batch < 1 || batch >= kMaxRows ? 0 : mi355::kv_slot_map_workspace(batch);
}

MI355_EXPORT int mi355_kv_slot_map_fwd(const mi355_kv_cache* cache, const int32_t* seq_lens, const int32_t* new_lens,
                                       int64_t* slots, int32_t* sequences, int64_t* positions, int64_t batch,
                                       int64_t tokens, void* workspace, int64_t workspace_bytes, void* stream) {
  static const char* fn = "mi355_kv_slot_map_fwd";
  mi355::clear_error();
  int st = check_cache(fn, cache);
  if (st != MI355_OK) return st;
  if (batch < 0 || tokens < 0) return bad(fn, "sizes out of range");
  if (tokens == 0) return MI355_OK;
  if (batch >= kMaxRows || tokens >= (int64_t{1} << 31))
    return beyond(fn, "size beyond the kernel's limits (batch < 2^24, tokens < 2^31)");
  if (batch < 1) return bad(fn, "tokens of no sequence");
  if (seq_lens == nullptr || new_lens == nullptr || slots == nullptr || sequences == nullptr || positions == nullptr)
    return bad(fn, "null pointer");
  st = check_pages(fn, cache, workspace, workspace_bytes, mi355::kv_slot_map_workspace(batch));
  if (st != MI355_OK) return st;
  return mi355::kv_slot_map_launch(*cache, seq_lens, new_lens, slots, sequences, positions, batch, tokens, workspace,
                                   static_cast<hipStream_t>(stream));
}
