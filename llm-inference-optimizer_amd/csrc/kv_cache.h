// The paged key/value cache as kernels see it, and its element formats.
//
// A pool of pages [pages, kv_heads, page_size, head_dim] for keys and one for
// values; the token in slot s of sequence b lies in page table[b][s /
// page_size] at place s % page_size.  Formats: 16-bit values, or one-byte
// codes (int8, e4m3) with an fp32 scale per token and head in
// [pages, kv_heads, page_size]: value = code * scale.
//
// Sizes that come from device memory (page numbers, lengths) are checked where
// they are used: a slot outside the table or on a page outside the pool has no
// place -- it is not written, reads as zero and is not attended to.
#pragma once

#include "common.h"

namespace mi355 {

enum { KV_16BIT = MI355_KV_16BIT, KV_INT8 = MI355_KV_INT8, KV_E4M3 = MI355_KV_E4M3 };

struct KvCache {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  const int32_t* table;
  int64_t table_stride;
  int32_t pages, table_width, heads, page_size, d;

  __device__ __forceinline__ int32_t capacity() const { return table_width * page_size; }

  // Row of a slot in [pages * heads * page_size] for head h; -1 without one.
  __device__ __forceinline__ int64_t row(int64_t b, int64_t slot, int h) const {
    if (slot < 0 || slot >= capacity()) return -1;
    const int32_t i = static_cast<int32_t>(slot) / page_size;
    const int32_t page = table[b * table_stride + i];
    if (page < 0 || page >= pages) return -1;
    return (static_cast<int64_t>(page) * heads + h) * page_size + (static_cast<int32_t>(slot) - i * page_size);
  }
};

inline KvCache kv_cache_args(const mi355_kv_cache& c) {
  return {c.k, c.v, c.k_scale, c.v_scale, c.page_table, c.table_stride, static_cast<int32_t>(c.pages),
          static_cast<int32_t>(c.table_width), static_cast<int32_t>(c.kv_heads), static_cast<int32_t>(c.page_size),
          static_cast<int32_t>(c.head_dim)};
}

template <int FMT> constexpr float kv_top() { return FMT == KV_INT8 ? 127.0f : 448.0f; }

// Four codes of one dword as fp32.
template <int FMT> __device__ __forceinline__ void decode4(uint32_t d, float (&f)[4]) {
  if constexpr (FMT == KV_INT8) {
    f[0] = static_cast<float>(static_cast<int8_t>(d & 0xffu));
    f[1] = static_cast<float>(static_cast<int8_t>((d >> 8) & 0xffu));
    f[2] = static_cast<float>(static_cast<int8_t>((d >> 16) & 0xffu));
    f[3] = static_cast<float>(static_cast<int8_t>(d >> 24));
  } else {
    f[0] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(d), 0);
    f[1] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(d), 1);
    f[2] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(d), 2);
    f[3] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(d), 3);
  }
}

// fp32 values divided by their scale (|f| <= the format's largest code, up to
// the division's rounding) -> four codes, rounded to nearest, ties to even.
template <int FMT> __device__ __forceinline__ uint32_t encode4(const float (&f)[4]) {
  if constexpr (FMT == KV_INT8) {
    uint32_t d = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      d |= (static_cast<uint32_t>(static_cast<int>(__builtin_rintf(f[i]))) & 0xffu) << (8 * i);
    return d;
  } else {
    int d = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
    d = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], d, true);
    return static_cast<uint32_t>(d);
  }
}

}  // namespace mi355
