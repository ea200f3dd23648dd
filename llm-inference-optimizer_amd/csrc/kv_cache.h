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

// x / scale, correctly rounded, for rc = 1 / scale correctly rounded: the
// remainder of the first quotient is exact in one fma.  A third of a division's
// instructions.
__device__ __forceinline__ float quotient(float x, float scale, float rc) {
  const float q = x * rc;
  return __builtin_fmaf(__builtin_fmaf(-q, scale, x), rc, q);
}

// Quotients (at most the format's largest code, up to their rounding) -> four
// codes, rounded to nearest, ties to even.
template <int FMT> __device__ __forceinline__ uint32_t encode4(const float (&f)[4]) {
  if constexpr (FMT == KV_INT8) {
    // 1.5 * 2^23 + f has f, rounded to an integer, in its low bits
    uint32_t t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = as_u32(f[i] + 12582912.0f);
    return __builtin_amdgcn_perm(t[1], t[0], 0x0c0c0400u) | __builtin_amdgcn_perm(t[3], t[2], 0x04000c0cu);
  } else {
    int d = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
    d = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], d, true);
    return static_cast<uint32_t>(d);
  }
}

}  // namespace mi355
