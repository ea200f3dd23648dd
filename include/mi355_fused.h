/*
 * mi355_fused.h -- C ABI of the MI355X (gfx950) fused RMSNorm and SiLU-and-mul
 * kernels, the fused gate/up projections, the weight-only int8 (W8A16)
 * linear with its quantiser, the 16-bit linear of the MLP's down projection,
 * what lies between an attention block's projections (rotary positions, a
 * paged and quantised key/value cache, and attention over it, shared prefixes
 * among it), page tables made from lengths, and drawing the next tokens.
 *
 * The reference has no FFI: its boundary is a pair of Python launchers that
 * hand torch tensors to Triton kernels.  Each entry point below replaces one of
 * those launches with a plain-pointer call, so a host binding (ctypes, a torch
 * extension, C++) can drive the HIP kernels without any torch type crossing the
 * boundary.
 *
 * Conventions shared by every entry point:
 *   - Pointers are device pointers (HBM).  Sizes are element counts.
 *   - `stream` is a hipStream_t passed as void* (NULL = the legacy default
 *     stream).  Work is enqueued on that stream only: no allocation, no host
 *     synchronisation, no memset, so every call may be recorded into a HIP
 *     graph.
 *   - The return value is MI355_OK (0) or a negative MI355_ERR_* code; the
 *     message for the most recent failure on the calling thread is returned by
 *     mi355_last_error().  Nothing throws across the ABI.
 *   - Calls are reentrant; the library holds no locks.  A call only reads its
 *     inputs and writes its outputs; outputs must not overlap inputs unless
 *     the pointers are identical and the strides match (in-place use).
 */
#ifndef MI355_FUSED_H
#define MI355_FUSED_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MI355_ABI_VERSION 1

/* Element types understood by the kernels (storage type; arithmetic is fp32). */
enum mi355_dtype {
  MI355_F32 = 0,
  MI355_F16 = 1,
  MI355_BF16 = 2
};

/* Status codes. */
enum mi355_status {
  MI355_OK = 0,
  MI355_ERR_INVALID = -1,     /* bad pointer, size, stride or dtype code */
  MI355_ERR_UNSUPPORTED = -2, /* valid request the library cannot serve */
  MI355_ERR_HIP = -3          /* the HIP runtime reported an error */
};

/* Version of this ABI; callers check it equals MI355_ABI_VERSION. */
int mi355_abi_version(void);

/* Message describing the last failure on the calling thread ("" if none). */
const char* mi355_last_error(void);

/*
 * RMSNorm over the last dimension, one row at a time:
 *   var_r  = (sum_j x[r,j]^2) / n            (fp32 accumulation)
 *   rstd_r = 1 / sqrt(var_r + eps)
 *   y[r,j] = (x[r,j] * rstd_r) * w[j]        (fp32, rounded once to y_dtype)
 *
 * Replaces the launch of `_rmsnorm_fwd_kernel` in the reference's
 * `fused_rmsnorm` (src/kernels/fused_rmsnorm_triton.py:52-71, kernel body
 * :23-49).  The reference's launcher reuses x's row stride for the output
 * (:66-68) and makes x contiguous first (:60); here both row strides are
 * explicit, so a row-strided view needs no copy.
 *
 *   x       [rows, x_row_stride] elements of x_dtype; row r starts at
 *           x + r * x_row_stride and its n elements are contiguous.
 *   weight  [n] elements of w_dtype, contiguous.
 *   y       [rows, y_row_stride] elements of y_dtype.
 *   rows    >= 0 (0 is a no-op), n >= 1, both row strides >= n.
 *   y_dtype must equal x_dtype or be MI355_F32 (the fp32 value before the
 *   final rounding, used to check the kernel's arithmetic on its own).
 */
int mi355_rmsnorm_fwd(const void* x, const void* weight, void* y,
                      int64_t rows, int64_t n,
                      int64_t x_row_stride, int64_t y_row_stride,
                      float eps,
                      int x_dtype, int w_dtype, int y_dtype,
                      void* stream);

/*
 * Residual add fused with RMSNorm, per row:
 *   h[r,j]            = x[r,j] + residual[r,j]   (fp32 add, rounded to x_dtype)
 *   residual_out[r,j] = h[r,j]
 *   y[r,j]            = RMSNorm(h)[r,j]          (as mi355_rmsnorm_fwd)
 *
 * The reference has no kernel for this; it is the "fused RMSNorm + residual"
 * its design plans (docs/architecture-cuda.md:94) for the decoder's
 * `hidden = residual + attn_out; normed = post_attention_layernorm(hidden)`
 * (the HF Qwen2 decoder layer, and src/engine/paged_engine.py:138-141).  h is
 * rounded exactly where the unfused add rounds it, so the results equal the
 * add followed by mi355_rmsnorm_fwd bit for bit, in one pass over the rows:
 * read x and residual, write residual_out and y.
 *
 *   x, residual, residual_out: x_dtype, [rows, *_row_stride], rows contiguous.
 *   weight [n] of w_dtype; y [rows, y_row_stride] of y_dtype (x_dtype or fp32).
 *   residual_out may be residual and y may be x (in place, same strides);
 *   y must not overlap residual or residual_out.
 */
int mi355_add_rmsnorm_fwd(const void* x, const void* residual, const void* weight,
                          void* y, void* residual_out,
                          int64_t rows, int64_t n,
                          int64_t x_row_stride, int64_t residual_row_stride,
                          int64_t y_row_stride, int64_t residual_out_row_stride,
                          float eps,
                          int x_dtype, int w_dtype, int y_dtype,
                          void* stream);

/*
 * SiLU-and-mul, the activation step of a SwiGLU MLP, over flat memory:
 *   out[i] = (g * sigmoid(g)) * u,  g = gate[i], u = up[i]   (fp32, rounded once)
 *
 * Replaces the launch of `_silu_mul_fwd_kernel` in the reference's
 * `fused_silu_mul` (src/kernels/fused_swiglu_triton.py:39-53, kernel body
 * :20-36).  gate, up and out are `numel` contiguous elements; gate and up
 * share in_dtype; out_dtype must equal in_dtype or be MI355_F32.
 */
int mi355_silu_mul_fwd(const void* gate, const void* up, void* out,
                       int64_t numel, int in_dtype, int out_dtype,
                       void* stream);

/*
 * Gate/up projections fused with SiLU-and-mul, for decode-sized batches:
 *   g[m,n]   = sum_k x[m,k] * w_gate[n,k]     (fp32 accumulation, MFMA)
 *   u[m,n]   = sum_k x[m,k] * w_up[n,k]
 *   out[m,n] = (g * sigmoid(g)) * u           (fp32, rounded once to out_dtype)
 *
 * The reference's FusedMLP (src/engine/fused_norm_activation_patch.py:60-64)
 * computes `fused_silu_mul(gate_proj(x), up_proj(x))`: two GEMMs whose
 * results are rounded to x's dtype, written to HBM and read back by the
 * SiLU-and-mul launch this call also replaces (src/kernels/
 * fused_swiglu_triton.py:39-53).  This entry point is the "fused activation
 * with the up/gate projections" its design plans (docs/architecture-cuda.md:94):
 * g and u never leave registers and are not rounded before the activation,
 * so results differ from the unfused chain by that intermediate rounding
 * (they are closer to the exact value).  Weights use nn.Linear's layout,
 * [n_out, k] row-major, as in HF's gate_proj / up_proj.
 *
 * rows <= 32 stream the weights once at HBM bandwidth; more rows run an
 * LDS-tiled MFMA GEMM over both weight matrices with SiLU-and-mul in its
 * epilogue (32-row weight-streaming tiles when a row stride is too large for
 * the tiled kernel's buffer descriptors).
 *
 *   x        [rows, x_row_stride] of dtype, 16-byte aligned.
 *   w_gate, w_up  [n_out, w_row_stride] of dtype, 16-byte aligned.
 *   out      [rows, out_row_stride] of out_dtype.
 *   dtype    MI355_F16 or MI355_BF16; out_dtype = dtype or MI355_F32.
 *   k, x_row_stride and w_row_stride are multiples of 8 (MI355_ERR_UNSUPPORTED
 *   otherwise); strides >= k (x, w) and >= n_out (out).  rows == 0 or
 *   n_out == 0 is a no-op.  Limits: x_row_stride and w_row_stride < 2^24,
 *   rows <= 2097120.  out must not overlap the inputs.
 */
int mi355_gate_up_silu_fwd(const void* x, const void* w_gate, const void* w_up, void* out,
                           int64_t rows, int64_t k, int64_t n_out,
                           int64_t x_row_stride, int64_t w_row_stride, int64_t out_row_stride,
                           int dtype, int out_dtype,
                           void* stream);

/*
 * Weight-only int8 linear (W8A16), per output feature n and row m:
 *   acc[m,n] = sum_k x[m,k] * w_q[n,k]           (fp32 accumulation; int8 and
 *                                                 16-bit x meet exactly in fp16/bf16)
 *   out[m,n] = acc[m,n] * scale[n] + bias[n]     (one fma in fp32, rounded once)
 *
 * Replaces the launch of `_w8a16_matmul_kernel` in the reference's
 * `w8a16_linear` (src/kernels/w8a16_matmul_triton.py:102-134, kernel body
 * :39-86), which QuantizedLinearInt8.forward calls (src/quantization/
 * int8.py:62-63).  The scale is applied once to the accumulator, as there.
 *
 *   x       [rows, x_row_stride] of x_dtype (MI355_F16 or MI355_BF16).
 *   w_q     [n, w_row_stride] int8, nn.Linear's layout (out_features rows).
 *   scale   [n] of scale_dtype (the reference's float32; fp16/bf16 accepted).
 *   bias    [n] of bias_dtype, or NULL (then bias_dtype is ignored).
 *   out     [rows, out_row_stride] of out_dtype = x_dtype or MI355_F32.
 *   rows >= 0, k >= 1, n >= 0 (rows == 0 or n == 0 is a no-op); strides >= k
 *   (x, w_q) and >= n (out).  Any alignment and k are served; the fast kernels
 *   need k and w_row_stride multiples of 16, x_row_stride a multiple of 8 and
 *   16-byte aligned x and w_q.  Limits: x_row_stride < 2^23, w_row_stride <
 *   2^24, n < 2^31 - 128, rows <= 4194240.  out must not overlap the inputs.
 *   Calls with the same shapes give identical bits (fixed summation order).
 */
int mi355_w8a16_linear_fwd(const void* x, const void* w_q, const void* scale, const void* bias, void* out,
                           int64_t rows, int64_t k, int64_t n,
                           int64_t x_row_stride, int64_t w_row_stride, int64_t out_row_stride,
                           int x_dtype, int scale_dtype, int bias_dtype, int out_dtype,
                           void* stream);

/*
 * The same with a workspace, which lets calls of 17 to about 1500 rows whose
 * output holds too few tiles for the CUs split K (two kernels, no allocation).
 * mi355_w8a16_linear_workspace returns the bytes such a call wants on the
 * current device, 0 where it would not use them; `workspace` is 16-byte
 * aligned device memory of `workspace_bytes` that no other work touches until
 * the call's kernels end (its contents need no preparation and are left
 * undefined).  NULL, or fewer bytes than wanted, runs mi355_w8a16_linear_fwd.
 */
int64_t mi355_w8a16_linear_workspace(int64_t rows, int64_t k, int64_t n);
int mi355_w8a16_linear_ws_fwd(const void* x, const void* w_q, const void* scale, const void* bias, void* out,
                              int64_t rows, int64_t k, int64_t n,
                              int64_t x_row_stride, int64_t w_row_stride, int64_t out_row_stride,
                              int x_dtype, int scale_dtype, int bias_dtype, int out_dtype,
                              void* workspace, int64_t workspace_bytes,
                              void* stream);

/*
 * Int8 gate/up projections fused with SiLU-and-mul (W8A16 weights), per row
 * m and output feature n:
 *   g[m,n] = (sum_k x[m,k] * wq_gate[n,k]) * scale_gate[n]     (fp32 sums)
 *   u[m,n] = (sum_k x[m,k] * wq_up[n,k])   * scale_up[n]
 *   out[m,n] = round(g * sigmoid(g) * u)                       (fp32, one rounding)
 *
 * No counterpart in the reference: its quantised model runs
 * QuantizedLinearInt8 gate_proj and up_proj (two `w8a16_linear` launches,
 * src/quantization/int8.py:62-63, each rounding to x's dtype) and then the
 * SiLU-and-mul kernel (src/engine/fused_norm_activation_patch.py:60-64).
 * This entry point is that chain as one kernel, without the intermediate
 * roundings -- the int8 form of mi355_gate_up_silu_fwd.  Decode rows (<= 32)
 * stream both int8 matrices once at HBM bandwidth; more rows run the tiled
 * MFMA GEMM.
 *
 *   x        [rows, x_row_stride] of x_dtype (MI355_F16 or MI355_BF16).
 *   wq_gate, wq_up  [n_out, w_row_stride] int8 (QuantizedLinearInt8.weight_q).
 *   scale_gate, scale_up  [n_out] of scale_dtype (the quantiser's fp32).
 *   out      [rows, out_row_stride] of out_dtype = x_dtype or MI355_F32.
 *   Same shape rules, alignment preferences and limits as
 *   mi355_w8a16_linear_fwd (any k and alignment are served; no bias).
 */
int mi355_gate_up_silu_w8a16_fwd(const void* x, const void* wq_gate, const void* wq_up,
                                 const void* scale_gate, const void* scale_up, void* out,
                                 int64_t rows, int64_t k, int64_t n_out,
                                 int64_t x_row_stride, int64_t w_row_stride, int64_t out_row_stride,
                                 int x_dtype, int scale_dtype, int out_dtype,
                                 void* stream);

/*
 * Per-output-channel symmetric int8 quantisation of a weight matrix, per row n:
 *   amax     = max_k |w[n,k]|
 *   scale[n] = max(amax / 127, 1e-8)                     (fp32, IEEE division)
 *   w_q[n,k] = clamp(round_half_even(w[n,k] / scale[n]), -127, 127)
 *
 * The arithmetic of the reference's QuantizedLinearInt8.from_linear
 * (src/quantization/int8.py:45-50), bit for bit: w is widened to fp32
 * (`linear.weight.detach().float()`), the scale is clamped below at 1e-8 and
 * the quotient rounded with torch.round's ties-to-even.
 *
 *   w      [n, w_row_stride] of w_dtype (fp32, fp16 or bf16).
 *   w_q    [n, q_row_stride] int8 (output).   scale  [n] fp32 (output).
 *   n >= 0 (0 is a no-op), 1 <= k < 2^31, strides >= k.  Rows holding NaN or
 *   Inf get unspecified codes (the reference's are undefined there too).
 */
int mi355_quantize_int8_fwd(const void* w, void* w_q, void* scale,
                            int64_t n, int64_t k, int64_t w_row_stride, int64_t q_row_stride,
                            int w_dtype, void* stream);

/*
 * 16-bit linear (nn.Linear's forward with fp16 / bf16 weights), per row m
 * and output feature n:
 *   acc[m,n] = sum_k x[m,k] * weight[n,k]     (fp32 accumulation, MFMA)
 *   out[m,n] = acc[m,n] + bias[n]             (fp32, rounded once to out_dtype)
 *
 * Replaces the down projection of the reference's FusedMLP,
 * `self.down_proj(activated)` (src/engine/fused_norm_activation_patch.py:64),
 * an nn.Linear that torch runs on hipBLASLt.  At decode batch sizes that call
 * streams the whole weight matrix for a few rows; rows <= 32 here (64 on
 * outputs narrower than 128 64-column tiles) read every weight byte once at
 * HBM bandwidth on MFMA.  More rows run the LDS-tiled MFMA GEMM.  The fp32 sums
 * run in this library's own order, so results may differ from hipBLASLt's
 * in the last output bit.
 *
 *   x       [rows, x_row_stride] of dtype (MI355_F16 or MI355_BF16).
 *   weight  [n, w_row_stride] of dtype, nn.Linear's layout.
 *   bias    [n] of bias_dtype, or NULL (then bias_dtype is ignored).
 *   out     [rows, out_row_stride] of out_dtype = dtype or MI355_F32.
 *   rows >= 0, k >= 1, n >= 0 (rows == 0 or n == 0 is a no-op); strides >= k
 *   (x, weight) and >= n (out).  Any alignment and k are served; the fast
 *   kernels need k and both input row strides multiples of 8 and 16-byte
 *   aligned x and weight.  Limits: x_row_stride and w_row_stride < 2^22,
 *   n < 2^31 - 256, rows <= 2097120.  out must not overlap the inputs.
 *   Calls with the same shapes give identical bits (fixed summation order).
 */
int mi355_linear16_fwd(const void* x, const void* weight, const void* bias, void* out,
                       int64_t rows, int64_t k, int64_t n,
                       int64_t x_row_stride, int64_t w_row_stride, int64_t out_row_stride,
                       int dtype, int bias_dtype, int out_dtype,
                       void* stream);

/* The same with a workspace: the rules of mi355_w8a16_linear_ws_fwd. */
int64_t mi355_linear16_workspace(int64_t rows, int64_t k, int64_t n);
int mi355_linear16_ws_fwd(const void* x, const void* weight, const void* bias, void* out,
                          int64_t rows, int64_t k, int64_t n,
                          int64_t x_row_stride, int64_t w_row_stride, int64_t out_row_stride,
                          int dtype, int bias_dtype, int out_dtype,
                          void* workspace, int64_t workspace_bytes,
                          void* stream);

/*
 * Rotary positions of x [batch, tokens, heads, head_dim].  With R = rotary_dim
 * and, for token (b, t) and pair j < R / 2,
 *   a = positions[b, t] * inv_freq[j],  c = scale cos a,  s = scale sin a:
 *   y0 = x0 c - x1 s,  y1 = x1 c + x0 s         (fp32, rounded once)
 * for the pairs (x[j], x[j + R / 2]) (interleaved = 0, the layout of Qwen2 and
 * Llama) or (x[2j], x[2j + 1]) (interleaved = 1); elements from R on are
 * copied.  Angles are formed and reduced in 64 bits, so far positions lose
 * nothing.  Longer contexts are a matter of inv_freq and scale.
 *
 *   x          dtype (fp32, fp16, bf16); strides in elements, head_dim
 *              contiguous; any strides >= 0 and any alignment.
 *   y          [batch, tokens, heads, head_dim] of dtype, contiguous; must not
 *              overlap x.
 *   positions  int64 by two strides (0 for one row of positions for all).
 *   inv_freq   fp32 [R / 2]; R even, 0 <= R <= head_dim, R <= 256.  With R = 0
 *              neither is read, and both may be NULL.
 *   batch * tokens < 2^24, heads <= 65535, head_dim < 2^20
 *   (MI355_ERR_UNSUPPORTED beyond).  Nothing to do for 0 elements.
 */
int mi355_rotary_fwd(const void* x, void* y, const int64_t* positions, const float* inv_freq,
                     int64_t batch, int64_t tokens, int64_t heads, int64_t head_dim, int64_t rotary_dim,
                     int64_t x_stride_b, int64_t x_stride_t, int64_t x_stride_h,
                     int64_t pos_stride_b, int64_t pos_stride_t,
                     float scale, int interleaved, int dtype, void* stream);

/* Element formats of a key/value cache. */
enum mi355_kv_format {
  MI355_KV_16BIT = 0, /* values of the call's dtype, no scales */
  MI355_KV_INT8 = 1,  /* int8 codes with a scale per token and head: value = code * scale */
  MI355_KV_E4M3 = 2   /* 8-bit floats (4 exponent, 3 mantissa bits, largest 448), likewise */
};

/*
 * A paged key/value cache.  The token in slot s of sequence b lies on page
 * page_table[b * table_stride + s / page_size] at place s % page_size.  One
 * page per sequence makes a static cache.  The library keeps nothing of the
 * struct after a call.
 *
 * page_table and the lengths that calls take are device memory: their values
 * are checked by the kernels.  A slot beyond the table, or on a page number
 * outside [0, pages), has no place: it is not written, reads as zero and is
 * not attended to.  A slot that two sequences share is theirs to keep whole.
 */
typedef struct mi355_kv_cache {
  void* k;                   /* [pages, kv_heads, page_size, head_dim], contiguous, 16-byte aligned */
  void* v;                   /* the same */
  float* k_scale;            /* [pages, kv_heads, page_size], 16-byte aligned; NULL for 16-bit values */
  float* v_scale;            /* the same */
  const int32_t* page_table; /* [batch, table_stride], table_width of them in use */
  int64_t table_stride;
  int64_t table_width;       /* table_width * page_size < 2^30 */
  int64_t pages;             /* < 2^31 */
  int64_t kv_heads;          /* 1 .. 65535 */
  int64_t page_size;         /* a multiple of 16 */
  int64_t head_dim;          /* a multiple of 16, at most 256 */
  int format;                /* enum mi355_kv_format */
} mi355_kv_cache;

/*
 * Writes the keys and values of `tokens` new tokens per sequence into slots
 * seq_lens[b] + t, rotating the keys (and queries, if given) on the way:
 *   kr = rotary(k) (as mi355_rotary_fwd, kept in fp32)
 *   scale = max(max|row| / top, 1e-8), code = round(row / scale)   per token and head,
 * top = 127 (int8, ties to even) or 448 (e4m3); 16-bit caches round once.  A
 * row that holds an infinity or a NaN reads back as NaN.  Tokens from
 * new_lens[b] on (NULL: none) are padding and not written; their queries are
 * rotated all the same.
 *
 *   k, v      [batch, tokens, kv_heads, head_dim] of dtype (fp16, bf16) by
 *             three strides each (strides[0..2] of k: batch, token, head;
 *             [3..5] of v; [6..8] of q), head_dim contiguous, rows 16-byte
 *             aligned.
 *   q, q_out  [batch, tokens, q_heads, head_dim] likewise, q_out contiguous;
 *             both NULL (q_heads = 0) to rotate no queries.
 *   inv_freq  NULL (rotary_dim = 0): nothing is rotated, positions is not read.
 *   batch * tokens < 2^24, q_heads + 2 kv_heads <= 65535.
 */
int mi355_kv_cache_append_fwd(const mi355_kv_cache* cache, const void* k, const void* v, const void* q, void* q_out,
                              const int32_t* seq_lens, const int32_t* new_lens,
                              const int64_t* positions, const float* inv_freq,
                              int64_t batch, int64_t tokens, int64_t q_heads, int64_t rotary_dim,
                              const int64_t* strides, int64_t pos_stride_b, int64_t pos_stride_t,
                              float scale, int interleaved, int dtype, void* stream);

/*
 * Reads slots start[b] + i, i < tokens, as values of dtype (code * scale,
 * rounded once) into k_out, v_out [batch, kv_heads, tokens, head_dim]
 * (contiguous, 16-byte aligned); zeros from slot end[b] on.  start may be NULL (0).
 * batch * tokens * kv_heads < 2^26.
 */
int mi355_kv_cache_read_fwd(const mi355_kv_cache* cache, void* k_out, void* v_out,
                            const int32_t* start, const int32_t* end, int64_t batch, int64_t tokens,
                            int dtype, void* stream);

/*
 * Moves kept tokens together: slot seq_lens[b] + i becomes what slot
 * seq_lens[b] + kept[b, i] held before the call, for i < kept_lens[b] (NULL:
 * max_kept) -- the accepted path of a tree of drafted tokens, in any order and
 * with repeats.  Codes and scales are moved as they are.  A negative kept[b, i]
 * or a slot without a place leaves its destination as it was.
 *   kept int32 [batch, kept_stride], max_kept <= 128.
 */
int mi355_kv_cache_keep_fwd(const mi355_kv_cache* cache, const int32_t* seq_lens, const int32_t* kept,
                            const int32_t* kept_lens, int64_t batch, int64_t max_kept, int64_t kept_stride,
                            void* stream);

/*
 * Attention of `tokens` new tokens per sequence over the cache, which holds
 * them already in slots seq_lens[b] + t (mi355_kv_cache_append_fwd).  Query
 * head h reads key/value head h / (q_heads / kv_heads).  Token t sees every
 * slot below seq_lens[b] and the new token j iff tree_mask[b, t, j] != 0
 * (NULL: j <= t, a chain):
 *   S[s] = scale * q . K[s],  out = sum_s exp(S[s]) V[s] / sum_s exp(S[s])
 * over the slots it sees, with fp32 sums and one rounding.  What it does not
 * see has no influence, NaN and infinities included.  An infinite 16-bit value
 * that it sees makes its element infinite, however small its weight; a NaN, or
 * both infinities, NaN; a value whose scale is not finite, all of them NaN.
 * A token that sees nothing, and padding (t >= new_lens[b]; NULL: none), gets
 * zeros, as does one whose scores are all -infinity.
 *
 *   q     [batch, tokens, q_heads, head_dim] of dtype (fp16, bf16) by three
 *         strides (batch, token, head), head_dim contiguous, rows 16-byte
 *         aligned.   out: the same shape, contiguous, 16-byte aligned.
 *   tree_mask  bytes [batch, tokens, tokens] by mask_stride_b (0: one tree for
 *         all sequences) and mask_stride_t; the last dimension contiguous.
 *   tokens <= 128, q_heads a multiple of kv_heads and at most 65535,
 *   batch * tokens * q_heads < 2^24 (MI355_ERR_UNSUPPORTED beyond).
 *
 * The cache is split over workgroups where sequences are few or long, and
 * joined by a second kernel.  mi355_tree_attention_workspace returns the bytes
 * that this wants on the current device; `workspace` is 16-byte aligned device
 * memory that no other work touches until the call's kernels end (its contents
 * need no preparation).  NULL or less of it: each sequence and head is one
 * workgroup's work.  Equal arguments give equal bits.
 */
int64_t mi355_tree_attention_workspace(const mi355_kv_cache* cache, int64_t batch, int64_t tokens, int64_t q_heads);
int mi355_tree_attention_fwd(const mi355_kv_cache* cache, const void* q, void* out,
                             const int32_t* seq_lens, const int32_t* new_lens,
                             const uint8_t* tree_mask, int64_t mask_stride_b, int64_t mask_stride_t,
                             int64_t batch, int64_t tokens, int64_t q_heads, const int64_t* q_strides,
                             float scale, int dtype, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * Attention as mi355_tree_attention_fwd computes it, for a batch whose
 * sequences share prefixes.  Sequence b is a member of group g if groups[g] <=
 * b < groups[g + 1] (groups int32 [group_count + 1], ascending; NULL: groups of
 * batch / group_count sequences each), and the slots below
 *   shared_b = min(prefix_lens[g], seq_lens[b])
 * are those that the page table names for the group's first sequence: they are
 * read once for all members, whose own entries for them are not looked at.  From
 * shared_b on a sequence's slots are its own.  A sequence of no group shares
 * nothing; group_count 0 is allowed.  Group boundaries are clamped to
 * [0, batch]; of descending ones, the first group that fits is taken.
 *
 * The other arguments, limits and rules (masks, padding, infinities) are those
 * of mi355_tree_attention_fwd.  Without a workspace of the size asked for, a wave
 * computes each query row by itself: right, and slow.
 */
int64_t mi355_shared_prefix_attention_workspace(const mi355_kv_cache* cache, int64_t batch, int64_t tokens,
                                                int64_t q_heads, int64_t group_count);
int mi355_shared_prefix_attention_fwd(const mi355_kv_cache* cache, const void* q, void* out,
                                      const int32_t* seq_lens, const int32_t* new_lens,
                                      const int32_t* prefix_lens, const int32_t* groups, int64_t group_count,
                                      const uint8_t* tree_mask, int64_t mask_stride_b, int64_t mask_stride_t,
                                      int64_t batch, int64_t tokens, int64_t q_heads, const int64_t* q_strides,
                                      float scale, int dtype, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * A page table in which every sequence has pages for its slots below
 * end_b = max(0, seq_lens[b]) + max(0, new_lens[b]) (new_lens NULL: 0):
 *   need_b = ceil(end_b / page_size)
 *   table_out[b, c] = page_table[b, c]  for c < need_b, where that names a page
 *                   = a free page       for other c < need_b
 *                   = -1                for c >= need_b
 * Free are the pages that no entry of the first kind names: several sequences
 * may name one page, and a page is free when none of them needs it any more
 * (a sequence that ended has length 0).  Free pages are handed out in ascending
 * order, to entries in the order of b, then c; when there are no more, -1.
 * missing[b]: pages of need_b that sequence b did not get, those beyond the
 * table's width among them.  The table is the only state.
 *
 *   Of the cache page_table, its sizes, pages and page_size are read; k, v and
 *   scales may be NULL.  table_out int32 [batch, out_stride], out_stride >=
 *   table_width: the cache's own table (with its stride), or memory that does
 *   not overlap it.  missing int32 [batch].  batch < 2^24, batch * table_width
 *   < 2^31, pages < 2^30 (MI355_ERR_UNSUPPORTED beyond).
 *   workspace: at least mi355_kv_cache_reserve_workspace bytes of 16-byte
 *   aligned device memory that no other work touches until the call's kernels
 *   end (its contents need no preparation).
 */
int64_t mi355_kv_cache_reserve_workspace(const mi355_kv_cache* cache, int64_t batch);
int mi355_kv_cache_reserve_fwd(const mi355_kv_cache* cache, const int32_t* seq_lens, const int32_t* new_lens,
                               int32_t* table_out, int64_t out_stride, int32_t* missing, int64_t batch,
                               void* workspace, int64_t workspace_bytes, void* stream);

/*
 * Where the tokens of a packed batch go: new_lens[0] tokens of sequence 0, then
 * new_lens[1] of sequence 1, ... (negative: 0).  For packed token j, token t of
 * sequence b:
 *   sequences[j] = b,  positions[j] = max(0, seq_lens[b]) + t
 *   slots[j] = page * page_size + positions[j] % page_size with the page that
 *              page_table names for the position, -1 where it names none
 * Rows from the number of tokens on get slot -1, sequence -1 and position 0.
 *
 *   slots, positions int64 [tokens]; sequences int32 [tokens].  batch < 2^24,
 *   tokens < 2^31 (MI355_ERR_UNSUPPORTED beyond).  Of the cache page_table, its
 *   sizes, pages and page_size are read.  workspace: as for
 *   mi355_kv_cache_reserve_fwd, of mi355_kv_slot_map_workspace bytes.
 */
int64_t mi355_kv_slot_map_workspace(int64_t batch);
int mi355_kv_slot_map_fwd(const mi355_kv_cache* cache, const int32_t* seq_lens, const int32_t* new_lens,
                          int64_t* slots, int32_t* sequences, int64_t* positions, int64_t batch, int64_t tokens,
                          void* workspace, int64_t workspace_bytes, void* stream);

/*
 * Draws a token per row of logits x from the distribution that temperature,
 * top-k, top-p and min-p leave, with one given uniform number u per row.
 * With M the largest logit, w_i = exp((x_i - M) / temperature) and tokens ranked
 * by x (equal ones by index), a token is kept if all of these hold:
 *   its rank is below top_k                               (top_k <= 0: no limit)
 *   the tokens ranked before it have less than top_p of
 *   the weight of those that top_k keeps                  (top_p >= 1: no limit)
 *   w_i >= min_p                                          (min_p <= 0: no limit)
 * (the first is always kept, alone if min_p > 1).  tokens[r] is the first i, in
 * the order of the vocabulary, up to which the kept weights sum to more than u
 * times their total; logprobs[r] (NULL: not wanted) the logarithm of w_i / total,
 * as which it was drawn.  temperature <= 0 (or NaN): the first token of rank 0,
 * logarithm 0.  u is clamped to [0, 1 - 2^-24], NaN to 0.  -infinity and NaN have
 * weight 0; where the largest logit is +infinity, those that are have weight 1 and
 * others 0.  A row without any other logit than -infinity and NaN gets token -1
 * and logarithm -infinity.  Weights and sums are of 64 bits.
 *
 *   logits      [rows, row_stride] of dtype (fp32, fp16, bf16), vocab elements
 *               of each row contiguous, any alignment.  vocab < 2^20.
 *   uniform     fp32 [rows].   tokens int64 [rows].   logprobs fp32 [rows].
 *   temperature, top_p, min_p (fp32 [rows]) and top_k (int32 [rows]): a setting
 *               per row, or NULL: the *_all value for every row.
 *   rows < 2^20, row_stride >= vocab.  workspace: as for
 *   mi355_kv_cache_reserve_fwd, of mi355_sample_tokens_workspace bytes.
 */
int64_t mi355_sample_tokens_workspace(int64_t rows, int64_t vocab);
int mi355_sample_tokens_fwd(const void* logits, const float* uniform, int64_t* tokens, float* logprobs,
                            const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                            float temperature_all, int32_t top_k_all, float top_p_all, float min_p_all,
                            int64_t rows, int64_t vocab, int64_t row_stride, int dtype,
                            void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MI355_FUSED_H */
