/*
 * kino_q8.h - 8-bit serving entry points of libkino_b200.so (conventions of kino.h: caller-owned
 * device pointers, no allocation, asynchronous on `stream`, a kino_status from every call).
 *
 * Values are held as 8-bit codes times an fp32 scale for a group: a token's row, a weight's output
 * channel, or the tokens of one cache block and head. With top = 127 (KINO_Q8_INT8) or 448
 * (KINO_Q8_E4M3): scale = amax / top, code = x * top / amax to the nearest code, ties to even. A
 * group whose scale would be below 2^-126 is zeros with scale 0; one with an infinity or a NaN
 * gets the scale NaN and codes 0 and reads back as NaN. The NaN pattern of e4m3 is never written and not expected.
 *
 * Sizes that the host cannot see (lengths, token starts, block tables) are checked by the kernels:
 * what does not fit is skipped, nothing out of range is touched, and kino_device_status() then
 * returns KINO_EINVAL.
 *
 * These operators have no counterpart in the reference, whose weights are packed and whose
 * activations and caches stay in bf16.
 */
#ifndef KINO_Q8_H
#define KINO_Q8_H

#include "kino.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ABI version of this header (1); bumped on any signature change or addition. */
int kino_q8_abi_version(void);

#define KINO_Q8_INT8 0
#define KINO_Q8_E4M3 1

/* Codes and scales of token rows, with an optional residual addition and RMS norm in front:
 *   h = residual ? bf16(x + residual) : x                       (stored to `hidden` if given)
 *   y = norm ? h * rsqrt(mean(h^2) + eps) * (weight + weight_offset) : h      (fp32)
 *   scales[row], codes[row, :] = quantised y[row, :]
 * x, residual, hidden: rows x dim bf16 at their own row strides (multiples of 8, 16-byte aligned);
 * hidden may be x or residual. weight: [dim] bf16 or NULL (then no weight and no offset). codes:
 * contiguous rows x dim bytes, 8-byte aligned; scales: [rows] fp32. dim % 8 == 0, dim <= 131072.
 * Row strides are not looked at where there is one row. Rows whose squares or weighted values leave
 * fp32's range are normed in 64 bits, and a row of zeros has scale 0 whatever eps is. */
kino_status kino_q8_rows(const void* x, int64_t ldx, const void* residual, int64_t ld_residual,
                         const void* weight, float weight_offset, float eps, int norm,
                         void* hidden, int64_t ld_hidden, void* codes, float* scales, int format,
                         int64_t rows, int64_t dim, void* stream);

/* out[i, j] = bf16(float(sum_k x[i, k] * w[j, k]) * x_scales[i] * w_scales[j] + bias[j]): int8
 * codes, the sum exact in int32 (k < 131072). x: m x k at row stride ldx, w: n x k at ldw (bytes,
 * multiples of 16, 16-byte aligned), out: bf16 m x n at ldo (a multiple of 8). k % 16 == 0,
 * n % 8 == 0. bias: [n] bf16 or NULL; scales and bias 16-byte aligned. */
kino_status kino_q8_linear(const void* x, int64_t ldx, const float* x_scales, const void* w,
                           int64_t ldw, const float* w_scales, const void* bias, void* out,
                           int64_t ldo, int64_t m, int64_t n, int64_t k, void* stream);

/* A K/V cache held in blocks: codes (num_blocks, heads, block, dim) contiguous bytes, 16-byte
 * aligned; scales (num_blocks, heads) fp32. heads <= 65535; dim 64 or 128; block 16, 32, 64 or
 * 128 tokens. Token t of sequence b is slot t % block of cache block
 * table[b * ld_table + t / block]. */
typedef struct kino_q8_cache {
  void* k_codes;
  void* v_codes;
  float* k_scales;
  float* v_scales;
  int64_t num_blocks;
  int64_t heads;
  int64_t dim;
  int64_t block;
  int format;              /* KINO_Q8_* */
  const int32_t* table;    /* device (batch, table_blocks) at row stride ld_table */
  int64_t ld_table;
  int64_t table_blocks;
  const int32_t* lengths;  /* device (batch): tokens held */
  int64_t batch;
} kino_q8_cache;

/* Quantises new tokens into the cache. k, v: (rows, heads, dim) bf16, row strides ld_k / ld_v and
 * head strides hs_k / hs_v in elements (multiples of 8, 16-byte aligned). Sequence b's tokens are
 * rows [token_starts[b], token_starts[b + 1]) (device, batch + 1 entries; rows behind the last
 * start are not read), or rows / batch each when token_starts is NULL; they take positions
 * lengths[b] on (cache->lengths is what was held before and is not changed). A block that already
 * holds tokens of the sequence keeps the larger of its scale and the new tokens'; where the scale
 * grows the earlier codes are rounded to it. Slots behind the new tokens stay as they were. A
 * cache block may be written for one sequence only in a call. */
kino_status kino_q8_cache_write(const kino_q8_cache* cache, const void* k, int64_t ld_k,
                                int64_t hs_k, const void* v, int64_t ld_v, int64_t hs_v,
                                const int32_t* token_starts, int64_t rows, void* stream);

/* k_out, v_out (batch, tokens, heads, dim) bf16 contiguous, 16-byte aligned: tokens [0, tokens) of
 * every sequence, bf16(code * scale), zeros from a sequence's length on. */
kino_status kino_q8_cache_read(const kino_q8_cache* cache, void* k_out, void* v_out,
                               int64_t tokens, void* stream);

typedef struct kino_q8_attention_args {
  const void* q;           /* (rows, q_heads, dim) bf16, row and head strides in elements */
  int64_t ld_q, hs_q;      /* (multiples of 8, 16-byte aligned) */
  void* out;               /* the same shape, bf16; may be q at the same strides */
  int64_t ld_out, hs_out;
  const int32_t* token_starts; /* device (batch + 1), or NULL: rows / batch rows a sequence */
  int64_t rows;
  int64_t q_heads;         /* a multiple of the cache's heads: group = q_heads / heads <= 128 */
  float scale;             /* softmax scale, positive or zero */
  int causal;
  void* workspace;         /* kino_q8_attention_workspace_size bytes, 16-byte aligned */
  int64_t workspace_bytes;
} kino_q8_attention_args;

/* Workspace bytes of kino_q8_attention (partial results of items that several CTAs share), which
 * depend on the shapes alone; -1 for invalid arguments. */
int64_t kino_q8_attention_workspace_size(const kino_q8_cache* cache,
                                         const kino_q8_attention_args* args);

/* softmax(q k^T * scale) v over a sequence's cached tokens [0, lengths[b]), query head h on cache
 * head h / group. The n query tokens of a sequence are its last n tokens: with `causal` query i
 * sees keys up to position lengths[b] - n + i. A query that sees no key gives zeros; one with an
 * infinity or a NaN gives NaN where it sees a key. Rows in front of the first start and behind the
 * last are not written, and nothing comes of their values. */
kino_status kino_q8_attention(const kino_q8_cache* cache, const kino_q8_attention_args* args,
                              void* stream);

#ifdef __cplusplus
}
#endif

#endif
