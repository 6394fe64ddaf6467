/*
 * pkh3_paged.h -- C ABI of libpkh3attn.so for a K/V cache in pages: keys and values of many sequences, of unequal length,
 * that grow as rows arrive, and the attention of new rows over them.
 *
 * The reference has no counterpart (its model attends within one packed document, src/pika_h3/core/wrapper.py:192-204, and
 * keeps nothing between two calls); the rows are those of its attention module all the same: QK-RMSNorm and rotation of
 * what `to_q/to_k/to_v` give (src/pika_h3/core/loader.py:9), head dim 128.
 *
 *   pkh3_paged_write            new keys (norm, rotation) and values into their sequences' pages, in bf16 or rounded to e4m3
 *   pkh3_paged_read             keys and values of the same rows back out of the pages
 *   pkh3_paged_attn             softmax(q k^T * scale) v of the new rows over all keys of their sequence
 *   pkh3_paged_workspace_bytes  scratch of pkh3_paged_attn
 *   pkh3_paged_record_bytes     what a page takes per key/value head
 *
 * Conventions (pointers, streams, errors) are those of pkh3_attn.h.
 *
 * The pool.  `pages` is [n_pages][kv_heads][pkh3_paged_record_bytes()]: a page holds 64 keys, per head a record of operand
 * images as the attention kernel reads them -- 16 KiB of K and 16 KiB of V, or with PKH3_PAGED_FP8 8 KiB each and 128 bytes
 * of scales.  A pool needs no clearing: what lies behind a sequence's last key is never part of a result, whatever it is.
 * With PKH3_PAGED_FP8 every key has two scales per head, one for K and one for V: the smallest power of two that is at least
 * max|x| / 448 (formed in float32, 2^-126 at least; 1 for a row of zeros), and x / scale is rounded to the nearest
 * e4m3 value.  (Stored values below 2^-126 may come back as 0.)  A row's values do not depend on the rows around it, so
 * what is written once stays as it is.  What is not finite is stored as NaN there, and as it is in bf16.  A NaN in a key makes
 * the results of the rows that see the key NaN; a value that is not finite reaches the results of those rows too and, under
 * PKH3_PAGED_CAUSAL, may reach those of rows of the same sequence and call in front of it (their weight of 0 times it is NaN).
 * Keys that the batch does not hold (behind a length, on a page that is not there) reach nothing, whatever their memory holds.
 *
 * The batch.  B sequences share the pool.  Sequence b owns the rows starts[b] .. starts[b+1]-1 of the call (n of them) and has
 * lengths[b] keys, those of the call's rows among them where they are written; its i-th row stands at position
 * lengths[b] - n + i.  Key j lies in page table[b * table_stride + j / 64], place j % 64.  The arrays live in device memory
 * and are read by the kernels only; what they hold is taken this way, and nothing else is touched whatever it is:
 *   - starts outside [0, rows] and lengths outside [0, 64 * table_pages] are brought there; a sequence that ends before it
 *     begins has no rows;
 *   - a table entry outside [0, n_pages) is a page that is not there: its keys are seen by nobody, writes to it are dropped,
 *     reads of it give zeros;
 *   - a row in front of position 0 (more new rows than keys) is not written, reads as zeros, and sees no key under
 *     PKH3_PAGED_CAUSAL (without it, it sees them all);
 *   - a row's place goes by starts and lengths as they are, so that none comes to another's: row r of the call stands at
 *     lengths[b] - starts[b+1] + r.  pkh3_paged_write writes the rows of the call whose place is in the table, and under PKH3_PAGED_CAUSAL a row sees what
 *     is stored up to its own place.  A sequence that has grown past its table loses the rows behind it and keeps what is stored.  (pkh3_paged_read
 *     alone goes by the values brought into range: of such a sequence it gives the last rows of the table.)
 * Rows that belong to no sequence are neither read nor written.  starts must not decrease, and no two places that one call
 * writes may be the same.
 */
#ifndef PKH3_PAGED_H
#define PKH3_PAGED_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define PKH3_PAGE_KEYS 64
#define PKH3_PAGED_MAX_SEQUENCES 1024

enum {
  PKH3_PAGED_FP8 = 1u << 0,   /* the pool holds e4m3 values with a scale per key, head and side */
  PKH3_PAGED_CAUSAL = 1u << 1 /* pkh3_paged_attn: a row sees the keys up to its own position, not all of its sequence */
};

typedef struct pkh3_paged_args {
  void* pages;             /* the pool, 256-byte aligned */
  int64_t n_pages;
  const int32_t* starts;   /* [B + 1] */
  const int32_t* lengths;  /* [B] */
  const int32_t* table;    /* [B][table_stride], table_pages entries of each used */
  int64_t table_stride;
  /* bf16 rows, [rows, heads, 128], addressed as base + row*ss + head*sh + d; 16-byte aligned, strides multiples of 8
     elements.  write: k and v in; read: k and v out, which must not overlap each other; attn: q in, o out (`o` may be `q`
     with q's strides, and must not overlap it otherwise).  What a call does not use is not looked at */
  const void* q;
  void* k;
  void* v;
  void* o;
  int64_t q_ss, q_sh, k_ss, k_sh, v_ss, v_sh, o_ss, o_sh;
  int32_t B, table_pages, rows, kv_heads;
  int32_t heads;           /* attn: query heads, a multiple of kv_heads; query head h reads the cache's head h / (heads / kv_heads) */
  int32_t D;
  float softmax_scale;     /* attn; <= 0 selects 1/sqrt(D) */
  float norm_eps;
  /* the rows that come in (write: k, attn: q): x * rsqrt(mean(x^2) + eps) * w (NULL: no norm), then the rotation by tables
     [rows, D/2], a row of them per row of the call */
  const float* norm_w;
  const float* rope_cos;
  const float* rope_sin;
  int32_t rope_mode;
  uint32_t flags;
  void* workspace;         /* attn: 256-byte aligned scratch.  Every call writes it before it reads it; calls that may overlap need one each */
  size_t workspace_bytes;
} pkh3_paged_args;

/* Bytes of one page of one kv head (0 on unknown flags; PKH3_PAGED_CAUSAL makes no difference). */
size_t pkh3_paged_record_bytes(uint32_t flags);

/* Keys and values of the call's rows into the pages.  Nothing else of the pool is written. */
int pkh3_paged_write(const pkh3_paged_args* a, void* stream);

/* Keys and values of the call's rows out of the pages, as the values they stand for. */
int pkh3_paged_read(const pkh3_paged_args* a, void* stream);

/* Scratch of pkh3_paged_attn for these sizes (B, table_pages, rows, heads, kv_heads) and flags, 0 on invalid ones; does not
   depend on what the batch's arrays hold.  103 MB are enough for any call. */
size_t pkh3_paged_workspace_bytes(const pkh3_paged_args* a);

/* Attention of the call's rows over their sequences' keys.  A row that sees no key gets zeros.  Results depend on the
   arguments and on what the batch's arrays hold, never on timing.  How the work is cut into blocks of rows goes by the sizes of the call (rows, B, heads,
   table_pages), for the whole of it: blocks of 16 rows keep what the rounding of q to bf16 after norm or rotation leaves, larger ones do not, and the
   rounded weights differ, so the last bits of a sequence's result may depend on the batch that it is in.  A chunk over a long context among many sequences
   without rows is slow: B is best the number of sequences that have some. */
int pkh3_paged_attn(const pkh3_paged_args* a, void* stream);

#ifdef __cplusplus
}
#endif
#endif
