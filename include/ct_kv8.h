/* ct_kv8.h -- 8-bit paged key/value cache: operators of libct_b200.so for hosts
 * that run their own decode loop.
 *
 * No counterpart in the reference, whose cache is a dense fp32 region
 * [B, MAX_SEQ, DEC_D] (backends/backend.h:214-217); backend_linear_to_kvcache_batch
 * and backend_sdp_attn_batch_decode_* of ct_backend.h write and read that one.
 * The operators here keep K and V in one byte per value with a scale for each
 * block of 16 token rows and head:
 *
 *   ct_kv8_append   projection rows -> 8-bit blocks of a sequence's pages
 *   ct_kv8_attn     attention of query rows over a sequence's pages, from one
 *                   row (decode) to whole prompts, optionally with a sliding
 *                   window and a few first tokens that stay visible
 *   ct_kv8_reserve, ct_kv8_fork, ct_kv8_free, ct_kv8_trim, ct_kv8_compact,
 *   ct_kv8_copy_pages   the pages: growing, sharing (beams), releasing,
 *                   releasing what a window has passed, defragmenting, copying
 *
 * Conventions.  Every pointer inside the structs and every array argument is
 * DEVICE memory of the current device; the structs themselves are host memory,
 * read during the call.  Calls launch on `stream` (a cudaStream_t, NULL = the
 * default stream), never synchronise and allocate nothing, so all of them may be
 * captured into a CUDA graph; scratch space is the caller's (`ws`, 256-byte
 * aligned, no particular contents, not shared by calls that may overlap).  The
 * calls need no backend_init.  Calls that change the same pages, tables, lengths
 * or refs must be ordered by the caller (one stream, or events).  They return CT_OK, CT_EINVAL (a bad argument;
 * nothing was launched), CT_ENOMEM (ws too small; nothing was launched) or
 * CT_EDEVICE (a CUDA call failed, or an error was already pending).  What only
 * the device can see (a page number outside the pool, a length beyond the
 * table, no free page left) makes the kernel leave that row, page or sequence
 * out and record a code in the device status word: ct_kv8_status.
 */
#ifndef CT_KV8_H
#define CT_KV8_H

#include <stddef.h>
#include <stdint.h>

#include "ct_engine.h"   /* CT_OK and the error codes */

#ifdef __cplusplus
extern "C" {
#endif

#define CT_KV8_ROWS 16        /* token rows of a page, and of a scale's block */

#define CT_KV8_E4M3 0         /* codes are E4M3 floats (largest 448) */
#define CT_KV8_INT8 1         /* codes are integers -127 .. 127 */

#define CT_KV8_F32 0          /* type of k / v, or of q and out */
#define CT_KV8_BF16 1

/* A pool of pages.  Page p holds CT_KV8_ROWS token rows of every layer:
 *   codes  [n_pages][n_layers][K, V][kv_heads][CT_KV8_ROWS][head_dim], 16-byte aligned
 *   scales [n_pages][n_layers][K, V][kv_heads], fp32
 * A value is code * scale of its block.  ct_kv8_append writes scales that are
 * powers of two; the attention takes any finite scale >= 0.  A scale of NaN
 * marks a block into which a NaN was written: all its values read as NaN.  The
 * E4M3 codes 0x7F and 0xFF (NaN) are not used: rows below a sequence's length
 * must not hold them, rows behind it may hold anything.
 *   refs   [n_pages]: how many sequences hold the page, 0 = free.  May be NULL
 * for ct_kv8_append and ct_kv8_attn, when the caller assigns pages itself.
 * head_dim is 64 or 128; n_layers and kv_heads are 4096 at most, and
 * n_pages * n_layers * kv_heads is below 2^30. */
typedef struct {
    uint8_t *codes;
    float *scales;
    int *refs;
    int n_pages, n_layers, kv_heads, head_dim;
    int format;               /* CT_KV8_E4M3 or CT_KV8_INT8 */
} ct_kv8_cache;

/* Sequences (at most 65535): row s of `table` lists the pages of sequence s in order
 * (token row t is row t % 16 of page table[s * table_stride + t / 16]); len[s]
 * is its number of token rows.  An entry of -1 is a page that was released. */
typedef struct {
    int *table;               /* [n_seqs][table_stride] */
    int *len;                 /* [n_seqs] */
    int n_seqs, table_stride;
} ct_kv8_seqs;

/* Write the K and V rows of this call into `layer`.
 * k, v: [n_rows][kv_heads * head_dim] of `type`, row strides ldk / ldv in
 * elements; 16-byte aligned, strides a multiple of 16 bytes.  Sequence s owns
 * rows row_start[s] .. row_start[s + 1] - 1, at most max_rows of them;
 * row_start NULL means row s for each sequence (a decode step; max_rows = 1),
 * and none for a sequence of length 0.  len[s] already counts the rows: they are
 * token rows len[s] - n .. len[s] - 1.
 *
 * Each block takes the smallest power of two as its scale that brings its
 * largest finite magnitude within the codes' range; a block that already held
 * rows keeps its scale or grows it, and then its earlier rows are rounded once
 * more, to the new scale (E4M3 codes lose nothing unless they become
 * subnormal; int8 codes move by at most half a step of the new scale).  Values
 * are rounded to nearest, ties to even.  An infinity becomes the block's
 * largest code; a NaN makes the block's scale NaN until the page is begun anew.
 * Rows of a page at or behind len[s] are left as they were.
 * With refs given, a page that is not held exactly once is not written
 * (status): two sequences may share full pages only, as ct_kv8_fork
 * leaves them.  max_rows up to 1 << 20. */
int ct_kv8_append(const ct_kv8_cache *c, int layer, const ct_kv8_seqs *s, const void *k, int ldk, const void *v,
                  int ldv, int type, int n_rows, const int *row_start, int max_rows, void *stream);

/* out[r][h] = softmax_j(scale * q[r][h] . K[j][h / g]) V[j][h / g], g = heads / kv_heads,
 * over the rows j of r's sequence that r sees.
 * q, out: [n_rows][heads * head_dim] of `type`, row strides ldq / ldo in
 * elements; 16-byte aligned, strides a multiple of 16 bytes.  Rows belong to
 * sequences as in ct_kv8_append, but with row_start NULL a sequence of length 0
 * has its row too (which sees nothing); row i of the n rows of sequence s is its
 * token row t = len[s] - n + i.  It sees every row j < len[s] or, with causal, those
 * with j <= t; with window > 0 (causal only) of these the ones with
 * j > t - window or j < sinks.  A row that sees nothing gets zeros.  Rows of
 * out that belong to no sequence are left as they were.
 * max_rows, max_len: upper bounds of the rows and of len[s] of any sequence
 * (when one is exceeded that sequence's rows of out are left as they were: status).
 * Products, sums and the softmax are fp32; K and V codes enter them exactly,
 * queries and probabilities as fp16 numbers scaled by powers of two: two each
 * (22 bits) for fp32 rows, one (11 bits) for bf16 rows.  What lies far below a
 * row's largest keeps fewer: a query's elements are exact to 2^-25 of its largest
 * (so bf16 ones are held exactly down to 2^-17 of it), products of probability and
 * V scale to 2^-33 of the row's largest such product, and a probability below 2^-96
 * of the largest may count as 0.  A query with an infinity or a NaN gives a row of
 * NaN.  A result depends on the sizes of the call (n_seqs, table_stride, max_rows,
 * max_len, heads, window, sinks: they decide how the keys are cut into pieces), not on
 * the other sequences' contents, and is the same each time.  out may be q itself.
 * ws: at least ct_kv8_attn_ws_bytes of the same arguments.  It is n_rows * heads *
 * (head_dim + 2) floats for each piece that the bounds max_rows and max_len allow for:
 * a gigabyte and more for long fp32 prompts, none for most short calls. */
int ct_kv8_attn(const ct_kv8_cache *c, int layer, const ct_kv8_seqs *s, const void *q, int ldq, void *out, int ldo,
                int type, int n_rows, const int *row_start, int max_rows, int max_len, int heads, float scale,
                int causal, int window, int sinks, void *ws, size_t ws_bytes, void *stream);
/* 0 when the arguments are bad (and for some calls that need no workspace). */
size_t ct_kv8_attn_ws_bytes(const ct_kv8_cache *c, const ct_kv8_seqs *s, int type, int n_rows, int max_rows,
                            int max_len, int heads, int causal, int window, int sinks);

/* ---- pages ------------------------------------------------------------------
 * Free pages are those with refs 0, and are always taken lowest number first,
 * in the order of the sequences that need them; the result of each call is a
 * function of its inputs alone.  refs must be given. */

/* len[s] += add[s] (add >= 0), with pages for the new rows written into the
 * table.  When free pages run out, the sequences from the first unserved one
 * on that needs a page stay as they were (status); so does a sequence whose
 * table row is too short.  n_seqs * table_stride is below 2^31. */
int ct_kv8_reserve(const ct_kv8_cache *c, const ct_kv8_seqs *s, const int *add, void *ws, size_t ws_bytes,
                   void *stream);

/* dst[i] continues src[parents[i]]: it shares the parent's full pages (one more
 * holder each) and gets a copy of a started last page, all layers, codes and
 * scales.  dst must not overlap src and hold nothing (release it with
 * ct_kv8_free before); table entries behind the pages of dst[i] are left as
 * they were.  parents[i] < 0 gives an empty sequence.  A child for which no
 * free page is left, or whose table row is too short, ends empty (status). */
int ct_kv8_fork(const ct_kv8_cache *c, const ct_kv8_seqs *src, const int *parents, const ct_kv8_seqs *dst, void *ws,
                size_t ws_bytes, void *stream);

/* Release the sequences which[0 .. n - 1] (NULL: all of s, n ignored): one
 * holder less for each of their pages, len = 0.  An index listed twice counts
 * once.  Table entries stay as they were. */
int ct_kv8_free(const ct_kv8_cache *c, const ct_kv8_seqs *s, const int *which, int n, void *stream);

/* Release the pages that hold only rows j with sinks <= j < len[s] - window:
 * rows that no query from token row len[s] - 1 on sees with that window.
 * Their table entries become -1. */
int ct_kv8_trim(const ct_kv8_cache *c, const ct_kv8_seqs *s, int window, int sinks, void *stream);

/* Move the live pages to the start of the pool: with L live pages, those
 * numbered L or above move, in order, to the free pages below L.  s lists every
 * sequence that holds pages.  The new table (laid out as s->table; entries
 * behind a sequence's pages are left as they were) and the new refs are
 * written to table_out and refs_out, which may be s->table and c->refs;
 * n_live (NULL or one int) gets L.  The moved pages' old copies stay readable
 * until those pages are written again. */
int ct_kv8_compact(const ct_kv8_cache *c, const ct_kv8_seqs *s, int *refs_out, int *table_out, int *n_live, void *ws,
                   size_t ws_bytes, void *stream);

/* Copy pages src[i] -> dst[i], i < n (at most 4096), all layers, codes and
 * scales.  A pair with a page outside the pool, a dst that another pair also
 * writes, or a dst that is any pair's src, is not copied (status). */
int ct_kv8_copy_pages(const ct_kv8_cache *c, const int *src, const int *dst, int n, void *stream);

/* Workspace of ct_kv8_reserve, ct_kv8_fork (n_seqs = dst->n_seqs) and ct_kv8_compact. */
size_t ct_kv8_pages_ws_bytes(const ct_kv8_cache *c, int n_seqs);

/* Waits for the current device, then reads and clears its status word
 * (0 = nothing reported, 4 = something was out of range and left out, 6 = no
 * free page was left, 1 to 3 = a bounded wait inside a kernel gave up: its output
 * is not to be used); CT_EDEVICE when a CUDA call failed.  The word is the
 * library's own, one per device: ct_device_status and ct_engine_status read the
 * same one. */
int ct_kv8_status(void);

#ifdef __cplusplus
}
#endif
#endif
