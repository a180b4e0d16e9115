/*
 * ramvamp_paged.h — C ABI of rotary positions and of a paged KV cache on
 * gfx950: a pool of pages that a batch of independent sequences draws on, the
 * rows written to it (K rotated on the way), read back, and attended by one new
 * token of each sequence. No reference counterpart: the reference runs one
 * sequence over one linear cache (kv/mod.rs:132-148) and rotates whole heads in
 * NeoX order without scaling (primitives/rope.rs:82-105); where these calls do
 * what it does they round as it does.
 *
 * Conventions of ramvamp_attn.h, and:
 *  - Tensor pointers are device pointers, aligned to an element, on the cache's
 *    device; RV_HOST_PTRS is RV_ERR_UNSUPPORTED. Rows of f32 inputs and outputs
 *    may lie further apart than their width: `*_stride` is the elements from one
 *    row to the next, at least the width (RV_PRIM_LENGTH_MISMATCH, a = width,
 *    b = stride; not looked at for a single row).
 *  - What the device reads from device memory (page ids, positions, lengths,
 *    sequence numbers) is checked on the device: a row or sequence that names
 *    what is not there is refused by itself, as its call says, nothing out of
 *    bounds is touched, and one such refusal is recorded for
 *    rv_paged_device_status. It must not change between the call and the end of
 *    its work: outputs of a call under which it did are undefined (nothing out of
 *    bounds is touched all the same, and later calls are as ever).
 */
#ifndef RAMVAMP_PAGED_H
#define RAMVAMP_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include "ramvamp_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Recorded by the device (rv_paged_device_status). */
#define RV_PAGED_PAGE_OUT_OF_RANGE 56     /* a layer, b row of the call, c the table's entry (as u32), d pages of the cache */
#define RV_PAGED_SEQUENCE_OUT_OF_RANGE 57 /* a layer, b row of the call, c sequence (as u32), d sequences of the table */
#define RV_PAGED_POSITION_OUT_OF_RANGE 58 /* a layer, b row of the call, c position or length (as u32), d positions of a table row */

/* ---- rotary positions --------------------------------------------------
 * The first rotary_dim values of a head are rotated in pairs, the rest pass
 * through: pair i is (i, i + rotary_dim / 2) with RV_ROPE_HALF, (2 i, 2 i + 1)
 * with RV_ROPE_INTERLEAVED. At position p pair i turns by p * f_i,
 *   f_i = theta^(-2 i / rotary_dim),
 * unless scaled for contexts `factor` times the trained one:
 *   RV_ROPE_LINEAR  f_i / factor;
 *   RV_ROPE_NTK     f_i of theta * factor^(rotary_dim / (rotary_dim - 2));
 *   RV_ROPE_YARN    f_i * (1 - r_i) + f_i / factor * r_i, r_i = (i - lo) / (hi - lo)
 *                   clamped to 0 .. 1, with lo = floor(pair(beta_fast)) >= 0, hi =
 *                   ceil(pair(beta_slow)) <= rotary_dim - 1, pair(b) = rotary_dim *
 *                   ln(trained_positions / (2 pi b)) / (2 ln theta), the pair that
 *                   makes b turns within the trained positions (hi - lo at least
 *                   0.001); cosine and sine times 0.1 ln(factor) + 1.
 * Angles, cosines and sines are computed in f64 and rounded to f32; the rotation
 * is y0 = x0 c - x1 s, y1 = x0 s + x1 c in f32, each operation rounded
 * (primitives/rope.rs:31-45). */
#define RV_ROPE_HALF 0u
#define RV_ROPE_INTERLEAVED 1u
#define RV_ROPE_UNSCALED 0u
#define RV_ROPE_LINEAR 1u
#define RV_ROPE_NTK 2u
#define RV_ROPE_YARN 3u

/* The frequencies of one model, in host memory: usable with any device and by
 * any number of threads; a call copies what it needs. */
typedef struct rv_rope rv_rope;

/* head_dim at most 512; rotary_dim even, 2 .. head_dim (RV_PRIM_INVALID_HEAD_DIM,
 * a = rotary_dim, b = head_dim). theta finite and positive (YARN: above 1), and so
 * that NTK's base and 2^31 f_i are finite.
 * factor (finite, at least 1) counts with a scaling, trained_positions (at least
 * 1) and the betas (finite, beta_fast > beta_slow > 0) with YARN alone; NTK needs
 * rotary_dim above 2. Else RV_ERR_UNSUPPORTED with `what`. */
int32_t rv_rope_new(size_t head_dim, size_t rotary_dim, uint32_t layout, double theta, uint32_t scaling,
                    double factor, size_t trained_positions, double beta_fast, double beta_slow, rv_rope** out,
                    rv_error* err);
void rv_rope_free(rv_rope* rope);
/* f_i of the rotary_dim / 2 pairs (n must be that many: RV_PRIM_LENGTH_MISMATCH)
 * and what cosine and sine are multiplied by; host memory, `gain` may be null. */
int32_t rv_rope_frequencies(const rv_rope* rope, double* freq, size_t n, double* gain, rv_error* err);
/* Row r of x, `width` f32 (whole heads: else RV_ATTN_Q_LEN_INDIVISIBLE), rotated at
 * positions[r] (i32; negative turns backwards) into row r of out. out may be x
 * itself (same stride), or rows beside x's in one buffer; any other overlap, also
 * with positions, is RV_ERR_UNSUPPORTED. Queued on `stream` of the current device. */
int32_t rv_rope_rows(const rv_rope* rope, const float* x, size_t x_stride, size_t rows, size_t width,
                     const int32_t* positions, float* out, size_t out_stride, void* stream, uint32_t flags,
                     rv_error* err);

/* ---- the paged cache -----------------------------------------------------
 * n_pages pages of page_rows rows in each of n_layers layers; a page id names
 * the same page in every layer. Row p of a sequence is row p % page_rows of the
 * page its table names at p / page_rows. Inside a page each kv head's rows are
 * contiguous. Element types are rv_kv_new's, with their roundings and limits; a
 * reader of a Q8_0 page sees f16(scale * code), as of a Q8_0 cache.
 * The caller owns the tables: which pages are free and whether two sequences
 * share one (a common prefix) is theirs to know. */
typedef struct rv_paged rv_paged;

/* A batch's tables on the device: page id p of sequence s is
 * ids[s * stride + p], p < pages. Entries past a sequence's rows are not read
 * as ids. */
typedef struct rv_page_table {
  const int32_t* ids;
  size_t n_seqs;
  size_t pages;
  size_t stride;
} rv_page_table;

/* Bytes of both planes (Q8_0: 34 per 32 elements). RV_KV_INVALID_DIMS as
 * rv_kv_projected_bytes (d = n_pages), also for page_rows not a power of two
 * from 8 to 1024; RV_ERR_UNSUPPORTED: head_dim above 512, n_kv_heads above
 * 65535, n_pages past 2^31 - 1. */
int32_t rv_paged_projected_bytes(size_t n_layers, size_t n_kv_heads, size_t head_dim, size_t n_pages,
                                 size_t page_rows, rv_elem elem, uint64_t* bytes, rv_error* err);
/* Zeroed pages on `device`. */
int32_t rv_paged_new(size_t n_layers, size_t n_kv_heads, size_t head_dim, size_t n_pages, size_t page_rows,
                     rv_elem elem, int device, rv_paged** out, rv_error* err);
/* Waits for the device's queued work before it frees the pages. */
void rv_paged_free(rv_paged* pg);
/* As rv_kv_set_tuning. RV_TUNE_PAGED_JOIN: how workgroups that share a
 * sequence's kv head join what they have: 0 within each XCD's L2 first where the
 * device deals workgroups to its XCDs in turn (checked when the cache is made),
 * else across them at once, 2 always so; other values are RV_ERR_UNSUPPORTED. */
#define RV_TUNE_PAGED_JOIN 1
int32_t rv_paged_set_tuning(rv_paged* pg, int32_t knob, int64_t value, rv_error* err);
/* As rv_kv_set_stream. Calls on one cache share its workspace: one stream at a
 * time, and so two graphs captured over one cache are replayed one after the
 * other. */
int32_t rv_paged_set_stream(rv_paged* pg, void* hip_stream, rv_error* err);
int32_t rv_paged_synchronize(rv_paged* pg, rv_error* err);
/* Waits for the stream, then returns and clears what a call recorded when the
 * device refused something since the last read (one of them, where there were
 * several): RV_OK or an RV_PAGED_* code. Not under capture. */
int32_t rv_paged_device_status(rv_paged* pg, rv_error* err);

/* Row r of k and v (kv heads * head_dim f32) becomes the row at positions[r] of
 * sequence seqs[r] (seqs null: sequence r). k_norm_w (may be null) is the
 * [head_dim] weight of a per-head RMSNorm of k with eps (primitives/norm.rs:
 * 18-90), then rope (may be null; its head_dim must be the cache's:
 * RV_PRIM_LENGTH_MISMATCH) rotates k at positions[r]; v is stored as given. A
 * negative position writes nothing (a padded batch's row). Refused on the
 * device, the row unwritten: a sequence the table does not have, a position
 * past the table row, a page the cache does not have. Rows of one call name
 * different places; of two that name one, it holds a mixture. */
int32_t rv_paged_append_rows(rv_paged* pg, size_t layer, const rv_rope* rope, const float* k, size_t k_stride,
                             const float* v, size_t v_stride, size_t rows, const int32_t* positions,
                             const int32_t* seqs, const rv_page_table* table, const float* k_norm_w,
                             size_t k_norm_len, float eps, uint32_t flags, rv_error* err);
/* The rows at positions[r] of sequence seqs[r], as attention reads them, into
 * row r of k and v (contiguous; either may be null): f32 of an F32 cache, else
 * f16. A row of a negative position or one refused on the device (as above) is
 * zeros. k and v overlap neither each other nor what the call reads
 * (RV_ERR_UNSUPPORTED). */
int32_t rv_paged_read_rows(rv_paged* pg, size_t layer, size_t rows, const int32_t* positions, const int32_t* seqs,
                           const rv_page_table* table, void* k, void* v, uint32_t flags, rv_error* err);

/* One new token of each of n_seqs sequences (at most the table's): row i of q
 * (q_dim post-RoPE f32) attends rows 0 .. lens[i] of sequence i, out row i the
 * softmax-weighted sum of v. A sequence of length 0 gets zeros. One whose
 * length is negative or past the table row, or that has a page the cache does
 * not have, is refused on the device: its out row (of the page: the heads')
 * is NaN. Rows of out behind the last are not touched. f32 arithmetic: f16 and
 * Q8_0 rows are matrix operands as stored, q and probabilities f16 hi + lo
 * halves scaled by powers of two (to 2^-22 of themselves, or 2^-38 of the
 * largest of a head's), sums in f32. V may be any finite values; scale * (q . k)
 * has to stay within f32's range, over f32 rows q . k and its partial sums too. An
 * infinity or NaN in a row that is attended reaches the outputs of that kv head's
 * query heads alone: NaN, but for an infinity of K that may, where it makes a score
 * minus infinity, leave its row without weight, and one of V that may stay an
 * infinity. What lies in rows past lens[i] never counts.
 * RV_ERR_UNSUPPORTED: n_seqs past 2^23, query heads past 65535, and tables whose
 * rows are more than 2^31 - 1 units (n_seqs * the tables' rows / 128 for each 16
 * query heads of a kv head; of every query head where head_dim is no multiple of
 * 8 or above 256). Checks, in order: q_dim, layer, the strides, the table, n_seqs,
 * out overlapping q, lens or the table (RV_ERR_UNSUPPORTED), the units. */
int32_t rv_paged_attention(rv_paged* pg, size_t layer, const float* q, size_t q_stride, size_t n_seqs, size_t q_dim,
                           const rv_page_table* table, const int32_t* lens, float scale, float* out,
                           size_t out_stride, uint32_t flags, rv_error* err);

/* The batch's step of one layer: q and k rows RMSNormed per head (either weight
 * may be null), rotated (rope may be null) at positions[i], k and v appended to
 * sequence i there, then attention over positions[i] + 1 rows. As
 * rv_paged_append_rows and rv_paged_attention one after the other; a negative
 * position gives zeros and writes nothing. out may overlap q, k, v and the weights,
 * all read before it is written, but not positions or the table
 * (RV_ERR_UNSUPPORTED). Positions and tables are read when
 * the step runs, so a captured step is replayed for every token (advance the
 * positions in the graph, or between replays on its stream); the first call of
 * a batch size may have to allocate and is not captured (RV_ERR_UNSUPPORTED). */
int32_t rv_paged_decode_step(rv_paged* pg, size_t layer, const rv_rope* rope, const float* q, size_t q_stride,
                             const float* k, size_t k_stride, const float* v, size_t v_stride, size_t n_seqs,
                             size_t q_dim, const float* q_norm_w, size_t q_norm_len, const float* k_norm_w,
                             size_t k_norm_len, float eps, const rv_page_table* table, const int32_t* positions,
                             float scale, float* out, size_t out_stride, uint32_t flags, rv_error* err);

#ifdef __cplusplus
}
#endif

#endif /* RAMVAMP_PAGED_H */
