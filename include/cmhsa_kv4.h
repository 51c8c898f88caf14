/* cmhsa_kv4.h -- C ABI of a paged KV cache held in 4 bits: store, read back, single-token attention, page copies (same
 * library and conventions as include/cmhsa.h: libcmhsa_hip.so, device pointers, no allocation, no synchronisation, status
 * codes of cmhsa.h, `stream` is a hipStream_t; the types CMHSA_F32 / BF16 / F16 are those of include/cmhsa_packed.h).
 *
 * cmhsa_fp32_decode_step reads an fp32 cache of one length for the whole batch: 512 bytes for a token's head of 64.  Here
 * a token's head of 64 takes 68, every sequence has a length of its own, and its tokens lie in pages of a common pool,
 * which sequences may share.
 *
 * NUMBERS.  Every 32 consecutive elements of a token's head are 32 e2m1 codes (sign and one of the magnitudes 0 0.5 1 1.5
 * 2 3 4 6) and one scale byte: exponent + 127 of a power of two, 255 = the block is not a number.  A block with largest
 * magnitude a is stored with the smallest 2^e, e >= -126, that has a <= 7 * 2^e (7 rounds to 6, the largest magnitude,
 * with no more than half a step's error), each element rounded to the nearest, ties to the even code.  A block that
 * holds a NaN or an infinity gets scale byte 255.
 * LAYOUT.  The pool is num_pages pages of num_kv_heads blocks; the block of (page, head) is
 *     K codes [page_size][head_dim / 2] | V codes [page_size][head_dim / 2] | K scales [page_size][head_dim / 32] | V scales [..]
 * = CMHSA_KV4_BLOCK_BYTES(page_size, head_dim) bytes; element 2i of a token's head is the low nibble of its byte i.
 * PAGE TABLE.  page_table[s * table_stride + n] is the page that holds the positions n * page_size .. of sequence s;
 * table_width entries a sequence.  An entry outside [0, num_pages) is no page: nothing is stored to it, it reads as zeros,
 * and attention leaves its positions out.
 */
#ifndef CMHSA_KV4_H
#define CMHSA_KV4_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define CMHSA_KV4_BLOCK_BYTES(page_size, head_dim) ((int64_t)(page_size) * (head_dim) / 16 * 17)
#define CMHSA_KV4_MIN_PAGE 16
#define CMHSA_KV4_MAX_PAGE 256

/* Requirements of all four calls: head_dim 64 or 128; page_size a power of two from 16 to 256; pages 16-B aligned,
 * page_stride (bytes) a multiple of 16 and at least num_kv_heads blocks; int32 arrays 4-B aligned.  Errors as in
 * include/cmhsa_packed.h; CMHSA_ERR_TOO_LARGE also for launches of 2^32 threads (append, gather: 32 a row and 512 elements of it; decode: 256 or 512
 * a sequence, K/V head and 16 query heads). */

/* Token r - cu_seqlens[s] of sequence s (row r of k and v: num_kv_heads * head_dim elements, row strides in elements,
 * multiples of 16 bytes) goes to position starts[s] + r - cu_seqlens[s] (starts NULL: 0).  Rows behind the last sequence
 * and positions outside [0, table_width * page_size) are not stored.  No two rows of a call may have one place. */
int cmhsa_kv4_append(const void *k, const void *v, int64_t k_row_stride, int64_t v_row_stride, int dtype,
                     uint8_t *pages, int64_t page_stride, int num_pages, int page_size,
                     const int *page_table, int64_t table_stride, int table_width,
                     const int *cu_seqlens, const int *starts, int num_seqs, int rows, int num_kv_heads, int head_dim, void *stream);

/* The way back: row r of k and v receives the values of position starts[s] + r - cu_seqlens[s] of its sequence (zeros
 * where there is no page).  zero_rest != 0 writes zeros to rows behind the last sequence, 0 leaves them as they were.
 * Values beyond the type's range become infinities (fp16). */
int cmhsa_kv4_gather(void *k, void *v, int64_t k_row_stride, int64_t v_row_stride, int dtype,
                     const uint8_t *pages, int64_t page_stride, int num_pages, int page_size,
                     const int *page_table, int64_t table_stride, int table_width,
                     const int *cu_seqlens, const int *starts, int num_seqs, int rows, int num_kv_heads, int head_dim, int zero_rest, void *stream);

/* One query token a sequence over the positions 0 .. lengths[s] - 1 of its pages (its own token appended before):
 *     o[s, h] = sum_j softmax_j( q[s, h] . K[j, g] / sqrt(head_dim) ) V[j, g]          g = h / (num_heads / num_kv_heads)
 * q, o: num_seqs rows of num_heads * head_dim elements of `dtype`, sharing no memory.  lengths: int32 in DEVICE memory, so that a captured
 * graph serves every step.  lengths[s] == 0, or outside [0, table_width * page_size]: nothing is read and o[s] = 0.
 * Scores of -inf (q . K beyond fp32's range) weigh 0; a sequence that has no other is not a number.
 * workspace: device memory of at least cmhsa_kv4_decode_workspace_bytes(..) bytes, 16-B aligned, contents irrelevant
 * before and after (NULL where that is 0); calls that overlap in time must not share one. */
size_t cmhsa_kv4_decode_workspace_bytes(int num_seqs, int table_width, int page_size, int num_heads, int num_kv_heads, int head_dim);
int cmhsa_kv4_decode(const void *q, void *o, int64_t q_row_stride, int64_t o_row_stride, int dtype,
                     const uint8_t *pages, int64_t page_stride, int num_pages, int page_size,
                     const int *page_table, int64_t table_stride, int table_width,
                     const int *lengths, int num_seqs, int num_heads, int num_kv_heads, int head_dim,
                     void *workspace, size_t workspace_bytes, void *stream);

/* Page dst[i] := page src[i] for i < count, in `layers` pools that lie layer_stride bytes apart, page_bytes bytes a page
 * (a multiple of 16).  src and dst are HOST arrays: they are checked (range, no page written twice, none both read and
 * written; BAD_SHAPE as for pages that overlap) before anything is launched, and a captured call keeps their values. */
int cmhsa_kv4_copy_pages(uint8_t *pages, int64_t layer_stride, int layers, int64_t page_stride, int num_pages, int64_t page_bytes,
                         const int *src, const int *dst, int count, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* CMHSA_KV4_H */
