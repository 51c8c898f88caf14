/* cmhsa_packed.h -- C ABI of causal attention over PACKED sequences of different lengths, with grouped heads, in fp32,
 * bf16 or fp16 (same library and conventions as include/cmhsa.h: libcmhsa_hip.so, device pointers, no allocation, no
 * synchronisation, status codes of cmhsa.h, `stream` is a hipStream_t).
 *
 * cmhsa_fp32_fwd takes a batch of equally long sequences with one K/V head per query head.  Here the rows of every
 * sequence lie one behind the other in one matrix: sequence s owns the query rows cu_q[s] .. cu_q[s+1] - 1 and the K/V
 * rows cu_k[s] .. cu_k[s+1] - 1 (nq and nk of them).  Function computed, for query row i (0 <= i < nq) of sequence s and
 * query head h, with K/V head g = h / (num_heads / num_kv_heads):
 *
 *     o[i, h] = sum_j softmax_j( q[i, h] . k[j, g] / sqrt(head_dim) ) v[j, g]        over  0 <= j <= nk - nq + i
 *
 * so the LAST query row sees the last key: nq == nk is a whole prompt, nq < nk a continuation of nk - nq earlier tokens.
 * A row that sees no key (nq > nk) is zero.  Keys that a row does not see take no part whatever they hold: a NaN or an
 * infinity there does not reach the row.  One that the row does see gives what the formula gives in floating point.
 */
#ifndef CMHSA_PACKED_H
#define CMHSA_PACKED_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define CMHSA_F32 0
#define CMHSA_BF16 1
#define CMHSA_F16 2

/* Where blocks of query rows are few and keys many (a continuation of long sequences, one prompt alone), the keys of a
 * block are cut between workgroups if there is device memory for their unfinished results: workspace, at least
 * cmhsa_packed_workspace_bytes(..) bytes (0 for most shapes), 16-B aligned, contents irrelevant before and after; calls
 * that overlap in time must not share one.  Without it (NULL, or too short) the call is right and slower. */
size_t cmhsa_packed_workspace_bytes(int num_seqs, int total_q, int total_k, int num_heads, int num_kv_heads, int head_dim, int dtype);

/* q, o: total_q rows of num_heads * head_dim elements; k, v: total_k rows of num_kv_heads * head_dim (row r at
 * ptr + r * row_stride elements; column slices of one QKV buffer are fine).  cu_q, cu_k: num_seqs + 1 ascending int32 in
 * DEVICE memory, cu[0] = 0 for packing without a gap; cu_k may be cu_q.  o shares no memory with q, k or v.  A value outside [0, total] is taken as the
 * nearest one inside, and what ends before it starts is empty: no value reads or writes out of range, but which rows are
 * written where they do not ascend is not said.
 * dtype: CMHSA_F32 / CMHSA_BF16 / CMHSA_F16 for all four.  Statistics and sums are fp32 for every type; a key's weight is its exponential
 * against a running maximum, up to 2^15, so that values of v beyond about 2^112 over the number of keys may overflow in the sums.
 * Up to 64 sequences a call get the faster layouts: short ones a wave each, the longest work first, keys cut between
 * workgroups.  Beyond, every (sequence, K/V head, 128 rows) is a workgroup of its own, whatever its length.
 * zero_rest != 0 writes zeros to the rows of o that belong to no sequence (those from cu_q[num_seqs] on); 0 leaves them
 * as they were.
 * Requirements: head_dim 64 or 128; num_heads a multiple of num_kv_heads; 16-B aligned pointers (cu: 4 B); row strides
 * multiples of 16 bytes and below 2^24 bytes.  total_q == 0 or num_seqs == 0 (without zero_rest) is a no-op.
 * CMHSA_ERR_TOO_LARGE also where total_q * num_heads / 128 + num_seqs * num_kv_heads reaches 2^24 workgroups.
 * Returns CMHSA_OK, CMHSA_ERR_NULL_POINTER, CMHSA_ERR_BAD_SHAPE, CMHSA_ERR_HEAD_DIM, CMHSA_ERR_ALIGNMENT,
 * CMHSA_ERR_TOO_LARGE or a positive hipError_t. */
int cmhsa_packed_fwd(const void *q, const void *k, const void *v, void *o,
                     int64_t q_row_stride, int64_t k_row_stride, int64_t v_row_stride, int64_t o_row_stride,
                     const int *cu_q, const int *cu_k, int num_seqs, int total_q, int total_k,
                     int num_heads, int num_kv_heads, int head_dim, int dtype, int zero_rest,
                     void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* CMHSA_PACKED_H */
