/*
 * vq_cache.h -- the vector-quantised key-value cache of libvqhip.so: training of float codebooks, quantising
 * keys and values as they are written, reading them back, and attention over the paged codes.  No counterpart
 * in VQ_Full.py, whose three steps (LBG iteration :77-90, encode :124-125, decode :160-169) these are for float
 * vectors and squared distance.
 *
 * The vector of one token and one head, `dim` numbers, is cut into parts = dim / sub sub-vectors; each is stored
 * as one byte, the number of its nearest codeword.
 *   codebook   (cb_heads, K, dim), row-major; row k holds codeword k of every sub-vector side by side;
 *              cb_heads is `heads`, or 1: one codebook for all heads
 *   k_codes    (pages, heads, page, parts) bytes
 *   v_codes    (pages, heads, parts, page) bytes: the codes of a page's tokens lie side by side, as the second
 *              product of attention takes them
 *   slot       page number * page + place in the page
 * dim is 32, 64, 96, 128, 192 or 256; sub is 2, 4 or 8; K is 1 to 256; page is a multiple of 16, at most 2^20; heads is
 * at most 1024; pages and tokens are below 2^31.
 *
 * The conventions of vq_hip.h hold (device pointers, stream, status codes, vq_last_error, nothing allocated).
 * Every call reads its lengths, slots and page numbers on the device and may be captured into a HIP graph.
 * One workspace serves one call at a time.  Element type `dtype`: VQ_F32, VQ_BF16 or VQ_F16.  Tensors of vectors
 * are given by their strides in elements between tokens and between heads; the numbers of one vector lie side by
 * side, and vectors start at multiples of 16 bytes.  Codebooks, codes and workspaces start at multiples of 16 bytes.
 */
#ifndef VQ_CACHE_H
#define VQ_CACHE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define VQ_F32  0
#define VQ_BF16 1
#define VQ_F16  2

/* Quantises the keys and values of `tokens` tokens and stores their codes: code = argmin_k sum_e (x_e - c_ke)^2,
 * the sum taken left to right in fp64, the lowest k winning ties; a distance that is infinite or not a number is
 * never less than another, so a vector that has no finite distance gets code 0.  A token whose slot is outside
 * [0, pages * page) is not stored.  Slots should be distinct: of two tokens with one slot, each code is that of
 * either.  dtype (of k, v and the codebooks): VQ_BF16 or VQ_F16. */
int vq_cache_write(const void *k, int64_t k_token_stride, int64_t k_head_stride,
                   const void *v, int64_t v_token_stride, int64_t v_head_stride,
                   const int64_t *slots, int64_t tokens, const void *k_cb, const void *v_cb, int cb_heads,
                   int heads, int dim, int sub, int K, int dtype,
                   uint8_t *k_codes, uint8_t *v_codes, int64_t pages, int page, void *stream);

/* The vectors that the codes of `tokens` slots stand for: k_out and v_out, (tokens, heads, dim) of `dtype`.
 * A slot outside [0, pages * page) reads as zeros; a code of K or more reads as codeword K - 1. */
int vq_cache_read(const int64_t *slots, int64_t tokens, const void *k_cb, const void *v_cb, int cb_heads,
                  int heads, int dim, int sub, int K, int dtype,
                  const uint8_t *k_codes, const uint8_t *v_codes, int64_t pages, int page,
                  void *k_out, void *v_out, void *stream);

/* Causal attention of packed sequences' newest tokens over the cache.  Sequence b owns rows starts[b] to
 * starts[b + 1] of q (rows, q_heads, dim) and the first kv_lens[b] tokens of the pages table[b, 0 .. width); its
 * rows are the newest of those tokens: row i of n_q sees tokens 0 to kv_lens[b] - n_q + i.  Query heads are
 * grouped: head h reads cache head h / (q_heads / heads).  rows * q_heads / heads is below 2^30, width * page below 2^31,
 * q_heads at most 4096, seqs at most 65535.  out and lse overlap no other tensor of the call.
 *   out (rows, q_heads, dim) = softmax(scale * q k^T) v      lse (rows, q_heads, nullable) = log sum exp(scale * q k^T)
 * A row that sees no token, or whose scores are all minus infinity, gets zeros and minus infinity; one with a score that is NaN or plus
 * infinity (in fp32) gets NaN; rows of no sequence are left as they were.  Lengths past the table's width are cut to it; the tokens of a
 * page number outside [0, pages) are not seen.  Codewords have to be finite; a code of K or more stands for some codeword or for zeros.  max_q and
 * max_kv, the longest of the sequences' rows and lengths as the caller knows them, only shape the launch: any value of
 * 1 or more gives the same sums, up to the order of addition.
 * Scores, weights and sums are fp32, which holds the sums of bf16 values up to 2^120 divided by the number of tokens.  Weights are rounded to
 * `dtype` before they meet the values; their sum takes them unrounded.  Of fp16 a weight is off by half a step, or by 2^-19 of the
 * largest that its row has among the 32 tokens it is taken with.
 * `starts` rises, from 0 or more to `rows` or less.  dtype: VQ_BF16 or VQ_F16. */
size_t vq_cache_attention_ws_bytes(int64_t rows, int q_heads, int heads, int dim, int sub, int K, int seqs,
                                   int64_t max_q, int64_t max_kv);
int vq_cache_attention(const void *q, int64_t q_token_stride, int64_t q_head_stride, int64_t rows, int q_heads,
                       const void *k_cb, const void *v_cb, int cb_heads, int heads, int dim, int sub, int K, int dtype,
                       const uint8_t *k_codes, const uint8_t *v_codes, int64_t pages, int page,
                       const int32_t *table, int seqs, int width, const int32_t *kv_lens, const int32_t *starts,
                       int64_t max_q, int64_t max_kv, double scale, void *out, float *lse,
                       void *ws, size_t ws_bytes, void *stream);

/* The accumulating half of an LBG iteration of float codebooks: over `tokens` tokens' vectors x, for each head,
 * part and codeword, the sum and number of the vectors nearest to it (as in vq_cache_write), and for each head and part
 * the sum of the least squared distances.  A vector of which a number is 2^100 or more
 * in size, or no number, is left out of all three.  sums (heads, K, dim) fp64, counts (heads, parts, K) int64, dist
 * (heads, parts) fp64 are overwritten; the result does not depend on timing.  A sum is off by 2^-17 of its numbers' sizes added up at
 * most (products in fp32, 256 to 1024 vectors at a time, are added up exactly and rounded to fp32 once a chunk).  cb is (heads, K, dim)
 * fp32; x is of any of the three types.  A call takes 65535 chunks of 4096 tokens (268 million).  Adding several calls' sums, counts and dist gives
 * those of their tokens together. */
size_t vq_cache_lbg_ws_bytes(int64_t tokens, int heads, int dim, int sub, int K);
int vq_cache_lbg_accum(const void *x, int64_t token_stride, int64_t head_stride, int64_t tokens,
                       const float *cb, int heads, int dim, int sub, int K, int dtype,
                       double *sums, int64_t *counts, double *dist, void *ws, size_t ws_bytes, void *stream);

/* Both halves in one: the new codebook, the members' numbers (heads, parts, K) and the mean squared distance to the old codewords
 * (heads, parts).  cb_new may be cb. */
int vq_cache_lbg_iterate(const void *x, int64_t token_stride, int64_t head_stride, int64_t tokens,
                         const float *cb, int heads, int dim, int sub, int K, int dtype,
                         float *cb_new, int64_t *counts, double *mean_dist, void *ws, size_t ws_bytes, void *stream);

/* The closing half: cb_new = sums / counts, a codeword without members staying as it is in cb_old, and
 * mean_dist (heads, parts) = dist / the number of vectors (0 where there is none).  cb_new may be cb_old. */
int vq_cache_lbg_finish(const double *sums, const int64_t *counts, const double *dist, const float *cb_old,
                        int heads, int dim, int sub, int K, float *cb_new, double *mean_dist, void *stream);

#ifdef __cplusplus
}
#endif
#endif
