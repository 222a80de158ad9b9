/*
 * wkf_decode.h -- the operators of a decoder's attention block as it serves, next to the Tensor API of wkf_tensor.h
 * and in its manner: opaque handles, status codes with the message in wkf_last_error(), nodes that are only recorded
 * until something materialises them.  None of them has a counterpart in the reference.
 *
 *   wkf_tensor_mat_mul_q4   products with weights held in 4 bits, beside wkf_tensor_mat_mul
 *   wkf_tensor_norm_rope    the norm of every head and its rotation, beside wkf_tensor_layer_norm and wkf_tensor_rope
 *   wkf_kv_cache_*          keys and values in 8 bits with a scale for each block of tokens and head
 *   wkf_tensor_attend       attention over such a cache, beside wkf_tensor_softmax_last_dim
 *
 * A serving program keeps its results on the device: wkf_tensor_zeros makes a tensor that holds data,
 * wkf_tensor_materialize_into computes lazy tensors into such tensors, wkf_tensor_device_ptr says where one lies.
 *
 * Element types are those of the Tensor API (WKF_F32, WKF_F16); sums, softmax statistics and norms are kept in f32 and
 * results are rounded once.  On the way to f16 results a product with many rows may round weights to f16 too, an error like
 * the result's own; after wkf_device_set_exact_math(dev, 1) none does.  Every size below is in elements.
 */
#ifndef WKF_DECODE_H
#define WKF_DECODE_H

#include "wkf_tensor.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct wkf_q4 wkf_q4;
typedef struct wkf_kv_cache wkf_kv_cache;

/* ---- results that stay on the device ---- */

/* A tensor that holds data, all zeros, without an upload. */
int wkf_tensor_zeros(wkf_device* dev, int dtype, int rank, const size_t* shape, wkf_tensor** out);
/* Computes ts[i] and leaves its values in outs[i], a dense tensor that holds data (wkf_tensor_new, wkf_tensor_zeros) of
 * the same shape, dtype and device; one pass over the joint graph, as wkf_tensor_materialize_many.  An output may be a
 * leaf of any of the graphs: every value is computed from what the leaves held before the call.  The launches are
 * recorded on ts[0].  Tensors recorded earlier that have outs[i] among their leaves see the new values when they are
 * materialised next.  No two outputs may be the same tensor.  When it fails, some outputs may hold their new values already. */
int wkf_tensor_materialize_into(wkf_tensor* const* ts, int n, wkf_tensor* const* outs);
/* The device address of the first element of a tensor that holds data.  What has been launched on the device may still
 * be writing there: wkf_device_sync first.  The address is good until the last handle of the tensor is freed. */
int wkf_tensor_device_ptr(const wkf_tensor* t, void** out);

/* ---- weights in 4 bits ---- */

/* A matrix W [k, n] in 4 bits: W[i][j] = (codes[i][j] - zeros[i / group][j]) * scales[i / group][j].
 * codes: k * n bytes, row-major, each 0 .. 15.  scales: ceil(k / group) rows of n values of `scale_dtype`.  zeros: as many
 * bytes, each 0 .. 15, or NULL for 8 everywhere.  group is a multiple of 32; the last group of rows may be shorter.
 * All three are host memory and are copied; the matrix is laid out for the kernels once, here. */
int wkf_q4_new(wkf_device* dev, size_t k, size_t n, size_t group, const void* codes, int scale_dtype, const void* scales,
               const void* zeros, wkf_q4** out);
/* Tensors recorded with the weights keep them alive. */
void wkf_q4_free(wkf_q4* w);
int wkf_q4_shape(const wkf_q4* w, size_t* k, size_t* n, size_t* group);
/* x [..., M, k] times W [k, n]: [..., M, n] in x's dtype, with at most 2^20 - 1 rows of x in all.  With many rows of f16 each
 * weight may be rounded to f16 first, if none of them is too large or too small for its normal numbers (never with exact math). */
int wkf_tensor_mat_mul_q4(const wkf_tensor* x, const wkf_q4* w, wkf_tensor** out);

/* ---- the norm of a head and its rotation ---- */

/* For every row of t [heads, seq, dim] or [batch, heads, seq, dim]: y = x / sqrt(mean(x^2) + eps) * weight, rotated by its
 * position p as wkf_tensor_rope does (the half of the row at d and the half at d + dim / 2 turn by the angle whose cosine and
 * sine the tables hold in row p).  weight [dim]; cos and sin [max_positions, dim / 2] or [max_positions, dim].  The weight and the
 * tables are of t's dtype or of f32.  Row s of batch entry b has position positions[b] + s; positions is one number for each
 * batch entry (one for rank 3), or NULL for zeros.  dim is even and at most 1024.  Everything is computed in f32 and rounded once.
 * t may be a strided view whose last dimension is dense.  Sibling nodes of one wkf_tensor_materialize_many / _into call that
 * share tables, eps and positions and agree in batch, seq, dim and dtype (the heads of q and of k) run as ONE launch. */
int wkf_tensor_norm_rope(const wkf_tensor* t, const wkf_tensor* weight, const wkf_tensor* cos, const wkf_tensor* sin, float eps,
                         const size_t* positions, wkf_tensor** out);

/* ---- keys and values in 8 bits ---- */

/* A cache for `sequences` (at most 256) sequences of up to `capacity` tokens with `kv_heads` heads of `head_dim` (at most 256)
 * elements.  For each sequence, head and block of `block` tokens (32, 64 or 128) keys and values have one f32 scale each,
 * the largest finite magnitude of the block / 127; an element is the integer nearest to value / scale (ties to even).  The
 * originals of a sequence's last, unfinished block are kept in f32 beside it: a block's codes depend on its tokens, not
 * on the calls that brought them.  8 bits have no place for infinities (stored as the largest magnitude) and NaN (stored as 0). */
int wkf_kv_cache_create(wkf_device* dev, size_t sequences, size_t kv_heads, size_t head_dim, size_t capacity, size_t block,
                        wkf_kv_cache** out);
/* Tensors recorded with the cache keep it alive. */
void wkf_kv_cache_free(wkf_kv_cache* c);
/* Tokens of a sequence. */
int wkf_kv_cache_length(const wkf_kv_cache* c, size_t sequence, size_t* out);
/* Forgets the tokens of one sequence, or of all of them for (size_t)-1. */
int wkf_kv_cache_reset(wkf_kv_cache* c, size_t sequence);
/* Appends k and v, [sequences, kv_heads, S, head_dim] (or without the first dimension for one sequence), behind the tokens of
 * every sequence: the first counts[b] <= S tokens of sequence b (NULL: S of each).  Runs at once; k and v are materialised.
 * When a sequence would outgrow the capacity nothing is appended. */
int wkf_kv_cache_append(wkf_kv_cache* c, const wkf_tensor* k, const wkf_tensor* v, const size_t* counts);
/* What the cache holds for tokens first .. first + count: [2, sequences, kv_heads, count, head_dim], keys then values,
 * zeros behind the end of a sequence. */
int wkf_kv_cache_values(wkf_kv_cache* c, int dtype, size_t first, size_t count, wkf_tensor** out);
/* Attention of q [sequences, heads, S, head_dim] (or without the first dimension for one sequence) over the cache:
 * softmax(scale q k^T) v.  Head h reads key head h / (heads / kv_heads).  The S rows are the LAST tokens of each sequence, or
 * its last counts[b] <= S ones (then rows behind counts[b] give zeros); with causal != 0 a row sees the tokens up to its own,
 * else all of its sequence.  A row that sees no token gives zeros.  scale is finite and not negative.
 * With more than 16 rows of f16 for a key head its softmax weights may be rounded to f16 (never with exact math).  Weighted values
 * are summed in f32 before they are divided by the sum of the weights: values beyond 3.4e38 / tokens may overflow.
 * The node stands for the cache as it is now: materialising it after an append or a reset is WKF_ERR_INVALID_ARG. */
int wkf_tensor_attend(const wkf_tensor* q, wkf_kv_cache* c, float scale, int causal, const size_t* counts, wkf_tensor** out);

#ifdef __cplusplus
}
#endif
#endif
