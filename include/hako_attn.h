/*
 * hako_attn.h — a quantised key/value cache on the device and the attention
 * that reads it (C ABI).
 *
 * The part of a transformer block between the q/k/v matmuls and the output
 * projection, on caller-owned device buffers: the rotation of queries and
 * keys, the cache write, and attention over the cache for single tokens (a
 * batch may share a long prefix) and for whole packed prompts. The decoder of
 * hako_decode.h runs on these calls when it is given a cache type. In the
 * reference: src/model.c:105-137 with an fp32 cache, one token at a time.
 *
 * Everything outside the cache is fp32, and so is the arithmetic: products
 * with cached codes are carried to 22 bits or more (of a query's values, those
 * below 2^-16 of its head's largest to 2^-38 of that) and summed in fp32.
 * Conventions are those of hako_gpu.h: 0 or a negative HAKO_GPU_E* code with
 * hako_gpu_last_error() set, work enqueued on the library stream, device
 * pointers unless a comment says host. The attention calls use a library
 * workspace (see hako_gpu_capture_begin): make one call of a shape before
 * capturing it. It follows the cache's max_seq, not the lengths: for n_seq
 * sequences of single tokens up to n_seq * n_heads * (max_seq / 2048 + 1)
 * records of (head_dim + 3) * 4 bytes where n_seq * n_kv_heads fills the chip
 * (64 sequences of 28 heads of 128 in slots of 32768: 15 MB; 1024 in slots of
 * 131072: 1 GB), else a few MB. Drafted trees take n_seq * n_tree * n_heads
 * such records for each part of their keys, parts by the shape and max_seq (up
 * to 65536 records, 34 MB with heads of 128), prompts by their lengths (up to
 * 45 MB). Calls are made from one thread at a time.
 */
#pragma once
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#pragma GCC visibility push(default)

/* ── the cache ──
 * A cache row is one position of one key/value head: head_dim codes and one
 * fp32 scale; its values are code * scale.
 *
 * HAKO_KV_Q8: int8 codes by the q8_32 rule of hako_gpu_quantize_q8_32 over
 *   the whole row: scale = max|x| * RN(1/127), code = x * RN(127 / max|x|)
 *   rounded half to even, subnormals taken as 0.
 * HAKO_KV_F16: scale = the power of two not above max|x| (2^-126 at least),
 *   code = the half nearest to x / scale: no row overflows.
 *
 * A row that holds a NaN or an infinity gets codes 0 and the scale NaN: it
 * reads back as NaN throughout, and a query that sees it answers NaN. */
#define HAKO_KV_F16 1
#define HAKO_KV_Q8  2

typedef struct {
	int type;               /* HAKO_KV_* */
	int n_slots;            /* sequences the cache has room for */
	int max_seq;            /* positions per slot; max_seq * head_dim codes under 2 GiB */
	int n_kv_heads;
	int head_dim;           /* 64 or 128 */
	void *k, *v;            /* codes [n_slots][n_kv_heads][max_seq][head_dim], 16-byte aligned */
	float *k_scale, *v_scale; /* [n_slots][n_kv_heads][max_seq] */
} hako_gpu_kv;

/* Bytes of one of the two code arrays, and of one of the two scale arrays.
 * The arrays need no initial values: rows that were never written are never
 * read by a call whose lengths cover only written positions. */
int hako_gpu_kv_bytes(const hako_gpu_kv *kv, size_t *codes, size_t *scales);

/* A rotation of queries and keys: dims [0, rot_dim) of a head turn in pairs
 * (a, b) -> (a cos - b sin, a sin + b cos), every product and sum rounded to
 * fp32; dims past rot_dim stay. The pairs are (i, i + rot_dim/2), as the
 * reference's rope_neox (src/nn.c:32-42), or with `interleaved` (2i, 2i + 1).
 * The angles are the caller's, so any base, stretch for long contexts or
 * magnitude factor: table[p][i] = (cos, sin) of pair i at position p. */
typedef struct {
	const float *table;     /* [n_pos][rot_dim/2][2], 16-byte aligned */
	int n_pos;              /* positions of the table */
	int rot_dim;            /* a multiple of 8, 8..head_dim */
	int interleaved;        /* 0 or 1 */
} hako_gpu_rope;

/* n_tok new tokens: token i's key and value heads (k + i*kv_stride and
 * v + i*kv_stride, n_kv_heads*head_dim floats each) go to position pos[i] of
 * slot slot[i], the keys rotated first. With q not NULL its n_heads query
 * heads (q + i*q_stride) are rotated into q_out + i*q_out_stride; q_out may
 * be q with the same stride. rope NULL: no rotation, q must be NULL. slot
 * NULL: token i goes to slot i (n_tok <= n_slots).
 *
 * A token whose slot or position lies outside the cache, or whose position
 * lies outside the rope's table, is left out: nothing of it is written, so a
 * padded batch marks its padding with position -1. Two tokens of one call
 * must not name the same slot and position. Strides are in floats, multiples
 * of 4; k, v, q and q_out are 16-byte aligned. */
int hako_gpu_kv_append(const hako_gpu_kv *kv, const int *slot, const int *pos, int n_tok,
                       const float *k, const float *v, int64_t kv_stride, const hako_gpu_rope *rope,
                       const float *q, float *q_out, int n_heads, int64_t q_stride, int64_t q_out_stride);

/* The same with the rotation apart from the row: token i's keys and values go
 * to row pos[i], its key and queries are turned as at position turn[i]. For
 * rows that do not lie in the order of the text: drafted trees
 * (hako_search.h), where several nodes share a place in the text, or a slot
 * used as a ring, whose rows the window of a long text passes through. A token
 * whose turn lies outside the rope's table is left out too. */
int hako_gpu_kv_append_turned(const hako_gpu_kv *kv, const int *slot, const int *pos, const int *turn, int n_tok,
                              const float *k, const float *v, int64_t kv_stride, const hako_gpu_rope *rope,
                              const float *q, float *q_out, int n_heads, int64_t q_stride, int64_t q_out_stride);

/* The values of cached rows: token i's keys to k + i*kv_stride, its values to
 * v + i*kv_stride (either may be NULL), from position pos[i] of slot slot[i]
 * (slot NULL: slot i). The rows of a token outside the cache are left as they
 * were. Strides and alignment as above. */
int hako_gpu_kv_read(const hako_gpu_kv *kv, const int *slot, const int *pos, int n_tok,
                     float *k, float *v, int64_t kv_stride);

/* ── attention ──
 * out_h = sum over the positions p that a token sees of
 * softmax_p(scale * q_h . k_p) v_p, for each of its n_heads query heads; head
 * h reads key/value head h / (n_heads / n_kv_heads), at most 16 query heads to
 * one. A token that sees no position gets zeros. q and out hold head_dim
 * floats per head, heads one after the other, tokens q_stride and out_stride
 * floats apart (multiples of 4, 16-byte aligned); out may be q with the same
 * stride and overlaps it in no other way.
 *
 * A prefix in common: with prefix_len > 0 the positions below it are those of
 * slot prefix_slot for every sequence, the others its own slot's, so the
 * prefix is stored once and, for single tokens, read once for the batch.
 *
 * Values that a token does not see have no part in its output, whatever they
 * are; among those it sees, a contribution below 2^-24 of the largest value
 * row times the largest weight may round away. Keys and values of magnitudes
 * from 2^-80 to 2^80 are meant: outside, scores may overflow and small weights
 * and values be lost.
 *
 * The sums' order follows the shapes, not the timing: a call repeats itself
 * bit for bit. */

/* One token per sequence: sequence i's query (row i) over positions
 * [0, len[i]) of slot slot[i] (NULL: slot i). slot and len are device arrays,
 * read when the kernels run, so a captured call follows them; a len below 0
 * counts as 0 and above max_seq as max_seq, a slot outside the cache as len
 * 0. */
int hako_gpu_attn_decode(float *out, int64_t out_stride, const float *q, int64_t q_stride, const hako_gpu_kv *kv,
                         const int *slot, const int *len, int n_seq, int n_heads, float scale, int prefix_slot,
                         int prefix_len);

/* Whole prompts: sequence s has len[s] tokens (0: none) at positions
 * start[s].. of slot slot[s] (NULL: slot s), its rows of q and out after those
 * of the sequences before it. A token sees its own position and every one
 * before it: the tokens' keys and values are in the cache already. slot,
 * start and len are HOST arrays, taken by the call. */
int hako_gpu_attn_prompt(float *out, int64_t out_stride, const float *q, int64_t q_stride, const hako_gpu_kv *kv,
                         const int *slot, const int *start, const int *len, int n_seq, int n_heads, float scale,
                         int prefix_slot, int prefix_len);

/* ── a window, and a few first positions that stay ──
 * The same two for models (or layers) whose tokens look back a limited way: a
 * token at position t sees the positions p <= t with p > t - window (window
 * >= 1: its own and the window - 1 before it) or p < sinks (>= 0). Rows outside
 * that are not read, so a token's work does not grow with its position, and
 * the workspace of single tokens follows min(max_seq, sinks + window) in the
 * place of max_seq. Prefixes are not shared here. */
int hako_gpu_attn_decode_window(float *out, int64_t out_stride, const float *q, int64_t q_stride, const hako_gpu_kv *kv,
                                const int *slot, const int *len, int n_seq, int n_heads, float scale, int window,
                                int sinks);
int hako_gpu_attn_prompt_window(float *out, int64_t out_stride, const float *q, int64_t q_stride, const hako_gpu_kv *kv,
                                const int *slot, const int *start, const int *len, int n_seq, int n_heads, float scale,
                                int window, int sinks);

/* ── trees of drafted tokens ──
 * n_tree (1..64) nodes of each of n_seq sequences: node j of sequence s is row
 * s*n_tree + j of q and out, its keys and values are in row base[s] + j of slot
 * slot[s] (NULL: slot s). It sees the positions below base[s], and of the rows
 * from base[s] on those whose bits are set in seen[s*n_tree + j] (8-byte
 * aligned): bit i is node i. A node whose mask is 0 is not there: it gets
 * zeros. slot, base and seen are device arrays, read when the kernels run; a
 * base above max_seq counts as max_seq, and no row at max_seq or past it is
 * seen; a base below 0 or a slot outside the cache: the sequence gets zeros.
 * Rows from base on that no node of a sequence sees, as those of the nodes that
 * a padded tree lacks, need not have been written and may hold anything.
 * hako_gpu_tree_plan (hako_search.h) makes the masks of a tree from its
 * parents. A prefix in common as above. */
int hako_gpu_attn_tree(float *out, int64_t out_stride, const float *q, int64_t q_stride, const hako_gpu_kv *kv,
                       const int *slot, const int *base, const uint64_t *seen, int n_seq, int n_tree, int n_heads,
                       float scale, int prefix_slot, int prefix_len);

#pragma GCC visibility pop

#ifdef __cplusplus
}
#endif
