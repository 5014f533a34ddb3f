/*
 * hako_search.h — beams and trees of drafted tokens over the quantised cache
 * (C ABI).
 *
 * What decoding needs besides hako_attn.h when a step tries more than one
 * continuation. Beam search: the best continuations of all beams from a step's
 * logits, and the caches brought after them. Drafted trees (a small model's or
 * a table's guesses, checked in one pass): a tree's positions and masks, the
 * path that the model's own picks follow, and that path's rows moved together;
 * the attention between them is hako_gpu_attn_tree of hako_attn.h. In the
 * reference there is one sequence and one continuation (src/sample.c).
 *
 * Conventions are those of hako_gpu.h: 0 or a negative HAKO_GPU_E* code with
 * hako_gpu_last_error() set, work enqueued on the library stream. All arrays
 * are device arrays, read when the kernels run, so that a captured call
 * follows them; arrays that are written overlap no other array of the call.
 * Calls are made from one thread at a time.
 */
#pragma once
#include <stddef.h>
#include <stdint.h>

#include "hako_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#pragma GCC visibility push(default)

#define HAKO_MAX_BEAMS 16   /* beams of a request */
#define HAKO_MAX_PICK  32   /* continuations chosen for a request */
#define HAKO_MAX_TREE  64   /* nodes of a tree */

/* ── beams ──
 * One step of n_req requests with n_beams beams each; beam b of request r is
 * row r*n_beams + b of logits (vocab floats, at most 2^24, rows ld floats
 * apart), score and done. score is the sum of the log probabilities of the
 * beam's tokens (-inf: no beam there). A continuation of beam b by token t is worth
 *   score[b] + (logits[b][t] - log sum_j exp(logits[b][j])),
 * compared in 64 bits. The log is taken of 32-bit exponentials and good to
 * 2^-19 (2^-25 as a rule), so continuations of different beams that lie closer
 * than that may come in either order; those of one beam go by their logits
 * alone. done[b] != 0 marks a beam that has ended: its one
 * continuation is token eos at its own score. done may be NULL (none has).
 *
 * The n_pick (1..HAKO_MAX_PICK) best continuations of a request, best first,
 * equal ones by beam, and of a beam by larger logits, then by token, go to
 * row r of parent (the beam, 0..n_beams-1), token and score_out ([n_req]
 * [n_pick] each), and done_out (may be NULL) is 1 where the parent has ended
 * or the token is eos. Continuations worth -inf or NaN are none (a row with a
 * NaN or +inf has none at all); where a request has too few, the remaining
 * places get parent -1, token -1, score -inf, done 0.
 *
 * arrange != 0 (n_pick = n_beams): the same continuations in another order, so
 * that little has to be moved: a beam that survives is followed in its own
 * place by the best of its continuations, the other ones fill the places that
 * are left, best first. parent[r][p] is then the beam whose state belongs in
 * place p, and a place that is its own parent stays.
 *
 * Uses a library workspace (make one call of a shape before capturing it):
 * per row at most vocab / 1024 + 1 parts of n_pick * 8 + 12 bytes. */
int hako_gpu_beam_select(const float *logits, int64_t ld, int vocab, const float *score, const int *done, int eos,
                         int n_req, int n_beams, int n_pick, int arrange, int *parent, int *token, float *score_out,
                         int *done_out);

/* After it: beam p of request r takes the cache rows [since[r], len[r]) that
 * beam parent[r][p] of the request held, in all n_kv caches (of one shape, as
 * those of a model's layers, none twice; kv is a HOST array), as if all moved at once. A
 * parent outside 0..n_beams-1, or its own place, leaves a beam's rows as they
 * are. Beam b of request r is in slot slot[r*n_beams + b] (NULL: that number),
 * no two in one slot; a beam whose slot lies outside the cache neither takes
 * nor gives. since may be NULL (0); rows that all beams of a request share
 * need not be moved. n_beams is at most HAKO_MAX_BEAMS. */
int hako_gpu_kv_reorder(const hako_gpu_kv *kv, int n_kv, const int *slot, const int *parent, int n_req, int n_beams,
                        const int *since, const int *len);

/* ── drafted trees ──
 * A step takes n_seq trees of up to n_tree (1..HAKO_MAX_TREE) nodes, [n_seq]
 * [n_tree] in every array. Node 0 is the token that comes next in any case, a
 * node's parent comes before it: parent[0] = -1, 0 <= parent[j] < j. More
 * nodes of parent -1 are further roots. A node whose parent is anything else,
 * and every node after such a one, is not there: a padded tree ends in -2's.
 *
 * The cache holds positions below base[s] of slot[s] (NULL: slot s); node j's
 * keys and values go to row base[s] + j and are turned by its place in the
 * text, base[s] + its depth. A base below 0: the sequence has no nodes. */

/* A tree's plan: seen, for hako_gpu_attn_tree (bit i of node j: i is j or
 * leads to it; 0: not there), and for hako_gpu_kv_append_turned each node's
 * slot, row and turn (row and turn -1: not there, or past 2^31 - 1). Any of the four may be
 * NULL. It follows base; the layers of a step share it. */
int hako_gpu_tree_plan(const int *slot, const int *base, const int *parent, int n_seq, int n_tree, uint64_t *seen,
                       int *node_slot, int *row, int *turn);

/* The path that the model follows: from node 0 to the first child whose token
 * is the pick of the node before (pick[j]: the model's token after node j), as
 * far as there is one. path[s] gets the n_path[s] nodes, then -1's; next[s]
 * the pick of the last one, the token that comes next; new_base[s] = base[s] +
 * n_path[s]. A tree without node 0 has no path: n_path 0, next -1. base and
 * new_base may both be NULL. */
int hako_gpu_tree_accept(const int *parent, const int *token, const int *pick, const int *base, int n_seq, int n_tree,
                         int *path, int *n_path, int *next, int *new_base);

/* The path's rows together: row base[s] + path[s][d] to row base[s] + d for
 * d < n_path[s], as if all moved at once, in all n_kv caches (of one shape,
 * none twice; kv is a HOST array). Rows outside the cache, nodes outside the tree and a slot
 * outside the cache are left out, n_path past n_tree counts as n_tree. Then
 * positions below base[s] + n_path[s] are the text. No two sequences in one
 * slot. */
int hako_gpu_kv_keep(const hako_gpu_kv *kv, int n_kv, const int *slot, const int *base, const int *path,
                     const int *n_path, int n_seq, int n_tree);

#pragma GCC visibility pop

#ifdef __cplusplus
}
#endif
