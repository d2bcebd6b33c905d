/* Serving operators over a paged KV cache: page tables and slot maps built on the GPU, RoPE with the
 * key and value rows written into the pages, attention of one query row per table row over them, and
 * penalties, biases and grammar masks on the logits. None has a counterpart in the reference, whose KV
 * cache is one contiguous tensor per layer (src/models/vkllm_kvcache.c) and whose token choice is a
 * plain argmax.
 *
 * A step of a server that batches requests runs vkllm_b200_paged_release for the sequences that ended
 * and vkllm_b200_paged_append for the new tokens; then per layer vkllm_b200_paged_rope_write and
 * vkllm_b200_paged_attention; then vkllm_b200_logits_apply before VKLLM_OP_ARG_MAX.
 *
 * Common to all: arrays are device (or managed) memory of the device that is current at the call, which
 * also owns `stream`; the structs, and the arrays of vkllm_b200_paged_check, are host memory. The work is
 * enqueued on `stream` (a cudaStream_t, NULL = the legacy default stream) and nothing waits; nothing is
 * allocated, so every call can be captured into a CUDA graph, whose replays read the arrays anew.
 * VKLLM_ERR_ARGS: an argument does not fit (a pointer that is not the current device's among them),
 * nothing was enqueued. VKLLM_ERR_VULKAN: a CUDA error.
 * Lengths, counts, page ids and slots in device memory that do not fit are found by the kernels: they
 * set bits of the device word *status (zeroed by the caller, only ever OR-ed into) and lead to no access
 * outside the arrays. One thing on the device they cannot check, since no length is given for it: the entries
 * of bias_starts in struct vkllm_b200_logit_rules have to lie within the two lists. */
#ifndef VKLLM_B200_PAGED_H
#define VKLLM_B200_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include "vkllm_dtypes.h"
#include "vkllm_errors.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Slot of a token without a cache row (padding): vkllm_b200_paged_rope_write skips it. */
#define VKLLM_B200_NO_SLOT 0xffffffffu

/* Bits of *status. */
enum
{
    VKLLM_B200_PAGED_BAD_PAGE = 1,  /* a page id >= n_pages in the table or the free list */
    VKLLM_B200_PAGED_TOO_LONG = 2,  /* a length passes cols * page_rows */
    VKLLM_B200_PAGED_NO_PAGES = 4,  /* append: more pages wanted than free (or *n_free > n_pages) */
    VKLLM_B200_PAGED_TOO_MANY = 8,  /* append: more new tokens than max_tokens; release: more pages than n_pages */
    VKLLM_B200_PAGED_BAD_SLOT = 16, /* rope_write: a slot >= n_pages * page_rows other than NO_SLOT */
    VKLLM_B200_PAGED_BAD_WORKSPACE = 32, /* attention: the workspace was not zero at first, or two calls
                                          * used it at the same time; rows of out are missing, and the
                                          * workspace has to be zeroed before its next use */
};

/* The page table of a batch of sequence slots. Row s of a sequence's cache is row s % page_rows of page
 * table[seq * stride + s / page_rows].
 * Every page of a table that vkllm_b200_paged_append or _release gets, and of its free list, is held once.
 * vkllm_b200_paged_check finds a page that is held twice; the calls on the device do not look for one. They
 * would hand it out while the other holder still reads it, or twice, or let both write its rows. Pages are
 * shared in tables that only the attention gets, whose rows name pages of such a table's sequences; a
 * sequence outlives those that read its pages. */
struct vkllm_b200_paged_table
{
    uint32_t *table;      /* device, [n_seqs] rows of cols page ids */
    uint32_t *free_pages; /* device, n_pages entries: a stack of *n_free ids; attention needs none (NULL) */
    uint64_t stride;      /* entries from one sequence's row to the next, >= cols */
    uint32_t n_seqs, cols, page_rows, n_pages;
};

/* The key and value pools of one layer. Element d of row r of key head h of page p is at
 * p * page_stride + h * head_stride + r * row_stride + d (in elements), so pages of whole heads
 * ([page][head][row][d]) and of whole rows ([page][row][head][d]) both fit, as do pools whose pages
 * lie inside a larger page. */
struct vkllm_b200_paged_kv
{
    void *k, *v; /* device, 16-byte aligned */
    uint64_t page_stride, head_stride, row_stride; /* multiples of 16 bytes */
    uint32_t n_pages, page_rows; /* n_pages * page_rows < 2^32 */
    uint32_t kv_heads;           /* <= 65535, as are the query heads, a multiple of them */
    uint32_t head_dim; /* <= 256, head_dim * element size a multiple of 16 */
    uint32_t dtype;    /* vkllm_dtype_float16 or vkllm_dtype_float32: of the pools, q, k, v and out */
    uint32_t reserved; /* 0 */
};

/* Host only: checks host copies of a table (all pointers in host memory) as the kernels do, and that no
 * page is held twice. `n_free` ids of free_pages are looked at (0: free_pages may be NULL). Returns
 * VKLLM_ERR_OK, or VKLLM_ERR_ARGS with *status (may be NULL) set to the bits above and *bad_seq (may be
 * NULL) to the first sequence at fault, n_seqs when it is the free list. */
extern vkllm_err_t vkllm_b200_paged_check(const struct vkllm_b200_paged_table *t, const uint32_t *lens, uint32_t n_free,
                                          uint32_t *status, uint32_t *bad_seq);

/* Makes room for n_new[s] more rows in every sequence slot s and says where they go.
 *   lens      [n_seqs] rows that each slot holds; new_lens [n_seqs] receives lens + n_new
 *   n_free    [1] free pages; n_free_out [1] receives what is left
 *   starts    [n_seqs + 1] receives the first new token of each slot (tokens are packed, slot by slot)
 *   slots     [max_tokens] receives page * page_rows + row of each token, VKLLM_B200_NO_SLOT past the last
 *   positions [max_tokens] receives each token's position in its sequence, 0 past the last
 * Pages come off the top of the free list, slot by slot and in order, and are written behind the ones
 * in the table (none of which two slots may hold); the rest of the table stays as it is. All or nothing:
 * when a length, the free list or max_tokens does not allow it, *status says so and the call does what it
 * would do for n_new all 0.
 * new_lens may be lens and n_free_out may be n_free (advance in place); other arrays must not overlap.
 * n_seqs <= 16384. max_tokens may be 0 (slots and positions may then be NULL). */
extern vkllm_err_t vkllm_b200_paged_append(const struct vkllm_b200_paged_table *t, const uint32_t *lens,
                                           const uint32_t *n_new, const uint32_t *n_free, uint32_t *new_lens,
                                           uint32_t *n_free_out, uint32_t *starts, uint32_t *slots, uint32_t *positions,
                                           uint32_t max_tokens, uint32_t *status, void *stream);

/* Gives the pages of every slot s with done[s] != 0 (none of which another slot may hold) back to the free
 * list, slot by slot, page by page, onto its top, and sets new_lens[s] to 0; new_lens[s] = lens[s] for the
 * others. All or nothing, as above; the table stays as it is. new_lens may be lens, n_free_out may be n_free.
 * n_seqs <= 16384. */
extern vkllm_err_t vkllm_b200_paged_release(const struct vkllm_b200_paged_table *t, const uint32_t *lens,
                                            const uint32_t *done, const uint32_t *n_free, uint32_t *new_lens,
                                            uint32_t *n_free_out, uint32_t *status, void *stream);

/* RoPE of new tokens and their rows of the cache: q_out = rotated q, key row = rotated k, value row = v,
 * with the pairs and angles of VKLLM_OP_ROPE (elements 2w and 2w + 1 turned by positions[t] *
 * rope_base^(-2w / head_dim); src/shaders/vkllm_rope.comp). Sines and cosines are off by at most 2^-22, at
 * far positions as at near ones.
 *   q [n_tokens] rows of heads * head_dim, k and v of kv_heads * head_dim, q_out as q; row strides in
 *   elements, multiples of 16 bytes, pointers 16-byte aligned: q, k and v may be parts of one row.
 *   heads a multiple of kv_heads; rope_base > 1 (<= 0: 10000). q_out may be q (same stride); it must not
 *   overlap q, k or v otherwise.
 * A token whose slot is VKLLM_B200_NO_SLOT leaves the cache and its q_out row as they were, and its rows
 * are not read; a token whose slot is outside the pool leaves both as they were and sets
 * VKLLM_B200_PAGED_BAD_SLOT. The other slots must differ. n_tokens may be 0. */
extern vkllm_err_t vkllm_b200_paged_rope_write(const struct vkllm_b200_paged_kv *kv, const void *q, uint64_t q_stride,
                                               const void *k, uint64_t k_stride, const void *v, uint64_t v_stride,
                                               const uint32_t *positions, const uint32_t *slots, uint32_t n_tokens,
                                               uint32_t heads, float rope_base, void *q_out, uint64_t q_out_stride,
                                               uint32_t *status, void *stream);

/* Size of the workspace that vkllm_b200_paged_attention asks for (the same for every shape). */
#define VKLLM_B200_PAGED_WORKSPACE_BYTES (16u << 20)

/* Attention of one query row per row of the table: out = softmax(scale q . K) V over the lens[s] cached
 * rows of table row s, for the query in row s of q; query head h reads key head h / (heads / kv_heads). This
 * is plain attention at every length (unlike VKLLM_OP_MATMUL, nothing depends on lens[s] == head_dim).
 *   q, out [n_seqs] rows of heads * head_dim, row strides in elements (multiples of 16 bytes, pointers
 *          16-byte aligned), of the pools' type; out must not overlap q
 *   lens   [n_seqs]; a row with 0 rows of cache, or whose every score is -infinity, gets a row of zeros; rows
 *          of the cache past lens[s] have no effect whatever they hold (no number, infinities)
 * Row s of q goes with row s of the table and nothing else: the table of the sequence slots fits the packed
 * rows of vkllm_b200_paged_append and _rope_write only in a step with exactly one new token in every slot. For
 * any other step (slots without a new token, prompts) the call takes a table of its own, a row per packed
 * token: row i a copy of its slot's row, lens[i] = positions[i] + 1 (so a prompt is causal), 0 past the last.
 *   workspace  16-byte aligned, VKLLM_B200_PAGED_WORKSPACE_BYTES, zero before its first use; every call
 *          leaves it ready for the next. Calls (and replays of captured calls) that may run at the same
 *          time need a workspace each.
 * A length past cols * page_rows is cut to it and a page id >= n_pages has no keys; both set *status.
 * Rows of the table may share pages (a table of the attention's own, not one that append and release keep:
 * see struct vkllm_b200_paged_table). Scores, softmax and sums are fp32 (an infinite value among the rows that
 * count makes its element of out infinite or no number). The same inputs give the same bits on the same
 * device. n_seqs <= 65535. */
extern vkllm_err_t vkllm_b200_paged_attention(const struct vkllm_b200_paged_kv *kv,
                                              const struct vkllm_b200_paged_table *t, const void *q, uint64_t q_stride,
                                              uint32_t heads, const uint32_t *lens, float scale, void *out,
                                              uint64_t out_stride, void *workspace, uint64_t workspace_bytes,
                                              uint32_t *status, void *stream);

/* Rules on a batch of logit rows. Every pointer is device memory; NULL turns its rule off. Row r's tokens
 * so far are history[r * history_stride + i], i < history_lens[r] (at most history_stride), the first
 * prompt_lens[r] of them (NULL: none) its prompt, the others generated. */
struct vkllm_b200_logit_rules
{
    const uint32_t *history, *prompt_lens, *history_lens;
    const float *repetition;      /* [rows], > 0: x / r where x > 0, else x * r, for ids in the history */
    const float *frequency;       /* [rows]: x - frequency * (times generated) */
    const float *presence;        /* [rows]: x - presence for ids generated at least once */
    const uint32_t *bias_starts;  /* [rows + 1], ascending: row r's biases are entries bias_starts[r] up to
                                   * bias_starts[r + 1] of the two lists below, which the caller answers for:
                                   * both must be at least bias_starts[rows] long (a row that would end
                                   * before it starts has none) */
    const uint32_t *bias_ids;     /* x + the id's value; of an id listed twice the sum, in the list's order */
    const float *bias_values;
    const uint32_t *mask;         /* bit id % 32 of word id / 32 of a row: 0 makes the logit -infinity */
    uint64_t history_stride, mask_stride; /* elements and words from row to row; history_stride < 2^30.
                                           * A stride past 2560 sets twice the shared memory aside, whatever
                                           * the lengths, for 8192 ids instead of 4096. A row's history and
                                           * biases that take more than 3/4 of these are read again for every
                                           * 8192 (4096) ids of vocab */
};

/* out = logits under the rules, in the order of the struct (repetition, frequency and presence, biases,
 * mask), in fp32 and rounded once. logits and out are rows of `vocab` elements of `dtype`
 * (vkllm_dtype_float16 or vkllm_dtype_float32), strides in elements; out may be logits (same stride) and
 * must not overlap otherwise. Ids >= vocab in the history and the biases are ignored. A mask that leaves a
 * row nothing gives a row of -infinity. rows <= 65535. */
extern vkllm_err_t vkllm_b200_logits_apply(const struct vkllm_b200_logit_rules *rules, const void *logits,
                                           uint64_t logits_stride, uint32_t rows, uint32_t vocab, uint32_t dtype,
                                           void *out, uint64_t out_stride, void *stream);

#ifdef __cplusplus
}
#endif
#endif
