/*
 * moe_attn.h -- C host side of the attention half of a layer, over libmoe_cuda:
 * projection to queries, keys and values, rotary positions, the paged cache,
 * attention, output projection.  What mda_qwen_attn_rec is to the reference's
 * layer (src/qwen.c, between the two mda_qwen_res_rec of mda_qwen_layer_rec),
 * for a plain causal softmax with grouped heads and a cache that the reference
 * does not keep.  The calling thread's current device is the context's.
 */
#ifndef MOE_ATTN_H
#define MOE_ATTN_H

#include <stdbool.h>
#include <stdint.h>

#include "moe_cuda.h"

typedef struct moe_attn_t {
    moe_cuda_ctx_t *c;
    uint32_t d, heads, kv_heads, hd, rot;
    float theta;
    uint32_t cols;      /* columns of the projection, a multiple of 128 */
    uint32_t rows, keys; /* most rows of one call; most cached keys that one prompt call reads back */
    void *p, *p16, *o16, *k16, *v16;
} moe_attn_t;

/* the weights of one layer's attention */
typedef struct moe_attn_w_t {
    const void *qkv; /* fp16 [cols x d]: heads * hd rows of queries, kv_heads * hd of keys, as many of values, zero rows */
    const void *out; /* fp16 [d x heads * hd] */
} moe_attn_w_t;

/* (heads + 2 kv_heads) * hd rounded up to 128 */
uint32_t moe_attn_cols(uint32_t heads, uint32_t kv_heads, uint32_t hd);
/* rot: columns of a head that turn, 0 for none.  keys: 0 if no prompt call will have cached prefixes.  d % 128 == 0. */
bool moe_attn_open(moe_attn_t *q, moe_cuda_ctx_t *c, uint32_t d, uint32_t heads, uint32_t kv_heads, uint32_t hd, uint32_t rot, float theta,
                   uint32_t rows, uint32_t keys);
void moe_attn_close(moe_attn_t *q);

/* One call's rows.  All pointers but the structs are device pointers; a16 [rows x d] is the cast of the layer's input (amax
 * and sa its scale slot, as for moe_cuda_dense), out fp32 [rows x d]. */
typedef struct moe_attn_rows_t {
    uint32_t rows, seqs;
    const void *a16;
    const uint32_t *amax;
    uint32_t sa;
    const uint32_t *pos;  /* [rows]: places of the tokens in their sequences */
    const uint32_t *slot; /* [rows]: where the cache keeps them */
    const uint32_t *table; /* [seqs x table_stride]: pages of the sequences */
    uint32_t table_stride;
    float *out;
} moe_attn_rows_t;

/* Both return false, with nothing enqueued, if the call does not fit (more rows than q->rows or keys than q->keys, a step whose rows
 * are not its sequences), and if the context has failed by then; what a kernel refuses shows at the next flush. */
/* Prompts: sequence s has rows cu_q[s] .. cu_q[s+1]-1, from 0 on; the output of rows behind the last one (a padded batch) is 0.
 * cu_k NULL: the sequences begin with them; else every sequence has cu_k[s+1] - cu_k[s] keys in the cache by then, these rows' own
 * among them, rows_k in all (at most q->keys). */
bool moe_attn_prompt(moe_attn_t *q, const moe_cuda_kv_t *kv, const moe_attn_w_t *w, const moe_attn_rows_t *r, const uint32_t *cu_q,
                     const uint32_t *cu_k, uint32_t rows_k);
/* One new token per sequence (rows == seqs); len[s] tokens with it, max_len at most. */
bool moe_attn_step(moe_attn_t *q, const moe_cuda_kv_t *kv, const moe_attn_w_t *w, const moe_attn_rows_t *r, const uint32_t *len,
                   uint32_t max_len);

#endif
