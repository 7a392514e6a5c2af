/* moe_attn.c -- see moe_attn.h. */
#include "moe_attn.h"

#include <math.h>
#include <stdio.h>
#include <string.h>

uint32_t moe_attn_cols(uint32_t heads, uint32_t kv_heads, uint32_t hd) { return ((heads + 2u * kv_heads) * hd + 127u) / 128u * 128u; }

bool moe_attn_open(moe_attn_t *q, moe_cuda_ctx_t *c, uint32_t d, uint32_t heads, uint32_t kv_heads, uint32_t hd, uint32_t rot, float theta,
                   uint32_t rows, uint32_t keys) {
    memset(q, 0, sizeof(*q));
    q->c = c;
    q->d = d;
    q->heads = heads;
    q->kv_heads = kv_heads;
    q->hd = hd;
    q->rot = rot;
    q->theta = theta;
    q->cols = moe_attn_cols(heads, kv_heads, hd);
    q->rows = rows;
    q->keys = keys;
    uint64_t r = rows, kept = (uint64_t)keys * kv_heads * hd * sizeof(uint16_t);
    q->p = moe_cuda_alloc(c, r * q->cols * sizeof(float));
    q->p16 = moe_cuda_alloc(c, r * q->cols * sizeof(uint16_t));
    q->o16 = moe_cuda_alloc(c, r * heads * hd * sizeof(uint16_t));
    q->k16 = keys != 0 ? moe_cuda_alloc(c, kept) : NULL;
    q->v16 = keys != 0 ? moe_cuda_alloc(c, kept) : NULL;
    return moe_cuda_status(c) == MOE_OK;
}

void moe_attn_close(moe_attn_t *q) {
    void *all[] = {q->p, q->p16, q->o16, q->k16, q->v16};
    for (uint32_t i = 0; i < sizeof(all) / sizeof(all[0]); i += 1) {
        moe_cuda_free(q->c, all[i]);
    }
    memset(q, 0, sizeof(*q));
}

static const uint16_t *moe_attn_col(const moe_attn_t *q, uint32_t head) { return (const uint16_t *)q->p16 + (uint64_t)head * q->hd; }

/* Projection, positions, cache. */
static bool moe_attn_begin(moe_attn_t *q, const moe_cuda_kv_t *kv, const moe_attn_w_t *w, const moe_attn_rows_t *r) {
    if (r->rows > q->rows) {
        fprintf(stderr, "moe_attn: %u rows, room for %u\n", r->rows, q->rows);
        return false;
    }
    struct moe_pc_dense_t pd = {
        .rows = r->rows,
        .n = q->cols,
        .k = q->d,
        .sa = r->sa,
    };
    moe_cuda_dense(q->c, r->a16, w->qkv, q->p, r->amax, pd);
    struct moe_pc_rope_t pr = {
        .rows = r->rows,
        .heads = q->heads + 2u * q->kv_heads,
        .rot_heads = q->rot != 0 ? q->heads + q->kv_heads : 0,
        .hd = q->hd,
        .rot = q->rot,
        .stride = q->cols,
        .out_stride = q->cols,
        .theta = q->theta,
    };
    moe_cuda_rope(q->c, q->p, r->pos, q->p16, pr);
    struct moe_pc_kv_write_t pw = {
        .rows = r->rows,
        .stride = q->cols,
    };
    moe_cuda_kv_write(q->c, kv, moe_attn_col(q, q->heads), moe_attn_col(q, q->heads + q->kv_heads), r->slot, pw);
    return true;
}

static void moe_attn_end(moe_attn_t *q, const moe_attn_w_t *w, const moe_attn_rows_t *r) {
    struct moe_pc_dense_t pd = {
        .rows = r->rows,
        .n = q->d,
        .k = q->heads * q->hd,
        .sa = MDA_PC_NO_SLOT,
    };
    moe_cuda_dense(q->c, q->o16, w->out, r->out, r->amax, pd);
}

bool moe_attn_prompt(moe_attn_t *q, const moe_cuda_kv_t *kv, const moe_attn_w_t *w, const moe_attn_rows_t *r, const uint32_t *cu_q,
                     const uint32_t *cu_k, uint32_t rows_k) {
    if (r->rows == 0) return moe_cuda_status(q->c) == MOE_OK;
    if (cu_k != NULL && rows_k > q->keys) {
        fprintf(stderr, "moe_attn: %u keys, room for %u\n", rows_k, q->keys);
        return false;
    }
    if (!moe_attn_begin(q, kv, w, r)) return false;
    struct moe_pc_attn_t pa = {
        .seqs = r->seqs,
        .rows_q = r->rows,
        .rows_k = r->rows,
        .heads = q->heads,
        .kv_heads = q->kv_heads,
        .hd = q->hd,
        .q_stride = q->cols,
        .kv_stride = q->cols,
        .o_stride = q->heads * q->hd,
        .scale = 1.0f / sqrtf((float)q->hd),
    };
    if (cu_k == NULL) {
        moe_cuda_attn(q->c, q->p16, moe_attn_col(q, q->heads), moe_attn_col(q, q->heads + q->kv_heads), cu_q, cu_q, q->o16, pa);
    } else {
        struct moe_pc_kv_read_t pk = {
            .seqs = r->seqs,
            .rows = rows_k,
            .table_stride = r->table_stride,
            .stride = q->kv_heads * q->hd,
        };
        moe_cuda_kv_read(q->c, kv, r->table, cu_k, q->k16, q->v16, pk);
        pa.rows_k = rows_k;
        pa.kv_stride = q->kv_heads * q->hd;
        moe_cuda_attn(q->c, q->p16, q->k16, q->v16, cu_q, cu_k, q->o16, pa);
    }
    /* rows of a padded batch: nothing attends there, and an earlier call's output is not this one's */
    uint32_t row = q->heads * q->hd * (uint32_t)sizeof(uint16_t);
    if (r->seqs != 0) {
        moe_cuda_clear_behind(q->c, q->o16, cu_q + r->seqs, r->rows, row);
    } else { /* no sequence, so perhaps no offsets */
        moe_cuda_fill(q->c, q->o16, (uint64_t)r->rows * row, 0);
    }
    moe_attn_end(q, w, r);
    return moe_cuda_status(q->c) == MOE_OK;
}

bool moe_attn_step(moe_attn_t *q, const moe_cuda_kv_t *kv, const moe_attn_w_t *w, const moe_attn_rows_t *r, const uint32_t *len,
                   uint32_t max_len) {
    if (r->rows == 0) return moe_cuda_status(q->c) == MOE_OK;
    if (r->rows != r->seqs) {
        fprintf(stderr, "moe_attn: a step has one row per sequence\n");
        return false;
    }
    if (!moe_attn_begin(q, kv, w, r)) return false;
    struct moe_pc_attn_decode_t pa = {
        .seqs = r->seqs,
        .heads = q->heads,
        .max_len = max_len,
        .table_stride = r->table_stride,
        .q_stride = q->cols,
        .o_stride = q->heads * q->hd,
        .scale = 1.0f / sqrtf((float)q->hd),
    };
    moe_cuda_attn_decode(q->c, kv, q->p16, r->table, len, q->o16, pa);
    moe_attn_end(q, w, r);
    return moe_cuda_status(q->c) == MOE_OK;
}
