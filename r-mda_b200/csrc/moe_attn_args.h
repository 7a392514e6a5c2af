/* What the attention calls refuse, as plain C: each function returns NULL or the
 * reason.  Apart from the kernels so that it can be checked without a GPU. */
#ifndef MOE_ATTN_ARGS_H
#define MOE_ATTN_ARGS_H

#include <stddef.h>

#include "../../include/moe_cuda.h"

#define MOE_ATTN_MAX_GROUP 16u

#ifdef __CUDACC__
#define MOE_BOTH __host__ __device__
#else
#define MOE_BOTH
#endif

/* Parts that decode's join reads of a head which begins in SM `first`'s piece, of `sms` parts there are: n, or none if they
 * would pass the last.  What a piece that gave up leaves behind may be any number. */
MOE_BOTH static inline uint32_t moe_join_parts(uint32_t first, uint32_t n, uint32_t sms) { return first < sms && n <= sms - first ? n : 0u; }

static inline int moe_at16(const void *p) { return p != NULL && ((uintptr_t)p & 15u) == 0; }
static inline int moe_at4(const void *p) { return p != NULL && ((uintptr_t)p & 3u) == 0; }

/* Rows of `columns` fp16 values at a stride that 16-byte accesses can follow. */
static inline int moe_stride_ok(uint32_t stride, uint64_t columns) { return stride % 8u == 0 && stride >= columns; }

static inline const char *moe_rope_refusal(const void *x, const void *pos, const void *out, struct moe_pc_rope_t pc) {
    if (pc.heads == 0 || pc.hd == 0 || pc.hd % 8u != 0 || pc.hd > 65536u) return "rope: heads and hd (a multiple of 8) are at least one";
    if (pc.rot_heads > pc.heads) return "rope: rot_heads > heads";
    if (pc.rot_heads != 0 && (pc.rot == 0 || pc.rot % 8u != 0 || pc.rot > pc.hd || pc.rot > 512u)) return "rope: rot is a multiple of 8 up to hd and 512";
    if (pc.rot_heads != 0 && !(pc.theta > 0.0f && pc.theta <= 3.0e38f)) return "rope: theta is positive and finite";
    if ((uint64_t)pc.heads * pc.hd >= (1ull << 31)) return "rope: a row is too long";
    if (pc.stride % 4u != 0 || pc.stride < (uint64_t)pc.heads * pc.hd) return "rope: stride is a multiple of 4 and holds all heads";
    if (!moe_stride_ok(pc.out_stride, (uint64_t)pc.heads * pc.hd)) return "rope: out_stride is a multiple of 8 and holds all heads";
    if (pc.rows != 0 && (!moe_at16(x) || !moe_at16(out))) return "rope: x and out at 16-byte addresses";
    if (pc.rows != 0 && pc.rot_heads != 0 && !moe_at4(pos)) return "rope: pos";
    return NULL;
}

static inline const char *moe_kv_refusal(const moe_cuda_kv_t *kv) {
    if (kv == NULL) return "cache: null";
    if (kv->type != MOE_KV_F16 && kv->type != MOE_KV_E4M3) return "cache: type is MOE_KV_F16 or MOE_KV_E4M3";
    if (kv->hd != 64u && kv->hd != 128u) return "cache: hd is 64 or 128";
    if (kv->page < 16u || kv->page > 256u || (kv->page & (kv->page - 1u)) != 0) return "cache: page is a power of two from 16 to 256";
    if (kv->pages == 0 || (uint64_t)kv->pages * kv->page >= (1ull << 31)) return "cache: 1 to 2^31 - 1 slots";
    if (kv->kv_heads == 0 || kv->kv_heads > 1024u) return "cache: 1 to 1024 kv heads";
    if ((uint64_t)kv->pages * kv->page * kv->kv_heads >= (1ull << 31)) return "cache: slots * kv heads below 2^31";
    if (!moe_at16(kv->k) || !moe_at16(kv->v)) return "cache: k and v at 16-byte addresses";
    if (kv->type == MOE_KV_E4M3 && (!moe_at16(kv->k_scale) || !moe_at16(kv->v_scale))) return "cache: e4m3 needs scales, at 16-byte addresses";
    return NULL;
}

static inline const char *moe_kv_write_refusal(const moe_cuda_kv_t *kv, const void *k16, const void *v16, const void *slot,
                                               struct moe_pc_kv_write_t pc) {
    const char *why = moe_kv_refusal(kv);
    if (why != NULL) return why;
    if (!moe_stride_ok(pc.stride, (uint64_t)kv->kv_heads * kv->hd)) return "kv_write: stride is a multiple of 8 and holds all kv heads";
    if ((uint64_t)pc.rows * kv->kv_heads >= (1ull << 30)) return "kv_write: rows * kv_heads below 2^30";
    if (pc.rows != 0 && (!moe_at16(k16) || !moe_at16(v16) || !moe_at4(slot))) return "kv_write: k16 and v16 at 16-byte addresses, slot";
    return NULL;
}

static inline const char *moe_kv_read_refusal(const moe_cuda_kv_t *kv, const void *table, const void *cu, const void *k16, const void *v16,
                                              struct moe_pc_kv_read_t pc) {
    const char *why = moe_kv_refusal(kv);
    if (why != NULL) return why;
    if (!moe_stride_ok(pc.stride, (uint64_t)kv->kv_heads * kv->hd)) return "kv_read: stride is a multiple of 8 and holds all kv heads";
    if (pc.rows >= (1u << 31) || pc.seqs >= (1u << 20)) return "kv_read: rows below 2^31, seqs below 2^20";
    if (pc.rows != 0 && pc.seqs != 0 && (!moe_at16(k16) || !moe_at16(v16) || !moe_at4(table) || !moe_at4(cu)))
        return "kv_read: k16 and v16 at 16-byte addresses, table, cu";
    return NULL;
}

static inline const char *moe_clear_refusal(const void *out, const void *first, uint32_t rows, uint32_t row_bytes) {
    if (row_bytes % 16u != 0) return "clear_behind: rows of a multiple of 16 bytes";
    if (rows != 0 && row_bytes != 0 && (!moe_at16(out) || !moe_at4(first))) return "clear_behind: out at a 16-byte address, first";
    return NULL;
}

static inline const char *moe_heads_refusal(uint32_t heads, uint32_t kv_heads) {
    if (heads == 0 || kv_heads == 0 || heads % kv_heads != 0 || heads / kv_heads > MOE_ATTN_MAX_GROUP || kv_heads > 1024u)
        return "attention: 1 to 16 query heads for each of up to 1024 kv heads";
    return NULL;
}

static inline const char *moe_attn_refusal(const void *q16, const void *k16, const void *v16, const void *cu_q, const void *cu_k,
                                           const void *o16, struct moe_pc_attn_t pc) {
    const char *why = moe_heads_refusal(pc.heads, pc.kv_heads);
    if (why != NULL) return why;
    if (pc.hd != 64u && pc.hd != 128u) return "attn: hd is 64 or 128";
    if (!moe_stride_ok(pc.q_stride, (uint64_t)pc.heads * pc.hd) || !moe_stride_ok(pc.o_stride, (uint64_t)pc.heads * pc.hd) ||
        !moe_stride_ok(pc.kv_stride, (uint64_t)pc.kv_heads * pc.hd))
        return "attn: strides are multiples of 8 and hold all heads";
    if (pc.rows_q >= (1u << 31) || pc.rows_k >= (1u << 31) || pc.seqs >= (1u << 20)) return "attn: rows below 2^31, seqs below 2^20";
    if (!(pc.scale > 0.0f && pc.scale <= 1.0e4f)) return "attn: scale is positive, 10^4 at most";
    if (pc.rows_q != 0 && pc.seqs != 0) {
        if (!moe_at16(q16) || !moe_at16(o16) || !moe_at4(cu_q) || !moe_at4(cu_k)) return "attn: q16 and o16 at 16-byte addresses, cu_q, cu_k";
        if (pc.rows_k != 0 && (!moe_at16(k16) || !moe_at16(v16))) return "attn: k16 and v16 at 16-byte addresses";
    }
    return NULL;
}

static inline const char *moe_attn_decode_refusal(const moe_cuda_kv_t *kv, const void *q16, const void *table, const void *len,
                                                  const void *o16, struct moe_pc_attn_decode_t pc) {
    const char *why = moe_kv_refusal(kv);
    if (why == NULL) why = moe_heads_refusal(pc.heads, kv->kv_heads);
    if (why != NULL) return why;
    if (!moe_stride_ok(pc.q_stride, (uint64_t)pc.heads * kv->hd) || !moe_stride_ok(pc.o_stride, (uint64_t)pc.heads * kv->hd))
        return "attn_decode: strides are multiples of 8 and hold all heads";
    if (pc.seqs >= (1u << 20)) return "attn_decode: seqs below 2^20";
    if ((uint64_t)pc.table_stride * kv->page < pc.max_len || pc.max_len >= (1u << 31)) return "attn_decode: max_len needs more pages than a row of the table has";
    if (!(pc.scale > 0.0f && pc.scale <= 1.0e4f)) return "attn_decode: scale is positive, 10^4 at most";
    if (pc.seqs != 0 && (!moe_at16(q16) || !moe_at16(o16) || !moe_at4(len) || (pc.max_len != 0 && !moe_at4(table))))
        return "attn_decode: q16 and o16 at 16-byte addresses, table, len";
    return NULL;
}

#endif
