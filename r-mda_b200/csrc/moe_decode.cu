// Attention of one new token per sequence over the paged key-value cache.
//
// Bound by HBM: every cached key and value is read once, and a group of g query heads does 2 g operations per fp16 element.
// The work is a line: sequence by sequence, head by head, stages of 16 SG cached tokens.  Every warp of a full chip takes an
// equal piece of the line whatever the lengths are, so no SM waits for another, and walks it alone: its loads run through a
// ring in shared memory that only it uses (each lane copies exactly the 16-byte pieces it will need as matrix fragments,
// so the ring needs no barriers and no swizzle), and the ring keeps running across the ends of heads and sequences.
// A (sequence, head) that lies within one warp's piece is written out at once; the others leave their running maximum, sum and
// unnormalised output in the context's work area, and a second small kernel joins them in the line's order.
//
// Fragments: scores are computed as S^T = K Q^T (16 tokens x 8 heads x 16 per mma.sync) and outputs as O^T = V^T P^T, so groups
// of up to 8 heads waste nothing.  The order of K's columns inside a product is free (Q's is the same), and so is the
// order of V's columns across products; both are chosen such that a lane's operands are contiguous 16 bytes in the cache.
// P^T comes from S^T's accumulators by an 8x8 transpose (movmatrix).
#include "moe_attn.cuh"
#include "moe_tc.cuh"

namespace {

using moe_tc::pack_h2;
using moe_tc::smem_u32;

constexpr uint32_t DEC_WARPS = 8, DEC_THREADS = DEC_WARPS * 32;
constexpr float LOG2E = 1.4426950408889634f;
// Weights are exp2(x - max + WEIGHT_SHIFT): 2^10 at most, so that fp16 holds weights down to 2^-34 of the largest.
constexpr float WEIGHT_SHIFT = 10.0f;

struct DecArgs {
    const uint8_t *k, *v;
    const float *k_scale, *v_scale;
    const __half *q;
    const uint32_t *table, *len;
    __half *o;
    unsigned long long *base;  // [seqs + 1]: stages of all sequences before s, of one head
    float *part;               // [2 * warps][part_floats: g * hd outputs, g maxima, g sums]
    uint32_t pages, page, page_shift, kv_heads, group;
    uint32_t seqs, max_len, table_stride, q_stride, o_stride;
    uint32_t warps;            // of the grid; part of the line that each takes follows from it and the line's length
    float scale;
    uint32_t *status;
};

// Floats of one warp's unfinished head: a multiple of four, so that every one begins at 16 bytes.
__host__ __device__ __forceinline__ uint32_t part_floats(uint32_t group, uint32_t hd) { return (group * (hd + 2u) + 3u) & ~3u; }

// Stages (of `per` tokens) of sequence s; a length beyond max_len counts as none.
__device__ __forceinline__ uint32_t stages_of(const DecArgs &a, uint32_t s, uint32_t per) {
    const uint32_t n = a.len[s];
    return n > a.max_len ? 0u : (n + per - 1u) / per;
}

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <uint32_t BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void *src, bool valid) {  // not valid: zeros, nothing is read
    const uint32_t n = valid ? BYTES : 0u;
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint2 ld_shared8(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float ld_shared_f(uint32_t at) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Sizes of one stage of one warp's ring.
template <uint32_t HD, bool FP8>
struct Stage {
    static constexpr uint32_t ES = FP8 ? 1 : 2;
    static constexpr uint32_t SG = HD == 128 && !FP8 ? 1 : 2;       // groups of 16 tokens
    static constexpr uint32_t TOKENS = 16 * SG;
    static constexpr uint32_t KP = HD * ES / 64;                    // 16-byte pieces of a K row per lane (4 lanes a row)
    static constexpr uint32_t VB = HD * ES / 8 > 16 ? 16 : HD * ES / 8;  // bytes of a V piece (8 lanes a row)
    static constexpr uint32_t VP = HD * ES / 8 / VB;                // V pieces per token and lane
    static constexpr uint32_t K_BYTES = 2 * KP * 512;               // of 16 tokens
    static constexpr uint32_t V_BYTES = 4 * VP * VB * 32;
    static constexpr uint32_t GROUP_BYTES = K_BYTES + V_BYTES + (FP8 ? 128 : 0);
    static constexpr uint32_t BYTES = SG * GROUP_BYTES;
    // about 26 KB per warp: eight warps then keep 150 to 200 KB of an SM's shared memory in flight, three times what
    // HBM's latency asks for
    static constexpr uint32_t COUNT = 26000 / BYTES;
};

// A place on the line: stage `g` of head h of sequence s.
struct Place {
    uint32_t s, h, g, stages, len;
};

__device__ __forceinline__ void place_next(const DecArgs &a, Place &p, uint32_t per) {
    p.g += 1;
    if (p.g < p.stages) return;
    p.g = 0;
    p.h += 1;
    if (p.h < a.kv_heads) return;
    p.h = 0;
    do {
        p.s += 1;
        p.stages = p.s < a.seqs ? stages_of(a, p.s, per) : 1u;  // behind the last: anything, it is not used
    } while (p.stages == 0u);
    p.len = p.s < a.seqs ? a.len[p.s] : 0u;
}

// Where the j-th of `warps` pieces of a line of `total` stages begins.
__device__ __forceinline__ unsigned long long piece_begin(unsigned long long total, uint32_t j, uint32_t warps) {
    return total * j / warps;
}

template <uint32_t HD, uint32_t NT, bool FP8>
__global__ void __launch_bounds__(DEC_THREADS, 1) moe_attn_decode_kernel(DecArgs a) {
    using St = Stage<HD, FP8>;
    constexpr uint32_t MT = HD / 16, SG = St::SG, PER = St::TOKENS;
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ unsigned long long before[DEC_THREADS + 1];
    __shared__ unsigned long long warp_sum[DEC_WARPS];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, r = lane >> 2, c = lane & 3u;
    moe_pdl_begin();

    // ---- the line: stages before each thread's share of the sequences -----------------------------
    const uint32_t share = (a.seqs + DEC_THREADS - 1u) / DEC_THREADS;
    const uint32_t s_lo = min(threadIdx.x * share, a.seqs), s_hi = min(s_lo + share, a.seqs);
    unsigned long long mine = 0;
    for (uint32_t s = s_lo; s < s_hi; s += 1) mine += stages_of(a, s, PER);
    unsigned long long incl = mine;
#pragma unroll
    for (uint32_t o = 1; o < 32; o <<= 1) {
        const unsigned long long up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    unsigned long long first = incl - mine;
#pragma unroll
    for (uint32_t w = 0; w < DEC_WARPS; w += 1) first += w < warp ? warp_sum[w] : 0ull;
    before[threadIdx.x] = first;
    if (threadIdx.x == DEC_THREADS - 1u) before[DEC_THREADS] = first + mine;
    if (blockIdx.x == 0) {  // for the joining kernel
        unsigned long long at = first;
        for (uint32_t s = s_lo; s < s_hi; s += 1) {
            a.base[s] = at;
            at += stages_of(a, s, PER);
            if (a.len[s] > a.max_len) moe_deny(a.status, MOE_SITE_LENGTH);
        }
        if (threadIdx.x == DEC_THREADS - 1u) a.base[a.seqs] = first + mine;
    }
    __syncthreads();
    const unsigned long long total = before[DEC_THREADS] * a.kv_heads;
    const uint32_t warps = total < a.warps ? (uint32_t)total : a.warps;
    const uint32_t me = warp * gridDim.x + blockIdx.x;  // neighbours on the line run on different SMs
    if (me >= warps) return;
    const unsigned long long x0 = piece_begin(total, me, warps);
    uint32_t left = (uint32_t)(piece_begin(total, me + 1u, warps) - x0);

    // ---- its beginning -----------------------------------------------------------------------------
    uint32_t owner = 0;  // the last thread share that begins at or before x0 (and is not empty)
#pragma unroll
    for (uint32_t i = 0; i < DEC_THREADS / 32u; i += 1) {
        const uint32_t t = i * 32u + lane;
        const uint32_t has = __ballot_sync(0xffffffffu, before[t] * a.kv_heads <= x0 && x0 < before[t + 1u] * a.kv_heads);
        if (has != 0) owner = i * 32u + (uint32_t)__ffs((int)has) - 1u;
    }
    Place p;
    {
        unsigned long long at = before[owner] * a.kv_heads;
        p.s = owner * share;
        p.stages = stages_of(a, p.s, PER);
        while (x0 - at >= (unsigned long long)p.stages * a.kv_heads) {
            at += (unsigned long long)p.stages * a.kv_heads;
            p.s += 1;
            p.stages = stages_of(a, p.s, PER);
        }
        p.h = (uint32_t)((x0 - at) / p.stages);
        p.g = (uint32_t)(x0 - at - (unsigned long long)p.h * p.stages);
        p.len = a.len[p.s];
    }

    const uint32_t ring0 = smem_u32(ring) + warp * St::COUNT * St::BYTES;
    Place q = p;             // the next stage to load, and the pages of its groups
    uint32_t to_load = left;
    uint32_t pg[SG];
    auto look_up = [&]() {
#pragma unroll
        for (uint32_t i = 0; i < SG; i += 1) {
            const uint32_t t = q.g * PER + i * 16u;
            pg[i] = to_load != 0 && t < q.len ? a.table[(size_t)q.s * a.table_stride + (t >> a.page_shift)] : 0u;
        }
    };
    uint32_t bad = 0;  // bit to * SG + i: group i of the stage in ring place `to` lies on a refused page
    // Copies of the next stage into ring place `to`.
    auto load = [&](uint32_t to) {
        if (to_load != 0) {
            const uint32_t dst0 = ring0 + to * St::BYTES;
#pragma unroll
            for (uint32_t i = 0; i < SG; i += 1) {
                const uint32_t t = q.g * PER + i * 16u;
                const bool page_ok = pg[i] < a.pages;
                if (!page_ok && lane == 0) moe_deny(a.status, MOE_SITE_PAGE);
                bad = (bad & ~(1u << (to * SG + i))) | (page_ok ? 0u : 1u << (to * SG + i));
                const size_t row = ((((size_t)(page_ok ? pg[i] : 0u) * a.kv_heads + q.h) << a.page_shift) + (t & (a.page - 1u)));
                const uint32_t n = page_ok && t < q.len ? q.len - t : 0u;  // valid tokens from the group's first on
                const uint32_t dst = dst0 + i * St::GROUP_BYTES;
#pragma unroll
                for (uint32_t j = 0; j < 2u * St::KP; j += 1) {
                    const uint32_t tok = r + 8u * (j / St::KP), piece = (j % St::KP) * 4u + c;
                    copy_async<16>(dst + (j * 32u + lane) * 16u, a.k + (row + tok) * (HD * St::ES) + piece * 16u, tok < n);
                }
#pragma unroll
                for (uint32_t j = 0; j < 4u * St::VP; j += 1) {
                    const uint32_t e = j / St::VP, tok = 2u * c + (e & 1u) + (e >> 1) * 8u, piece = (j % St::VP) * 8u + r;
                    copy_async<St::VB>(dst + St::K_BYTES + (j * 32u + lane) * St::VB, a.v + (row + tok) * (HD * St::ES) + piece * St::VB,
                                       tok < n);
                }
                if (FP8 && lane < 8u) {
                    const float *from = (lane < 4u ? a.k_scale : a.v_scale) + row + (lane & 3u) * 4u;
                    copy_async<16>(dst + St::K_BYTES + St::V_BYTES + lane * 16u, from, n != 0);
                }
            }
            to_load -= 1;
            if (to_load != 0) place_next(a, q, PER);
            look_up();
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    look_up();
#pragma unroll
    for (uint32_t i = 0; i < St::COUNT - 1u; i += 1) load(i);

    const float to_log2 = a.scale * LOG2E;
    uint32_t qf[NT][HD / 32u][4];   // Q^T fragments: words 2i, 2i+1 feed product i of a piece's pair
    float o[MT][NT][4], top[NT][2], sum[NT][2];
    uint32_t place = 0, begun_at = p.g;
    bool fresh = true;
    while (left != 0) {
        if (fresh) {
            fresh = false;
            begun_at = p.g;
#pragma unroll
            for (uint32_t n = 0; n < NT; n += 1) {
                const uint32_t head = n * 8u + r;
                const __half *row = a.q + (size_t)p.s * a.q_stride + (size_t)(p.h * a.group + head) * HD;
#pragma unroll
                for (uint32_t j = 0; j < HD / 32u; j += 1) {
                    // fp16: piece j of 8 columns; e4m3: a piece is 16 columns, j counts its halves
                    const uint32_t col = FP8 ? ((j / 2u) * 4u + c) * 16u + (j & 1u) * 8u : (j * 4u + c) * 8u;
                    uint4 w = make_uint4(0, 0, 0, 0);
                    if (head < a.group) w = *reinterpret_cast<const uint4 *>(row + col);
                    qf[n][j][0] = w.x;
                    qf[n][j][1] = w.y;
                    qf[n][j][2] = w.z;
                    qf[n][j][3] = w.w;
                }
                top[n][0] = top[n][1] = -INFINITY;
                sum[n][0] = sum[n][1] = 0.0f;
#pragma unroll
                for (uint32_t i = 0; i < MT; i += 1) {
#pragma unroll
                    for (uint32_t e = 0; e < 4; e += 1) o[i][n][e] = 0.0f;
                }
            }
        }
        load(place == 0 ? St::COUNT - 1u : place - 1u);  // into the place whose stage has just been used
        asm volatile("cp.async.wait_group %0;" ::"n"(St::COUNT - 1u) : "memory");
        __syncwarp();
        const uint32_t at = ring0 + place * St::BYTES;

        // ---- scores: rows r and r + 8 of each group are tokens, columns 2c and 2c + 1 of each n are heads ----
        float x[SG][NT][4], inv[SG][2];
#pragma unroll
        for (uint32_t i = 0; i < SG; i += 1) {
            const uint32_t kb = at + i * St::GROUP_BYTES;
            float s[2][NT][4];
#pragma unroll
            for (uint32_t n = 0; n < NT; n += 1) {
#pragma unroll
                for (uint32_t e = 0; e < 4; e += 1) s[0][n][e] = s[1][n][e] = 0.0f;
            }
#pragma unroll
            for (uint32_t j = 0; j < St::KP; j += 1) {
                const uint4 lo = ld_shared16(kb + (j * 32u + lane) * 16u), hi = ld_shared16(kb + ((St::KP + j) * 32u + lane) * 16u);
                const uint32_t l[4] = {lo.x, lo.y, lo.z, lo.w}, h[4] = {hi.x, hi.y, hi.z, hi.w};
                if (!FP8) {
#pragma unroll
                    for (uint32_t n = 0; n < NT; n += 1) {
                        mma_16816(s[0][n], l[0], h[0], l[1], h[1], qf[n][j][0], qf[n][j][1]);
                        mma_16816(s[1][n], l[2], h[2], l[3], h[3], qf[n][j][2], qf[n][j][3]);
                    }
                } else {
#pragma unroll
                    for (uint32_t w = 0; w < 4; w += 1) {  // a word is four columns of the product
                        const uint32_t a0 = e4m3x2_to_h2(l[w] & 0xffffu), a2 = e4m3x2_to_h2(l[w] >> 16);
                        const uint32_t a1 = e4m3x2_to_h2(h[w] & 0xffffu), a3 = e4m3x2_to_h2(h[w] >> 16);
#pragma unroll
                        for (uint32_t n = 0; n < NT; n += 1) {
                            const uint32_t f = (w & 1u) * 2u;
                            mma_16816(s[w & 1u][n], a0, a1, a2, a3, qf[n][2u * j + w / 2u][f], qf[n][2u * j + w / 2u][f + 1u]);
                        }
                    }
                }
            }
            const uint32_t t0 = p.g * PER + i * 16u;
#pragma unroll
            for (uint32_t half = 0; half < 2; half += 1) {
                float ks = to_log2, lv = 0.0f;
                inv[i][half] = 1.0f;
                if (FP8) {
                    const uint32_t sc = kb + St::K_BYTES + St::V_BYTES + (r + 8u * half) * 4u;
                    const float vs = ld_shared_f(sc + 64u);
                    ks *= ld_shared_f(sc);
                    // V's scale enters as a part of the exponent, so that weights keep their precision whatever the scales are
                    lv = __log2f(vs);
                    inv[i][half] = __frcp_rn(vs);
                }
                const bool seen = t0 + r + 8u * half < p.len && (bad >> (place * SG + i) & 1u) == 0u;
#pragma unroll
                for (uint32_t n = 0; n < NT; n += 1) {
#pragma unroll
                    for (uint32_t e = 0; e < 2; e += 1) {
                        x[i][n][half * 2u + e] = seen ? (s[0][n][half * 2u + e] + s[1][n][half * 2u + e]) * ks + lv : -INFINITY;
                    }
                }
                if (!seen) inv[i][half] = 0.0f;
            }
        }

        // ---- softmax: running maximum of each head, weights, their sum ----
        bool moves = false;
        float shift[NT][2], keep[NT][2];
#pragma unroll
        for (uint32_t n = 0; n < NT; n += 1) {
#pragma unroll
            for (uint32_t e = 0; e < 2; e += 1) {
                float m = top[n][e];
#pragma unroll
                for (uint32_t i = 0; i < SG; i += 1) m = fmaxf(m, fmaxf(x[i][n][e], x[i][n][2u + e]));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                keep[n][e] = m == top[n][e] ? 1.0f : exp2_fast(top[n][e] - m);
                moves |= m != top[n][e];
                top[n][e] = m;
                shift[n][e] = m == -INFINITY ? 0.0f : m - WEIGHT_SHIFT;
                sum[n][e] *= keep[n][e];
            }
        }
        if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
            for (uint32_t i = 0; i < MT; i += 1) {
#pragma unroll
                for (uint32_t n = 0; n < NT; n += 1) {
#pragma unroll
                    for (uint32_t e = 0; e < 4; e += 1) o[i][n][e] *= keep[n][e & 1u];
                }
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < SG; i += 1) {
            uint32_t pf[NT][2];
#pragma unroll
            for (uint32_t n = 0; n < NT; n += 1) {
#pragma unroll
                for (uint32_t half = 0; half < 2; half += 1) {
                    const float w0 = exp2_fast(x[i][n][half * 2u] - shift[n][0]), w1 = exp2_fast(x[i][n][half * 2u + 1u] - shift[n][1]);
                    sum[n][0] += w0 * inv[i][half];
                    sum[n][1] += w1 * inv[i][half];
                    // weights round to fp16 for the product (11 bits, as many as the output has); their sum does not
                    pf[n][half] = transpose_8x8(pack_h2(w0, w1));
                }
            }
            // ---- outputs: O^T += V^T P^T, 16 columns of V at a time ----
            const uint32_t vb = at + i * St::GROUP_BYTES + St::K_BYTES;
            uint32_t w[4][MT];  // [token 2c, 2c+1, 2c+8, 2c+9][pairs of columns]: first MT / 2 words row r, then row r + 8
#pragma unroll
            for (uint32_t e = 0; e < 4; e += 1) {
                if (!FP8) {
#pragma unroll
                    for (uint32_t j = 0; j < St::VP; j += 1) {
                        const uint4 v = ld_shared16(vb + ((e * St::VP + j) * 32u + lane) * 16u);
                        w[e][4u * j] = v.x;
                        w[e][4u * j + 1u] = v.y;
                        w[e][4u * j + 2u] = v.z;
                        w[e][4u * j + 3u] = v.w;
                    }
                } else {
                    uint32_t v[4];
                    if (HD == 128) {
                        const uint4 y = ld_shared16(vb + (e * 32u + lane) * 16u);
                        v[0] = y.x;
                        v[1] = y.y;
                        v[2] = y.z;
                        v[3] = y.w;
                    } else {
                        const uint2 y = ld_shared8(vb + (e * 32u + lane) * 8u);
                        v[0] = y.x;
                        v[1] = y.y;
                    }
#pragma unroll
                    for (uint32_t j = 0; j < MT / 2u; j += 1) {
                        w[e][2u * j] = e4m3x2_to_h2(v[j] & 0xffffu);
                        w[e][2u * j + 1u] = e4m3x2_to_h2(v[j] >> 16);
                    }
                }
            }
#pragma unroll
            for (uint32_t m = 0; m < MT; m += 1) {
                const uint32_t sel = (m & 1u) != 0 ? 0x7632u : 0x5410u;
                const uint32_t a0 = __byte_perm(w[0][m / 2u], w[1][m / 2u], sel), a1 = __byte_perm(w[0][MT / 2u + m / 2u], w[1][MT / 2u + m / 2u], sel);
                const uint32_t a2 = __byte_perm(w[2][m / 2u], w[3][m / 2u], sel), a3 = __byte_perm(w[2][MT / 2u + m / 2u], w[3][MT / 2u + m / 2u], sel);
#pragma unroll
                for (uint32_t n = 0; n < NT; n += 1) mma_16816(o[m][n], a0, a1, a2, a3, pf[n][0], pf[n][1]);
            }
        }

        // ---- the end of this head, or of the warp's piece ----
        left -= 1;
        place = place + 1u == St::COUNT ? 0u : place + 1u;
        const bool head_ends = p.g + 1u == p.stages;
        if (head_ends || left == 0) {
            fresh = true;
            const bool whole = head_ends && begun_at == 0;
            // columns of row half f and tile m: fp16 at 128 columns f * 64 + r * 8 + m, else r * HD/8 + f * HD/16 + m
            const uint32_t col0 = r * (HD == 128 && !FP8 ? 8u : HD / 8u), colf = HD == 128 && !FP8 ? 64u : HD / 16u;
#pragma unroll
            for (uint32_t n = 0; n < NT; n += 1) {
#pragma unroll
                for (uint32_t e = 0; e < 2; e += 1) {
                    float l = sum[n][e];
                    l += __shfl_xor_sync(0xffffffffu, l, 4);
                    l += __shfl_xor_sync(0xffffffffu, l, 8);
                    l += __shfl_xor_sync(0xffffffffu, l, 16);
                    const uint32_t head = n * 8u + 2u * c + e;
                    if (head >= a.group) continue;
                    if (whole) {
                        const float f = l == 0.0f ? 0.0f : 1.0f / l;
                        __half *out = a.o + (size_t)p.s * a.o_stride + (size_t)(p.h * a.group + head) * HD + col0;
#pragma unroll
                        for (uint32_t half = 0; half < 2; half += 1) {
#pragma unroll
                            for (uint32_t m = 0; m < MT; m += 4) {
                                *reinterpret_cast<uint2 *>(out + half * colf + m) =
                                    make_uint2(pack_h2(o[m][n][half * 2u + e] * f, o[m + 1u][n][half * 2u + e] * f),
                                               pack_h2(o[m + 2u][n][half * 2u + e] * f, o[m + 3u][n][half * 2u + e] * f));
                            }
                        }
                    } else {
                        // place 0: the piece began inside this head; place 1: the head goes on in the next warp's piece
                        float *part = a.part + (size_t)(me * 2u + (begun_at == 0 ? 1u : 0u)) * part_floats(a.group, HD);
                        if (r == 0) {
                            part[a.group * HD + head] = top[n][e];
                            part[a.group * (HD + 1u) + head] = l;
                        }
                        part += head * HD + col0;
#pragma unroll
                        for (uint32_t half = 0; half < 2; half += 1) {
#pragma unroll
                            for (uint32_t m = 0; m < MT; m += 4) {
                                *reinterpret_cast<float4 *>(part + half * colf + m) =
                                    make_float4(o[m][n][half * 2u + e], o[m + 1u][n][half * 2u + e], o[m + 2u][n][half * 2u + e],
                                                o[m + 3u][n][half * 2u + e]);
                            }
                        }
                    }
                }
            }
        }
        if (left != 0) place_next(a, p, PER);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// One block per (sequence, kv head): joins the pieces of a head that several warps worked on, in the line's order, and writes
// zeros for an empty sequence.
template <uint32_t HD>
__global__ void __launch_bounds__(128) moe_attn_join_kernel(DecArgs a) {
    moe_pdl_begin();
    const uint32_t s = blockIdx.x / a.kv_heads, h = blockIdx.x - s * a.kv_heads;
    const unsigned long long b0 = a.base[s], stages = a.base[s + 1u] - b0;
    __half *out = a.o + (size_t)s * a.o_stride + (size_t)h * a.group * HD;
    const uint32_t units = a.group * HD / 4u;
    if (stages == 0) {
        for (uint32_t u = threadIdx.x; u < units; u += blockDim.x) *reinterpret_cast<uint2 *>(out + u * 4u) = make_uint2(0, 0);
        return;
    }
    const unsigned long long total = a.base[a.seqs] * a.kv_heads, x0 = b0 * a.kv_heads + h * stages, x1 = x0 + stages;
    const uint32_t warps = total < a.warps ? (uint32_t)total : a.warps;
    // the piece that holds x: the largest j with total * j / warps <= x
    const uint32_t w0 = (uint32_t)(((x0 + 1u) * warps - 1u) / total), w1 = (uint32_t)((x1 * warps - 1u) / total);
    if (w0 == w1) return;
    const uint32_t size = part_floats(a.group, HD);
    for (uint32_t u = threadIdx.x; u < units; u += blockDim.x) {
        const uint32_t head = u / (HD / 4u);
        float top = -INFINITY;
        for (uint32_t w = w0; w <= w1; w += 1) top = fmaxf(top, a.part[(size_t)(w * 2u + (w == w0 ? 1u : 0u)) * size + a.group * HD + head]);
        float sum = 0.0f;
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (uint32_t w = w0; w <= w1; w += 1) {
            const float *part = a.part + (size_t)(w * 2u + (w == w0 ? 1u : 0u)) * size;
            const float m = part[a.group * HD + head];
            const float f = m == top ? 1.0f : exp2_fast(m - top);
            const float4 v = *reinterpret_cast<const float4 *>(part + u * 4u);
            sum += f * part[a.group * (HD + 1u) + head];
            y.x += f * v.x;
            y.y += f * v.y;
            y.z += f * v.z;
            y.w += f * v.w;
        }
        const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
        *reinterpret_cast<uint2 *>(out + u * 4u) = make_uint2(pack_h2(y.x * f, y.y * f), pack_h2(y.z * f, y.w * f));
    }
}

template <uint32_t HD, uint32_t NT, bool FP8>
void decode_launch(moe_cuda_ctx *c, const DecArgs &a, uint32_t slot) {
    constexpr uint32_t smem = DEC_WARPS * Stage<HD, FP8>::COUNT * Stage<HD, FP8>::BYTES;
    if (!c->dec_attr_set[slot]) {
        MOE_CUDA_TRY(c, cudaFuncSetAttribute(moe_attn_decode_kernel<HD, NT, FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        c->dec_attr_set[slot] = true;
    }
    moe_run(c, moe_attn_decode_kernel<HD, NT, FP8>, (uint32_t)c->sm_count, DEC_THREADS, smem, a);
    MOE_LAUNCHED(c);
    moe_run(c, moe_attn_join_kernel<HD>, a.seqs * a.kv_heads, 128, 0, a);
    MOE_LAUNCHED(c);
}

}  // namespace

extern "C" void moe_cuda_attn_decode(moe_cuda_ctx_t *c, const moe_cuda_kv_t *kv, const void *q16, const uint32_t *table, const uint32_t *len,
                                     void *o16, struct moe_pc_attn_decode_t pc) {
    if (!MOE_LIVE(c)) return;
    const char *why = moe_attn_decode_refusal(kv, q16, table, len, o16, pc);
    MOE_REQUIRE(c, why == NULL, "%s", why);
    if (pc.seqs == 0) return;
    DecArgs a;
    a.k = (const uint8_t *)kv->k;
    a.v = (const uint8_t *)kv->v;
    a.k_scale = kv->k_scale;
    a.v_scale = kv->v_scale;
    a.q = (const __half *)q16;
    a.table = table;
    a.len = len;
    a.o = (__half *)o16;
    a.pages = kv->pages;
    a.page = kv->page;
    a.page_shift = moe_log2(kv->page);
    a.kv_heads = kv->kv_heads;
    a.group = pc.heads / kv->kv_heads;
    a.seqs = pc.seqs;
    a.max_len = pc.max_len;
    a.table_stride = pc.table_stride;
    a.q_stride = pc.q_stride;
    a.o_stride = pc.o_stride;
    a.warps = (uint32_t)c->sm_count * DEC_WARPS;
    a.scale = pc.scale;
    a.status = c->dev_status_dev;
    const size_t base_bytes = (((size_t)pc.seqs + 1u) * 8u + 255u) & ~(size_t)255u;
    const size_t part_bytes = (size_t)a.warps * 2u * part_floats(a.group, kv->hd) * 4u;
    if (base_bytes + part_bytes > c->work_bytes) {
        moe_fail(c, MOE_ERR_NOMEM, "attn_decode: %zu bytes of work area, the context has %zu", base_bytes + part_bytes, c->work_bytes);
        return;
    }
    a.base = (unsigned long long *)c->work;
    a.part = (float *)((uint8_t *)c->work + base_bytes);
    moe_on_device on(c);
    const bool fp8 = kv->type == MOE_KV_E4M3, wide = a.group > 8u;
    if (kv->hd == 128u) {
        if (fp8) wide ? decode_launch<128, 2, true>(c, a, 0) : decode_launch<128, 1, true>(c, a, 1);
        else wide ? decode_launch<128, 2, false>(c, a, 2) : decode_launch<128, 1, false>(c, a, 3);
    } else {
        if (fp8) wide ? decode_launch<64, 2, true>(c, a, 4) : decode_launch<64, 1, true>(c, a, 5);
        else wide ? decode_launch<64, 2, false>(c, a, 6) : decode_launch<64, 1, false>(c, a, 7);
    }
}
