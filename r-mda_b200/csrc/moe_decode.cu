// Attention of one new token per sequence over the paged key-value cache.
//
// Bound by HBM: every cached key and value is read once, and a group of g query heads does 2 g operations per fp16 element.
// The work is a line: sequence by sequence, head by head, stages of 16 or 32 cached tokens.  Every SM takes an equal piece of
// the line whatever the lengths are, and every warp an equal piece of that, so no one waits for another.  A warp walks its
// piece alone: its loads (TMA boxes of one page's tokens, swizzled) run through a ring in shared memory that only it uses, with
// barriers that only it waits at, and keep running across the ends of heads and sequences.  A (sequence, head) that lies within
// one warp's piece is written out at once; of the others each warp leaves its running maximum, sum and unnormalised output in
// shared memory, the SM's warps join them, and heads that reach over an SM's piece go through the context's work area to a
// second small kernel.  Everything is joined in the line's order.
//
// Scores are computed as S^T = K Q^T (16 tokens x 8 heads x 16 columns per mma.sync) and outputs as O^T = V^T P^T, so groups
// of up to 8 heads waste nothing; P^T comes from S^T's accumulators by an 8x8 transpose (movmatrix).  Operands come from shared
// memory by ldmatrix: fp16 as they are; of e4m3 a lane gets two pairs of neighbouring columns, which are converted in
// registers (the order of K's columns inside a product is free, Q's is the same).  A group is 8 of the 64 rows that the
// 5th-generation tensor cores' smallest product has, and the products are far from a bound here.
//
// One B200: 129 sequences of up to 8191 tokens, fp16, 4 kv heads of 128 (1.08 GB) 173 us, of which this kernel 166 = 6.5 TB/s, the
// copy rate; 16 of up to 16384, e4m3 (141 MB) 37 us, bound by the chain from codes to products in 8 warps (0.37 of the issue slots) and
// ~7 us of join and gaps; one of 777 tokens 9.3 us with the call, a chain of latencies: the line, the first loads, the joins.
#include "moe_attn.cuh"
#include "moe_tc.cuh"

namespace {

using namespace moe_tc;

constexpr float LOG2E = 1.4426950408889634f;
// Weights are taken against the running maximum less WEIGHT_SHIFT: 2^10 at most, so that fp16 holds weights down to 2^-34 of the largest.
constexpr float WEIGHT_SHIFT = 10.0f;

struct DecArgs {
    const float *k_scale, *v_scale;
    const __half *q;
    const uint32_t *table, *len;
    __half *o;
    uint4 *split;              // [SMs]: the head that begins in this SM's piece and goes on in others: sequence, kv head, first SM, SMs; 0 SMs: none
    float *part;               // [2 * SMs][part_floats: g * hd outputs, g maxima, g sums]: of a head begun earlier, of one that goes on
    uint32_t pages, page, page_shift, kv_heads, group;
    uint32_t seqs, max_len, table_stride, q_stride, o_stride;
    float scale;
    uint32_t *status;
    uint64_t wait_ns;
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
__device__ __forceinline__ void copy_async16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&v)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&v)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(at)
                 : "memory");
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

// Sizes of one stage of one warp's ring, and how many warps share an SM.
template <uint32_t HD, uint32_t NT, bool FP8>
struct Stage {
    static constexpr uint32_t WARPS = 8;
    static constexpr uint32_t THREADS = WARPS * 32;
    static constexpr uint32_t ROW = HD * (FP8 ? 1 : 2);             // bytes of a token's keys, or values
    static constexpr uint32_t LINE = ROW > 128 ? 128 : ROW;         // of them in one swizzled line; two halves if ROW is 256
    static constexpr uint32_t HALVES = ROW / LINE;
    static constexpr uint32_t SG = ROW == 256 ? 1 : 2;              // groups of 16 tokens
    static constexpr uint32_t TOKENS = 16 * SG;
    static constexpr uint32_t HALF_BYTES = TOKENS * LINE;
    static constexpr uint32_t K_BYTES = TOKENS * ROW;
    static constexpr uint32_t BYTES = 2 * K_BYTES;
    static constexpr uint32_t SCALES = FP8 ? 2 * TOKENS * 4 : 0;    // keys' scales, then values'
    static constexpr uint32_t PART = (8 * NT * (HD + 2) * 4 + 15) / 16 * 16;   // a part of a head, for the largest group
    static constexpr uint32_t ROOM = (218000 / WARPS - PART) / (BYTES + SCALES);
    static constexpr uint32_t COUNT = ROOM > 4 ? 4 : ROOM;
    static constexpr uint32_t RING = WARPS * COUNT * BYTES;
    static constexpr uint32_t PARTS = (RING + WARPS * COUNT * (SCALES + 8) + 15) / 16 * 16;   // where the parts of heads lie
    static constexpr uint32_t SMEM = PARTS + WARPS * PART + 1024;
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

// Bounded wait for a stage; false: gave up, the status says so.
__device__ __forceinline__ bool landed(uint32_t bar, uint32_t parity, const DecArgs &a) {
    uint32_t spins = 0;
    uint64_t t0 = 0;
    bool ok = true;
    while (!mbar_try_wait(bar, parity)) {
        spins += 1;
        if ((spins & 0xffu) != 0) continue;
        const uint64_t now = globaltimer_ns();
        if (t0 == 0) t0 = now;
        else if (now - t0 > a.wait_ns) {
            atomicCAS(a.status, 0u, (uint32_t)MOE_ERR_TIMEOUT | (42u << 8));
            ok = false;
            break;
        }
    }
    return __all_sync(0xffffffffu, ok);
}

// x * j / n, in 32 bits where they do (64-bit division takes hundreds of cycles).
__device__ __forceinline__ unsigned long long share_of(unsigned long long x, uint32_t j, uint32_t n) {
    return x < (1u << 22) ? (unsigned long long)((uint32_t)x * j / n) : x * j / n;   // j up to 2^10
}
// The last j with total * j / n <= x: the piece of n that holds stage x.
__device__ __forceinline__ uint32_t piece_of(unsigned long long x, unsigned long long total, uint32_t n) {
    return total < (1u << 22) ? (((uint32_t)x + 1u) * n - 1u) / (uint32_t)total : (uint32_t)(((x + 1u) * n - 1u) / total);
}

template <uint32_t HD, uint32_t NT, bool FP8>
__global__ void __launch_bounds__(Stage<HD, NT, FP8>::THREADS, 1)
moe_attn_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, DecArgs a) {
    using St = Stage<HD, NT, FP8>;
    constexpr uint32_t DEC_WARPS = St::WARPS, DEC_THREADS = St::THREADS;
    constexpr uint32_t MT = HD / 16, KS = HD / 16, SG = St::SG, PER = St::TOKENS;
    extern __shared__ uint8_t smem_raw[];
    __shared__ unsigned long long before[DEC_THREADS + 1];
    __shared__ unsigned long long warp_sum[DEC_WARPS];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, r = lane >> 2, c = lane & 3u;
    uint8_t *const smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *const my_ring = smem + warp * St::COUNT * St::BYTES;
    const uint32_t ring0 = smem_u32(my_ring), scales0 = smem_u32(smem) + St::RING + warp * St::COUNT * St::SCALES;
    const uint32_t bars0 = smem_u32(smem) + St::RING + DEC_WARPS * St::COUNT * St::SCALES + warp * St::COUNT * 8u;
    // parts of heads: a warp's first one, which begins before it, and its last one, which goes on behind it (in its ring, at the end)
    float *const ended = reinterpret_cast<float *>(smem + St::PARTS);
    auto goes_on = [&](uint32_t w) { return reinterpret_cast<float *>(smem + w * St::COUNT * St::BYTES); };
    __shared__ uint2 ended_of[DEC_WARPS], goes_on_of[DEC_WARPS];   // sequence and kv head; a sequence of ~0: none
    __shared__ bool begins[DEC_WARPS];   // the last one begins in the warp's piece
    __shared__ uint32_t behind;          // stages of the SM's last head behind its piece
    __shared__ bool gave_up;             // some warp's wait ran out: what it leaves is incomplete, `behind` may not have been written
    __shared__ uint4 over;               // the head that begins in the SM's piece and goes on behind it: sequence, kv head, first SM, SMs
    if (lane < St::COUNT) {
        mbar_init(bars0 + lane * 8u, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x == 0) {
        over = make_uint4(0, 0, 0, 0);
        behind = 0;
        gave_up = false;
    }
    moe_pdl_begin();

    // ---- the line: stages before each thread's share of the sequences -----------------------------
    const uint32_t share = (a.seqs + DEC_THREADS - 1u) / DEC_THREADS;
    const uint32_t s_lo = min(threadIdx.x * share, a.seqs), s_hi = min(s_lo + share, a.seqs);
    unsigned long long mine = 0;
    for (uint32_t s = s_lo; s < s_hi; s += 1) {
        const uint32_t n = a.len[s];
        if (n > a.max_len) {
            if (blockIdx.x == 0) moe_deny(a.status, MOE_SITE_LENGTH);   // here, before any return
        } else {
            mine += (n + PER - 1u) / PER;
        }
    }
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
    __syncthreads();
    const unsigned long long total = before[DEC_THREADS] * a.kv_heads;
    // SMs in use: as many as leave every warp at least a stage
    const uint32_t sms = (uint32_t)min((unsigned long long)gridDim.x, (total + DEC_WARPS - 1u) / DEC_WARPS);
    for (uint32_t s = warp * gridDim.x + blockIdx.x; s < a.seqs; s += DEC_WARPS * gridDim.x) {   // nothing to attend to: zeros
        if (stages_of(a, s, PER) != 0u) continue;
        __half *out = a.o + (size_t)s * a.o_stride;
        for (uint32_t i = lane * 8u; i < a.kv_heads * a.group * HD; i += 256u) *reinterpret_cast<uint4 *>(out + i) = make_uint4(0, 0, 0, 0);
    }
    if (blockIdx.x >= sms) {
        if (threadIdx.x == 0) a.split[blockIdx.x] = make_uint4(0, 0, 0, 0);
        return;
    }
    const unsigned long long sm0 = share_of(total, blockIdx.x, sms), sm1 = share_of(total, blockIdx.x + 1u, sms);
    const uint32_t warps = (uint32_t)min((unsigned long long)DEC_WARPS, sm1 - sm0);
    if (lane == 0) ended_of[warp] = goes_on_of[warp] = make_uint2(~0u, 0u);
    // a warp without a piece waits for the others at the first one's beginning
    const unsigned long long x0 = sm0 + (warp < warps ? share_of(sm1 - sm0, warp, warps) : 0ull);
    uint32_t left = warp < warps ? (uint32_t)(sm0 + share_of(sm1 - sm0, warp + 1u, warps) - x0) : 0u;

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
        const unsigned long long off = x0 - at;   // below stages * kv heads
        p.h = off < (1ull << 32) ? (uint32_t)off / p.stages : (uint32_t)(off / p.stages);
        p.g = (uint32_t)(off - (unsigned long long)p.h * p.stages);
        p.len = a.len[p.s];
    }

    auto sm_of = [&](unsigned long long x) { return piece_of(x, total, sms); };
    Place q = p;             // the next stage to load, and the pages of its boxes
    uint32_t to_load = left, pg[SG];
    const uint32_t box = a.page < PER ? a.page : PER;   // tokens of one box: a stage, or a page of 16 of a stage of 32
    auto look_up = [&]() {
#pragma unroll
        for (uint32_t i = 0; i < SG; i += 1) {
            const uint32_t t = q.g * PER + i * box;
            pg[i] = to_load != 0 && i * box < PER && t < q.len ? a.table[(size_t)q.s * a.table_stride + (t >> a.page_shift)] : 0u;
        }
    };
    uint32_t bad = 0;   // bit to * SG + i: box i of the stage in ring place `to` lies on a refused page
    // Copies of the next stage into ring place `to`.
    auto load = [&](uint32_t to) {
        if (to_load != 0) {
            const uint32_t bar = bars0 + to * 8u, dst = ring0 + to * St::BYTES;
            int32_t row[SG];
            uint32_t bytes = 0;
#pragma unroll
            for (uint32_t i = 0; i < SG; i += 1) {
                const uint32_t t = q.g * PER + i * box;
                const bool page_ok = pg[i] < a.pages, there = i * box < PER && t < q.len;
                if (there && !page_ok && lane == 0) moe_deny(a.status, MOE_SITE_PAGE);
                bad = (bad & ~(1u << (to * SG + i))) | ((page_ok ? 0u : 1u) << (to * SG + i));
                row[i] = there && page_ok ? (int32_t)(((pg[i] * a.kv_heads + q.h) << a.page_shift) + (t & (a.page - 1u))) : -1;
                bytes += row[i] >= 0 ? 2u * box * St::ROW : 0u;
                if (FP8 && row[i] >= 0 && lane < box / 2u) {
                    const uint32_t piece = lane % (box / 4u), is_v = lane / (box / 4u);
                    copy_async16(scales0 + to * St::SCALES + is_v * PER * 4u + i * box * 4u + piece * 16u,
                                 (is_v != 0 ? a.v_scale : a.k_scale) + row[i] + piece * 4u);
                }
            }
            if (elect_one()) {
                if (bytes != 0) mbar_expect_tx(bar, bytes);
                else mbar_arrive(bar);
#pragma unroll
                for (uint32_t i = 0; i < SG; i += 1) {
                    if (row[i] < 0) continue;
                    tma_load_3d(dst + i * box * St::LINE, &tm_k, bar, 0, row[i], 0);
                    tma_load_3d(dst + St::K_BYTES + i * box * St::LINE, &tm_v, bar, 0, row[i], 0);
                }
            }
            __syncwarp();
            to_load -= 1;
            if (to_load != 0) place_next(a, q, PER);
            look_up();
        }
        if (FP8) asm volatile("cp.async.commit_group;" ::: "memory");
    };
    look_up();
#pragma unroll
    for (uint32_t i = 0; i < St::COUNT - 1u; i += 1) load(i);

    // ldmatrix: lane l gives the address of row l % 8 of matrix l / 8.  Keys: matrices (tokens 0-7, 8-15) x (line piece 2s, 2s + 1);
    // values: the other way round.  Pieces of 16 bytes lie at piece ^ (row % 8) of a 128-byte line, piece ^ (row / 2 % 4) of a 64-byte one.
    auto piece_at = [&](uint32_t token, uint32_t piece) { return token * St::LINE + ((piece ^ (St::LINE == 128 ? token & 7u : (token >> 1) & 3u)) << 4); };
    const uint32_t k_at = piece_at((lane & 7u) + ((lane >> 3) & 1u) * 8u, lane >> 4);
    const uint32_t v_at = St::K_BYTES + piece_at((lane & 7u) + (lane >> 4) * 8u, (lane >> 3) & 1u);
    auto line_step = [](uint32_t at, uint32_t s) {   // two pieces on from `at`, s times: other bits of the same line, then the other half
        constexpr uint32_t PER_LINE = St::LINE / 32u;
        return (at ^ ((s % PER_LINE) * 32u)) + (s / PER_LINE) * St::HALF_BYTES;
    };
    const float to_log2 = a.scale * LOG2E;
    uint32_t qf[NT][KS][2];
    float o[MT][NT][4], top[NT][2], sum[NT][2];
    uint32_t place = 0, phase = 0, begun_at = p.g;
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
                for (uint32_t k = 0; k < KS; k += 1) {
                    qf[n][k][0] = qf[n][k][1] = 0;
                    if (head < a.group) {
                        if (FP8) {
                            const uint2 w = *reinterpret_cast<const uint2 *>(row + k * 16u + c * 4u);
                            qf[n][k][0] = w.x;
                            qf[n][k][1] = w.y;
                        } else {
                            qf[n][k][0] = *reinterpret_cast<const uint32_t *>(row + k * 16u + c * 2u);
                            qf[n][k][1] = *reinterpret_cast<const uint32_t *>(row + k * 16u + 8u + c * 2u);
                        }
                    }
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
        if (FP8) asm volatile("cp.async.wait_group %0;" ::"n"(St::COUNT - 1u) : "memory");
        if (!landed(bars0 + place * 8u, phase, a)) break;
        __syncwarp();
        const uint32_t at = ring0 + place * St::BYTES;
        // tokens of each group that are there; what their places hold beyond is nobody's and may be anything
        uint32_t valid[SG];
        bool all = true;
#pragma unroll
        for (uint32_t i = 0; i < SG; i += 1) {
            const uint32_t t0 = p.g * PER + i * 16u;
            const bool refused = (bad >> (place * SG + i * 16u / box) & 1u) != 0u;
            valid[i] = refused || t0 >= p.len ? 0u : min(16u, p.len - t0);
            all = all && valid[i] == 16u;
        }
        if (!all) {   // 0 x NaN is not 0: values that are not there become zeros
#pragma unroll
            for (uint32_t i = 0; i < SG; i += 1) {
                for (uint32_t u = valid[i] * (St::LINE / 16u) + lane; u < St::LINE; u += 32u) {
#pragma unroll
                    for (uint32_t h = 0; h < St::HALVES; h += 1)
                        *reinterpret_cast<uint4 *>(my_ring + place * St::BYTES + St::K_BYTES + h * St::HALF_BYTES + i * 16u * St::LINE + u * 16u) = make_uint4(0, 0, 0, 0);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before a later TMA load writes here
            __syncwarp();
        }

        // ---- scores: rows r and r + 8 of each group are tokens, columns 2c and 2c + 1 of each n are heads ----
        float x[SG][NT][4], inv[SG][2];
#pragma unroll
        for (uint32_t i = 0; i < SG; i += 1) {
            float s[2][NT][4];
#pragma unroll
            for (uint32_t n = 0; n < NT; n += 1) {
#pragma unroll
                for (uint32_t e = 0; e < 4; e += 1) s[0][n][e] = s[1][n][e] = 0.0f;
            }
            if (!FP8) {
#pragma unroll
                for (uint32_t k = 0; k < KS; k += 1) {
                    uint32_t f[4];
                    ldmatrix_x4(f, line_step(at + i * 16u * St::LINE + k_at, k));
#pragma unroll
                    for (uint32_t n = 0; n < NT; n += 1) mma_16816(s[k & 1u][n], f[0], f[1], f[2], f[3], qf[n][k][0], qf[n][k][1]);
                }
            } else {
#pragma unroll
                for (uint32_t k = 0; k < KS; k += 2) {   // a line piece is 16 columns: one product each
                    uint32_t f[4], lo[4], hi[4];
                    ldmatrix_x4(f, line_step(at + i * 16u * St::LINE + k_at, k / 2u));
#pragma unroll
                    for (uint32_t e = 0; e < 4; e += 1) e4m3x4_to_h2(f[e], lo[e], hi[e]);
#pragma unroll
                    for (uint32_t n = 0; n < NT; n += 1) {
                        mma_16816(s[0][n], lo[0], lo[1], hi[0], hi[1], qf[n][k][0], qf[n][k][1]);
                        mma_16816(s[1][n], lo[2], lo[3], hi[2], hi[3], qf[n][k + 1u][0], qf[n][k + 1u][1]);
                    }
                }
            }
#pragma unroll
            for (uint32_t half = 0; half < 2; half += 1) {
                float ks = to_log2, lv = 0.0f;
                inv[i][half] = 1.0f;
                if (FP8) {
                    const uint32_t sc = scales0 + place * St::SCALES + (i * 16u + r + 8u * half) * 4u;
                    const float vs = ld_shared_f(sc + PER * 4u);
                    ks *= ld_shared_f(sc);
                    // V's scale enters as a part of the exponent, so that weights keep their precision whatever the scales are
                    lv = __log2f(vs);
                    inv[i][half] = __fdividef(1.0f, vs);
                }
                const bool seen = r + 8u * half < valid[i];
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

        // ---- softmax: running reference (the maximum less WEIGHT_SHIFT) of each head, weights, their sum ----
        bool moves = false;
        float shift[NT][2], keep[NT][2];
#pragma unroll
        for (uint32_t n = 0; n < NT; n += 1) {
#pragma unroll
            for (uint32_t e = 0; e < 2; e += 1) {
                float m = fmaxf(x[0][n][e], x[0][n][2u + e]);
#pragma unroll
                for (uint32_t i = 1; i < SG; i += 1) m = fmaxf(m, fmaxf(x[i][n][e], x[i][n][2u + e]));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                // rounded up: to nearest, from 2^27 on, weights could pass fp16
                m = fmaxf(top[n][e], __fadd_ru(m, -WEIGHT_SHIFT));
                keep[n][e] = m == top[n][e] ? 1.0f : exp2_fast(top[n][e] - m);
                moves |= m != top[n][e];
                top[n][e] = m;
                shift[n][e] = m == -INFINITY ? 0.0f : m;
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
#pragma unroll
            for (uint32_t m = 0; m < MT; m += FP8 ? 2 : 1) {
                uint32_t f[4];
                ldmatrix_x4_trans(f, line_step(at + i * 16u * St::LINE + v_at, FP8 ? m / 2u : m));
                if (!FP8) {
#pragma unroll
                    for (uint32_t n = 0; n < NT; n += 1) mma_16816(o[m][n], f[0], f[1], f[2], f[3], pf[n][0], pf[n][1]);
                } else {
                    // a lane has columns 2r, 2r + 1 of two tokens: sorted by column and converted, row r and row r + 8 of the product
                    uint32_t lo[4], hi[4];
#pragma unroll
                    for (uint32_t e = 0; e < 4; e += 1) e4m3x4_to_h2(__byte_perm(f[e], 0u, 0x3120u), lo[e], hi[e]);
#pragma unroll
                    for (uint32_t n = 0; n < NT; n += 1) {
                        mma_16816(o[m][n], lo[0], hi[0], lo[2], hi[2], pf[n][0], pf[n][1]);
                        mma_16816(o[m + 1u][n], lo[1], hi[1], lo[3], hi[3], pf[n][0], pf[n][1]);
                    }
                }
            }
        }

        // ---- the end of this head, or of the warp's piece ----
        left -= 1;
        place += 1;
        if (place == St::COUNT) {
            place = 0;
            phase ^= 1u;
        }
        const bool head_ends = p.g + 1u == p.stages;
        bool whole_head = false;
        if (head_ends || left == 0) {
            fresh = true;
            whole_head = head_ends && begun_at == 0;
#pragma unroll
            for (uint32_t n = 0; n < NT; n += 1) {
                float l[2];
#pragma unroll
                for (uint32_t e = 0; e < 2; e += 1) {
                    l[e] = sum[n][e];
                    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 4);
                    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 8);
                    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 16);
                }
                if (whole_head) {
                    // transposed back, a lane has two neighbouring columns of head r; of e4m3 the tile's rows 8-15 are its odd columns
                    const float f0 = l[0] == 0.0f ? 0.0f : 1.0f / l[0], f1 = l[1] == 0.0f ? 0.0f : 1.0f / l[1];
                    const uint32_t head = n * 8u + r;
                    __half *out = a.o + (size_t)p.s * a.o_stride + (size_t)(p.h * a.group + head) * HD;
#pragma unroll
                    for (uint32_t m = 0; m < MT; m += 1) {
                        uint32_t y0 = transpose_8x8(pack_h2(o[m][n][0] * f0, o[m][n][1] * f1)), y1 = transpose_8x8(pack_h2(o[m][n][2] * f0, o[m][n][3] * f1));
                        if (head >= a.group) continue;
                        if (FP8) {
                            *reinterpret_cast<uint2 *>(out + m * 16u + c * 4u) = make_uint2(__byte_perm(y0, y1, 0x5410u), __byte_perm(y0, y1, 0x7632u));
                        } else {
                            *reinterpret_cast<uint32_t *>(out + m * 16u + c * 2u) = y0;
                            *reinterpret_cast<uint32_t *>(out + m * 16u + 8u + c * 2u) = y1;
                        }
                    }
                } else {
                    float *part = head_ends ? ended + warp * (St::PART / 4u) : goes_on(warp);
#pragma unroll
                    for (uint32_t e = 0; e < 2; e += 1) {
                        const uint32_t head = n * 8u + 2u * c + e;
                        if (head >= a.group) continue;
                        if (r == 0) {
                            part[a.group * HD + head] = top[n][e];
                            part[a.group * (HD + 1u) + head] = l[e];
                        }
#pragma unroll
                        for (uint32_t m = 0; m < MT; m += 1) {
                            part[head * HD + m * 16u + (FP8 ? 2u * r : r)] = o[m][n][e];
                            part[head * HD + m * 16u + (FP8 ? 2u * r + 1u : r + 8u)] = o[m][n][2u + e];
                        }
                    }
                }
            }
        }
        if (fresh && !whole_head && lane == 0) {
            if (head_ends) {
                ended_of[warp] = make_uint2(p.s, p.h);
            } else {
                goes_on_of[warp] = make_uint2(p.s, p.h);
                begins[warp] = begun_at == 0;
                if (warp + 1u == warps) behind = p.stages - p.g - 1u;
            }
        }
        if (left != 0) place_next(a, p, PER);
    }
    if (FP8) asm volatile("cp.async.wait_all;" ::: "memory");
    if (left != 0) {   // gave up: a bounded time for the copies in flight
        gave_up = true;
        for (uint32_t spin = 0; spin < (1u << 16); spin += 1) {
            bool done = true;
            for (uint32_t i = 0; i < St::COUNT; i += 1) done = mbar_try_wait(bars0 + i * 8u, i >= place ? phase : phase ^ 1u) && done;
            if (done) break;
        }
    }

    // ---- heads that go on from one warp to the next ------------------------------------------------
    __syncthreads();
    float *const begun_earlier = a.part + (size_t)blockIdx.x * 2u * part_floats(a.group, HD);
    const uint32_t at_top = a.group * HD, at_sum = a.group * (HD + 1u);
    // lane w looks at warp w: whether its last head goes on, and is one that an earlier warp has told of
    const uint2 key_of = lane < warps ? goes_on_of[lane] : make_uint2(~0u, 0u), key_before = lane != 0 && lane < warps ? goes_on_of[lane - 1u] : make_uint2(~0u, 0u);
    const uint2 end_of = lane < warps ? ended_of[lane] : make_uint2(~0u, 0u);
    const bool here_of = lane < warps && begins[lane];
    const uint32_t goes = __ballot_sync(0xffffffffu, key_of.x != ~0u), heres = __ballot_sync(0xffffffffu, here_of);
    const uint32_t starts = goes & __ballot_sync(0xffffffffu, here_of || key_of.x != key_before.x || key_of.y != key_before.y);
    for (uint32_t todo = starts; todo != 0u; todo &= todo - 1u) {
        const uint32_t w0 = (uint32_t)__ffs((int)todo) - 1u;
        const uint32_t stop = (~goes | starts) & (0xfffffffeu << w0);   // the first warp behind w0 whose last head is another
        const uint32_t w1 = stop != 0u ? min((uint32_t)__ffs((int)stop) - 1u, warps) : warps;
        const uint2 key = make_uint2(__shfl_sync(0xffffffffu, key_of.x, w0), __shfl_sync(0xffffffffu, key_of.y, w0));
        const uint32_t end_s = __shfl_sync(0xffffffffu, end_of.x, w1 & 31u), end_h = __shfl_sync(0xffffffffu, end_of.y, w1 & 31u);
        const bool ends = w1 < warps && end_s == key.x && end_h == key.y, here = (heres >> w0 & 1u) != 0u;
        const uint32_t n = w1 - w0 + (ends ? 1u : 0u);
        for (uint32_t head = warp; head < a.group; head += DEC_WARPS) {
            // lane i: the i-th part's maximum and sum
            const float *mine = lane < w1 - w0 ? goes_on(w0 + lane) : ended + (w1 < warps ? w1 : 0u) * (St::PART / 4u);
            float m = lane < n ? mine[at_top + head] : -INFINITY;
            const float own = m;
#pragma unroll
            for (uint32_t o = 16; o != 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float f_of = lane >= n ? 0.0f : own == m ? 1.0f : exp2_fast(own - m);
            float sum = lane < n ? f_of * mine[at_sum + head] : 0.0f;
#pragma unroll
            for (uint32_t o = 16; o != 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (uint32_t i = 0; i < DEC_WARPS + 1u; i += 1) {
                if (i >= n) break;
                const float *part = i < w1 - w0 ? goes_on(w0 + i) : ended + w1 * (St::PART / 4u);
                const float f = __shfl_sync(0xffffffffu, f_of, i);
                const float4 v = *reinterpret_cast<const float4 *>(part + head * HD + (lane < HD / 4u ? lane * 4u : 0u));
                y.x += f * v.x;
                y.y += f * v.y;
                y.z += f * v.z;
                y.w += f * v.w;
            }
            if (lane >= HD / 4u) continue;
            if (here && ends) {
                const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
                __half *out = a.o + (size_t)key.x * a.o_stride + (size_t)(key.y * a.group + head) * HD;
                *reinterpret_cast<uint2 *>(out + lane * 4u) = make_uint2(pack_h2(y.x * f, y.y * f), pack_h2(y.z * f, y.w * f));
            } else {
                float *to = begun_earlier + (here ? part_floats(a.group, HD) : 0u);
                *reinterpret_cast<float4 *>(to + head * HD + lane * 4u) = y;
                if (lane == 0) {
                    to[at_top + head] = m;
                    to[at_sum + head] = sum;
                }
            }
        }
        if (here && !ends && !gave_up && threadIdx.x == 0) over = make_uint4(key.x, key.y, blockIdx.x, sm_of(sm1 + behind - 1u) - blockIdx.x + 1u);
    }
    if (ended_of[0].x != ~0u) {   // begun in an earlier SM's piece, ended in this one's first warp
        for (uint32_t i = threadIdx.x; i < a.group * (HD + 2u); i += DEC_THREADS) begun_earlier[i] = ended[i];
    }

    if (threadIdx.x == 0) a.split[blockIdx.x] = over;
}

// Joins a head that begins in one SM's piece and goes on in others: a block for each SM and query head of a group, a warp for every
// fourth piece, always in the line's order.
constexpr uint32_t JOIN_WARPS = 4;
template <uint32_t HD>
__global__ void __launch_bounds__(JOIN_WARPS * 32) moe_attn_join_kernel(DecArgs a) {
    __shared__ float4 y_of[JOIN_WARPS][HD / 4];
    __shared__ float sum_of[JOIN_WARPS];
    moe_pdl_begin();
    const uint32_t first = blockIdx.x / a.group, head = blockIdx.x - first * a.group;
    const uint4 split = a.split[first];   // sequence, kv head, first SM, SMs
    const uint32_t n = moe_join_parts(first, split.w, gridDim.x / a.group);
    if (n == 0u) return;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, size = part_floats(a.group, HD);
    auto part_at = [&](uint32_t i) { return a.part + (size_t)((first + i) * 2u + (i == 0 ? 1u : 0u)) * size; };
    const uint32_t at_top = a.group * HD + head, at_sum = a.group * (HD + 1u) + head;
    float m = -INFINITY, sum = 0.0f;
    for (uint32_t i = lane; i < n; i += 32u) m = fmaxf(m, part_at(i)[at_top]);
#pragma unroll
    for (uint32_t o = 16; o != 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const bool mine = lane < HD / 4u;
#pragma unroll 4
    for (uint32_t i = warp; i < n; i += JOIN_WARPS) {
        const float *part = part_at(i);
        const float top = part[at_top], l = part[at_sum];
        const float4 v = *reinterpret_cast<const float4 *>(part + head * HD + (mine ? lane * 4u : 0u));
        const float f = top == m ? 1.0f : exp2_fast(top - m);
        sum += f * l;
        y.x += f * v.x;
        y.y += f * v.y;
        y.z += f * v.z;
        y.w += f * v.w;
    }
    if (mine) y_of[warp][lane] = y;
    if (lane == 0) sum_of[warp] = sum;
    __syncthreads();
    if (threadIdx.x >= HD / 4u) return;
    sum = 0.0f;
    y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (uint32_t w = 0; w < JOIN_WARPS; w += 1) {
        const float4 v = y_of[w][threadIdx.x];
        sum += sum_of[w];
        y.x += v.x;
        y.y += v.y;
        y.z += v.z;
        y.w += v.w;
    }
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
    __half *out = a.o + (size_t)split.x * a.o_stride + (size_t)(split.y * a.group + head) * HD;
    *reinterpret_cast<uint2 *>(out + threadIdx.x * 4u) = make_uint2(pack_h2(y.x * f, y.y * f), pack_h2(y.z * f, y.w * f));
}

template <uint32_t HD, uint32_t NT, bool FP8>
void decode_launch(moe_cuda_ctx *c, const moe_cuda_kv_t *kv, const DecArgs &a, uint32_t slot) {
    using St = Stage<HD, NT, FP8>;
    constexpr uint32_t smem = St::SMEM;
    static_assert(St::COUNT >= 2 && St::COUNT * St::SG <= 32 && smem + 4096 <= 227 * 1024 && St::PART <= St::COUNT * St::BYTES, "ring");
    CUtensorMap tk, tv;
    const uint64_t rows = (uint64_t)kv->pages * kv->kv_heads * kv->page;
    const uint32_t box = kv->page < St::TOKENS ? kv->page : St::TOKENS;
    if (!moe_tmap_bytes(c, &tk, kv->k, rows, St::ROW, St::LINE, box) || !moe_tmap_bytes(c, &tv, kv->v, rows, St::ROW, St::LINE, box)) return;
    if (!c->dec_attr_set[slot]) {
        MOE_CUDA_TRY(c, cudaFuncSetAttribute(moe_attn_decode_kernel<HD, NT, FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        c->dec_attr_set[slot] = true;
    }
    moe_run(c, moe_attn_decode_kernel<HD, NT, FP8>, (uint32_t)c->sm_count, St::THREADS, smem, tk, tv, a);
    MOE_LAUNCHED(c);
    moe_run(c, moe_attn_join_kernel<HD>, (uint32_t)c->sm_count * a.group, JOIN_WARPS * 32, 0, a);
    MOE_LAUNCHED(c);
}

}  // namespace

extern "C" void moe_cuda_attn_decode(moe_cuda_ctx_t *c, const moe_cuda_kv_t *kv, const void *q16, const uint32_t *table, const uint32_t *len,
                                     void *o16, struct moe_pc_attn_decode_t pc) {
    if (!MOE_LIVE(c)) return;
    const char *why = moe_attn_decode_refusal(kv, q16, table, len, o16, pc);
    MOE_REQUIRE(c, why == NULL, "%s", why);
    if (pc.seqs == 0) return;
    moe_on_device on(c);
    DecArgs a;
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
    a.scale = pc.scale;
    a.status = c->dev_status_dev;
    a.wait_ns = c->wait_ns;
    const size_t split_bytes = (size_t)c->sm_count * sizeof(uint4);
    const size_t part_bytes = split_bytes + (size_t)c->sm_count * 2u * part_floats(a.group, kv->hd) * 4u;
    if (part_bytes > c->work_bytes) {
        moe_fail(c, MOE_ERR_NOMEM, "attn_decode: %zu bytes of work area, the context has %zu", part_bytes, c->work_bytes);
        return;
    }
    a.split = (uint4 *)c->work;
    a.part = (float *)((uint8_t *)c->work + split_bytes);
    const bool fp8 = kv->type == MOE_KV_E4M3, wide = a.group > 8u;
    if (kv->hd == 128u) {
        if (fp8) wide ? decode_launch<128, 2, true>(c, kv, a, 0) : decode_launch<128, 1, true>(c, kv, a, 1);
        else wide ? decode_launch<128, 2, false>(c, kv, a, 2) : decode_launch<128, 1, false>(c, kv, a, 3);
    } else {
        if (fp8) wide ? decode_launch<64, 2, true>(c, kv, a, 4) : decode_launch<64, 1, true>(c, kv, a, 5);
        else wide ? decode_launch<64, 2, false>(c, kv, a, 6) : decode_launch<64, 1, false>(c, kv, a, 7);
    }
}
