// Causal attention over packed prompts on the 5th-generation tensor cores.
//
// o_i = sum_j p_ij v_j, p = softmax over the visible keys of scale * q_i k_j, one pass over the keys with a running maximum and
// sum.  Bound by the tensor pipe and, as closely, by the exponentials: a 128 x 128 tile of scores costs 512 cycles of products
// each for S = Q K^T and O += P V at head size 128, and 128 * 128 / 16 = 1024 cycles of the SM's exp2 unit.
//
// The query heads of one key-value head are rows of one tile: 128 / g tokens x g heads (g = heads / kv_heads), so a group reads
// its keys and values once, and a tile spans few tokens, which keeps what is computed above the diagonal small.  A CTA works
// on two such tiles (256 rows) against the same key blocks of 128, so that one tile's softmax runs under the other's products.
// Persistent CTAs, one per SM, walk a list of (tile pair, kv head), the longest first.  Roles:
//   warp 0     loads K and V blocks by TMA, a block to a load, and Q, each tile as soon as its last scores have been issued
//   warps 1, 3 issue the tcgen05.mma of the first and the second tile: S into tensor memory, then per block P V into the output
//              accumulator (P is read from tensor memory, where it overwrites its own S).  A warp of its own for each tile: a
//              look at a barrier takes some 200 cycles, and one tile's looks hide under the other's products
//   warp 2     makes V blocks that some row must not see in part safe (below)
//   warps 4-7, 8-11   softmax of the first and second tile, a row per thread
//   warps 12-15       scale and store the finished output of both tiles, while the softmax is at the next item
// What a tile waits for is softmax, then its products, then softmax again; so the softmax's own time counts, not only its
// throughput.  It takes scores two at a time where it can (f32x2 arithmetic, maxima of three), hands P over in two halves, and
// leaves a share of the exponentials to the multiply-add pipe: 2^x = 2^n * 2^f with n the nearest integer and a polynomial of
// degree 4 in f (fitted for the least relative error on [-1/2, 1/2], 2^-18.5, seven bits below P's rounding).
// The output accumulator is rescaled, by the softmax warps, only when a row's maximum has grown by more than 2^6; until then
// weights are taken against the older maximum, which stays inside fp16's range.
// A masked weight is 0, but 0 x NaN and 0 x infinity are not.  So the blocks that reach over the diagonal or the sequence's
// end are looked through before their product: their non-finite values become 0 in shared memory, and if there were any,
// the rows that do see them get them added at the end from global memory (a weight is positive, so infinities keep their sign).
// A NaN score makes the row's maximum NaN, and with it the whole row.
//
// One B200: a prompt of 8192 (32 heads of 128, 4 kv heads) 465 us = 1183 TFLOP/s, 0.71 of the measured bf16 rate, in bursts of a few
// milliseconds, and 532 us = 1033 for seconds on end, at 1515 MHz of 1965 under the 1000 W cap; one of 4096 128 us = 1073 and 143 us =
// 959 (1590 MHz); 13 prompts up to 1999 behind 517 cached tokens (12 heads of 64) 107 us, 103 captured; 32 windows of 384 (16 heads
// of 128, 2 kv heads) 50 us back to back, 45 captured, with the plan kernel.  On long prompts the tensor pipe is busy 0.58 and the exp2
// unit 0.44 of the time: what is left is the softmax's own turn, ~1700 cycles a tile and block, of which 768 are the exp2 unit's.  Short
// prompts are bound by the steps between items (~3500 cycles), by blocks cut by the diagonal and by the deal of few items.
#include "moe_attn.cuh"
#include "moe_tc.cuh"

#include <string.h>

namespace {

using namespace moe_tc;

constexpr uint32_t AT_THREADS = 512, TILE_ROWS = 128, BLOCK_KEYS = 128;
constexpr uint32_t HALF_BYTES = 128 * 128;       // 128 rows of 64 columns, one TMA box
constexpr float LOG2E = 1.4426950408889634f;
constexpr float GROW = 6.0f;                     // log2 of how far weights may pass the reference before a rescale
constexpr float SHIFT = 8.0f;                    // weights are at most 2^(GROW + SHIFT) = 2^14; fp16 then goes down to 2^-32 of the reference
// A row whose largest logit passes about 2^FAR (in log2 units) is scaled as if its exponent were that: powers of two come off the scale.
// The product of reference and scale is rounded before it is taken off, by 1 at most up to 2^(FAR + 2), so weights stay below
// 2^(GROW + SHIFT + 1); unbounded, they pass fp16.  fp32 scores are good to 2^-24 of themselves, so logits of that size to half a unit.
constexpr int32_t FAR = 23;
// Of every POLY_OF pairs of exponentials POLY_SHARE go to the multiply-add pipe.
constexpr uint32_t POLY_OF = 4, POLY_SHARE = 1;
// Items with a masked block that may be between their V check and their epilogue.  Each has such a block in the ring until its products
// are done: four items in a ring of eight places, one more per tile whose output has not been stored, and the one whose check begins.
constexpr uint32_t FLAGS = 8;

template <uint32_t HD>
struct Cfg {
    static constexpr uint32_t HALVES = HD / 64;
    static constexpr uint32_t TILE_BYTES = HALVES * HALF_BYTES;      // Q tile, K block or V block
    static constexpr uint32_t STAGES = HD == 128 ? 5 : 8;
    static constexpr uint32_t SMEM = (2 + STAGES) * TILE_BYTES;
};

template <uint32_t ST>
struct __align__(8) AttnBars {
    uint64_t kv_full[ST], kv_empty[ST];
    uint64_t v_landed[ST];   // masked V blocks: loaded; warp 2 then arrives at kv_full
    uint64_t q_full[2], q_empty[2];
    uint64_t s_full[2], p_full[2][2], o_full[2], o_empty[2];   // p_full: of each tile, keys 0-63 and 64-127
    uint64_t sum_full[2], sum_empty[2];
    uint64_t turn[2];        // the tile's softmax may begin: the other one's has ended
    uint64_t drain[2];       // at the end: all products issued have retired, and what waits for them has been told
    uint32_t tmem_base;
    uint32_t abort[3];       // a role gave up; places of the ring that each tile has been through
    uint32_t found[FLAGS];   // the item's masked V blocks held something that is not finite
    float sum[2][TILE_ROWS];
};

// A pair of tiles of one sequence: `left` queries from row q_row on, the sequence's keys from row k_row on.
struct Pair {
    uint32_t q_row, left, k_row, lk;
};

struct AttnArgs {
    const uint32_t *cu_q, *cu_k;
    const __half *v;
    __half *o;
    const uint4 *plan;       // NULL: one sequence, its pairs from the last to the first
    const uint32_t *pairs;   // number of entries of plan
    uint32_t rows_q, rows_k, kv_heads, group, tile_tokens;
    uint32_t kv_stride, o_stride;
    float scale;
    uint32_t far_top, far_scale;   // bits of the reference's exponent from which the scale is cut; those of the scale, and far_top more
    uint32_t *status;
    uint64_t wait_ns;
};

// Rows a .. b - 1 of a table of `rows`, whatever the caller's offsets are.
__device__ __forceinline__ uint32_t span(uint32_t a, uint32_t b, uint32_t rows) {
    return a <= b && b <= rows ? b - a : 0u;
}

// What a CTA has to do, in turn: round r takes item r * G + c, odd rounds from the other end, so that with falling costs every
// CTA gets about the same.
struct Items {
    uint32_t count, round, head;
    Pair p;            // of the next item, loaded one item ahead
    bool more;
    Pair one;
    uint32_t one_pairs;

    __device__ __forceinline__ void begin(const AttnArgs &a) {
        round = 0;
        if (a.plan == nullptr) {
            one.q_row = a.cu_q[0];
            one.left = span(a.cu_q[0], a.cu_q[1], a.rows_q);
            one.k_row = a.cu_k[0];
            one.lk = span(a.cu_k[0], a.cu_k[1], a.rows_k);
            one_pairs = (one.left + 2u * a.tile_tokens - 1u) / (2u * a.tile_tokens);
            count = one_pairs * a.kv_heads;
        } else {
            count = *a.pairs * a.kv_heads;
        }
        fetch(a);
    }
    __device__ __forceinline__ void fetch(const AttnArgs &a) {
        const uint32_t at = round * gridDim.x + ((round & 1u) != 0 ? gridDim.x - 1u - blockIdx.x : blockIdx.x);
        more = at < count;   // a round that is too short for this CTA is the last one
        if (!more) return;
        round += 1;
        const uint32_t i = at / a.kv_heads;
        head = at - i * a.kv_heads;
        if (a.plan == nullptr) {
            const uint32_t q0 = (one_pairs - 1u - i) * 2u * a.tile_tokens;
            p.q_row = one.q_row + q0;
            p.left = one.left - q0;
            p.k_row = one.k_row;
            p.lk = one.lk;
        } else {
            const uint4 e = a.plan[i];
            p.q_row = e.x;
            p.left = e.y;
            p.k_row = e.z;
            p.lk = e.w;
        }
    }
    __device__ __forceinline__ bool next(const AttnArgs &a, Pair &now, uint32_t &now_head) {
        if (!more) return false;
        now = p;
        now_head = head;
        fetch(a);
        return true;
    }
};

// Visible keys of the query `i` behind the pair's first one (may be negative).
__device__ __forceinline__ int32_t visible(const Pair &p, uint32_t i) { return (int32_t)p.lk - (int32_t)p.left + 1 + (int32_t)i; }

struct Blocks {
    uint32_t tile[2];   // key blocks that the tile's last query sees; 0: the tile has no query, or its queries no key
    bool has_b;
    uint32_t n;
    int32_t masked_from;  // blocks from here on are masked for some row
    __device__ __forceinline__ bool masks() const { return masked_from < (int32_t)n; }
};
__device__ __forceinline__ Blocks blocks_of(const Pair &p, uint32_t tile_tokens) {
    Blocks b;
    b.has_b = p.left > tile_tokens;
    const int32_t va = visible(p, min(p.left, tile_tokens) - 1u), vb = b.has_b ? visible(p, min(p.left, 2u * tile_tokens) - 1u) : 0;
    b.tile[0] = va > 0 ? ((uint32_t)va + BLOCK_KEYS - 1u) / BLOCK_KEYS : 0u;
    b.tile[1] = vb > 0 ? ((uint32_t)vb + BLOCK_KEYS - 1u) / BLOCK_KEYS : 0u;
    b.n = max(b.tile[0], b.tile[1]);
    const int32_t first = visible(p, 0);
    b.masked_from = first > 0 ? first / (int32_t)BLOCK_KEYS : 0;
    return b;
}

// V as the second operand of P V: [keys][columns] with the columns contiguous ("MN-major"), 128-byte swizzle: 64-column
// groups HALF_BYTES apart, groups of 8 keys 1024 bytes apart.
__device__ __forceinline__ uint64_t v_desc(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3ffffu) >> 4) | ((uint64_t)(HALF_BYTES >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// D[tmem] (+)= A[tmem] * B
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
        :
        : "r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accum)
        : "memory");
}
// A box of some heads of some rows, from 64-column half `half` on.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int32_t head, int32_t row, int32_t half = 0) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        :
        : "r"(dst), "l"((uint64_t)map), "r"(bar), "r"(0), "r"(head), "r"(row), "r"(half)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]),
        "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]),
        "r"(v[31])
        : "memory");
}
// Waits for this thread's loads; what was loaded into v is used behind it only.
__device__ __forceinline__ void tmem_ld_wait32(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]),
                   "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]),
                   "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]),
                   "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_nan(float x, float y) {
    float z;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
    return z;
}
__device__ __forceinline__ float max_nan(float x, float y, float z) {
    float m;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(x), "f"(y), "f"(z));
    return m;
}
// Two fp32 values in one register pair.
__device__ __forceinline__ uint64_t two(float x, float y) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
    return v;
}
__device__ __forceinline__ void apart(uint64_t v, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(x), "l"(y), "l"(z));
    return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(x), "l"(y));
    return v;
}
// 2^x for two x below 127 (what lies below -126 counts as -126); not for NaN.
__device__ __forceinline__ void exp2_poly(uint64_t x, float &y0, float &y1) {
    float a, b;
    apart(x, a, b);
    x = two(fmaxf(a, -126.0f), fmaxf(b, -126.0f));
    const uint64_t magic = two(12582912.0f, 12582912.0f), minus = two(-12582912.0f, -12582912.0f), one = two(-1.0f, -1.0f);
    const uint64_t t = add2(x, magic);                  // the nearest integer in the low bits
    const uint64_t f = fma2(add2(t, minus), one, x);    // [-1/2, 1/2]
    uint64_t v = fma2(two(0.0095701f, 0.0095701f), f, two(0.05591786f, 0.05591786f));
    v = fma2(v, f, two(0.24024745f, 0.24024745f));
    v = fma2(v, f, two(0.69312181f, 0.69312181f));
    v = fma2(v, f, two(0.99999926f, 0.99999926f));
    float n0, n1;
    apart(t, n0, n1);
    apart(v, y0, y1);
    y0 = __uint_as_float(__float_as_uint(y0) + (__float_as_uint(n0) << 23));
    y1 = __uint_as_float(__float_as_uint(y1) + (__float_as_uint(n1) << 23));
}
__device__ __forceinline__ void store32(__half *to, const uint32_t (&w)[8], bool whole) {   // 32 bytes, at once if they are aligned
    if (whole) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                     "r"(w[5]), "r"(w[6]), "r"(w[7])
                     : "memory");
    } else {
        reinterpret_cast<uint4 *>(to)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<uint4 *>(to)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
}

// mbar_wait in two parts: the first looks stand where the wait is (a call would hold a softmax thread's registers to a calling
// convention), all that bounds it is out of line.  Each role's step from item to item runs code that the others' have pushed
// out of the instruction cache, so the code is kept short: with the whole wait in every place 32 windows of 384 took 47.3 us captured,
// with this 43.5.
// Some waits last an item, however many keys it has, so the limit is for the time in which neither tile has moved: abort[1] and [2].
__device__ __noinline__ bool wait_long(uint32_t bar, uint32_t parity, volatile uint32_t *abort, uint32_t *status, uint32_t site, uint64_t wait_ns) {
    uint32_t spins = 0, moved = 0;
    uint64_t t0 = 0;
    while (!mbar_try_wait(bar, parity)) {
        spins += 1;
        if ((spins & 0xffu) != 0) continue;
        if (*abort != 0) return false;
        const uint64_t now = globaltimer_ns();
        const uint32_t at = abort[1] + abort[2];
        if (t0 == 0 || at != moved) {
            t0 = now;
            moved = at;
        } else if (now - t0 > wait_ns) {
            *abort = 1;
            atomicCAS(status, 0u, (uint32_t)MOE_ERR_TIMEOUT | (site << 8));
            return false;
        }
    }
    return true;
}

__device__ __forceinline__ bool wait_here(uint32_t bar, uint32_t parity, volatile uint32_t *abort, uint32_t *status, uint32_t site, uint64_t wait_ns) {
#pragma unroll 1
    for (uint32_t i = 0; i < 64u; i += 1) {
        if (mbar_try_wait(bar, parity)) return true;
    }
    return wait_long(bar, parity, abort, status, site, wait_ns);
}

template <uint32_t HD>
__global__ void __launch_bounds__(AT_THREADS, 1)
moe_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                AttnArgs a) {
    using C = Cfg<HD>;
    constexpr uint32_t ST = C::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    AttnBars<ST> *bars = reinterpret_cast<AttnBars<ST> *>(smem + C::SMEM);
    const uint32_t q_smem = smem_u32(smem), ring = q_smem + 2u * C::TILE_BYTES;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    volatile uint32_t *abort = bars->abort;

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < ST; i += 1) {
            mbar_init(smem_u32(&bars->kv_full[i]), 1);
            mbar_init(smem_u32(&bars->kv_empty[i]), 2);
            mbar_init(smem_u32(&bars->v_landed[i]), 1);
        }
        for (uint32_t i = 0; i < 2; i += 1) {
            mbar_init(smem_u32(&bars->q_full[i]), 1);
            mbar_init(smem_u32(&bars->q_empty[i]), 1);
            mbar_init(smem_u32(&bars->s_full[i]), 1);
            mbar_init(smem_u32(&bars->p_full[i][0]), TILE_ROWS);
            mbar_init(smem_u32(&bars->p_full[i][1]), TILE_ROWS);
            mbar_init(smem_u32(&bars->sum_full[i]), TILE_ROWS);
            mbar_init(smem_u32(&bars->sum_empty[i]), TILE_ROWS);
            mbar_init(smem_u32(&bars->turn[i]), 4);
            mbar_init(smem_u32(&bars->drain[i]), 1);
            mbar_init(smem_u32(&bars->o_full[i]), 1);
            mbar_init(smem_u32(&bars->o_empty[i]), TILE_ROWS);
        }
        bars->abort[0] = bars->abort[1] = bars->abort[2] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&bars->tmem_base)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // all 512 columns are this CTA's, so they begin at 0
    constexpr uint32_t tmem = 0;   // S of the two tiles at 0 and 128, O at 256 and 256 + HD

    moe_pdl_begin();

    Items items;
    items.begin(a);
    Pair p;
    uint32_t head;
#define AT_WAIT(bar, parity, site) wait_here(smem_u32(bar), (parity), abort, a.status, (site), a.wait_ns)

    if (blockIdx.x == 0 && threadIdx.x == 0 && a.plan == nullptr &&
        (a.cu_q[0] > a.cu_q[1] || a.cu_q[1] > a.rows_q || a.cu_k[0] > a.cu_k[1] || a.cu_k[1] > a.rows_k)) {
        moe_deny(a.status, MOE_SITE_ROWS);
    }
    if (warp < 4u) {
        if (warp == 0) {
            // ---------------- loads: ring places K(n-1), V(n-1), K(n-2), V(n-2), ... of each item in turn ----------------
            if (lane == 0) {
                uint32_t at = 0, issued = 0, parity = 0, masked = 0, landed = 0, q_loads[2] = {0, 0};
                bool ok = true;
                while (ok && items.next(a, p, head)) {
                    const Blocks b = blocks_of(p, a.tile_tokens);
                    if (b.n == 0) continue;
                    for (uint32_t i = 0; i < 2u * b.n; i += 1) {
                        const uint32_t j = b.n - 1u - i / 2u, s = at % ST, ph = (at / ST) & 1u;
                        const bool is_v = (i & 1u) != 0;
                        if (!AT_WAIT(&bars->kv_empty[s], ph ^ 1u, 32)) {
                            ok = false;
                            break;
                        }
                        const bool m = is_v && (int32_t)j >= b.masked_from;
                        const uint32_t full = smem_u32(m ? &bars->v_landed[s] : &bars->kv_full[s]);
                        mbar_expect_tx(full, C::TILE_BYTES);
                        tma_load_4d(ring + s * C::TILE_BYTES, is_v ? &tm_v : &tm_k, full, (int32_t)head, (int32_t)(p.k_row + j * BLOCK_KEYS));
                        issued |= 1u << s;
                        parity = (parity & ~(1u << s)) | (ph << s);
                        masked = (masked & ~(1u << s)) | ((m ? 1u : 0u) << s);
                        landed ^= (m ? 1u : 0u) << s;   // the next masked use's parity
                        at += 1u;
                        // Q behind the item's first two blocks, for which there is room earlier
                        for (uint32_t tile = 0; tile < 2u && i == 1 && ok; tile += 1) {
                            if (b.tile[tile] == 0) continue;
                            const uint32_t q_bar = smem_u32(&bars->q_full[tile]);
                            ok = AT_WAIT(&bars->q_empty[tile], ~q_loads[tile] & 1u, 31);
                            if (!ok) break;
                            mbar_expect_tx(q_bar, a.group * a.tile_tokens * HD * 2u);
                            // a group of an odd size leaves rows of the tile free, so each half is placed by itself
                            for (uint32_t half = 0; half < C::HALVES; half += 1) {
                                tma_load_4d(q_smem + tile * C::TILE_BYTES + half * HALF_BYTES, &tm_q, q_bar, (int32_t)(head * a.group),
                                            (int32_t)(p.q_row + tile * a.tile_tokens), (int32_t)half);
                            }
                            q_loads[tile] += 1;
                        }
                        if (!ok) break;
                    }
                }
                if (*abort != 0) {
                    // unwinding: give copies already issued a bounded time to land
                    for (uint32_t s = 0; s < ST; s += 1) {
                        for (uint32_t spin = 0; (issued >> s & 1u) != 0 && spin < (1u << 16); spin += 1) {
                            if ((masked >> s & 1u) != 0) {
                                if (mbar_try_wait(smem_u32(&bars->v_landed[s]), ~landed >> s & 1u)) break;
                            } else if (mbar_try_wait(smem_u32(&bars->kv_full[s]), parity >> s & 1u)) {
                                break;
                            }
                        }
                    }
                    for (uint32_t tile = 0; tile < 2; tile += 1) {
                        for (uint32_t spin = 0; q_loads[tile] != 0 && spin < (1u << 16); spin += 1) {
                            if (mbar_try_wait(smem_u32(&bars->q_full[tile]), (q_loads[tile] - 1u) & 1u)) break;
                        }
                    }
                }
            }
            __syncwarp();
        } else if (warp == 1 || warp == 3) {
            // ---------------- MMA issue: a whole warp runs each tile's loop, one elected lane issues ----------------
            const uint32_t t = warp >> 1;
            const uint32_t s_at = tmem + t * 128u, o_at = tmem + 256u + t * HD;
            const uint64_t qd = umma_desc(q_smem + t * C::TILE_BYTES);
            uint32_t at = 0, q_phase = 0, p_phase = 0, o_phase = 1;
            bool ok = true;
            const uint32_t idesc_s = umma_idesc(128, BLOCK_KEYS), idesc_o = umma_idesc(128, HD) | (1u << 16);  // V: MN-major
            // S of the block in ring place `slot`; last: the item's last use of Q
            auto scores = [&](uint32_t slot, bool mine, bool last) {
                tc_fence_after();
                if (elect_one()) {
                    if (mine) {
                        const uint64_t kd = umma_desc(ring + slot * C::TILE_BYTES);
#pragma unroll
                        for (uint32_t k = 0; k < HD / 16u; k += 1) {
                            const uint64_t off = (uint64_t)((k / 4u) * (HALF_BYTES >> 4) + (k % 4u) * 2u);
                            umma_f16(s_at, qd + off, kd + off, idesc_s, k != 0 ? 1u : 0u);
                        }
                        umma_commit(smem_u32(&bars->s_full[t]));
                    }
                    umma_commit(smem_u32(&bars->kv_empty[slot]));
                    if (last && mine) umma_commit(smem_u32(&bars->q_empty[t]));
                }
                __syncwarp();
            };
            while (ok && items.next(a, p, head)) {
                const Blocks b = blocks_of(p, a.tile_tokens);
                if (b.n == 0) continue;
                uint32_t ks = at % ST;
                ok = AT_WAIT(&bars->kv_full[ks], (at / ST) & 1u, 34) && (b.tile[t] == 0 || AT_WAIT(&bars->q_full[t], q_phase, 33));
                __syncwarp();
                if (!ok) break;
                if (b.tile[t] != 0) q_phase ^= 1u;
                scores(ks, b.n == b.tile[t], b.n == 1u);
                for (uint32_t j = b.n; j-- > 0;) {
                    const uint32_t vi = at + 1u, vs = vi % ST;
                    at += 2u;
                    ks = at % ST;
                    ok = AT_WAIT(&bars->kv_full[vs], (vi / ST) & 1u, 35) && (j == 0 || AT_WAIT(&bars->kv_full[ks], (at / ST) & 1u, 34));
                    if (j < b.tile[t]) {
                        const bool first = j + 1u == b.tile[t];
                        if (first) {
                            ok = ok && AT_WAIT(&bars->o_empty[t], o_phase, 37);
                            o_phase ^= 1u;
                        }
#pragma unroll
                        for (uint32_t part = 0; part < 2u; part += 1) {
                            ok = ok && AT_WAIT(&bars->p_full[t][part], p_phase, 38);
                            __syncwarp();
                            tc_fence_after();
                            if (ok && elect_one()) {
                                const uint64_t vd = v_desc(ring + vs * C::TILE_BYTES) + part * 512u;
#pragma unroll
                                for (uint32_t k = 0; k < BLOCK_KEYS / 32u; k += 1) {
                                    umma_f16_ts(o_at, s_at + part * 32u + k * 8u, vd + k * 128u, idesc_o, first && part == 0 && k == 0 ? 0u : 1u);
                                }
                                if (j == 0 && part == 1u) umma_commit(smem_u32(&bars->o_full[t]));
                            }
                            __syncwarp();
                        }
                        p_phase ^= 1u;
                    }
                    __syncwarp();
                    if (!ok) break;
                    if (j != 0) scores(ks, j - 1u < b.tile[t], j == 1u);
                    if (elect_one()) {
                        umma_commit(smem_u32(&bars->kv_empty[vs]));
                        abort[1u + t] = at;
                    }
                    __syncwarp();
                }
            }
            __syncwarp();
            // Arrivals at the ring's last barriers may be under way still, and products when unwinding: the shared memory and tensor
            // memory are theirs until then.  A bounded time for them.
            if (elect_one()) umma_commit(smem_u32(&bars->drain[t]));
            __syncwarp();
            for (uint32_t spin = 0; spin < (1u << 16); spin += 1) {
                if (mbar_try_wait(smem_u32(&bars->drain[t]), 0)) break;
            }
            __syncwarp();
        } else if (warp == 2) {
            // ---------------- V blocks that reach over the diagonal or the sequence's end ----------------
            uint32_t at = 0, n_item = 0, landed = 0;
            bool ok = true;
            while (ok && items.next(a, p, head)) {
                const Blocks b = blocks_of(p, a.tile_tokens);
                if (!b.masks()) {   // no wait here holds this warp back: an item without a masked block has no flag
                    at += 2u * b.n;
                    continue;
                }
                volatile uint32_t *found = &bars->found[n_item % FLAGS];
                if (lane == 0) *found = 0;
                __syncwarp();
                for (uint32_t j = b.n; j-- > 0 && (int32_t)j >= b.masked_from;) {
                    const uint32_t vi = at + 2u * (b.n - 1u - j) + 1u, vs = vi % ST;
                    if (!AT_WAIT(&bars->v_landed[vs], landed >> vs & 1u, 39)) {
                        ok = false;
                        break;
                    }
                    landed ^= 1u << vs;
                    __syncwarp();
                    uint8_t *block = smem + (2u + vs) * C::TILE_BYTES;
                    uint32_t top[4] = {0, 0, 0, 0};   // the largest exponents and mantissas of both halves
#pragma unroll 8
                    for (uint32_t i = lane; i < C::TILE_BYTES / 16u; i += 32u) {
                        const uint4 w = *reinterpret_cast<const uint4 *>(block + i * 16u);
                        top[0] = __vmaxu2(top[0], w.x & 0x7fff7fffu);
                        top[1] = __vmaxu2(top[1], w.y & 0x7fff7fffu);
                        top[2] = __vmaxu2(top[2], w.z & 0x7fff7fffu);
                        top[3] = __vmaxu2(top[3], w.w & 0x7fff7fffu);
                    }
                    const uint32_t most = __vmaxu2(__vmaxu2(top[0], top[1]), __vmaxu2(top[2], top[3]));
                    if (__any_sync(0xffffffffu, (most & 0xffffu) >= 0x7c00u || (most >> 16) >= 0x7c00u)) {
                        for (uint32_t i = lane; i < C::TILE_BYTES / 4u; i += 32u) {
                            uint32_t *w = reinterpret_cast<uint32_t *>(block + i * 4u);
                            uint32_t x = *w;
                            if ((x & 0x7c00u) == 0x7c00u) x &= 0xffff0000u;
                            if ((x & 0x7c000000u) == 0x7c000000u) x &= 0xffffu;
                            *w = x;
                        }
                        if (lane == 0) *found = 1;
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&bars->kv_full[vs]));
                }
                at += 2u * b.n;
                n_item += 1;
            }
            __syncwarp();
        }
    } else if (warp < 12u) {
        // ---------------- softmax: a row per thread ----------------
        const uint32_t t = (warp - 4u) >> 2, row = (warp & 3u) * 32u + lane;
        const uint32_t my_token = row / a.group;
        const uint32_t lanes = ((warp & 3u) * 32u) << 16;
        const uint32_t s_at = tmem + t * 128u + lanes, o_at = tmem + 256u + t * HD + lanes;
        const float to_log2 = a.scale * LOG2E;
        uint32_t s_phase = 0, sum_phase = 1, turn_phase = t == 0 ? 1u : 0u;   // the first tile begins
        bool ok = true;
        while (ok && items.next(a, p, head)) {
            const Blocks b = blocks_of(p, a.tile_tokens);
            const uint32_t n = b.tile[t], both = min(b.tile[0], b.tile[1]);   // blocks that both tiles have
            if (n == 0) continue;
            const int32_t tile_first = visible(p, t * a.tile_tokens);
            float top = -INFINITY, sum = 0.0f;   // top: the reference that weights are taken against, in score units
            for (uint32_t j = n; j-- > 0;) {
                if (!AT_WAIT(&bars->s_full[t], s_phase, 40)) {
                    ok = false;
                    break;
                }
                s_phase ^= 1u;
                __syncwarp();
                tc_fence_after();
                if ((int32_t)((j + 1u) * BLOCK_KEYS) > tile_first) {
                    // some rows do not see all of the block: what they do not see becomes -infinity where it lies, so that the code
                    // below, which every block runs, is short (straight through once a block, it is bound by its own fetching); done
                    // while the other tile has its turn
                    const int32_t seen = tile_first + (int32_t)my_token - (int32_t)(j * BLOCK_KEYS);   // columns below it are visible
#pragma unroll 1
                    for (int32_t i = 0; i < 4; i += 1) {
                        if (__all_sync(0xffffffffu, seen >= i * 32 + 32)) continue;
                        uint32_t s[32];
                        tmem_ld32(s_at + (uint32_t)i * 32u, s);
                        tmem_ld_wait32(s);
#pragma unroll
                        for (int32_t e = 0; e < 32; e += 1) {
                            if (e >= seen - i * 32) s[e] = 0xff800000u;
                        }
                        tmem_st32(s_at + (uint32_t)i * 32u, s);
                    }
                    tmem_st_wait();
                }
                // The two tiles' softmaxes take turns, block by block (masks come before): alone on the SM's units one is done twice as fast, and
                // the other one's products run meanwhile.  Left to themselves they fall into step.
                const bool turns = j < both;
                if (turns) {
                    if (!AT_WAIT(&bars->turn[t], turn_phase, 45)) {
                        ok = false;
                        break;
                    }
                    turn_phase ^= 1u;
                }
                __syncwarp();
                // Scores are read twice, 32 columns at a time and each piece while the one before it is worked on: a whole row in
                // registers would cost the other warps theirs.
                uint32_t s[2][32];
                float m[2] = {-INFINITY, -INFINITY};
                tmem_ld32(s_at, s[0]);
#pragma unroll 1
                for (uint32_t half = 0; half < 2; half += 1) {
#pragma unroll
                    for (uint32_t i = 0; i < 2; i += 1) {
                        tmem_ld_wait32(s[i]);
                        tmem_ld32(s_at + ((half * 64u + i * 32u + 32u) & 127u), s[i ^ 1u]);   // behind the last piece the first again
#pragma unroll
                        for (uint32_t e = 0; e < 32; e += 4) {
                            m[0] = max_nan(m[0], __uint_as_float(s[i][e]), __uint_as_float(s[i][e + 1]));
                            m[1] = max_nan(m[1], __uint_as_float(s[i][e + 2]), __uint_as_float(s[i][e + 3]));
                        }
                    }
                }
                const float now = max_nan(m[0], m[1]);
                const bool grows = now != -INFINITY && !((now - top) * to_log2 <= GROW);   // also from -infinity, and to NaN
                if (j + 1u == n) {
                    top = now;
                } else if (__any_sync(0xffffffffu, grows)) {
                    // P V of the blocks before has completed: this S was issued behind it
                    const float f = grows ? exp2_fast((top - now) * to_log2) : 1.0f;
                    if (grows) top = now;
                    sum *= f;
                    tmem_ld_wait();
#pragma unroll 1
                    for (uint32_t i = 0; i < HD / 16u; i += 1) {
                        uint32_t o[16];
                        tmem_ld16(o_at + i * 16u, o);
                        tmem_ld_wait();
#pragma unroll
                        for (uint32_t e = 0; e < 16; e += 1) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st16(o_at + i * 16u, o);
                    }
                }
                // against -infinity everything is -infinity: weights 0; against infinity or NaN everything is NaN
                const float scale = __uint_as_float(a.far_scale - max(__float_as_uint(top) & 0x7f800000u, a.far_top));
                const float base = top == -INFINITY ? 0.0f : SHIFT - top * scale + (top - top);
                const uint64_t scale2 = two(scale, scale), base2 = two(base, base);
                uint64_t part[2] = {0, 0};
#pragma unroll
                for (uint32_t i = 0; i < 4; i += 1) {
                    tmem_ld_wait32(s[i & 1u]);
                    if (i < 3) tmem_ld32(s_at + (i + 1u) * 32u, s[(i + 1u) & 1u]);
                    uint32_t w[16];
#pragma unroll
                    for (uint32_t e = 0; e < 16; e += 1) {
                        const uint64_t z = fma2(two(__uint_as_float(s[i & 1u][2 * e]), __uint_as_float(s[i & 1u][2 * e + 1])), scale2, base2);
                        float x, y;
                        if (e % POLY_OF < POLY_SHARE) {
                            exp2_poly(z, x, y);
                        } else {
                            apart(z, x, y);
                            x = exp2_fast(x);
                            y = exp2_fast(y);
                        }
                        part[e & 1u] = add2(part[e & 1u], two(x, y));
                        // weights round to fp16 for the product (11 bits, as many as the output has); their sum does not
                        w[e] = pack_h2(x, y);
                    }
                    if (i == 2 && turns && lane == 0) mbar_arrive(smem_u32(&bars->turn[t ^ 1u]));
                    tmem_st16(s_at + i * 16u, w);
                    if ((i & 1u) != 0) {
                        tmem_st_wait();
                        tc_fence_before();
                        mbar_arrive(smem_u32(&bars->p_full[t][i / 2u]));
                    }
                }
                float x, y;
                apart(add2(part[0], part[1]), x, y);
                sum += x + y;
            }
            if (!ok || !AT_WAIT(&bars->sum_empty[t], sum_phase, 41)) break;
            sum_phase ^= 1u;
            bars->sum[t][row] = sum;
            mbar_arrive(smem_u32(&bars->sum_full[t]));
        }
    } else {
        // ---------------- output: a row per thread ----------------
        const uint32_t row = (warp & 3u) * 32u + lane, my_token = row / a.group, my_head = row - my_token * a.group;
        const uint32_t lanes = ((warp & 3u) * 32u) << 16;
        const bool whole = ((uintptr_t)a.o & 31u) == 0 && a.o_stride % 16u == 0;
        uint32_t phase = 0, n_item = 0;   // phase: a bit for each tile
        bool ok = true;
        while (ok && items.next(a, p, head)) {
            const Blocks b = blocks_of(p, a.tile_tokens);
            const uint32_t flag = n_item % FLAGS;
            if (b.masks()) n_item += 1;
#pragma unroll 1
            for (uint32_t t = 0; t < 2; t += 1) {
                const uint32_t token = t * a.tile_tokens + my_token;   // behind the pair's first
                const bool mine = my_token < a.tile_tokens && token < p.left;
                __half *out = a.o + (size_t)(p.q_row + token) * a.o_stride + (size_t)(head * a.group + my_head) * HD;
                if ((t == 0 ? b.tile[0] : b.tile[1]) == 0) {   // no query, or none that sees a key
                    if (mine) {
#pragma unroll 1
                        for (uint32_t i = 0; i < HD; i += 8) *reinterpret_cast<uint4 *>(out + i) = make_uint4(0, 0, 0, 0);
                    }
                    continue;
                }
                ok = ok && AT_WAIT(&bars->sum_full[t], phase >> t & 1u, 43) && AT_WAIT(&bars->o_full[t], phase >> t & 1u, 44);
                if (!ok) break;
                phase ^= 1u << t;
                __syncwarp();
                tc_fence_after();
                const float sum = bars->sum[t][row];
                mbar_arrive(smem_u32(&bars->sum_empty[t]));
                const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
                const bool extra = b.masks() && *(volatile uint32_t *)&bars->found[flag] != 0;
                const int32_t vis = visible(p, token);
#pragma unroll 1
                for (uint32_t i = 0; i < HD / 16u; i += 1) {
                    uint32_t o[16];
                    tmem_ld16(tmem + 256u + t * HD + lanes + i * 16u, o);
                    tmem_ld_wait();
                    if (mine) {
                        if (extra) {
                            for (int32_t key = b.masked_from * (int32_t)BLOCK_KEYS; key < vis; key += 1) {
                                const __half *v = a.v + (size_t)(p.k_row + (uint32_t)key) * a.kv_stride + (size_t)head * HD + i * 16u;
#pragma unroll
                                for (uint32_t e = 0; e < 16; e += 1) {
                                    const float x = __half2float(v[e]);
                                    if (!isfinite(x)) o[e] = __float_as_uint(__uint_as_float(o[e]) + x);
                                }
                            }
                        }
                        uint32_t w[8];
#pragma unroll
                        for (uint32_t e = 0; e < 8; e += 1) w[e] = pack_h2(__uint_as_float(o[2 * e]) * f, __uint_as_float(o[2 * e + 1]) * f);
                        store32(out + i * 16u, w, whole);
                    }
                    __syncwarp();
                }
                tc_fence_before();
                mbar_arrive(smem_u32(&bars->o_empty[t]));
            }
        }
    }
#undef AT_WAIT
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// The list of tile pairs, those with the most key blocks first (counting sort over 1024 classes of cost; the order within a
// class does not matter to any result).
constexpr uint32_t PLAN_THREADS = 1024, CLASSES = 1024;
__global__ void __launch_bounds__(PLAN_THREADS) moe_attn_plan_kernel(AttnArgs a, uint32_t seqs, uint4 *plan, uint32_t *pairs, uint32_t most_pairs) {
    __shared__ uint32_t place[CLASSES];
    __shared__ uint32_t warp_sum[32];
    __shared__ uint32_t most;
    moe_pdl_begin();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, step = 2u * a.tile_tokens;
    place[threadIdx.x] = 0;
    if (threadIdx.x == 0) most = 1;
    __syncthreads();
    uint32_t longest = 0;
    for (uint32_t s = threadIdx.x; s < seqs; s += PLAN_THREADS) {
        if (a.cu_q[s] > a.cu_q[s + 1u] || a.cu_q[s + 1u] > a.rows_q || a.cu_k[s] > a.cu_k[s + 1u] || a.cu_k[s + 1u] > a.rows_k)
            moe_deny(a.status, MOE_SITE_ROWS);
        longest = max(longest, span(a.cu_k[s], a.cu_k[s + 1u], a.rows_k));
    }
    atomicMax(&most, longest);
    __syncthreads();
    const uint32_t per = (most / BLOCK_KEYS + 1u) / CLASSES + 1u;   // key blocks of one class
    for (uint32_t pass = 0; pass < 2; pass += 1) {
        for (uint32_t s = warp; s < seqs; s += PLAN_THREADS / 32u) {
            Pair p;
            const uint32_t q0 = a.cu_q[s], lq = span(q0, a.cu_q[s + 1u], a.rows_q);
            p.k_row = a.cu_k[s];
            p.lk = span(p.k_row, a.cu_k[s + 1u], a.rows_k);
            for (uint32_t i = lane * step; i < lq; i += 32u * step) {
                p.q_row = q0 + i;
                p.left = lq - i;
                const uint32_t n = min(CLASSES - 1u, blocks_of(p, a.tile_tokens).n / per), cls = CLASSES - 1u - n;
                const uint32_t at = atomicAdd(&place[cls], 1u);
                if (pass != 0 && at < most_pairs) plan[at] = make_uint4(p.q_row, p.left, p.k_row, p.lk);   // offsets that fall (denied above) may give more
            }
        }
        __syncthreads();
        if (pass != 0) break;
        const uint32_t mine = place[threadIdx.x];
        uint32_t incl = mine;
#pragma unroll
        for (uint32_t o = 1; o < 32; o <<= 1) {
            const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        if (lane == 31) warp_sum[warp] = incl;
        __syncthreads();
        uint32_t before = 0;
        for (uint32_t w = 0; w < warp; w += 1) before += warp_sum[w];
        place[threadIdx.x] = before + incl - mine;
        if (threadIdx.x == PLAN_THREADS - 1u) *pairs = min(before + incl, most_pairs);
        __syncthreads();
    }
}

template <uint32_t HD>
void attn_launch(moe_cuda_ctx *c, const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv, const AttnArgs &a, uint32_t grid, uint32_t slot) {
    constexpr uint32_t smem = Cfg<HD>::SMEM + sizeof(AttnBars<Cfg<HD>::STAGES>) + 1024;
    static_assert(smem <= 227 * 1024, "shared memory of one SM");
    if (!c->attn_attr_set[slot]) {
        MOE_CUDA_TRY(c, cudaFuncSetAttribute(moe_attn_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        c->attn_attr_set[slot] = true;
    }
    moe_run(c, moe_attn_kernel<HD>, grid, AT_THREADS, smem, tq, tk, tv, a);
    MOE_LAUNCHED(c);
}

}  // namespace

extern "C" void moe_cuda_attn(moe_cuda_ctx_t *c, const void *q16, const void *k16, const void *v16, const uint32_t *cu_q, const uint32_t *cu_k,
                              void *o16, struct moe_pc_attn_t pc) {
    if (!MOE_LIVE(c)) return;
    const char *why = moe_attn_refusal(q16, k16, v16, cu_q, cu_k, o16, pc);
    MOE_REQUIRE(c, why == NULL, "%s", why);
    if (pc.rows_q == 0 || pc.seqs == 0) return;
    moe_on_device on(c);
    AttnArgs a;
    a.cu_q = cu_q;
    a.cu_k = cu_k;
    a.v = (const __half *)v16;
    a.o = (__half *)o16;
    a.plan = NULL;
    a.pairs = NULL;
    a.rows_q = pc.rows_q;
    a.rows_k = pc.rows_k;
    a.kv_heads = pc.kv_heads;
    a.group = pc.heads / pc.kv_heads;
    a.tile_tokens = TILE_ROWS / a.group;
    a.kv_stride = pc.kv_stride;
    a.o_stride = pc.o_stride;
    a.scale = pc.scale;
    const float to_log2 = pc.scale * LOG2E;
    uint32_t bits;
    memcpy(&bits, &to_log2, sizeof(bits));
    const int32_t far = 127 + FAR - ((int32_t)(bits >> 23) - 127);
    a.far_top = (uint32_t)(far < 255 ? far : 255) << 23;   // 255: not even infinity's; else the scale keeps an exponent of 22 there
    a.far_scale = bits + a.far_top;
    a.status = c->dev_status_dev;
    a.wait_ns = c->wait_ns;
    const uint64_t pairs = (uint64_t)pc.rows_q / (2u * a.tile_tokens) + pc.seqs;   // at most
    MOE_REQUIRE(c, pairs * pc.kv_heads < (1ull << 31), "attn: too many tiles");
    CUtensorMap tq, tk, tv;
    if (!moe_tmap_heads_f16(c, &tq, q16, pc.rows_q, pc.heads, pc.hd, pc.q_stride, a.group, a.tile_tokens, 1)) return;
    if (pc.rows_k == 0) {
        tk = tv = tq;   // never loaded from
    } else if (!moe_tmap_heads_f16(c, &tk, k16, pc.rows_k, pc.kv_heads, pc.hd, pc.kv_stride, 1, BLOCK_KEYS, pc.hd / 64u) ||
               !moe_tmap_heads_f16(c, &tv, v16, pc.rows_k, pc.kv_heads, pc.hd, pc.kv_stride, 1, BLOCK_KEYS, pc.hd / 64u)) {
        return;
    }
    if (pc.seqs > 1u) {
        const size_t need = 256 + (size_t)pairs * sizeof(uint4);
        if (need > c->work_bytes) {
            moe_fail(c, MOE_ERR_NOMEM, "attn: %zu bytes of work area, the context has %zu", need, c->work_bytes);
            return;
        }
        a.pairs = (const uint32_t *)c->work;
        a.plan = (const uint4 *)((uint8_t *)c->work + 256);
        moe_run(c, moe_attn_plan_kernel, 1, PLAN_THREADS, 0, a, pc.seqs, (uint4 *)a.plan, (uint32_t *)a.pairs, (uint32_t)pairs);
        MOE_LAUNCHED(c);
    }
    const uint64_t items = pairs * pc.kv_heads;
    const uint32_t grid = items < (uint64_t)c->sm_count ? (uint32_t)items : (uint32_t)c->sm_count;
    if (pc.hd == 128u) attn_launch<128>(c, tq, tk, tv, a, grid, 0);
    else attn_launch<64>(c, tq, tk, tv, a, grid, 1);
}
