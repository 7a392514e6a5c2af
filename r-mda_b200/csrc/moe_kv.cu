// The steps around attention that move rows: rotary positions with the fp32 -> fp16 rounding of the projection's output,
// keys and values into the paged cache (fp16, or e4m3 with a power-of-two scale per token and head) and back out of it.
// Each reads its input once and writes its output once.  The floor is HBM's, but what bound the first forms of all three was
// instruction issue: hence multiplications for divisions, fp16x2 arithmetic, and a thread that has keys and values of a head.
// One B200, back to back: rope of 4096 rows of 40 heads of 128, half rotated, 25.6 us = 4.9 TB/s (0.75 of the copy rate); write of
// 16384 rows of 16 heads of 128 as e4m3 38 us = 5.4 TB/s (34 captured); read of 12 prefixes of up to 8191 tokens, e4m3, 31.4 us = 5.5
// TB/s.  Steps of 16 to 1003 rows take 1.6 to 2.5 us on the GPU.
#include "moe_attn.cuh"

namespace {

constexpr uint32_t ROPE_THREADS = 256, ROPE_BLOCKS = 6;   // blocks of an SM

struct RopeArgs {
    const float *x;
    const uint32_t *pos;
    __half *out;
    moe_pc_rope_t pc;
    uint32_t half, pairs, tails, plain;   // pieces of 4 columns in a row: pairs of pieces to turn, the rest of turned heads, the other heads
    moe_divisor by_half, by_tail;         // pieces of one head's first half, and of its rest
};

__device__ __forceinline__ uint2 to_f16x4(float a, float b, float c, float d) {
    const __half2 lo = __floats2half2_rn(a, b), hi = __floats2half2_rn(c, d);
    return make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
}

// y = x rotated: (x_i, x_{i + rot/2}) turn by pos * theta^(-2i/rot).  Far positions times a frequency need more than 24
// bits before the whole turns are taken off, so angles are in turns and in double until their fraction is left; a block
// makes the frequencies once and a row's sines once, for all its heads.  A thread takes both halves of a pair, so every
// column is read once; two pairs are under way at a time.
__global__ void __launch_bounds__(ROPE_THREADS, ROPE_BLOCKS) moe_rope_kernel(RopeArgs a) {
    __shared__ float4 turn[2][ROPE_THREADS / 2];   // (cos, sin) of two neighbours
    const uint32_t half = a.half;
    double freq = 0.0;  // turns per position of pair threadIdx.x
    if (threadIdx.x < half) freq = exp2(-(double)threadIdx.x / (double)half * log2((double)a.pc.theta)) * 0.15915494309189535;
    moe_pdl_begin();
    // Sines of the next row are made while this one is turned.
    auto sines = [&](uint32_t r, float4 *to) {
        if (threadIdx.x >= half || r >= a.pc.rows) return;
        double t = (double)a.pos[r] * freq;
        t -= rint(t);
        float s, c;
        sincospif((float)(2.0 * t), &s, &c);
        reinterpret_cast<float2 *>(to)[threadIdx.x] = make_float2(c, s);
    };
    uint32_t buf = 0;
    sines(blockIdx.x, turn[0]);
    for (uint32_t r = blockIdx.x; r < a.pc.rows; r += gridDim.x) {
        const float *xr = a.x + (size_t)r * a.pc.stride;
        __half *yr = a.out + (size_t)r * a.pc.out_stride;
        __syncthreads();
        if (a.pc.rows - r > gridDim.x) sines(r + gridDim.x, turn[buf ^ 1u]);
        for (uint32_t u0 = threadIdx.x; u0 < a.tails + a.plain; u0 += 2u * ROPE_THREADS) {
            float4 v[2];
            uint32_t col[2];
#pragma unroll
            for (uint32_t j = 0; j < 2; j += 1) {
                const uint32_t u = u0 + j * ROPE_THREADS;
                if (u < a.tails) {
                    const uint32_t head = moe_quotient(u, a.by_tail);
                    col[j] = head * a.pc.hd + a.pc.rot + (u - head * a.by_tail.d) * 4u;
                } else {
                    col[j] = a.pc.rot_heads * a.pc.hd + (u - a.tails) * 4u;
                }
                if (u < a.tails + a.plain) v[j] = *reinterpret_cast<const float4 *>(xr + col[j]);
            }
#pragma unroll
            for (uint32_t j = 0; j < 2; j += 1) {
                if (u0 + j * ROPE_THREADS < a.tails + a.plain) *reinterpret_cast<uint2 *>(yr + col[j]) = to_f16x4(v[j].x, v[j].y, v[j].z, v[j].w);
            }
        }
        for (uint32_t u0 = threadIdx.x; u0 < a.pairs; u0 += 2u * ROPE_THREADS) {
            float4 lo[2], hi[2];
            uint32_t col[2], i[2];
#pragma unroll
            for (uint32_t j = 0; j < 2; j += 1) {
                const uint32_t u = u0 + j * ROPE_THREADS;
                if (u >= a.pairs) continue;
                const uint32_t head = moe_quotient(u, a.by_half);
                i[j] = (u - head * a.by_half.d) * 4u;
                col[j] = head * a.pc.hd + i[j];
                lo[j] = *reinterpret_cast<const float4 *>(xr + col[j]);
                hi[j] = *reinterpret_cast<const float4 *>(xr + col[j] + half);
            }
#pragma unroll
            for (uint32_t j = 0; j < 2; j += 1) {
                if (u0 + j * ROPE_THREADS >= a.pairs) continue;
                const float4 t0 = turn[buf][i[j] / 2u], t1 = turn[buf][i[j] / 2u + 1u];
                const float4 x = lo[j], y = hi[j];
                *reinterpret_cast<uint2 *>(yr + col[j]) =
                    to_f16x4(x.x * t0.x - y.x * t0.y, x.y * t0.z - y.y * t0.w, x.z * t1.x - y.z * t1.y, x.w * t1.z - y.w * t1.w);
                *reinterpret_cast<uint2 *>(yr + col[j] + half) =
                    to_f16x4(y.x * t0.x + x.x * t0.y, y.y * t0.z + x.y * t0.w, y.z * t1.x + x.z * t1.y, y.w * t1.z + x.w * t1.w);
            }
        }
        buf ^= 1u;
    }
}

struct KvArgs {
    uint8_t *k, *v;
    float *k_scale, *v_scale;
    uint32_t pages, page, page_shift, kv_heads;
    moe_divisor by_heads;
    uint32_t *status;
};

// Index of a slot's head row among all [pages][kv_heads][page] rows.
__device__ __forceinline__ size_t kv_row(const KvArgs &kv, uint32_t slot, uint32_t head) {
    return (((size_t)(slot >> kv.page_shift) * kv.kv_heads + head) << kv.page_shift) + (slot & (kv.page - 1u));
}

__device__ __forceinline__ __half2 as_h2(uint32_t w) { return *reinterpret_cast<const __half2 *>(&w); }
__device__ __forceinline__ uint32_t as_word(__half2 h) { return *reinterpret_cast<const uint32_t *>(&h); }

// Eight fp16 values (two per word) as e4m3 codes of value * f * g, rounded once to nearest even, clipped to the largest code.
// f and g are powers of two: the fp16 products are exact wherever the code is not 0 (what they make subnormal is below
// 2^-14, and half of the least code is 2^-10).
__device__ __forceinline__ uint2 to_e4m3(const uint32_t (&w)[4], __half2 f, __half2 g) {
    uint32_t p[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; i += 1) {
        const uint32_t y = as_word(__hmul2(__hmul2(as_h2(w[i]), f), g));
        asm("{\n\t.reg .b16 c;\n\tcvt.rn.satfinite.e4m3x2.f16x2 c, %1;\n\tcvt.u32.u16 %0, c;\n\t}\n" : "=r"(p[i]) : "r"(y));
    }
    return make_uint2(p[0] | (p[1] << 16), p[2] | (p[3] << 16));
}

// The least power of two s with amax <= 448 s, from amax's bits: 448 = 1.75 * 2^8.
__device__ __forceinline__ int32_t e4m3_exponent(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    return amax == 0.0f ? 0 : (int32_t)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
}

constexpr uint32_t KV_THREADS = 256;

// Codes of a vector that LPV lanes hold, eight values each, and its scale's exponent.
template <uint32_t LPV>
__device__ __forceinline__ uint2 quantise(uint4 x, int32_t &e) {
    uint32_t w[4] = {x.x, x.y, x.z, x.w};
    const __half2 most = __hmax2(__hmax2(__habs2(as_h2(w[0])), __habs2(as_h2(w[1]))), __hmax2(__habs2(as_h2(w[2])), __habs2(as_h2(w[3]))));
    uint32_t top = as_word(__hmax2(most, __half2half2(__ushort_as_half(0))));   // passes over NaN
    top = max(top & 0xffffu, top >> 16);   // not negative: ordered like their bits
#pragma unroll
    for (uint32_t o = LPV / 2u; o != 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    e = e4m3_exponent(__half2float(__ushort_as_half((unsigned short)min(top, 0x7bffu))));
    // times 2^-e in two steps, in three beyond 2^30 (it may be up to 2^32)
    if (e < -30) {
#pragma unroll
        for (uint32_t i = 0; i < 4; i += 1) w[i] = as_word(__hmul2(as_h2(w[i]), __half2half2(__ushort_as_half(0x4400))));   // 4
    }
    const int32_t rest = e < -30 ? e + 2 : e, e0 = max(-15, rest), e1 = rest - e0;
    return to_e4m3(w, __half2half2(__ushort_as_half((unsigned short)((15 - e0) << 10))), __half2half2(__ushort_as_half((unsigned short)((15 - e1) << 10))));
}

// A unit is one head of one row, keys and values: LPV = hd / 8 lanes with 16 bytes of each.
template <bool FP8, uint32_t LPV>
__global__ void __launch_bounds__(KV_THREADS, 8) moe_kv_write_kernel(const __half *k16, const __half *v16, const uint32_t *slot, KvArgs kv,
                                                                      moe_pc_kv_write_t pc) {
    moe_pdl_begin();
    const uint32_t total = pc.rows * kv.kv_heads;  // below 2^30
    const uint32_t lane = threadIdx.x % LPV, step = gridDim.x * (KV_THREADS / LPV), limit = kv.pages << kv.page_shift;
    for (uint32_t u0 = blockIdx.x * (KV_THREADS / LPV); u0 < total; u0 += step) {
        const uint32_t u = u0 + threadIdx.x / LPV;
        const bool in = u < total;
        const uint32_t row = in ? moe_quotient(u, kv.by_heads) : 0u, head = in ? u - row * kv.kv_heads : 0u;
        const uint32_t at = in ? slot[row] : MDA_PC_NO_SLOT;
        uint4 x = make_uint4(0, 0, 0, 0), y = x;
        if (in) {
            const size_t from = (size_t)row * pc.stride + (head * LPV + lane) * 8u;
            x = *reinterpret_cast<const uint4 *>(k16 + from);
            y = *reinterpret_cast<const uint4 *>(v16 + from);
        }
        const bool keep = at < limit;
        if (!keep && at != MDA_PC_NO_SLOT && lane == 0) moe_deny(kv.status, MOE_SITE_SLOT);
        const size_t to = keep ? kv_row(kv, at, head) : 0;
        if (!FP8) {
            if (keep) {
                *reinterpret_cast<uint4 *>(kv.k + (to * LPV + lane) * 16u) = x;
                *reinterpret_cast<uint4 *>(kv.v + (to * LPV + lane) * 16u) = y;
            }
        } else {
            int32_t ek, ev;
            const uint2 ck = quantise<LPV>(x, ek), cv = quantise<LPV>(y, ev);
            if (keep) {
                *reinterpret_cast<uint2 *>(kv.k + (to * LPV + lane) * 8u) = ck;
                *reinterpret_cast<uint2 *>(kv.v + (to * LPV + lane) * 8u) = cv;
                if (lane < 2u) (lane == 0 ? kv.k_scale : kv.v_scale)[to] = __uint_as_float((uint32_t)(127 + (lane == 0 ? ek : ev)) << 23);
            }
        }
    }
}

// code * scale in fp16's range.  fp16 values of an amax above 57344 are kept at scale 256, and 63488 to 65504 of them round to code
// 256: 65536, which is no fp16 value, reads as the largest one.  What lies beyond is infinite: an infinity is kept as 448 * 256.
__device__ __forceinline__ float in_f16(float y) { return fabsf(y) <= 65536.0f ? fminf(fmaxf(y, -65504.0f), 65504.0f) : y; }

// Eight codes as fp16 values of code * scale, rounded once.
__device__ __forceinline__ uint4 from_e4m3(uint2 c, float scale) {
    uint32_t o[4];
    e4m3x4_to_h2(c.x, o[0], o[1]);
    e4m3x4_to_h2(c.y, o[2], o[3]);
    const uint32_t bits = __float_as_uint(scale), e = bits >> 23;
    if ((bits & 0x807fffffu) == 0u && e >= 127u - 14u && e <= 127u + 7u) {   // a power of two that fp16 has, 448 of it too: one rounding all the same
        const __half2 f = __half2half2(__ushort_as_half((unsigned short)((e - 112u) << 10)));
#pragma unroll
        for (uint32_t i = 0; i < 4; i += 1) o[i] = as_word(__hmul2(as_h2(o[i]), f));
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; i += 1) {
            const float2 y = __half22float2(as_h2(o[i]));
            o[i] = as_word(__floats2half2_rn(in_f16(y.x * scale), in_f16(y.y * scale)));
        }
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

constexpr uint32_t READ_ROWS = 64;  // most rows a block takes at a time

template <bool FP8, uint32_t LPV>
__global__ void __launch_bounds__(KV_THREADS, 6) moe_kv_read_kernel(const uint32_t *table, const uint32_t *cu, __half *k16, __half *v16, KvArgs kv,
                                                                  moe_pc_kv_read_t pc, uint32_t tile) {
    __shared__ uint32_t slots[2][READ_ROWS];
    moe_pdl_begin();
    const uint32_t total_rows = cu[pc.seqs], last = min(total_rows, pc.rows);
    const uint32_t lane = threadIdx.x % LPV;
    // Offsets that fall or pass the rows are refused: a thread loads those of a sequence here and looks at them at the end.
    uint32_t mine = blockIdx.x * KV_THREADS + threadIdx.x, begin = 0, end = 0;
    if (mine < pc.seqs) {
        begin = cu[mine];
        end = cu[mine + 1u];
    }
    // Slots of a tile's rows, a row per thread; those of the next tile are looked up while this one is copied.
    auto look_up = [&](uint64_t r0, uint32_t *to) {
        if (threadIdx.x >= tile || r0 + threadIdx.x >= last) return;
        const uint32_t r = (uint32_t)r0 + threadIdx.x;
        uint32_t lo = 0, hi = pc.seqs, stop = total_rows;  // the sequence of row r: cu[lo] <= r < cu[hi] = stop
        while (hi - lo > 1u) {
            const uint32_t mid = (lo + hi) / 2u, at = cu[mid];
            if (at <= r) {
                lo = mid;
            } else {
                hi = mid;
                stop = at;
            }
        }
        const uint32_t first = cu[lo], place = r - first;
        uint32_t s = MDA_PC_NO_SLOT;
        // rows before the first sequence are no one's, and a sequence that passes the rows (refused at the end) is left
        if (r >= first && stop <= pc.rows) {
            if (place >> kv.page_shift < pc.table_stride) {
                const uint32_t pg = table[(size_t)lo * pc.table_stride + (place >> kv.page_shift)];
                if (pg < kv.pages) s = (pg << kv.page_shift) + (place & (kv.page - 1u));
            }
            if (s == MDA_PC_NO_SLOT) moe_deny(kv.status, MOE_SITE_PAGE);
        }
        to[threadIdx.x] = s;
    };
    uint32_t buf = 0;
    const uint64_t step = (uint64_t)gridDim.x * tile;
    look_up((uint64_t)blockIdx.x * tile, slots[0]);
    for (uint64_t r0 = (uint64_t)blockIdx.x * tile; r0 < last; r0 += step) {
        const uint32_t n = min(tile, last - (uint32_t)r0);
        __syncthreads();
        look_up(r0 + step, slots[buf ^ 1u]);
        const uint32_t *at = slots[buf];
        buf ^= 1u;
        constexpr uint32_t UN = 2, VPB = KV_THREADS / LPV;
        const uint32_t total = n * kv.kv_heads;
        for (uint32_t u0 = threadIdx.x / LPV; u0 < total; u0 += UN * VPB) {
            // Loads without branches between them, so that all are under way at once: units that are not there load slot 0.
            uint4 x[UN], y[UN];
            float ks[UN], vs[UN];
            size_t to[UN];
            bool ok[UN];
#pragma unroll
            for (uint32_t j = 0; j < UN; j += 1) {
                const uint32_t u = min(u0 + j * VPB, total - 1u);
                const uint32_t row = moe_quotient(u, kv.by_heads), head = u - row * kv.kv_heads, s = at[row];
                ok[j] = u0 + j * VPB < total && s != MDA_PC_NO_SLOT;
                to[j] = (size_t)((uint32_t)r0 + row) * pc.stride + (head * LPV + lane) * 8u;
                const size_t from = kv_row(kv, s != MDA_PC_NO_SLOT ? s : 0u, head);
                if (FP8) {
                    const uint2 c = *reinterpret_cast<const uint2 *>(kv.k + (from * LPV + lane) * 8u), d = *reinterpret_cast<const uint2 *>(kv.v + (from * LPV + lane) * 8u);
                    x[j] = make_uint4(c.x, c.y, 0, 0);
                    y[j] = make_uint4(d.x, d.y, 0, 0);
                    ks[j] = kv.k_scale[from];
                    vs[j] = kv.v_scale[from];
                } else {
                    x[j] = *reinterpret_cast<const uint4 *>(kv.k + (from * LPV + lane) * 16u);
                    y[j] = *reinterpret_cast<const uint4 *>(kv.v + (from * LPV + lane) * 16u);
                }
            }
#pragma unroll
            for (uint32_t j = 0; j < UN; j += 1) {
                if (!ok[j]) continue;
                *reinterpret_cast<uint4 *>(k16 + to[j]) = FP8 ? from_e4m3(make_uint2(x[j].x, x[j].y), ks[j]) : x[j];
                *reinterpret_cast<uint4 *>(v16 + to[j]) = FP8 ? from_e4m3(make_uint2(y[j].x, y[j].y), vs[j]) : y[j];
            }
        }
    }
    while (mine < pc.seqs) {
        if (begin > end || end > pc.rows) moe_deny(kv.status, MOE_SITE_ROWS);
        mine += gridDim.x * KV_THREADS;
        if (mine >= pc.seqs) break;
        begin = cu[mine];
        end = cu[mine + 1u];
    }
}

// Almost always nothing to do: a block looks at *first and ends.
__global__ void __launch_bounds__(KV_THREADS) moe_clear_behind_kernel(uint4 *out, const uint32_t *first, uint32_t rows, uint32_t row16) {
    moe_pdl_begin();
    const uint64_t end = (uint64_t)rows * row16, step = (uint64_t)gridDim.x * KV_THREADS;
    for (uint64_t i = (uint64_t)*first * row16 + blockIdx.x * KV_THREADS + threadIdx.x; i < end; i += step) out[i] = make_uint4(0, 0, 0, 0);
}

KvArgs kv_args(moe_cuda_ctx *c, const moe_cuda_kv_t *kv) {
    KvArgs a;
    a.k = (uint8_t *)kv->k;
    a.v = (uint8_t *)kv->v;
    a.k_scale = kv->k_scale;
    a.v_scale = kv->v_scale;
    a.pages = kv->pages;
    a.page = kv->page;
    a.page_shift = moe_log2(kv->page);
    a.kv_heads = kv->kv_heads;
    a.by_heads = moe_divide_by(kv->kv_heads);
    a.status = c->dev_status_dev;
    return a;
}

}  // namespace

extern "C" void moe_cuda_rope(moe_cuda_ctx_t *c, const float *x, const uint32_t *pos, void *out, struct moe_pc_rope_t pc) {
    if (!MOE_LIVE(c)) return;
    const char *why = moe_rope_refusal(x, pos, out, pc);
    MOE_REQUIRE(c, why == NULL, "%s", why);
    if (pc.rows == 0) return;
    moe_on_device on(c);
    RopeArgs a;
    a.x = x;
    a.pos = pos;
    a.out = (__half *)out;
    a.pc = pc;
    a.half = pc.rot_heads != 0 ? pc.rot / 2u : 0u;
    const uint32_t tail = pc.rot_heads != 0 ? (pc.hd - pc.rot) / 4u : 0u;
    a.by_half = moe_divide_by(a.half != 0 ? a.half / 4u : 1u);
    a.by_tail = moe_divide_by(tail != 0 ? tail : 1u);
    a.pairs = pc.rot_heads * (a.half / 4u);
    a.tails = pc.rot_heads * tail;
    a.plain = (pc.heads - pc.rot_heads) * (pc.hd / 4u);
    const uint32_t most = (uint32_t)c->sm_count * ROPE_BLOCKS;
    moe_run(c, moe_rope_kernel, pc.rows < most ? pc.rows : most, ROPE_THREADS, 0, a);
    MOE_LAUNCHED(c);
}

extern "C" void moe_cuda_kv_write(moe_cuda_ctx_t *c, const moe_cuda_kv_t *kv, const void *k16, const void *v16, const uint32_t *slot,
                                  struct moe_pc_kv_write_t pc) {
    if (!MOE_LIVE(c)) return;
    const char *why = moe_kv_write_refusal(kv, k16, v16, slot, pc);
    MOE_REQUIRE(c, why == NULL, "%s", why);
    if (pc.rows == 0) return;
    moe_on_device on(c);
    const KvArgs a = kv_args(c, kv);
    const uint64_t threads = (uint64_t)pc.rows * kv->kv_heads * (kv->hd / 8u);
    const uint64_t blocks = (threads + KV_THREADS - 1u) / KV_THREADS, most = (uint64_t)c->sm_count * 8u;
    const uint32_t grid = (uint32_t)(blocks < most ? blocks : most);
    const __half *k = (const __half *)k16, *v = (const __half *)v16;
    if (kv->type == MOE_KV_E4M3) {
        if (kv->hd == 128u) moe_run(c, moe_kv_write_kernel<true, 16>, grid, KV_THREADS, 0, k, v, slot, a, pc);
        else moe_run(c, moe_kv_write_kernel<true, 8>, grid, KV_THREADS, 0, k, v, slot, a, pc);
    } else {
        if (kv->hd == 128u) moe_run(c, moe_kv_write_kernel<false, 16>, grid, KV_THREADS, 0, k, v, slot, a, pc);
        else moe_run(c, moe_kv_write_kernel<false, 8>, grid, KV_THREADS, 0, k, v, slot, a, pc);
    }
    MOE_LAUNCHED(c);
}

extern "C" void moe_cuda_kv_read(moe_cuda_ctx_t *c, const moe_cuda_kv_t *kv, const uint32_t *table, const uint32_t *cu, void *k16, void *v16,
                                 struct moe_pc_kv_read_t pc) {
    if (!MOE_LIVE(c)) return;
    const char *why = moe_kv_read_refusal(kv, table, cu, k16, v16, pc);
    MOE_REQUIRE(c, why == NULL, "%s", why);
    if (pc.rows == 0 || pc.seqs == 0) return;
    moe_on_device on(c);
    const KvArgs a = kv_args(c, kv);
    // Rows of a tile: eight tiles to each of the 6 x SMs blocks, so that they end together (51 k rows of 4 heads of 128 in e4m3: 32 us;
    // one tile to a block 40 us), 4 to 64 rows
    uint32_t tile = pc.rows / ((uint32_t)c->sm_count * 48u);
    tile = tile > READ_ROWS ? READ_ROWS : tile < 4u ? 4u : tile;
    const uint64_t blocks = ((uint64_t)pc.rows + tile - 1u) / tile, most = (uint64_t)c->sm_count * 6u;
    const uint32_t grid = (uint32_t)(blocks < most ? blocks : most);
    __half *k = (__half *)k16, *v = (__half *)v16;
    if (kv->type == MOE_KV_E4M3) {
        if (kv->hd == 128u) moe_run(c, moe_kv_read_kernel<true, 16>, grid, KV_THREADS, 0, table, cu, k, v, a, pc, tile);
        else moe_run(c, moe_kv_read_kernel<true, 8>, grid, KV_THREADS, 0, table, cu, k, v, a, pc, tile);
    } else {
        if (kv->hd == 128u) moe_run(c, moe_kv_read_kernel<false, 16>, grid, KV_THREADS, 0, table, cu, k, v, a, pc, tile);
        else moe_run(c, moe_kv_read_kernel<false, 8>, grid, KV_THREADS, 0, table, cu, k, v, a, pc, tile);
    }
    MOE_LAUNCHED(c);
}

extern "C" void moe_cuda_clear_behind(moe_cuda_ctx_t *c, void *out, const uint32_t *first, uint32_t rows, uint32_t row_bytes) {
    if (!MOE_LIVE(c)) return;
    const char *why = moe_clear_refusal(out, first, rows, row_bytes);
    MOE_REQUIRE(c, why == NULL, "%s", why);
    if (rows == 0 || row_bytes == 0) return;
    moe_on_device on(c);
    moe_run(c, moe_clear_behind_kernel, (uint32_t)c->sm_count, KV_THREADS, 0, (uint4 *)out, first, rows, row_bytes / 16u);
    MOE_LAUNCHED(c);
}
