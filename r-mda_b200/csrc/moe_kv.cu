// The steps around attention that move rows: rotary positions with the fp32 -> fp16 rounding of the projection's output,
// keys and values into the paged cache (fp16, or e4m3 with a power-of-two scale per token and head) and back out of it.
// All three are bound by HBM; each reads its input once and writes its output once.
#include <cuda_fp8.h>

#include "moe_attn.cuh"

namespace {

constexpr uint32_t ROPE_THREADS = 256;

// y = x rotated: (x_i, x_{i + rot/2}) turn by pos * theta^(-2i/rot).  Far positions times a frequency need more than 24
// bits before the whole turns are taken off, so angles are in turns and in double until their fraction is left; a block
// makes the frequencies once and a row's sines once, for all its heads.
__global__ void __launch_bounds__(ROPE_THREADS) moe_rope_kernel(const float *x, const uint32_t *pos, __half *out, moe_pc_rope_t pc) {
    __shared__ float2 turn[2][ROPE_THREADS];
    const uint32_t half = pc.rot_heads != 0 ? pc.rot / 2u : 0u, hd4 = pc.hd / 4u, units = pc.heads * hd4;
    double freq = 0.0;  // turns per position of pair threadIdx.x
    if (threadIdx.x < half) freq = exp2(-(double)threadIdx.x / (double)half * log2((double)pc.theta)) * 0.15915494309189535;
    moe_pdl_begin();
    uint32_t buf = 0;
    for (uint32_t r = blockIdx.x; r < pc.rows; r += gridDim.x) {
        if (threadIdx.x < half) {
            double t = (double)pos[r] * freq;
            t -= rint(t);
            float s, c;
            sincospif((float)(2.0 * t), &s, &c);
            turn[buf][threadIdx.x] = make_float2(c, s);
        }
        __syncthreads();
        const float *xr = x + (size_t)r * pc.stride;
        __half *yr = out + (size_t)r * pc.out_stride;
        for (uint32_t u0 = threadIdx.x; u0 < units; u0 += 4u * ROPE_THREADS) {
            float4 a[4], b[4];
            int32_t at[4];  // first pair of this unit; -1: not rotated; with bit 30: the unit is the pairs' second half
#pragma unroll
            for (uint32_t j = 0; j < 4; j += 1) {
                const uint32_t u = u0 + j * ROPE_THREADS;
                at[j] = -1;
                if (u >= units) continue;
                a[j] = *reinterpret_cast<const float4 *>(xr + u * 4u);
                const uint32_t head = u / hd4, col = (u - head * hd4) * 4u;
                if (head < pc.rot_heads && col < 2u * half) {
                    const bool second = col >= half;
                    at[j] = (int32_t)(second ? (col - half) | (1u << 30) : col);
                    b[j] = *reinterpret_cast<const float4 *>(xr + u * 4u + (second ? 0 : half) - (second ? half : 0));
                }
            }
#pragma unroll
            for (uint32_t j = 0; j < 4; j += 1) {
                const uint32_t u = u0 + j * ROPE_THREADS;
                if (u >= units) continue;
                float v[4] = {a[j].x, a[j].y, a[j].z, a[j].w};
                if (at[j] >= 0) {
                    const float w[4] = {b[j].x, b[j].y, b[j].z, b[j].w};
                    const float sign = (at[j] >> 30) != 0 ? 1.0f : -1.0f;
#pragma unroll
                    for (uint32_t k = 0; k < 4; k += 1) {
                        const float2 cs = turn[buf][(at[j] & 0xffff) + k];
                        v[k] = v[k] * cs.x + sign * w[k] * cs.y;
                    }
                }
                const __half2 lo = __floats2half2_rn(v[0], v[1]), hi = __floats2half2_rn(v[2], v[3]);
                *reinterpret_cast<uint2 *>(yr + u * 4u) =
                    make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
            }
        }
        buf ^= 1u;
    }
}

struct KvArgs {
    uint8_t *k, *v;
    float *k_scale, *v_scale;
    uint32_t pages, page, page_shift, kv_heads;
    uint32_t *status;
};

// Index of a slot's head row among all [pages][kv_heads][page] rows.
__device__ __forceinline__ size_t kv_row(const KvArgs &kv, uint32_t slot, uint32_t head) {
    return (((size_t)(slot >> kv.page_shift) * kv.kv_heads + head) << kv.page_shift) + (slot & (kv.page - 1u));
}

__device__ __forceinline__ float f16_bits(uint32_t w, uint32_t i) {
    return __half2float(__ushort_as_half((unsigned short)(i != 0 ? w >> 16 : w & 0xffffu)));
}

// Eight fp16 values (two per word) as e4m3 codes of value * inv, rounded once to nearest even, clipped to the largest code.
__device__ __forceinline__ uint2 to_e4m3(uint4 x, float inv) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t p[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; i += 1) {
        p[i] = __nv_cvt_float2_to_fp8x2(make_float2(f16_bits(w[i], 0) * inv, f16_bits(w[i], 1) * inv), __NV_SATFINITE, __NV_E4M3);
    }
    return make_uint2(p[0] | (p[1] << 16), p[2] | (p[3] << 16));
}

// The least power of two s with amax <= 448 s, from amax's bits: 448 = 1.75 * 2^8.
__device__ __forceinline__ int32_t e4m3_exponent(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    return amax == 0.0f ? 0 : (int32_t)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
}

constexpr uint32_t KV_THREADS = 256;

// LPV = hd / 8 lanes hold one head's keys or values of one row, 16 bytes each.
template <bool FP8, uint32_t LPV>
__global__ void __launch_bounds__(KV_THREADS) moe_kv_write_kernel(const __half *k16, const __half *v16, const uint32_t *slot, KvArgs kv,
                                                                   moe_pc_kv_write_t pc) {
    moe_pdl_begin();
    const uint32_t per_row = 2u * kv.kv_heads, total = pc.rows * per_row;  // below 2^31
    const uint32_t lane = threadIdx.x % LPV, step = gridDim.x * (KV_THREADS / LPV);
    const uint64_t limit = (uint64_t)kv.pages * kv.page;
    constexpr uint32_t UN = 2;
    for (uint32_t u0 = blockIdx.x * (KV_THREADS / LPV) + threadIdx.x / LPV; u0 - threadIdx.x / LPV < total; u0 += UN * step) {
        uint4 x[UN];
        uint32_t at[UN], vec[UN];
#pragma unroll
        for (uint32_t j = 0; j < UN; j += 1) {
            const uint32_t u = u0 + j * step;
            const bool in = u < total && u >= u0;
            const uint32_t row = in ? u / per_row : 0u;
            vec[j] = in ? u - row * per_row : 0u;
            at[j] = in ? slot[row] : MDA_PC_NO_SLOT;
            const bool is_v = vec[j] >= kv.kv_heads;
            const uint32_t head = is_v ? vec[j] - kv.kv_heads : vec[j];
            x[j] = make_uint4(0, 0, 0, 0);
            if (in) x[j] = *reinterpret_cast<const uint4 *>((is_v ? v16 : k16) + (size_t)row * pc.stride + (head * LPV + lane) * 8u);
        }
#pragma unroll
        for (uint32_t j = 0; j < UN; j += 1) {
            const bool is_v = vec[j] >= kv.kv_heads;
            const uint32_t head = is_v ? vec[j] - kv.kv_heads : vec[j];
            const bool keep = at[j] < limit;
            if (!keep && at[j] != MDA_PC_NO_SLOT && lane == 0) moe_deny(kv.status, MOE_SITE_SLOT);
            const size_t row = keep ? kv_row(kv, at[j], head) : 0;
            uint8_t *dst = is_v ? kv.v : kv.k;
            if (!FP8) {
                if (keep) *reinterpret_cast<uint4 *>(dst + (row * LPV + lane) * 16u) = x[j];
            } else {
                const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
                float amax = 0.0f;  // fmaxf passes over NaN
#pragma unroll
                for (uint32_t i = 0; i < 4; i += 1) amax = fmaxf(amax, fmaxf(fabsf(f16_bits(w[i], 0)), fabsf(f16_bits(w[i], 1))));
#pragma unroll
                for (uint32_t o = LPV / 2u; o != 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                const int32_t e = e4m3_exponent(fminf(amax, 65504.0f));
                const uint2 code = to_e4m3(x[j], __uint_as_float((uint32_t)(127 - e) << 23));
                if (keep) {
                    *reinterpret_cast<uint2 *>(dst + (row * LPV + lane) * 8u) = code;
                    if (lane == 0) (is_v ? kv.v_scale : kv.k_scale)[row] = __uint_as_float((uint32_t)(127 + e) << 23);
                }
            }
        }
    }
}

constexpr uint32_t READ_ROWS = 64;  // most rows a block takes at a time

template <bool FP8, uint32_t LPV>
__global__ void __launch_bounds__(KV_THREADS) moe_kv_read_kernel(const uint32_t *table, const uint32_t *cu, __half *k16, __half *v16, KvArgs kv,
                                                                  moe_pc_kv_read_t pc, uint32_t tile) {
    __shared__ uint32_t at[READ_ROWS];
    moe_pdl_begin();
    const uint32_t last = min(cu[pc.seqs], pc.rows);
    const uint32_t lane = threadIdx.x % LPV, per_row = 2u * kv.kv_heads;
    for (uint64_t r0 = (uint64_t)blockIdx.x * tile; r0 < last; r0 += (uint64_t)gridDim.x * tile) {
        const uint32_t n = min(tile, last - (uint32_t)r0);
        __syncthreads();
        if (threadIdx.x < n) {
            const uint32_t r = (uint32_t)r0 + threadIdx.x;
            uint32_t lo = 0, hi = pc.seqs;  // the sequence of row r: cu[lo] <= r < cu[hi]
            while (hi - lo > 1u) {
                const uint32_t mid = (lo + hi) / 2u;
                if (cu[mid] <= r) lo = mid;
                else hi = mid;
            }
            const uint32_t first = cu[lo], place = r - first;
            uint32_t s = MDA_PC_NO_SLOT;
            if (r >= first && place >> kv.page_shift < pc.table_stride) {
                const uint32_t pg = table[(size_t)lo * pc.table_stride + (place >> kv.page_shift)];
                if (pg < kv.pages) s = (pg << kv.page_shift) + (place & (kv.page - 1u));
            }
            if (s == MDA_PC_NO_SLOT) moe_deny(kv.status, MOE_SITE_PAGE);
            at[threadIdx.x] = s;
        }
        __syncthreads();
        constexpr uint32_t UN = 4, VPB = KV_THREADS / LPV;
        const uint32_t total = n * per_row;
        for (uint32_t u0 = threadIdx.x / LPV; u0 < total; u0 += UN * VPB) {
            uint4 x[UN];
            float scale[UN];
            uint32_t row[UN];
#pragma unroll
            for (uint32_t j = 0; j < UN; j += 1) {
                const uint32_t u = u0 + j * VPB;
                row[j] = u < total ? u / per_row : ~0u;
                if (row[j] != ~0u && at[row[j]] == MDA_PC_NO_SLOT) row[j] = ~0u;
                if (row[j] == ~0u) continue;
                const uint32_t vec = u - row[j] * per_row;
                const bool is_v = vec >= kv.kv_heads;
                const size_t src = kv_row(kv, at[row[j]], is_v ? vec - kv.kv_heads : vec);
                const uint8_t *from = is_v ? kv.v : kv.k;
                if (FP8) {
                    const uint2 c = *reinterpret_cast<const uint2 *>(from + (src * LPV + lane) * 8u);
                    x[j] = make_uint4(c.x, c.y, 0, 0);
                    scale[j] = (is_v ? kv.v_scale : kv.k_scale)[src];
                } else {
                    x[j] = *reinterpret_cast<const uint4 *>(from + (src * LPV + lane) * 16u);
                }
            }
#pragma unroll
            for (uint32_t j = 0; j < UN; j += 1) {
                if (row[j] == ~0u) continue;
                const uint32_t vec = u0 + j * VPB - row[j] * per_row;
                const bool is_v = vec >= kv.kv_heads;
                if (FP8) {
                    const uint32_t c[2] = {x[j].x, x[j].y};
                    uint32_t o[4];
#pragma unroll
                    for (uint32_t i = 0; i < 4; i += 1) {
                        const uint32_t h2 = e4m3x2_to_h2((i & 1u) != 0 ? c[i / 2u] >> 16 : c[i / 2u] & 0xffffu);
                        const __half2 y = __floats2half2_rn(f16_bits(h2, 0) * scale[j], f16_bits(h2, 1) * scale[j]);
                        o[i] = *reinterpret_cast<const uint32_t *>(&y);
                    }
                    x[j] = make_uint4(o[0], o[1], o[2], o[3]);
                }
                __half *dst = is_v ? v16 : k16;
                *reinterpret_cast<uint4 *>(dst + (r0 + row[j]) * (size_t)pc.stride + ((is_v ? vec - kv.kv_heads : vec) * LPV + lane) * 8u) = x[j];
            }
        }
    }
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
    const uint32_t most = (uint32_t)c->sm_count * 8u;  // resident blocks of 256 threads
    moe_run(c, moe_rope_kernel, pc.rows < most ? pc.rows : most, ROPE_THREADS, 0, x, pos, (__half *)out, pc);
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
    const uint64_t threads = (uint64_t)pc.rows * 2u * kv->kv_heads * (kv->hd / 8u);
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
    // rows per block: 64 share the look-ups best, fewer when that would leave SMs without a block
    uint32_t tile = pc.rows / ((uint32_t)c->sm_count * 4u);
    tile = tile > READ_ROWS ? READ_ROWS : tile < 4u ? 4u : tile;
    const uint64_t blocks = ((uint64_t)pc.rows + tile - 1u) / tile, most = (uint64_t)c->sm_count * 8u;
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
