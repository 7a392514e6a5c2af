// What the attention calls share: refusals, the device-side refusal, the context's device, small conversions.
#pragma once

#include "moe_attn_args.h"
#include "moe_common.cuh"

// Kinds of device-side refusals (MOE_ERR_ARG | kind << 8 in the status word).
enum { MOE_SITE_SLOT = 1, MOE_SITE_PAGE = 2, MOE_SITE_LENGTH = 3, MOE_SITE_ROWS = 4 };

// The calling thread's current device is the context's for as long as this lives.
struct moe_on_device {
    int before;
    bool moved;
    explicit moe_on_device(const moe_cuda_ctx *c) : before(0), moved(false) {
        if (cudaGetDevice(&before) == cudaSuccess && before != c->device) moved = cudaSetDevice(c->device) == cudaSuccess;
    }
    ~moe_on_device() {
        if (moved) (void)cudaSetDevice(before);
    }
    moe_on_device(const moe_on_device &) = delete;
    moe_on_device &operator=(const moe_on_device &) = delete;
};

static inline uint32_t moe_log2(uint32_t power_of_two) {
    uint32_t n = 0;
    while ((1u << n) < power_of_two) n += 1;
    return n;
}

// Division of numbers below 2^31 by a number that the host knows: q = (mulhi(m, n) + n) >> s with 2^s >= d and
// m = floor(2^32 (2^s - d) / d) + 1, exact by the round-up method of Granlund and Montgomery.
struct moe_divisor {
    uint32_t d, m, s;
};
static inline moe_divisor moe_divide_by(uint32_t d) {
    moe_divisor v = {d, 0, 0};
    while ((1u << v.s) < d) v.s += 1;
    v.m = (uint32_t)(((((uint64_t)1 << v.s) - d) << 32) / d + 1u);
    return v;
}
__device__ __forceinline__ uint32_t moe_quotient(uint32_t n, const moe_divisor &v) { return (__umulhi(v.m, n) + n) >> v.s; }

__device__ __forceinline__ void moe_deny(uint32_t *status, uint32_t kind) { atomicCAS(status, 0u, (uint32_t)MOE_ERR_ARG | (kind << 8)); }

// Four e4m3 codes as two pairs of fp16 values; exact, NaN stays NaN.
__device__ __forceinline__ void e4m3x4_to_h2(uint32_t codes, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}\n"
        : "=r"(lo), "=r"(hi)
        : "r"(codes));
}
