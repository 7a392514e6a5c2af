// Causal attention over packed prompts: one warp per (query row, head), keys in lanes.  The plain kernel.
#include "moe_attn.cuh"

namespace {

struct AttnArgs {
    const __half *q, *k, *v;
    const uint32_t *cu_q, *cu_k;
    __half *o;
    moe_pc_attn_t pc;
    uint32_t group;
};

template <uint32_t HD>
__global__ void __launch_bounds__(128) moe_attn_kernel(AttnArgs a) {
    __shared__ float qs[4][HD];
    moe_pdl_begin();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint64_t total = (uint64_t)min(a.cu_q[a.pc.seqs], a.pc.rows_q) * a.pc.heads;
    for (uint64_t w = (uint64_t)blockIdx.x * 4u + warp; w < total; w += (uint64_t)gridDim.x * 4u) {
        const uint32_t row = (uint32_t)(w / a.pc.heads), head = (uint32_t)(w % a.pc.heads), kh = head / a.group;
        uint32_t lo = 0, hi = a.pc.seqs;
        while (hi - lo > 1u) {
            const uint32_t mid = (lo + hi) / 2u;
            if (a.cu_q[mid] <= row) lo = mid;
            else hi = mid;
        }
        const int64_t k0 = a.cu_k[lo], k1 = min(a.cu_k[lo + 1u], a.pc.rows_k), lk = max(k1 - k0, (int64_t)0);
        const int64_t seen = (int64_t)row - a.cu_q[lo + 1u] + lk + 1;
        for (uint32_t d = lane; d < HD; d += 32u) qs[warp][d] = __half2float(a.q[(size_t)row * a.pc.q_stride + head * HD + d]) * a.pc.scale;
        __syncwarp();
        float m = -INFINITY, l = 0.0f, o[HD / 32u] = {};
        for (int64_t j0 = 0; j0 < seen; j0 += 32) {
            const int64_t j = j0 + lane;
            float s = -INFINITY;
            if (j < seen) {
                const __half *kr = a.k + (size_t)(k0 + j) * a.pc.kv_stride + kh * HD;
                s = 0.0f;
                for (uint32_t d = 0; d < HD; d += 1) s += qs[warp][d] * __half2float(kr[d]);
            }
            float t = s;
            for (uint32_t x = 16; x != 0; x >>= 1) t = fmaxf(t, __shfl_xor_sync(~0u, t, x));
            t = fmaxf(m, t);
            const float keep = m == t ? 1.0f : expf(m - t), p = t == -INFINITY ? 0.0f : expf(s - t);
            float sum = p;
            for (uint32_t x = 16; x != 0; x >>= 1) sum += __shfl_xor_sync(~0u, sum, x);
            l = l * keep + sum;
            m = t;
            for (uint32_t i = 0; i < HD / 32u; i += 1) o[i] *= keep;
            for (uint32_t x = 0; x < 32u && j0 + x < seen; x += 1) {
                const float pj = __shfl_sync(~0u, p, x);
                const __half *vr = a.v + (size_t)(k0 + j0 + x) * a.pc.kv_stride + kh * HD;
                for (uint32_t i = 0; i < HD / 32u; i += 1) o[i] += pj * __half2float(vr[i * 32u + lane]);
            }
        }
        for (uint32_t i = 0; i < HD / 32u; i += 1) {
            a.o[(size_t)row * a.pc.o_stride + head * HD + i * 32u + lane] = __float2half(l == 0.0f ? 0.0f : o[i] / l);
        }
        __syncwarp();
    }
}

}  // namespace

extern "C" void moe_cuda_attn(moe_cuda_ctx_t *c, const void *q16, const void *k16, const void *v16, const uint32_t *cu_q, const uint32_t *cu_k,
                              void *o16, struct moe_pc_attn_t pc) {
    if (!MOE_LIVE(c)) return;
    const char *why = moe_attn_refusal(q16, k16, v16, cu_q, cu_k, o16, pc);
    MOE_REQUIRE(c, why == NULL, "%s", why);
    if (pc.rows_q == 0 || pc.seqs == 0) return;
    moe_on_device on(c);
    AttnArgs a = {(const __half *)q16, (const __half *)k16, (const __half *)v16, cu_q, cu_k, (__half *)o16, pc, pc.heads / pc.kv_heads};
    const uint32_t grid = (uint32_t)c->sm_count * 16u;
    if (pc.hd == 128u) moe_run(c, moe_attn_kernel<128>, grid, 128, 0, a);
    else moe_run(c, moe_attn_kernel<64>, grid, 128, 0, a);
    MOE_LAUNCHED(c);
}
