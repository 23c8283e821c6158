/* logprob.hip — log probabilities of tokens from rows of logits (PLOW_DOP_X_LOGPROB): given tokens, entropy, log of
 * the sum of exponentials, most likely tokens.
 *
 *   d_j = c (x_j - m), m = max_j x_j;  Z = sum_j exp(d_j);  T = sum_j exp(d_j) d_j
 *   logprob_i = d_i - ln Z;  entropy = ln Z - T / Z;  lse = c m + ln Z
 *
 * (the entropy is taken from sums over the shifted values: no difference of large numbers). */
#include "common.h"
#include "kernels.h"

#define LP_THREADS 256u
#define LP_NONE 0xFFFFFFFFu

__device__ __forceinline__ float lp_at(const LogprobRun& r, size_t row, uint32_t i) {
    if (r.mask && !((r.mask[row * r.mask_pitch + (i >> 5)] >> (i & 31u)) & 1u)) return -__builtin_inff();
    return r.f32 ? ((const float*)r.logits)[row * r.pitch + i] : bf2f(((const bf16_t*)r.logits)[row * r.pitch + i]);
}
/* order of alternatives: a larger key first; NaN (either sign) above +inf, -0 and +0 alike */
__device__ __forceinline__ uint32_t lp_key(float x) { return x != x ? 0xFFFFFFFFu : route_ord(x + 0.0f); }

__device__ __forceinline__ float lp_block_sum(float v, float* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0u) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}
__device__ __forceinline__ unsigned long long lp_block_max(unsigned long long v, unsigned long long* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const unsigned long long u = __shfl_xor(v, o, 64);
        v = u > v ? u : v;
    }
    __syncthreads();
    if ((threadIdx.x & 63u) == 0u) red[threadIdx.x >> 6] = v;
    __syncthreads();
    unsigned long long m = red[0];
    for (int w = 1; w < 4; w++) m = red[w] > m ? red[w] : m;
    return m;
}

/* a workgroup per row: one pass for the maximum, one for the sums, one for each alternative */
__global__ __launch_bounds__(LP_THREADS) void k_logprob_plain(LogprobRun r) {
    __shared__ float red[4];
    __shared__ unsigned long long red64[4];
    const float NINF = -__builtin_inff();
    for (size_t row = blockIdx.x; row < r.T; row += gridDim.x) {
        float m = NINF;
        for (uint32_t i = threadIdx.x; i < r.V; i += LP_THREADS) m = fmaxf(m, lp_at(r, row, i));
        /* (fmaxf passes over NaN: the sums below carry it) */
        const unsigned long long mk = lp_block_max(route_ord(m), red64);
        const uint32_t mo = (uint32_t)mk;
        m = __uint_as_float((mo & 0x80000000u) ? mo & 0x7FFFFFFFu : ~mo);
        const float base = m == NINF ? 0.0f : m;
        float z = 0.0f, t = 0.0f;
        for (uint32_t i = threadIdx.x; i < r.V; i += LP_THREADS) {
            const float x = lp_at(r, row, i);
            if (x == NINF) continue;
            const float d = (x - base) * r.scale, e = expf(d);
            z += e;
            t = fmaf(e, fmaxf(d, -1000.0f), t); /* e = 0 there; -inf times 0 would not be */
        }
        z = lp_block_sum(z, red);
        t = lp_block_sum(t, red);
        const float logz = logf(z);
        auto logp = [&](float x) { return x == NINF ? (z != z ? z : NINF) : (x - base) * r.scale - logz; };
        if (threadIdx.x == 0) {
            if (r.entropy) r.entropy[row] = z == 0.0f ? 0.0f : logz - t / z;
            if (r.lse) r.lse[row] = base * r.scale + logz;
        }
        for (uint32_t j = threadIdx.x; j < r.n; j += LP_THREADS) {
            const uint32_t id = r.ids[row * r.n + j];
            r.logprob[row * r.n + j] = id == LP_NONE ? 0.0f : id >= r.V ? __builtin_nanf("") : logp(lp_at(r, row, id));
        }
        unsigned long long prev = ~0ull;
        for (uint32_t a = 0; a < r.A; a++) {
            unsigned long long best = 0ull; /* key, then the lowest id */
            for (uint32_t i = threadIdx.x; i < r.V; i += LP_THREADS) {
                const float x = lp_at(r, row, i);
                if (x == NINF) continue;
                const unsigned long long k = ((unsigned long long)lp_key(x) << 32) | (uint32_t)~i;
                if (k < prev && k > best) best = k;
            }
            best = lp_block_max(best, red64);
            if (threadIdx.x == 0) {
                const uint32_t id = best ? ~(uint32_t)best : LP_NONE;
                if (r.alt_ids) r.alt_ids[row * r.A + a] = id;
                if (r.alt_logprob) r.alt_logprob[row * r.A + a] = best ? logp(lp_at(r, row, id)) : (z != z ? z : NINF);
            }
            prev = best ? best : 0ull;
        }
        __syncthreads();
    }
}

int launch_logprob(const LogprobRun& r, hipStream_t st) {
    k_logprob_plain<<<r.T < (1u << 20) ? r.T : (1u << 20), LP_THREADS, 0, st>>>(r);
    return 0;
}
