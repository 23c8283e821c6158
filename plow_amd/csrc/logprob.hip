/* logprob.hip — log probabilities of tokens from rows of logits (PLOW_DOP_X_LOGPROB): given tokens, entropy, log of
 * the sum of exponentials, most likely tokens.
 *
 *   d_j = c (x_j - m), m = max_j x_j;  Z = sum_j exp(d_j);  T = sum_j exp(d_j) d_j
 *   logprob_i = d_i - ln Z;  entropy = ln Z - T / Z;  lse = c m + ln Z
 *
 * (the entropy comes from sums over the shifted values: no difference of large numbers). One pass over the logits: a
 * wave walks its part of a row with 4 KB of loads in flight, every lane keeps its own running maximum and both sums
 * (f32, in units of log 2; when the maximum rises by D they become 2^-D Z and 2^-D (T - D Z)), and the wave keeps the
 * best 64 tokens sorted over its lanes. A tile whose largest value lies below the A-th best token found so far, nearly
 * every one after the first few, costs the list one comparison; tokens at or above it go to a buffer of the wave, and
 * 64 of them at a time are sorted and merged into the list. The first tile's bar is the A-th largest of the 64 lanes'
 * own maxima. Tokens are ordered by a 64-bit key (value, lowest id first), so the order in which they are met does not
 * matter.
 *
 * A workgroup's four waves share a row; with few rows a row is split over up to 64 waves, whose results a second
 * launch joins (a lane per part). Sums are joined in a fixed order. */
#include "common.h"
#include "kernels.h"
#include "tuning.h"

#define LP_WAVES 4u
#define LP_NONE 0xFFFFFFFFu
#define LP_MAX_PARTS 64u /* a lane of the joining wave each */
typedef unsigned long long u64;

/* lanes of the wave exchange data through LDS: nothing is emitted, but no read or write moves across it */
__device__ __forceinline__ void lp_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

/* ---- lanes exchanged within the wave, without LDS ---- */
template <int CTRL>
__device__ __forceinline__ uint32_t lp_dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
/* the value of lane ^ O */
template <int O>
__device__ __forceinline__ uint32_t lp_xor(uint32_t v) {
    if (O == 1) return lp_dpp<0xB1>(v);              /* quad_perm 1,0,3,2 */
    if (O == 2) return lp_dpp<0x4E>(v);              /* quad_perm 2,3,0,1 */
    if (O == 4) return lp_dpp<0x1B>(lp_dpp<0x141>(v)); /* row_half_mirror (^ 7), then quad_perm 3,2,1,0 (^ 3) */
    if (O == 8) return lp_dpp<0x128>(v);             /* row_ror 8 */
    if (O == 16) {
        const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false); /* s[0]: even rows' values in both, s[1]: odd rows' */
        return (threadIdx.x & 16u) ? s[0] : s[1];
    }
    const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return (threadIdx.x & 32u) ? s[0] : s[1];
}
template <int O>
__device__ __forceinline__ u64 lp_xor64(u64 v) {
    return ((u64)lp_xor<O>((uint32_t)(v >> 32)) << 32) | lp_xor<O>((uint32_t)v);
}
template <int O>
__device__ __forceinline__ float lp_xorf(float v) { return __uint_as_float(lp_xor<O>(__float_as_uint(v))); }

/* one stage of a bitonic network over the wave: lanes O apart, the larger key to the lower lane where `down` */
template <int O>
__device__ __forceinline__ u64 lp_stage(u64 k, bool down) {
    const u64 o = lp_xor64<O>(k);
    const bool lower = (threadIdx.x & (uint32_t)O) == 0u;
    return (lower == down) == (k > o) ? k : o;
}
template <int O>
__device__ __forceinline__ u64 lp_stages(u64 k, bool down) {
    k = lp_stage<O>(k, down);
    if constexpr (O > 1) k = lp_stages<O / 2>(k, down);
    return k;
}
/* the wave's 64 keys, largest first */
__device__ __forceinline__ u64 lp_sort(u64 k) {
    const uint32_t l = threadIdx.x;
    k = lp_stages<1>(k, (l & 2u) == 0u);
    k = lp_stages<2>(k, (l & 4u) == 0u);
    k = lp_stages<4>(k, (l & 8u) == 0u);
    k = lp_stages<8>(k, (l & 16u) == 0u);
    k = lp_stages<16>(k, (l & 32u) == 0u);
    return lp_stages<32>(k, true);
}
/* the 64 largest of two lists that are sorted largest first, sorted */
__device__ __forceinline__ u64 lp_merge(u64 a, u64 b) {
    b = lp_xor64<32>(b), b = lp_xor64<16>(b), b = lp_xor64<8>(b), b = lp_xor64<4>(b), b = lp_xor64<2>(b), b = lp_xor64<1>(b); /* reversed */
    return lp_stages<32>(a > b ? a : b, true);
}
__device__ __forceinline__ u64 lp_lane(u64 k, uint32_t lane) {
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), (int)lane), lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)k, (int)lane);
    return ((u64)hi << 32) | lo;
}

/* order of the tokens: NaN (either sign) above +inf, -0 and +0 alike, equal values by lowest id; 0 = none (-inf) */
__device__ __forceinline__ u64 lp_key(float x, uint32_t id) {
    if (x == -__builtin_inff()) return 0ull;
    return ((u64)(x != x ? 0xFFFFFFFFu : route_ord(x + 0.0f)) << 32) | (uint32_t)~id;
}
__device__ __forceinline__ float lp_value(u64 key) { /* of a key that is not 0 (NaN: some NaN) */
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float((o & 0x80000000u) ? o & 0x7FFFFFFFu : ~o);
}

/* maximum, Z and T (in units of log 2) of a set of logits */
struct LpSums {
    float m, z, t;
};
/* the sums re-based on a maximum m >= s.m. Clamped where 2^D is 0 anyway: no -inf times 0 (an empty set has m = -inf);
 * a NaN in z stays */
__device__ __forceinline__ void lp_rebase(LpSums& s, float m, float c2) {
    const float D = fmaxf((s.m - m) * c2, -1000.0f), f = __builtin_amdgcn_exp2f(D);
    s.t = f * (s.t + D * s.z), s.z = f * s.z, s.m = m;
}
template <int O>
__device__ __forceinline__ void lp_sums_with(LpSums& s, float c2) {
    LpSums o = {lp_xorf<O>(s.m), lp_xorf<O>(s.z), lp_xorf<O>(s.t)};
    const float m = fmaxf(s.m, o.m);
    lp_rebase(s, m, c2), lp_rebase(o, m, c2);
    s.z += o.z, s.t += o.t;
}
__device__ __forceinline__ void lp_sums_wave(LpSums& s, float c2) {
    lp_sums_with<1>(s, c2), lp_sums_with<2>(s, c2), lp_sums_with<4>(s, c2), lp_sums_with<8>(s, c2), lp_sums_with<16>(s, c2), lp_sums_with<32>(s, c2);
}

/* ---- a wave's walk over vectors [lo, hi) of 16 bytes of a row; vector V / VEC is the row's ragged end ---- */
template <bool F32, bool MASK, bool ALT>
__device__ __forceinline__ void lp_scan(const LogprobRun& r, size_t row, uint32_t lo, uint32_t hi, float c2, u64* buf, LpSums& s, u64& list) {
    constexpr uint32_t VEC = F32 ? 4u : 8u, U = 4u;
    const uint32_t lane = threadIdx.x & 63u, full = r.V / VEC, tail = r.V % VEC;
    const uint8_t* const x = (const uint8_t*)r.logits + row * r.pitch * (F32 ? 4u : 2u);
    const uint8_t* const mk = MASK ? (const uint8_t*)(r.mask + row * r.mask_pitch) : nullptr;
    const float NINF = -__builtin_inff();
    const uint32_t A = ALT ? r.A : 0u;
    s.m = NINF, s.z = 0.0f, s.t = 0.0f;
    list = 0ull;
    u64 bar = 0ull; /* the A-th best of the list: what is not above it cannot be among the A best */
    uint32_t held = 0u; /* keys in the buffer */

    auto flush = [&]() { /* up to 64 of them into the list */
        lp_wave_sync();
        const u64 k = lane < held ? buf[lane] : 0ull, more = lane + 64u < held ? buf[64u + lane] : 0ull;
        list = lp_merge(list, lp_sort(k));
        lp_wave_sync();
        held = held > 64u ? held - 64u : 0u;
        if (lane < held) buf[lane] = more;
        lp_wave_sync();
        const u64 b = lp_lane(list, A - 1u);
        bar = b > bar ? b : bar;
    };

    bool first = true;
    for (uint32_t v0 = lo; v0 < hi; v0 += 64u * U) {
        uint32_t raw[U][4], bits[U];
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            const uint32_t v = v0 + u * 64u + lane;
            bits[u] = v < hi ? (F32 ? 0xFu : 0xFFu) : 0u; /* values of the vector that exist and are allowed */
            if (v < hi && v < full) {
                __builtin_memcpy(raw[u], x + (size_t)v * 16u, 16); /* rows are aligned to an element only */
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 4u; i++) raw[u][i] = 0u;
                if (v < hi) {
                    bits[u] = (1u << tail) - 1u;
                    for (uint32_t i = 0; i < tail; i++) {
                        if (F32) {
                            const uint32_t w = *(const uint32_t*)(x + ((size_t)v * VEC + i) * 4u);
#pragma unroll
                            for (uint32_t j = 0; j < 4u; j++)
                                if (j == i) raw[u][j] = w;
                        } else {
                            const uint32_t w = (uint32_t)*(const uint16_t*)(x + ((size_t)v * VEC + i) * 2u) << (16u * (i & 1u));
#pragma unroll
                            for (uint32_t j = 0; j < 4u; j++)
                                if (j == i / 2u) raw[u][j] |= w;
                        }
                    }
                }
            }
            if (MASK && v < hi) bits[u] &= F32 ? (uint32_t)mk[v >> 1] >> (4u * (v & 1u)) : (uint32_t)mk[v];
        }
        float val[U * VEC];
        const bool some_out = MASK || v0 + 64u * U > (hi < full ? hi : full); /* the same in every lane */
#pragma unroll
        for (uint32_t u = 0; u < U; u++)
#pragma unroll
            for (uint32_t j = 0; j < VEC; j++)
                val[u * VEC + j] = __uint_as_float(F32 ? raw[u][j & 3u] : (j & 1u) ? raw[u][j / 2u] & 0xFFFF0000u : raw[u][j / 2u] << 16);
        if (some_out) {
#pragma unroll
            for (uint32_t u = 0; u < U; u++)
#pragma unroll
                for (uint32_t j = 0; j < VEC; j++)
                    if (!((bits[u] >> j) & 1u)) val[u * VEC + j] = NINF;
        }
        float top = val[0];
#pragma unroll
        for (uint32_t i = 1; i < U * VEC; i++) top = fmaxf(top, val[i]); /* (passes over NaN: Z carries it) */

        lp_rebase(s, fmaxf(s.m, top), c2);
        const float base = s.m == NINF ? 0.0f : s.m;
#pragma unroll
        for (uint32_t i = 0; i < U * VEC; i++) {
            const float d = (val[i] - base) * c2, e = __builtin_amdgcn_exp2f(d);
            s.z += e;
            s.t = fmaf(e, fmaxf(d, -1000.0f), s.t); /* e = 0 there */
        }

        if (ALT) {
            if (first) {
                /* A of this tile's tokens lie at or above the A-th largest of the lanes' own best */
                u64 best = 0ull;
#pragma unroll
                for (uint32_t i = 0; i < U * VEC; i++) {
                    const u64 k = lp_key(val[i], (v0 + (i / VEC) * 64u + lane) * VEC + i % VEC);
                    best = k > best ? k : best;
                }
                const u64 b = lp_lane(lp_sort(best), A - 1u);
                bar = b ? b - 1ull : 0ull;
                first = false;
            }
            const bool near = bar == 0ull || !(top < lp_value(bar)) || s.z != s.z;
            if (__ballot(near && top != NINF) || __ballot(s.z != s.z)) {
#pragma unroll
                for (uint32_t i = 0; i < U * VEC; i++) {
                    const u64 k = lp_key(val[i], (v0 + (i / VEC) * 64u + lane) * VEC + i % VEC);
                    const u64 m = __ballot(k > bar);
                    if (m) {
                        if (k > bar) buf[held + (uint32_t)__popcll(m & ((1ull << lane) - 1ull))] = k;
                        held += (uint32_t)__popcll(m);
                        if (held >= 64u) flush();
                    }
                }
            }
        }
    }
    if (ALT && held) flush();
    lp_sums_wave(s, c2);
}

/* what is written for a row whose sums and (in the wave's lanes) list are whole; by one wave */
template <bool ALT>
__device__ __forceinline__ void lp_write(const LogprobRun& r, size_t row, const LpSums& s, u64 list) {
    const uint32_t lane = threadIdx.x & 63u;
    const float NINF = -__builtin_inff(), LN2 = 0.69314718055994531f;
    const float base = s.m == NINF ? 0.0f : s.m, logz = logf(s.z);
    const bool bad = s.z != s.z;
    auto logp = [&](float x) { return bad ? s.z : x == NINF ? NINF : (x - base) * r.scale - logz; };
    if (lane == 0u) {
        if (r.entropy) r.entropy[row] = s.z == 0.0f ? 0.0f : logz - s.t * LN2 / s.z;
        if (r.lse) r.lse[row] = bad ? s.z : base * r.scale + logz;
    }
    for (uint32_t j = lane; j < r.n; j += WAVE) {
        const uint32_t id = r.ids[row * r.n + j];
        float v = 0.0f; /* asks for nothing */
        if (id != LP_NONE) {
            v = __builtin_nanf("");
            if (id < r.V) {
                const bool ok = !r.mask || ((r.mask[row * r.mask_pitch + (id >> 5)] >> (id & 31u)) & 1u);
                v = logp(!ok ? NINF : r.f32 ? ((const float*)r.logits)[row * r.pitch + id] : bf2f(((const bf16_t*)r.logits)[row * r.pitch + id]));
            }
        }
        r.logprob[row * r.n + j] = v;
    }
    if (ALT && lane < r.A) {
        if (r.alt_ids) r.alt_ids[row * r.A + lane] = list ? ~(uint32_t)list : LP_NONE;
        if (r.alt_logprob) r.alt_logprob[row * r.A + lane] = logp(list ? lp_value(list) : NINF);
    }
}

struct LpParts { /* rows split over parts: their sums and lists in scratch */
    uint32_t n;    /* parts per row, 0 = a workgroup per row */
    LpSums* sums;  /* [T][n] */
    u64* lists;    /* [T][n][A] */
};

template <bool F32, bool MASK, bool ALT>
__global__ __launch_bounds__(LP_WAVES* WAVE) void k_logprob(LogprobRun r, LpParts p, float c2) {
    __shared__ u64 buf[LP_WAVES][ALT ? 128 : 1];
    __shared__ LpSums part[LP_WAVES];
    const uint32_t lane = threadIdx.x & 63u, wv = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    constexpr uint32_t VEC = F32 ? 4u : 8u;
    const uint64_t nv = (r.V + VEC - 1u) / VEC;
    const uint32_t per_row = p.n ? p.n / LP_WAVES : 1u, parts = per_row * LP_WAVES;
    const size_t row = blockIdx.x / per_row;
    const uint32_t at = (uint32_t)(blockIdx.x % per_row) * LP_WAVES + wv;
    LpSums s;
    u64 list;
    lp_scan<F32, MASK, ALT>(r, row, (uint32_t)(nv * at / parts), (uint32_t)(nv * (at + 1u) / parts), c2, buf[wv], s, list);
    if (p.n) {
        if (lane == 0u) p.sums[row * p.n + at] = s;
        if (ALT && lane < r.A) p.lists[(row * p.n + at) * r.A + lane] = list;
        return;
    }
    if (lane == 0u) part[wv] = s;
    if (ALT) buf[wv][lane] = list;
    __syncthreads();
    if (wv) return;
#pragma unroll
    for (uint32_t w = 1; w < LP_WAVES; w++) {
        LpSums o = part[w];
        const float m = fmaxf(s.m, o.m);
        lp_rebase(s, m, c2), lp_rebase(o, m, c2);
        s.z += o.z, s.t += o.t;
        if (ALT) list = lp_merge(list, buf[w][lane]);
    }
    lp_write<ALT>(r, row, s, list);
}

/* a wave per row: a lane per part */
template <bool ALT>
__global__ __launch_bounds__(WAVE) void k_logprob_join(LogprobRun r, LpParts p, float c2) {
    __shared__ u64 buf[128];
    const uint32_t lane = threadIdx.x;
    const size_t row = blockIdx.x;
    const bool mine = lane < p.n;
    LpSums s = {-__builtin_inff(), 0.0f, 0.0f};
    if (mine) s = p.sums[row * p.n + lane];
    u64 list = 0ull;
    if (ALT) {
        const u64* const l = p.lists + (row * p.n + (mine ? lane : 0u)) * r.A;
        /* A tokens lie at or above the A-th largest of the parts' own best */
        u64 k = mine ? l[0] : 0ull;
        u64 bar = lp_lane(lp_sort(k), r.A - 1u);
        bar = bar ? bar - 1ull : 0ull;
        uint32_t held = 0u;
        for (uint32_t j = 0;;) {
            const u64 m = __ballot(k > bar);
            if (!m) break; /* the lists fall: nothing further on is above the bar either */
            if (k > bar) buf[held + (uint32_t)__popcll(m & ((1ull << lane) - 1ull))] = k;
            held += (uint32_t)__popcll(m);
            j++;
            const u64 next = mine && j < r.A && k > bar ? l[j] : 0ull;
            const bool last = __ballot(next > bar) == 0ull;
            while (held >= 64u || (last && held)) {
                lp_wave_sync();
                const u64 c = lane < held ? buf[lane] : 0ull, more = lane + 64u < held ? buf[64u + lane] : 0ull;
                list = lp_merge(list, lp_sort(c));
                lp_wave_sync();
                held = held > 64u ? held - 64u : 0u;
                if (lane < held) buf[lane] = more;
                const u64 b = lp_lane(list, r.A - 1u);
                bar = b > bar ? b : bar;
            }
            k = next;
        }
    }
    lp_sums_wave(s, c2);
    lp_write<ALT>(r, row, s, list);
}

template <bool F32, bool MASK>
static void lp_launch(const LogprobRun& r, const LpParts& p, uint32_t grid, float c2, hipStream_t st) {
    if (r.A) k_logprob<F32, MASK, true><<<grid, LP_WAVES * WAVE, 0, st>>>(r, p, c2);
    else k_logprob<F32, MASK, false><<<grid, LP_WAVES * WAVE, 0, st>>>(r, p, c2);
}

int launch_logprob(const LogprobRun& r, hipStream_t st) {
    const uint32_t n_cu = plow_moe_n_cu();
    if (!n_cu) return PLOW_MOE_EDEVICE;
    /* few rows: as many workgroups per row as give every CU four, up to LP_MAX_PARTS waves of a whole tile each */
    const uint32_t tile = (r.f32 ? 4u : 8u) * 256u * LP_WAVES;
    uint32_t wgs = r.T < 4u * n_cu ? (4u * n_cu + r.T - 1u) / r.T : 1u;
    const uint32_t most = r.V / tile < LP_MAX_PARTS / LP_WAVES ? r.V / tile : LP_MAX_PARTS / LP_WAVES;
    if (wgs > most) wgs = most;
    LpParts p = {};
    const float c2 = r.scale * 1.44269504088896341f; /* log2(e) */
    if (wgs >= 2u && r.ws) {
        const uint32_t n = wgs * LP_WAVES;
        const size_t lists = (size_t)r.T * n * r.A * 8u, sums = (size_t)r.T * n * sizeof(LpSums);
        if (lists + sums <= r.ws_bytes) p.n = n, p.lists = (u64*)r.ws, p.sums = (LpSums*)((uint8_t*)r.ws + lists);
    }
    const uint64_t grid = (uint64_t)r.T * (p.n ? p.n / LP_WAVES : 1u);
    if (grid > 0x7FFFFFFFull) return PLOW_MOE_EINVAL;
    if (r.f32) {
        if (r.mask) lp_launch<true, true>(r, p, (uint32_t)grid, c2, st);
        else lp_launch<true, false>(r, p, (uint32_t)grid, c2, st);
    } else {
        if (r.mask) lp_launch<false, true>(r, p, (uint32_t)grid, c2, st);
        else lp_launch<false, false>(r, p, (uint32_t)grid, c2, st);
    }
    if (p.n) {
        if (r.A) k_logprob_join<true><<<r.T, WAVE, 0, st>>>(r, p, c2);
        else k_logprob_join<false><<<r.T, WAVE, 0, st>>>(r, p, c2);
    }
    return 0;
}
