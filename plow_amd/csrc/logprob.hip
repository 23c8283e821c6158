/* logprob.hip — log probabilities of tokens from rows of logits (PLOW_DOP_X_LOGPROB): given tokens, entropy, log of
 * the sum of exponentials, most likely tokens.
 *
 *   d_j = c (x_j - m), m = max_j x_j;  Z = sum_j exp(d_j);  T = sum_j exp(d_j) d_j
 *   logprob_i = d_i - ln Z;  entropy = ln Z - T / Z;  lse = c m + ln Z
 *
 * (the entropy comes from sums over the shifted values: no difference of large numbers). One pass over the logits: a
 * wave walks its part of a row, the next 4 KB of loads under this tile's arithmetic; every lane keeps its own running
 * maximum and both sums (f32, in units of log 2; when the maximum rises by D they become 2^-D Z and 2^-D (T - D Z)).
 *
 * The best A tokens: A of the row's tokens lie at or above the A-th largest of the lanes' running maxima, so what lies
 * below that bar needs no further look: a comparison per tile. Tokens at or above it go, unsorted, to a buffer of the
 * wave in LDS, a few dozen in all; the waves of a workgroup share the highest bar. The survivors of a row are sorted
 * once, by 64-bit keys (value, lowest id first), so the order in which they are met does not matter. (With a sorted
 * list per wave, 64 tokens merged at a time, one row of 120001 with 20 alternatives took 16.0 us for 12.9, 64 masked
 * rows of 32000 with 5 took 18.4 for 14.8.)
 * Where many tokens tie at the bar the buffer is sorted and merged into such a list after all, whose A-th key is an
 * exact bar.
 *
 * A workgroup's four waves share a row; with few rows a row is split over up to 64 waves, whose results a second
 * launch joins. Sums are joined in a fixed order.
 *
 * 2048 rows of 120001 bf16 without alternatives take 108 us = 4.5 TB/s, the rate of a large copy; vector instructions fill
 * 67 % of their issue slots, an exponential counted as one though it takes four. One row of 120001 f32
 * with 20 alternatives takes 13 us, 64 masked rows of 32000 with 5 15 us: two launches, 8 and 5 us, of which the bytes
 * are 1 us. */
#include "common.h"
#include "kernels.h"
#include "tuning.h"

#define LP_WAVES 4u
#define LP_NONE 0xFFFFFFFFu
#define LP_MAX_PARTS 64u /* a lane of a joining wave each */
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

#define LP_BUF 256u  /* keys a wave's buffer holds */
#define LP_KEEP 80u  /* LDS bytes of a lane's tile, 64 of them used: lanes on different banks */
#define LP_LIST 64u  /* keys a part of a split row hands on, at least PLOW_LOGPROB_MAX_ALT */

__device__ __forceinline__ uint32_t lp_ord(float x) { return route_ord(x); }
__device__ __forceinline__ float lp_unord(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? o & 0x7FFFFFFFu : ~o); }
/* a lower bound of the A-th largest of the wave's 64 values (its upper 16 bits are that value's; -inf: no bound). The
 * values are ordered as unsigned numbers, whose bits are found from the top */
__device__ __forceinline__ float lp_ath(float v, uint32_t A) {
    const uint32_t k = lp_ord(v);
    uint32_t t = 0u;
#pragma unroll
    for (int b = 31; b >= 16; b--) {
        const uint32_t c = t | (1u << b);
        t = (uint32_t)__popcll(__ballot(k >= c)) >= A ? c : t;
    }
    return t <= 0x007FFFFFu ? -__builtin_inff() : lp_unord(t);
}

/* The best A tokens met so far, in one wave: a buffer of tokens none of which need be among them, and, once that has
 * run over, a list sorted over the lanes whose A-th key is `bar`. bar_v: no token with a smaller value counts. */
struct LpBest {
    u64 list, bar;
    float bar_v;
    uint32_t held, A;
    u64* buf;
    __device__ __forceinline__ void init(uint32_t a, u64* b) { list = 0ull, bar = 0ull, bar_v = -__builtin_inff(), held = 0u, A = a, buf = b; }
    __device__ __forceinline__ void raise(float v) { bar_v = v > bar_v ? v : bar_v; }
    /* the lanes' keys that `take` names (the buffer has room for 64) */
    __device__ __forceinline__ void push(u64 k, bool take) {
        const u64 m = __ballot(take);
        if (take) buf[held + __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u))] = k;
        held += (uint32_t)__popcll(m);
    }
    __device__ __forceinline__ void prune() { /* what the bar has left behind since leaves the buffer */
        const uint32_t lane = threadIdx.x & 63u, n = held;
        u64 k[LP_BUF / 64u];
        lp_wave_sync();
#pragma unroll
        for (uint32_t r = 0; r < LP_BUF / 64u; r++) k[r] = r * 64u + lane < n ? buf[r * 64u + lane] : 0ull;
        lp_wave_sync();
        held = 0u;
#pragma unroll
        for (uint32_t r = 0; r < LP_BUF / 64u; r++) push(k[r], k[r] > bar && !(lp_value(k[r]) < bar_v));
        lp_wave_sync();
    }
    __device__ __forceinline__ void sort_in() { /* the whole buffer into the list */
        const uint32_t lane = threadIdx.x & 63u;
        lp_wave_sync();
        for (uint32_t at = 0; at < held; at += 64u) {
            const u64 k = lp_sort(at + lane < held ? buf[at + lane] : 0ull);
            list = lp_lane(list, 0u) == 0ull ? k : lp_merge(list, k); /* (the first 64 are the list) */
        }
        lp_wave_sync();
        held = 0u;
        bar = lp_lane(list, A - 1u);
        if (bar) raise(lp_value(bar));
    }
};

/* One tile of N values per lane into the sums and the best tokens. id0, id_at(i): the tile's lowest id and the id of
 * this lane's value i; stash() keeps the lane's values where
 * value_at(i), i not a constant, finds them; wg_bar: the workgroup's bar, as lp_ord. */
template <int N, bool ALT, class IdAt, class Stash, class ValueAt>
__device__ __forceinline__ void lp_tile(const float (&val)[N], LpSums& s, LpBest& best, uint32_t* wg_bar, float c2, uint32_t id0, IdAt id_at, Stash stash, ValueAt value_at) {
    const float NINF = -__builtin_inff();
    float top = val[0];
#pragma unroll
    for (int i = 1; i < N; i++) top = fmaxf(top, val[i]); /* (passes over NaN: Z carries it) */
    lp_rebase(s, fmaxf(s.m, top), c2);
    const float base = s.m == NINF ? 0.0f : s.m;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float d = (val[i] - base) * c2, e = __builtin_amdgcn_exp2f(d);
        s.z += e;
        s.t = fmaf(e, fmaxf(d, -1000.0f), s.t); /* e = 0 there */
    }
    if (!ALT) return;

    best.raise(lp_unord(*(volatile uint32_t*)wg_bar));
    if (!__ballot(!(top < best.bar_v) || s.z != s.z)) return;
    const float own = lp_ath(s.m, best.A);
    if (own > best.bar_v) {
        best.raise(own);
        if ((threadIdx.x & 63u) == 0u) atomicMax(wg_bar, lp_ord(own));
    }
    /* above the bar, or at it unless all that still come at it have higher ids than an exact bar's; NaN is always in */
    const bool past = best.bar_v == NINF || (best.bar != 0ull && lp_value(best.bar) == best.bar_v && ~(uint32_t)best.bar < id0);
    const float bar = best.bar_v;
    uint32_t mine = 0u;
#pragma unroll
    for (int i = 0; i < N; i++) mine |= (past ? !(val[i] <= bar) : !(val[i] < bar)) ? 1u << i : 0u;
    /* One of each lane's at a time: most lanes have none, few have two. A register cannot be named by a number, so the
     * lanes that have any put theirs into LDS first (read again from memory, which is busy, each turn waits for it). */
    if (mine) stash();
    while (__ballot(mine != 0u)) {
        const uint32_t i = mine ? (uint32_t)__ffs((int)mine) - 1u : 0u;
        const u64 k = mine ? lp_key(value_at(i), id_at(i)) : 0ull;
        mine &= mine - 1u;
        if (best.held > LP_BUF - 64u) {
            best.prune();
            if (best.held > LP_BUF - 64u) best.sort_in(); /* ties at the bar, a row that rises */
        }
        best.push(k, k > best.bar);
    }
}

/* ---- a wave's walk over the vectors [lo, hi) of 16 bytes of a row, and with `tail` the values behind its last one ---- */
template <bool F32, bool MASK, bool ALT>
__device__ __forceinline__ void lp_scan(const LogprobRun& r, size_t row, uint32_t lo, uint32_t hi, bool tail, float c2, uint32_t* wg_bar, uint8_t* keep, LpSums& s, LpBest& best) {
    constexpr uint32_t VEC = F32 ? 4u : 8u, U = 4u, N = U * VEC;
    const uint32_t lane = threadIdx.x & 63u;
    const uint8_t* const x = (const uint8_t*)r.logits + row * r.pitch * (F32 ? 4u : 2u);
    const uint32_t* const mw = MASK ? r.mask + row * r.mask_pitch : nullptr;
    const uint8_t* const mk = (const uint8_t*)mw;
    const float NINF = -__builtin_inff();
    s.m = NINF, s.z = 0.0f, s.t = 0.0f;
    auto value = [&](uint32_t id) { /* one logit, as the mask leaves it */
        if (MASK && !((mw[id >> 5] >> (id & 31u)) & 1u)) return NINF;
        return F32 ? *(const float*)(x + (size_t)id * 4u) : bf2f(*(const bf16_t*)(x + (size_t)id * 2u));
    };

    /* The next tile's loads go out ahead of this one's arithmetic, none of them under a condition: a vector past the
     * end is the last one again and counts as -inf. */
    uint32_t raw[2][U][4];
    uint8_t bits[2][U];
    auto load = [&](uint32_t b, uint32_t v0) {
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            uint32_t v = v0 + u * 64u + lane;
            v = v < hi ? v : hi - 1u;
            __builtin_memcpy(raw[b][u], x + (size_t)v * 16u, 16); /* rows are aligned to an element only */
            if (MASK) bits[b][u] = F32 ? mk[v >> 1] : mk[v];
        }
    };
    auto tile = [&](uint32_t b, uint32_t v0) {
        float val[N];
#pragma unroll
        for (uint32_t u = 0; u < U; u++)
#pragma unroll
            for (uint32_t j = 0; j < VEC; j++)
                val[u * VEC + j] = __uint_as_float(F32 ? raw[b][u][j & 3u] : (j & 1u) ? raw[b][u][j / 2u] & 0xFFFF0000u : raw[b][u][j / 2u] << 16);
        if (MASK || v0 + 64u * U > hi) { /* the same in every lane */
#pragma unroll
            for (uint32_t u = 0; u < U; u++) {
                const uint32_t v = v0 + u * 64u + lane;
                const uint32_t ok = v >= hi ? 0u : !MASK ? 0xFFu : F32 ? (uint32_t)bits[b][u] >> (4u * (v & 1u)) : (uint32_t)bits[b][u];
#pragma unroll
                for (uint32_t j = 0; j < VEC; j++)
                    if (!((ok >> j) & 1u)) val[u * VEC + j] = NINF;
            }
        }
        auto id_at = [&](uint32_t i) { return (v0 + (i / VEC) * 64u + lane) * VEC + i % VEC; };
        uint8_t* const kept = ALT ? keep + lane * LP_KEEP : nullptr; /* this lane's 64 bytes */
        lp_tile<(int)N, ALT>(val, s, best, wg_bar, c2, v0 * VEC, id_at,
                             [&]() {
#pragma unroll
                                 for (uint32_t u = 0; u < U; u++) __builtin_memcpy(__builtin_assume_aligned(kept + u * 16u, 16), raw[b][u], 16);
                             },
                             [&](uint32_t i) { return F32 ? *(const float*)(kept + i * 4u) : bf2f(*(const bf16_t*)(kept + i * 2u)); });
    };
    if (lo < hi) {
        load(0u, lo);
        for (uint32_t v0 = lo;;) {
            load(1u, v0 + 64u * U);
            tile(0u, v0);
            if ((v0 += 64u * U) >= hi) break;
            load(0u, v0 + 64u * U);
            tile(1u, v0);
            if ((v0 += 64u * U) >= hi) break;
        }
    }
    if (tail) {
        const uint32_t id0 = r.V / VEC * VEC, id = id0 + lane;
        float val[1] = {id < r.V ? value(id) : NINF};
        lp_tile<1, ALT>(val, s, best, wg_bar, c2, id0, [&](uint32_t) { return id; }, []() {}, [&](uint32_t) { return val[0]; });
    }
    if (ALT) {
        best.raise(lp_unord(*(volatile uint32_t*)wg_bar));
        best.prune();
        if (lp_lane(best.list, 0u) != 0ull) best.sort_in();
    }
    lp_sums_wave(s, c2);
}

/* what is written for a row whose sums and (in the wave's lanes) list are whole; by one wave */
template <bool ALT>
__device__ __forceinline__ void lp_write(const LogprobRun& r, size_t row, const LpSums& s, u64 list) {
    const uint32_t lane = threadIdx.x & 63u;
    const float NINF = -__builtin_inff(), LN2 = 0.69314718055994531f;
    const float base = s.m == NINF ? 0.0f : s.m, logz = logf(s.z);
    const bool bad = s.z != s.z;
    /* halves: the difference of two finite logits may be past the largest f32 where c times it is not */
    auto logp = [&](float x) { return bad ? s.z : x == NINF ? NINF : (0.5f * x - 0.5f * base) * (2.0f * r.scale) - logz; };
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

/* rows split over parts: what each hands on, in scratch */
struct LpPart {
    LpSums sums;
    uint32_t n; /* keys of its list */
    float bar;  /* A tokens of the row lie at or above it */
};
struct LpParts {
    uint32_t n;     /* parts per row, 0 = a workgroup per row */
    LpPart* part;   /* [T][n] */
    u64* lists;     /* [T][n][LP_LIST] */
};

template <bool F32, bool MASK, bool ALT>
__global__ __launch_bounds__(LP_WAVES* WAVE) void k_logprob(LogprobRun r, LpParts p, float c2) {
    __shared__ u64 buf[LP_WAVES][ALT ? LP_BUF : 1u];
    __shared__ u64 last[ALT ? LP_BUF : 1u];
    __shared__ __attribute__((aligned(16))) uint8_t keep[LP_WAVES][ALT ? WAVE * LP_KEEP : 1u];
    __shared__ LpPart part[LP_WAVES];
    __shared__ uint32_t wg_bar;
    const uint32_t lane = threadIdx.x & 63u, wv = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    constexpr uint32_t VEC = F32 ? 4u : 8u;
    const uint64_t nv = r.V / VEC;
    const uint32_t per_row = p.n ? p.n / LP_WAVES : 1u, parts = per_row * LP_WAVES;
    const size_t row = blockIdx.x / per_row;
    const uint32_t at = (uint32_t)(blockIdx.x % per_row) * LP_WAVES + wv;
    LpSums s;
    LpBest best;
    if (ALT) {
        if (threadIdx.x == 0u) wg_bar = lp_ord(-__builtin_inff());
        __syncthreads();
        best.init(r.A, buf[wv]);
    }
    lp_scan<F32, MASK, ALT>(r, row, (uint32_t)(nv * at / parts), (uint32_t)(nv * (at + 1u) / parts), r.V % VEC != 0u && at == parts - 1u, c2, &wg_bar, ALT ? &keep[wv][0] : nullptr, s, best);
    if (ALT && best.held > (p.n ? LP_LIST : LP_BUF - 64u)) best.sort_in();
    const bool sorted = ALT && lp_lane(best.list, 0u) != 0ull; /* then the buffer is empty */
    const uint32_t n = !ALT ? 0u : sorted ? (uint32_t)__popcll(__ballot(best.list != 0ull)) : best.held;
    if (p.n) {
        if (lane == 0u) p.part[row * p.n + at] = {s, n, ALT ? best.bar_v : 0.0f};
        if (ALT && lane < n) p.lists[(row * p.n + at) * LP_LIST + lane] = sorted ? best.list : buf[wv][lane];
        return;
    }
    if (ALT && sorted) buf[wv][lane] = best.list;
    if (lane == 0u) part[wv] = {s, n, 0.0f};
    __syncthreads();
    if (wv) return;
    LpBest all;
    if (ALT) {
        all.init(r.A, last);
        all.raise(lp_unord(wg_bar));
    }
#pragma unroll 1
    for (uint32_t w = 0; w < LP_WAVES; w++) {
        if (w) {
            LpSums o = part[w].sums;
            const float m = fmaxf(s.m, o.m);
            lp_rebase(s, m, c2), lp_rebase(o, m, c2);
            s.z += o.z, s.t += o.t;
        }
        if (ALT)
            for (uint32_t j = 0; j < part[w].n; j += 64u) {
                const u64 k = j + lane < part[w].n ? buf[w][j + lane] : 0ull;
                if (all.held > LP_BUF - 64u) all.sort_in();
                all.push(k, k > all.bar && !(lp_value(k) < all.bar_v));
            }
    }
    if (ALT) all.sort_in();
    lp_write<ALT>(r, row, s, ALT ? all.list : 0ull);
}

/* a workgroup per row: 8 waves fetch the parts' lists, all of them on their way at once, and keep what lies at or above
 * the A-th largest of the parts' maxima and above every part's own bar; one wave sorts that */
#define LP_JOIN_WAVES 8u
template <bool ALT>
__global__ __launch_bounds__(ALT ? LP_JOIN_WAVES * WAVE : WAVE) void k_logprob_join(LogprobRun r, LpParts p, float c2) {
    __shared__ u64 kept[ALT ? LP_MAX_PARTS * LP_LIST : 1u];
    __shared__ u64 buf[ALT ? LP_BUF : 1u];
    __shared__ uint32_t n_kept;
    const uint32_t lane = threadIdx.x & 63u, wv = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const size_t row = blockIdx.x;
    u64 k[LP_MAX_PARTS / LP_JOIN_WAVES];
    if (ALT) {
        if (threadIdx.x == 0u) n_kept = 0u;
#pragma unroll
        for (uint32_t j = 0; j < LP_MAX_PARTS / LP_JOIN_WAVES; j++) { /* (what lies behind a list's end is not used) */
            const uint32_t q = j * LP_JOIN_WAVES + wv;
            k[j] = p.lists[(row * p.n + (q < p.n ? q : 0u)) * LP_LIST + lane];
        }
    }
    LpPart mine = {{-__builtin_inff(), 0.0f, 0.0f}, 0u, -__builtin_inff()};
    if (lane < p.n) mine = p.part[row * p.n + lane];
    LpSums s = mine.sums;
    float bar = -__builtin_inff();
    if (ALT) {
        bar = mine.bar;
        bar = fmaxf(bar, lp_xorf<1>(bar)), bar = fmaxf(bar, lp_xorf<2>(bar)), bar = fmaxf(bar, lp_xorf<4>(bar));
        bar = fmaxf(bar, lp_xorf<8>(bar)), bar = fmaxf(bar, lp_xorf<16>(bar)), bar = fmaxf(bar, lp_xorf<32>(bar));
        bar = fmaxf(bar, lp_ath(s.m, r.A));
        __syncthreads();
#pragma unroll
        for (uint32_t j = 0; j < LP_MAX_PARTS / LP_JOIN_WAVES; j++) {
            const uint32_t q = j * LP_JOIN_WAVES + wv;
            if (q >= p.n) continue; /* the same in every lane */
            const bool take = lane < (uint32_t)__builtin_amdgcn_readlane((int)mine.n, (int)q) && !(lp_value(k[j]) < bar);
            const u64 m = __ballot(take);
            if (!m) continue;
            uint32_t at = 0u;
            if (lane == 0u) at = atomicAdd(&n_kept, (uint32_t)__popcll(m));
            at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
            if (take) kept[at + __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u))] = k[j];
        }
        __syncthreads();
    }
    if (wv) return;
    LpBest all;
    if (ALT) {
        all.init(r.A, buf);
        const uint32_t n = n_kept;
        for (uint32_t j = 0; j < n; j += 64u) {
            const u64 c = j + lane < n ? kept[j + lane] : 0ull;
            if (all.held > LP_BUF - 64u) all.sort_in();
            all.push(c, c > all.bar);
        }
        all.sort_in();
    }
    lp_sums_wave(s, c2);
    lp_write<ALT>(r, row, s, ALT ? all.list : 0ull);
}

template <bool F32, bool MASK>
static void lp_launch(const LogprobRun& r, const LpParts& p, uint32_t grid, float c2, hipStream_t st) {
    if (r.A) k_logprob<F32, MASK, true><<<grid, LP_WAVES * WAVE, 0, st>>>(r, p, c2);
    else k_logprob<F32, MASK, false><<<grid, LP_WAVES * WAVE, 0, st>>>(r, p, c2);
}

int launch_logprob(const LogprobRun& r, hipStream_t st) {
    const uint32_t n_cu = plow_moe_n_cu();
    if (!n_cu) return PLOW_MOE_EDEVICE;
    /* few rows: as many workgroups per row as give every CU two, up to LP_MAX_PARTS waves of a whole tile each. Rows of
     * 120001 with a workgroup per row / so / with four per CU: 1 row f32 A = 20 34 / 13 / 13 us, 64 rows bf16 A = 5 41 /
     * 18 / 24, 300 rows 46 / 41 / 42, 600 rows 57 / 58 / 68 (each part hands on candidates of its own). */
    const uint32_t tile = (r.f32 ? 4u : 8u) * 256u * LP_WAVES;
    uint32_t wgs = r.T < 2u * n_cu ? (2u * n_cu + r.T - 1u) / r.T : 1u;
    const uint32_t most = r.V / tile < LP_MAX_PARTS / LP_WAVES ? r.V / tile : LP_MAX_PARTS / LP_WAVES;
    if (wgs > most) wgs = most;
    LpParts p = {};
    const float c2 = r.scale * 1.44269504088896341f; /* log2(e) */
    if (wgs >= 2u && r.ws) {
        const uint32_t n = wgs * LP_WAVES;
        const size_t lists = r.A ? (size_t)r.T * n * LP_LIST * 8u : 0u, parts = (size_t)r.T * n * sizeof(LpPart);
        if (lists + parts <= r.ws_bytes) p.n = n, p.lists = (u64*)r.ws, p.part = (LpPart*)((uint8_t*)r.ws + lists);
    }
    const uint64_t grid = (uint64_t)r.T * (p.n ? p.n / LP_WAVES : 1u);
    if (grid >= (1ull << 24)) return PLOW_MOE_EINVAL; /* (256 threads each in 32 bits) */
    if (r.f32) {
        if (r.mask) lp_launch<true, true>(r, p, (uint32_t)grid, c2, st);
        else lp_launch<true, false>(r, p, (uint32_t)grid, c2, st);
    } else {
        if (r.mask) lp_launch<false, true>(r, p, (uint32_t)grid, c2, st);
        else lp_launch<false, false>(r, p, (uint32_t)grid, c2, st);
    }
    if (p.n) {
        if (r.A) k_logprob_join<true><<<r.T, LP_JOIN_WAVES * WAVE, 0, st>>>(r, p, c2);
        else k_logprob_join<false><<<r.T, WAVE, 0, st>>>(r, p, c2);
    }
    return 0;
}
