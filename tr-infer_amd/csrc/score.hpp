// Routing by scores, one row by a wave (trk_route_scores, trk_moe_mx4): sigmoid or softmax scores, a bias that moves the choice
// but not the weights, groups, top-k, renormalised weights.
//
// A row is 4 E bytes and some ten operations a logit; what bounds the kernel is the chain of steps of a row (scores,
// groups, selection) with few waves, and their instructions with many.  So keys are compared in 32 bits with a bound
// on what 32 bits get wrong.  Where two group sums or keys that decide something are nearer than that (some rows in a
// thousand), the sums, or the few keys in question, are taken in 64 bits; a row with more than 64 keys in question (many
// equal ones) is done in 64 bits from the start.
#pragma once

#include "route.hpp"

namespace trk {

// the larger key, the lower index among equal ones; an index of ~0 is no candidate
__device__ __forceinline__ bool better(double ka, uint32_t ia, double kb, uint32_t ib) {
    return ka > kb || (ka == kb && ia < ib);
}

__device__ __forceinline__ void wave_best(double& k, uint32_t& i) {
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const double ko = __shfl_xor(k, d);
        const uint32_t io = __shfl_xor(i, d);
        if (better(ko, io, k, i)) k = ko, i = io;
    }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// Every key in 64 bits, the best ones by k rounds over the wave.  `key`: E doubles of LDS.
static __device__ void score_row(const float* __restrict__ lg, const float* __restrict__ bias, uint32_t E, const ScorePolicy& p,
                          uint32_t lane, double* key, uint32_t* __restrict__ ids, float* __restrict__ w,
                          uint32_t* __restrict__ n_sel) {
    const double NONE = -__builtin_inf();
    const uint32_t gs = E / p.n_group;
    double mx = NONE, denom = 1.0;
    if (p.score == TRK_SCORE_SOFTMAX) {
        for (uint32_t i = lane; i < E; i += WAVE) mx = ::fmax(mx, (double)lg[i]);  // NaN loses
#pragma unroll
        for (int d = 32; d; d >>= 1) mx = ::fmax(mx, __shfl_xor(mx, d));
        double s = 0.0;
        for (uint32_t i = lane; i < E; i += WAVE)
            if (lg[i] > -__builtin_inff()) s += ::exp((double)lg[i] - mx);
        denom = wave_sum(s);
    }
    auto score = [&](float l) {
        return p.score == TRK_SCORE_SOFTMAX ? ::exp((double)l - mx) / denom : 1.0 / (1.0 + ::exp(-(double)l));
    };
    // what a group's best two are summed from: without a bias the keys are logits
    const bool by_score = !bias && p.n_group > 1 && p.group_top == 2;
    for (uint32_t i = lane; i < E; i += WAVE) {
        const float l = lg[i];
        double k = bias || by_score ? score(l) + (bias ? (double)bias[i] : 0.0) : (double)l;
        key[i] = l > -__builtin_inff() && k > NONE ? k : NONE;  // NaN compares false
    }
    wave_sync();
    uint32_t kept = p.n_group == 1 ? 1u : 0u;  // bit g: group g may be chosen from
    if (p.n_group > 1) {
        double worth = NONE;
        if (lane < p.n_group) {
            double a = NONE, b = NONE;
            for (uint32_t i = 0; i < gs; i++) {
                const double k = key[lane * gs + i];
                if (k > a)
                    b = a, a = k;
                else if (k > b)
                    b = k;
            }
            worth = p.group_top == 2 && b > NONE ? a + b : a;
        }
        for (uint32_t r = 0; r < p.topk_group; r++) {
            double bw = worth;
            uint32_t bi = lane < p.n_group && worth > NONE ? lane : 0xffffffffu;
            wave_best(bw, bi);
            if (bi == 0xffffffffu) break;
            kept |= 1u << bi;
            if (lane == bi) worth = NONE;
        }
        if (by_score) {  // the choice itself goes by the logits
            wave_sync();
            for (uint32_t i = lane; i < E; i += WAVE) key[i] = lg[i] > -__builtin_inff() ? (double)lg[i] : NONE;
            wave_sync();
        }
    }
    uint32_t n = 0, mine = 0xffffffffu;
    for (; n < p.k; n++) {
        double bk = NONE;
        uint32_t bi = 0xffffffffu;
        for (uint32_t i = lane; i < E; i += WAVE)
            if ((kept >> (i / gs) & 1u) && key[i] > NONE && better(key[i], i, bk, bi)) bk = key[i], bi = i;
        wave_best(bk, bi);
        if (bi == 0xffffffffu) break;
        if (bi % WAVE == lane) key[bi] = NONE;
        if (lane == n) mine = bi;
    }
    double s = lane < n ? score(lg[mine]) : 0.0;
    if (p.renorm) {
        const double sum = wave_sum(s);
        s = sum > 0.0 ? s / sum : sum;  // every score underflowed: zeros; NaN stays
    }
    if (lane < p.k) {
        ids[lane] = mine;
        w[lane] = lane < n ? (float)(s * (double)p.factor) : 0.0f;
    }
    if (lane == 0) *n_sel = n;
}

// ---- 32 bits, and what they may be off by ----------------------------------------------------------

template <int CTRL>
__device__ __forceinline__ float dpp_or(float v, float none) {  // lanes without a source get `none`
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float wave_sum32(float v) {
    v += dpp_or<0x111>(v, 0.0f);  // row_shr:1, 2, 4, 8: lane 15 of each row has its sum
    v += dpp_or<0x112>(v, 0.0f);
    v += dpp_or<0x114>(v, 0.0f);
    v += dpp_or<0x118>(v, 0.0f);
    return rdl(v, 15) + rdl(v, 31) + (rdl(v, 47) + rdl(v, 63));
}

// The two largest of a and b's two each
__device__ __forceinline__ void merge2(float& a1, float& a2, float b1, float b2) {
    a2 = __builtin_fmaxf(__builtin_fminf(a1, b1), __builtin_fmaxf(a2, b2));
    a1 = __builtin_fmaxf(a1, b1);
}

constexpr float LOG2E = 1.44269504f;
constexpr uint32_t SC_CAND = 64 + 34;  // LDS entries a wave: candidates, then the best in order

// One row; false where 64 bits have to decide.  NJ: logits a lane holds.  Lanes are split evenly over the groups.  What the
// policy asks for is in the template: with branches on it between a row's loads they wait for one another.
template <int NJ, bool SOFT, bool BIAS, bool GROUPED>
__device__ __forceinline__ bool score_row32(const float* __restrict__ lg, const float* __restrict__ bias, uint32_t E,
                                            const ScorePolicy& p, uint32_t lane, uint2* cand, uint32_t* __restrict__ ids,
                                            float* __restrict__ w, uint32_t* __restrict__ n_sel) {
    const float NONE = -__builtin_inff();
    const uint32_t gs = E / p.n_group, L = p.group_lanes, g = lane / L, r0 = lane % L;
    float v[NJ], key[NJ];
    uint32_t idx[NJ];
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const uint32_t r = r0 + L * j;
        const bool in = g < p.n_group && r < gs;
        idx[j] = in ? g * gs + r : 0;
        v[j] = lg[idx[j]];
        key[j] = BIAS ? bias[idx[j]] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const bool in = g < p.n_group && r0 + L * j < gs;
        v[j] = in && v[j] > NONE ? v[j] : NONE;  // NaN compares false
    }
    float mx = 0.0f, denom = 1.0f, tol = 0.0f, scale = 1.0f;
    const bool sums = GROUPED && p.group_top == 2;
    const bool scored = BIAS || sums;  // else keys are logits
    if constexpr (SOFT) {
        uint32_t mk = 0;
#pragma unroll
        for (int j = 0; j < NJ; j++) mk = mk > fkey(v[j]) ? mk : fkey(v[j]);
        mk = wave_max_u32(mk);
        if (mk == fkey(__builtin_inff())) return false;  // scores that are NaN
        mx = fkey_inv(mk);
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < NJ; j++) s += __builtin_amdgcn_exp2f((v[j] - mx) * LOG2E);
        denom = wave_sum32(s);
        scale = 1.0f / denom;  // the largest score
        // (l - mx) log2 e and its power are off by d 3 2^-24 + 2^-23 at distance d, where d e^-d <= 0.37; the sum by 38
        // roundings and its terms': a score by less than 2^-18 of the largest
        tol = scale * 0x1p-18f;
    } else {
        // s (1 - s) |l| <= 0.23: the argument's two roundings, the power's, the sum's and the reciprocal's make less
        // than 2^-22
        tol = 0x1p-22f;
    }
    float a1 = NONE, a2 = NONE;  // of this lane's keys
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        if (BIAS || GROUPED) {  // (groups by their best logit alone: the logits again, below)
            const float s = SOFT ? __builtin_amdgcn_exp2f((v[j] - mx) * LOG2E) * scale
                                 : __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-v[j] * LOG2E));
            const float k = s + key[j];
            key[j] = v[j] > NONE && k > NONE ? (scored ? k : v[j]) : NONE;
        } else {
            key[j] = v[j];
        }
        merge2(a1, a2, key[j], NONE);
    }
    // score and key in 64 bits; the softmax's sum too, once one of them is asked for
    double denom64 = 0.0;
    auto sum64 = [&] {
        if (!SOFT || denom64 != 0.0) return;
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < NJ; j++) s += v[j] > NONE ? ::exp((double)v[j] - (double)mx) : 0.0;
        denom64 = wave_sum(s);
    };
    auto key64 = [&](float l, float b) {
        const double s = SOFT ? ::exp((double)l - (double)mx) / denom64 : 1.0 / (1.0 + ::exp(-(double)l));
        return s + (BIAS ? (double)b : 0.0);
    };
    if constexpr (GROUPED) {
        if (L > 1) merge2(a1, a2, dpp_f<0xB1>(a1), dpp_f<0xB1>(a2));    // lane ^ 1
        if (L > 2) merge2(a1, a2, dpp_f<0x4E>(a1), dpp_f<0x4E>(a2));    // ^ 2
        if (L > 4) merge2(a1, a2, dpp_f<0x141>(a1), dpp_f<0x141>(a2));  // mirrored in 8: the other quad
        if (L > 8) merge2(a1, a2, dpp_f<0x140>(a1), dpp_f<0x140>(a2));  // mirrored in 16: the other 8
        if (L > 16) merge2(a1, a2, __shfl_xor(a1, 16), __shfl_xor(a2, 16));
        const float worth = g >= p.n_group ? NONE : sums && a2 > NONE ? a1 + a2 : a1;
        uint32_t rank = 0;
        for (uint32_t i = 0; i < p.n_group; i++) {
            const float o = rdl(worth, i * L);
            rank += o > worth || (o == worth && i < g) ? 1u : 0u;
        }
        bool kept = rank < p.topk_group && worth > NONE;
        // the worst group kept and the best one dropped; a sum of two keys is off by twice a key and a rounding, and -inf below
        // the lowest number: its group (key 1) is there, and its place open
        const uint32_t there = fkey(worth), drop = a1 > NONE && there == 0u ? 1u : there;
        const uint32_t lo = ~wave_max_u32(kept ? ~there : 0u), hi = wave_max_u32(kept ? 0u : drop);
        if (scored && hi) {
            const float fl = fkey_inv(lo), fh = fkey_inv(hi);
            // of a sum: its keys' errors, their roundings and its own
            const float both = __builtin_fabsf(a1) + (a2 > NONE ? __builtin_fabsf(a2) : 0.0f);
            const float big = __uint_as_float(wave_max_u32(g < p.n_group && a1 > NONE ? __float_as_uint(both) : 0u));
            if (!(fl - fh > 4.0f * tol + 0x1p-22f * big)) {  // so too where one is no number, or none is kept
                sum64();
                double d1 = (double)NONE, d2 = (double)NONE;
#pragma unroll
                for (int j = 0; j < NJ; j++) {
                    const double k = key[j] > NONE ? key64(v[j], BIAS ? bias[idx[j]] : 0.0f) : (double)NONE;
                    d2 = ::fmax(d2, ::fmin(d1, k)), d1 = ::fmax(d1, k);
                }
                for (uint32_t d = 1; d < L; d *= 2) {
                    const double o1 = __shfl_xor(d1, d), o2 = __shfl_xor(d2, d);
                    d2 = ::fmax(::fmin(d1, o1), ::fmax(d2, o2)), d1 = ::fmax(d1, o1);
                }
                const double w64 = g >= p.n_group ? (double)NONE : sums && d2 > (double)NONE ? d1 + d2 : d1;
                rank = 0;
                for (uint32_t i = 0; i < p.n_group; i++) {
                    const double o = __shfl(w64, i * L);
                    rank += o > w64 || (o == w64 && i < g) ? 1u : 0u;
                }
                kept = rank < p.topk_group && w64 > (double)NONE;
            }
        }
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            key[j] = !kept ? NONE : BIAS ? key[j] : v[j];  // without a bias the choice goes by the logits
        }
    }
    // Selection as route_select's: the kk-th largest of the lanes' maxima, cut to 16 bits, bounds the kk-th largest key
    // from below; the keys that reach it are ranked.  kk = k + 1 where the next key has to be told from the k-th.
    const uint32_t kk = p.k + (BIAS ? 1u : 0u);
    uint32_t fk[NJ], lmax = 0;
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        fk[j] = fkey(key[j]);
        lmax = lmax > fk[j] ? lmax : fk[j];
    }
    uint32_t T = 0;
#pragma unroll
    for (int b = 30; b >= 16; b -= 2) {
        const uint32_t t1 = T | (1u << b), t2 = T | (2u << b), t3 = T | (3u << b);
        const uint32_t c1 = (uint32_t)__popcll(__ballot(lmax >= t1));
        const uint32_t c2 = (uint32_t)__popcll(__ballot(lmax >= t2));
        const uint32_t c3 = (uint32_t)__popcll(__ballot(lmax >= t3));
        T = c3 >= kk ? t3 : (c2 >= kk ? t2 : (c1 >= kk ? t1 : T));
    }
    if (BIAS && T > 1u) {  // and what 32 bits may have put below it
        const float f = fkey_inv(T);
        T = fkey(f - 2.0f * tol - 0x1p-22f * __builtin_fabsf(f));
    }
    T = T > 1u ? T : 1u;
    uint32_t C = 0;
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const bool c = fk[j] >= T;
        const uint64_t m = __ballot(c);
        const uint32_t at = C + __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u));
        if (c && at < 64u) cand[at] = make_uint2(fk[j], idx[j]);
        C += (uint32_t)__popcll(m);
    }
    if (C > 64u) return false;
    wave_sync();
    const uint2 me = lane < C ? cand[lane] : make_uint2(0u, 0xffffffffu);
    uint32_t rank = 0;
    for (uint32_t t = 0; t < C; t++) {
        const uint32_t kt = (uint32_t)__builtin_amdgcn_readlane((int)me.x, (int)t);
        const uint32_t it = (uint32_t)__builtin_amdgcn_readlane((int)me.y, (int)t);
        rank += kt > me.x || (kt == me.x && it < me.y) ? 1u : 0u;
    }
    if (lane < C && rank < kk) cand[64 + rank] = me;
    wave_sync();
    const uint32_t have = C < kk ? C : kk, n = have < p.k ? have : p.k;
    const uint2 best = lane < have ? cand[64 + lane] : make_uint2(0u, 0xffffffffu);
    uint32_t mine = best.y;
    if constexpr (BIAS) {
        const uint32_t next = (uint32_t)__shfl_down((int)best.x, 1);
        const float k0 = fkey_inv(best.x), k1 = fkey_inv(next);
        const bool close = !(k0 - k1 > 2.0f * tol + 0x1p-22f * __builtin_fmaxf(__builtin_fabsf(k0), __builtin_fabsf(k1)));
        if (__ballot(lane + 1 < have && close)) {  // the candidates once more, by their keys in 64 bits
            sum64();
            const double k = lane < C ? key64(lg[me.y], bias[me.y]) : -__builtin_inf();
            rank = 0;
            for (uint32_t t = 0; t < C; t++) {
                const double kt = __shfl(k, t);
                const uint32_t it = (uint32_t)__builtin_amdgcn_readlane((int)me.y, (int)t);
                rank += kt > k || (kt == k && it < me.y) ? 1u : 0u;
            }
            wave_sync();
            if (lane < C && rank < kk) cand[64 + rank] = me;
            wave_sync();
            mine = lane < have ? cand[64 + lane].y : 0xffffffffu;
        }
    }
    // the weights in 64 bits, a lane each: sigmoids that 32 bits lose below their sum still have their ratios.  A softmax
    // that stays as it is takes its sum in 64 bits too: in 32 it is off by up to 5 2^-24, and other rows (score_row) would
    // have other bits.  2048 x 512 4.2 -> 5.7 us, 16384 x 256 10.8 -> 14.7.
    if (SOFT && !p.renorm) sum64();
    double s = 0.0;
    if (lane < n) {
        const double l = (double)lg[mine];
        s = SOFT ? ::exp(l - (double)mx) / (p.renorm ? 1.0 : denom64) : 1.0 / (1.0 + ::exp(-l));
    }
    if (p.renorm) {
        double sum = s;
        for (int d = n > 32 ? 32 : n > 16 ? 16 : n > 8 ? 8 : n > 4 ? 4 : n > 2 ? 2 : 1; d; d >>= 1) sum += __shfl_xor(sum, d);
        s = sum > 0.0 ? s / sum : sum;
    }
    if (lane < p.k) {
        ids[lane] = lane < n ? mine : 0xffffffffu;
        w[lane] = lane < n ? (float)(s * (double)p.factor) : 0.0f;
    }
    if (lane == 0) *n_sel = n;
    return true;
}

// p.group_lanes for E experts; returns the logits that a lane then holds.
inline uint32_t score_lanes(ScorePolicy& p, uint32_t E) {
    p.group_lanes = WAVE;
    while (p.group_lanes * p.n_group > WAVE) p.group_lanes /= 2;
    return (E / p.n_group + p.group_lanes - 1) / p.group_lanes;
}

}  // namespace trk
