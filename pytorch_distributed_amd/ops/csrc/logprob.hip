// Log-probabilities of given tokens with entropy and the best alternatives, and their gradient.
//
//   z = x / T,  m = max x,  s = sum exp((x - m) / T),  u = sum exp((x - m) / T) (x - m) / T
//   logprob = (x_t - m) / T - log s,   entropy = log s - u / s,   logsumexp = m / T + log s
//   dx_i = (p_i (dlse - dlp - dent (logp_i + entropy)) + dlp [i = t]) / T,   p_i = exp(logp_i)
//
// Exponents are formed as 2^(x c - r), c = log2(e) / T, r = m c rounded: one fused multiply-add per value.  r's rounding
// is common to all values of a row and cancels, because s is taken relative to r and logp = (x c - r) - log2 s.
// (m, log2 s) is what the forward pass keeps for the backward pass: their sum would round p by |lse| 2^-24.
// A logit of -inf is a masked token: p = 0, no share in the entropy, gradient 0.  A row with nothing but -inf: logprob
// and logsumexp -inf, entropy 0, gradient 0.  An ignored row is not read: 0 everywhere, alternatives -1.
// A token outside the vocabulary gives NaN (log-probability and gradient row) and reads nothing.
#include "seq.h"
#pragma clang fp reassociate(off)       // (x - m) / T stays what it is: x / T and m / T alone may overflow

struct LogprobArgs {
    const void* logits; long long ld; long long rows; int vocab;
    const void* tokens; int tok64; long long ignore;
    float inv_t, c; int top_k;                          // 1 / T, log2(e) / T
    float* logprob; float* entropy; float* lse;         // [rows]
    float* stat_m; float* stat_l2;                      // [rows]: m, log2 s, for the backward pass (null: none follows)
    float* top_lp; long long* top_id;                   // [rows][top_k]
    // backward
    const float* d_lp; const float* d_ent; const float* d_lse;  // [rows], any may be null
    void* d_logits;                                     // [rows][vocab], contiguous
    // long rows cut into `splits` parts (forward): what each part leaves for the joining launch
    int splits; float* part_stat; unsigned long long* part_top;     // [rows][splits][4], [rows][splits][top_k]
};
#define LP_MAX_TOP 32
#define LP_SHORT 1024       // rows up to here are held in registers by one wave or a part of one

__device__ __forceinline__ long long lp_token(const LogprobArgs& p, long long row) {
    return p.tok64 ? ((const long long*)p.tokens)[row] : (long long)((const int*)p.tokens)[row];
}

// Order of the alternatives as one unsigned number: larger value first (NaN above all, -0 = +0), then the lower index.
__device__ __forceinline__ uint64_t lp_key(float x, int i) {
    uint32_t b = __builtin_bit_cast(uint32_t, x);
    if (b == 0x80000000u) b = 0u;
    b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    if (x != x) b = 0xfffffffeu;         // (all ones would be above every "key < last")
    return ((uint64_t)b << 32) | (uint32_t)~i;
}
__device__ __forceinline__ int lp_key_index(uint64_t k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float lp_key_value(uint64_t k) {         // (0 for -0: its log-probability is the same)
    const uint32_t b = (uint32_t)(k >> 32);
    return __builtin_bit_cast(float, (b & 0x80000000u) ? (b & 0x7fffffffu) : ~b);
}
__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t t = __shfl_xor((unsigned long long)v, o, 64);
        v = t > v ? t : v;
    }
    return v;
}

// softmax statistics of a part of a row: its maximum m, and relative to r = m c rounded: s = sum 2^d, u = sum 2^d d,
// d = x c - r
struct LpStat { float m, s, u; };
#define LP_LN2 0.693147180559945309f
// The rounding of r is at most |r| 2^-24: below LP_NEAR 2^(its rounding) stays near 1.  Rows whose maximum lies beyond it
// (logits of more than 7e6 T, masks of the type's lowest value in every place) are walked once more with d = (x - m) c.
// A part's s stays below 2^32 for each of its values up to LP_FAR, where r is rounded to multiples of 64.  A part beyond that,
// nothing but masks of a low value, takes d = (x - m) c too: how it stands to another part's r is not known, and need not be,
// because a row whose maximum is near drops it.
#define LP_NEAR 1.0e7f
#define LP_FAR 1.0e9f
__device__ __forceinline__ float lp_exp2(float d) { return __builtin_amdgcn_exp2f(d); }
__device__ __forceinline__ float lp_ref(float m, float c) {
    float r = m * c;
    asm("" : "+v"(r));          // r is this rounded product wherever it is used: no contraction into an fma
    return r;
}
__device__ __forceinline__ bool lp_near(float r) { return fabsf(r) < LP_NEAR; }
// `st` seen from the maximum m >= st.m.  No part of it turns into 0 * inf, unless the row is walked: the shift is cut off where
// 2^shift is 0, and s < 2^62 times a shift of 2e9, or a far part's s < 2^30 times the cut-off, is finite.
__device__ __forceinline__ LpStat lp_shift(LpStat st, float m, float c) {
    const float d = st.m == m ? 0.f : fmaxf(lp_ref(st.m, c) - lp_ref(m, c), -1.0e20f), e = lp_exp2(d);
    return LpStat{m, st.s * e, e * __builtin_fmaf(d, st.s, st.u)};
}
__device__ __forceinline__ LpStat lp_merge(LpStat a, LpStat b, float c) {
    const float m = fmaxf(a.m, b.m);
    a = lp_shift(a, m, c);
    b = lp_shift(b, m, c);
    return LpStat{m, a.s + b.s, a.u + b.u};
}
// NX values (-inf where there is none); bm >= each of them
template <int NX>
__device__ __forceinline__ void lp_add(LpStat& st, const float (&x)[NX], float bm, float c) {
    st = lp_shift(st, fmaxf(st.m, bm), c);
    const float r = st.m == -INFINITY ? 0.f : lp_ref(st.m, c);
    float s = 0.f, u = 0.f;
    if (fabsf(r) < LP_FAR) {
#pragma unroll
        for (int i = 0; i < NX; ++i) {
            const float d = __builtin_fmaf(x[i], c, -r), e = lp_exp2(d);
            s += e;                                             // (NaN for a NaN)
            u = __builtin_fmaf(e, fmaxf(d, -1000.f), u);        // (0 for -inf)
        }
    } else {            // (NaN for +inf)
#pragma unroll
        for (int i = 0; i < NX; ++i) {
            const float d = (x[i] - st.m) * c, e = lp_exp2(d);
            s += e;
            u = __builtin_fmaf(e, fmaxf(d, -1000.f), u);
        }
    }
    st.s += s;
    st.u += u;
}
// over groups of G lanes
template <int G>
__device__ __forceinline__ LpStat lp_across(LpStat st, float c) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1)
        st = lp_merge(st, LpStat{__shfl_xor(st.m, o, 64), __shfl_xor(st.s, o, 64), __shfl_xor(st.u, o, 64)}, c);
    return st;
}

__device__ __forceinline__ void lp_ignored_row(const LogprobArgs& p, long long row) {
    p.logprob[row] = 0.f; p.entropy[row] = 0.f; p.lse[row] = 0.f;
    if (p.stat_m) { p.stat_m[row] = 0.f; p.stat_l2[row] = 0.f; }
    for (int k = 0; k < p.top_k; ++k) { p.top_lp[row * p.top_k + k] = 0.f; p.top_id[row * p.top_k + k] = -1; }
}

// What the row's values become.  NEAR: d = x c - r; otherwise d = (x - m) c, for rows whose m c leaves 32 bits, and for
// short rows, which cost nothing either way.
struct LpRow {
    float m, r, c, l2; bool near, empty;
    __device__ __forceinline__ LpRow(float m_, float l2_, float c_, bool short_row) : m(m_), c(c_), l2(l2_) {
        r = lp_ref(m, c);
        near = !short_row && lp_near(r);
        empty = m == -INFINITY && l2 == l2;     // nothing but -inf
    }
    __device__ __forceinline__ float log2p(float x) const { return (near ? __builtin_fmaf(x, c, -r) : (x - m) * c) - l2; }
    __device__ __forceinline__ float logp(float x, float inv_t) const {
        if (empty) return -INFINITY;
        const float v = log2p(x) * LP_LN2;      // (x c may leave 32 bits where x / T does not)
        return v == -INFINITY && x > -INFINITY ? (x - m) * inv_t - l2 * LP_LN2 : v;
    }
};
// s = 0 for a row of nothing but -inf; NaN where the row holds NaN or +inf
__device__ __forceinline__ float lp_log2_sum(LpStat st) {
    if (st.m == INFINITY || st.s != st.s) return __builtin_nanf("");
    return st.s == 0.f ? 0.f : __builtin_amdgcn_logf(st.s);
}
// The given token's logit, NaN for a token outside the vocabulary.  (Its load is issued with the row's, not behind its sums.)
template <typename T>
__device__ __forceinline__ float lp_given(const LogprobArgs& p, const T* x, long long tok) {
    return tok >= 0 && tok < p.vocab ? to_f32(x[tok]) : __builtin_nanf("");
}
__device__ __forceinline__ void lp_finish_row(const LogprobArgs& p, long long row, float xt, LpStat st, const LpRow& q) {
    p.logprob[row] = xt == xt ? q.logp(xt, p.inv_t) : xt;
    p.entropy[row] = q.empty ? 0.f : (q.l2 - st.u / st.s) * LP_LN2;
    p.lse[row] = q.empty ? -INFINITY : q.near ? (q.r + q.l2) * LP_LN2 : __builtin_fmaf(q.m, p.inv_t, q.l2 * LP_LN2);
    if (p.stat_m) { p.stat_m[row] = st.m; p.stat_l2[row] = q.l2; }
}
__device__ __forceinline__ void lp_put_alternative(const LogprobArgs& p, long long row, int k, uint64_t key, const LpRow& q) {
    p.top_id[row * p.top_k + k] = lp_key_index(key);
    p.top_lp[row * p.top_k + k] = q.logp(lp_key_value(key), p.inv_t);
}

// Rows that the running statistics cannot take: nothing but -inf, NaN, +inf, or |m c| beyond LP_NEAR.  Whole workgroup, two walks and one more for each alternative.
template <typename T>
__device__ __forceinline__ void lp_walk_row(const LogprobArgs& p, long long row, float xt, LpStat* part, uint64_t* best) {
    const T* x = (const T*)p.logits + row * p.ld;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    float m = -INFINITY, bad = 0.f;
    for (int i = tid; i < p.vocab; i += 256) {
        const float v = to_f32(x[i]);
        m = fmaxf(m, v);
        if (v != v) bad = v;
    }
    m = wave_max(m);
    bad = wave_sum(bad);
    __syncthreads();                // (earlier reads of part[] and best[])
    if (lane == 0) part[wave] = LpStat{m, bad, 0.f};
    __syncthreads();
    m = fmaxf(fmaxf(part[0].m, part[1].m), fmaxf(part[2].m, part[3].m));
    bad = part[0].s + part[1].s + part[2].s + part[3].s;
    // the form of d that LpRow, here and in the backward pass, takes for this maximum: s is relative to it
    const float r = lp_ref(m, p.c);
    const bool near = lp_near(r);
    float s = bad, u = 0.f;
    if (m > -INFINITY)
        for (int i = tid; i < p.vocab; i += 256) {
            const float v = to_f32(x[i]), d = near ? __builtin_fmaf(v, p.c, -r) : (v - m) * p.c, e = lp_exp2(d);
            s += e;
            u += e > 0.f ? e * d : 0.f;
        }
    s = wave_sum(s);
    u = wave_sum(u);
    __syncthreads();
    if (lane == 0) part[wave] = LpStat{m, s, u};
    __syncthreads();
    const LpStat st{m, (part[0].s + part[1].s) + (part[2].s + part[3].s), (part[0].u + part[1].u) + (part[2].u + part[3].u)};
    const LpRow q(m, lp_log2_sum(st), p.c, false);
    if (tid == 0) lp_finish_row(p, row, xt, st, q);
    uint64_t last = ~0ull;
    for (int k = 0; k < p.top_k; ++k) {
        uint64_t b = 0;
        for (int i = tid; i < p.vocab; i += 256) {
            const uint64_t key = lp_key(to_f32(x[i]), i);
            if (key < last && key > b) b = key;
        }
        b = wave_max_u64(b);
        __syncthreads();            // (the previous round's reads of best[])
        if (lane == 0) best[wave] = b;
        __syncthreads();
        last = best[0];
        for (int w = 1; w < 4; ++w) last = best[w] > last ? best[w] : last;
        if (tid == 0) lp_put_alternative(p, row, k, last, q);
    }
    __syncthreads();
}
__device__ __forceinline__ bool lp_ordinary(LpStat st, float c) {
    return st.s > 0.f && st.s < INFINITY && lp_near(lp_ref(st.m, c));
}
// The top_k largest of n distinct keys (0: none) in LDS, by counting what is above each: whole workgroup
template <typename F>
__device__ __forceinline__ void lp_rank(const uint64_t* keys, int n, int top_k, F put) {
    for (int i = threadIdx.x; i < n; i += 256) {
        const uint64_t mine = keys[i];
        int above = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) above += keys[j] > mine ? 1 : 0;
        if (above < top_k && mine != 0) put(above, mine);
    }
}

// ---- rows of up to LP_SHORT tokens: G lanes hold E tokens each --------------------------------------------------------
// One load, butterfly sums within the G lanes, no LDS.  Bound by the launch: 4096 x 18 fp32 (0.3 MB) 3.6 us forward, 3.2 us
// backward, where the smallest launches of this file take 2.3.
template <typename T, int E, int G>
__global__ __launch_bounds__(256) void logprob_short_kernel(LogprobArgs p) {
    const int lane = threadIdx.x & 63, l = lane & (G - 1);
    const long long step = (long long)gridDim.x * (256 / G);
    // (every lane of a wave takes every round: the shuffles want them all)
    for (long long r0 = (long long)blockIdx.x * (256 / G); r0 < p.rows; r0 += step) {
        const long long row = r0 + threadIdx.x / G;
        const bool on = row < p.rows;
        const long long tok = on ? lp_token(p, row) : p.ignore;
        const bool live = on && tok != p.ignore;
        const T* x = (const T*)p.logits + (live ? row : 0) * p.ld;
        const float xt = live && l == 0 ? lp_given(p, x, tok) : 0.f;
        float xs[E], m = -INFINITY, bad = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = l + e * G;
            xs[e] = live && i < p.vocab ? to_f32(x[i]) : -INFINITY;
            m = fmaxf(m, xs[e]);
            if (xs[e] != xs[e]) bad = xs[e];
        }
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        float s = bad, u = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = m == -INFINITY ? -INFINITY : (xs[e] - m) * p.c, ex = lp_exp2(d);
            s += ex;
            u += ex > 0.f ? ex * d : 0.f;
        }
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) { s += __shfl_xor(s, o, 64); u += __shfl_xor(u, o, 64); }
        const LpStat st{m, s, u};
        const LpRow q(m, lp_log2_sum(st), p.c, true);
        if (l == 0 && on) {
            if (live) lp_finish_row(p, row, xt, st, q);
            else lp_ignored_row(p, row);
        }
        uint64_t last = ~0ull;
        for (int k = 0; k < p.top_k; ++k) {
            uint64_t b = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int i = l + e * G;
                const uint64_t key = i < p.vocab ? lp_key(xs[e], i) : 0;
                if (key < last && key > b) b = key;
            }
#pragma unroll
            for (int o = G / 2; o > 0; o >>= 1) {
                const uint64_t t = __shfl_xor((unsigned long long)b, o, 64);
                b = t > b ? t : b;
            }
            last = b;
            if (l == 0 && live) lp_put_alternative(p, row, k, last, q);
        }
    }
}

// ---- long rows ---------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint64_t lp_lane(uint64_t v, int lane) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) |
           (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
__device__ __forceinline__ uint64_t lp_next_lane(uint64_t v) {      // lane i gets lane i - 1's (0x138: wave_shr by one)
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), 0x138, 0xf, 0xf, false);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)v, 0x138, 0xf, 0xf, false);
    return ((uint64_t)hi << 32) | lo;
}
// LDS written by some lanes of a wave and read by others
__device__ __forceinline__ void lp_wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
#define LP_FIRST 128       // keys that a wave's first batch may hold in LDS
// A wave's best keys, sorted over its lanes, and what a value has to reach (`strict`: to exceed) to come among them.
struct LpList {
    uint64_t key; float lim; bool strict, full;
    __device__ __forceinline__ LpList() : key(0), lim(-INFINITY), strict(false), full(false) {}
    __device__ __forceinline__ bool passes(float v) const { return strict ? v > lim : v >= lim; }
    // k-th largest of the lanes' t: at least k values of the first batch reach it
    __device__ __forceinline__ void first_limit(float t, int k) {
        const int lane = threadIdx.x & 63;
        int above = 0;
#pragma unroll 16
        for (int o = 0; o < 64; ++o) {
            const float other = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, t), o));
            above += (other > t || (other == t && o < lane)) ? 1 : 0;
        }
        const uint64_t who = __ballot(above == k - 1);
        if (who) lim = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, t), __builtin_ctzll(who)));
    }
    // the lanes of `todo` offer a key each (all lanes take part)
    __device__ __forceinline__ void insert(uint64_t todo, uint64_t mine, int k) {
        const int lane = threadIdx.x & 63;
        while (todo) {
            const int src = __builtin_ctzll(todo);
            todo &= todo - 1;
            const uint64_t q = lp_lane(mine, src);
            const int pos = __builtin_popcountll(__ballot(key > q));
            if (pos >= k) continue;
            const uint64_t up = lp_next_lane(key);
            key = lane < pos ? key : (lane == pos ? q : up);
        }
        settle(k);
    }
    // the first values at once: n <= LP_FIRST keys in `from` (this wave's LDS), ordered by counting what is above each
    __device__ __forceinline__ void fill(const uint64_t* from, uint64_t* sorted, int n, int k) {
        const int lane = threadIdx.x & 63;
        lp_wave_fence();
        const uint64_t q0 = lane < n ? from[lane] : 0, q1 = lane + 64 < n ? from[lane + 64] : 0;
        int a0 = 0, a1 = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
            const uint64_t o = from[j];
            a0 += o > q0 ? 1 : 0;
            a1 += o > q1 ? 1 : 0;
        }
        if (q0 != 0 && a0 < 64) sorted[a0] = q0;
        if (q1 != 0 && a1 < 64) sorted[a1] = q1;
        lp_wave_fence();
        key = lane < n ? sorted[lane] : 0;
        settle(k);
    }
    __device__ __forceinline__ void settle(int k) {
        const uint64_t kth = lp_lane(key, k - 1);
        if (kth == 0) return;
        const float v = lp_key_value(kth);
        if (!full || v > lim) { lim = v; strict = false; }      // equal values of this batch may have lower indices
        full = true;
    }
};

// A workgroup reads a row (or one of its splits) once, in 16-byte loads, the next four in flight while four are worked on.
// Each thread keeps running statistics, shifted once per 32 or 16 values.  The alternatives: each wave keeps its best keys
// sorted over its lanes.  A value is looked at again only if it passes the wave's k-th best, which the first batch sets to
// the k-th largest of the lanes' maxima; a wave of n values then inserts about k (2 + ln(n / 2048)) of them, each by a
// ballot and a shift by one lane.  That is for rows in no particular order; of values in ascending order every one is inserted
// (1024 x 32000 bf16, 8 alternatives: 34 us in random order, 622 ascending; 1 x 131072, 20: 10 + 5 and 27 + 15).  FILL: the first batch, which is all that a wave of a split row mostly sees, is ordered
// at once instead (1 row of 131072 bf16, 20 alternatives: 11.4 -> 10.0 us; in the loop over a whole row the same code costs
// more than it saves: 4096 rows 248 -> 277 us).
//
// 4096 x 32000 bf16 without alternatives, a tenth of the rows ignored: 48.5 us for 236 MB, 4.9 TB/s (a sum of 256 MB: 5.7).
// 4096 x 131072 bf16 with 8 alternatives: 247 us, 4.3 TB/s, in one process, 261 to 280 in others of the same build (a sum of 1
// GB reads 4.0 TB/s).  Half of every row masked with the type's lowest value: 4096 x 32000 45 us, as without.  Split rows are bound by the
// latency of the chain of loads, joins and the second launch: 1 x 131072 10.0 + 4.6 us.  (Workgroups of 1024 threads with a
// shared limit, so that fewer parts are joined: 16 to 32 us.)
template <typename T, bool TOP, bool FILL>
__global__ __launch_bounds__(256, 4) void logprob_long_kernel(LogprobArgs p) {
    constexpr int VEC = 16 / sizeof(T), U = 2, NX = U * VEC;
    __shared__ LpStat part[4];
    __shared__ uint64_t keys[4 * LP_MAX_TOP], firsts[FILL ? 4 : 1][LP_FIRST], sorted[FILL ? 4 : 1][64];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const float c = p.c;
    const long long units = p.rows * p.splits;
    for (long long unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const long long row = unit / p.splits;
        const int split = (int)(unit - row * p.splits);
        const long long tok = lp_token(p, row);
        if (tok == p.ignore) {
            if (tid == 0 && p.splits == 1) lp_ignored_row(p, row);
            continue;
        }
        const T* x = (const T*)p.logits + row * p.ld;
        const float xt = p.splits == 1 && tid == 0 ? lp_given(p, x, tok) : 0.f;
        // head: tokens in front of the first 16-byte boundary; behind the vectors the tail
        const int head = min((int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T), p.vocab);
        const int nvec = (p.vocab - head) / VEC, tail = (p.vocab - head) - nvec * VEC;
        const int per = (nvec + p.splits - 1) / p.splits, v0 = min(split * per, nvec), v1 = min(v0 + per, nvec);
        const vec16<T>* xv = reinterpret_cast<const vec16<T>*>(x + head);
        LpStat st{-INFINITY, 0.f, 0.f};
        LpList list;
        auto fetch = [&](vec16<T> (&raw)[U], int b) {
            if (b + U * 256 <= v1) {
#pragma unroll
                for (int u = 0; u < U; ++u) raw[u] = xv[b + u * 256 + tid];
            } else {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int v = b + u * 256 + tid;
                    if (v < v1) {
                        raw[u] = xv[v];
                    } else {
#pragma unroll
                        for (int j = 0; j < VEC; ++j) raw[u].e[j] = from_f32<T>(-INFINITY);
                    }
                }
            }
        };
        auto take = [&](const vec16<T> (&raw)[U], int b) {
            float xs[NX], bm = -INFINITY;
#pragma unroll
            for (int i = 0; i < NX; ++i) { xs[i] = to_f32(raw[i / VEC].e[i % VEC]); bm = fmaxf(bm, xs[i]); }
            lp_add<NX>(st, xs, bm, c);
            if (!TOP) return;
            if (b == v0) list.first_limit(bm, p.top_k);
            else if (list.full) list.strict = true;         // an equal value of a later batch has a higher index
            if (__ballot(list.passes(bm)) == 0) return;
            uint32_t mask = 0;
#pragma unroll
            for (int i = 0; i < NX; ++i)
                if (list.passes(xs[i]) && b + (i / VEC) * 256 + tid < v1) mask |= 1u << i;
            bool first = FILL && b == v0;
            int count = 0;              // of the first batch's keys
            for (uint64_t todo = __ballot(mask != 0); todo; todo = __ballot(mask != 0)) {
                const int slot = __builtin_ctz(mask | 0x80000000u);
                mask &= mask - 1;
                float v = xs[0];
#pragma unroll
                for (int i = 1; i < NX; ++i) v = slot == i ? xs[i] : v;
                const uint64_t key = lp_key(v, head + (b + (slot / VEC) * 256 + tid) * VEC + slot % VEC);
                const int more = __builtin_popcountll(todo);
                if (first && count + more <= LP_FIRST) {
                    if (todo >> lane & 1) firsts[wave][count + __builtin_popcountll(todo & ((1ull << lane) - 1))] = key;
                    count += more;
                    continue;
                }
                if (FILL && first) list.fill(firsts[wave], sorted[wave], count, p.top_k);
                first = false;
                list.insert(todo, key, p.top_k);
            }
            if (FILL && first) list.fill(firsts[wave], sorted[wave], count, p.top_k);
        };
        vec16<T> even[U], odd[U];
        fetch(even, v0);
        for (int b = v0; b < v1; b += 2 * 256 * U) {
            fetch(odd, b + 256 * U);
            take(even, b);
            if (b + 256 * U >= v1) break;
            fetch(even, b + 2 * 256 * U);
            take(odd, b + 256 * U);
        }
        if (split == 0 && wave == 0 && head + tail > 0) {       // at most 14 single tokens
            const bool valid = lane < head + tail;
            const int i = lane < head ? lane : head + nvec * VEC + (lane - head);
            float xs[1] = {valid ? to_f32(x[i]) : -INFINITY};
            lp_add<1>(st, xs, xs[0], c);
            if (TOP) {
                list.strict = false;
                list.insert(__ballot(valid && list.passes(xs[0])), lp_key(xs[0], i), p.top_k);
            }
        }
        st = lp_across<64>(st, c);
        if (lane == 0) part[wave] = st;
        if (lane < p.top_k) keys[wave * p.top_k + lane] = list.key;
        __syncthreads();
        st = lp_merge(lp_merge(part[0], part[1], c), lp_merge(part[2], part[3], c), c);
        if (p.splits > 1) {
            if (tid == 0) {
                float* o = p.part_stat + unit * 4;
                o[0] = st.m; o[1] = st.s; o[2] = st.u;
            }
            if (tid < p.top_k) p.part_top[unit * p.top_k + tid] = 0;     // (a split may hold fewer than top_k tokens)
            __syncthreads();
            lp_rank(keys, 4 * p.top_k, p.top_k, [&](int k, uint64_t key) { p.part_top[unit * p.top_k + k] = key; });
        } else if (!lp_ordinary(st, c)) {
            lp_walk_row<T>(p, row, xt, part, keys);
        } else {
            const LpRow q(st.m, lp_log2_sum(st), c, false);
            if (tid == 0) lp_finish_row(p, row, xt, st, q);
            lp_rank(keys, 4 * p.top_k, p.top_k, [&](int k, uint64_t key) { lp_put_alternative(p, row, k, key, q); });
        }
        __syncthreads();            // part[] and keys[] are reused by the next unit
    }
}
// Joins the splits of a row, one per lane.  Of their sorted lists only keys that reach the k-th largest of the lists' first ceil(k /
// splits) entries can be among the best: mostly k and a few more.
#define LP_JOIN_KEYS 1024
template <typename T>
__global__ __launch_bounds__(256) void logprob_join_kernel(LogprobArgs p) {
    __shared__ uint64_t keys[LP_JOIN_KEYS], heads[128], limit;
    __shared__ LpStat part[4];
    __shared__ int count;
    const long long row = blockIdx.x;
    const long long tok = lp_token(p, row);
    const int tid = threadIdx.x, lane = tid & 63, k = p.top_k, n = p.splits * k;
    if (tok == p.ignore) {
        if (tid == 0) lp_ignored_row(p, row);
        return;
    }
    // everything this row needs is asked for at once
    const float xt = tid == 0 ? lp_given(p, (const T*)p.logits + row * p.ld, tok) : 0.f;
    float4 own{-INFINITY, 0.f, 0.f, 0.f};       // (every wave merges all splits: no exchange between waves)
    if (lane < p.splits) own = reinterpret_cast<const float4*>(p.part_stat)[row * p.splits + lane];
    constexpr int PER = LP_JOIN_KEYS / 256;
    uint64_t mine[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) mine[j] = tid + j * 256 < n ? p.part_top[row * n + tid + j * 256] : 0;
    if (tid == 0) { count = 0; limit = 0; }
    const LpStat st = lp_across<64>(LpStat{own.x, own.y, own.z}, p.c);
    if (!lp_ordinary(st, p.c)) {
        lp_walk_row<T>(p, row, xt, part, keys);
        return;
    }
    const LpRow q(st.m, lp_log2_sum(st), p.c, false);
    if (tid == 0) lp_finish_row(p, row, xt, st, q);
    if (k == 0) return;
    const int deep = (k + p.splits - 1) / p.splits, nh = deep * p.splits;       // k <= nh < k + splits <= 96
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = tid + j * 256, split = i / k, at = i - split * k;
        if (i < n && at < deep) heads[split * deep + at] = mine[j];
    }
    __syncthreads();
    lp_rank(heads, nh, k, [&](int r, uint64_t key) { if (r == k - 1) limit = key; });
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j)
        if (mine[j] != 0 && mine[j] >= limit) keys[atomicAdd(&count, 1)] = mine[j];     // (any order: lp_rank sorts)
    __syncthreads();
    lp_rank(keys, count, k, [&](int r, uint64_t key) { lp_put_alternative(p, row, r, key, q); });
}

// ---- gradient ----------------------------------------------------------------------------------------------------------
// One pass: each logit read once, each gradient written once, nothing summed (p comes from the forward pass's statistics).
// Bound by memory: 4096 x 32000 bf16, a tenth of the rows ignored, 78 us for 498 MB, 6.4 TB/s, part of the logits still in
// the memory-side cache from the forward pass (a copy of 256 MB reaches 5.4).
struct LpGrad {
    LpRow q; float dent, dlp, k0, inv_t; long long tok; bool zero;
    __device__ __forceinline__ LpGrad(const LogprobArgs& p, long long row, bool short_row)
        : q(p.stat_m[row], p.stat_l2[row], p.c, short_row), tok(lp_token(p, row)) {
        zero = tok == p.ignore || q.empty;
        dlp = p.d_lp ? p.d_lp[row] : 0.f;
        dent = p.d_ent ? p.d_ent[row] : 0.f;
        k0 = (p.d_lse ? p.d_lse[row] : 0.f) - dlp - dent * p.entropy[row];
        if (tok < 0 || tok >= p.vocab) k0 = __builtin_nanf("");
        inv_t = p.inv_t;
        k0 *= inv_t;
        dlp *= inv_t;
        dent *= inv_t * LP_LN2;         // (with log2p below)
    }
    // without the taken token's own dlp
    template <bool NEAR> __device__ __forceinline__ float of(float x) const {
        const float lp = (NEAR ? __builtin_fmaf(x, q.c, -q.r) : (x - q.m) * q.c) - q.l2;
        return lp_exp2(lp) * __builtin_fmaf(-dent, fmaxf(lp, -1000.f), k0);
    }
    __device__ __forceinline__ float at(float x, int i) const {
        if (zero) return 0.f;
        const float d = q.near ? of<true>(x) : of<false>(x);
        return i == tok ? d + dlp : d;
    }
};
template <typename T, int E, int G>
__global__ __launch_bounds__(256) void logprob_short_bwd_kernel(LogprobArgs p) {
    const int l = threadIdx.x & (G - 1);
    const long long step = (long long)gridDim.x * (256 / G);
    for (long long row = (long long)blockIdx.x * (256 / G) + threadIdx.x / G; row < p.rows; row += step) {
        const LpGrad g(p, row, true);
        const T* x = (const T*)p.logits + row * p.ld;
        T* dx = (T*)p.d_logits + row * p.vocab;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = l + e * G;
            if (i < p.vocab) dx[i] = from_f32<T>(g.at(g.zero ? 0.f : to_f32(x[i]), i));
        }
    }
}
#define LP_BWD_U 4      // 16-byte loads in flight per thread (with cached stores 2 / 4 / 8 took 111 / 107 / 115 us)
template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void logprob_long_bwd_kernel(LogprobArgs p, int parts) {
    constexpr int VEC = 16 / sizeof(T), U = LP_BWD_U;
    const int tid = threadIdx.x;
    const long long units = p.rows * parts;
    for (long long unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const long long row = unit / parts;
        const int part = (int)(unit - row * parts);
        const LpGrad g(p, row, false);
        const T* x = (const T*)p.logits + row * p.ld;
        T* dx = (T*)p.d_logits + row * p.vocab;
        const int head = min((int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T), p.vocab);
        const int nvec = (p.vocab - head) / VEC, tail = (p.vocab - head) - nvec * VEC;
        const bool wide = (reinterpret_cast<uintptr_t>(dx + head) & 15) == 0;      // both on the 16-byte grid together
        const int taken = g.zero ? -1 : (int)min(max(g.tok, -1ll), (long long)p.vocab) - head;  // counted from the first vector
        const int v0 = part * (256 * U) + tid;
        vec16<T> q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (v0 + u * 256 < nvec && !g.zero) q[u] = *reinterpret_cast<const vec16<T>*>(x + head + (long long)(v0 + u * 256) * VEC);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int v = v0 + u * 256;
            if (v >= nvec) continue;
            float d[VEC];
            if (g.zero) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) d[j] = 0.f;
            } else if (g.q.near) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) d[j] = g.of<true>(to_f32(q[u].e[j]));
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) d[j] = g.of<false>(to_f32(q[u].e[j]));
            }
            if (taken >= v * VEC && taken < v * VEC + VEC) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) d[j] += taken - v * VEC == j ? g.dlp : 0.f;
            }
            vec16<T> o;
#pragma unroll
            for (int j = 0; j < VEC; ++j) o.e[j] = from_f32<T>(d[j]);
            T* to = dx + head + (long long)v * VEC;
            if (wide) {
                store16<STREAM>(to, o);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) to[j] = o.e[j];
            }
        }
        if (part == 0 && tid < head + tail) {
            const int i = tid < head ? tid : head + nvec * VEC + (tid - head);
            dx[i] = from_f32<T>(g.at(g.zero ? 0.f : to_f32(x[i]), i));
        }
    }
}

// ---- entries -----------------------------------------------------------------------------------------------------------
static bool lp_ok(const LogprobArgs& p) {
    return p.rows >= 0 && p.vocab > 0 && p.vocab < (1 << 30) && p.ld >= 0 && p.top_k >= 0 && p.top_k <= LP_MAX_TOP &&
           p.top_k <= p.vocab;
}
// Parts a long row is cut into: as many as give the card about 1024 workgroups, none shorter than 4096 tokens, and no
// more than the joining launch can order at once.
static int lp_splits(long long rows, int vocab, int top_k) {
    if (vocab <= LP_SHORT || rows >= 512 || rows == 0) return 1;
    long long s = (1024 + rows - 1) / rows;
    if (s > vocab / 4096) s = vocab / 4096;
    if (s > 64) s = 64;
    if (top_k > 0 && s > LP_JOIN_KEYS / top_k) s = LP_JOIN_KEYS / top_k;
    return s < 2 ? 1 : (int)s;
}
PDA_EXPORT int pda_logprob_splits(long long rows, int vocab, int top_k) { return lp_splits(rows, vocab, top_k); }

template <typename T, int E, int G>
static void lp_launch_short(const LogprobArgs& p, bool backward, hipStream_t stream) {
    const long long blocks = (p.rows + 256 / G - 1) / (256 / G);
    const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536)), block(256);
    if (backward) hipLaunchKernelGGL((logprob_short_bwd_kernel<T, E, G>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((logprob_short_kernel<T, E, G>), grid, block, 0, stream, p);
}
template <typename T>
static void lp_launch(const LogprobArgs& p, bool backward, hipStream_t stream) {
    if (p.vocab <= 8) lp_launch_short<T, 1, 8>(p, backward, stream);
    else if (p.vocab <= 32) lp_launch_short<T, 1, 32>(p, backward, stream);
    else if (p.vocab <= 256) lp_launch_short<T, 4, 64>(p, backward, stream);
    else if (p.vocab <= LP_SHORT) lp_launch_short<T, 16, 64>(p, backward, stream);
    else if (backward) {
        constexpr int PART = 256 * LP_BWD_U * (16 / sizeof(T));
        const int parts = (p.vocab + PART - 1) / PART;
        const long long units = p.rows * parts;
        const dim3 grid((unsigned)(units < 1048576 ? units : 1048576)), block(256);
        if (seq_streams(p.rows * p.vocab * (long long)sizeof(T)))
            hipLaunchKernelGGL((logprob_long_bwd_kernel<T, true>), grid, block, 0, stream, p, parts);
        else hipLaunchKernelGGL((logprob_long_bwd_kernel<T, false>), grid, block, 0, stream, p, parts);
    } else {
        const long long units = p.rows * p.splits;
        const dim3 grid((unsigned)(units < 1048576 ? units : 1048576)), block(256);
        if (p.top_k > 0 && p.splits > 1) hipLaunchKernelGGL((logprob_long_kernel<T, true, true>), grid, block, 0, stream, p);
        else if (p.top_k > 0) hipLaunchKernelGGL((logprob_long_kernel<T, true, false>), grid, block, 0, stream, p);
        else hipLaunchKernelGGL((logprob_long_kernel<T, false, false>), grid, block, 0, stream, p);
        if (p.splits > 1) hipLaunchKernelGGL(logprob_join_kernel<T>, dim3((unsigned)p.rows), dim3(256), 0, stream, p);
    }
}
static int lp_run(const LogprobArgs* args, int dtype, bool backward, hipStream_t stream) {
    const LogprobArgs p = *args;
    if (!lp_ok(p) || dtype < SEQ_F32 || dtype > SEQ_F16) return SEQ_REFUSED;
    if (p.rows == 0) return 0;
    if (backward) {
        if (p.stat_m == nullptr || p.stat_l2 == nullptr) return SEQ_REFUSED;
    } else {
        if (p.splits != lp_splits(p.rows, p.vocab, p.top_k)) return SEQ_REFUSED;
        if (p.splits > 1 && (p.part_stat == nullptr || (p.top_k > 0 && p.part_top == nullptr))) return SEQ_REFUSED;
    }
    if (dtype == SEQ_F32) lp_launch<elem_f32>(p, backward, stream);
    else if (dtype == SEQ_BF16) lp_launch<elem_bf16>(p, backward, stream);
    else lp_launch<elem_f16>(p, backward, stream);
    return seq_launched();
}
PDA_EXPORT int pda_logprob(const LogprobArgs* args, int dtype, hipStream_t stream) { return lp_run(args, dtype, false, stream); }
PDA_EXPORT int pda_logprob_bwd(const LogprobArgs* args, int dtype, hipStream_t stream) { return lp_run(args, dtype, true, stream); }
