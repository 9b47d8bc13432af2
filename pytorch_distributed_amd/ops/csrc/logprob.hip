// Log-probabilities of given tokens with entropy and the best alternatives, and their gradient.
//
//   z = x / T,  m = max x,  s = sum exp((x - m) / T),  u = sum exp((x - m) / T) (x - m) / T
//   logprob = (x_t - m) / T - log s,   entropy = log s - u / s,   logsumexp = m / T + log s
//   dx_i = (p_i (dlse - dlp - dent (logp_i + entropy)) + dlp [i = t]) / T,   p_i = exp(logp_i)
//
// (m, log s) is what the forward pass keeps for the backward pass: their sum would round p by |lse| 2^-24.
// A logit of -inf is a masked token: p = 0, no share in the entropy, gradient 0.  A row with nothing but -inf: logprob
// and logsumexp -inf, entropy 0, gradient 0.  An ignored row is not read: 0 everywhere, alternatives -1.
// A token outside the vocabulary gives NaN (log-probability and gradient row) and reads nothing.
#include "seq.h"
#pragma clang fp reassociate(off)       // (x - m) / T stays what it is: x / T and m / T alone may overflow

struct LogprobArgs {
    const void* logits; long long ld; long long rows; int vocab;
    const void* tokens; int tok64; long long ignore;
    float inv_t; int top_k;
    float* logprob; float* entropy; float* lse;         // [rows]
    float* stat_m; float* stat_ls;                      // [rows], for the backward pass
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
__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t t = __shfl_xor((unsigned long long)v, o, 64);
        v = t > v ? t : v;
    }
    return v;
}

// softmax statistics of a part of a row: running maximum m, and s, u relative to it, with u in units of log 2:
// s = sum 2^d, u = sum 2^d d, d = (x - m) c, c = log2(e) / T
struct LpStat { float m, s, u; };
#define LP_LN2 0.693147180559945309f
#define LP_LOG2E 1.44269504088896341f
__device__ __forceinline__ float lp_exp2(float d) { return __builtin_amdgcn_exp2f(d); }
// `st` seen from the maximum m >= st.m (no part of it may turn into 0 * inf: the shift is cut off where 2^shift is 0)
__device__ __forceinline__ LpStat lp_shift(LpStat st, float m, float c) {
    const float d = st.m == m ? 0.f : fmaxf((st.m - m) * c, -1.0e20f), e = lp_exp2(d);
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
    const float m = st.m == -INFINITY ? 0.f : st.m;
    float s = 0.f, u = 0.f;
#pragma unroll
    for (int i = 0; i < NX; ++i) {
        const float d = (x[i] - m) * c, e = lp_exp2(d);
        s += e;                                             // (NaN for a NaN, and for +inf - +inf)
        u = __builtin_fmaf(e, fmaxf(d, -1000.f), u);        // (0 for -inf)
    }
    st.s += s;
    st.u += u;
}
template <int G>
__device__ __forceinline__ LpStat lp_across(LpStat st, float c) {   // over groups of G lanes
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1)
        st = lp_merge(st, LpStat{__shfl_xor(st.m, o, 64), __shfl_xor(st.s, o, 64), __shfl_xor(st.u, o, 64)}, c);
    return st;
}

__device__ __forceinline__ void lp_ignored_row(const LogprobArgs& p, long long row) {
    p.logprob[row] = 0.f; p.entropy[row] = 0.f; p.lse[row] = 0.f;
    p.stat_m[row] = 0.f; p.stat_ls[row] = 0.f;
    for (int k = 0; k < p.top_k; ++k) { p.top_lp[row * p.top_k + k] = 0.f; p.top_id[row * p.top_k + k] = -1; }
}
__device__ __forceinline__ bool lp_empty(LpStat st) { return st.m == -INFINITY && st.s == 0.f; }
__device__ __forceinline__ bool lp_not_a_number(LpStat st) { return st.m == INFINITY || st.s != st.s; }
__device__ __forceinline__ float lp_log_sum(LpStat st) { return lp_not_a_number(st) ? __builtin_nanf("") : __logf(st.s); }
template <typename T>
__device__ __forceinline__ void lp_finish_row(const LogprobArgs& p, long long row, long long tok, LpStat st) {
    const T* x = (const T*)p.logits + row * p.ld;
    const bool empty = lp_empty(st);
    const float ls = empty ? 0.f : lp_log_sum(st);
    float lp = __builtin_nanf("");
    if (tok >= 0 && tok < p.vocab) lp = empty ? -INFINITY : (to_f32(x[tok]) - st.m) * p.inv_t - ls;
    p.logprob[row] = lp;
    p.entropy[row] = empty ? 0.f : ls - st.u / st.s * LP_LN2;
    p.lse[row] = empty ? -INFINITY : st.m * p.inv_t + ls;
    p.stat_m[row] = st.m;
    p.stat_ls[row] = ls;
}
template <typename T>
__device__ __forceinline__ void lp_put_alternative(const LogprobArgs& p, long long row, int k, uint64_t key, LpStat st, float ls) {
    const int id = lp_key_index(key);
    const float x = to_f32(((const T*)p.logits + row * p.ld)[id]);
    p.top_id[row * p.top_k + k] = id;
    p.top_lp[row * p.top_k + k] = lp_empty(st) ? -INFINITY : (x - st.m) * p.inv_t - ls;
}

// The alternatives of a row that holds NaN, by top_k walks over it (float comparisons cannot order those): whole workgroup
template <typename T>
__device__ void lp_walk_top(const LogprobArgs& p, long long row, LpStat st, float ls, uint64_t* best) {
    const T* x = (const T*)p.logits + row * p.ld;
    const int tid = threadIdx.x;
    uint64_t last = ~0ull;
    for (int k = 0; k < p.top_k; ++k) {
        uint64_t b = 0;
        for (int i = tid; i < p.vocab; i += 256) {
            const uint64_t key = lp_key(to_f32(x[i]), i);
            if (key < last && key > b) b = key;
        }
        b = wave_max_u64(b);
        __syncthreads();            // (the previous round's reads of best[])
        if ((tid & 63) == 0) best[tid >> 6] = b;
        __syncthreads();
        last = best[0];
        for (int w = 1; w < 4; ++w) last = best[w] > last ? best[w] : last;
        if (tid == 0) lp_put_alternative<T>(p, row, k, last, st, ls);
    }
    __syncthreads();
}
// The top_k largest of n distinct keys in LDS, by counting what is above each: whole workgroup
template <typename F>
__device__ __forceinline__ void lp_rank(const uint64_t* keys, int n, int top_k, F put) {
    for (int i = threadIdx.x; i < n; i += 256) {
        const uint64_t mine = keys[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += keys[j] > mine ? 1 : 0;
        if (above < top_k && mine != 0) put(above, mine);
    }
}

// ---- rows of up to LP_SHORT tokens: G lanes hold E tokens each --------------------------------------------------------
template <typename T, int E, int G>
__global__ __launch_bounds__(256) void logprob_short_kernel(LogprobArgs p) {
    const int lane = threadIdx.x & 63, l = lane & (G - 1);
    const float c = p.inv_t * LP_LOG2E;
    const long long step = (long long)gridDim.x * (256 / G);
    // (every lane of a wave takes every round: the shuffles want them all)
    for (long long r0 = (long long)blockIdx.x * (256 / G); r0 < p.rows; r0 += step) {
        const long long row = r0 + threadIdx.x / G;
        const bool on = row < p.rows;
        const long long tok = on ? lp_token(p, row) : p.ignore;
        const bool live = on && tok != p.ignore;
        const T* x = (const T*)p.logits + (live ? row : 0) * p.ld;
        float xs[E], bm = -INFINITY;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = l + e * G;
            xs[e] = live && i < p.vocab ? to_f32(x[i]) : -INFINITY;
            bm = fmaxf(bm, xs[e]);
        }
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) bm = fmaxf(bm, __shfl_xor(bm, o, 64));
        LpStat st{-INFINITY, 0.f, 0.f};
        lp_add<E>(st, xs, bm, c);
        st = lp_across<G>(st, c);
        if (l == 0 && on) {
            if (live) lp_finish_row<T>(p, row, tok, st);
            else lp_ignored_row(p, row);
        }
        const float ls = lp_log_sum(st);
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
            if (l == 0 && live) lp_put_alternative<T>(p, row, k, last, st, ls);
        }
    }
}

// ---- long rows ---------------------------------------------------------------------------------------------------------
// A workgroup reads a row (or one of its splits) once, in 16-byte loads, four in flight per thread.  Each thread keeps
// running statistics, shifted once per 32 or 16 values.  The alternatives: each wave keeps its best keys sorted over its
// lanes.  A value is looked at again only if it passes the wave's k-th best, which the first batch sets to the k-th largest
// of the lanes' maxima; a wave of n values then inserts about k (2 + ln(n / 2048)) of them, each by a ballot and a shift.
template <typename T>
__global__ __launch_bounds__(256) void logprob_long_kernel(LogprobArgs p) {
    constexpr int VEC = 16 / sizeof(T), U = 4, NX = U * VEC;
    __shared__ LpStat part[4];
    __shared__ uint64_t keys[4 * LP_MAX_TOP];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const float c = p.inv_t * LP_LOG2E;
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
        // head: tokens in front of the first 16-byte boundary; behind the vectors the tail
        const int head = min((int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T), p.vocab);
        const int nvec = (p.vocab - head) / VEC, tail = (p.vocab - head) - nvec * VEC;
        const int per = (nvec + p.splits - 1) / p.splits, v0 = min(split * per, nvec), v1 = min(v0 + per, nvec);
        LpStat st{-INFINITY, 0.f, 0.f};
        uint64_t list = 0;                  // lane i: the wave's i-th best key so far
        float lim = -INFINITY;              // what a value has to reach (or, `strict`, to exceed) to get into it
        bool strict = false, filled = false;
        auto offer = [&](float v, int index, bool valid) {
            const bool pass = valid && (strict ? v > lim : v >= lim);
            uint64_t todo = __ballot(pass);
            if (todo == 0) return;
            const uint64_t key = lp_key(v, index);
            while (todo) {
                const int src = __builtin_ctzll(todo);
                todo &= todo - 1;
                const uint64_t k = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(key >> 32), src) << 32) |
                                   (uint32_t)__builtin_amdgcn_readlane((int)key, src);
                const uint64_t above = __ballot(list > k);
                const int pos = __builtin_popcountll(above);
                if (pos >= p.top_k) continue;
                const uint64_t up = __shfl_up((unsigned long long)list, 1, 64);
                list = lane < pos ? list : (lane == pos ? k : up);
            }
            const uint64_t kth = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(list >> 32), p.top_k - 1) << 32) |
                                 (uint32_t)__builtin_amdgcn_readlane((int)list, p.top_k - 1);
            if (kth != 0) {
                uint32_t b = (uint32_t)(kth >> 32);
                b = (b & 0x80000000u) ? (b & 0x7fffffffu) : ~b;
                const float v = __builtin_bit_cast(float, b);
                if (!filled || v > lim) { lim = v; strict = false; }
                filled = true;
            }
        };
        bool first = true;
        for (int b = v0; b < v1; b += 256 * U) {
            float xs[NX], bm = -INFINITY;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int v = b + u * 256 + tid;
                if (v < v1) {
                    const vec16<T> q = *reinterpret_cast<const vec16<T>*>(x + head + (long long)v * VEC);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) xs[u * VEC + j] = to_f32(q.e[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) xs[u * VEC + j] = -INFINITY;
                }
            }
#pragma unroll
            for (int i = 0; i < NX; ++i) bm = fmaxf(bm, xs[i]);
            lp_add<NX>(st, xs, bm, c);
            if (p.top_k == 0) continue;
            if (first) {        // the k-th largest of the lanes' maxima: k values reach it
                first = false;
                float t = bm;
                int above = 0;
                for (int o = 0; o < 64; ++o) {
                    const float other = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, t), o));
                    above += (other > t || (other == t && o < lane)) ? 1 : 0;
                }
                const uint64_t who = __ballot(above == p.top_k - 1);
                lim = who ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, t), __builtin_ctzll(who)))
                          : -INFINITY;
            } else if (filled) {
                strict = true;  // an equal value of a later batch has a higher index
            }
            if (__ballot(strict ? bm > lim : bm >= lim) == 0) continue;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int v = b + u * 256 + tid;
#pragma unroll
                for (int j = 0; j < VEC; ++j) offer(xs[u * VEC + j], head + v * VEC + j, v < v1);
            }
        }
        if (split == 0 && wave == 0 && head + tail > 0) {       // at most 14 single tokens
            const bool valid = lane < head + tail;
            const int i = lane < head ? lane : head + nvec * VEC + (lane - head);
            float xs[1] = {valid ? to_f32(x[i]) : -INFINITY};
            lp_add<1>(st, xs, xs[0], c);
            strict = false;
            if (p.top_k > 0) offer(xs[0], i, valid);
        }
        st = lp_across<64>(st, c);
        if (lane == 0) part[wave] = st;
        if (lane < p.top_k) keys[wave * p.top_k + lane] = list;
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
        } else {
            if (tid == 0) lp_finish_row<T>(p, row, tok, st);
            const float ls = lp_log_sum(st);
            if (p.top_k > 0) {
                if (lp_not_a_number(st)) lp_walk_top<T>(p, row, st, ls, keys);
                else lp_rank(keys, 4 * p.top_k, p.top_k, [&](int k, uint64_t key) { lp_put_alternative<T>(p, row, k, key, st, ls); });
            }
        }
        __syncthreads();            // part[] and keys[] are reused by the next unit
    }
}
// joins the splits of a row
template <typename T>
__global__ __launch_bounds__(256) void logprob_join_kernel(LogprobArgs p) {
    __shared__ uint64_t keys[1024];
    const long long row = blockIdx.x;
    const long long tok = lp_token(p, row);
    const int tid = threadIdx.x, lane = tid & 63, n = p.splits * p.top_k;
    if (tok == p.ignore) {
        if (tid == 0) lp_ignored_row(p, row);
        return;
    }
    const float c = p.inv_t * LP_LOG2E;
    LpStat st{-INFINITY, 0.f, 0.f};         // (every wave merges all splits: no exchange between waves)
    for (int s = lane; s < p.splits; s += 64) {
        const float* q = p.part_stat + (row * p.splits + s) * 4;
        st = lp_merge(st, LpStat{q[0], q[1], q[2]}, c);
    }
    st = lp_across<64>(st, c);
    const float ls = lp_log_sum(st);
    if (tid == 0) lp_finish_row<T>(p, row, tok, st);
    if (p.top_k == 0) return;
    if (lp_not_a_number(st)) {
        lp_walk_top<T>(p, row, st, ls, keys);
        return;
    }
    for (int i = tid; i < n; i += 256) keys[i] = p.part_top[row * n + i];
    __syncthreads();
    lp_rank(keys, n, p.top_k, [&](int k, uint64_t key) { lp_put_alternative<T>(p, row, k, key, st, ls); });
}

// ---- gradient ----------------------------------------------------------------------------------------------------------
// One pass: each logit read once, each gradient written once.
struct LpGrad { float m, ls, dent, dlp, k0, inv_t; long long tok; bool zero; };
__device__ __forceinline__ LpGrad lp_grad_of(const LogprobArgs& p, long long row) {
    LpGrad g;
    g.tok = lp_token(p, row);
    g.m = p.stat_m[row];
    g.ls = p.stat_ls[row];
    g.zero = g.tok == p.ignore || (g.m == -INFINITY && g.ls == g.ls);       // ignored, or nothing but -inf
    g.dlp = p.d_lp ? p.d_lp[row] : 0.f;
    g.dent = p.d_ent ? p.d_ent[row] : 0.f;
    g.k0 = (p.d_lse ? p.d_lse[row] : 0.f) - g.dlp - g.dent * p.entropy[row];
    if (g.tok < 0 || g.tok >= p.vocab) g.k0 = __builtin_nanf("");
    g.inv_t = p.inv_t;
    return g;
}
__device__ __forceinline__ float lp_grad(const LpGrad& g, float x, int i) {
    const float lp = (x - g.m) * g.inv_t - g.ls, pr = lp_exp2(lp * LP_LOG2E);
    float d = pr * (g.k0 - g.dent * fmaxf(lp, -1000.f));
    if (i == g.tok) d += g.dlp;
    return g.zero ? 0.f : d * g.inv_t;
}
template <typename T, int E, int G>
__global__ __launch_bounds__(256) void logprob_short_bwd_kernel(LogprobArgs p) {
    const int l = threadIdx.x & (G - 1);
    const long long step = (long long)gridDim.x * (256 / G);
    for (long long row = (long long)blockIdx.x * (256 / G) + threadIdx.x / G; row < p.rows; row += step) {
        const LpGrad g = lp_grad_of(p, row);
        const T* x = (const T*)p.logits + row * p.ld;
        T* dx = (T*)p.d_logits + row * p.vocab;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = l + e * G;
            if (i < p.vocab) dx[i] = from_f32<T>(lp_grad(g, g.zero ? 0.f : to_f32(x[i]), i));
        }
    }
}
template <typename T>
__global__ __launch_bounds__(256) void logprob_long_bwd_kernel(LogprobArgs p, int parts) {
    constexpr int VEC = 16 / sizeof(T), U = 4;
    const int tid = threadIdx.x;
    const long long units = p.rows * parts;
    for (long long unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const long long row = unit / parts;
        const int part = (int)(unit - row * parts);
        const LpGrad g = lp_grad_of(p, row);
        const T* x = (const T*)p.logits + row * p.ld;
        T* dx = (T*)p.d_logits + row * p.vocab;
        const int head = min((int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T), p.vocab);
        const int nvec = (p.vocab - head) / VEC, tail = (p.vocab - head) - nvec * VEC;
        const bool wide = (reinterpret_cast<uintptr_t>(dx + head) & 15) == 0;      // both on the 16-byte grid together
        const int v0 = part * (256 * U);
        vec16<T> q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int v = v0 + u * 256 + tid;
            if (v < nvec && !g.zero) q[u] = *reinterpret_cast<const vec16<T>*>(x + head + (long long)v * VEC);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int v = v0 + u * 256 + tid;
            if (v >= nvec) continue;
            vec16<T> o;
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                o.e[j] = from_f32<T>(lp_grad(g, g.zero ? 0.f : to_f32(q[u].e[j]), head + v * VEC + j));
            T* to = dx + head + (long long)v * VEC;
            if (wide) {
                *reinterpret_cast<vec16<T>*>(to) = o;
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) to[j] = o.e[j];
            }
        }
        if (part == 0 && tid < head + tail) {
            const int i = tid < head ? tid : head + nvec * VEC + (tid - head);
            dx[i] = from_f32<T>(lp_grad(g, g.zero ? 0.f : to_f32(x[i]), i));
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
    if (top_k > 0 && s > 1024 / top_k) s = 1024 / top_k;
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
        constexpr int PART = 256 * 4 * (16 / sizeof(T));
        const int parts = (p.vocab + PART - 1) / PART;
        const long long units = p.rows * parts;
        hipLaunchKernelGGL(logprob_long_bwd_kernel<T>, dim3((unsigned)(units < 1048576 ? units : 1048576)), dim3(256), 0,
                           stream, p, parts);
    } else {
        const long long units = p.rows * p.splits;
        hipLaunchKernelGGL(logprob_long_kernel<T>, dim3((unsigned)(units < 1048576 ? units : 1048576)), dim3(256), 0, stream, p);
        if (p.splits > 1) hipLaunchKernelGGL(logprob_join_kernel<T>, dim3((unsigned)p.rows), dim3(256), 0, stream, p);
    }
}
static int lp_run(const LogprobArgs* args, int dtype, bool backward, hipStream_t stream) {
    const LogprobArgs p = *args;
    if (!lp_ok(p) || dtype < SEQ_F32 || dtype > SEQ_F16) return SEQ_REFUSED;
    if (p.rows == 0) return 0;
    if (!backward) {
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
