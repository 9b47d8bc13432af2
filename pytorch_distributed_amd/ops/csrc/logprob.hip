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
};
#define LP_MAX_TOP 32

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

// softmax statistics of a part of a row: running maximum m, s and u relative to it
struct LpStat { float m, s, u; };
__device__ __forceinline__ LpStat lp_merge(LpStat a, LpStat b, float inv_t) {
    const float m = fmaxf(a.m, b.m);
    if (m == -INFINITY) return LpStat{m, a.s + b.s, a.u + b.u};
    const float da = a.m == m ? 0.f : fmaxf((a.m - m) * inv_t, -3.0e38f);
    const float db = b.m == m ? 0.f : fmaxf((b.m - m) * inv_t, -3.0e38f);
    const float ea = __expf(da), eb = __expf(db);
    LpStat r;
    r.m = m;
    r.s = a.s * ea + b.s * eb;
    r.u = (ea > 0.f ? ea * (a.u + da * a.s) : 0.f) + (eb > 0.f ? eb * (b.u + db * b.s) : 0.f);
    if (a.s != a.s || b.s != b.s) r.s = a.s + b.s;
    return r;
}
__device__ __forceinline__ void lp_add(LpStat& st, float x, float inv_t) {
    if (x > st.m) {
        st = lp_merge(st, LpStat{x, 1.f, 0.f}, inv_t);
    } else {
        const float d = (x - st.m) * inv_t, e = st.m == -INFINITY ? (x == x ? 0.f : x) : __expf(d);
        st.s += e;
        st.u += e > 0.f ? e * d : 0.f;
    }
}
__device__ __forceinline__ LpStat lp_wave(LpStat st, float inv_t) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        st = lp_merge(st, LpStat{__shfl_xor(st.m, o, 64), __shfl_xor(st.s, o, 64), __shfl_xor(st.u, o, 64)}, inv_t);
    return st;
}

__device__ __forceinline__ void lp_ignored_row(const LogprobArgs& p, long long row) {
    p.logprob[row] = 0.f; p.entropy[row] = 0.f; p.lse[row] = 0.f;
    p.stat_m[row] = 0.f; p.stat_ls[row] = 0.f;
    for (int k = 0; k < p.top_k; ++k) { p.top_lp[row * p.top_k + k] = 0.f; p.top_id[row * p.top_k + k] = -1; }
}
__device__ __forceinline__ bool lp_empty(LpStat st) { return st.m == -INFINITY && st.s == 0.f; }
__device__ __forceinline__ float lp_log_sum(LpStat st) { return st.m == INFINITY ? __builtin_nanf("") : __logf(st.s); }
template <typename T>
__device__ __forceinline__ void lp_finish_row(const LogprobArgs& p, long long row, long long tok, LpStat st) {
    const T* x = (const T*)p.logits + row * p.ld;
    const bool empty = lp_empty(st);
    const float ls = empty ? 0.f : lp_log_sum(st);
    float lp = __builtin_nanf("");
    if (tok >= 0 && tok < p.vocab) lp = empty ? -INFINITY : (to_f32(x[tok]) - st.m) * p.inv_t - ls;
    p.logprob[row] = lp;
    p.entropy[row] = empty ? 0.f : ls - st.u / st.s;
    p.lse[row] = empty ? -INFINITY : st.m * p.inv_t + ls;
    p.stat_m[row] = st.m;
    p.stat_ls[row] = ls;
}
__device__ __forceinline__ float lp_alternative(float x, LpStat st, float ls, float inv_t) {
    return lp_empty(st) ? -INFINITY : (x - st.m) * inv_t - ls;
}

// one workgroup per row; the alternatives by top_k walks over the row
template <typename T>
__global__ __launch_bounds__(256) void logprob_row_kernel(LogprobArgs p) {
    __shared__ LpStat part[4];
    __shared__ uint64_t best[4];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const long long tok = lp_token(p, row);
        if (tok == p.ignore) {
            if (tid == 0) lp_ignored_row(p, row);
            continue;
        }
        const T* x = (const T*)p.logits + row * p.ld;
        LpStat st{-INFINITY, 0.f, 0.f};
        for (int i = tid; i < p.vocab; i += 256) lp_add(st, to_f32(x[i]), p.inv_t);
        st = lp_wave(st, p.inv_t);
        if (lane == 0) part[wave] = st;
        __syncthreads();
        st = lp_merge(lp_merge(part[0], part[1], p.inv_t), lp_merge(part[2], part[3], p.inv_t), p.inv_t);
        if (tid == 0) lp_finish_row<T>(p, row, tok, st);
        const float ls = lp_log_sum(st);
        uint64_t last = ~0ull;
        for (int k = 0; k < p.top_k; ++k) {
            uint64_t b = 0;
            for (int i = tid; i < p.vocab; i += 256) {
                const uint64_t key = lp_key(to_f32(x[i]), i);
                if (key < last && key > b) b = key;
            }
            b = wave_max_u64(b);
            __syncthreads();        // (the previous round's reads of best[])
            if (lane == 0) best[wave] = b;
            __syncthreads();
            last = best[0];
            for (int w = 1; w < 4; ++w) last = best[w] > last ? best[w] : last;
            if (tid == 0) {
                const int id = lp_key_index(last);
                p.top_id[row * p.top_k + k] = id;
                p.top_lp[row * p.top_k + k] = lp_alternative(to_f32(x[id]), st, ls, p.inv_t);
            }
        }
        __syncthreads();            // part[] and best[] are reused by the next row
    }
}

template <typename T>
__global__ __launch_bounds__(256) void logprob_bwd_kernel(LogprobArgs p) {
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const long long tok = lp_token(p, row);
        const T* x = (const T*)p.logits + row * p.ld;
        T* dx = (T*)p.d_logits + row * p.vocab;
        const float m = p.stat_m[row], ls = p.stat_ls[row];
        if (tok == p.ignore || (m == -INFINITY && ls == ls)) {     // ignored, or nothing but -inf
            for (int i = threadIdx.x; i < p.vocab; i += 256) dx[i] = from_f32<T>(0.f);
            continue;
        }
        const float dlp = p.d_lp ? p.d_lp[row] : 0.f, dent = p.d_ent ? p.d_ent[row] : 0.f;
        float k0 = (p.d_lse ? p.d_lse[row] : 0.f) - dlp - dent * p.entropy[row];
        if (tok < 0 || tok >= p.vocab) k0 = __builtin_nanf("");
        for (int i = threadIdx.x; i < p.vocab; i += 256) {
            const float lp = (to_f32(x[i]) - m) * p.inv_t - ls, pr = __expf(lp);
            float g = pr * (k0 - dent * fmaxf(lp, -1000.f));
            if (i == tok) g += dlp;
            dx[i] = from_f32<T>(g * p.inv_t);
        }
    }
}

static bool lp_ok(const LogprobArgs& p) {
    return p.rows >= 0 && p.vocab > 0 && p.ld >= 0 && p.top_k >= 0 && p.top_k <= LP_MAX_TOP && p.top_k <= p.vocab;
}

PDA_EXPORT int pda_logprob(const LogprobArgs* args, int dtype, hipStream_t stream) {
    const LogprobArgs p = *args;
    if (!lp_ok(p)) return SEQ_REFUSED;
    if (p.rows == 0) return 0;
    const dim3 grid((unsigned)(p.rows < 65536 ? p.rows : 65536)), block(256);
    if (dtype == SEQ_F32) hipLaunchKernelGGL(logprob_row_kernel<elem_f32>, grid, block, 0, stream, p);
    else if (dtype == SEQ_BF16) hipLaunchKernelGGL(logprob_row_kernel<elem_bf16>, grid, block, 0, stream, p);
    else if (dtype == SEQ_F16) hipLaunchKernelGGL(logprob_row_kernel<elem_f16>, grid, block, 0, stream, p);
    else return SEQ_REFUSED;
    return seq_launched();
}

PDA_EXPORT int pda_logprob_bwd(const LogprobArgs* args, int dtype, hipStream_t stream) {
    const LogprobArgs p = *args;
    if (!lp_ok(p)) return SEQ_REFUSED;
    if (p.rows == 0) return 0;
    const dim3 grid((unsigned)(p.rows < 65536 ? p.rows : 65536)), block(256);
    if (dtype == SEQ_F32) hipLaunchKernelGGL(logprob_bwd_kernel<elem_f32>, grid, block, 0, stream, p);
    else if (dtype == SEQ_BF16) hipLaunchKernelGGL(logprob_bwd_kernel<elem_bf16>, grid, block, 0, stream, p);
    else if (dtype == SEQ_F16) hipLaunchKernelGGL(logprob_bwd_kernel<elem_f16>, grid, block, 0, stream, p);
    else return SEQ_REFUSED;
    return seq_launched();
}
