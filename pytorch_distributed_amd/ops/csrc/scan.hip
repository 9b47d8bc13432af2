// Gated linear recurrence over sequences, its backward pass and its single-token step.
//
//   h_t = a_t h_{t-1} + u_t        a = gate | sigmoid(gate),  u = x | (1 - a) x
//   G_t = dh_t + a_{t+1} G_{t+1}   dx = G | (1 - a) G,  da = G h_{t-1} | G (h_{t-1} - x),  dgate = da | da a (1 - a),
//                                  dh0 = a_0 G_0
//
// a h is formed as h - (1 - a) h where a logit gate is above 1/2, with 1 - sigmoid(g) taken as sigmoid(-g): rounding a gate
// next to 1 would be repeated over the whole memory of the recurrence, while 1 - a keeps its own precision (and a does
// below 1/2).  States are 32 bits wide throughout; h is rounded once, where it is stored in x's type.
#include "seq.h"
#pragma clang fp reassociate(off)       // h - c h must not become (1 - c) h

struct ScanArgs {
    const void* x; const void* gate; const void* dh;
    long long xs[3], gs[3], ds[3];          // element strides (batch, step, channel) of x, gate, dh
    const float* h0; const float* dlast;    // [B][D], may be null
    const void* lengths; int len64;         // [B] or null: steps from the length on are no part of a sequence
    void* h; float* last;                   // [B][T][D] contiguous, [B][D]
    float* hist;                            // backward pass: h_{t-1} in 32 bits, [B][T][D]
    void* dx; void* dg; float* dh0;
    int B, T, D, logit, mix, reverse;
};

struct Gate { float a, c; };                // a and c = 1 - a
__device__ __forceinline__ Gate gate_of(float g, int logit) {
    if (!logit) return Gate{g, 1.f - g};
    const float e = __expf(-fabsf(g)), r = 1.f / (1.f + e);     // sigmoid(|g|); the other side is e r
    return g >= 0.f ? Gate{r, e * r} : Gate{e * r, r};
}
__device__ __forceinline__ float decayed(float h, Gate g, int logit) {      // a h
    return logit && g.c <= 0.5f ? __builtin_fmaf(-g.c, h, h) : g.a * h;
}
__device__ __forceinline__ float scan_step(float h, float x, Gate g, int logit, int mix) {
    return decayed(h, g, logit) + (mix ? g.c * x : x);
}
__device__ __forceinline__ int scan_length(const ScanArgs& p, int b) {
    if (p.lengths == nullptr) return p.T;
    const long long n = p.len64 ? ((const long long*)p.lengths)[b] : (long long)((const int*)p.lengths)[b];
    return (int)(n < 0 ? 0 : (n > p.T ? p.T : n));
}

// one thread per sequence and channel
template <typename T>
__global__ __launch_bounds__(64) void scan_fwd_kernel(ScanArgs p) {
    const long long id = (long long)blockIdx.x * 64 + threadIdx.x;
    if (id >= (long long)p.B * p.D) return;
    const int b = (int)(id / p.D), d = (int)(id - (long long)b * p.D), n = scan_length(p, b);
    const T* x = (const T*)p.x + b * p.xs[0] + d * p.xs[2];
    const T* g = (const T*)p.gate + b * p.gs[0] + d * p.gs[2];
    T* out = (T*)p.h + (long long)b * p.T * p.D + d;
    float h = p.h0 ? p.h0[id] : 0.f;
    for (int i = 0; i < n; ++i) {
        const long long t = p.reverse ? n - 1 - i : i;
        h = scan_step(h, to_f32(x[t * p.xs[1]]), gate_of(to_f32(g[t * p.gs[1]]), p.logit), p.logit, p.mix);
        out[t * p.D] = from_f32<T>(h);
    }
    for (long long t = n; t < p.T; ++t) out[t * p.D] = from_f32<T>(0.f);
    p.last[id] = h;
}

template <typename T>
__global__ __launch_bounds__(64) void scan_bwd_kernel(ScanArgs p) {
    const long long id = (long long)blockIdx.x * 64 + threadIdx.x;
    if (id >= (long long)p.B * p.D) return;
    const int b = (int)(id / p.D), d = (int)(id - (long long)b * p.D), n = scan_length(p, b);
    const T* x = (const T*)p.x + b * p.xs[0] + d * p.xs[2];
    const T* g = (const T*)p.gate + b * p.gs[0] + d * p.gs[2];
    const T* dh = p.dh ? (const T*)p.dh + b * p.ds[0] + d * p.ds[2] : nullptr;
    const long long base = (long long)b * p.T * p.D + d;
    float h = p.h0 ? p.h0[id] : 0.f;
    for (int i = 0; i < n; ++i) {
        const long long t = p.reverse ? n - 1 - i : i;
        p.hist[base + t * p.D] = h;
        h = scan_step(h, to_f32(x[t * p.xs[1]]), gate_of(to_f32(g[t * p.gs[1]]), p.logit), p.logit, p.mix);
    }
    float carry = p.dlast ? p.dlast[id] : 0.f;
    for (int i = n - 1; i >= 0; --i) {
        const long long t = p.reverse ? n - 1 - i : i;
        const float xv = to_f32(x[t * p.xs[1]]);
        const Gate ga = gate_of(to_f32(g[t * p.gs[1]]), p.logit);
        const float gr = carry + (dh ? to_f32(dh[t * p.ds[1]]) : 0.f);
        const float prev = p.hist[base + t * p.D];
        float da = gr * (p.mix ? prev - xv : prev);
        if (p.logit) da *= ga.a * ga.c;
        ((T*)p.dx)[base + t * p.D] = from_f32<T>(p.mix ? gr * ga.c : gr);
        ((T*)p.dg)[base + t * p.D] = from_f32<T>(da);
        carry = decayed(gr, ga, p.logit);
    }
    for (long long t = n; t < p.T; ++t) {
        ((T*)p.dx)[base + t * p.D] = from_f32<T>(0.f);
        ((T*)p.dg)[base + t * p.D] = from_f32<T>(0.f);
    }
    if (p.dh0) p.dh0[id] = carry;
}

struct ScanStepArgs {
    const void* x; const void* gate; const float* state; float* state_out; void* h;
    long long xs[2], gs[2], ss[2], os[2];       // element strides (request, channel)
    int B, D, logit, mix;
};
template <typename T>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanStepArgs p) {
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    if (id >= (long long)p.B * p.D) return;
    const int b = (int)(id / p.D), d = (int)(id - (long long)b * p.D);
    const float x = to_f32(((const T*)p.x)[b * p.xs[0] + d * p.xs[1]]);
    const Gate g = gate_of(to_f32(((const T*)p.gate)[b * p.gs[0] + d * p.gs[1]]), p.logit);
    const float h = scan_step(p.state[b * p.ss[0] + d * p.ss[1]], x, g, p.logit, p.mix);
    p.state_out[b * p.os[0] + d * p.os[1]] = h;
    ((T*)p.h)[id] = from_f32<T>(h);
}

static bool scan_ok(const ScanArgs& p) {
    return p.B >= 0 && p.T >= 0 && p.D >= 0 && (long long)p.B * p.D < (1ll << 31);
}
PDA_EXPORT int pda_scan_fwd(const ScanArgs* args, int dtype, hipStream_t stream) {
    const ScanArgs p = *args;
    if (!scan_ok(p)) return SEQ_REFUSED;
    if ((long long)p.B * p.D == 0) return 0;
    const dim3 grid((unsigned)(((long long)p.B * p.D + 63) / 64)), block(64);
    if (dtype == SEQ_F32) hipLaunchKernelGGL(scan_fwd_kernel<elem_f32>, grid, block, 0, stream, p);
    else if (dtype == SEQ_BF16) hipLaunchKernelGGL(scan_fwd_kernel<elem_bf16>, grid, block, 0, stream, p);
    else if (dtype == SEQ_F16) hipLaunchKernelGGL(scan_fwd_kernel<elem_f16>, grid, block, 0, stream, p);
    else return SEQ_REFUSED;
    return seq_launched();
}
PDA_EXPORT int pda_scan_bwd(const ScanArgs* args, int dtype, hipStream_t stream) {
    const ScanArgs p = *args;
    if (!scan_ok(p)) return SEQ_REFUSED;
    if ((long long)p.B * p.D == 0) return 0;
    const dim3 grid((unsigned)(((long long)p.B * p.D + 63) / 64)), block(64);
    if (dtype == SEQ_F32) hipLaunchKernelGGL(scan_bwd_kernel<elem_f32>, grid, block, 0, stream, p);
    else if (dtype == SEQ_BF16) hipLaunchKernelGGL(scan_bwd_kernel<elem_bf16>, grid, block, 0, stream, p);
    else if (dtype == SEQ_F16) hipLaunchKernelGGL(scan_bwd_kernel<elem_f16>, grid, block, 0, stream, p);
    else return SEQ_REFUSED;
    return seq_launched();
}
PDA_EXPORT int pda_scan_step(const ScanStepArgs* args, int dtype, hipStream_t stream) {
    const ScanStepArgs p = *args;
    if (p.B < 0 || p.D < 0 || (long long)p.B * p.D >= (1ll << 31)) return SEQ_REFUSED;
    if ((long long)p.B * p.D == 0) return 0;
    const dim3 grid((unsigned)(((long long)p.B * p.D + 255) / 256)), block(256);
    if (dtype == SEQ_F32) hipLaunchKernelGGL(scan_step_kernel<elem_f32>, grid, block, 0, stream, p);
    else if (dtype == SEQ_BF16) hipLaunchKernelGGL(scan_step_kernel<elem_bf16>, grid, block, 0, stream, p);
    else if (dtype == SEQ_F16) hipLaunchKernelGGL(scan_step_kernel<elem_f16>, grid, block, 0, stream, p);
    else return SEQ_REFUSED;
    return seq_launched();
}
