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
    float* carry;                           // [B][tiles][D]: the state in front of every tile (null: no backward pass)
    float* sums;                            // [B][chunks][2][D]: the chunks' partial recurrences (chunks > 1)
    void* dx; void* dg; float* dh0;
    int B, T, D, logit, mix, reverse;
    int chunks;                             // ScanPlan
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

// A workgroup owns CL * VEC channels of one sequence and walks its steps in tiles of SUB * L: thread (sub, cl) takes L
// consecutive steps of VEC channels.  Within a tile every thread runs its L steps from 0, keeping the products of gates A
// and the partial states H; the threads' ends are scanned across the wave and, through LDS, across the waves; then
// h = A h_in + H.  x and gate are read once and h is written once, in 16-byte accesses; nothing crosses workgroups.
// 32 (16-bit) or 16 (32-bit) channels per workgroup are 64 contiguous bytes per step: the narrowest slab that still uses
// whole sectors, because it is the number of slabs that fills the card.
//
// The backward pass walks the tiles from the end.  It runs the states of a tile again, from the 32-bit state in front of
// the tile that the forward pass left in `carry` (1 / tile length of the traffic), instead of reading h: that is one
// tensor less, and the gate's gradient sees unrounded states.
//
// Where the slabs do not fill the card, the steps are cut into chunks: scan_sum_kernel leaves every chunk's product of
// gates and end state, and each chunk's workgroup folds those in front of it before it starts.  x and gate are then read
// twice.
template <typename T> struct ScanShape { static constexpr int VEC = 16 / sizeof(T), CL = 4, L = 32 / VEC, NT = 256; };
struct ScanRow { static constexpr int VEC = 1, CL = 1, L = 8, NT = 1024; };     // few channels: one per workgroup

struct ScanWhere { int b, chunk, ch0, nch, n; };
template <typename S>
__device__ __forceinline__ ScanWhere scan_where(const ScanArgs& p) {
    const int nslab = (p.D + S::CL * S::VEC - 1) / (S::CL * S::VEC);
    ScanWhere w;
    const int rest = (int)blockIdx.x / nslab;
    w.ch0 = (((int)blockIdx.x - rest * nslab) * S::CL + (int)threadIdx.x % S::CL) * S::VEC;
    w.nch = min(max(p.D - w.ch0, 0), S::VEC);
    w.b = rest / p.chunks;
    w.chunk = rest - w.b * p.chunks;
    w.n = scan_length(p, w.b);
    return w;
}

template <typename T, int VEC> struct Raw { T e[VEC]; };
// VEC channels at `row`: one 16-byte access where the layout allows it, else element by element
template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> scan_load(const T* row, long long cs, bool wide, int nch) {
    Raw<T, VEC> r;
    if (VEC * sizeof(T) == 16 && wide) {
        const vec16<T> v = *reinterpret_cast<const vec16<T>*>(row);
#pragma unroll
        for (int i = 0; i < VEC; ++i) r.e[i] = v.e[i];
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) r.e[i] = i < nch ? row[i * cs] : from_f32<T>(0.f);
    }
    return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void scan_store(T* row, const float (&v)[VEC], bool wide, int nch) {
    if (VEC * sizeof(T) == 16 && wide) {
        vec16<T> o;
#pragma unroll
        for (int i = 0; i < VEC; ++i) o.e[i] = from_f32<T>(v[i]);
        *reinterpret_cast<vec16<T>*>(row) = o;
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (i < nch) row[i] = from_f32<T>(v[i]);
    }
}
template <typename T, int VEC>
__device__ __forceinline__ bool scan_wide(const void* base, const long long (&s)[3], int D) {
    return VEC * sizeof(T) == 16 && s[2] == 1 && D % VEC == 0 && s[0] % VEC == 0 && s[1] % VEC == 0 &&
           (reinterpret_cast<uintptr_t>(base) & 15) == 0;
}

// joins a later part (a, h) behind an earlier one (pa, ph): state -> a (pa state + ph) + h
#define SCAN_JOIN(a, h, pa, ph) do { h = __builtin_fmaf(a, ph, h); a *= pa; } while (0)

// Exclusive scan of the threads' parts over the workgroup, in step order (UP) or against it, applied to the state `in` in
// front of the tile: -> the state in front of this thread's steps; `in` becomes the state behind the tile.
// part: [waves][CL * VEC] in LDS; the caller separates two uses of one buffer by a barrier.
template <typename S, bool UP>
__device__ __forceinline__ void scan_across(float (&A)[S::VEC], float (&H)[S::VEC], float (&in)[S::VEC], float2* part) {
    constexpr int NW = S::NT / 64, W = S::CL * S::VEC;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, cl = threadIdx.x % S::CL;
#pragma unroll
    for (int o = S::CL; o < 64; o <<= 1) {
        const bool on = UP ? lane >= o : lane < 64 - o;
#pragma unroll
        for (int v = 0; v < S::VEC; ++v) {
            const float pa = UP ? __shfl_up(A[v], o, 64) : __shfl_down(A[v], o, 64);
            const float ph = UP ? __shfl_up(H[v], o, 64) : __shfl_down(H[v], o, 64);
            if (on) SCAN_JOIN(A[v], H[v], pa, ph);
        }
    }
    const bool end = UP ? lane >= 64 - S::CL : lane < S::CL;
    if (end) {
#pragma unroll
        for (int v = 0; v < S::VEC; ++v) part[wave * W + cl * S::VEC + v] = make_float2(A[v], H[v]);
    }
    const bool first = UP ? lane < S::CL : lane >= 64 - S::CL;
#pragma unroll
    for (int v = 0; v < S::VEC; ++v) {
        const float pa = UP ? __shfl_up(A[v], S::CL, 64) : __shfl_down(A[v], S::CL, 64);
        const float ph = UP ? __shfl_up(H[v], S::CL, 64) : __shfl_down(H[v], S::CL, 64);
        A[v] = first ? 1.f : pa;
        H[v] = first ? 0.f : ph;
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < S::VEC; ++v) {
        float mine = in[v];
#pragma unroll
        for (int k = 0; k < NW; ++k) {
            const int w = UP ? k : NW - 1 - k;
            if (w == wave) mine = in[v];
            const float2 t = part[w * W + cl * S::VEC + v];
            in[v] = __builtin_fmaf(t.x, in[v], t.y);
        }
        H[v] = __builtin_fmaf(A[v], mine, H[v]);
    }
}

// the state in front of this workgroup's chunk: `in` carried over the chunks before it (UP) or behind it
template <typename S, bool UP>
__device__ __forceinline__ void scan_fold_chunks(const ScanArgs& p, const ScanWhere& w, float (&in)[S::VEC]) {
    const int k0 = UP ? 0 : p.chunks - 1;
    for (int k = k0; k != w.chunk; k += UP ? 1 : -1) {
        const float* s = p.sums + ((long long)w.b * p.chunks + k) * 2 * p.D + w.ch0;
#pragma unroll
        for (int v = 0; v < S::VEC; ++v)
            if (v < w.nch) in[v] = __builtin_fmaf(s[v], in[v], s[p.D + v]);
    }
}

// tiles [first, last) of a chunk
template <typename S> struct ScanTiles {
    static constexpr int SUB = S::NT / S::CL, TILE = SUB * S::L;
    int tiles, per, first, last;
    __device__ __forceinline__ ScanTiles(const ScanArgs& p, int chunk) {
        tiles = (p.T + TILE - 1) / TILE;
        per = (tiles + p.chunks - 1) / p.chunks;
        first = min(chunk * per, tiles);
        last = min(first + per, tiles);
    }
};

template <typename T, typename S, bool LOGIT>
__global__ __launch_bounds__(S::NT) void scan_fwd_kernel(ScanArgs p) {
    constexpr int VEC = S::VEC, L = S::L, TILE = ScanTiles<S>::TILE;
    __shared__ float2 part[2][S::NT / 64 * S::CL * VEC];
    const ScanWhere w = scan_where<S>(p);
    const ScanTiles<S> tl(p, w.chunk);
    const int sub = threadIdx.x / S::CL;
    const bool xw = scan_wide<T, VEC>(p.x, p.xs, p.D), gw = scan_wide<T, VEC>(p.gate, p.gs, p.D), ow = p.D % VEC == 0;
    const T* x = (const T*)p.x + w.b * p.xs[0] + w.ch0 * p.xs[2];
    const T* g = (const T*)p.gate + w.b * p.gs[0] + w.ch0 * p.gs[2];
    T* out = (T*)p.h + (long long)w.b * p.T * p.D + w.ch0;
    float in[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) in[v] = p.h0 && v < w.nch ? p.h0[(long long)w.b * p.D + w.ch0 + v] : 0.f;
    scan_fold_chunks<S, true>(p, w, in);
    for (int tile = tl.first; tile < tl.last; ++tile) {
        const int i0 = tile * TILE + sub * L;
        if (p.carry != nullptr && sub == 0) {
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                if (v < w.nch) p.carry[((long long)w.b * tl.tiles + tile) * p.D + w.ch0 + v] = in[v];
        }
        float A[L][VEC], H[L][VEC];
        if (tile * TILE < w.n) {
            Raw<T, VEC> xr[L], gr[L];
#pragma unroll
            for (int l = 0; l < L; ++l) {
                const int i = min(i0 + l, w.n - 1);
                const long long t = p.reverse ? w.n - 1 - i : i;
                xr[l] = scan_load<T, VEC>(x + t * p.xs[1], p.xs[2], xw && w.nch > 0, w.nch);
                gr[l] = scan_load<T, VEC>(g + t * p.gs[1], p.gs[2], gw && w.nch > 0, w.nch);
            }
            float a[VEC], h[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) { a[v] = 1.f; h[v] = 0.f; }
#pragma unroll
            for (int l = 0; l < L; ++l) {
                const bool on = i0 + l < w.n;
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const Gate ga = gate_of(to_f32(gr[l].e[v]), LOGIT);
                    const float hv = scan_step(h[v], to_f32(xr[l].e[v]), ga, LOGIT, p.mix), av = decayed(a[v], ga, LOGIT);
                    h[v] = on ? hv : h[v];
                    a[v] = on ? av : a[v];
                    A[l][v] = a[v];
                    H[l][v] = h[v];
                }
            }
            scan_across<S, true>(a, h, in, part[tile & 1]);     // (two buffers: one barrier per tile)
#pragma unroll
            for (int l = 0; l < L; ++l) {
#pragma unroll
                for (int v = 0; v < VEC; ++v) H[l][v] = __builtin_fmaf(A[l][v], h[v], H[l][v]);
            }
        }
#pragma unroll
        for (int l = 0; l < L; ++l) {
            const int i = i0 + l;
            if (i >= p.T || w.nch == 0) continue;
            const bool on = i < w.n;
            const long long t = on && p.reverse ? w.n - 1 - i : i;
            float o[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) o[v] = on ? H[l][v] : 0.f;
            scan_store<T, VEC>(out + t * p.D, o, ow, w.nch);
        }
    }
    if (w.chunk == p.chunks - 1 && sub == 0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v)
            if (v < w.nch) p.last[(long long)w.b * p.D + w.ch0 + v] = in[v];
    }
}

template <typename T, typename S, bool LOGIT>
__global__ __launch_bounds__(S::NT) void scan_bwd_kernel(ScanArgs p) {
    constexpr int VEC = S::VEC, L = S::L, TILE = ScanTiles<S>::TILE;
    __shared__ float2 part[2][S::NT / 64 * S::CL * VEC];
    const ScanWhere w = scan_where<S>(p);
    const ScanTiles<S> tl(p, w.chunk);
    const int sub = threadIdx.x / S::CL;
    const bool xw = scan_wide<T, VEC>(p.x, p.xs, p.D) && w.nch > 0, gw = scan_wide<T, VEC>(p.gate, p.gs, p.D) && w.nch > 0,
               dw = scan_wide<T, VEC>(p.dh, p.ds, p.D) && w.nch > 0, ow = p.D % VEC == 0;
    const T* x = (const T*)p.x + w.b * p.xs[0] + w.ch0 * p.xs[2];
    const T* g = (const T*)p.gate + w.b * p.gs[0] + w.ch0 * p.gs[2];
    const T* dh = (const T*)p.dh + w.b * p.ds[0] + w.ch0 * p.ds[2];
    const long long base = (long long)w.b * p.T * p.D + w.ch0;
    float rin[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) rin[v] = p.dlast && v < w.nch ? p.dlast[(long long)w.b * p.D + w.ch0 + v] : 0.f;
    scan_fold_chunks<S, false>(p, w, rin);
    for (int tile = tl.last - 1; tile >= tl.first; --tile) {
        const int i0 = tile * TILE + sub * L;
        float dx[L][VEC], dg[L][VEC];
        if (tile * TILE < w.n) {
            Raw<T, VEC> xr[L], gr[L], dr[L];
#pragma unroll
            for (int l = 0; l < L; ++l) {
                const int i = min(i0 + l, w.n - 1);
                const long long t = p.reverse ? w.n - 1 - i : i;
                gr[l] = scan_load<T, VEC>(g + t * p.gs[1], p.gs[2], gw, w.nch);
                xr[l] = scan_load<T, VEC>(x + t * p.xs[1], p.xs[2], xw, w.nch);
                if (p.dh != nullptr) {
                    dr[l] = scan_load<T, VEC>(dh + t * p.ds[1], p.ds[2], dw, w.nch);
                } else {
#pragma unroll
                    for (int v = 0; v < VEC; ++v) dr[l].e[v] = from_f32<T>(0.f);
                }
            }
            float hin[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                hin[v] = v < w.nch ? p.carry[((long long)w.b * tl.tiles + tile) * p.D + w.ch0 + v] : 0.f;
            // the tile's states again: prev[l] = the state in front of step l, first relative to the thread's start
            float PA[L][VEC], prev[L][VEC], a[VEC], h[VEC];
            Gate ga[L][VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) { a[v] = 1.f; h[v] = 0.f; }
#pragma unroll
            for (int l = 0; l < L; ++l) {
                const bool on = i0 + l < w.n;
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    ga[l][v] = gate_of(to_f32(gr[l].e[v]), LOGIT);
                    PA[l][v] = a[v];
                    prev[l][v] = h[v];
                    const float hv = scan_step(h[v], to_f32(xr[l].e[v]), ga[l][v], LOGIT, p.mix);
                    const float av = decayed(a[v], ga[l][v], LOGIT);
                    h[v] = on ? hv : h[v];
                    a[v] = on ? av : a[v];
                }
            }
            scan_across<S, true>(a, h, hin, part[0]);
#pragma unroll
            for (int l = 0; l < L; ++l) {
#pragma unroll
                for (int v = 0; v < VEC; ++v) prev[l][v] = __builtin_fmaf(PA[l][v], h[v], prev[l][v]);
            }
            // r = a G, carried from later steps to earlier ones; PA and q relative to the thread's end
            float q[L][VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) { a[v] = 1.f; h[v] = 0.f; }
#pragma unroll
            for (int l = L - 1; l >= 0; --l) {
                const bool on = i0 + l < w.n;
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    PA[l][v] = a[v];
                    q[l][v] = h[v];
                    const float hv = decayed(h[v] + to_f32(dr[l].e[v]), ga[l][v], LOGIT), av = decayed(a[v], ga[l][v], LOGIT);
                    h[v] = on ? hv : h[v];
                    a[v] = on ? av : a[v];
                }
            }
            scan_across<S, false>(a, h, rin, part[1]);
#pragma unroll
            for (int l = 0; l < L; ++l) {
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const float xv = to_f32(xr[l].e[v]);
                    const float G = to_f32(dr[l].e[v]) + __builtin_fmaf(PA[l][v], h[v], q[l][v]);
                    float da = G * (p.mix ? prev[l][v] - xv : prev[l][v]);
                    if (LOGIT) da *= ga[l][v].a * ga[l][v].c;
                    dx[l][v] = p.mix ? G * ga[l][v].c : G;
                    dg[l][v] = da;
                }
            }
        }
#pragma unroll
        for (int l = 0; l < L; ++l) {
            const int i = i0 + l;
            if (i >= p.T || w.nch == 0) continue;
            const bool on = i < w.n;
            const long long t = on && p.reverse ? w.n - 1 - i : i;
            float ox[VEC], og[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) { ox[v] = on ? dx[l][v] : 0.f; og[v] = on ? dg[l][v] : 0.f; }
            scan_store<T, VEC>((T*)p.dx + base + t * p.D, ox, ow, w.nch);
            scan_store<T, VEC>((T*)p.dg + base + t * p.D, og, ow, w.nch);
        }
    }
    if (w.chunk == 0 && sub == 0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v)
            if (v < w.nch) p.dh0[(long long)w.b * p.D + w.ch0 + v] = rin[v];
    }
}

// Product of gates and end state of every chunk, from 0 (forward: UP) or of the gradient's recurrence (r = a (dh + r)).
// A thread walks a run of its own through the chunk; the runs are joined once.
template <typename T, typename S, bool LOGIT, bool UP>
__global__ __launch_bounds__(S::NT) void scan_sum_kernel(ScanArgs p) {
    constexpr int VEC = S::VEC, TILE = ScanTiles<S>::TILE, SUB = ScanTiles<S>::SUB, U = 4;
    __shared__ float2 part[S::NT / 64 * S::CL * VEC];
    const ScanWhere w = scan_where<S>(p);
    const ScanTiles<S> tl(p, w.chunk);
    const int sub = threadIdx.x / S::CL;
    const T* v1 = UP ? (const T*)p.x : (const T*)p.dh;
    const long long s0 = UP ? p.xs[0] : p.ds[0], s1 = UP ? p.xs[1] : p.ds[1], s2 = UP ? p.xs[2] : p.ds[2];
    const bool vw = (UP ? scan_wide<T, VEC>(p.x, p.xs, p.D) : scan_wide<T, VEC>(p.dh, p.ds, p.D)) && w.nch > 0;
    const bool gw = scan_wide<T, VEC>(p.gate, p.gs, p.D) && w.nch > 0;
    const T* g = (const T*)p.gate + w.b * p.gs[0] + w.ch0 * p.gs[2];
    v1 += w.b * s0 + w.ch0 * s2;
    const int begin = tl.first * TILE, end = min(tl.last * TILE, w.n), run = (max(end - begin, 0) + SUB - 1) / SUB;
    const int i0 = begin + sub * run, i1 = min(i0 + run, end);
    float a[VEC], h[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) { a[v] = 1.f; h[v] = 0.f; }
    for (int k = i0; k < i1; k += U) {
        Raw<T, VEC> gr[U], vr[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = min(k + u, i1 - 1), i = UP ? j : i0 + (i1 - 1 - j);
            const long long t = p.reverse ? w.n - 1 - i : i;
            gr[u] = scan_load<T, VEC>(g + t * p.gs[1], p.gs[2], gw, w.nch);
            if (UP || p.dh != nullptr) {
                vr[u] = scan_load<T, VEC>(v1 + t * s1, s2, vw, w.nch);
            } else {
#pragma unroll
                for (int v = 0; v < VEC; ++v) vr[u].e[v] = from_f32<T>(0.f);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool on = k + u < i1;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const Gate ga = gate_of(to_f32(gr[u].e[v]), LOGIT);
                const float xv = to_f32(vr[u].e[v]);
                const float hv = UP ? scan_step(h[v], xv, ga, LOGIT, p.mix) : decayed(h[v] + xv, ga, LOGIT);
                const float av = decayed(a[v], ga, LOGIT);
                h[v] = on ? hv : h[v];
                a[v] = on ? av : a[v];
            }
        }
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, cl = threadIdx.x % S::CL;
#pragma unroll
    for (int o = S::CL; o < 64; o <<= 1) {      // thread s takes in the o / CL threads in front of it (UP) or behind it
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const float pa = UP ? __shfl_up(a[v], o, 64) : __shfl_down(a[v], o, 64);
            const float ph = UP ? __shfl_up(h[v], o, 64) : __shfl_down(h[v], o, 64);
            if (UP ? lane >= o : lane < 64 - o) SCAN_JOIN(a[v], h[v], pa, ph);
        }
    }
    if (UP ? lane >= 64 - S::CL : lane < S::CL) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) part[wave * S::CL * VEC + cl * VEC + v] = make_float2(a[v], h[v]);
    }
    __syncthreads();
    if ((int)threadIdx.x < S::CL) {
        float* out = p.sums + ((long long)w.b * p.chunks + w.chunk) * 2 * p.D + w.ch0;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            float ta = 1.f, th = 0.f;
#pragma unroll
            for (int k = 0; k < S::NT / 64; ++k) {
                const float2 t = part[(UP ? k : S::NT / 64 - 1 - k) * S::CL * VEC + cl * VEC + v];
                th = __builtin_fmaf(t.x, th, t.y);
                ta *= t.x;
            }
            if (v < w.nch) { out[v] = ta; out[p.D + v] = th; }
        }
    }
}

// How a problem is cut (the forward and the backward pass of one call agree on it: a function of the sizes alone).
struct ScanPlan { int row, tile, tiles, slabs, chunks; };
static ScanPlan scan_plan(int B, int T, int D, int dtype) {
    ScanPlan k;
    k.row = D < 8;
    const int width = k.row ? 1 : (dtype == SEQ_F32 ? 16 : 32);
    k.tile = k.row ? ScanRow::NT * ScanRow::L : (dtype == SEQ_F32 ? 64 * ScanShape<elem_f32>::L : 64 * ScanShape<elem_bf16>::L);
    k.tiles = (T + k.tile - 1) / k.tile;
    k.slabs = (D + width - 1) / width;
    const long long groups = (long long)B * k.slabs;
    k.chunks = 1;
    if (groups < 256 && k.tiles > 1) {
        const long long want = (512 + groups - 1) / groups;
        k.chunks = (int)(want < k.tiles ? want : k.tiles);
        if (k.chunks > 64) k.chunks = 64;
    }
    return k;
}

static bool scan_ok(const ScanArgs& p) {
    return p.B >= 0 && p.T >= 0 && p.D >= 0 && (long long)p.B * p.D < (1ll << 31) && (unsigned)p.T < (1u << 30);
}

// tiles and chunks of a problem: the caller's carry is [B][tiles][D], its sums [B][chunks][2][D] floats
PDA_EXPORT int pda_scan_plan(int B, int T, int D, int dtype, int* tiles, int* chunks) {
    const ScanPlan k = scan_plan(B, T, D, dtype);
    *tiles = k.tiles;
    *chunks = k.chunks;
    return 0;
}

template <typename T, typename S, bool LOGIT>
static void scan_launch(const ScanArgs& p, const ScanPlan& k, bool backward, hipStream_t stream) {
    const dim3 grid((unsigned)((long long)p.B * k.slabs * k.chunks)), block(S::NT);
    if (!backward) {
        if (k.chunks > 1) hipLaunchKernelGGL((scan_sum_kernel<T, S, LOGIT, true>), grid, block, 0, stream, p);
        hipLaunchKernelGGL((scan_fwd_kernel<T, S, LOGIT>), grid, block, 0, stream, p);
    } else {
        if (k.chunks > 1) hipLaunchKernelGGL((scan_sum_kernel<T, S, LOGIT, false>), grid, block, 0, stream, p);
        hipLaunchKernelGGL((scan_bwd_kernel<T, S, LOGIT>), grid, block, 0, stream, p);
    }
}
template <typename T>
static void scan_dispatch(const ScanArgs& p, const ScanPlan& k, bool backward, hipStream_t stream) {
    if (k.row) {
        if (p.logit) scan_launch<T, ScanRow, true>(p, k, backward, stream);
        else scan_launch<T, ScanRow, false>(p, k, backward, stream);
    } else {
        if (p.logit) scan_launch<T, ScanShape<T>, true>(p, k, backward, stream);
        else scan_launch<T, ScanShape<T>, false>(p, k, backward, stream);
    }
}
static int scan_run(const ScanArgs* args, int dtype, bool backward, hipStream_t stream) {
    ScanArgs p = *args;
    if (!scan_ok(p) || dtype < SEQ_F32 || dtype > SEQ_F16) return SEQ_REFUSED;
    if ((long long)p.B * p.D == 0) return 0;
    const ScanPlan k = scan_plan(p.B, p.T, p.D, dtype);
    if (p.chunks != k.chunks || (k.chunks > 1 && p.sums == nullptr) || (backward && k.tiles > 0 && p.carry == nullptr))
        return SEQ_REFUSED;
    if ((long long)p.B * k.slabs * k.chunks >= (1ll << 31) / ScanRow::NT * 2) return SEQ_REFUSED;
    if (dtype == SEQ_F32) scan_dispatch<elem_f32>(p, k, backward, stream);
    else if (dtype == SEQ_BF16) scan_dispatch<elem_bf16>(p, k, backward, stream);
    else scan_dispatch<elem_f16>(p, k, backward, stream);
    return seq_launched();
}
PDA_EXPORT int pda_scan_fwd(const ScanArgs* args, int dtype, hipStream_t stream) { return scan_run(args, dtype, false, stream); }
PDA_EXPORT int pda_scan_bwd(const ScanArgs* args, int dtype, hipStream_t stream) { return scan_run(args, dtype, true, stream); }

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
