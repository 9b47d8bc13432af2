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
#include <type_traits>
#pragma clang fp reassociate(off)       // h - c h must not become (1 - c) h

struct ScanArgs {
    const void* x; const void* gate; const void* dh;
    long long xs[3], gs[3], ds[3];          // element strides (batch, step, channel) of x, gate, dh
    const float* h0; const float* dlast;    // [B][D], may be null
    const void* lengths; int len64;         // [B] or null: steps from the length on are no part of a sequence
    void* h; float* last;                   // [B][T][D] contiguous, [B][D]
    float* carry;                           // [B][carries][D]: the state in front of every carry_len steps (null: not kept)
    float* sums;                            // [B][chunks][2][D]: the chunks' partial recurrences (chunks > 1)
    void* dx; void* dg; float* dh0;
    int B, T, D, logit, mix, reverse;
    int chunks, chunk_len, carry_len, carries;      // ScanPlan
};

// k = a where a <= 1/2, else -c (its sign bit says which, also that of -0: a step that does not exist, and a gate saturated at
// 1, have c = 0); c = 1 - a.  For decay gates k = a.
struct Gate { float k, c; };
template <bool LOGIT>
__device__ __forceinline__ Gate gate_of(float g) {
    if (!LOGIT) return Gate{g, 1.f - g};
    const float e = __builtin_amdgcn_exp2f(g * 1.44269504088896341f), c = __builtin_amdgcn_rcpf(1.f + e);     // a = e c
    return Gate{c <= 0.5f ? -c : e * c, c};
}
__device__ __forceinline__ float acc_fma(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double acc_fma(double a, double b, double c) { return __builtin_fma(a, b, c); }
template <bool LOGIT, typename Acc>
__device__ __forceinline__ Acc decayed(Acc h, Gate g) {             // a h
    return LOGIT ? acc_fma((Acc)g.k, h, __builtin_bit_cast(int, g.k) < 0 ? h : (Acc)0) : (Acc)g.k * h;
}
template <bool LOGIT, bool MIX, typename Acc>
__device__ __forceinline__ Acc scan_step(Acc h, float x, Gate g) {
    return MIX ? acc_fma((Acc)g.c, (Acc)x, decayed<LOGIT>(h, g)) : decayed<LOGIT>(h, g) + (Acc)x;
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
// 64 (16-bit) or 32 (32-bit) channels per workgroup are 128 contiguous bytes per step, a whole cache line: slabs of 64 bytes
// give twice the workgroups, but every line is then fetched by two of them (1 x 65521 x 512 fp32 in an earlier form of these
// kernels: 98 + 152 us forward against 64 + 107).
//
// The backward pass walks the tiles from the end.  It runs the states of a tile again, from the 32-bit state in front of
// the tile that the forward pass left in `carry` (1 / tile length of the traffic), instead of reading h: that is one
// tensor less, and the gate's gradient sees unrounded states.
//
// Where the slabs do not fill the card, the steps are cut into chunks: scan_sum_kernel leaves every chunk's product of
// gates and end state, and each chunk's workgroup folds those in front of it before it starts.  x and gate are then read
// twice.
//
// Measured at 8 x 2048 x 2048 bf16, sigmoid gates, leaky average, lengths of 1024 to 2048 (256 workgroups, one per CU):
// forward 53 us for 168 MB (3.2 TB/s), backward 98 us for 285 MB (2.9 TB/s).  Loads, arithmetic and stores of a tile follow
// one another on a CU that holds one workgroup (backward: one wave per SIMD, which issues about 2500 vector instructions a
// tile, 10000 of the tile's 15000 cycles), and the longest sequence sets the time.  At 1 x 65521 x 512 fp32 (16 slabs, 256
// workgroups): 56 + 75 us forward for 268 + 403 MB, 47 + 142 us backward for 268 + 671 MB, 4.7 to 5.7 TB/s: bound by memory, a
// third of it the second reading.
#define SCAN_CL 8
// scan_sum_kernel, either direction: 128 / 256 / 512 threads take 65 + 62 / 54 + 47 / 60 + 50 us (forward + backward) at
// 1 x 65521 x 512 fp32
template <typename T> struct ScanSum {
    typedef float Acc;
    static constexpr int VEC = 16 / sizeof(T), CL = SCAN_CL, L = 1, NT = 256;
};
// a forward tile holds a whole number of backward tiles: the forward pass leaves the state in front of each of those
template <typename T> struct ScanFwd {
    typedef float Acc;
    typedef ScanSum<T> Sum;
    static constexpr int VEC = 16 / sizeof(T), CL = SCAN_CL, L = 32 / VEC, NT = 512;
};
template <typename T> struct ScanBwd {
    typedef float Acc;
    static constexpr int VEC = 16 / sizeof(T), CL = SCAN_CL, L = 32 / VEC, NT = 256;
};
// Fewer than 8 channels: one sequence of one channel per workgroup, of 16 waves or of one.  Latency is all that counts
// there, so a workgroup's states and products are 64 bits wide: a constant gate such as 0.99 rounds every product the same
// way, which left 5e-7 of 12500 discounted returns in 32 bits.  What passes through memory is rounded to 32: the sums of
// chunks, once for every 8192 steps or more, and the state that the backward pass starts a tile from.
// (16 x 12500 fp32 returns: 8.7 us, of which the loads of the two tiles that a workgroup walks are most; 8 forward + 21
// backward with a gradient, 11 for 1 x 25000, 10 + 5 forward and 10 + 14 backward for 1 x 65536 in 8 chunks.)
struct ScanRow { typedef double Acc; typedef ScanRow Sum; static constexpr int VEC = 1, CL = 1, L = 8, NT = 1024; };
struct ScanWave { typedef double Acc; typedef void Sum; static constexpr int VEC = 1, CL = 1, L = 8, NT = 64; };
// The lanes of a wave: SW consecutive ones hold consecutive runs of steps of one group of VEC channels, so that a scan
// over steps moves along a DPP row.
template <typename S> struct ScanLane {
    static constexpr int SW = 64 / S::CL, W = S::CL * S::VEC;
    int cl, sub;
    __device__ __forceinline__ ScanLane() : cl(((int)threadIdx.x & 63) / SW), sub((int)(threadIdx.x >> 6) * SW + ((int)threadIdx.x & (SW - 1))) {}
};

// How a kernel touches memory: element by element (any strides), in 16-byte accesses (contiguous channels on the 16-byte
// grid), or so with stores past the caches.  All of a call's tensors decide together: rows of 2047 bf16 channels, or one
// stride-0 gradient (that of h.sum()), take the first way.  8 x 2048 x 2048 bf16, no lengths: 49 us forward and 102 backward,
// with the gradient of h.sum() 248 backward, with 2047 channels 153 and 354; 8 x 2048 fp32 with 1024 / 1023 channels 41 + 78 /
// 75 + 152.
#define SCAN_ANY 0
#define SCAN_WIDE 1
#define SCAN_STREAM 2

struct ScanWhere { int b, chunk, ch0, nch, n; };
template <typename S>
__device__ __forceinline__ ScanWhere scan_where(const ScanArgs& p) {
    const int nslab = (p.D + S::CL * S::VEC - 1) / (S::CL * S::VEC);
    ScanWhere w;
    const int id = blockIdx.x;
    const int rest = id / nslab;
    w.ch0 = ((id - rest * nslab) * S::CL + ScanLane<S>().cl) * S::VEC;
    w.nch = min(max(p.D - w.ch0, 0), S::VEC);
    w.b = rest / p.chunks;
    w.chunk = rest - w.b * p.chunks;
    w.n = scan_length(p, w.b);
    return w;
}

// VEC elements in whole registers (16-bit ones in pairs)
template <typename T, int VEC> struct Raw {
    static constexpr int PER = VEC == 1 ? 1 : 4 / (int)sizeof(T), NW = VEC / PER;
    uint32_t w[NW];
    __device__ __forceinline__ void put(int i, T v) {
        const uint32_t bits = bits_of(v);
        w[i / PER] = i % PER == 0 ? bits : (w[i / PER] | bits << 16);
    }
    __device__ __forceinline__ float get(int i) const { return value_of<T>(w[i / PER], i % PER); }
};
// VEC channels at `row`: one 16-byte access where the layout allows it, else element by element
template <typename T, int VEC, bool WIDE>
__device__ __forceinline__ Raw<T, VEC> scan_load(const T* row, long long cs, int nch) {
    Raw<T, VEC> r;
    if constexpr (WIDE) {
        const uint4 v = *reinterpret_cast<const uint4*>(row);
        r.w[0] = v.x;
        r.w[1] = v.y;
        r.w[2] = v.z;
        r.w[3] = v.w;
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) r.put(i, i < nch ? row[i * cs] : from_f32<T>(0.f));
    }
    return r;
}
// What a step that does not exist reads: it leaves the state as it is (a = 1, u = 0).
template <typename T, int VEC, bool LOGIT>
__device__ __forceinline__ Raw<T, VEC> scan_no_gate() {
    Raw<T, VEC> r;
#pragma unroll
    for (int v = 0; v < VEC; ++v) r.put(v, from_f32<T>(LOGIT ? INFINITY : 1.f));
    return r;
}
template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> scan_nothing() {
    Raw<T, VEC> r;
#pragma unroll
    for (int v = 0; v < VEC; ++v) r.put(v, from_f32<T>(0.f));
    return r;
}

// The L steps from i0 of one tensor, in the recurrence's order; steps from n on read `none`.  A thread of a one-channel scan
// whose steps are contiguous takes four 32-bit values at a time: element by element its loads would pass the L1 cache
// (64 KB of steps in flight per workgroup) once each.
template <typename T, typename S, int MODE>
__device__ __forceinline__ void scan_fetch(Raw<T, S::VEC> (&r)[S::L], const T* base, long long ts, long long cs, int i0, int n,
                                           int nch, bool reverse, const Raw<T, S::VEC>& none) {
    constexpr int L = S::L;
    if constexpr (S::VEC == 1 && MODE == SCAN_WIDE) {
        if (i0 + L <= n) {
            const T* from = base + (reverse ? n - i0 - L : i0);
#pragma unroll
            for (int l = 0; l < L; l += 4) {
                uint32_t w[4];
                __builtin_memcpy(w, from + l, 16);      // (on the 4-byte grid)
#pragma unroll
                for (int j = 0; j < 4; ++j) r[reverse ? L - 1 - l - j : l + j].w[0] = w[j];
            }
            return;
        }
    }
#pragma unroll
    for (int l = 0; l < L; ++l) {
        const int i = i0 + l;
        if (i < n && nch > 0) r[l] = scan_load<T, S::VEC, MODE != SCAN_ANY && S::VEC != 1>(base + (reverse ? n - 1 - i : i) * ts, cs, nch);
        else r[l] = none;
    }
}
// on = false stores zeros (whole words of them: half the selects of 16-bit elements one by one)
template <typename T, int VEC, int MODE>
__device__ __forceinline__ void scan_store(T* row, const float (&v)[VEC], int nch, bool on) {
    if constexpr (MODE != SCAN_ANY && VEC != 1) {
        vec16<T> o;
#pragma unroll
        for (int i = 0; i < VEC; ++i) o.e[i] = from_f32<T>(v[i]);
        seq_u32x4 w = __builtin_bit_cast(seq_u32x4, o);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = on ? w[i] : 0u;
        store16<MODE == SCAN_STREAM>(row, __builtin_bit_cast(vec16<T>, w));
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (i < nch) row[i] = from_f32<T>(on ? v[i] : 0.f);
    }
}
// joins a later part (a, h) behind an earlier one (pa, ph): state -> a (pa state + ph) + h
#define SCAN_JOIN(a, h, pa, ph) do { h = acc_fma(a, ph, h); a *= pa; } while (0)
template <typename Acc> struct alignas(2 * sizeof(Acc)) Part { Acc a, h; };

template <int CTRL, int BANKS>
__device__ __forceinline__ float dpp_move(float none, float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v),
                                                                 CTRL, 0xf, BANKS, false));
}
template <int CTRL, int BANKS>
__device__ __forceinline__ double dpp_move(double none, double v) {
    const uint2 n = __builtin_bit_cast(uint2, none), w = __builtin_bit_cast(uint2, v);
    return __builtin_bit_cast(double, make_uint2(__builtin_amdgcn_update_dpp(n.x, w.x, CTRL, 0xf, BANKS, false),
                                                 __builtin_amdgcn_update_dpp(n.y, w.y, CTRL, 0xf, BANKS, false)));
}
template <int O, bool UP, int BANKS = 0xf, typename Acc>
__device__ __forceinline__ Acc dpp_shift(Acc none, Acc v) {             // lane i of a row of 16 gets lane i -+ O's, or `none`
    return dpp_move<(UP ? 0x110 : 0x100) + O, BANKS>(none, v);
}
template <int O, bool UP>
__device__ __forceinline__ float dpp_neighbour(float v) {               // the same without `none`: lanes that have no such neighbour are
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), (UP ? 0x110 : 0x100) + O, 0xf, 0xf, true));
}                                                                       // replaced by the caller (saves a move each)
template <bool UP, typename Acc>
__device__ __forceinline__ Acc wave_shift(Acc v) {                      // lane i of the wave gets lane i -+ 1's
    return dpp_move<UP ? 0x138 : 0x130, 0xf>((Acc)0, v);
}
__device__ __forceinline__ float scan_lane(float v, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
__device__ __forceinline__ double scan_lane(double v, int lane) {
    const uint2 w = __builtin_bit_cast(uint2, v);
    return __builtin_bit_cast(double, make_uint2(__builtin_amdgcn_readlane(w.x, lane), __builtin_amdgcn_readlane(w.y, lane)));
}
template <int O, int SW, bool UP, typename Acc>
__device__ __forceinline__ void scan_lanes_step(Acc& A, Acc& H) {
    if constexpr (O < SW) {
        constexpr int BANKS = SW == 8 && O == 4 ? (UP ? 0xa : 0x5) : 0xf;      // (the lanes of a group that have a partner)
        Acc pa, ph;
        if constexpr (SW < 16 && BANKS == 0xf) {
            const int i = threadIdx.x & (SW - 1);
            const bool on = UP ? i >= O : i < SW - O;
            pa = dpp_neighbour<O, UP>(A);
            ph = dpp_neighbour<O, UP>(H);
            pa = on ? pa : (Acc)1;
            ph = on ? ph : (Acc)0;
        } else {
            pa = dpp_shift<O, UP, BANKS>((Acc)1, A);
            ph = dpp_shift<O, UP, BANKS>((Acc)0, H);
        }
        SCAN_JOIN(A, H, pa, ph);
    }
}
// inclusive over the SW lanes of a channel group
template <int SW, bool UP, typename Acc>
__device__ __forceinline__ void scan_lanes(Acc& A, Acc& H) {
    static_assert(SW == 8 || SW == 16 || SW == 64, "");
    scan_lanes_step<1, SW, UP>(A, H);
    scan_lanes_step<2, SW, UP>(A, H);
    scan_lanes_step<4, SW, UP>(A, H);
    scan_lanes_step<8, SW, UP>(A, H);
    if constexpr (SW == 64) {       // the four rows of 16
        const int row = (threadIdx.x >> 4) & 3, at = UP ? row : 3 - row;
        Acc pa = 1, ph = 0, ta = 1, th = 0;
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const int end = UP ? 16 * k + 15 : 48 - 16 * k;
            const Acc a = scan_lane(A, end), h = scan_lane(H, end);
            th = acc_fma(a, th, h);
            ta *= a;
            pa = at > k ? ta : pa;
            ph = at > k ? th : ph;
        }
        SCAN_JOIN(A, H, pa, ph);
    }
}
// Exclusive scan of the threads' parts over the workgroup, in step order (UP) or against it, applied to the state `in` in
// front of the tile: H becomes the state in front of this thread's steps, `in` the state behind the tile.
// part: [waves][CL * VEC] in LDS; the caller separates two uses of one buffer by a barrier.
template <typename S, bool UP, typename Acc>
__device__ __forceinline__ void scan_across(Acc (&A)[S::VEC], Acc (&H)[S::VEC], Acc (&in)[S::VEC], Part<Acc>* part) {
    constexpr int NW = S::NT / 64, W = S::CL * S::VEC, SW = ScanLane<S>::SW;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), cl = ScanLane<S>().cl, i = threadIdx.x & (SW - 1);
#pragma unroll
    for (int v = 0; v < S::VEC; ++v) scan_lanes<SW, UP>(A[v], H[v]);
    if (i == (UP ? SW - 1 : 0)) {
#pragma unroll
        for (int v = 0; v < S::VEC; ++v) part[wave * W + cl * S::VEC + v] = Part<Acc>{A[v], H[v]};
    }
    const bool first = i == (UP ? 0 : SW - 1);
#pragma unroll
    for (int v = 0; v < S::VEC; ++v) {      // exclusive: the neighbour's
        Acc pa, ph;
        if constexpr (SW <= 16) {
            pa = dpp_neighbour<1, UP>(A[v]);
            ph = dpp_neighbour<1, UP>(H[v]);
        } else {
            pa = wave_shift<UP>(A[v]);
            ph = wave_shift<UP>(H[v]);
        }
        A[v] = first ? (Acc)1 : pa;
        H[v] = first ? (Acc)0 : ph;
    }
    __syncthreads();
    Acc mine[S::VEC];
    const Part<Acc>* t = part + (UP ? 0 : (NW - 1) * W) + cl * S::VEC;
    const int at = UP ? wave : NW - 1 - wave;
#pragma unroll
    for (int k = 0; k < NW; ++k, t += UP ? W : -W) {
        if (k == at) {
#pragma unroll
            for (int v = 0; v < S::VEC; ++v) mine[v] = in[v];
        }
#pragma unroll
        for (int v = 0; v < S::VEC; ++v) in[v] = acc_fma(t[v].a, in[v], t[v].h);
    }
#pragma unroll
    for (int v = 0; v < S::VEC; ++v) H[v] = acc_fma(A[v], mine[v], H[v]);
}

// `in` carried over the chunks in front of this workgroup's (UP) or behind it: one chunk per thread row and round
template <typename S, bool UP, typename Acc>
__device__ __forceinline__ void scan_fold_chunks(const ScanArgs& p, const ScanWhere& w, Acc (&in)[S::VEC], Part<Acc>* part) {
    constexpr int SUB = S::NT / S::CL;
    const int count = UP ? w.chunk : p.chunks - 1 - w.chunk, sub = ScanLane<S>().sub;
    for (int base = 0; base < count; base += SUB) {
        const int j = base + (UP ? sub : SUB - 1 - sub), k = UP ? j : p.chunks - 1 - j;
        Acc A[S::VEC], H[S::VEC];
#pragma unroll
        for (int v = 0; v < S::VEC; ++v) {
            const bool on = j < count && v < w.nch;
            const float* s = p.sums + ((long long)w.b * p.chunks + (on ? k : 0)) * 2 * p.D + (on ? w.ch0 + v : 0);
            A[v] = on ? s[0] : 1.f;
            H[v] = on ? s[p.D] : 0.f;
        }
        scan_across<S, UP>(A, H, in, part);
        __syncthreads();        // (part is used again)
    }
}

// tiles [first, last) of a chunk
template <typename S> struct ScanTiles {
    static constexpr int SUB = S::NT / S::CL, TILE = SUB * S::L;
    int first, last;
    __device__ __forceinline__ ScanTiles(const ScanArgs& p, int chunk) {
        const int begin = min(chunk * p.chunk_len, p.T), end = min(begin + p.chunk_len, p.T);      // chunk_len: whole tiles
        first = begin / TILE;
        last = (end + TILE - 1) / TILE;
        if (begin >= end) last = first;
    }
};

// The next tile's loads are issued as soon as this tile's registers are free, over the joins and the stores.  (A second set
// of registers, loaded a whole tile ahead, took 65 us instead of 54 at 8 x 2048 x 2048 bf16: 240 registers a thread.)
template <typename T, typename S, bool LOGIT, bool MIX, int MODE>
__global__ __launch_bounds__(S::NT) void scan_fwd_kernel(ScanArgs p) {
    typedef typename S::Acc Acc;
    constexpr int VEC = S::VEC, L = S::L, TILE = ScanTiles<S>::TILE;
    __shared__ Part<Acc> part[2][S::NT / 64 * S::CL * VEC];
    const ScanWhere w = scan_where<S>(p);
    const ScanTiles<S> tl(p, w.chunk);
    const int sub = ScanLane<S>().sub;
    const T* x = (const T*)p.x + w.b * p.xs[0] + w.ch0 * p.xs[2];
    const T* g = (const T*)p.gate + w.b * p.gs[0] + w.ch0 * p.gs[2];
    T* out = (T*)p.h + (long long)w.b * p.T * p.D + w.ch0;
    struct Set { Raw<T, VEC> x[L], g[L]; };
    auto fetch = [&](Set& s, int tile) {
        const int i0 = tile * TILE + sub * L;
        scan_fetch<T, S, MODE>(s.x, x, p.xs[1], p.xs[2], i0, w.n, w.nch, p.reverse, scan_nothing<T, VEC>());
        scan_fetch<T, S, MODE>(s.g, g, p.gs[1], p.gs[2], i0, w.n, w.nch, p.reverse, scan_no_gate<T, VEC, LOGIT>());
    };
    Set s;
    fetch(s, tl.first);
    Acc in[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) in[v] = p.h0 && v < w.nch ? p.h0[(long long)w.b * p.D + w.ch0 + v] : 0.f;
    scan_fold_chunks<S, true>(p, w, in, part[0]);
    for (int tile = tl.first; tile < tl.last; ++tile) {
        const int i0 = tile * TILE + sub * L;
        Acc A[L][VEC], H[L][VEC], a[VEC], h[VEC];
        const bool some = tile * TILE < w.n;
        if (some) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) { a[v] = 1; h[v] = 0; }
#pragma unroll
            for (int l = 0; l < L; ++l) {
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const Gate ga = gate_of<LOGIT>(s.g[l].get(v));
                    h[v] = scan_step<LOGIT, MIX>(h[v], s.x[l].get(v), ga);
                    a[v] = decayed<LOGIT>(a[v], ga);
                    A[l][v] = a[v];
                    H[l][v] = h[v];
                }
            }
            if (tile + 1 < tl.last) fetch(s, tile + 1);
            scan_across<S, true>(a, h, in, part[tile & 1]);     // (two buffers: one barrier per tile)
        } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) h[v] = 0;
        }
        if (p.carry != nullptr && i0 % p.carry_len == 0 && i0 < p.T) {
            float* c = p.carry + ((long long)w.b * p.carries + i0 / p.carry_len) * p.D + w.ch0;
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                if (v < w.nch) c[v] = (float)h[v];
        }
        if constexpr (VEC == 1 && MODE == SCAN_WIDE) {
            if (i0 + L <= w.n && p.D == 1) {
                float o[L];
#pragma unroll
                for (int l = 0; l < L; ++l) o[p.reverse ? L - 1 - l : l] = (float)acc_fma(A[l][0], h[0], H[l][0]);
                __builtin_memcpy(out + (p.reverse ? w.n - i0 - L : i0), o, sizeof(o));      // (32-bit elements)
                continue;
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
            for (int v = 0; v < VEC; ++v) o[v] = (float)acc_fma(A[l][v], h[v], H[l][v]);
            scan_store<T, VEC, MODE>(out + t * p.D, o, w.nch, on);
        }
    }
    if (w.chunk == p.chunks - 1 && sub == 0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v)
            if (v < w.nch) p.last[(long long)w.b * p.D + w.ch0 + v] = (float)in[v];
    }
}

template <typename T, typename S, bool LOGIT, bool MIX, int MODE>
__global__ __launch_bounds__(S::NT) void scan_bwd_kernel(ScanArgs p) {
    typedef typename S::Acc Acc;
    constexpr int VEC = S::VEC, L = S::L, TILE = ScanTiles<S>::TILE;
    __shared__ Part<Acc> part[2][S::NT / 64 * S::CL * VEC];
    const ScanWhere w = scan_where<S>(p);
    const ScanTiles<S> tl(p, w.chunk);
    const int sub = ScanLane<S>().sub;
    const T* x = (const T*)p.x + w.b * p.xs[0] + w.ch0 * p.xs[2];
    const T* g = (const T*)p.gate + w.b * p.gs[0] + w.ch0 * p.gs[2];
    const T* dh = (const T*)p.dh + w.b * p.ds[0] + w.ch0 * p.ds[2];
    const long long base = (long long)w.b * p.T * p.D + w.ch0;
    struct Set { Raw<T, VEC> x[L], g[L], d[L]; float hin[VEC]; };
    auto fetch = [&](Set& s, int tile) {
        const int i0 = tile * TILE + sub * L, n = w.n;
        scan_fetch<T, S, MODE>(s.g, g, p.gs[1], p.gs[2], i0, n, w.nch, p.reverse, scan_no_gate<T, VEC, LOGIT>());
        scan_fetch<T, S, MODE>(s.x, x, p.xs[1], p.xs[2], i0, n, w.nch, p.reverse, scan_nothing<T, VEC>());
        scan_fetch<T, S, MODE>(s.d, dh, p.ds[1], p.ds[2], i0, p.dh != nullptr ? n : 0, w.nch, p.reverse, scan_nothing<T, VEC>());
#pragma unroll
        for (int v = 0; v < VEC; ++v)
            s.hin[v] = v < w.nch ? p.carry[((long long)w.b * p.carries + tile) * p.D + w.ch0 + v] : 0.f;
    };
    Set s;
    if (tl.last > tl.first) fetch(s, tl.last - 1);
    Acc rin[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) rin[v] = p.dlast && v < w.nch ? p.dlast[(long long)w.b * p.D + w.ch0 + v] : 0.f;
    scan_fold_chunks<S, false>(p, w, rin, part[0]);
    for (int tile = tl.last - 1; tile >= tl.first; --tile) {
        const int i0 = tile * TILE + sub * L;
        // per step: G = q + P r_in, dx = G c or G, dgate = G wt
        Acc P[L][VEC], q[L][VEC], a[VEC], h[VEC];
        float wt[L][VEC], cc[L][VEC];
        const bool some = tile * TILE < w.n;
        if (some) {
            Gate ga[L][VEC];
            Acc hin[VEC];
            // the tile's states again: wt = the state in front of step l (- x), first relative to the thread's start
#pragma unroll
            for (int v = 0; v < VEC; ++v) { a[v] = 1; h[v] = 0; hin[v] = s.hin[v]; }
#pragma unroll
            for (int l = 0; l < L; ++l) {
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const float xv = s.x[l].get(v);
                    ga[l][v] = gate_of<LOGIT>(s.g[l].get(v));
                    P[l][v] = a[v];
                    q[l][v] = MIX ? h[v] - (Acc)xv : h[v];
                    h[v] = scan_step<LOGIT, MIX>(h[v], xv, ga[l][v]);
                    a[v] = decayed<LOGIT>(a[v], ga[l][v]);
                }
            }
            scan_across<S, true>(a, h, hin, part[0]);
#pragma unroll
            for (int l = 0; l < L; ++l) {
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    wt[l][v] = (float)acc_fma(P[l][v], h[v], q[l][v]);
                    if (LOGIT) wt[l][v] *= decayed<LOGIT>(ga[l][v].c, ga[l][v]);      // a c
                }
            }
            // r = a G, carried from later steps to earlier ones; P and q relative to the thread's end
#pragma unroll
            for (int v = 0; v < VEC; ++v) { a[v] = 1; h[v] = 0; }
#pragma unroll
            for (int l = L - 1; l >= 0; --l) {
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    P[l][v] = a[v];
                    q[l][v] = h[v] + (Acc)s.d[l].get(v);
                    h[v] = decayed<LOGIT>(q[l][v], ga[l][v]);
                    a[v] = decayed<LOGIT>(a[v], ga[l][v]);
                    if (MIX) cc[l][v] = ga[l][v].c;
                }
            }
        }
        if (tile > tl.first) fetch(s, tile - 1);
        if (some) scan_across<S, false>(a, h, rin, part[1]);
#pragma unroll
        for (int l = 0; l < L; ++l) {
            const int i = i0 + l;
            if (i >= p.T || w.nch == 0) continue;
            const bool on = i < w.n;
            const long long t = on && p.reverse ? w.n - 1 - i : i;
            float ox[VEC], og[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float G = (float)acc_fma(P[l][v], h[v], q[l][v]);
                ox[v] = MIX ? G * cc[l][v] : G;
                og[v] = G * wt[l][v];
            }
            scan_store<T, VEC, MODE>((T*)p.dx + base + t * p.D, ox, w.nch, on);
            scan_store<T, VEC, MODE>((T*)p.dg + base + t * p.D, og, w.nch, on);
        }
    }
    if (w.chunk == 0 && sub == 0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v)
            if (v < w.nch) p.dh0[(long long)w.b * p.D + w.ch0 + v] = (float)rin[v];
    }
}

// Product of gates and end state of every chunk, from 0 (forward: UP) or of the gradient's recurrence (r = a (dh + r)).
// A thread walks a run of its own through the chunk; the runs are joined once.
template <typename T, typename S, bool LOGIT, bool MIX, bool UP, int MODE>
__global__ __launch_bounds__(S::NT) void scan_sum_kernel(ScanArgs p) {
    typedef typename S::Acc Acc;
    constexpr int VEC = S::VEC, SUB = ScanTiles<S>::SUB, U = 4;
    __shared__ Part<Acc> part[S::NT / 64 * S::CL * VEC];
    const ScanWhere w = scan_where<S>(p);
    const int sub = ScanLane<S>().sub;
    const T* v1 = UP ? (const T*)p.x : (const T*)p.dh;
    const long long s0 = UP ? p.xs[0] : p.ds[0], s1 = UP ? p.xs[1] : p.ds[1], s2 = UP ? p.xs[2] : p.ds[2];
    const T* g = (const T*)p.gate + w.b * p.gs[0] + w.ch0 * p.gs[2];
    v1 += w.b * s0 + w.ch0 * s2;
    const int begin = min(w.chunk * p.chunk_len, p.T), end = min(min(begin + p.chunk_len, p.T), w.n), run = (max(end - begin, 0) + SUB - 1) / SUB;
    const int i0 = begin + sub * run, i1 = w.nch > 0 ? min(i0 + run, end) : i0;
    Acc a[VEC], h[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) { a[v] = 1; h[v] = 0; }
    for (int k = i0; k < i1; k += U) {
        Raw<T, VEC> gr[U], vr[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = min(k + u, i1 - 1), i = UP ? j : i0 + (i1 - 1 - j);
            const long long t = p.reverse ? w.n - 1 - i : i;
            gr[u] = scan_load<T, VEC, MODE != SCAN_ANY && VEC != 1>(g + t * p.gs[1], p.gs[2], w.nch);
            if (UP || p.dh != nullptr) {
                vr[u] = scan_load<T, VEC, MODE != SCAN_ANY && VEC != 1>(v1 + t * s1, s2, w.nch);
            } else {
#pragma unroll
                for (int v = 0; v < VEC; ++v) vr[u].put(v, from_f32<T>(0.f));
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool on = k + u < i1;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const Gate ga = gate_of<LOGIT>(gr[u].get(v));
                const float xv = vr[u].get(v);
                const Acc hv = UP ? scan_step<LOGIT, MIX>(h[v], xv, ga) : decayed<LOGIT>(h[v] + (Acc)xv, ga);
                const Acc av = decayed<LOGIT>(a[v], ga);
                h[v] = on ? hv : h[v];
                a[v] = on ? av : a[v];
            }
        }
    }
    constexpr int SW = ScanLane<S>::SW;
    const int wave = threadIdx.x >> 6, cl = ScanLane<S>().cl, li = threadIdx.x & (SW - 1);
#pragma unroll
    for (int v = 0; v < VEC; ++v) scan_lanes<SW, UP>(a[v], h[v]);
    if (li == (UP ? SW - 1 : 0)) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) part[wave * S::CL * VEC + cl * VEC + v] = Part<Acc>{a[v], h[v]};
    }
    __syncthreads();
    if (wave == 0 && li == 0) {
        float* out = p.sums + ((long long)w.b * p.chunks + w.chunk) * 2 * p.D + w.ch0;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            Acc ta = 1, th = 0;
#pragma unroll
            for (int k = 0; k < S::NT / 64; ++k) {
                const Part<Acc> t = part[(UP ? k : S::NT / 64 - 1 - k) * S::CL * VEC + cl * VEC + v];
                th = acc_fma(t.a, th, t.h);
                ta *= t.a;
            }
            if (v < w.nch) { out[v] = (float)ta; out[p.D + v] = (float)th; }
        }
    }
}

// How a problem is cut (the forward and the backward pass of one call agree on it: a function of the sizes alone).
//
// Chunks: where the slabs are fewer than the 256 CUs and there are at least SCAN_CHUNK_TILES tiles, the steps are cut into
// as many chunks as give every CU one workgroup.  Forward + backward with the cut against without, sigmoid gates, leaky
// average: 8 tiles, 32 slabs (1 x 2048 x 2048 bf16) 19 + 25 us against 42 + 87; 8 tiles, 128 slabs 46 + 69 against 43 + 89;
// 16 tiles, 16 slabs (1 x 8192 x 512 fp32) 22 + 29 against more than 77 + 160.  With fewer tiles what it gains depends on the
// slabs: 4 tiles, 128 slabs (4 x 1024 x 2048 bf16) 29 + 40 against 25 + 47, 4 tiles, 16 slabs (1 x 2048 x 512 fp32) 18 + 26
// against 28 + 56: the rule leaves both as they are.  From 129 to 255 slabs a cut would give some CUs two workgroups: not taken.  (Chunks
// taken in turns that fit the memory-side cache, so that the second reading finds them there: 323 us against 326 us at
// 1 x 65521 x 512 fp32 with gradient, not worth it.)
#define SCAN_CHUNK_TILES 8
#define SCAN_ROUND 256
struct ScanPlan { int kind, slabs, chunks, chunk_len, carry_len, carries; };
#define SCAN_KIND_SLAB 0
#define SCAN_KIND_ROW 1
#define SCAN_KIND_WAVE 2
template <typename F, typename B>
static void scan_cut(ScanPlan& k, long long groups, int T) {
    static_assert(ScanTiles<F>::TILE % ScanTiles<B>::TILE == 0, "whole backward tiles");
    const int tile = ScanTiles<F>::TILE, tiles = (T + tile - 1) / tile;
    k.carry_len = ScanTiles<B>::TILE;
    k.carries = (T + k.carry_len - 1) / k.carry_len;
    k.chunks = 1;
    k.chunk_len = (tiles > 0 ? tiles : 1) * tile;
    if (groups <= 0 || groups >= SCAN_ROUND || tiles < SCAN_CHUNK_TILES) return;
    const int want = (int)(SCAN_ROUND / groups < tiles ? SCAN_ROUND / groups : tiles), per = (tiles + want - 1) / want;
    k.chunks = (tiles + per - 1) / per;
    k.chunk_len = per * tile;
}
static ScanPlan scan_plan(int B, int T, int D, int dtype) {
    ScanPlan k;
    const int width = D < 8 ? 1 : SCAN_CL * (dtype == SEQ_F32 ? 4 : 8);
    k.slabs = (D + width - 1) / width;
    const long long groups = (long long)B * k.slabs;
    k.kind = D >= 8 ? SCAN_KIND_SLAB : (T <= 4 * ScanTiles<ScanWave>::TILE || groups >= 1024) ? SCAN_KIND_WAVE : SCAN_KIND_ROW;
    if (k.kind == SCAN_KIND_ROW) scan_cut<ScanRow, ScanRow>(k, groups, T);
    else if (k.kind == SCAN_KIND_WAVE) scan_cut<ScanWave, ScanWave>(k, groups, T);
    else if (dtype == SEQ_F32) scan_cut<ScanFwd<elem_f32>, ScanBwd<elem_f32>>(k, groups, T);
    else scan_cut<ScanFwd<elem_bf16>, ScanBwd<elem_bf16>>(k, groups, T);
    return k;
}

static bool scan_ok(const ScanArgs& p) {
    return p.B >= 0 && p.T >= 0 && p.D >= 0 && (long long)p.B * p.D < (1ll << 31) && (unsigned)p.T < (1u << 30);
}

// what the caller allocates: carry is [B][carries][D] floats, sums [B][chunks][2][D] (chunks > 1)
PDA_EXPORT int pda_scan_plan(int B, int T, int D, int dtype, int* carries, int* chunks) {
    if (B < 0 || T < 0 || D < 0 || (unsigned)T >= (1u << 30) || dtype < SEQ_F32 || dtype > SEQ_F16) return SEQ_REFUSED;
    const ScanPlan k = scan_plan(B, T, D, dtype);
    *carries = k.carries;
    *chunks = k.chunks;
    return 0;
}

template <typename T, typename F, typename B, bool LOGIT, bool MIX, int MODE>
static void scan_launch(const ScanArgs& p, const ScanPlan& k, bool backward, hipStream_t stream) {
    constexpr int READ = MODE == SCAN_STREAM ? SCAN_WIDE : MODE;
    const dim3 grid((unsigned)((long long)p.B * k.slabs * k.chunks)), fwd(F::NT), bwd(B::NT);
    typedef typename F::Sum Sum;
    if constexpr (!std::is_same<F, ScanWave>::value) {      // (which never has chunks)
        const dim3 sum(Sum::NT);
        if (k.chunks > 1 && !backward) hipLaunchKernelGGL((scan_sum_kernel<T, Sum, LOGIT, MIX, true, READ>), grid, sum, 0, stream, p);
        if (k.chunks > 1 && backward) hipLaunchKernelGGL((scan_sum_kernel<T, Sum, LOGIT, false, false, READ>), grid, sum, 0, stream, p);
    }
    if (!backward) hipLaunchKernelGGL((scan_fwd_kernel<T, F, LOGIT, MIX, MODE>), grid, fwd, 0, stream, p);
    else hipLaunchKernelGGL((scan_bwd_kernel<T, B, LOGIT, MIX, MODE>), grid, bwd, 0, stream, p);
}
template <typename T, typename F, typename B, int MODE>
static void scan_forms(const ScanArgs& p, const ScanPlan& k, bool backward, hipStream_t stream) {
    if (p.logit && p.mix) scan_launch<T, F, B, true, true, MODE>(p, k, backward, stream);
    else if (p.logit) scan_launch<T, F, B, true, false, MODE>(p, k, backward, stream);
    else if (p.mix) scan_launch<T, F, B, false, true, MODE>(p, k, backward, stream);
    else scan_launch<T, F, B, false, false, MODE>(p, k, backward, stream);
}
static bool scan_wide(const void* base, const long long* s, int D, int vec) {
    return s[2] == 1 && D % vec == 0 && s[0] % vec == 0 && s[1] % vec == 0 && (reinterpret_cast<uintptr_t>(base) & 15) == 0;
}
template <typename T>
static void scan_dispatch(const ScanArgs& p, const ScanPlan& k, bool backward, hipStream_t stream) {
    constexpr int VEC = 16 / sizeof(T);
    const bool wide = scan_wide(p.x, p.xs, p.D, VEC) && scan_wide(p.gate, p.gs, p.D, VEC) &&
                      (!backward || p.dh == nullptr || scan_wide(p.dh, p.ds, p.D, VEC));
    if constexpr (sizeof(T) == 4) {     // one channel whose steps are contiguous
        const bool steps = p.D == 1 && p.xs[1] == 1 && p.gs[1] == 1 && (!backward || p.dh == nullptr || p.ds[1] == 1);
        if (steps && k.kind == SCAN_KIND_ROW) return scan_forms<T, ScanRow, ScanRow, SCAN_WIDE>(p, k, backward, stream);
        if (steps && k.kind == SCAN_KIND_WAVE) return scan_forms<T, ScanWave, ScanWave, SCAN_WIDE>(p, k, backward, stream);
    }
    if (k.kind == SCAN_KIND_ROW) scan_forms<T, ScanRow, ScanRow, SCAN_ANY>(p, k, backward, stream);
    else if (k.kind == SCAN_KIND_WAVE) scan_forms<T, ScanWave, ScanWave, SCAN_ANY>(p, k, backward, stream);
    else if (!wide) scan_forms<T, ScanFwd<T>, ScanBwd<T>, SCAN_ANY>(p, k, backward, stream);
    else if (seq_streams((long long)p.B * p.T * p.D * (long long)sizeof(T)))
        scan_forms<T, ScanFwd<T>, ScanBwd<T>, SCAN_STREAM>(p, k, backward, stream);
    else scan_forms<T, ScanFwd<T>, ScanBwd<T>, SCAN_WIDE>(p, k, backward, stream);
}
static int scan_run(const ScanArgs* args, int dtype, bool backward, hipStream_t stream) {
    ScanArgs p = *args;
    if (!scan_ok(p) || dtype < SEQ_F32 || dtype > SEQ_F16) return SEQ_REFUSED;
    if ((long long)p.B * p.D == 0) return 0;
    const ScanPlan k = scan_plan(p.B, p.T, p.D, dtype);
    if (p.chunks != k.chunks || (k.chunks > 1 && p.sums == nullptr) || (backward && k.carries > 0 && p.carry == nullptr))
        return SEQ_REFUSED;
    p.chunk_len = k.chunk_len;
    p.carry_len = k.carry_len;
    p.carries = k.carries;
    const int nt = k.kind == SCAN_KIND_WAVE ? ScanWave::NT : k.kind == SCAN_KIND_ROW ? ScanRow::NT : ScanFwd<elem_f32>::NT;
    if ((long long)p.B * k.slabs * k.chunks >= (1ll << 32) / nt) return SEQ_REFUSED;    // (a launch's threads)
    if (dtype == SEQ_F32) scan_dispatch<elem_f32>(p, k, backward, stream);
    else if (dtype == SEQ_BF16) scan_dispatch<elem_bf16>(p, k, backward, stream);
    else scan_dispatch<elem_f16>(p, k, backward, stream);
    return seq_launched();
}
PDA_EXPORT int pda_scan_fwd(const ScanArgs* args, int dtype, hipStream_t stream) { return scan_run(args, dtype, false, stream); }
PDA_EXPORT int pda_scan_bwd(const ScanArgs* args, int dtype, hipStream_t stream) { return scan_run(args, dtype, true, stream); }

// One step of every request, a thread per element.  Bound by the launch: 64 x 2048 bf16 (1.8 MB) 2.7 us; 512 x 8192 (59 MB)
// 12.9 us, 4.6 TB/s; 4096 x 8192 (470 MB) 111 us, 4.2 TB/s.
struct ScanStepArgs {
    const void* x; const void* gate; const float* state; float* state_out; void* h;
    long long xs[2], gs[2], ss[2], os[2];       // element strides (request, channel)
    int B, D, logit, mix;
};
template <typename T, bool LOGIT, bool MIX>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanStepArgs p) {
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    if (id >= (long long)p.B * p.D) return;
    const int b = (int)(id / p.D), d = (int)(id - (long long)b * p.D);
    const float x = to_f32(((const T*)p.x)[b * p.xs[0] + d * p.xs[1]]);
    const Gate g = gate_of<LOGIT>(to_f32(((const T*)p.gate)[b * p.gs[0] + d * p.gs[1]]));
    float h = scan_step<LOGIT, MIX>(p.state[b * p.ss[0] + d * p.ss[1]], x, g);
    asm("" : "+v"(h));          // what is returned is the stored state rounded, not a second rounding of the exact one
    p.state_out[b * p.os[0] + d * p.os[1]] = h;
    ((T*)p.h)[id] = from_f32<T>(h);
}
template <typename T>
static void scan_step_launch(const ScanStepArgs& p, hipStream_t stream) {
    const dim3 grid((unsigned)(((long long)p.B * p.D + 255) / 256)), block(256);
    if (p.logit && p.mix) hipLaunchKernelGGL((scan_step_kernel<T, true, true>), grid, block, 0, stream, p);
    else if (p.logit) hipLaunchKernelGGL((scan_step_kernel<T, true, false>), grid, block, 0, stream, p);
    else if (p.mix) hipLaunchKernelGGL((scan_step_kernel<T, false, true>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((scan_step_kernel<T, false, false>), grid, block, 0, stream, p);
}
PDA_EXPORT int pda_scan_step(const ScanStepArgs* args, int dtype, hipStream_t stream) {
    const ScanStepArgs p = *args;
    if (p.B < 0 || p.D < 0 || (long long)p.B * p.D >= (1ll << 31)) return SEQ_REFUSED;
    if ((long long)p.B * p.D == 0) return 0;
    if (dtype == SEQ_F32) scan_step_launch<elem_f32>(p, stream);
    else if (dtype == SEQ_BF16) scan_step_launch<elem_bf16>(p, stream);
    else if (dtype == SEQ_F16) scan_step_launch<elem_f16>(p, stream);
    else return SEQ_REFUSED;
    return seq_launched();
}
