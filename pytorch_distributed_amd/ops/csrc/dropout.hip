// Dropout whose mask is a function of (seed, step counter, site, element) and is regenerated in the backward pass.
//
//   key  = mix(mix(seed + G (1 + counter)) + G (1 + site)),  key2 = mix(key)          G = 2^64 / golden ratio
//   word = mix(key + G (1 + i / 4)),  u = 16 bits of word for element i               mix = common.h's 64-bit finaliser
//   dropped: u < hi, or u == hi and the high half of mix(key2 + G (1 + i)) < lo       (hi, lo) = p in 48 bits
//   y = x / (1 - p) where kept, 0 where dropped (also where x is not finite), + residual;  dx = dy / (1 - p) where kept
//
// One 64-bit hash decides four elements: two 64-bit products (about 30 issue cycles) spread over four elements is what
// leaves the kernel bound by memory instead of by the integer pipe.  16 bits alone would round p to multiples of 2^-16;
// the second hash is taken only where they tie (one element in 65536), so p is honoured to 2^-48.
#include "seq.h"

struct DropoutArgs {
    const void* x; const void* residual; void* y;
    const long long* counter;       // read by the forward pass ...
    long long* used;                // ... which leaves the value here for the backward pass (null in the backward pass)
    unsigned long long seed; unsigned int site, hi, lo; float scale; long long n;
};

struct DropKey { uint64_t key, key2; uint32_t hi, lo; };
__device__ __forceinline__ DropKey drop_key(const DropoutArgs& p, long long ctr) {
    const uint64_t key = hash_u64(hash_u64(p.seed + SEQ_GOLDEN * (1ull + (uint64_t)ctr)) + SEQ_GOLDEN * (1ull + p.site));
    return DropKey{key, hash_u64(key), p.hi, p.lo};
}
// bit j: element 4 g + j is kept
__device__ __forceinline__ uint32_t drop_group(const DropKey& k, long long g) {
    const uint64_t word = hash_u64(k.key + SEQ_GOLDEN * (1ull + (uint64_t)g));
    uint32_t keep = 0, tie = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t u = (uint32_t)(word >> (16 * j)) & 0xffffu;
        keep |= (u > k.hi ? 1u : 0u) << j;
        tie |= (u == k.hi ? 1u : 0u) << j;
    }
    while (tie) {       // one element in 65536
        const int j = __builtin_ctz(tie);
        tie &= tie - 1;
        if ((uint32_t)(hash_u64(k.key2 + SEQ_GOLDEN * (1ull + (uint64_t)(4 * g + j))) >> 32) >= k.lo) keep |= 1u << j;
    }
    return keep;
}

// A thread takes 16 bytes (one or two groups of four) of each tensor at a time, DROP_U of them in flight.  Bound by memory:
// 16384 x 4096 bf16 with residual 70 us for 403 MB (5.7 TB/s), its backward pass 45 us for 268 MB (6.0 TB/s); a copy of 256
// MB reaches 5.4.  128 x 512 fp32: 3.0 us, the launch.
#define DROP_U 2
template <typename T, bool RESIDUAL, bool STREAM>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutArgs p) {
    constexpr int VEC = 16 / sizeof(T), U = DROP_U;
    const long long ctr = *p.counter;
    const DropKey key = drop_key(p, ctr);
    if (p.used != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *p.used = ctr;
    const long long nvec = p.n / VEC, step = (long long)gridDim.x * 256 * U;
    const vec16<T>* x = (const vec16<T>*)p.x;
    const vec16<T>* r = (const vec16<T>*)p.residual;
    for (long long b = (long long)blockIdx.x * 256 * U + threadIdx.x; b < nvec; b += step) {
        vec16<T> xr[U], rr[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long v = b + u * 256;
            if (v < nvec) {
                xr[u] = x[v];
                if (RESIDUAL) rr[u] = r[v];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long v = b + u * 256;
            if (v >= nvec) continue;
            vec16<T> o;
#pragma unroll
            for (int h = 0; h < VEC / 4; ++h) {
                const uint32_t keep = drop_group(key, v * (VEC / 4) + h);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float y = (keep >> j) & 1u ? to_f32(xr[u].e[4 * h + j]) * p.scale : 0.f;
                    if (RESIDUAL) y += to_f32(rr[u].e[4 * h + j]);
                    o.e[4 * h + j] = from_f32<T>(y);
                }
            }
            store16<STREAM>((T*)p.y + v * VEC, o);
        }
    }
    const int tail = (int)(p.n - nvec * VEC);       // at most 7 elements
    if (blockIdx.x == 0 && (int)threadIdx.x < tail) {
        const long long i = nvec * VEC + threadIdx.x;
        float y = (drop_group(key, i >> 2) >> (i & 3)) & 1u ? to_f32(((const T*)p.x)[i]) * p.scale : 0.f;
        if (RESIDUAL) y += to_f32(((const T*)p.residual)[i]);
        ((T*)p.y)[i] = from_f32<T>(y);
    }
}
// the same element by element, for tensors off the 16-byte grid
template <typename T>
__global__ __launch_bounds__(256) void dropout_any_kernel(DropoutArgs p) {
    const long long ctr = *p.counter;
    const DropKey key = drop_key(p, ctr);
    if (p.used != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *p.used = ctr;
    const long long groups = (p.n + 3) >> 2, step = (long long)gridDim.x * 256;
    for (long long g = (long long)blockIdx.x * 256 + threadIdx.x; g < groups; g += step) {
        const uint32_t keep = drop_group(key, g);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const long long i = g * 4 + j;
            if (i >= p.n) break;
            float y = (keep >> j) & 1u ? to_f32(((const T*)p.x)[i]) * p.scale : 0.f;
            if (p.residual != nullptr) y += to_f32(((const T*)p.residual)[i]);
            ((T*)p.y)[i] = from_f32<T>(y);
        }
    }
}

template <typename T>
static void dropout_launch(const DropoutArgs& p, hipStream_t stream) {
    const uintptr_t grid16 = (uintptr_t)p.x | (uintptr_t)p.residual | (uintptr_t)p.y;
    const bool wide = (grid16 & 15) == 0;
    const long long per = wide ? 256 * DROP_U * (16 / (long long)sizeof(T)) : 1024;
    long long blocks = (p.n + per - 1) / per;
    blocks = blocks < 1 ? 1 : (blocks > 1048576 ? 1048576 : blocks);
    const dim3 grid((unsigned)blocks), block(256);
    const bool past = seq_streams(p.n * (long long)sizeof(T));
    if (!wide) hipLaunchKernelGGL(dropout_any_kernel<T>, grid, block, 0, stream, p);
    else if (p.residual && past) hipLaunchKernelGGL((dropout_kernel<T, true, true>), grid, block, 0, stream, p);
    else if (p.residual) hipLaunchKernelGGL((dropout_kernel<T, true, false>), grid, block, 0, stream, p);
    else if (past) hipLaunchKernelGGL((dropout_kernel<T, false, true>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((dropout_kernel<T, false, false>), grid, block, 0, stream, p);
}

PDA_EXPORT int pda_dropout(const DropoutArgs* args, int dtype, hipStream_t stream) {
    const DropoutArgs p = *args;
    if (p.n < 0 || p.counter == nullptr || p.hi > 65536u) return SEQ_REFUSED;
    if (p.n == 0 && p.used == nullptr) return 0;
    if (dtype == SEQ_F32) dropout_launch<elem_f32>(p, stream);
    else if (dtype == SEQ_BF16) dropout_launch<elem_bf16>(p, stream);
    else if (dtype == SEQ_F16) dropout_launch<elem_f16>(p, stream);
    else return SEQ_REFUSED;
    return seq_launched();
}
