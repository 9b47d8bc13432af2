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

template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutArgs p) {
    const long long ctr = *p.counter;
    const uint64_t key = hash_u64(hash_u64(p.seed + SEQ_GOLDEN * (1ull + (uint64_t)ctr)) + SEQ_GOLDEN * (1ull + p.site));
    const uint64_t key2 = hash_u64(key);
    if (p.used != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *p.used = ctr;
    const long long groups = (p.n + 3) >> 2, step = (long long)gridDim.x * 256;
    for (long long g = (long long)blockIdx.x * 256 + threadIdx.x; g < groups; g += step) {
        const uint64_t word = hash_u64(key + SEQ_GOLDEN * (1ull + (uint64_t)g));
        for (int j = 0; j < 4; ++j) {
            const long long i = g * 4 + j;
            if (i >= p.n) break;
            const uint32_t u = (uint32_t)(word >> (16 * j)) & 0xffffu;
            bool keep = u > p.hi;
            if (u == p.hi) keep = (uint32_t)(hash_u64(key2 + SEQ_GOLDEN * (1ull + (uint64_t)i)) >> 32) >= p.lo;
            float v = keep ? to_f32(((const T*)p.x)[i]) * p.scale : 0.f;
            if (p.residual != nullptr) v += to_f32(((const T*)p.residual)[i]);
            ((T*)p.y)[i] = from_f32<T>(v);
        }
    }
}

PDA_EXPORT int pda_dropout(const DropoutArgs* args, int dtype, hipStream_t stream) {
    const DropoutArgs p = *args;
    if (p.n < 0 || p.counter == nullptr || p.hi > 65536u) return SEQ_REFUSED;
    if (p.n == 0 && p.used == nullptr) return 0;
    long long blocks = (p.n + 1023) / 1024;
    blocks = blocks < 1 ? 1 : (blocks > 8192 ? 8192 : blocks);
    const dim3 grid((unsigned)blocks), block(256);
    if (dtype == SEQ_F32) hipLaunchKernelGGL(dropout_kernel<elem_f32>, grid, block, 0, stream, p);
    else if (dtype == SEQ_BF16) hipLaunchKernelGGL(dropout_kernel<elem_bf16>, grid, block, 0, stream, p);
    else if (dtype == SEQ_F16) hipLaunchKernelGGL(dropout_kernel<elem_f16>, grid, block, 0, stream, p);
    else return SEQ_REFUSED;
    return seq_launched();
}
