// Shared by the sequence-policy operators (logprob.hip, scan.hip, dropout.hip): element types, host-side checks.
#pragma once
#include "common.h"

// Element types of the operators' tensors; every sum, softmax statistic and recurrent state is a 32-bit float, and a
// value is rounded to a 16-bit type once, where it is stored.
struct elem_f32 { float v; };
struct elem_bf16 { bf16_t v; };
struct elem_f16 { _Float16 v; };
__device__ __forceinline__ float to_f32(elem_f32 e) { return e.v; }
__device__ __forceinline__ float to_f32(elem_bf16 e) { return bf2f(e.v); }
__device__ __forceinline__ float to_f32(elem_f16 e) { return (float)e.v; }
template <typename T> __device__ __forceinline__ T from_f32(float f);
template <> __device__ __forceinline__ elem_f32 from_f32<elem_f32>(float f) { return elem_f32{f}; }
template <> __device__ __forceinline__ elem_bf16 from_f32<elem_bf16>(float f) { return elem_bf16{f2bf(f)}; }
template <> __device__ __forceinline__ elem_f16 from_f32<elem_f16>(float f) { return elem_f16{(_Float16)f}; }

// 16 bytes of elements
template <typename T> struct alignas(16) vec16 { T e[16 / sizeof(T)]; };

// dtype codes of the C entries (ops/_seq.py TYPE_CODES)
#define SEQ_F32 0
#define SEQ_BF16 1
#define SEQ_F16 2

// Entries return 0, -1 for arguments they refuse (nothing was launched), or the HIP error of the launch.
#define SEQ_REFUSED (-1)
static inline int seq_launched() { return (int)hipGetLastError(); }

// 64-bit finaliser of the counter hash in common.h (all 64 bits of it; hash_u32 returns the low half)
#define SEQ_GOLDEN 0x9e3779b97f4a7c15ULL
__host__ __device__ __forceinline__ uint64_t hash_u64(uint64_t x) {
    x ^= x >> 33; x *= 0xff51afd7ed558ccdULL; x ^= x >> 33; x *= 0xc4ceb9fe1a85ec53ULL; x ^= x >> 33;
    return x;
}
