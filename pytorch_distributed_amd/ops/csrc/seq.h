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

// bits of an element, and the element in the low (0) or high (1) half of a register
__device__ __forceinline__ uint32_t bits_of(elem_f32 e) { return __builtin_bit_cast(uint32_t, e.v); }
__device__ __forceinline__ uint32_t bits_of(elem_bf16 e) { return e.v; }
__device__ __forceinline__ uint32_t bits_of(elem_f16 e) { return __builtin_bit_cast(unsigned short, e.v); }
template <typename T> __device__ __forceinline__ float value_of(uint32_t w, int half);
template <> __device__ __forceinline__ float value_of<elem_f32>(uint32_t w, int) { return __builtin_bit_cast(float, w); }
template <> __device__ __forceinline__ float value_of<elem_bf16>(uint32_t w, int half) {
    return __builtin_bit_cast(float, half ? w & 0xffff0000u : w << 16);
}
template <> __device__ __forceinline__ float value_of<elem_f16>(uint32_t w, int half) {
    return (float)__builtin_bit_cast(_Float16, (unsigned short)(half ? w >> 16 : w));
}

// 16 bytes of elements
template <typename T> struct alignas(16) vec16 { T e[16 / sizeof(T)]; };

// 16-byte store.  STREAM: past the caches.  An output that does not fit the 256 MB memory-side cache next to its inputs only
// pushes them out of it: the gradient of 4096 x 32000 bf16 logits (262 MB) took 107 us through the caches and 78 us past
// them, and the next forward pass over the same logits 65 and 48 us.  Outputs that do fit stay for whoever reads them next.
typedef __attribute__((ext_vector_type(4))) int seq_i32x4;
typedef __attribute__((ext_vector_type(4))) unsigned seq_u32x4;
#define SEQ_STREAM_BYTES (96ll << 20)
template <bool STREAM, typename T>
__device__ __forceinline__ void store16(T* to, const vec16<T>& v) {
    if (STREAM) __builtin_nontemporal_store(__builtin_bit_cast(seq_i32x4, v), reinterpret_cast<seq_i32x4*>(to));
    else *reinterpret_cast<vec16<T>*>(to) = v;
}
static inline bool seq_streams(long long bytes) { return bytes >= SEQ_STREAM_BYTES; }

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
