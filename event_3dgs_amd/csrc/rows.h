// rows.h -- row-wise helpers of the learned-feature operators (features.hip, distill.hip): element types, packs of
// consecutive elements, loads by a runtime type, reductions over a group of lanes.
#pragma once
#include "common.h"

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

enum { E3_F32 = 0, E3_F16 = 1, E3_BF16 = 2 };     // E3DGS_F32 / _F16 / _BF16 (include/e3dgs_hip.h)

// V consecutive elements, loaded and stored as one memory instruction (V * sizeof(T) = 16 bytes, or a single element).
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

// elements of a 16-byte pack
template <typename T>
struct Wide {
    static constexpr int N = 16 / (int)sizeof(T);
};

// A 16-byte pack that is kept in registers across phases of a kernel: four words that the compiler does not split into
// elements (a 16-bit element would take a register of its own).
typedef uint32_t words_t __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ float word_elem(words_t q, int j);
template <>
__device__ __forceinline__ float word_elem<float>(words_t q, int j) { return __uint_as_float(q[j]); }
template <>
__device__ __forceinline__ float word_elem<bf16_t>(words_t q, int j) {
    return __uint_as_float(j & 1 ? q[j >> 1] & 0xFFFF0000u : q[j >> 1] << 16);
}
template <>
__device__ __forceinline__ float word_elem<f16_t>(words_t q, int j) {
    const uint16_t h = (uint16_t)(j & 1 ? q[j >> 1] >> 16 : q[j >> 1]);
    return (float)__builtin_bit_cast(f16_t, h);
}
// Makes the compiler forget what it knows about a pack, so that it converts the elements again in the next phase instead of
// holding their fp32 values.
__device__ __forceinline__ void forget(words_t& q) { asm volatile("" : "+v"(q)); }
__device__ __forceinline__ void forget(uint32_t& x) { asm volatile("" : "+v"(x)); }

// Stores of a large result.  Past E3_STREAM_BYTES (half of the 256 MB Infinity Cache) the reader of a result finds little of
// it there, while ordinary stores push the running kernel's inputs out and hold its reads up: such a result is streamed past
// the cache.  A lookup of 192 MB of rows takes 55 us with ordinary and 30 us with streamed stores, and with a layer norm
// behind it 122 us and 104 us; at 134 MB and below the reader loses more than the writer gains (lookup + layer norm of
// 8192 x 4096 fp32: 86 us ordinary, 88 us streamed).  A template argument: the compiler joins the two stores of a runtime
// choice into an ordinary one.
constexpr size_t E3_STREAM_BYTES = 128u << 20;
template <bool STREAM, typename T, int V>
__device__ __forceinline__ void put(T* p, const Pack<T, V>& r) {
    if constexpr (!STREAM) *reinterpret_cast<Pack<T, V>*>(p) = r;
    else if constexpr (sizeof(r) == 16) __builtin_nontemporal_store(__builtin_bit_cast(words_t, r), reinterpret_cast<words_t*>(p));
    else if constexpr (sizeof(r) == 8) __builtin_nontemporal_store(__builtin_bit_cast(unsigned long long, r), reinterpret_cast<unsigned long long*>(p));
    else if constexpr (sizeof(r) == 4) __builtin_nontemporal_store(__builtin_bit_cast(uint32_t, r), reinterpret_cast<uint32_t*>(p));
    else __builtin_nontemporal_store(__builtin_bit_cast(uint16_t, r), reinterpret_cast<uint16_t*>(p));
}

static inline size_t e3_elem_bytes(int dtype) { return dtype == E3_F32 ? 4 : 2; }

// The bits of one element, and a pack on its way from memory.  A single 16-bit value is loaded into a register of its own: loads
// that fill the halves of one register wait for each other.
template <typename T>
using Bits = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
template <typename T>
__device__ __forceinline__ T bits_elem(uint32_t v) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, v);
    else return __builtin_bit_cast(T, (uint16_t)v);
}
template <typename T, int V>
struct Held {
    Pack<T, V> p;
    __device__ __forceinline__ void load(const T* src) { p = *reinterpret_cast<const Pack<T, V>*>(src); }
    __device__ __forceinline__ float value(int j) const { return (float)p.v[j]; }
};
template <typename T>
struct Held<T, 1> {
    uint32_t bits;
    __device__ __forceinline__ void load(const T* src) { bits = *reinterpret_cast<const Bits<T>*>(src); }
    __device__ __forceinline__ float value(int) const { return (float)bits_elem<T>(bits); }
};

// Whether rows at `p`, `stride` elements apart and `dim` long, can be read as packs of `bytes` bytes (a power of two).
static inline bool e3_rows_packs(const void* p, size_t stride, size_t dim, int dtype, size_t bytes) {
    const size_t n = bytes / e3_elem_bytes(dtype);
    return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0 && stride % n == 0 && dim % n == 0;
}
static inline bool e3_rows_wide(const void* p, size_t stride, size_t dim, int dtype) {
    return e3_rows_packs(p, stride, dim, dtype, 16);
}

// One element of an array whose type is a launch argument (uniform branch): parameters and labels, which are read once per
// workgroup or row, so that the kernels need no instance per combination of types.
__device__ __forceinline__ float load_elem(const void* __restrict__ p, size_t i, int dtype) {
    if (dtype == E3_F32) return reinterpret_cast<const float*>(p)[i];
    if (dtype == E3_F16) return (float)reinterpret_cast<const f16_t*>(p)[i];
    return (float)reinterpret_cast<const bf16_t*>(p)[i];
}
__device__ __forceinline__ long long load_index(const void* __restrict__ p, size_t i, int bytes) {
    return bytes == 8 ? reinterpret_cast<const long long*>(p)[i] : (long long)reinterpret_cast<const int*>(p)[i];
}

// The same for labels, whose loads should be in flight together: without a branch on the type (a branch waits for its own
// load), as the halves of a value, the second one only counting where the type has it.
__device__ __forceinline__ float load_elem_flat(const void* __restrict__ p, size_t i, int dtype) {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + (dtype == E3_F32 ? 2 * i : i);
    const uint32_t lo = h[0], hi = h[dtype == E3_F32 ? 1 : 0];
    const float f16 = (float)__builtin_bit_cast(f16_t, (uint16_t)lo);
    return dtype == E3_F32 ? __uint_as_float(hi << 16 | lo) : dtype == E3_F16 ? f16 : __uint_as_float(lo << 16);
}
__device__ __forceinline__ long long load_index_flat(const void* __restrict__ p, size_t i, int bytes) {
    const int* w = reinterpret_cast<const int*>(p) + (bytes == 8 ? 2 * i : i);
    const int lo = w[0], hi = w[bytes == 8 ? 1 : 0];
    return (long long)(bytes == 8 ? hi : lo >> 31) << 32 | (uint32_t)lo;
}

// Sum / maximum over aligned groups of G lanes (G a power of two, 1 .. 64): every lane of the group gets the result, and
// every lane adds in the same tree, so the result does not depend on the lane.
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = 1; o < G; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}
template <int G>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int o = 1; o < G; o <<= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
