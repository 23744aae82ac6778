// Loads and stores of bf16, fp16 and fp32 elements as fp32, for passes that take any of the
// three (layer norm, AdamW).
#pragma once

#include "common.hpp"

namespace haste {

template <int DT>
constexpr int kElemBytes = DT == HASTE_DTYPE_F32 ? 4 : 2;

template <int DT>
__device__ __forceinline__ float load_elem(const void* p, int64_t i) {
    if constexpr (DT == HASTE_DTYPE_F32) return static_cast<const float*>(p)[i];
    const uint32_t h = static_cast<const uint16_t*>(p)[i];
    return DT == HASTE_DTYPE_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
}

// Rounded to nearest even.
template <int DT>
__device__ __forceinline__ void store_elem(void* p, int64_t i, float f) {
    if constexpr (DT == HASTE_DTYPE_F32)
        static_cast<float*>(p)[i] = f;
    else
        static_cast<uint16_t*>(p)[i] =
            (uint16_t)(DT == HASTE_DTYPE_BF16 ? f32_to_bf16_rne(f) : f32_to_f16_rne(f));
}

// f as an element of type DT holds it.
template <int DT>
__device__ __forceinline__ float round_elem(float f) {
    if constexpr (DT == HASTE_DTYPE_F32) return f;
    return DT == HASTE_DTYPE_BF16 ? bf16_bits_to_f32(f32_to_bf16_rne(f))
                                  : f16_bits_to_f32(f32_to_f16_rne(f));
}

// V elements (4 or 8) as they lie in memory, read and written with the alignment of one element
// (gfx950 takes 16-byte accesses at any address).
template <int DT, int V>
struct Elems {
    uint32_t q[V * kElemBytes<DT> / 4];
};
typedef u32x4 __attribute__((aligned(2))) u32x4_a2;
typedef u32x2 __attribute__((aligned(2))) u32x2_a2;

// NT: non-temporal, for what is met once.
template <int DT, int V, bool NT = false>
__device__ __forceinline__ Elems<DT, V> load(const void* p, int64_t i) {
    const char* a = static_cast<const char*>(p) + i * kElemBytes<DT>;
    constexpr int W = V * kElemBytes<DT> / 4;
    Elems<DT, V> v;
    if constexpr (W == 2) {
        const u32x2_a2* s = reinterpret_cast<const u32x2_a2*>(a);
        const u32x2 x = NT ? __builtin_nontemporal_load(s) : *s;
        v.q[0] = x[0];
        v.q[1] = x[1];
    } else {
#pragma unroll
        for (int k = 0; k < W / 4; ++k) {
            const u32x4_a2* s = reinterpret_cast<const u32x4_a2*>(a) + k;
            const u32x4 x = NT ? __builtin_nontemporal_load(s) : *s;
#pragma unroll
            for (int j = 0; j < 4; ++j) v.q[4 * k + j] = x[j];
        }
    }
    return v;
}

template <int DT, int V, bool NT = false>
__device__ __forceinline__ void store(void* p, int64_t i, const Elems<DT, V>& v) {
    char* a = static_cast<char*>(p) + i * kElemBytes<DT>;
    constexpr int W = V * kElemBytes<DT> / 4;
    if constexpr (W == 2) {
        u32x2_a2* d = reinterpret_cast<u32x2_a2*>(a);
        const u32x2 x = {v.q[0], v.q[1]};
        if (NT) __builtin_nontemporal_store(x, d);
        else *d = x;
    } else {
#pragma unroll
        for (int k = 0; k < W / 4; ++k) {
            u32x4_a2* d = reinterpret_cast<u32x4_a2*>(a) + k;
            const u32x4 x = {v.q[4 * k], v.q[4 * k + 1], v.q[4 * k + 2], v.q[4 * k + 3]};
            if (NT) __builtin_nontemporal_store(x, d);
            else *d = x;
        }
    }
}

// The first `count` of V elements, zeros after them; none where count <= 0.
template <int DT, int V>
__device__ __forceinline__ Elems<DT, V> load_part(const void* p, int64_t i, int64_t count) {
    if (count >= V) return load<DT, V>(p, i);
    Elems<DT, V> v{};
#pragma unroll
    for (int e = 0; e < V - 1; ++e)
        if (e < count) {
            if constexpr (DT == HASTE_DTYPE_F32) v.q[e] = static_cast<const uint32_t*>(p)[i + e];
            else v.q[e / 2] |= (uint32_t)static_cast<const uint16_t*>(p)[i + e] << (16 * (e & 1));
        }
    return v;
}

template <int DT, int V>
__device__ __forceinline__ void store_part(void* p, int64_t i, const Elems<DT, V>& v,
                                           int64_t count) {
    if (count >= V) return store<DT, V>(p, i, v);
#pragma unroll
    for (int e = 0; e < V - 1; ++e)
        if (e < count) {
            if constexpr (DT == HASTE_DTYPE_F32) static_cast<uint32_t*>(p)[i + e] = v.q[e];
            else static_cast<uint16_t*>(p)[i + e] = (uint16_t)(v.q[e / 2] >> (16 * (e & 1)));
        }
}

template <int DT, int V>
__device__ __forceinline__ void unpack(const Elems<DT, V>& v, float* f) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
        if constexpr (DT == HASTE_DTYPE_F32) {
            f[e] = __uint_as_float(v.q[e]);
        } else {
            const uint32_t h = (e & 1) ? v.q[e / 2] >> 16 : v.q[e / 2] & 0xFFFFu;
            f[e] = DT == HASTE_DTYPE_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
        }
    }
}

// Rounded to nearest even.
template <int DT, int V>
__device__ __forceinline__ Elems<DT, V> pack(const float* f) {
    Elems<DT, V> v;
    if constexpr (DT == HASTE_DTYPE_F32) {
#pragma unroll
        for (int e = 0; e < V; ++e) v.q[e] = __float_as_uint(f[e]);
    } else {
#pragma unroll
        for (int e = 0; e < V / 2; ++e)
            v.q[e] = DT == HASTE_DTYPE_BF16
                         ? pack2_rne<BF16>(f[2 * e], f[2 * e + 1])
                         : f32_to_f16_rne(f[2 * e]) | f32_to_f16_rne(f[2 * e + 1]) << 16;
    }
    return v;
}

inline bool elem_dtype(int32_t dt) {
    return dt == HASTE_DTYPE_BF16 || dt == HASTE_DTYPE_F16 || dt == HASTE_DTYPE_F32;
}
inline int elem_bytes(int32_t dt) { return dt == HASTE_DTYPE_F32 ? 4 : 2; }
inline bool elem_aligned(const void* p, int32_t dt) {
    return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(elem_bytes(dt) - 1)) == 0;
}

}  // namespace haste
