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

// Eight elements as they lie in memory, read and written with the alignment of one element
// (gfx950 takes 16-byte accesses at any address).
template <int DT>
struct Elems8 {
    u32x4 q[DT == HASTE_DTYPE_F32 ? 2 : 1];
};
typedef u32x4 __attribute__((aligned(2))) u32x4_a2;

template <int DT, bool NT = false>
__device__ __forceinline__ Elems8<DT> load8(const void* p, int64_t i) {
    const u32x4_a2* a =
        reinterpret_cast<const u32x4_a2*>(static_cast<const char*>(p) + i * kElemBytes<DT>);
    Elems8<DT> v;
    if constexpr (NT) {
        v.q[0] = __builtin_nontemporal_load(a);
        if constexpr (DT == HASTE_DTYPE_F32) v.q[1] = __builtin_nontemporal_load(a + 1);
    } else {
        v.q[0] = a[0];
        if constexpr (DT == HASTE_DTYPE_F32) v.q[1] = a[1];
    }
    return v;
}

template <int DT, bool NT = false>
__device__ __forceinline__ void store8(void* p, int64_t i, const Elems8<DT>& v) {
    u32x4_a2* a = reinterpret_cast<u32x4_a2*>(static_cast<char*>(p) + i * kElemBytes<DT>);
    if constexpr (NT) {
        __builtin_nontemporal_store(v.q[0], a);
        if constexpr (DT == HASTE_DTYPE_F32) __builtin_nontemporal_store(v.q[1], a + 1);
    } else {
        a[0] = v.q[0];
        if constexpr (DT == HASTE_DTYPE_F32) a[1] = v.q[1];
    }
}

// The first `count` of eight elements, zeros after them; none where count <= 0.
template <int DT>
__device__ __forceinline__ Elems8<DT> load8_part(const void* p, int64_t i, int64_t count) {
    if (count >= 8) return load8<DT>(p, i);
    Elems8<DT> v;
    v.q[0] = u32x4{0, 0, 0, 0};
    if constexpr (DT == HASTE_DTYPE_F32) v.q[1] = v.q[0];
#pragma unroll
    for (int e = 0; e < 7; ++e)
        if (e < count) {
            if constexpr (DT == HASTE_DTYPE_F32)
                v.q[e / 4][e & 3] = static_cast<const uint32_t*>(p)[i + e];
            else
                v.q[0][e / 2] |= (uint32_t)static_cast<const uint16_t*>(p)[i + e] << (16 * (e & 1));
        }
    return v;
}

template <int DT>
__device__ __forceinline__ void store8_part(void* p, int64_t i, const Elems8<DT>& v, int64_t count) {
    if (count >= 8) return store8<DT>(p, i, v);
#pragma unroll
    for (int e = 0; e < 7; ++e)
        if (e < count) {
            if constexpr (DT == HASTE_DTYPE_F32)
                static_cast<uint32_t*>(p)[i + e] = v.q[e / 4][e & 3];
            else
                static_cast<uint16_t*>(p)[i + e] = (uint16_t)(v.q[0][e / 2] >> (16 * (e & 1)));
        }
}

template <int DT>
__device__ __forceinline__ void unpack8(const Elems8<DT>& v, float* f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (DT == HASTE_DTYPE_F32) {
            f[e] = __uint_as_float(v.q[e / 4][e & 3]);
        } else {
            const uint32_t h = (e & 1) ? v.q[0][e / 2] >> 16 : v.q[0][e / 2] & 0xFFFFu;
            f[e] = DT == HASTE_DTYPE_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
        }
    }
}

// Rounded to nearest even.
template <int DT>
__device__ __forceinline__ Elems8<DT> pack8(const float* f) {
    Elems8<DT> v;
    if constexpr (DT == HASTE_DTYPE_F32) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v.q[e / 4][e & 3] = __float_as_uint(f[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v.q[0][e] = DT == HASTE_DTYPE_BF16 ? pack2_rne<BF16>(f[2 * e], f[2 * e + 1])
                                               : f32_to_f16_rne(f[2 * e]) | f32_to_f16_rne(f[2 * e + 1]) << 16;
    }
    return v;
}

// Four elements, as Elems8.
template <int DT>
struct Elems4 {
    uint32_t q[DT == HASTE_DTYPE_F32 ? 4 : 2];
};
typedef u32x2 __attribute__((aligned(2))) u32x2_a2;

template <int DT, bool NT = false>
__device__ __forceinline__ Elems4<DT> load4(const void* p, int64_t i) {
    const char* a = static_cast<const char*>(p) + i * kElemBytes<DT>;
    if constexpr (DT == HASTE_DTYPE_F32) {
        const u32x4_a2* v = reinterpret_cast<const u32x4_a2*>(a);
        const u32x4 x = NT ? __builtin_nontemporal_load(v) : *v;
        return Elems4<DT>{{x[0], x[1], x[2], x[3]}};
    } else {
        const u32x2_a2* v = reinterpret_cast<const u32x2_a2*>(a);
        const u32x2 x = NT ? __builtin_nontemporal_load(v) : *v;
        return Elems4<DT>{{x[0], x[1]}};
    }
}

template <int DT, bool NT = false>
__device__ __forceinline__ void store4(void* p, int64_t i, const Elems4<DT>& x) {
    char* a = static_cast<char*>(p) + i * kElemBytes<DT>;
    if constexpr (DT == HASTE_DTYPE_F32) {
        u32x4_a2* v = reinterpret_cast<u32x4_a2*>(a);
        const u32x4 y = {x.q[0], x.q[1], x.q[2], x.q[3]};
        if (NT) __builtin_nontemporal_store(y, v);
        else *v = y;
    } else {
        u32x2_a2* v = reinterpret_cast<u32x2_a2*>(a);
        const u32x2 y = {x.q[0], x.q[1]};
        if (NT) __builtin_nontemporal_store(y, v);
        else *v = y;
    }
}

template <int DT>
__device__ __forceinline__ Elems4<DT> load4_part(const void* p, int64_t i, int64_t count) {
    if (count >= 4) return load4<DT>(p, i);
    Elems4<DT> v{};
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (e < count) {
            if constexpr (DT == HASTE_DTYPE_F32) v.q[e] = static_cast<const uint32_t*>(p)[i + e];
            else v.q[e / 2] |= (uint32_t)static_cast<const uint16_t*>(p)[i + e] << (16 * (e & 1));
        }
    return v;
}

template <int DT>
__device__ __forceinline__ void store4_part(void* p, int64_t i, const Elems4<DT>& v, int64_t count) {
    if (count >= 4) return store4<DT>(p, i, v);
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (e < count) {
            if constexpr (DT == HASTE_DTYPE_F32) static_cast<uint32_t*>(p)[i + e] = v.q[e];
            else static_cast<uint16_t*>(p)[i + e] = (uint16_t)(v.q[e / 2] >> (16 * (e & 1)));
        }
}

template <int DT>
__device__ __forceinline__ void unpack4(const Elems4<DT>& v, float* f) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (DT == HASTE_DTYPE_F32) {
            f[e] = __uint_as_float(v.q[e]);
        } else {
            const uint32_t h = (e & 1) ? v.q[e / 2] >> 16 : v.q[e / 2] & 0xFFFFu;
            f[e] = DT == HASTE_DTYPE_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
        }
    }
}

// Rounded to nearest even.
template <int DT>
__device__ __forceinline__ Elems4<DT> pack4(const float* f) {
    Elems4<DT> v;
    if constexpr (DT == HASTE_DTYPE_F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v.q[e] = __float_as_uint(f[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 2; ++e)
            v.q[e] = DT == HASTE_DTYPE_BF16 ? pack2_rne<BF16>(f[2 * e], f[2 * e + 1])
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
