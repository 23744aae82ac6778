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

inline bool elem_dtype(int32_t dt) {
    return dt == HASTE_DTYPE_BF16 || dt == HASTE_DTYPE_F16 || dt == HASTE_DTYPE_F32;
}
inline int elem_bytes(int32_t dt) { return dt == HASTE_DTYPE_F32 ? 4 : 2; }
inline bool elem_aligned(const void* p, int32_t dt) {
    return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(elem_bytes(dt) - 1)) == 0;
}

}  // namespace haste
