// Layer norm over rows, forward and backward.
#include <algorithm>

#include "elements.hpp"

namespace haste {
namespace {

constexpr int kRowThreads = 256;

// The sum of v over the workgroup, in every thread.  `part` [kRowThreads / 64] is free again
// after the next barrier.
__device__ __forceinline__ float group_sum(float v, float* part) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
    for (int k = 0; k < kRowThreads / 64; ++k) v += part[k];
    return v;
}

// A workgroup to a row; the row is read again from cache for each of its passes.
template <int DT, int WT>
__global__ __launch_bounds__(kRowThreads) void ln_fwd_kernel(
    const char* x, int64_t ldx, const char* res, int64_t ldres, const void* w, const void* b,
    char* y, char* h, float* stats, int64_t D, float eps) {
    __shared__ float part[kRowThreads / 64];
    constexpr int S = kElemBytes<DT>;
    const int64_t row = blockIdx.x;
    x += row * ldx * S;
    y += row * D * S;
    if (res) {
        res += row * ldres * S;
        h += row * D * S;
    }
    auto get = [&](int64_t i) {
        const float f = load_elem<DT>(x, i);
        return res ? round_elem<DT>(f + load_elem<DT>(res, i)) : f;
    };
    float s = 0.f;
    for (int64_t i = threadIdx.x; i < D; i += kRowThreads) s += get(i);
    const float mean = group_sum(s, part) / (float)D;
    s = 0.f;
    for (int64_t i = threadIdx.x; i < D; i += kRowThreads) {
        const float d = get(i) - mean;
        s += d * d;
    }
    const float rstd = 1.f / sqrtf(group_sum(s, part) / (float)D + eps);
    for (int64_t i = threadIdx.x; i < D; i += kRowThreads) {
        const float f = get(i);
        if (res) store_elem<DT>(h, i, f);
        const float n = (f - mean) * rstd * load_elem<WT>(w, i);
        store_elem<DT>(y, i, b ? n + load_elem<WT>(b, i) : n);
    }
    if (stats && threadIdx.x == 0) {
        stats[2 * row] = mean;
        stats[2 * row + 1] = rstd;
    }
}

template <int DT, int WT>
__global__ __launch_bounds__(kRowThreads) void ln_dx_kernel(
    const char* dy, int64_t lddy, const char* dh, int64_t lddh, const char* h, int64_t ldh,
    const void* w, const float* stats, char* dx, int64_t D) {
    __shared__ float part[kRowThreads / 64];
    constexpr int S = kElemBytes<DT>;
    const int64_t row = blockIdx.x;
    dy += row * lddy * S;
    h += row * ldh * S;
    dx += row * D * S;
    if (dh) dh += row * lddh * S;
    const float mean = stats[2 * row], rstd = stats[2 * row + 1];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t i = threadIdx.x; i < D; i += kRowThreads) {
        const float a = load_elem<DT>(dy, i) * load_elem<WT>(w, i);
        s1 += a;
        s2 += a * ((load_elem<DT>(h, i) - mean) * rstd);
    }
    const float c1 = group_sum(s1, part) / (float)D, c2 = group_sum(s2, part) / (float)D;
    for (int64_t i = threadIdx.x; i < D; i += kRowThreads) {
        const float n = (load_elem<DT>(h, i) - mean) * rstd;
        float d = rstd * (load_elem<DT>(dy, i) * load_elem<WT>(w, i) - c1 - n * c2);
        if (dh) d += load_elem<DT>(dh, i);
        store_elem<DT>(dx, i, d);
    }
}

// 64 columns to a workgroup, four rows at a time.
template <int DT, int WT>
__global__ __launch_bounds__(kRowThreads) void ln_dw_kernel(const char* dy, int64_t lddy,
                                                            const char* h, int64_t ldh,
                                                            const float* stats, void* dw, void* db,
                                                            int64_t N, int64_t D) {
    __shared__ float part[2][kRowThreads];
    constexpr int S = kElemBytes<DT>;
    const int64_t c = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    float sw = 0.f, sb = 0.f;
    if (c < D)
        for (int64_t r = threadIdx.x >> 6; r < N; r += kRowThreads / 64) {
            const float g = load_elem<DT>(dy + r * lddy * S, c);
            sw += g * ((load_elem<DT>(h + r * ldh * S, c) - stats[2 * r]) * stats[2 * r + 1]);
            sb += g;
        }
    part[0][threadIdx.x] = sw;
    part[1][threadIdx.x] = sb;
    __syncthreads();
    if (threadIdx.x >= 64 || c >= D) return;
    for (int k = 1; k < kRowThreads / 64; ++k) {
        sw += part[0][k * 64 + threadIdx.x];
        sb += part[1][k * 64 + threadIdx.x];
    }
    if (dw) store_elem<WT>(dw, c, sw);
    if (db) store_elem<WT>(db, c, sb);
}

int ln_types(const char* fn, int32_t dtype, int32_t w_dtype) {
    HASTE_CHECK_ARG(elem_dtype(dtype), "%s: rows must be bf16, fp16 or fp32 (dtype code %d)", fn,
                    (int)dtype);
    HASTE_CHECK_ARG(w_dtype == dtype || w_dtype == HASTE_DTYPE_F32,
                    "%s: weights must be of the rows' dtype or fp32 (dtype code %d)", fn,
                    (int)w_dtype);
    return HASTE_OK;
}

// A matrix of rows `ld` apart that is read.
int ln_rows(const char* fn, const char* what, const void* p, int64_t ld, int64_t D, int32_t dtype) {
    HASTE_CHECK_ARG(p != nullptr, "%s: %s is NULL", fn, what);
    HASTE_CHECK_ARG(elem_aligned(p, dtype), "%s: %s is not aligned to its elements", fn, what);
    HASTE_CHECK_ARG(ld == 0 || ld >= D, "%s: row pitch of %s is short (%lld < %lld)", fn, what,
                    (long long)ld, (long long)D);
    return HASTE_OK;
}

#define HASTE_TRY(expr)                        \
    do {                                       \
        const int rc_ = (expr);                \
        if (rc_ != HASTE_OK) return rc_;       \
    } while (0)

// `call` with DT and WT for the types of a call.
#define HASTE_LN_TYPES(call)                                                                 \
    do {                                                                                     \
        if (dtype == HASTE_DTYPE_F32) call(HASTE_DTYPE_F32, HASTE_DTYPE_F32);                \
        else if (dtype == HASTE_DTYPE_BF16 && w_dtype == dtype)                              \
            call(HASTE_DTYPE_BF16, HASTE_DTYPE_BF16);                                        \
        else if (dtype == HASTE_DTYPE_BF16) call(HASTE_DTYPE_BF16, HASTE_DTYPE_F32);         \
        else if (w_dtype == dtype) call(HASTE_DTYPE_F16, HASTE_DTYPE_F16);                   \
        else call(HASTE_DTYPE_F16, HASTE_DTYPE_F32);                                         \
    } while (0)

}  // namespace
}  // namespace haste

extern "C" int haste_layer_norm(const void* x, int64_t ldx, const void* res, int64_t ldres,
                                const void* w, const void* b, void* y, void* h, float* stats,
                                int64_t N, int64_t D, double eps, int32_t dtype, int32_t w_dtype,
                                void* stream) {
    const char* fn = "haste_layer_norm";
    HASTE_CHECK_ARG(N >= 0 && D > 0, "%s: bad sizes N=%lld D=%lld", fn, (long long)N, (long long)D);
    HASTE_CHECK_ARG(N < (int64_t)1 << 31 && D < (int64_t)1 << 31, "%s: matrix too large", fn);
    HASTE_CHECK_ARG(eps >= 0.0, "%s: eps must be >= 0", fn);
    HASTE_TRY(haste::ln_types(fn, dtype, w_dtype));
    if (N == 0) return HASTE_OK;
    HASTE_TRY(haste::ln_rows(fn, "x", x, ldx, D, dtype));
    if (res) {
        HASTE_TRY(haste::ln_rows(fn, "res", res, ldres, D, dtype));
        HASTE_TRY(haste::ln_rows(fn, "h", h, D, D, dtype));
    }
    HASTE_TRY(haste::ln_rows(fn, "w", w, D, D, w_dtype));
    HASTE_CHECK_ARG(haste::elem_aligned(b, w_dtype), "%s: b is not aligned to its elements", fn);
    HASTE_TRY(haste::ln_rows(fn, "y", y, D, D, dtype));
    HASTE_CHECK_ARG(haste::elem_aligned(stats, HASTE_DTYPE_F32), "%s: stats is misaligned", fn);
#define HASTE_LN_FWD(DT, WT)                                                                   \
    haste::ln_fwd_kernel<DT, WT><<<dim3((unsigned)N), dim3(haste::kRowThreads), 0,             \
                                   static_cast<hipStream_t>(stream)>>>(                        \
        static_cast<const char*>(x), ldx, static_cast<const char*>(res), ldres, w, b,          \
        static_cast<char*>(y), static_cast<char*>(h), stats, D, (float)eps)
    HASTE_LN_TYPES(HASTE_LN_FWD);
#undef HASTE_LN_FWD
    HASTE_CHECK_LAUNCH(fn);
    return HASTE_OK;
}

extern "C" int64_t haste_layer_norm_bwd_workspace_size(int64_t N, int64_t D) {
    return N < 0 || D < 0 ? HASTE_ERR_INVALID_ARG : 16;
}

extern "C" int haste_layer_norm_bwd(const void* dy, int64_t lddy, const void* dh, int64_t lddh,
                                    const void* h, int64_t ldh, const void* w, const float* stats,
                                    void* dx, void* dw, void* db, void* ws, int64_t ws_bytes,
                                    int64_t N, int64_t D, int32_t dtype, int32_t w_dtype,
                                    void* stream) {
    const char* fn = "haste_layer_norm_bwd";
    HASTE_CHECK_ARG(N >= 0 && D > 0, "%s: bad sizes N=%lld D=%lld", fn, (long long)N, (long long)D);
    HASTE_CHECK_ARG(N < (int64_t)1 << 31 && D < (int64_t)1 << 31, "%s: matrix too large", fn);
    HASTE_TRY(haste::ln_types(fn, dtype, w_dtype));
    if (N > 0) {
        HASTE_TRY(haste::ln_rows(fn, "dy", dy, lddy, D, dtype));
        if (dh) HASTE_TRY(haste::ln_rows(fn, "dh", dh, lddh, D, dtype));
        HASTE_TRY(haste::ln_rows(fn, "h", h, ldh, D, dtype));
        HASTE_TRY(haste::ln_rows(fn, "w", w, D, D, w_dtype));
        HASTE_CHECK_ARG(stats != nullptr && haste::elem_aligned(stats, HASTE_DTYPE_F32),
                        "%s: stats is NULL or misaligned", fn);
        HASTE_CHECK_ARG(haste::elem_aligned(dx, dtype), "%s: dx is not aligned to its elements", fn);
    }
    HASTE_CHECK_ARG(haste::elem_aligned(dw, w_dtype) && haste::elem_aligned(db, w_dtype),
                    "%s: dw or db is not aligned to its elements", fn);
    if (dw || db) {
        const int64_t need = haste_layer_norm_bwd_workspace_size(N, D);
        HASTE_CHECK_ARG(ws != nullptr && haste::aligned16(ws), "%s: workspace is NULL or misaligned",
                        fn);
        if (ws_bytes < need) {
            haste::set_error("%s: workspace too small (%lld < %lld bytes)", fn, (long long)ws_bytes,
                             (long long)need);
            return HASTE_ERR_WORKSPACE;
        }
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
#define HASTE_LN_BWD(DT, WT)                                                                     \
    do {                                                                                         \
        if (dx && N > 0)                                                                         \
            haste::ln_dx_kernel<DT, WT><<<dim3((unsigned)N), dim3(haste::kRowThreads), 0, st>>>( \
                static_cast<const char*>(dy), lddy, static_cast<const char*>(dh), lddh,          \
                static_cast<const char*>(h), ldh, w, stats, static_cast<char*>(dx), D);          \
        if (dw || db)                                                                            \
            haste::ln_dw_kernel<DT, WT><<<dim3((unsigned)haste::ceil_div(D, 64)),                \
                                          dim3(haste::kRowThreads), 0, st>>>(                    \
                static_cast<const char*>(dy), lddy, static_cast<const char*>(h), ldh, stats, dw, \
                db, N, D);                                                                       \
    } while (0)
    HASTE_LN_TYPES(HASTE_LN_BWD);
#undef HASTE_LN_BWD
    HASTE_CHECK_LAUNCH(fn);
    return HASTE_OK;
}
