// The norm of many gradients, and AdamW steps of many tensors with states in 32 or in 8 bits.
#include <algorithm>
#include <cmath>

#include "elements.hpp"

namespace haste {
namespace {

constexpr int kBlock = 128;    // elements of an 8-bit state that share a scale
constexpr int kMaxSegs = 60;   // tensors of one launch: their table fills its 4 KB of arguments

struct AdamSeg {
    void* w;
    const void* g;
    void* m;
    void* v;
    uint8_t* ms;
    uint8_t* vs;
    int64_t n;
    uint32_t blk0;    // first workgroup of this tensor
    uint32_t stream;
};
struct AdamBatch {
    AdamSeg s[kMaxSegs];
    int32_t count;
};
struct AdamArgs {
    float b1, c1, b2, c2;  // beta1, 1 - beta1, beta2, 1 - beta2
    float decay, lr, rcorr, eps;  // 1 - lr wd, lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t)
    uint32_t k0, k1;
    int32_t do_sr;
    const float* grad_scale;
};

struct GradSeg {
    const void* g;
    int64_t n;
    int32_t dtype;
    uint32_t blk0;
};
struct GradBatch {
    GradSeg s[kMaxSegs];
    int32_t count;
};

// The four words of Philox4x32-10 (philox_w0's function).
__device__ __forceinline__ u32x4 philox_words(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t k0,
                                              uint32_t k1) {
    uint32_t c3 = 0u;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
        c0 = __builtin_amdgcn_bitop3_b32((uint32_t)(p1 >> 32), c1, k0, 0x96);
        c2 = __builtin_amdgcn_bitop3_b32((uint32_t)(p0 >> 32), c3, k1, 0x96);
        c1 = (uint32_t)p1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return u32x4{c0, c1, c2, c3};
}

// |x| in units of its spacing with MANT mantissa bits and smallest normal 2^LOW, plus `up` in
// [0, 1), cut to a whole number; `unit` is that spacing.
template <int MANT, int LOW>
__device__ __forceinline__ float cut_units(float x, float up, float* unit) {
    const uint32_t e = max(__float_as_uint(x) & 0x7F800000u, (uint32_t)(127 + LOW) << 23);
    *unit = __uint_as_float(e - ((uint32_t)MANT << 23));
    return floorf(fabsf(x) * __uint_as_float((254u << 23) - (e - ((uint32_t)MANT << 23))) + up);
}

// x as an e4m3 code, rounded by the 16 bits r; with KEEP what is above zero stays so.  |x| is
// below 2^8 or not finite (NaN then).
template <bool KEEP>
__device__ __forceinline__ uint32_t cut_e4m3(float x, uint32_t r) {
    float unit;
    float t = cut_units<3, -6>(x, (float)r * 0x1p-16f, &unit);
    if (KEEP && x > 0.f) t = fmaxf(t, 1.f);
    t = copysignf(t * unit, x);
    if (!(fabsf(x) < 512.f)) return 0x7Fu;
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(t, t, 0, false) & 0xFFu;
}

__device__ __forceinline__ float e4m3_to_f32(uint32_t c) {
    return __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
}

// w as 16 bits of type WT, rounded by the 16 bits r.
template <int WT>
__device__ __forceinline__ uint32_t cut_16(float w, uint32_t r) {
    if constexpr (WT == HASTE_DTYPE_BF16) return sr_bf16(w, r);
    if (!(fabsf(w) < 65536.f)) return f32_to_f16_rne(w);
    float unit;
    const float t = cut_units<10, -14>(w, (float)(r >> 3) * 0x1p-13f, &unit);
    return f32_to_f16_rne(copysignf(t * unit, w));
}

template <typename B>
__device__ __forceinline__ int find_seg(const B& b, uint32_t blk) {
    int t = 0;
    for (int k = 1; k < b.count; ++k)
        if (blk >= b.s[k].blk0) t = k;
    return t;
}

// A thread to an element, a workgroup to a block of 128.
template <int WT, int GT, bool Q8>
__global__ __launch_bounds__(kBlock) void adamw_kernel(const AdamBatch b, const AdamArgs a) {
    __shared__ float top[2][kBlock / 64];
    float gs = 1.f;
    if (a.grad_scale) {
        gs = *a.grad_scale;
        if (gs != gs) return;
    }
    const AdamSeg& s = b.s[find_seg(b, blockIdx.x)];
    const int64_t blk = blockIdx.x - s.blk0;
    const int64_t i = blk * kBlock + threadIdx.x;
    const bool in = i < s.n;
    const float g = in ? load_elem<GT>(s.g, i) * gs : 0.f;
    float w = in ? load_elem<WT>(s.w, i) : 0.f;
    float m = 0.f, u;
    if constexpr (Q8) {
        m = e4m3_to_f32(static_cast<uint8_t*>(s.m)[i]) *
            __uint_as_float((uint32_t)s.ms[blk] << 23);
        u = e4m3_to_f32(static_cast<uint8_t*>(s.v)[i]) *
            __uint_as_float((uint32_t)s.vs[blk] << 23);
        m = a.b1 * m + a.c1 * g;
        u = sqrtf(a.b2 * (u * u) + a.c2 * (g * g));
    } else {
        float v = 0.f;
        if (in) {
            m = a.b1 * static_cast<float*>(s.m)[i] + a.c1 * g;
            v = a.b2 * static_cast<float*>(s.v)[i] + a.c2 * (g * g);
            static_cast<float*>(s.m)[i] = m;
            static_cast<float*>(s.v)[i] = v;
        }
        u = sqrtf(v);
    }
    w = w * a.decay - a.lr * (m / (u * a.rcorr + a.eps));
    uint32_t r = 0, rm = 0, ru = 0;
    if constexpr (Q8) {
        const int64_t k = i / 4;
        const u32x4 q = philox_words((uint32_t)k, (uint32_t)(k >> 32), s.stream, a.k0, a.k1);
        r = q[i & 3] & 0xFFFFu;
        rm = q[i & 3] >> 16;
        ru = q[(i + 1) & 3] >> 16;
    } else if (WT != HASTE_DTYPE_F32 && a.do_sr) {
        const int64_t k = i / 8;
        const u32x4 q = philox_words((uint32_t)k, (uint32_t)(k >> 32), s.stream, a.k0, a.k1);
        r = (q[(i & 7) >> 1] >> (16 * (i & 1))) & 0xFFFFu;
    }
    if (in) {
        if (WT != HASTE_DTYPE_F32 && a.do_sr)
            static_cast<uint16_t*>(s.w)[i] = (uint16_t)cut_16<WT>(w, r);
        else
            store_elem<WT>(s.w, i, w);
    }
    if constexpr (Q8) {
        float tm = fabsf(m) < INFINITY ? fabsf(m) : 0.f, tu = u < INFINITY ? u : 0.f;
        for (int o = 32; o; o >>= 1) {
            tm = fmaxf(tm, __shfl_xor(tm, o));
            tu = fmaxf(tu, __shfl_xor(tu, o));
        }
        if ((threadIdx.x & 63) == 0) {
            top[0][threadIdx.x >> 6] = tm;
            top[1][threadIdx.x >> 6] = tu;
        }
        __syncthreads();
        const int em = max((int)(__float_as_uint(fmaxf(top[0][0], top[0][1])) >> 23) - 7, 1);
        const int eu = max((int)(__float_as_uint(fmaxf(top[1][0], top[1][1])) >> 23) - 7, 1);
        static_cast<uint8_t*>(s.m)[i] =
            (uint8_t)cut_e4m3<false>(m * __uint_as_float((uint32_t)(254 - em) << 23), rm);
        static_cast<uint8_t*>(s.v)[i] =
            (uint8_t)cut_e4m3<true>(u * __uint_as_float((uint32_t)(254 - eu) << 23), ru);
        if (threadIdx.x == 0) {
            s.ms[blk] = (uint8_t)em;
            s.vs[blk] = (uint8_t)eu;
        }
    }
}

constexpr int kNormThreads = 256;
constexpr int kNormElems = 16384;       // elements of a workgroup
constexpr int kNormParts = 2048;        // partial sums of a launch

__device__ __forceinline__ double wave_sum(double v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// part[block] = the sum of squares of the block's pieces, every gridDim.x-th of the launch's.
__global__ __launch_bounds__(kNormThreads) void grad_norm_kernel(const GradBatch b, uint32_t pieces,
                                                                 double* part) {
    __shared__ double sums[kNormThreads / 64];
    double total = 0.0;
    for (uint32_t p = blockIdx.x; p < pieces; p += gridDim.x) {
        const GradSeg& s = b.s[find_seg(b, p)];
        const int64_t i0 = (int64_t)(p - s.blk0) * kNormElems;
        const int64_t i1 = min(s.n, i0 + kNormElems);
        for (int64_t i = i0 + threadIdx.x; i < i1; i += kNormThreads) {
            const float g = s.dtype == HASTE_DTYPE_BF16  ? load_elem<HASTE_DTYPE_BF16>(s.g, i)
                            : s.dtype == HASTE_DTYPE_F16 ? load_elem<HASTE_DTYPE_F16>(s.g, i)
                                                         : load_elem<HASTE_DTYPE_F32>(s.g, i);
            total += (double)g * (double)g;
        }
    }
    total = wave_sum(total);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = total;
    __syncthreads();
    if (threadIdx.x) return;
    for (int k = 1; k < kNormThreads / 64; ++k) total += sums[k];
    part[blockIdx.x] = total;
}

__global__ __launch_bounds__(kNormThreads) void grad_norm_final_kernel(const double* part,
                                                                       int64_t parts, float max_norm,
                                                                       float* out) {
    __shared__ double sums[kNormThreads / 64];
    double total = 0.0;
    for (int64_t i = threadIdx.x; i < parts; i += kNormThreads) total += part[i];
    total = wave_sum(total);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = total;
    __syncthreads();
    if (threadIdx.x) return;
    for (int k = 1; k < kNormThreads / 64; ++k) total += sums[k];
    const float norm = (float)sqrt(total);
    out[0] = norm;
    out[1] = norm < INFINITY ? fminf(1.f, max_norm / (norm + 1e-6f)) : NAN;
}

template <int WT, int GT, bool Q8>
int launch_adamw(const haste_adamw_tensor* ts, int count, const AdamArgs& a, hipStream_t st) {
    for (int base = 0; base < count;) {
        AdamBatch b;
        b.count = 0;
        int64_t blocks = 0;
        for (; base < count && b.count < kMaxSegs; ++base) {
            const haste_adamw_tensor& t = ts[base];
            if (t.n == 0) continue;
            b.s[b.count++] = AdamSeg{t.w, t.g, t.m, t.v, t.m_scale, t.v_scale, t.n,
                                     (uint32_t)blocks, t.stream};
            blocks += ceil_div(t.n, kBlock);
            HASTE_CHECK_ARG(blocks < (int64_t)1 << 31, "haste_adamw_step: tensors too large");
        }
        if (b.count == 0) break;
        adamw_kernel<WT, GT, Q8><<<dim3((unsigned)blocks), dim3(kBlock), 0, st>>>(b, a);
        HASTE_CHECK_LAUNCH("haste_adamw_step");
    }
    return HASTE_OK;
}

}  // namespace
}  // namespace haste

extern "C" int haste_adamw_step(const haste_adamw_tensor* tensors, int32_t count, int32_t w_dtype,
                                int32_t g_dtype, int32_t state_bits, double lr, double beta1,
                                double beta2, double eps, double wd, int64_t step, int32_t do_sr,
                                uint64_t seed, const float* grad_scale, void* stream) {
    const char* fn = "haste_adamw_step";
    HASTE_CHECK_ARG(count >= 0 && (count == 0 || tensors != nullptr), "%s: bad tensor list", fn);
    HASTE_CHECK_ARG(haste::elem_dtype(w_dtype) && haste::elem_dtype(g_dtype),
                    "%s: weights and gradients must be bf16, fp16 or fp32 (dtype codes %d, %d)", fn,
                    (int)w_dtype, (int)g_dtype);
    HASTE_CHECK_ARG(state_bits == 8 || state_bits == 32, "%s: states must have 8 or 32 bits (got %d)",
                    fn, (int)state_bits);
    HASTE_CHECK_ARG(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0,
                    "%s: betas must be in [0, 1) and eps >= 0", fn);
    HASTE_CHECK_ARG(step >= 1, "%s: step must be >= 1 (got %lld)", fn, (long long)step);
    HASTE_CHECK_ARG((reinterpret_cast<uintptr_t>(grad_scale) & 3u) == 0, "%s: grad_scale misaligned",
                    fn);
    const bool q8 = state_bits == 8;
    for (int k = 0; k < count; ++k) {
        const haste_adamw_tensor& t = tensors[k];
        HASTE_CHECK_ARG(t.n >= 0, "%s: tensor %d: n must be >= 0", fn, k);
        if (t.n == 0) continue;
        HASTE_CHECK_ARG(t.w && t.g && t.m && t.v && (!q8 || (t.m_scale && t.v_scale)),
                        "%s: tensor %d: null pointer", fn, k);
        const uintptr_t st = reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v);
        HASTE_CHECK_ARG(haste::elem_aligned(t.w, w_dtype) && haste::elem_aligned(t.g, g_dtype) &&
                            (st & (q8 ? 7u : 15u)) == 0,
                        "%s: tensor %d is misaligned", fn, k);
    }
    haste::AdamArgs a{};
    a.b1 = (float)beta1;
    a.c1 = (float)(1.0 - beta1);
    a.b2 = (float)beta2;
    a.c2 = (float)(1.0 - beta2);
    a.decay = (float)(1.0 - lr * wd);
    a.lr = (float)(lr / (1.0 - std::pow(beta1, (double)step)));
    a.rcorr = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
    a.eps = (float)eps;
    a.k0 = (uint32_t)seed;
    a.k1 = (uint32_t)(seed >> 32);
    a.do_sr = do_sr != 0;
    a.grad_scale = grad_scale;
    hipStream_t st = static_cast<hipStream_t>(stream);
#define HASTE_ADAMW(WT, GT)                                                                 \
    if (w_dtype == WT && g_dtype == GT)                                                     \
        return q8 ? haste::launch_adamw<WT, GT, true>(tensors, count, a, st)                \
                  : haste::launch_adamw<WT, GT, false>(tensors, count, a, st)
    HASTE_ADAMW(HASTE_DTYPE_BF16, HASTE_DTYPE_BF16);
    HASTE_ADAMW(HASTE_DTYPE_BF16, HASTE_DTYPE_F16);
    HASTE_ADAMW(HASTE_DTYPE_BF16, HASTE_DTYPE_F32);
    HASTE_ADAMW(HASTE_DTYPE_F16, HASTE_DTYPE_BF16);
    HASTE_ADAMW(HASTE_DTYPE_F16, HASTE_DTYPE_F16);
    HASTE_ADAMW(HASTE_DTYPE_F16, HASTE_DTYPE_F32);
    HASTE_ADAMW(HASTE_DTYPE_F32, HASTE_DTYPE_BF16);
    HASTE_ADAMW(HASTE_DTYPE_F32, HASTE_DTYPE_F16);
    HASTE_ADAMW(HASTE_DTYPE_F32, HASTE_DTYPE_F32);
#undef HASTE_ADAMW
    return HASTE_ERR_UNSUPPORTED;
}

extern "C" int64_t haste_grad_norm_workspace_size(int32_t count) {
    if (count < 0) return HASTE_ERR_INVALID_ARG;
    return haste::ceil_div(std::max(count, 1), haste::kMaxSegs) * haste::kNormParts *
           (int64_t)sizeof(double);
}

extern "C" int haste_grad_norm(const haste_grad_tensor* tensors, int32_t count, double max_norm,
                               float* out, void* ws, int64_t ws_bytes, void* stream) {
    const char* fn = "haste_grad_norm";
    HASTE_CHECK_ARG(count >= 0 && (count == 0 || tensors != nullptr), "%s: bad tensor list", fn);
    HASTE_CHECK_ARG(out != nullptr && (reinterpret_cast<uintptr_t>(out) & 3u) == 0,
                    "%s: out is NULL or misaligned", fn);
    HASTE_CHECK_ARG(max_norm >= 0.0, "%s: max_norm must be >= 0", fn);
    HASTE_CHECK_ARG(ws != nullptr && (reinterpret_cast<uintptr_t>(ws) & 7u) == 0,
                    "%s: workspace is NULL or misaligned", fn);
    if (ws_bytes < haste_grad_norm_workspace_size(count)) {
        haste::set_error("%s: workspace too small (%lld < %lld bytes)", fn, (long long)ws_bytes,
                         (long long)haste_grad_norm_workspace_size(count));
        return HASTE_ERR_WORKSPACE;
    }
    for (int k = 0; k < count; ++k) {
        const haste_grad_tensor& t = tensors[k];
        HASTE_CHECK_ARG(t.n >= 0, "%s: tensor %d: n must be >= 0", fn, k);
        HASTE_CHECK_ARG(haste::elem_dtype(t.dtype),
                        "%s: tensor %d must be bf16, fp16 or fp32 (dtype code %d)", fn, k,
                        (int)t.dtype);
        HASTE_CHECK_ARG(t.n == 0 || (t.g && haste::elem_aligned(t.g, t.dtype)),
                        "%s: tensor %d is NULL or misaligned", fn, k);
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    double* part = static_cast<double*>(ws);
    int64_t parts = 0;
    for (int base = 0; base < count;) {
        haste::GradBatch b;
        b.count = 0;
        int64_t pieces = 0;
        for (; base < count && b.count < haste::kMaxSegs; ++base) {
            const haste_grad_tensor& t = tensors[base];
            if (t.n == 0) continue;
            b.s[b.count++] = haste::GradSeg{t.g, t.n, t.dtype, (uint32_t)pieces};
            pieces += haste::ceil_div(t.n, (int64_t)haste::kNormElems);
            HASTE_CHECK_ARG(pieces < (int64_t)1 << 31, "%s: tensors too large", fn);
        }
        if (b.count == 0) break;
        const int64_t blocks = std::min<int64_t>(pieces, haste::kNormParts);
        haste::grad_norm_kernel<<<dim3((unsigned)blocks), dim3(haste::kNormThreads), 0, st>>>(
            b, (uint32_t)pieces, part + parts);
        HASTE_CHECK_LAUNCH(fn);
        parts += blocks;
    }
    haste::grad_norm_final_kernel<<<dim3(1), dim3(haste::kNormThreads), 0, st>>>(
        part, parts, (float)max_norm, out);
    HASTE_CHECK_LAUNCH(fn);
    return HASTE_OK;
}
