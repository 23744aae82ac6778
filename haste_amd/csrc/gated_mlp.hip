// The gated feed-forward block, y = (act(x Wg^T) * (x Wu^T)) Wd^T, and its gradients (gated_mlp.hpp has
// the formulas).  Bound by its matrix products: 6 N D H operations forward, 12 N D H backward, as
//   forward   [g | u] with h in the epilogue;  y
//   backward  dh with dg and du in the epilogue;  dx over both;  dWg and dWu;  dWd
// A few tokens in serving are bound by reading the weights once and take kernels of their own.
// Measured in bf16 at widths 768 and 2048: one row 4.8 + 4.9 us (9.4 MB, two launches' latency); 509 rows 11 + 10
// + 4 us (latency of few workgroups); 65,536 rows forward 565 to 626 (412 GFLOP, and 1.07 GB written) + 233 us,
// backward 430 to 455 + 427 + 410 + 224 us.  At 16,384 rows, widths 4096 and 8192: 1913 + 978 and 1126 + 1944 +
// 1823 + 917 us, 1.13 to 1.2 PFLOP/s.
#include <algorithm>

#include "gated_mlp.hpp"
#include "gemm.hpp"
#include "launches.hpp"

namespace haste {
namespace {

template <typename Tile, int DT, typename Epilogue>
__global__ __launch_bounds__(Tile::kThreads, 2) void gemm_kernel(GemmArgs g, int batches, int act,
                                                                 Epilogue out) {
    __shared__ __attribute__((aligned(16))) char lds[Tile::kLdsBytes];
    GemmPlace p;
    if (!gemm_place(g, batches, &p)) return;
    Tile t;
    t.run(g, lds, p.tm, p.tn, p.batch, p.split);
    const int lane = threadIdx.x & 63;
    constexpr int F = Tile::kDual ? Tile::FN / 2 : Tile::FN;
    // f(row of tiles, row of C, first column of the lane, its sums)
    auto rows = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
        for (int fm = 0; fm < Tile::FM; ++fm) {
            f32x4 v[F], w[F];
#pragma unroll
            for (int k = 0; k < F; ++k) {
                v[k] = t.acc[k][fm];
                w[k] = t.acc[Tile::FN - F + k][fm];
            }
            const int n = t.n0 + gather_columns<F>(v, lane);
            if (Tile::kDual) gather_columns<F>(w, lane);
            f(fm, t.m0 + fm * 16 + (lane & 15), n, v, w);
        }
    };
    if constexpr (std::is_same<Epilogue, PlainOut>::value) {
        rows([&](int, int m, int n, auto& v, auto&) __attribute__((always_inline)) {
            if (m < g.M && n < g.N) out.template put<DT, F>(p.split, p.batch, m, n, v);
        });
    } else if constexpr (std::is_same<Epilogue, GatedGrad>::value) {
        // the next rows' kept values are on their way while these are used
        Kept<DT> slope[2], kept_act[2];
        const int col = min(t.n0 + 16 * (lane >> 4), (int)out.ld - 16);
        auto fetch = [&](int fm) __attribute__((always_inline)) {
            const int m = min(t.m0 + fm * 16 + (lane & 15), g.M - 1);
            const char* block = out.kept.template block<DT>(m, col);
            slope[fm & 1] = load_kept<DT>(block, m, col);
            kept_act[fm & 1] = load_kept<DT>(block + kKeptBlock<DT>, m, col);
        };
        fetch(0);
        rows([&](int fm, int m, int n, auto& v, auto&) __attribute__((always_inline)) {
            if (fm + 1 < Tile::FM) fetch(fm + 1);
            if (m < g.M && n < out.ld) out.template put<DT, F>(m, n, v, slope[fm & 1], kept_act[fm & 1]);
        });
    } else {
        with_activation(act, [&](auto a) __attribute__((always_inline)) {
            rows([&](int, int m, int n, auto& vg, auto& vu) __attribute__((always_inline)) {
                if (m < g.M && n < out.ld) out.template put<DT, decltype(a)::value, F>(m, n, vg, vu);
            });
        });
    }
}

// --------------------------------------------------------------- a few rows ----
// Up to 16 NG rows of x against 16 rows of the weights (of both, DUAL): the waves share K, and read
// the weights straight into registers, at any alignment.  fp32 weights are split there; x is too (DUAL), or
// comes as its parts, `plane` bytes apart.
template <typename T, int NG, bool DUAL, int WAVES, typename Epilogue>
__global__ __launch_bounds__(64 * WAVES) void few_rows_kernel(const char* x, int64_t ldx, int64_t plane,
                                                             const char* w0, int64_t ldw0,
                                                             const char* w1, int64_t ldw1, int M, int N,
                                                             int K, int act, Epilogue out) {
    constexpr int DT = T::code, NW = DUAL ? 2 : 1, P = DT == HASTE_DTYPE_F32 ? 3 : 1, SZ = kElemBytes<DT>;
    typedef typename std::conditional<P == 3, BF16, T>::type MT;
    __shared__ f32x4 sums[WAVES][NG * NW][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15;
    const int n = blockIdx.x * 16 + r;
    const char* w[2] = {w0 + (int64_t)min(n, N - 1) * ldw0 * SZ,
                        DUAL ? w1 + (int64_t)min(n, N - 1) * ldw1 * SZ : w0};
    f32x4 acc[NG * NW];
#pragma unroll
    for (int i = 0; i < NG * NW; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    struct Piece {
        u32x4 p[P];
    };
    // eight elements: one fragment, or three
    auto piece = [](const char* p, int64_t i, int64_t count) __attribute__((always_inline)) {
        Piece f;
        if constexpr (P == 1) {
            const Elems<DT, 8> v = load_part<DT, 8>(p, i, count);
            f.p[0] = u32x4{v.q[0], v.q[1], v.q[2], v.q[3]};
        } else {
            float v[8];
            unpack<DT, 8>(load_part<DT, 8>(p, i, count), v);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t lo[3], hi[3];
                split_f32(v[2 * k], lo);
                split_f32(v[2 * k + 1], hi);
#pragma unroll
                for (int j = 0; j < P; ++j) f.p[j][k] = lo[j] | hi[j] << 16;
            }
        }
        return f;
    };
    auto rows = [&](int i, int k) __attribute__((always_inline)) {
        const int m = 16 * i + r, count = m < M ? K - k : 0;
        if constexpr (P == 1 || DUAL) return piece(x + (int64_t)m * ldx * SZ, k, count);
        Piece f;
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const Elems<HASTE_DTYPE_BF16, 8> v =
                load_part<HASTE_DTYPE_BF16, 8>(x + j * plane + (int64_t)m * ldx * 2, k, count);
            f.p[j] = u32x4{v.q[0], v.q[1], v.q[2], v.q[3]};
        }
        return f;
    };
#pragma unroll 4
    for (int k0 = wave * 32; k0 < K; k0 += 32 * WAVES) {
        const int k = k0 + 8 * (lane >> 4);
        Piece fw[NW], fx[NG];
#pragma unroll
        for (int i = 0; i < NW; ++i) fw[i] = piece(w[i], k, n < N ? K - k : 0);
#pragma unroll
        for (int i = 0; i < NG; ++i) fx[i] = rows(i, k);
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int j = 0; j < NW; ++j) {
                f32x4& c = acc[i * NW + j];
                if constexpr (P == 1) {
                    c = mfma16x16x32<MT>(fw[j].p[0], fx[i].p[0], c);
                } else {
#pragma unroll
                    for (int q = 0; q < 6; ++q)
                        c = mfma16x16x32<MT>(fw[j].p[kPartsOfB >> (2 * q) & 3], fx[i].p[kPartsOfA >> (2 * q) & 3], c);
                }
            }
    }
#pragma unroll
    for (int i = 0; i < NG * NW; ++i) sums[wave][i][lane] = acc[i];
    __syncthreads();
    for (int i = wave; i < NG; i += WAVES) {
        f32x4 s[NW][1];
#pragma unroll
        for (int j = 0; j < NW; ++j) {
            s[j][0] = sums[0][i * NW + j][lane];
            for (int v = 1; v < WAVES; ++v) s[j][0] += sums[v][i * NW + j][lane];
        }
        const int m = 16 * i + r, col = blockIdx.x * 16 + 4 * (lane >> 4);
        if (m >= M) continue;
        if constexpr (DUAL) {
            if (col < out.ld)
                with_activation(act, [&](auto a) __attribute__((always_inline)) {
                    out.template put<DT, decltype(a)::value, 1>(m, col, s[0], s[1]);
                });
        } else {
            if (col < N) out.template put<DT, 1>(0, 0, m, col, s[0]);
        }
    }
}

// Matrices [R, C] of any pitch as rows of P (a multiple of 8) elements on 16 bytes, with zeros behind C;
// fp32 ones as their three parts.  One launch for all that a call has (or as many as they need: `first` is
// the launch's first workgroup).
constexpr int kMaxPacks = 5;
struct Packs {
    struct {
        const char* src;
        char* dst;
        int64_t ld, R, C, P;
        uint32_t block0;  // its first workgroup
    } m[kMaxPacks];
    int count;
};
template <bool F32>
__global__ __launch_bounds__(256) void pack_rows_kernel(Packs p, uint32_t first) {
    constexpr int DT = F32 ? HASTE_DTYPE_F32 : HASTE_DTYPE_BF16;
    const uint32_t block = first + blockIdx.x;
    int k = 0;
    for (int j = 1; j < p.count; ++j) k = block >= p.m[j].block0 ? j : k;
    const auto& m = p.m[k];
    const int64_t i = (int64_t)(block - m.block0) * 256 + threadIdx.x, pieces = m.P / 8;
    if (i >= m.R * pieces) return;
    const int64_t r = i / pieces, c = i % pieces * 8;
    const Elems<DT, 8> v = load_part<DT, 8>(m.src + r * m.ld * kElemBytes<DT>, c, m.C - c);
    if constexpr (F32) {
        float f[8];
        unpack<DT, 8>(v, f);
        const f32x4 w[2] = {{f[0], f[1], f[2], f[3]}, {f[4], f[5], f[6], f[7]}};
        put_operand<DT, 2>(m.dst, m.R * m.P * 2, r * m.P + c, w);
    } else {
        store<DT, 8>(m.dst, r * m.P + c, v);
    }
}

// ------------------------------------------------------------------ host ----
constexpr int64_t kMaxSide = (int64_t)1 << 20;  // a tile's rows span less than 2^31 bytes
constexpr int kFewRows = 64;

int64_t round8(int64_t n) { return ceil_div(n, 8) * 8; }
int64_t round16(int64_t n) { return ceil_div(n, 16) * 16; }  // (the pitch of h and its like)
int64_t kept_blocks(int64_t H) { return ceil_div(H, 64); }
// h, dg or du: of the type, fp32 as three bf16 parts.
int64_t hidden_bytes(int64_t N, int64_t ld, int32_t dtype) {
    return N * ld * 2 * (dtype == HASTE_DTYPE_F32 ? 3 : 1);
}

// A matrix as the kernels take it.
struct Matrix {
    const void* p;
    int64_t ld, rows, cols;
    int64_t plane = 0;  // fp32 as three parts: bytes between them
};
bool plain_rows(const Matrix& m) { return aligned16(m.p) && m.ld % 8 == 0 && m.cols % 8 == 0; }

// The workspace's places, handed out in order.
struct Space {
    char* base;
    int64_t used = 0;
    void* take(int64_t bytes) {
        void* p = base ? base + used : nullptr;
        used += ceil_div(bytes, 256) * 256;
        return p;
    }
};

struct Product {
    Matrix a[2], b[2];  // two of each where the mode has two, of one pitch
    int64_t M, N, K;
};

template <int DT>
struct TypeOf;
template <>
struct TypeOf<HASTE_DTYPE_BF16> {
    typedef BF16 type;
};
template <>
struct TypeOf<HASTE_DTYPE_F16> {
    typedef F16 type;
};
template <>
struct TypeOf<HASTE_DTYPE_F32> {
    typedef F32Parts type;
};

template <typename Tile>
GemmArgs gemm_args(const Product& p, int segments, int splits) {
    GemmArgs g{};
    for (int i = 0; i < 2; ++i) {
        g.a.base[i] = static_cast<const char*>(p.a[i].p);
        g.b.base[i] = static_cast<const char*>(p.b[i].p);
    }
    g.a.ld = p.a[0].ld;
    g.b.ld = p.b[0].ld;
    g.a.plane = p.a[0].plane;
    g.b.plane = p.b[0].plane;
    g.M = (int)p.M;
    g.N = (int)p.N;
    g.K = (int)p.K;
    g.tiles_m = (int)ceil_div(p.M, Tile::BM);
    g.tiles_n = (int)ceil_div(p.N, Tile::kCols);
    g.steps = (int)ceil_div(p.K, Tile::KS);
    g.splits = (int)std::max<int64_t>(1, std::min<int64_t>(splits, (int64_t)g.steps * segments * Tile::kProducts));
    return g;
}

template <typename Tile, int DT, typename Epilogue>
void launch_tiles(const GemmArgs& g, int batches, int act, const Epilogue& out, hipStream_t st) {
    const int64_t n = (int64_t)g.tiles_m * g.tiles_n * batches * g.splits;
    gemm_kernel<Tile, DT, Epilogue><<<dim3((unsigned)(ceil_div(n, 8) * 8)), dim3(Tile::kThreads), 0, st>>>(
        g, batches, act, out);
}

// How a product is cut.  Tiles of 256 x 256 (a workgroup to a CU) where they fill most of the GPU's 256
// CUs, by themselves or with K in parts; else of 128 x 128, two workgroups to a CU; else, where those
// leave half of the CUs idle, of 64 x 128: the time is then that of a tile's steps and epilogue (509 rows,
// H = 2048: 28.8 -> 24.9 us for the block; 512 rows, H = 8192, with the first rule left out: 162 -> 198).
enum class Tiles { kLarge, kSmall, kLow };
struct Cut {
    Tiles tiles;
    int splits;
};
template <GemmMode MODE, int DT>
Cut cut_of(const Product& p, bool may_split) {
    const int64_t batches = MODE == GemmMode::kBatch ? 2 : 1;
    const int64_t products = DT == HASTE_DTYPE_F32 ? 6 : 1;
    const int64_t steps = ceil_div(p.K, 32) * (MODE == GemmMode::kSegments ? 2 : 1) * products;
    auto tiles = [&](int64_t rows, int64_t cols) {
        return ceil_div(p.M, rows) * ceil_div(p.N, MODE == GemmMode::kDual ? cols / 2 : cols) * batches;
    };
    const int64_t big = tiles(256, 256), small = tiles(128, 128), low = tiles(64, 128);
    // (16 steps to a part at least)
    auto splits = [&](int64_t n) {
        return may_split ? std::max<int64_t>(1, std::min(256 / n, steps / 16)) : 1;
    };
    if (small == 0) return Cut{Tiles::kSmall, 1};
    if (big >= 192) return Cut{Tiles::kLarge, 1};
    if (may_split && steps / 32 >= ceil_div(192, big)) return Cut{Tiles::kLarge, (int)(256 / big)};
    if (small * splits(small) <= 128) return Cut{Tiles::kLow, (int)splits(low)};
    return Cut{Tiles::kSmall, (int)splits(small)};
}

template <int DT, GemmMode MODE, bool AK, bool BK_, typename Epilogue>
void product(const Product& p, Cut cut, int act, const Epilogue& out, hipStream_t st) {
    constexpr int batches = MODE == GemmMode::kBatch ? 2 : 1, segments = MODE == GemmMode::kSegments ? 2 : 1;
    typedef typename TypeOf<DT>::type T;
    typedef GemmTile<T, MODE, AK, BK_, 8, 4, 2, 4, 4> Large;
    typedef GemmTile<T, MODE, AK, BK_, 4, 4, 2, 2, 4> Small;
    if constexpr (!std::is_same<Epilogue, PlainOut>::value && DT != HASTE_DTYPE_F32) {
        // An epilogue that moves 8 to 10 bytes an element takes longer than a short K: two workgroups
        // to a CU, of 256 x 128, overlap one's with the other's products (65536 x 2048 elements, K =
        // 768: h 585 -> 565 us, dg and du 473 -> 430; 16384 x 8192, K = 4096: 1922 -> 2193, 1131 ->
        // 1308, since they load half as much again).  In between, for the whole forward of 65536 x 2048:
        // K = 1280 1097 -> 1119 us, 1536 1245 -> 1284, 2048 1549 -> 1635; 16384 x 8192: K = 1280 the same.
        typedef GemmTile<T, MODE, AK, BK_, 8, 4, 2, 2, 3> Half;
        if (cut.tiles == Tiles::kLarge && p.K <= 1024)
            return launch_tiles<Half, DT>(gemm_args<Half>(p, segments, cut.splits), batches, act, out, st);
    }
    typedef GemmTile<T, MODE, AK, BK_, 2, 4, 2, 2, 4> Low;
    if (cut.tiles == Tiles::kLarge)
        launch_tiles<Large, DT>(gemm_args<Large>(p, segments, cut.splits), batches, act, out, st);
    else if (cut.tiles == Tiles::kSmall)
        launch_tiles<Small, DT>(gemm_args<Small>(p, segments, cut.splits), batches, act, out, st);
    else
        launch_tiles<Low, DT>(gemm_args<Low>(p, segments, cut.splits), batches, act, out, st);
}

// A product without an epilogue, its parts of K joined by a second launch.  `parts` has room for
// plain_parts() bytes.
template <int DT, GemmMode MODE>
int64_t plain_parts(const Product& p) {
    const int splits = cut_of<MODE, DT>(p, true).splits;
    return splits == 1 ? 0
                       : splits * (MODE == GemmMode::kBatch ? 2 : 1) * p.M * (ceil_div(p.N, 16) * 16) * 4;
}
template <int DT, GemmMode MODE, bool AK, bool BK_>
void plain(const Product& p, void* c0, void* c1, void* parts, hipStream_t st) {
    const Cut cut = cut_of<MODE, DT>(p, true);
    const int splits = cut.splits;
    PlainOut out{{c0, c1}, p.N, splits > 1 ? static_cast<float*>(parts) : nullptr, (int)p.M, (int)p.N,
                 MODE == GemmMode::kBatch ? 2 : 1};
    product<DT, MODE, AK, BK_>(p, cut, 0, out, st);
    if (splits > 1) {
        const int64_t n = out.batches * p.M * (out.pitch() / 4);
        sum_parts_kernel<DT><<<dim3((unsigned)ceil_div(n, 256)), dim3(256), 0, st>>>(out, splits);
    }
}

struct Sizes {
    int64_t N, D, H, O;
};

// Matrices with 16-byte rows (fp32: their parts): themselves, or copies in the workspace, made by one launch.
struct Packer {
    Packs packs{};
    uint32_t blocks = 0;  // (five matrices of up to 2^40 elements, 2^11 to a workgroup: under 2^32)
    template <int DT>
    Matrix add(const Matrix& m, Space& ws, bool used, bool as_it_lies = true) {
        constexpr bool parts = DT == HASTE_DTYPE_F32;
        if (!parts && as_it_lies && plain_rows(m)) return m;
        const int64_t P = round8(m.cols), plane = parts ? m.rows * P * 2 : 0;
        void* to = ws.take(m.rows * P * 2 * (parts ? 3 : 1));
        if (used && m.rows > 0) {
            packs.m[packs.count++] = {static_cast<const char*>(m.p), static_cast<char*>(to), m.ld,
                                      m.rows, m.cols, P, blocks};
            blocks += (uint32_t)ceil_div(m.rows * (P / 8), 256);
        }
        return Matrix{to, P, m.rows, m.cols, plane};
    }
    // Two operands of one product, which have one pitch: both as they lie or both as copies.
    template <int DT>
    void add_pair(Matrix& a, Matrix& b, Space& ws, bool used) {
        const bool as_they_lie = plain_rows(a) && plain_rows(b) && a.ld == b.ld;
        a = add<DT>(a, ws, used, as_they_lie);
        b = add<DT>(b, ws, used, as_they_lie);
    }
    template <int DT>
    void launch(hipStream_t st) const {
        in_launches_of(blocks, 256, [&](int64_t first, int64_t count) {
            pack_rows_kernel<DT == HASTE_DTYPE_F32>
                <<<dim3((unsigned)count), dim3(256), 0, st>>>(packs, (uint32_t)first);
        });
    }
};

template <int DT>
int64_t forward(const Sizes& s, Matrix x, Matrix wg, Matrix wu, Matrix wd, const GatedOut& out, void* y,
                int act, char* base, bool launch, hipStream_t st) {
    Space ws{base};
    if (s.N <= kFewRows) {
        if (!launch) return 0;
        typedef typename TypeOf<DT>::type T;
        const char *xc = static_cast<const char*>(x.p), *gc = static_cast<const char*>(wg.p),
                   *uc = static_cast<const char*>(wu.p), *dc = static_cast<const char*>(wd.p),
                   *hc = static_cast<const char*>(out.h);
        const dim3 g1((unsigned)ceil_div(out.ld, 16)), g2((unsigned)ceil_div(s.O, 16));
        const PlainOut po{{y, nullptr}, s.O, nullptr, (int)s.N, (int)s.O, 1};
        auto run = [&](auto groups) {
            constexpr int NG = decltype(groups)::value;
            few_rows_kernel<T, NG, true, 8, GatedOut><<<g1, dim3(512), 0, st>>>(
                xc, x.ld, 0, gc, wg.ld, uc, wu.ld, (int)s.N, (int)s.H, (int)s.D, act, out);
            few_rows_kernel<T, NG, false, 16, PlainOut><<<g2, dim3(1024), 0, st>>>(
                hc, out.ld, out.plane, dc, wd.ld, nullptr, 0, (int)s.N, (int)s.O, (int)s.H, 0, po);
        };
        if (s.N <= 16) run(std::integral_constant<int, 1>());
        else if (s.N <= 32) run(std::integral_constant<int, 2>());
        else run(std::integral_constant<int, 4>());
        return 0;
    }
    Packer packer;
    x = packer.add<DT>(x, ws, true);
    packer.add_pair<DT>(wg, wu, ws, true);
    wd = packer.add<DT>(wd, ws, true);
    const Matrix h{out.h, out.ld, s.N, s.H, out.plane};
    const Product p1{{x, x}, {wg, wu}, s.N, s.H, s.D};
    const Product p2{{h, h}, {wd, wd}, s.N, s.O, s.H};
    void* parts = ws.take(plain_parts<DT, GemmMode::kPlain>(p2));
    if (launch) {
        packer.launch<DT>(st);
        product<DT, GemmMode::kDual, true, true>(p1, cut_of<GemmMode::kDual, DT>(p1, false), act, out,
                                                 st);
        plain<DT, GemmMode::kPlain, true, true>(p2, y, nullptr, parts, st);
    }
    return ws.used;
}

struct Grads {
    void *dx, *dwg, *dwu, *dwd;
};

template <int DT>
int64_t backward(const Sizes& s, Matrix x, Matrix wg, Matrix wu, Matrix wd, Matrix dy,
                 void* kept, const void* h, int64_t ld, const Grads& to, char* base,
                 bool launch, hipStream_t st) {
    Space ws{base};
    const int64_t plane = DT == HASTE_DTYPE_F32 ? s.N * ld * 2 : 0, bytes = hidden_bytes(s.N, ld, DT);
    void *dg = ws.take(bytes), *du = ws.take(bytes);
    Packer packer;
    if (s.N > 0) {  // (without rows the products of K = 0 read nothing)
        x = packer.add<DT>(x, ws, to.dwg || to.dwu);
        packer.add_pair<DT>(wg, wu, ws, to.dx);
        wd = packer.add<DT>(wd, ws, to.dx || to.dwg || to.dwu);
        dy = packer.add<DT>(dy, ws, true);
    }
    const Matrix mg{dg, ld, s.N, s.H, plane}, mu{du, ld, s.N, s.H, plane}, mh{h, ld, s.N, s.H, plane};
    const Product p1{{dy, dy}, {wd, wd}, s.N, s.H, s.O};
    const Product p2{{mg, mu}, {wg, wu}, s.N, s.D, s.H};
    const Product p3{{mg, mu}, {x, x}, s.H, s.D, s.N};
    const Product p4{{dy, dy}, {mh, mh}, s.O, s.H, s.N};
    void* parts = ws.take(std::max({plain_parts<DT, GemmMode::kSegments>(p2),
                                    plain_parts<DT, GemmMode::kBatch>(p3),
                                    plain_parts<DT, GemmMode::kPlain>(p4)}));
    if (launch) {
        packer.launch<DT>(st);
        if (s.N > 0 && (to.dx || to.dwg || to.dwu)) {
            const GatedGrad out{{kept, kept_blocks(s.H)}, dg, du, ld, plane, (int)s.H};
            product<DT, GemmMode::kPlain, true, false>(p1, cut_of<GemmMode::kPlain, DT>(p1, false), 0, out,
                                                       st);
        }
        if (s.N > 0 && to.dx) plain<DT, GemmMode::kSegments, true, false>(p2, to.dx, nullptr, parts, st);
        if (to.dwg || to.dwu) plain<DT, GemmMode::kBatch, false, false>(p3, to.dwg, to.dwu, parts, st);
        if (to.dwd) plain<DT, GemmMode::kPlain, false, false>(p4, to.dwd, nullptr, parts, st);
    }
    return ws.used;
}

// `call` with DT.
#define HASTE_MLP_TYPES(call)                              \
    (dtype == HASTE_DTYPE_F32    ? call(HASTE_DTYPE_F32)   \
     : dtype == HASTE_DTYPE_BF16 ? call(HASTE_DTYPE_BF16)  \
                                 : call(HASTE_DTYPE_F16))

int mlp_sizes(const char* fn, int64_t N, int64_t D, int64_t H, int64_t O, int32_t dtype) {
    HASTE_CHECK_ARG(N >= 0 && D > 0 && H > 0 && O > 0, "%s: bad sizes N=%lld D=%lld H=%lld O=%lld", fn,
                    (long long)N, (long long)D, (long long)H, (long long)O);
    HASTE_CHECK_ARG(D <= kMaxSide && H <= kMaxSide && O <= kMaxSide && N < (int64_t)1 << 30,
                    "%s: too large (D, H and O up to 2^20, N below 2^30)", fn);
    // (so that a product's launch has fewer than 2^32 threads, 512 to a tile of 256 x 256)
    HASTE_CHECK_ARG(N * std::max(D, O) < (int64_t)1 << 34, "%s: too large (N D and N O below 2^34)", fn);
    HASTE_CHECK_ARG(elem_dtype(dtype), "%s: matrices must be bf16, f16 or f32", fn);
    return HASTE_OK;
}
int mlp_matrix(const char* fn, const char* what, const Matrix& m, int32_t dtype) {
    HASTE_CHECK_ARG(m.p != nullptr && elem_aligned(m.p, dtype), "%s: %s is NULL or misaligned", fn, what);
    HASTE_CHECK_ARG(m.ld >= m.cols && m.ld <= 4 * kMaxSide, "%s: row pitch of %s (%lld) must be %lld to 2^22",
                    fn, what, (long long)m.ld, (long long)m.cols);
    return HASTE_OK;
}
int mlp_hidden(const char* fn, const char* what, const void* p) {
    HASTE_CHECK_ARG(p != nullptr && aligned16(p), "%s: %s is NULL or misaligned", fn, what);
    return HASTE_OK;
}
int mlp_space(const char* fn, const void* ws, int64_t have, int64_t need) {
    HASTE_CHECK_ARG(need == 0 || (ws != nullptr && aligned16(ws)), "%s: workspace is NULL or misaligned", fn);
    if (have < need) {
        set_error("%s: workspace too small (%lld < %lld bytes)", fn, (long long)have, (long long)need);
        return HASTE_ERR_WORKSPACE;
    }
    return HASTE_OK;
}
int mlp_act(const char* fn, int32_t act) {
    HASTE_CHECK_ARG(act == HASTE_ACT_SILU || act == HASTE_ACT_GELU || act == HASTE_ACT_GELU_TANH,
                    "%s: unknown activation %d", fn, (int)act);
    return HASTE_OK;
}

}  // namespace
}  // namespace haste

extern "C" int64_t haste_gated_mlp_workspace_size(int64_t N, int64_t D, int64_t H, int64_t O,
                                                  int32_t dtype, int32_t backward,
                                                  int32_t aligned) {
    HASTE_TRY(haste::mlp_sizes("haste_gated_mlp_workspace_size", N, D, H, O, dtype));
    const haste::Sizes s{N, D, H, O};
    const int64_t ld = haste::round16(H);
    // (an odd pitch: the matrix counts as one to be copied)
    auto any = [&](int64_t rows, int64_t cols) {
        return haste::Matrix{nullptr, aligned ? cols : cols | 1, rows, cols};
    };
    const haste::Matrix x = any(N, D), wg = any(H, D), wd = any(O, H), dy = any(N, O);
#define HASTE_MLP(DT)                                                                                   \
    (backward ? haste::backward<DT>(s, x, wg, wg, wd, dy, nullptr, nullptr, ld, haste::Grads{}, \
                                    nullptr, false, nullptr)                                          \
              : haste::forward<DT>(s, x, wg, wg, wd, haste::GatedOut{{nullptr, 0}, nullptr, ld, 0, (int)H},     \
                                   nullptr, 0, nullptr, false, nullptr))
    return HASTE_MLP_TYPES(HASTE_MLP);
#undef HASTE_MLP
}

extern "C" int64_t haste_gated_mlp_kept_size(int64_t N, int64_t H, int32_t dtype) {
    HASTE_TRY(haste::mlp_sizes("haste_gated_mlp_kept_size", N, 1, H, 1, dtype));
    return haste::ceil_div(N, 16) * haste::kept_blocks(H) * 2 *
           (dtype == HASTE_DTYPE_F32 ? haste::kKeptBlock<HASTE_DTYPE_F32> : haste::kKeptBlock<HASTE_DTYPE_BF16>);
}

extern "C" int haste_gated_mlp(const void* x, int64_t ldx, const void* wg, int64_t ldg, const void* wu,
                               int64_t ldu, const void* wd, int64_t ldd, void* y, void* kept,
                               void* h, int64_t N, int64_t D, int64_t H, int64_t O, int32_t act,
                               int32_t dtype, void* ws, int64_t ws_bytes, void* stream) {
    const char* fn = "haste_gated_mlp";
    HASTE_TRY(haste::mlp_sizes(fn, N, D, H, O, dtype));
    HASTE_TRY(haste::mlp_act(fn, act));
    if (N == 0) return HASTE_OK;
    const haste::Sizes s{N, D, H, O};
    const haste::Matrix mx{x, ldx, N, D}, mg{wg, ldg, H, D}, mu{wu, ldu, H, D}, md{wd, ldd, O, H};
    HASTE_TRY(haste::mlp_matrix(fn, "x", mx, dtype));
    HASTE_TRY(haste::mlp_matrix(fn, "the gate's weight", mg, dtype));
    HASTE_TRY(haste::mlp_matrix(fn, "the up weight", mu, dtype));
    HASTE_TRY(haste::mlp_matrix(fn, "the down weight", md, dtype));
    HASTE_CHECK_ARG(y != nullptr && haste::elem_aligned(y, dtype), "%s: y is NULL or misaligned", fn);
    HASTE_TRY(haste::mlp_hidden(fn, "h", h));
    if (kept) HASTE_TRY(haste::mlp_hidden(fn, "kept", kept));
    const haste::GatedOut out{{kept, haste::kept_blocks(H)}, h, haste::round16(H),
                              dtype == HASTE_DTYPE_F32 ? N * haste::round16(H) * 2 : 0, (int)H};
    hipStream_t st = static_cast<hipStream_t>(stream);
    auto run = [&](char* base, bool launch) {
#define HASTE_MLP(DT) haste::forward<DT>(s, mx, mg, mu, md, out, y, act, base, launch, st)
        return HASTE_MLP_TYPES(HASTE_MLP);
#undef HASTE_MLP
    };
    HASTE_TRY(haste::mlp_space(fn, ws, ws_bytes, run(nullptr, false)));
    run(static_cast<char*>(ws), true);
    HASTE_CHECK_LAUNCH(fn);
    return HASTE_OK;
}

extern "C" int haste_gated_mlp_bwd(const void* x, int64_t ldx, const void* wg, int64_t ldg,
                                   const void* wu, int64_t ldu, const void* wd, int64_t ldd,
                                   const void* dy, int64_t lddy, const void* kept,
                                   const void* h, void* dx, void* dwg, void* dwu, void* dwd, int64_t N,
                                   int64_t D, int64_t H, int64_t O, int32_t dtype, void* ws,
                                   int64_t ws_bytes, void* stream) {
    const char* fn = "haste_gated_mlp_bwd";
    HASTE_TRY(haste::mlp_sizes(fn, N, D, H, O, dtype));
    const haste::Sizes s{N, D, H, O};
    const haste::Matrix mx{x, ldx, N, D}, mg{wg, ldg, H, D}, mu{wu, ldu, H, D}, md{wd, ldd, O, H},
        my{dy, lddy, N, O};
    HASTE_CHECK_ARG(haste::elem_aligned(dx, dtype) && haste::elem_aligned(dwg, dtype) &&
                        haste::elem_aligned(dwu, dtype) && haste::elem_aligned(dwd, dtype),
                    "%s: a gradient is misaligned", fn);
    HASTE_CHECK_ARG((dwg == nullptr) == (dwu == nullptr), "%s: dwg and dwu are computed together", fn);
    if (N > 0) {
        HASTE_TRY(haste::mlp_matrix(fn, "x", mx, dtype));
        HASTE_TRY(haste::mlp_matrix(fn, "the gate's weight", mg, dtype));
        HASTE_TRY(haste::mlp_matrix(fn, "the up weight", mu, dtype));
        HASTE_TRY(haste::mlp_matrix(fn, "the down weight", md, dtype));
        HASTE_TRY(haste::mlp_matrix(fn, "dy", my, dtype));
        HASTE_TRY(haste::mlp_hidden(fn, "kept", kept));
        HASTE_TRY(haste::mlp_hidden(fn, "h", h));
    }
    if (N == 0 && !dwg && !dwd) return HASTE_OK;
    const haste::Grads to{dx, dwg, dwu, dwd};
    hipStream_t st = static_cast<hipStream_t>(stream);
    auto run = [&](char* base, bool launch) {
#define HASTE_MLP(DT) \
    haste::backward<DT>(s, mx, mg, mu, md, my, const_cast<void*>(kept), h, haste::round16(H), to, base, launch, st)
        return HASTE_MLP_TYPES(HASTE_MLP);
#undef HASTE_MLP
    };
    HASTE_TRY(haste::mlp_space(fn, ws, ws_bytes, run(nullptr, false)));
    run(static_cast<char*>(ws), true);
    HASTE_CHECK_LAUNCH(fn);
    return HASTE_OK;
}
