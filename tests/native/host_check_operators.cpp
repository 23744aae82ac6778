// host_check_operators.cpp -- drives the host-side code of the encoder's operators (layer norm,
// gradient norm, AdamW: argument checks and workspace sizing) without a GPU, for the
// AddressSanitizer / UndefinedBehaviorSanitizer build of `make -C haste_amd sanitize_operators`
// (host code only; no kernel is launched).  Prints "host_check_operators OK" and exits 0 when
// every check held; a sanitizer report aborts the run.
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <limits>

#include "../../include/haste_ffi.h"

static int failures = 0;
#define EXPECT(cond)                                                                                  \
    do {                                                                                              \
        if (!(cond)) {                                                                                \
            std::fprintf(stderr, "host_check_operators: %s:%d: %s\n", __FILE__, __LINE__, #cond);     \
            ++failures;                                                                               \
        }                                                                                             \
    } while (0)

static void expect_rejected(int rc) {
    EXPECT(rc < 0);
    EXPECT(std::strlen(haste_last_error()) > 0);
}

// (an address that no check follows)
static char* at(uintptr_t a) { return reinterpret_cast<char*>(a); }

static void workspaces() {
    const int64_t Ns[] = {0, 1, 16, 8192, 1000000, ((int64_t)1 << 31) - 1};
    const int64_t Ds[] = {1, 7, 8, 768, 8192, 12289, 70000, ((int64_t)1 << 31) - 1};
    for (int64_t N : Ns)
        for (int64_t D : Ds) {
            const int64_t size = haste_layer_norm_bwd_workspace_size(N, D);
            EXPECT(size >= 8 * D && size <= 512 * 8 * (D + 8));
        }
    EXPECT(haste_layer_norm_bwd_workspace_size(-1, 8) < 0);
    EXPECT(haste_layer_norm_bwd_workspace_size(8, -1) < 0);
    int64_t last = 0;
    for (int32_t n : {0, 1, 200, 201, 1000, std::numeric_limits<int32_t>::max()}) {
        const int64_t size = haste_grad_norm_workspace_size(n);
        EXPECT(size > 0 && size >= last);
        last = size;
    }
    EXPECT(haste_grad_norm_workspace_size(-1) < 0);
}

static void layer_norms() {
    const double nan = std::nan("");
    for (int32_t dt = -1; dt <= 5; ++dt)
        for (int32_t wdt = -1; wdt <= 5; ++wdt) {
            // every pointer missing
            expect_rejected(haste_layer_norm(nullptr, 8, nullptr, 0, nullptr, nullptr, nullptr, nullptr,
                                             nullptr, 4, 8, 1e-5, dt, wdt, nullptr));
            expect_rejected(haste_layer_norm_bwd(nullptr, 8, nullptr, 0, nullptr, 8, nullptr, nullptr,
                                                 nullptr, nullptr, nullptr, nullptr, 0, 4, 8, dt, wdt,
                                                 nullptr));
        }
    float* stats = reinterpret_cast<float*>(at(512));
    for (int64_t N : {(int64_t)-1, (int64_t)4, (int64_t)1 << 31})
        for (int64_t D : {(int64_t)0, (int64_t)1 << 31, std::numeric_limits<int64_t>::max()}) {
            expect_rejected(haste_layer_norm(at(64), 8, nullptr, 0, at(64), nullptr, at(64), nullptr,
                                             stats, N, D, 1e-5, 0, 0, nullptr));
            expect_rejected(haste_layer_norm_bwd(at(64), 8, nullptr, 0, at(64), 8, at(64), stats, at(64),
                                                 at(64), at(64), at(64), 1 << 30, N, D, 0, 0, nullptr));
        }
    for (double eps : {-1.0, nan})
        expect_rejected(haste_layer_norm(at(64), 8, nullptr, 0, at(64), nullptr, at(64), nullptr, stats, 4,
                                         8, eps, 0, 0, nullptr));
    for (int64_t ld : {(int64_t)7, (int64_t)-8, std::numeric_limits<int64_t>::min()})
        expect_rejected(haste_layer_norm(at(64), ld, nullptr, 0, at(64), nullptr, at(64), nullptr, stats, 4,
                                         8, 1e-5, 0, 0, nullptr));
    expect_rejected(haste_layer_norm_bwd(at(64), 8, nullptr, 0, at(64), 8, at(64), stats, at(64), at(64),
                                         at(64), at(64), 16, 4, 8, 0, 0, nullptr));
    // no rows
    EXPECT(haste_layer_norm(nullptr, 8, nullptr, 0, nullptr, nullptr, nullptr, nullptr, nullptr, 0, 8, 1e-5,
                            0, 0, nullptr) == HASTE_OK);
}

static void norms_and_steps() {
    float* out = reinterpret_cast<float*>(at(64));
    const int64_t size = haste_grad_norm_workspace_size(3);
    const int64_t bad_n[] = {-1, (int64_t)1 << 44, std::numeric_limits<int64_t>::max()};
    for (int64_t n : bad_n) {
        haste_grad_tensor t[3] = {{nullptr, 0, 0}, {nullptr, 0, 2}, {at(64), n, 0}};
        expect_rejected(haste_grad_norm(t, 3, 1.0, out, at(64), size, nullptr));
    }
    haste_grad_tensor g[3] = {{at(64), 5, 0}, {at(66), 5, 2}, {at(64), 5, 1}};
    expect_rejected(haste_grad_norm(g, 3, 1.0, out, at(64), size, nullptr));  // misaligned
    expect_rejected(haste_grad_norm(g, 3, std::nan(""), out, at(64), size, nullptr));
    expect_rejected(haste_grad_norm(g, 3, 1.0, out, at(64), size - 1, nullptr));
    expect_rejected(haste_grad_norm(nullptr, 3, 1.0, out, at(64), size, nullptr));

    uint8_t* sc = reinterpret_cast<uint8_t*>(at(64));
    const haste_adamw_tensor good{at(64), at(64), at(64), at(64), sc, sc, 10, 0};
    haste_adamw_tensor empty[200];
    for (auto& t : empty) t = haste_adamw_tensor{nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 0, 0};
    for (int32_t bits : {8, 32})
        for (int32_t w = 0; w <= 2; ++w)
            for (int32_t gd = 0; gd <= 2; ++gd) {
                EXPECT(haste_adamw_step(empty, 200, w, gd, bits, 1e-3, 0.9, 0.999, 1e-8, 0.01, 1, 1, 7,
                                        nullptr, nullptr) == HASTE_OK);
                for (int k = 0; k < 7; ++k) {
                    haste_adamw_tensor t = good;
                    if (k == 0) t.w = nullptr;
                    if (k == 1) t.g = nullptr;
                    if (k == 2) t.m = nullptr;
                    if (k == 3) t.v = at(68);
                    if (k == 4) t.n = (int64_t)1 << 40;
                    if (k == 5) t.stream = 1u << 24;
                    if (k == 6) t.n = std::numeric_limits<int64_t>::min();
                    expect_rejected(haste_adamw_step(&t, 1, w, gd, bits, 1e-3, 0.9, 0.999, 1e-8, 0.01, 1, 1,
                                                     7, nullptr, nullptr));
                }
                for (int64_t step : {(int64_t)0, std::numeric_limits<int64_t>::min()})
                    expect_rejected(haste_adamw_step(&good, 1, w, gd, bits, 1e-3, 0.9, 0.999, 1e-8, 0.01,
                                                     step, 1, 7, nullptr, nullptr));
                EXPECT(haste_adamw_step(empty, 200, w, gd, bits, 1e-3, 0.0, 0.0, 0.0, 0.0,
                                        std::numeric_limits<int64_t>::max(), 0, ~0ull, nullptr,
                                        nullptr) == HASTE_OK);
            }
    expect_rejected(haste_adamw_step(&good, 1, 0, 0, 16, 1e-3, 0.9, 0.999, 1e-8, 0.01, 1, 1, 7, nullptr, nullptr));
    expect_rejected(haste_adamw_step(&good, -1, 0, 0, 8, 1e-3, 0.9, 0.999, 1e-8, 0.01, 1, 1, 7, nullptr, nullptr));
    expect_rejected(haste_adamw_step(&good, 1, 0, 0, 8, 1e-3, 1.0, 0.999, 1e-8, 0.01, 1, 1, 7, nullptr, nullptr));
}

int main() {
    workspaces();
    layer_norms();
    norms_and_steps();
    if (failures) return 1;
    std::puts("host_check_operators OK");
    return 0;
}
