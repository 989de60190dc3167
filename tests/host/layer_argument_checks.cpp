// The layer entry points (nerf_embedding_*, nerf_rmsnorm_*, nerf_gated_mlp_*) in the sanitizer build, beside
// abi_argument_checks.cpp: every refusal that returns before a launch, every documented no-op, and the workspace sizes over the
// whole range of shapes -- their arithmetic is what -fsanitize=undefined is for.  No GPU is needed and none is touched.
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <initializer_list>

#include "../../include/nerf_hip.h"

static int g_fail = 0;
#define EXPECT(cond)                                                                  \
    do {                                                                              \
        if (!(cond)) { printf("FAIL %s:%d: %s   [%s]\n", __FILE__, __LINE__, #cond, nerf_last_error()); ++g_fail; } \
    } while (0)
#define REFUSED(call) EXPECT((call) == NERF_EINVAL && strlen(nerf_last_error()) > 0)

// non-null "device pointers" that are never dereferenced
static void* const P = (void*)0x1000;
static void* const ODD = (void*)0x1002;
static const int64_t* const IDX = (const int64_t*)0x1000;
static float* const F = (float*)0x1000;

static uint64_t g_seed = 1;
static int64_t draw(int64_t most) {         // 1 .. most, spread over its logarithm
    g_seed = g_seed * 6364136223846793005ull + 1442695040888963407ull;
    int bits = 0;
    while (most >> bits) ++bits;
    const int64_t v = (int64_t)(g_seed >> 11) & ((1ll << ((g_seed >> 5) % bits + 1)) - 1);
    return v < 1 ? 1 : v > most ? most : v;
}

static void embedding() {
    const int64_t kRows = 0x7fffffff, kDim = 1 << 20;
    for (int dt = 0; dt < 3; ++dt) {
        const int64_t need = nerf_embedding_bwd_workspace_bytes(dt, 5, 8, 4);
        EXPECT(need > 0);
        EXPECT(nerf_embedding_fwd(P, dt, 5, 8, IDX, 0, 1.f, P, nullptr) == 0);
        EXPECT(nerf_embedding_fwd(nullptr, dt, 0, 8, nullptr, 0, 1.f, nullptr, nullptr) == 0);
        REFUSED(nerf_embedding_fwd(nullptr, dt, 5, 8, IDX, 4, 1.f, P, nullptr));
        REFUSED(nerf_embedding_fwd(P, dt, 5, 8, nullptr, 4, 1.f, P, nullptr));
        REFUSED(nerf_embedding_fwd(P, dt, 5, 8, IDX, 4, 1.f, nullptr, nullptr));
        const int64_t bad[][3] = {{-1, 8, 4}, {kRows + 1, 8, 4}, {5, 0, 4}, {5, kDim + 1, 4}, {5, 8, -1}, {5, 8, kRows + 1}, {INT64_MIN, 8, 4},
                                  {5, INT64_MAX, 4}, {5, 8, INT64_MAX}};
        for (auto& b : bad) {
            REFUSED(nerf_embedding_fwd(P, dt, b[0], b[1], IDX, b[2], 1.f, P, nullptr));
            EXPECT(nerf_embedding_bwd_workspace_bytes(dt, b[0], b[1], b[2]) < 0);
            REFUSED(nerf_embedding_bwd(IDX, P, dt, b[2], b[0], b[1], 1.f, P, P, INT64_MAX, nullptr));
        }
        EXPECT(nerf_embedding_bwd(IDX, P, dt, 4, 0, 8, 1.f, nullptr, nullptr, 0, nullptr) == 0);
        REFUSED(nerf_embedding_bwd(nullptr, P, dt, 4, 5, 8, 1.f, P, P, need, nullptr));
        REFUSED(nerf_embedding_bwd(IDX, nullptr, dt, 4, 5, 8, 1.f, P, P, need, nullptr));
        REFUSED(nerf_embedding_bwd(IDX, P, dt, 4, 5, 8, 1.f, nullptr, P, need, nullptr));
        REFUSED(nerf_embedding_bwd(IDX, P, dt, 4, 5, 8, 1.f, P, nullptr, need, nullptr));
        REFUSED(nerf_embedding_bwd(IDX, P, dt, 4, 5, 8, 1.f, P, ODD, need, nullptr));
        REFUSED(nerf_embedding_bwd(IDX, P, dt, 4, 5, 8, 1.f, P, P, need - 1, nullptr));
        EXPECT(nerf_embedding_bwd_workspace_bytes(dt, kRows, kDim, kRows) > 0);
        for (int i = 0; i < 20000; ++i) {
            const int64_t e = draw(kRows), d = draw(kDim), r = draw(kRows);
            EXPECT(nerf_embedding_bwd_workspace_bytes(dt, e, d, r) >= 16 * r);      // two buffers of pairs at the least
        }
    }
    REFUSED(nerf_embedding_fwd(P, 3, 5, 8, IDX, 4, 1.f, P, nullptr));
    REFUSED(nerf_embedding_bwd(IDX, P, -1, 4, 5, 8, 1.f, P, P, 1 << 20, nullptr));
    EXPECT(nerf_embedding_bwd_workspace_bytes(3, 5, 8, 4) < 0);
}

static void rmsnorm() {
    const int64_t kRows = 0x7fffffff, kDim = 1 << 24;
    const float nan = __builtin_nanf("");
    const int64_t need = nerf_rmsnorm_bwd_workspace_bytes(3, 8);
    for (int dt = 0; dt < 3; ++dt) {
        EXPECT(nerf_rmsnorm_fwd(nullptr, nullptr, nullptr, dt, dt, 0, 8, 0.f, nullptr, nullptr, nullptr) == 0);
        REFUSED(nerf_rmsnorm_fwd(nullptr, nullptr, P, dt, 0, 3, 8, 0.f, nullptr, P, nullptr));
        REFUSED(nerf_rmsnorm_fwd(P, nullptr, nullptr, dt, 0, 3, 8, 0.f, nullptr, P, nullptr));
        REFUSED(nerf_rmsnorm_fwd(P, nullptr, P, dt, 0, 3, 8, 0.f, nullptr, nullptr, nullptr));
        REFUSED(nerf_rmsnorm_fwd(P, P, P, dt, 0, 3, 8, 0.f, nullptr, P, nullptr));       // a residual and nowhere to put the sum
        REFUSED(nerf_rmsnorm_fwd(P, nullptr, P, dt, dt == 1 ? 2 : 1 + (dt == 0), 3, 8, 0.f, nullptr, P, nullptr));
        for (float eps : {-1.f, nan}) {
            REFUSED(nerf_rmsnorm_fwd(P, nullptr, P, dt, 0, 3, 8, eps, nullptr, P, nullptr));
            REFUSED(nerf_rmsnorm_bwd(P, P, P, nullptr, dt, 0, 3, 8, eps, P, P, P, need, nullptr));
        }
        const int64_t bad[][2] = {{-1, 8}, {kRows + 1, 8}, {3, 0}, {3, kDim + 1}, {INT64_MIN, 8}, {3, INT64_MAX}, {INT64_MAX, INT64_MAX}};
        for (auto& b : bad) {
            REFUSED(nerf_rmsnorm_fwd(P, nullptr, P, dt, 0, b[0], b[1], 0.f, nullptr, P, nullptr));
            REFUSED(nerf_rmsnorm_bwd(P, P, P, nullptr, dt, 0, b[0], b[1], 0.f, P, P, P, INT64_MAX, nullptr));
            EXPECT(nerf_rmsnorm_bwd_workspace_bytes(b[0], b[1]) < 0);
        }
        REFUSED(nerf_rmsnorm_bwd(nullptr, P, P, nullptr, dt, 0, 3, 8, 0.f, P, P, P, need, nullptr));
        REFUSED(nerf_rmsnorm_bwd(P, nullptr, P, nullptr, dt, 0, 3, 8, 0.f, P, P, P, need, nullptr));
        REFUSED(nerf_rmsnorm_bwd(P, P, nullptr, nullptr, dt, 0, 3, 8, 0.f, P, P, P, need, nullptr));
        REFUSED(nerf_rmsnorm_bwd(P, P, P, nullptr, dt, 0, 3, 8, 0.f, P, P, nullptr, need, nullptr));
        REFUSED(nerf_rmsnorm_bwd(P, P, P, nullptr, dt, 0, 3, 8, 0.f, P, P, ODD, need, nullptr));
        REFUSED(nerf_rmsnorm_bwd(P, P, P, nullptr, dt, 0, 3, 8, 0.f, P, P, P, need - 1, nullptr));
    }
    REFUSED(nerf_rmsnorm_fwd(P, nullptr, P, 4, 4, 3, 8, 0.f, nullptr, P, nullptr));
    for (int i = 0; i < 20000; ++i) {
        const int64_t r = draw(kRows), d = draw(kDim);
        EXPECT(nerf_rmsnorm_bwd_workspace_bytes(r, d) >= 4 * d);
    }
    EXPECT(nerf_rmsnorm_bwd_workspace_bytes(kRows, kDim) > 0 && nerf_rmsnorm_bwd_workspace_bytes(0, kDim) > 0);
}

static void gated() {
    const int64_t kRows = 1 << 26, kWidth = 1 << 16;
    const int64_t huge = INT64_MAX;
    for (int dt = 0; dt < 3; ++dt) {
        const int64_t m = 4, k = 200, f = 264, n = 200, need = nerf_gated_mlp_fwd_workspace_bytes(dt, m, k, f, n),
                      back = nerf_gated_mlp_bwd_workspace_bytes(dt, m, k, f, n);
        EXPECT(need > 0 && back > 0 && nerf_gated_mlp_saved_floats(dt, m, k, f, n) >= 2 * m * f);
        EXPECT(nerf_gated_mlp_alone_workspace_bytes(dt, m, k, f, n) == need);
        EXPECT(nerf_gated_mlp_fwd(nullptr, nullptr, dt, 0, k, f, n, 0, nullptr, nullptr, nullptr, 0, nullptr) == 0);
        EXPECT(nerf_gated_mlp_bwd(nullptr, nullptr, nullptr, nullptr, dt, 0, k, f, n, 0, nullptr, nullptr, dt, nullptr, 0, nullptr) == 0);
        REFUSED(nerf_gated_mlp_fwd(nullptr, P, dt, m, k, f, n, 0, P, nullptr, P, need, nullptr));
        REFUSED(nerf_gated_mlp_fwd(P, nullptr, dt, m, k, f, n, 0, P, nullptr, P, need, nullptr));
        REFUSED(nerf_gated_mlp_fwd(P, P, dt, m, k, f, n, 0, nullptr, nullptr, P, need, nullptr));
        REFUSED(nerf_gated_mlp_fwd(P, P, dt, m, k, f, n, 0, P, nullptr, nullptr, need, nullptr));
        REFUSED(nerf_gated_mlp_fwd(P, P, dt, m, k, f, n, 0, P, nullptr, P, need - 1, nullptr));
        REFUSED(nerf_gated_mlp_fwd(P, P, dt, m, k, f, n, 3, P, nullptr, P, need, nullptr));
        REFUSED(nerf_gated_mlp_fwd(P, P, dt, m, k, f, n, -1, P, nullptr, P, need, nullptr));
        REFUSED(nerf_gated_mlp_fwd(ODD, P, dt, m, k, f, n, 0, P, nullptr, P, need, nullptr));
        REFUSED(nerf_gated_mlp_fwd(P, ODD, dt, m, k, f, n, 0, P, nullptr, P, need, nullptr));
        REFUSED(nerf_gated_mlp_fwd(P, P, dt, m, k, f, n, 0, P, nullptr, ODD, need, nullptr));
        // a narrow block whose g and u are kept needs a workspace that the same one alone does not
        EXPECT(dt == 0 || nerf_gated_mlp_alone_workspace_bytes(dt, 900, 100, 128, 64) == 0);
        REFUSED(nerf_gated_mlp_fwd(P, P, dt, 900, 100, 128, 64, 0, P, F, nullptr, 0, nullptr));
        REFUSED(nerf_gated_mlp_bwd(nullptr, P, P, F, dt, m, k, f, n, 0, P, P, dt, P, back, nullptr));
        REFUSED(nerf_gated_mlp_bwd(P, nullptr, P, F, dt, m, k, f, n, 0, P, P, dt, P, back, nullptr));
        REFUSED(nerf_gated_mlp_bwd(P, P, nullptr, F, dt, m, k, f, n, 0, P, P, dt, P, back, nullptr));
        REFUSED(nerf_gated_mlp_bwd(P, P, P, nullptr, dt, m, k, f, n, 0, P, P, dt, P, back, nullptr));
        REFUSED(nerf_gated_mlp_bwd(P, P, P, F, dt, m, k, f, n, 0, P, P, dt, nullptr, back, nullptr));
        REFUSED(nerf_gated_mlp_bwd(P, P, P, F, dt, m, k, f, n, 0, P, P, dt, P, back - 1, nullptr));
        REFUSED(nerf_gated_mlp_bwd(ODD, P, P, F, dt, m, k, f, n, 0, P, P, dt, P, back, nullptr));
        REFUSED(nerf_gated_mlp_bwd(P, ODD, P, F, dt, m, k, f, n, 0, P, P, dt, P, back, nullptr));
        REFUSED(nerf_gated_mlp_bwd(P, P, ODD, F, dt, m, k, f, n, 0, P, P, dt, P, back, nullptr));
        REFUSED(nerf_gated_mlp_bwd(P, P, P, F, dt, m, k, f, n, 0, P, P, dt, ODD, back, nullptr));
        REFUSED(nerf_gated_mlp_bwd(P, P, P, F, dt, m, k, f, n, 0, P, P, dt == 1 ? 2 : 1, P, back, nullptr));
        REFUSED(nerf_gated_mlp_bwd(P, P, P, F, dt, m, k, f, n, 7, P, P, dt, P, back, nullptr));
        const int64_t bad[][4] = {{-1, 8, 8, 8}, {kRows + 1, 8, 8, 8}, {4, 0, 8, 8}, {4, 8, 0, 8}, {4, 8, 8, 0}, {4, kWidth + 1, 8, 8},
                                  {4, 8, kWidth + 1, 8}, {4, 8, 8, kWidth + 1}, {kRows, 8, kWidth, 8}, {kRows, kWidth, kWidth, kWidth},
                                  {INT64_MIN, 8, 8, 8}, {huge, huge, huge, huge}, {4, huge, 8, 8}, {4, 8, INT64_MIN, 8}};
        for (auto& b : bad) {
            REFUSED(nerf_gated_mlp_fwd(P, P, dt, b[0], b[1], b[2], b[3], 0, P, nullptr, P, huge, nullptr));
            REFUSED(nerf_gated_mlp_bwd(P, P, P, F, dt, b[0], b[1], b[2], b[3], 0, P, P, dt, P, huge, nullptr));
            EXPECT(nerf_gated_mlp_saved_floats(dt, b[0], b[1], b[2], b[3]) < 0 && nerf_gated_mlp_fwd_workspace_bytes(dt, b[0], b[1], b[2], b[3]) < 0 &&
                   nerf_gated_mlp_alone_workspace_bytes(dt, b[0], b[1], b[2], b[3]) < 0 && nerf_gated_mlp_bwd_workspace_bytes(dt, b[0], b[1], b[2], b[3]) < 0);
        }
        for (int i = 0; i < 20000; ++i) {
            const int64_t r = draw(kRows), a = draw(kWidth), h = draw(kWidth), o = draw(kWidth);
            const int64_t s = nerf_gated_mlp_saved_floats(dt, r, a, h, o), w = nerf_gated_mlp_fwd_workspace_bytes(dt, r, a, h, o),
                          l = nerf_gated_mlp_alone_workspace_bytes(dt, r, a, h, o), b = nerf_gated_mlp_bwd_workspace_bytes(dt, r, a, h, o);
            EXPECT((s < 0) == (w < 0) && (s < 0) == (l < 0) && (s < 0) == (b < 0) && l <= w);
            if (s < 0) continue;
            EXPECT(b > 0 && (s == 0 || s >= 2 * r * h));
        }
    }
    REFUSED(nerf_gated_mlp_fwd(P, P, 3, 4, 8, 8, 8, 0, P, nullptr, P, huge, nullptr));
    REFUSED(nerf_gated_mlp_bwd(P, P, P, F, -1, 4, 8, 8, 8, 0, P, P, 0, P, huge, nullptr));
    EXPECT(nerf_gated_mlp_saved_floats(3, 4, 8, 8, 8) < 0 && nerf_gated_mlp_fwd_workspace_bytes(3, 4, 8, 8, 8) < 0);
}

int main() {
    embedding();
    rmsnorm();
    gated();
    if (g_fail) { printf("%d checks failed\n", g_fail); return 1; }
    printf("all layer argument checks passed\n");
    return 0;
}
