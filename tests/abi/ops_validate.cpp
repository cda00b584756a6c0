// Host side of the operators in include/gsage_ops.h under AddressSanitizer + UndefinedBehaviorSanitizer, without a GPU:
// every entry point is called with arguments it must refuse and with empty inputs it must accept.  All of these return
// before anything is launched.  Pointers marked "device" are never dereferenced on the host; they point into a small host
// array only so that they are non-null and aligned.
#include <cmath>
#include <cstdint>
#include <cstdio>

#include "gsage_ops.h"

static int failures = 0;

#define REFUSED(code, call)                                                                          \
    do {                                                                                             \
        const int rc_ = (call);                                                                      \
        const char *msg_ = gs_last_error();                                                          \
        if (rc_ != (code) || !msg_ || !msg_[0]) {                                                    \
            std::printf("line %d: expected %d with a message, got %d (%s)\n", __LINE__, (code), rc_, msg_ ? msg_ : ""); \
            ++failures;                                                                              \
        }                                                                                            \
    } while (0)

#define ACCEPTED(call)                                                                               \
    do {                                                                                             \
        const int rc_ = (call);                                                                      \
        if (rc_ != GS_OK) { std::printf("line %d: expected GS_OK, got %d (%s)\n", __LINE__, rc_, gs_last_error()); ++failures; } \
    } while (0)

#define EXPECT(cond)                                                                                 \
    do { if (!(cond)) { std::printf("line %d: %s\n", __LINE__, #cond); ++failures; } } while (0)

int main() {
    alignas(256) static char arena[8192];
    float *f = reinterpret_cast<float *>(arena);
    void *p = arena, *odd = arena + 1;
    int32_t *i32 = reinterpret_cast<int32_t *>(arena + 1024);
    int64_t *i64 = reinterpret_cast<int64_t *>(arena + 2048);
    uint64_t *u64 = reinterpret_cast<uint64_t *>(arena + 4096);

    // ---- dropout ----
    ACCEPTED(gs_dropout(nullptr, 0, GS_F32, 0.5, 1, nullptr, 0, nullptr, nullptr));
    REFUSED(GS_EINVAL, gs_dropout(p, -1, GS_F32, 0.5, 1, nullptr, 0, p, nullptr));
    REFUSED(GS_EINVAL, gs_dropout(p, 8, 3, 0.5, 1, nullptr, 0, p, nullptr));
    REFUSED(GS_EINVAL, gs_dropout(p, 8, GS_F32, 1.0, 1, nullptr, 0, p, nullptr));
    REFUSED(GS_EINVAL, gs_dropout(p, 8, GS_F32, -0.25, 1, nullptr, 0, p, nullptr));
    REFUSED(GS_EINVAL, gs_dropout(p, 8, GS_F32, std::nan(""), 1, nullptr, 0, p, nullptr));
    REFUSED(GS_EINVAL, gs_dropout(nullptr, 8, GS_F32, 0.5, 1, nullptr, 0, p, nullptr));
    REFUSED(GS_EINVAL, gs_dropout(p, 8, GS_F32, 0.5, 1, nullptr, 0, nullptr, nullptr));
    REFUSED(GS_EINVAL, gs_dropout(odd, 8, GS_BF16, 0.5, 1, nullptr, 0, p, nullptr));
    REFUSED(GS_EINVAL, gs_dropout(p, 8, GS_F16, 0.5, 1, reinterpret_cast<uint64_t *>(arena + 4100), 0, p, nullptr));
    REFUSED(GS_EINVAL, gs_dropout(p, 64, GS_F32, 0.5, 1, u64, 0, arena + 64, nullptr));          // in part the same memory
    REFUSED(GS_ELIMIT, gs_dropout(p, INT64_MAX / 4, GS_BF16, 0.5, 1, nullptr, 0, p, nullptr));

    // ---- attention over neighbors ----
    gs_neighbors uniform{nullptr, 10, 4, i32, 40, 0, 100}, ragged{i64, 10, 0, i32, 40, 0, 100}, dense{nullptr, 10, 4, nullptr, 40, 0, 40};
    gs_neighbors none{nullptr, 0, 4, i32, 0, 0, 100}, broken{nullptr, 10, 4, i32, 41, 0, 100};
    gs_neighbors huge{i64, 10, 0, i32, (int64_t)1 << 31, 0, 100}, rows{nullptr, 10, 4, i32, 40, 0, (int64_t)1 << 31};
    EXPECT(gs_neighbor_attention_workspace(&uniform, 2, 1, 64, GS_F32) == 0);                   // short lists leave no pieces
    EXPECT(gs_neighbor_attention_workspace(&ragged, 2, 1, 64, GS_F32) > 0);
    EXPECT(gs_neighbor_attention_workspace(&broken, 2, 1, 64, GS_F32) == 0);
    EXPECT(gs_neighbor_attention_workspace(nullptr, 2, 1, 64, GS_F32) == 0);
    const auto fwd = [&](const gs_neighbors *nb, int heads, int kv, int dim, int dtype) {
        return gs_neighbor_attention_fwd(p, p, p, nb, heads, kv, dim, dtype, 1.f, p, f, arena, sizeof arena, nullptr);
    };
    ACCEPTED(fwd(&none, 2, 1, 64, GS_F32));
    REFUSED(GS_EINVAL, fwd(nullptr, 2, 1, 64, GS_F32));
    REFUSED(GS_EINVAL, fwd(&broken, 2, 1, 64, GS_F32));
    REFUSED(GS_EINVAL, fwd(&uniform, 3, 2, 64, GS_F32));
    REFUSED(GS_EINVAL, fwd(&uniform, 0, 1, 64, GS_F32));
    REFUSED(GS_EINVAL, fwd(&uniform, 2, 1, 0, GS_F32));
    REFUSED(GS_EINVAL, fwd(&uniform, 2, 1, 64, 7));
    REFUSED(GS_ELIMIT, fwd(&uniform, 2, 1, 257, GS_F32));
    REFUSED(GS_ELIMIT, fwd(&uniform, 2048, 1, 64, GS_F32));
    REFUSED(GS_ELIMIT, fwd(&huge, 2, 1, 64, GS_F32));
    REFUSED(GS_ELIMIT, fwd(&rows, 2, 1, 64, GS_F32));
    REFUSED(GS_EINVAL, gs_neighbor_attention_fwd(nullptr, p, p, &uniform, 2, 1, 64, GS_F32, 1.f, p, f, arena, sizeof arena, nullptr));
    REFUSED(GS_EINVAL, gs_neighbor_attention_fwd(p, nullptr, p, &uniform, 2, 1, 64, GS_F32, 1.f, p, f, arena, sizeof arena, nullptr));
    REFUSED(GS_EINVAL, gs_neighbor_attention_fwd(p, p, p, &uniform, 2, 1, 64, GS_F32, 1.f, p, nullptr, arena, sizeof arena, nullptr));
    REFUSED(GS_EINVAL, gs_neighbor_attention_fwd(p, odd, p, &uniform, 2, 1, 64, GS_BF16, 1.f, p, f, arena, sizeof arena, nullptr));
    REFUSED(GS_EINVAL, gs_neighbor_attention_fwd(p, p, p, &ragged, 2, 1, 64, GS_F32, 1.f, p, f, arena, 16, nullptr));
    REFUSED(GS_EINVAL, gs_neighbor_attention_fwd(p, p, p, &ragged, 2, 1, 64, GS_F32, 1.f, p, f, nullptr, 1 << 20, nullptr));

    EXPECT(gs_neighbor_attention_bwd_workspace(&uniform, 2, 1, 64, GS_F32, 40) > 0);
    EXPECT(gs_neighbor_attention_bwd_workspace(&uniform, 2, 1, 64, GS_F32, -1) == 0);
    const auto bwd = [&](const gs_neighbors *nb, const int64_t *inv, int64_t n_inv, void *gq, void *gk, size_t ws) {
        return gs_neighbor_attention_bwd(p, p, p, nb, 2, 1, 8, GS_F32, 1.f, p, f, p, inv, i32, n_inv, gq, gk, nullptr, arena, ws, nullptr);
    };
    ACCEPTED(bwd(&uniform, nullptr, 0, nullptr, nullptr, 0));                                    // nothing wanted
    ACCEPTED(gs_neighbor_attention_bwd(p, p, nullptr, &dense, 2, 1, 8, GS_F32, 1.f, p, f, p, nullptr, nullptr, 0, nullptr, nullptr,
                                       p, arena, 0, nullptr));                                   // g_v without values: not wanted
    REFUSED(GS_EINVAL, bwd(&uniform, nullptr, 0, p, p, sizeof arena));                           // rows by id without their lists
    REFUSED(GS_EINVAL, bwd(&uniform, i64, 41, p, p, sizeof arena));                              // more entries than edges
    REFUSED(GS_EINVAL, bwd(&uniform, i64, 40, p, p, 8));
    REFUSED(GS_EINVAL, bwd(&broken, i64, 40, p, p, sizeof arena));
    REFUSED(GS_EINVAL, gs_neighbor_attention_bwd(p, p, p, &uniform, 2, 1, 8, GS_F32, 1.f, p, f, nullptr, i64, i32, 40, p, p, p, arena,
                                                 sizeof arena, nullptr));

    // ---- catalog ----
    EXPECT(gs_catalog_workspace(0, 100, 32, GS_F32, 0) == 0);
    EXPECT(gs_catalog_workspace(10, 0, 32, GS_F32, 5) > 0);
    EXPECT(gs_catalog_workspace(10, 100, 32, GS_F32, 65) == 0);
    EXPECT(gs_catalog_workspace(10, 100, 257, GS_F32, 5) == 0);
    EXPECT(gs_catalog_workspace((int64_t)1 << 30, (int64_t)1 << 30, 256, GS_F32, 64) > 0);
    EXPECT(gs_catalog_bwd_workspace(10, 100, 32, GS_F32) > 0);
    EXPECT(gs_catalog_bwd_workspace(-1, 100, 32, GS_F32) == 0);
    const auto rank = [&](int64_t nu, int64_t ni, int dim, int dtype, float scale, int k, void *ws, size_t bytes) {
        return gs_catalog_fwd(p, nu, p, ni, dim, dtype, nullptr, scale, nullptr, nullptr, nullptr, nullptr, k, f, i32, ws, bytes, nullptr);
    };
    ACCEPTED(rank(0, 100, 32, GS_F32, 1.f, 5, nullptr, 0));
    REFUSED(GS_EINVAL, rank(-1, 100, 32, GS_F32, 1.f, 5, arena, sizeof arena));
    REFUSED(GS_EINVAL, rank(10, 100, 0, GS_F32, 1.f, 5, arena, sizeof arena));
    REFUSED(GS_EINVAL, rank(10, 100, 32, 9, 1.f, 5, arena, sizeof arena));
    REFUSED(GS_EINVAL, rank(10, 100, 32, GS_F32, 0.f, 5, arena, sizeof arena));
    REFUSED(GS_EINVAL, rank(10, 100, 32, GS_F32, -1.f, 5, arena, sizeof arena));
    REFUSED(GS_EINVAL, rank(10, 100, 32, GS_F32, INFINITY, 5, arena, sizeof arena));
    REFUSED(GS_EINVAL, rank(10, 100, 32, GS_F32, NAN, 5, arena, sizeof arena));
    REFUSED(GS_EINVAL, rank(10, 100, 32, GS_F32, 1.f, -1, arena, sizeof arena));
    REFUSED(GS_ELIMIT, rank(10, 100, 32, GS_F32, 1.f, 65, arena, sizeof arena));
    REFUSED(GS_ELIMIT, rank(10, 100, 257, GS_F32, 1.f, 5, arena, sizeof arena));
    REFUSED(GS_ELIMIT, rank(10, (int64_t)1 << 31, 32, GS_F32, 1.f, 5, arena, sizeof arena));
    REFUSED(GS_EINVAL, rank(10, 100, 32, GS_F32, 1.f, 5, arena, 64));
    REFUSED(GS_EINVAL, rank(10, 100, 32, GS_F32, 1.f, 5, arena + 16, (size_t)1 << 40));
    REFUSED(GS_EINVAL, rank(10, 100, 32, GS_F32, 1.f, 5, nullptr, (size_t)1 << 40));
    REFUSED(GS_EINVAL, gs_catalog_fwd(p, 10, nullptr, 100, 32, GS_F32, nullptr, 1.f, nullptr, f, f, f, 0, nullptr, nullptr, arena, (size_t)1 << 40, nullptr));
    REFUSED(GS_EINVAL, gs_catalog_fwd(p, 10, p, 100, 32, GS_F32, nullptr, 1.f, nullptr, f, f, f, 5, nullptr, i32, arena, (size_t)1 << 40, nullptr));
    REFUSED(GS_EINVAL, gs_catalog_fwd(odd, 10, p, 100, 32, GS_BF16, nullptr, 1.f, nullptr, f, f, f, 0, nullptr, nullptr, arena, (size_t)1 << 40, nullptr));

    const auto back = [&](int64_t nu, int64_t ni, const float *lse, const float *entropy, const float *g_entropy, void *gu, void *ws, size_t bytes) {
        return gs_catalog_bwd(p, nu, p, ni, 32, GS_F32, nullptr, 1.f, i32, lse, entropy, f, g_entropy, gu, nullptr, nullptr, ws, bytes, nullptr);
    };
    ACCEPTED(back(10, 100, f, f, f, nullptr, nullptr, 0));                                       // nothing wanted
    ACCEPTED(back(0, 100, f, f, f, p, nullptr, 0));                                              // no users
    REFUSED(GS_EINVAL, back(10, 100, nullptr, f, f, p, arena, (size_t)1 << 40));
    REFUSED(GS_EINVAL, back(10, 100, f, nullptr, f, p, arena, (size_t)1 << 40));
    REFUSED(GS_EINVAL, back(10, 100, f, f, f, p, arena, 64));
    REFUSED(GS_EINVAL, back(10, 100, f, f, f, p, arena + 32, (size_t)1 << 40));
    REFUSED(GS_ELIMIT, gs_catalog_bwd(p, 10, p, 100, 300, GS_F32, nullptr, 1.f, i32, f, f, f, f, p, p, f, arena, (size_t)1 << 40, nullptr));

    if (failures) { std::printf("%d failures\n", failures); return 1; }
    std::printf("ops_validate ok\n");
    return 0;
}
