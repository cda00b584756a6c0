// Gradients of the log probabilities and the entropy over a catalog (layout and tile product: catalog.h).
//
//     dz[n][j] = p_j (A_n + B_n log p_j) + [j = target_n] g_n,   A = -(g + g_entropy entropy),  B = -g_entropy
//     g_user = scale dz item,   g_item = scale dz^T user,   g_bias = column sums of dz
// Two launches of one kernel.  A wave owns 32 rows of one table and streams tiles of the other: the tile product gives
// it 32 x 32 scores with its own row in the lane, dz is formed in place, cut into bf16 pieces (two for 16-bit tables,
// three for fp32: what a piece leaves out is 2^-16 or 2^-24 of an element, well under the rounding of the result) and
// multiplied with the same streamed rows, cols layout, into the accumulators of the 32 gradients.  Nothing of the scores or dz goes
// through memory; the scores are computed twice.  The streamed table is cut into shares so that the launch fills
// the chip; the shares' sums are added in share order by a second launch.
#include "catalog.h"

namespace {

using namespace gs;

struct Stats {                                      // per user, padded to whole tiles
    float *lse2, *a, *b2, *g;
    int32_t *target;
};

// lse2 = 1e14 silences a user: padding, or one for whom nothing is on offer.
__global__ __launch_bounds__(kCatThreads)
void catalog_stats_kernel(Stats s, int64_t n_users, int64_t n_padded, int64_t n_items, const int32_t *targets, const float *lse,
                          const float *entropy, const float *g_log_prob, const float *g_entropy) {
    const int64_t n = (int64_t)blockIdx.x * kCatThreads + threadIdx.x;
    if (n >= n_padded) return;
    float l = 1e14f, a = 0.f, b = 0.f, g = 0.f;
    int32_t t = -1;
    if (n < n_users && lse[n] != -INFINITY) {
        l = lse[n] * kLog2e;
        if (targets && g_log_prob && targets[n] >= 0 && targets[n] < n_items) { t = targets[n]; g = g_log_prob[n]; }
        const float ge = g_entropy ? g_entropy[n] : 0.f;
        a = -(g + (g_entropy ? ge * entropy[n] : 0.f));
        b = -ge * kLn2;
    }
    s.lse2[n] = l; s.a[n] = a; s.b2[n] = b; s.g[n] = g; s.target[n] = t;
}

struct BwdArgs {
    const uint4 *own, *stream_rows, *stream_cols;
    const float *bias2;
    Stats st;
    float *part;                                    // [shares][own tiles * 32][blocks * 32]
    float *part_bias;                               // [shares][own tiles * 32], items only, nullable
    int own_tiles, stream_tiles, shares, tiles_per_share;
    float scale2;
};

template <int P, int DB, bool USERS>
__global__ __launch_bounds__(kCatThreads)
void catalog_bwd_kernel(BwdArgs a) {
    constexpr int KC = 2 * DB, NZ = P == 3 ? 3 : 2, MOST = P == 3 ? 2 : 1;
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int64_t task = (int64_t)blockIdx.x * (kCatThreads / 64) + (threadIdx.x >> 6);
    if (task >= (int64_t)a.own_tiles * a.shares) return;
    const int tile = (int)(task % a.own_tiles), share = (int)(task / a.own_tiles);
    const int t0 = share * a.tiles_per_share, t1 = min(t0 + a.tiles_per_share, a.stream_tiles);
    const int mine = tile * 32 + (lane & 31);

    Fragment<P> own[KC];
    {
        const uint4 *src = a.own + (size_t)tile * KC * P * 64 + lane;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) own[kc] = load_fragment<P>(src, kc);
    }
    float lse2 = 0.f, ca = 0.f, cb = 0.f, cg = 0.f, bias = 0.f, sum = 0.f;
    int target = -1;
    if (USERS) { lse2 = a.st.lse2[mine]; ca = a.st.a[mine]; cb = a.st.b2[mine]; cg = a.st.g[mine]; target = a.st.target[mine]; }
    else bias = a.bias2[mine];
    f32x16 out[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) out[d][r] = 0.f;

    for (int t = t0; t < t1; ++t) {
        const uint4 *rows = a.stream_rows + (size_t)t * KC * P * 64 + lane, *cols = a.stream_cols + (size_t)t * KC * P * 64 + lane;
        f32x16 acc;
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[r] = 0.f;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
            const Fragment<P> f = load_fragment<P>(rows, kc);
            multiply<P, P, 2>(acc, f.p, own[kc].p);
        }
        float dz[16];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int at = t * 32 + 8 * g + 4 * half;
            float x[4], y[4], w[4];
            if (USERS) *reinterpret_cast<float4 *>(x) = *reinterpret_cast<const float4 *>(a.bias2 + at);
            else {
                *reinterpret_cast<float4 *>(x) = *reinterpret_cast<const float4 *>(a.st.lse2 + at);
                *reinterpret_cast<float4 *>(y) = *reinterpret_cast<const float4 *>(a.st.a + at);
                *reinterpret_cast<float4 *>(w) = *reinterpret_cast<const float4 *>(a.st.b2 + at);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 4 * g + i;
                const float lp = USERS ? __builtin_fmaf(acc[r], a.scale2, x[i]) - lse2 : __builtin_fmaf(acc[r], a.scale2, bias) - x[i];
                dz[r] = fast_exp2(lp) * (USERS ? __builtin_fmaf(cb, lp, ca) : __builtin_fmaf(w[i], lp, y[i]));
            }
        }
        // the targets: rarely in this tile
        if (USERS) {
            const int local = target - t * 32;
            if (__any(target >= 0 && (unsigned)local < 32u)) {
                const bool on = target >= 0 && (unsigned)local < 32u && a.bias2[target >= 0 && (unsigned)local < 32u ? target : 0] > kFloor;
#pragma unroll
                for (int r = 0; r < 16; ++r) dz[r] += on && local == row_of_reg(r, lane) ? cg : 0.f;
            }
        } else {
            const int tg = a.st.target[t * 32 + (lane & 31)];
            if (__any(tg >= 0 && (tg >> 5) == tile)) {
                const float g = a.st.g[t * 32 + (lane & 31)];
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int src = row_of_reg(r, lane);
                    const int tr = __shfl(tg, src, 64);
                    const float gr = __shfl(g, src, 64);
                    dz[r] += tr == mine && bias > kFloor ? gr : 0.f;
                }
            }
        }
        if (!USERS && a.part_bias)
#pragma unroll
            for (int r = 0; r < 16; ++r) sum += dz[r];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            bf16x8 z[NZ];
#pragma unroll
            for (int p = 0; p < NZ; ++p) {
                uint32_t word[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t lo = next_piece(dz[8 * h + 2 * i]), hi = next_piece(dz[8 * h + 2 * i + 1]);
                    word[i] = (lo >> 16) | hi;
                }
                z[p] = *reinterpret_cast<const bf16x8 *>(word);
            }
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const Fragment<P> f = load_fragment<P>(cols, h * DB + d);
                multiply<NZ, P, MOST>(out[d], z, f.p);
            }
        }
    }
    float *dst = a.part + ((size_t)share * a.own_tiles + tile) * 32 * (DB * 32) + (lane & 31);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) dst[(size_t)row_of_reg(r, lane) * (DB * 32) + d * 32] = out[d][r];
    if (!USERS && a.part_bias) {
        sum += __shfl_xor(sum, 32, 64);
        if (lane < 32) a.part_bias[(size_t)share * a.own_tiles * 32 + mine] = sum;
    }
}

// Adds the shares in order.
template <class T>
__global__ __launch_bounds__(kCatThreads)
void catalog_bwd_join_kernel(const float *part, int shares, int64_t rows, int64_t padded, int dim, int width, float scale, T *out) {
    const int64_t i = (int64_t)blockIdx.x * kCatThreads + threadIdx.x;
    if (i >= rows * dim) return;
    const int64_t row = i / dim;
    const int d = (int)(i - row * dim);
    float s = 0.f;
    for (int k = 0; k < shares; ++k) s += part[((size_t)k * padded + row) * width + d];
    out[i] = (T)(s * scale);
}

struct Space {
    size_t user_rows, user_cols, item_rows, item_cols, bias2, stats, part, part_bias, total;
    int user_shares, user_per, item_shares, item_per;
};

constexpr int64_t kWaves = 4096;

void shares_of(int64_t own, int64_t stream, int *shares, int *per) {
    int64_t s = own ? kWaves / own : 1;
    if (s > stream / 4) s = stream / 4;
    if (s < 1) s = 1;
    *per = stream ? (int)((stream + s - 1) / s) : 1;
    *shares = (int)((stream + *per - 1) / *per);
}

Space space_of(int64_t n_users, int64_t n_items, int dim, int dtype) {
    Space s;
    const int64_t ut = tiles_of(n_users), it = tiles_of(n_items);
    const size_t row = (size_t)32 * blocks_of(dim) * 32 * sizeof(float);
    shares_of(ut, it, &s.user_shares, &s.user_per);
    shares_of(it, ut, &s.item_shares, &s.item_per);
    size_t off = 0;
    s.user_rows = off; off += align256(layout_bytes(n_users, dim, dtype));
    s.user_cols = off; off += align256(layout_bytes(n_users, dim, dtype));
    s.item_rows = off; off += align256(layout_bytes(n_items, dim, dtype));
    s.item_cols = off; off += align256(layout_bytes(n_items, dim, dtype));
    s.bias2 = off; off += align256((size_t)it * 32 * sizeof(float));
    s.stats = off; off += 5 * align256((size_t)ut * 32 * sizeof(float));
    const size_t pu = ut * s.user_shares * row, pi = it * s.item_shares * row;
    s.part = off; off += align256(pu > pi ? pu : pi);
    s.part_bias = off; off += align256((size_t)it * s.item_shares * 32 * sizeof(float));
    s.total = off;
    return s;
}

template <int P, bool USERS>
void launch_bwd(const BwdArgs &a, int blocks, hipStream_t stream) {
    const dim3 grid((unsigned)(((int64_t)a.own_tiles * a.shares + kCatThreads / 64 - 1) / (kCatThreads / 64)));
    if (blocks == 1) catalog_bwd_kernel<P, 1, USERS><<<grid, kCatThreads, 0, stream>>>(a);
    else if (blocks == 2) catalog_bwd_kernel<P, 2, USERS><<<grid, kCatThreads, 0, stream>>>(a);
    else if (blocks == 4) catalog_bwd_kernel<P, 4, USERS><<<grid, kCatThreads, 0, stream>>>(a);
    else catalog_bwd_kernel<P, 8, USERS><<<grid, kCatThreads, 0, stream>>>(a);
}

template <bool USERS>
int run_side(const BwdArgs &a, int pieces, int blocks, hipStream_t stream) {
    if (a.shares > 0) {
        if (pieces == 1) launch_bwd<1, USERS>(a, blocks, stream);
        else if (pieces == 2) launch_bwd<2, USERS>(a, blocks, stream);
        else launch_bwd<3, USERS>(a, blocks, stream);
    }
    return gs::check_launch("gs_catalog_bwd");
}

int run_join(const BwdArgs &a, int dtype, int64_t rows, int dim, int width, float scale, const float *part, void *out, hipStream_t stream) {
    const dim3 grid((unsigned)((rows * dim + kCatThreads - 1) / kCatThreads));
    const int64_t padded = (int64_t)a.own_tiles * 32;
    if (dtype == GS_F32) catalog_bwd_join_kernel<float><<<grid, kCatThreads, 0, stream>>>(part, a.shares, rows, padded, dim, width, scale, static_cast<float *>(out));
    else if (dtype == GS_BF16) catalog_bwd_join_kernel<__bf16><<<grid, kCatThreads, 0, stream>>>(part, a.shares, rows, padded, dim, width, scale, static_cast<__bf16 *>(out));
    else catalog_bwd_join_kernel<_Float16><<<grid, kCatThreads, 0, stream>>>(part, a.shares, rows, padded, dim, width, scale, static_cast<_Float16 *>(out));
    return gs::check_launch("gs_catalog_bwd (join)");
}

}  // namespace

extern "C" size_t gs_catalog_bwd_workspace(int64_t n_users, int64_t n_items, int dim, int dtype) {
    if (gs::check_catalog("gs_catalog_bwd_workspace", n_users, n_items, dim, dtype, 1.f)) return 0;
    return space_of(n_users, n_items, dim, dtype).total;
}

extern "C" int gs_catalog_bwd(const void *user, int64_t n_users, const void *item, int64_t n_items, int dim, int dtype,
                              const float *bias, float scale, const int32_t *targets, const float *lse, const float *entropy,
                              const float *g_log_prob, const float *g_entropy, void *g_user, void *g_item, float *g_bias,
                              void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "gs_catalog_bwd";
    if (int rc = gs::check_catalog(what, n_users, n_items, dim, dtype, scale)) return rc;
    if (n_users == 0) g_user = nullptr;
    if (n_items == 0) g_item = g_bias = nullptr;
    if (!g_user && !g_item && !g_bias) return GS_OK;
    if ((n_users && (!user || !lse || (g_entropy && !entropy))) || (n_items && !item))
        return gs::fail(GS_EINVAL, "%s: null pointer argument", what);
    const int size = gs::dtype_size(dtype);
    if (((uintptr_t)user | (uintptr_t)item | (uintptr_t)g_user | (uintptr_t)g_item) & (size - 1))
        return gs::fail(GS_EINVAL, "%s: pointer not aligned to its element", what);
    const Space sp = space_of(n_users, n_items, dim, dtype);
    if (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < sp.total)
        return gs::fail(GS_EINVAL, "%s: 256-byte aligned workspace of %zu bytes needed, %zu given", what, sp.total, workspace_bytes);
    char *ws = static_cast<char *>(workspace);
    hipStream_t s = (hipStream_t)stream;
    const int blocks = gs::blocks_of(dim), pieces = gs::pieces_of(dtype);
    const bool items = g_item || g_bias;
    const int ut = (int)gs::tiles_of(n_users), it = (int)gs::tiles_of(n_items);
    const size_t each = gs::align256((size_t)ut * 32 * sizeof(float));
    Stats st;
    st.lse2 = reinterpret_cast<float *>(ws + sp.stats);
    st.a = reinterpret_cast<float *>(ws + sp.stats + each);
    st.b2 = reinterpret_cast<float *>(ws + sp.stats + 2 * each);
    st.g = reinterpret_cast<float *>(ws + sp.stats + 3 * each);
    st.target = reinterpret_cast<int32_t *>(ws + sp.stats + 4 * each);
    if (ut) {
        catalog_stats_kernel<<<dim3((unsigned)((ut * 32 + gs::kCatThreads - 1) / gs::kCatThreads)), gs::kCatThreads, 0, s>>>(
            st, n_users, (int64_t)ut * 32, n_items, targets, lse, entropy, g_log_prob, g_entropy);
        if (int rc = gs::check_launch("gs_catalog_bwd (statistics)")) return rc;
    }
    gs::Layout l{};
    l.x = user; l.n_rows = n_users; l.dim = dim; l.blocks = blocks;
    l.rows = reinterpret_cast<uint4 *>(ws + sp.user_rows);
    l.cols = items ? reinterpret_cast<uint4 *>(ws + sp.user_cols) : nullptr;
    if (int rc = gs::launch_layout(l, dtype, s)) return rc;
    l.x = item; l.n_rows = n_items; l.bias = bias;
    l.rows = reinterpret_cast<uint4 *>(ws + sp.item_rows);
    l.cols = g_user ? reinterpret_cast<uint4 *>(ws + sp.item_cols) : nullptr;
    l.bias2 = reinterpret_cast<float *>(ws + sp.bias2);
    if (int rc = gs::launch_layout(l, dtype, s)) return rc;

    BwdArgs a;
    a.bias2 = l.bias2;
    a.st = st;
    a.part = reinterpret_cast<float *>(ws + sp.part);
    a.part_bias = nullptr;
    a.scale2 = scale * gs::kLog2e;
    if (g_user) {
        a.own = reinterpret_cast<const uint4 *>(ws + sp.user_rows);
        a.stream_rows = reinterpret_cast<const uint4 *>(ws + sp.item_rows);
        a.stream_cols = reinterpret_cast<const uint4 *>(ws + sp.item_cols);
        a.own_tiles = ut; a.stream_tiles = it; a.shares = n_items ? sp.user_shares : 0; a.tiles_per_share = sp.user_per;
        if (int rc = run_side<true>(a, pieces, blocks, s)) return rc;
        if (int rc = run_join(a, dtype, n_users, dim, blocks * 32, scale, a.part, g_user, s)) return rc;
    }
    if (items) {
        a.own = reinterpret_cast<const uint4 *>(ws + sp.item_rows);
        a.stream_rows = reinterpret_cast<const uint4 *>(ws + sp.user_rows);
        a.stream_cols = reinterpret_cast<const uint4 *>(ws + sp.user_cols);
        a.own_tiles = it; a.stream_tiles = ut; a.shares = n_users ? sp.item_shares : 0; a.tiles_per_share = sp.item_per;
        a.part_bias = g_bias ? reinterpret_cast<float *>(ws + sp.part_bias) : nullptr;
        if (int rc = run_side<false>(a, pieces, blocks, s)) return rc;
        if (g_item)
            if (int rc = run_join(a, dtype, n_items, dim, blocks * 32, scale, a.part, g_item, s)) return rc;
        if (g_bias)
            if (int rc = run_join(a, GS_F32, n_items, 1, 1, 1.f, a.part_bias, g_bias, s)) return rc;
    }
    return GS_OK;
}
