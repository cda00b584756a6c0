// Gradients of the log probabilities and the entropy over a catalog (layout and tile product: catalog.h).
//
//     dz[n][j] = p_j (A_n + B_n log p_j) + [j = target_n] g_n,   A = -(g + g_entropy entropy),  B = -g_entropy
//     g_user = scale dz item,   g_item = scale dz^T user,   g_bias = column sums of dz
// One launch for both tables.  A wave owns 32 rows of one table and streams tiles of the other: the tile product gives
// it 32 x 32 scores with its own row in the lane, dz is formed in place, cut into as many bf16 pieces as the tables'
// elements have (which leaves out 2^-8 of an element for bf16 tables, 2^-16 for fp16, nothing for fp32; many elements add up
// to a result that is itself rounded to the tables' type) and multiplied, pieces i and k with i + k below their number,
// with the same streamed rows, cols layout, into the accumulators of the 32 gradients.  Nothing of the scores
// or dz goes through memory; the scores are computed twice.  The streamed table is cut into shares so that the launch fills
// the chip; the shares' sums are added in share order by a second launch.
//
// Targets: where one is predicted well, g and -g p cancel, and what a cut leaves out of -g p would stand where g (1 - p) should
// (bf16: 2^-9 of g against the 1e-4 of it that p = 0.9999 leaves).  So a tile that holds targets is followed by a second product
// of matrices that are zero elsewhere: g and what the cut left of -g p, in three pieces, and the product of fp16's second pieces.  The sum then lacks nothing but fp32
// roundings of g.  All targets of a tile cost one such product (4096 users and items of 32 fp32, every user's target an item of its
// own: 47 us with the call, 75 us with a loop over the targets; all the same item: 49 and 106 us).
//
// 4096 users, 100 000 items of 64 bf16: 335 to 390 us for 105 + 52 GFLOP (scores twice, two gradients), bound by issue: the vector ALU
// is busy 68% of the time (2 x 410M dz at an exponential and about ten more instructions each), the matrix cores 33%, one after the
// other.
#include "catalog.h"

#include <algorithm>

namespace {

using namespace gs;

struct Side {                                       // one of the two gradients
    const uint4 *own, *stream_rows, *stream_cols;
    float *part;                                    // [shares][own tiles * 32][blocks * 32]
    void *out;                                      // items': written at once where there is one share
    int64_t own_rows;
    int own_tiles, stream_tiles, shares, tiles_per_share;
};

struct BwdArgs {
    Side users, items;
    const float *bias2;
    const Stats *stats;                             // of the users' tiles
    float *part_bias, *g_bias;                      // [shares][own tiles * 32]; nullable
    int user_blocks, item_blocks, dim;
    float scale, scale2;
};

// Fragments of a streamed tile: rows, cols and, of users, their statistics.  Where two tiles do not fit into LDS (fp32 of
// more than 128 elements) every wave reads its own from L2.
template <int P, int DB, bool USERS> constexpr int kTile = 4 * DB * P + (USERS ? 0 : 1);
template <int P, int DB> constexpr bool kStaged = fits_lds(kTile<P, DB, false>);

template <class T, int DB, bool USERS>
__device__ __forceinline__ void backward(const BwdArgs &a, const Side &side, uint32_t block, uint4 *stage) {
    constexpr int P = Pieces<T>::P, KC = 2 * DB, W = kCatThreads / 64;
    constexpr int F = kTile<P, DB, USERS>, ST = kStaged<P, DB> ? tiles_per_stage(F) : 1;
    constexpr bool STAGED = kStaged<P, DB>;
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t lds = __builtin_amdgcn_readfirstlane((uint32_t)reinterpret_cast<uintptr_t>(stage));
    const uint32_t tile_blocks = (side.own_tiles + W - 1) / W;
    const int tile_mine = (int)(block % tile_blocks) * W + wave, share = (int)(block / tile_blocks);
    const bool live = tile_mine < side.own_tiles;   // a wave past the last tile repeats it and writes nothing
    const int tile = live ? tile_mine : side.own_tiles - 1;
    const int t0 = share * side.tiles_per_share, t1 = min(t0 + side.tiles_per_share, side.stream_tiles);
    const int mine = tile * 32 + (lane & 31);
    const auto issue = [&](int t, int to) {
#pragma unroll
        for (int k = 0; k < ST; ++k)
            if (t + k < t1)
#pragma unroll
                for (int i = 0; i < (F + W - 1) / W; ++i) {
                    const int f = i * W + wave;
                    if (f >= F) continue;
                    const uint4 *src = f < KC * P ? side.stream_rows + ((size_t)(t + k) * KC * P + f) * 64
                                       : f < 2 * KC * P ? side.stream_cols + ((size_t)(t + k) * KC * P + f - KC * P) * 64
                                                        : reinterpret_cast<const uint4 *>(a.stats + t + k);
                    fragment_to_lds(src, lane, lds + ((to * ST + k) * F + f) * 1024);
                }
    };
    if (STAGED) issue(t0, 0);

    Fragment<P> own[KC];
    {
        const uint4 *src = side.own + (size_t)tile * KC * P * 64;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) own[kc] = load_fragment<P>(src, kc, lane);
    }
    float lse2 = 0.f, ca = 0.f, cb = 0.f, bias = 0.f, sum = 0.f, g = 0.f;
    int target = -1;
    if (USERS) {
        const Stats &st = a.stats[tile];
        const int i = lane & 31;
        lse2 = st.lse2[i]; ca = st.a[i]; cb = st.b2[i];
        g = st.g[i]; target = st.target[i];
    } else bias = a.bias2[mine];
    f32x16 out[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) out[d][r] = 0.f;

    for (int t = t0; t < t1; ++t) {
        const uint4 *rows, *cols;
        const Stats *st;
        if constexpr (STAGED) {
            const int at = (t - t0) % ST, from = (t - t0) / ST % 2;
            if (at == 0) {
                stage_ready();
                if (t + ST < t1) issue(t + ST, from ^ 1);
            }
            rows = stage + (from * ST + at) * F * 64;
            cols = rows + KC * P * 64;
            st = reinterpret_cast<const Stats *>(cols + KC * P * 64);
        } else {
            rows = side.stream_rows + (size_t)t * KC * P * 64;
            cols = side.stream_cols + (size_t)t * KC * P * 64;
            st = a.stats + t;
        }
        f32x16 acc;
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[r] = 0.f;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
            const Fragment<P> it = load_fragment<P>(rows, kc, lane);
            multiply<P, P, 2>(acc, it.p, own[kc].p);
        }
        float dz[16];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int i = 8 * q + 4 * half;
            float x[4], y[4], w[4];
            if (USERS) *reinterpret_cast<float4 *>(x) = *reinterpret_cast<const float4 *>(a.bias2 + t * 32 + i);
            else {
                *reinterpret_cast<float4 *>(x) = *reinterpret_cast<const float4 *>(st->lse2 + i);
                *reinterpret_cast<float4 *>(y) = *reinterpret_cast<const float4 *>(st->a + i);
                *reinterpret_cast<float4 *>(w) = *reinterpret_cast<const float4 *>(st->b2 + i);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int r = 4 * q + k;
                const float lp = USERS ? __builtin_fmaf(acc[r], a.scale2, x[k]) - lse2 : __builtin_fmaf(acc[r], a.scale2, bias) - x[k];
                dz[r] = fast_exp2(lp) * (USERS ? __builtin_fmaf(cb, lp, ca) : __builtin_fmaf(w[k], lp, y[k]));
            }
        }
        if (!USERS && a.g_bias) {                   // (a tile's elements first: thousands one by one would cost digits)
            float x[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) x[r] = dz[2 * r] + dz[2 * r + 1];
            sum += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        }
        bf16x8 last[2];                             // fp16: the piece whose product with the elements' second one is left out
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            bf16x8 z[P];
            cut_pieces<P>(dz + 8 * h, z);           // (dz keeps what is left of it: nothing of fp32)
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const Fragment<P> ct = load_fragment<P>(cols, h * DB + d, lane);
                multiply<P, P, P - 1>(out[d], z, ct.p);
            }
            last[h] = z[P - 1];
        }
        // targets: rarely in this tile
        const int tg = USERS ? target - t * 32 : st->target[lane & 31] - tile * 32;
        if (!__any((unsigned)tg < 32u)) continue;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            // (a half of the streamed rows at a time: the lane's target there, or the lane is the target's user)
            if (!__any((unsigned)tg < 32u && (USERS ? tg : lane & 31) >> 4 == h)) continue;
            float w[8];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int i = 16 * h + 8 * q + 4 * half;
                int32_t to[4];
                float gr[4];
                if (!USERS) {
                    *reinterpret_cast<int4 *>(to) = *reinterpret_cast<const int4 *>(st->target + i);
                    *reinterpret_cast<float4 *>(gr) = *reinterpret_cast<const float4 *>(st->g + i);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const bool hit = USERS ? tg == i + k : to[k] == mine && !(bias < kFloor);       // (not on offer: nothing)
                    w[4 * q + k] = hit ? (USERS ? g : gr[k]) + (P < 3 ? dz[8 * h + 4 * q + k] : 0.f) : 0.f;
                    if (!USERS) sum += hit ? gr[k] : 0.f;
                    if (P == 2 && !hit) last[h][4 * q + k] = (__bf16)0.f;
                }
            }
            bf16x8 z[3];
            cut_pieces<3>(w, z);
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const Fragment<P> ct = load_fragment<P>(cols, h * DB + d, lane);
                multiply<3, P, 2>(out[d], z, ct.p);
                if constexpr (P == 2) multiply<1, 1, 0>(out[d], last + h, ct.p + 1);
            }
        }
    }
    if (!live) return;
    if (!USERS && side.out && side.shares == 1) {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int64_t row = (int64_t)tile * 32 + row_of_reg(r, lane);
                const int col = d * 32 + (lane & 31);
                if (row < side.own_rows && col < a.dim) static_cast<T *>(side.out)[row * a.dim + col] = (T)(out[d][r] * a.scale);
            }
    } else if (side.out) {
        float *dst = side.part + ((size_t)share * side.own_tiles + tile) * 32 * (DB * 32) + (lane & 31);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) dst[(size_t)row_of_reg(r, lane) * (DB * 32) + d * 32] = out[d][r];
    }
    if (!USERS && a.g_bias) {
        sum += __shfl_xor(sum, 32, 64);
        if (lane < 32 && side.shares > 1) a.part_bias[(size_t)share * side.own_tiles * 32 + mine] = sum;
        else if (lane < 32 && mine < side.own_rows) a.g_bias[mine] = sum;
    }
}

// Three waves per SIMD where 168 registers do (4096 users, 100 000 items of 64 fp32: 1174 us, 1210 with 170 and two).
constexpr int waves_of(int registers) { return registers <= 112 ? 3 : waves_for(registers); }

// Both gradients in one launch: the first blocks own users, the others items.
template <class T, int DB>
__global__ __launch_bounds__(kCatThreads, waves_of(8 * DB * Pieces<T>::P + 16 * DB + 32))
void catalog_bwd_kernel(BwdArgs a) {
    extern __shared__ uint4 stage[];
    if ((int)blockIdx.x < a.user_blocks) backward<T, DB, true>(a, a.users, blockIdx.x, stage);
    else backward<T, DB, false>(a, a.items, blockIdx.x - a.user_blocks, stage);
}

// Adds the shares in a fixed order: users' elements, then items', then the bias.
struct JoinArgs {
    int64_t first;                                  // the element that the launch begins with
    const float *user_part, *item_part, *bias_part;
    int user_shares, item_shares, dim, width;
    int64_t user_n, item_n, bias_n, user_padded, item_padded;          // *_n: elements to write, 0 for none
    float scale;
    void *g_user, *g_item;
    float *g_bias;
};

// A block takes 32 elements, N threads each.
template <class T, int N>
__global__ __launch_bounds__(32 * N)
void catalog_bwd_join_kernel(JoinArgs a) {
    __shared__ float sums[N][32];
    const int part_of = threadIdx.x >> 5;
    int64_t i = a.first + (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
    const bool in = i < a.user_n + a.item_n + a.bias_n;
    const bool user = i < a.user_n, item = !user && i < a.user_n + a.item_n;
    const float *part = a.bias_part;
    int64_t each = a.item_padded;
    int shares = in ? (user ? a.user_shares : a.item_shares) : 0;
    if (user || item) {
        if (item) i -= a.user_n;
        const int64_t row = i / a.dim;
        part = (user ? a.user_part : a.item_part) + row * a.width + (i - row * a.dim);
        each = (user ? a.user_padded : a.item_padded) * a.width;
    } else {
        i -= a.user_n + a.item_n;
        part += i;
    }
    float s = 0.f;
#pragma unroll 8
    for (int k = part_of; k < shares; k += N) s += part[(size_t)k * each];
    sums[part_of][threadIdx.x & 31] = s;
    __syncthreads();
    if (part_of || !in) return;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) s += sums[k][threadIdx.x];
    if (user) static_cast<T *>(a.g_user)[i] = (T)(s * a.scale);
    else if (item) static_cast<T *>(a.g_item)[i] = (T)(s * a.scale);
    else a.g_bias[i] = s;
}

struct Space {
    size_t user_rows, user_cols, item_rows, item_cols, bias2, stats, user_part, item_part, part_bias, total;
    int user_shares, user_per, item_shares, item_per;
};

constexpr int64_t kBlocks = 512;                    // blocks each side is cut into: with the other's, four waves per SIMD

void shares_of(int64_t own, int64_t stream, int *shares, int *per) {
    constexpr int W = kCatThreads / 64;
    int64_t s = own ? kBlocks / ((own + W - 1) / W) : 1;
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
    s.stats = off; off += (size_t)ut * sizeof(Stats);
    s.user_part = off; off += align256(ut * s.user_shares * row);
    s.item_part = off; off += s.item_shares > 1 ? align256(it * s.item_shares * row) : 0;
    s.part_bias = off; off += s.item_shares > 1 ? align256((size_t)it * s.item_shares * 32 * sizeof(float)) : 0;
    s.total = off;
    return s;
}

template <class T, int DB>
int launch_bwd(const BwdArgs &a, hipStream_t stream) {
    constexpr int P = Pieces<T>::P, FU = kTile<P, DB, true>, FI = kTile<P, DB, false>;
    constexpr int users = FU * tiles_per_stage(FU), items = FI * tiles_per_stage(FI);
    constexpr int lds = kStaged<P, DB> ? 2 * (users > items ? users : items) * 1024 : 0;
    const auto kernel = catalog_bwd_kernel<T, DB>;
    if (lds > 64 * 1024) {
        const hipError_t e = gs::raise_lds_limit(reinterpret_cast<const void *>(kernel), lds);
        if (e != hipSuccess) return gs::fail(GS_ELAUNCH, "gs_catalog_bwd: LDS limit: %s", hipGetErrorString(e));
    }
    kernel<<<dim3((unsigned)(a.user_blocks + a.item_blocks)), kCatThreads, lds, stream>>>(a);
    return gs::check_launch("gs_catalog_bwd");
}

template <class T>
int run_bwd(const BwdArgs &a, JoinArgs j, int blocks, hipStream_t stream) {
    if (a.user_blocks + a.item_blocks) {
        if (int rc = blocks == 1 ? launch_bwd<T, 1>(a, stream) : blocks == 2 ? launch_bwd<T, 2>(a, stream)
                   : blocks == 4 ? launch_bwd<T, 4>(a, stream) : launch_bwd<T, 8>(a, stream))
            return rc;
    }
    const int64_t elements = j.user_n + j.item_n + j.bias_n;
    // 32 threads an element where a side has many shares (five users against 70 000 items leave 441: 19 us with eight)
    const int each = (j.user_n && j.user_shares > 64) || (j.item_n + j.bias_n && j.item_shares > 64) ? 32 : 8;
    for (j.first = 0; j.first < elements; j.first += gs::kMostThreads / each) {
        const dim3 grid((unsigned)((std::min(gs::kMostThreads / each, elements - j.first) + 31) / 32));
        if (each == 32) catalog_bwd_join_kernel<T, 32><<<grid, 1024, 0, stream>>>(j);
        else catalog_bwd_join_kernel<T, 8><<<grid, 256, 0, stream>>>(j);
        if (int rc = gs::check_launch("gs_catalog_bwd (join)")) return rc;
    }
    return GS_OK;
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
    if (n_users + n_items >= (int64_t)1 << 31)      // (a wave for 32 rows of either table, in one launch)
        return gs::fail(GS_ELIMIT, "%s: %lld users and %lld items (less than 2^31 together)", what, (long long)n_users, (long long)n_items);
    const Space sp = space_of(n_users, n_items, dim, dtype);
    if (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < sp.total)
        return gs::fail(GS_EINVAL, "%s: 256-byte aligned workspace of %zu bytes needed, %zu given", what, sp.total, workspace_bytes);
    char *ws = static_cast<char *>(workspace);
    hipStream_t s = (hipStream_t)stream;
    const int blocks = gs::blocks_of(dim);
    constexpr int W = gs::kCatThreads / 64;
    const bool items = g_item || g_bias;
    const int ut = (int)gs::tiles_of(n_users), it = (int)gs::tiles_of(n_items);
    gs::Layout lu{}, li{};
    lu.x = user; lu.n_rows = n_users;
    lu.rows = reinterpret_cast<uint4 *>(ws + sp.user_rows);
    lu.cols = items ? reinterpret_cast<uint4 *>(ws + sp.user_cols) : nullptr;
    lu.stats = reinterpret_cast<gs::Stats *>(ws + sp.stats);
    lu.from = gs::StatsFrom{n_items, targets, lse, entropy, g_log_prob, g_entropy};
    li.x = item; li.n_rows = n_items; li.bias = bias;
    li.rows = reinterpret_cast<uint4 *>(ws + sp.item_rows);
    li.cols = g_user ? reinterpret_cast<uint4 *>(ws + sp.item_cols) : nullptr;
    li.bias2 = reinterpret_cast<float *>(ws + sp.bias2);
    if (int rc = gs::launch_layouts(lu, li, dim, dtype, s)) return rc;

    // a side without anything to stream has no shares: the join writes its zeros
    BwdArgs a{};
    a.bias2 = li.bias2;
    a.stats = lu.stats;
    a.dim = dim;
    a.scale = scale;
    a.scale2 = scale * gs::kLog2e;
    a.g_bias = g_bias;
    a.part_bias = reinterpret_cast<float *>(ws + sp.part_bias);
    JoinArgs j{};
    j.dim = dim; j.width = blocks * 32; j.scale = scale;
    j.g_user = g_user; j.g_item = g_item; j.g_bias = g_bias;
    j.user_padded = (int64_t)ut * 32; j.item_padded = (int64_t)it * 32;
    if (g_user) {
        a.users = Side{lu.rows, li.rows, li.cols, reinterpret_cast<float *>(ws + sp.user_part), g_user, n_users, ut, it,
                       n_items ? sp.user_shares : 0, sp.user_per};
        a.user_blocks = (ut + W - 1) / W * a.users.shares;
        j.user_part = a.users.part; j.user_shares = a.users.shares;
        j.user_n = n_users * dim;
    }
    if (items) {
        a.items = Side{li.rows, lu.rows, lu.cols, reinterpret_cast<float *>(ws + sp.item_part), g_item, n_items, it, ut,
                       n_users ? sp.item_shares : 0, sp.item_per};
        a.item_blocks = (it + W - 1) / W * a.items.shares;
        j.item_part = a.items.part; j.bias_part = a.part_bias; j.item_shares = a.items.shares;
        if (a.items.shares != 1) { j.item_n = g_item ? n_items * dim : 0; j.bias_n = g_bias ? n_items : 0; }
    }
    if (dtype == GS_F32) return run_bwd<float>(a, j, blocks, s);
    if (dtype == GS_BF16) return run_bwd<__bf16>(a, j, blocks, s);
    return run_bwd<_Float16>(a, j, blocks, s);
}
