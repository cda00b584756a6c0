// Gradients of the attention over neighbors (the dealing of edges: attention.h).
//
// With P = exp(s - lse), recomputed edge by edge, and delta = <g_out, out> (which is sum_e P_e <g_out, v_e>):
//     ds_e = P_e (<g_out, v_e> - delta) scale      g_q = sum over a parent's edges of ds_e k_e
//     g_k[row] = sum over the edges that read it of ds_e q,    g_v[row] = the same sum of P_e g_out
// Two walks.  The parents' walk is the forward's, with sums in place of the running softmax; it also leaves delta and, for
// ragged neighborhoods, the parent of every edge.  The rows' walk is the same with the roles exchanged: the row's keys
// and values stay in registers and the queries and g_out of the edges that read it arrive, so a row's gradient is summed
// in registers in the order of its list, and no atomics are needed.
#include "attention.h"

namespace {

using gs::Neighbors;
using gs::RowPart;

struct BwdArgs {
    Neighbors nb;
    const void *q, *k, *v, *out, *g_out;
    const float *lse;
    void *g_q, *g_k, *g_v;
    float *delta;                                   // [n_parents][heads]
    int32_t *edge_parent;                           // [n_edges], ragged neighborhoods only
    const int64_t *inv_indptr;
    const int32_t *inv_edges;
    float *piece;                                   // parents: [workers][2][heads][dim]; rows: [workers][2][kv_heads][2][dim]
    float scale;
    int heads, kv_heads, dim, chunk, parts;
    uint32_t n_inv;
};

template <class T, int L, int G, bool ALIGNED>
__global__ __launch_bounds__(gs::kAttnThreads)
void attn_bwd_parents_kernel(BwdArgs a) {
    constexpr int E = gs::Pack<T>::E, U = 4;
    constexpr uint32_t W = 64 / L;
    const int lane = threadIdx.x & (L - 1);
    const uint32_t w = blockIdx.x * (gs::kAttnThreads / L) + threadIdx.x / L;
    const int share = a.heads / a.kv_heads;
    const int j = blockIdx.y / a.parts, h0 = j * share + (blockIdx.y % a.parts) * G;
    const int n_heads = min(G, (j + 1) * share - h0);
    const uint32_t C = a.chunk;
    const T *K = static_cast<const T *>(a.k) + (int64_t)j * a.dim, *V = a.v ? static_cast<const T *>(a.v) + (int64_t)j * a.dim : nullptr;
    const int64_t stride = (int64_t)a.kv_heads * a.dim;
    const float scale2 = a.scale * gs::kLog2e;

    gs::Walk walk(a.nb, w, C, L);
    while (walk.next()) {
        const int64_t p = walk.p;
        const uint32_t begin = walk.begin, end = walk.end;
        if (a.edge_parent && blockIdx.y == 0)
            for (uint32_t i = begin + lane; i < end; i += L) a.edge_parent[i] = (int32_t)p;

        float q[G][E], go[G][E], acc[G][E], delta[G], lse2[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            RowPart<T, L, ALIGNED> r, o, d;
            const int64_t at = p * a.heads + h0 + g;
            lse2[g] = -INFINITY;
            if (g < n_heads) {
                r.load(static_cast<const T *>(a.q) + at * a.dim, lane, a.dim);
                o.load(static_cast<const T *>(a.out) + at * a.dim, lane, a.dim);
                d.load(static_cast<const T *>(a.g_out) + at * a.dim, lane, a.dim);
                lse2[g] = a.lse[at] * gs::kLog2e;
            } else { r.zero(); o.zero(); d.zero(); }
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                q[g][i] = r.at(i) * scale2;
                go[g][i] = d.at(i);
                dot += d.at(i) * o.at(i);
                acc[g][i] = 0.f;
            }
            delta[g] = gs::lanes_sum<L>(dot);
            if (g < n_heads && begin == walk.sb && lane == 0) a.delta[at] = delta[g];
        }
        for (uint32_t e = begin; e < end; e += U) {
            int32_t row[U];
            RowPart<T, L, ALIGNED> kr[U], vr[U];
#pragma unroll
            for (int u = 0; u < U; ++u) row[u] = e + u < end ? a.nb.row_of(e + u) : -1;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (row[u] >= 0) kr[u].load(K + (int64_t)row[u] * stride, lane, a.dim); else kr[u].zero();
                if (V) { if (row[u] >= 0) vr[u].load(V + (int64_t)row[u] * stride, lane, a.dim); else vr[u].zero(); }
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float s = 0.f, dp = 0.f;
#pragma unroll
                    for (int i = 0; i < E; ++i) {
                        s += q[g][i] * kr[u].at(i);
                        dp += go[g][i] * (V ? vr[u].at(i) : kr[u].at(i));
                    }
                    s = gs::lanes_sum<L>(s);
                    dp = gs::lanes_sum<L>(dp);
                    const bool live = row[u] >= 0 && lse2[g] != -INFINITY;
                    const float ds = live ? gs::fast_exp2(s - lse2[g]) * (dp - delta[g]) : 0.f;
#pragma unroll
                    for (int i = 0; i < E; ++i) acc[g][i] += ds * kr[u].at(i);
                }
            }
        }
        const bool complete = walk.complete(), merge = walk.inside(w, C, W);
        if (a.g_q) {
#pragma unroll
            for (int g = 0; g < G; ++g) {
                if (merge)
#pragma unroll
                    for (int o = L; o < 64; o *= 2)
#pragma unroll
                        for (int i = 0; i < E; ++i) acc[g][i] += __shfl_xor(acc[g][i], o, 64);
                if (g >= n_heads || (merge && w % W)) continue;
#pragma unroll
                for (int i = 0; i < E; ++i) acc[g][i] *= a.scale;
                if (complete) {
                    gs::store_row<T, L, ALIGNED>(static_cast<T *>(a.g_q) + (p * a.heads + h0 + g) * a.dim, lane, a.dim, acc[g]);
                } else {
                    const size_t at = walk.place(w) * a.heads + h0 + g;
#pragma unroll
                    for (int i = 0; i < E; ++i) {
                        const int d = gs::element_of<T, L, ALIGNED>(lane, i);
                        if (d < a.dim) a.piece[at * a.dim + d] = acc[g][i];
                    }
                }
            }
        }
    }
}

// The rows' walk: list entry x of row r is edge inv_edges[x] (or x itself where rows are not read by id: then row x
// has the one entry x).
template <class T, int L, int G, bool ALIGNED>
__global__ __launch_bounds__(gs::kAttnThreads)
void attn_bwd_rows_kernel(BwdArgs a) {
    constexpr int E = gs::Pack<T>::E;
    constexpr int U = G == 1 ? 4 : G == 2 ? 2 : 1;
    constexpr uint32_t W = 64 / L;
    const int lane = threadIdx.x & (L - 1);
    const uint32_t w = blockIdx.x * (gs::kAttnThreads / L) + threadIdx.x / L;
    const int share = a.heads / a.kv_heads, j = blockIdx.y;
    Neighbors rows;                                 // the lists of the rows, walked as the parents' are
    rows.indptr = a.inv_indptr;
    rows.ids = nullptr;
    rows.n_parents = a.nb.n_rows;
    rows.n_child = 1;
    rows.n_edges = a.n_inv;
    const uint32_t C = a.chunk;
    const T *Q = static_cast<const T *>(a.q), *GO = static_cast<const T *>(a.g_out);
    const int64_t stride = (int64_t)a.kv_heads * a.dim;
    const float scale2 = a.scale * gs::kLog2e;
    int64_t first = 0, last = a.nb.n_edges;         // edges that belong to a parent
    if (!a.inv_indptr && a.nb.indptr) { first = a.nb.indptr[0]; last = a.nb.indptr[a.nb.n_parents]; }

    gs::Walk walk(rows, w, C, L);
    while (walk.next()) {
        const int64_t r = walk.p;
        const uint32_t end = walk.end;
        float key[E], val[E], gk[E], gv[E];
        {
            RowPart<T, L, ALIGNED> kr, vr;
            kr.load(static_cast<const T *>(a.k) + r * stride + (int64_t)j * a.dim, lane, a.dim);
            if (a.v) vr.load(static_cast<const T *>(a.v) + r * stride + (int64_t)j * a.dim, lane, a.dim); else vr = kr;
#pragma unroll
            for (int i = 0; i < E; ++i) { key[i] = kr.at(i) * scale2; val[i] = vr.at(i); gk[i] = 0.f; gv[i] = 0.f; }
        }
        bool read = false;
        for (uint32_t e = walk.begin; e < end; e += U) {
            int32_t p[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                p[u] = -1;
                if (e + u < end) {
                    const int64_t x = a.inv_indptr ? (int64_t)a.inv_edges[e + u] : (int64_t)(e + u);
                    if (x >= first && x < last && (uint64_t)x < a.nb.n_edges) {
                        p[u] = a.nb.indptr ? a.edge_parent[x] : (int32_t)((uint32_t)x / a.nb.n_child);
                        if ((uint64_t)(int64_t)p[u] >= (uint64_t)a.nb.n_parents) p[u] = -1;
                    }
                }
                read |= p[u] >= 0;
            }
            for (int h0 = j * share; h0 < (j + 1) * share; h0 += G) {
                RowPart<T, L, ALIGNED> qr[U][G], gr[U][G];
                float lse2[U][G], delta[U][G];
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        lse2[u][g] = -INFINITY;
                        delta[u][g] = 0.f;
                        if (p[u] >= 0 && h0 + g < (j + 1) * share) {
                            const int64_t at = (int64_t)p[u] * a.heads + h0 + g;
                            qr[u][g].load(Q + at * a.dim, lane, a.dim);
                            gr[u][g].load(GO + at * a.dim, lane, a.dim);
                            lse2[u][g] = a.lse[at] * gs::kLog2e;
                            delta[u][g] = a.delta[at];
                        } else { qr[u][g].zero(); gr[u][g].zero(); }
                    }
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        float s = 0.f, dp = 0.f;
#pragma unroll
                        for (int i = 0; i < E; ++i) { s += key[i] * qr[u][g].at(i); dp += val[i] * gr[u][g].at(i); }
                        s = gs::lanes_sum<L>(s);
                        dp = gs::lanes_sum<L>(dp);
                        const float pr = lse2[u][g] != -INFINITY ? gs::fast_exp2(s - lse2[u][g]) : 0.f;
                        const float ds = pr * (dp - delta[u][g]) * a.scale;
#pragma unroll
                        for (int i = 0; i < E; ++i) { gk[i] += ds * qr[u][g].at(i); gv[i] += pr * gr[u][g].at(i); }
                    }
            }
        }
        const bool complete = walk.complete();
        if (!a.v)
#pragma unroll
            for (int i = 0; i < E; ++i) gk[i] += gv[i];
        if (complete) {
            if (a.inv_indptr || read) {
                const int64_t at = r * stride + (int64_t)j * a.dim;
                if (a.g_k) gs::store_row<T, L, ALIGNED>(static_cast<T *>(a.g_k) + at, lane, a.dim, gk);
                if (a.g_v) gs::store_row<T, L, ALIGNED>(static_cast<T *>(a.g_v) + at, lane, a.dim, gv);
            }
        } else {
            if (walk.inside(w, C, W)) {
#pragma unroll
                for (int o = L; o < 64; o *= 2)
#pragma unroll
                    for (int i = 0; i < E; ++i) { gk[i] += __shfl_xor(gk[i], o, 64); gv[i] += __shfl_xor(gv[i], o, 64); }
                if (w % W) continue;
            }
            const size_t at = (walk.place(w) * a.kv_heads + j) * 2;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const int d = gs::element_of<T, L, ALIGNED>(lane, i);
                if (d < a.dim) { a.piece[at * a.dim + d] = gk[i]; a.piece[(at + 1) * a.dim + d] = gv[i]; }
            }
        }
    }
}

// Adds the pieces of the lists that were cut, in worker order, and writes zeros for empty ones.  `sets` vectors of dim
// floats per (list, y): the parents' walk has one (y a head), the rows' two (y a key head).  Few pieces: one wave alone.
constexpr uint32_t kFewPieces = 16;

template <class T>
__global__ __launch_bounds__(gs::kJoinWaves * 64)
void attn_bwd_join_kernel(Neighbors seg, const float *piece, int per_slot, int sets, int dim, int chunk, int per_wave, T *out0,
                          T *out1) {
    constexpr int N = gs::kJoinWaves;
    __shared__ float part[N][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, y = blockIdx.y;
    const int64_t mine = (int64_t)lane * gridDim.x + blockIdx.x;
    uint32_t b = 0, e = 0;
    if (mine < seg.n_parents) seg.range(mine, b, e);
    const bool mine_todo = mine < seg.n_parents && gs::needs_join(b, e, chunk);
    const bool many = mine_todo && e > b && gs::PieceList(b, e, chunk, per_wave).count() > kFewPieces;
    unsigned long long few = __ballot(mine_todo && !many), long_ones = __ballot(many);
    const auto add = [&](uint32_t sb, uint32_t se, uint32_t i0, uint32_t step, int set, float (&acc)[4]) {
        const gs::PieceList list(sb, se, chunk, per_wave);
        const uint32_t n = list.count();
#pragma unroll 4
        for (uint32_t i = i0; i < n; i += step) {
            const size_t at = ((list.place(i) * per_slot + y) * sets + set) * dim;
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (lane + 64 * c < dim) acc[c] += piece[at + lane + 64 * c];
        }
    };
    for (int turn = 0; few; ++turn, few &= few - 1) {
        if (turn % N != wave) continue;
        const int src = __builtin_ctzll(few);
        const uint32_t sb = __shfl(b, src, 64), se = __shfl(e, src, 64);
        const int64_t p = (int64_t)src * gridDim.x + blockIdx.x;
        for (int set = 0; set < sets; ++set) {
            T *out = set ? out1 : out0;
            if (!out) continue;
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            if (se > sb) add(sb, se, 0, 1, set, acc);
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (lane + 64 * c < dim) out[(p * per_slot + y) * dim + lane + 64 * c] = (T)acc[c];
        }
    }
    for (; long_ones; long_ones &= long_ones - 1) {
        const int src = __builtin_ctzll(long_ones);
        const uint32_t sb = __shfl(b, src, 64), se = __shfl(e, src, 64);
        const int64_t p = (int64_t)src * gridDim.x + blockIdx.x;
        for (int set = 0; set < sets; ++set) {
            T *out = set ? out1 : out0;
            if (!out) continue;
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            add(sb, se, wave, N, set, acc);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i) part[wave][lane + 64 * i] = acc[i];
            __syncthreads();
            if (threadIdx.x < dim) {
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < N; ++i) sum += part[i][threadIdx.x];
                out[(p * per_slot + y) * dim + threadIdx.x] = (T)sum;
            }
        }
    }
}

template <class T, int L, bool ALIGNED>
void launch_parents(const BwdArgs &a, int64_t workers, hipStream_t stream) {
    const int share = a.heads / a.kv_heads, g = share >= 3 ? 4 : share;
    BwdArgs b = a;
    b.parts = (share + g - 1) / g;
    const dim3 grid((unsigned)((workers * L + gs::kAttnThreads - 1) / gs::kAttnThreads), (unsigned)(a.kv_heads * b.parts));
    if (g == 1) attn_bwd_parents_kernel<T, L, 1, ALIGNED><<<grid, gs::kAttnThreads, 0, stream>>>(b);
    else if (g == 2) attn_bwd_parents_kernel<T, L, 2, ALIGNED><<<grid, gs::kAttnThreads, 0, stream>>>(b);
    else attn_bwd_parents_kernel<T, L, 4, ALIGNED><<<grid, gs::kAttnThreads, 0, stream>>>(b);
}

template <class T, int L, bool ALIGNED>
void launch_rows(const BwdArgs &a, int64_t workers, hipStream_t stream) {
    const int share = a.heads / a.kv_heads;
    const dim3 grid((unsigned)((workers * L + gs::kAttnThreads - 1) / gs::kAttnThreads), (unsigned)a.kv_heads);
    if (share == 1) attn_bwd_rows_kernel<T, L, 1, ALIGNED><<<grid, gs::kAttnThreads, 0, stream>>>(a);
    else if (share == 2) attn_bwd_rows_kernel<T, L, 2, ALIGNED><<<grid, gs::kAttnThreads, 0, stream>>>(a);
    else attn_bwd_rows_kernel<T, L, 4, ALIGNED><<<grid, gs::kAttnThreads, 0, stream>>>(a);
}

#define GS_BY_LANES(f, ...)                                                \
    do {                                                                   \
        if (aligned) {                                                     \
            if (lanes == 4) f<T, 4, true>(__VA_ARGS__);                    \
            else if (lanes == 8) f<T, 8, true>(__VA_ARGS__);               \
            else if (lanes == 16) f<T, 16, true>(__VA_ARGS__);             \
            else if (lanes == 32) f<T, 32, true>(__VA_ARGS__);             \
            else f<T, 64, true>(__VA_ARGS__);                              \
        } else {                                                           \
            if (lanes == 4) f<T, 4, false>(__VA_ARGS__);                   \
            else if (lanes == 8) f<T, 8, false>(__VA_ARGS__);              \
            else if (lanes == 16) f<T, 16, false>(__VA_ARGS__);            \
            else if (lanes == 32) f<T, 32, false>(__VA_ARGS__);            \
            else f<T, 64, false>(__VA_ARGS__);                             \
        }                                                                  \
    } while (0)

struct Plan {
    gs::Deal parents, rows;
    size_t off_parent, off_piece, total;
};

// The pieces of both walks share a region: the second walk starts when the first one's pieces are joined.
Plan make_plan(const gs_neighbors *nb, int heads, int kv_heads, int dim, int dtype, int64_t n_inv) {
    Plan p;
    const int lanes = gs::lanes_for(dim, gs::dtype_size(dtype));
    p.parents = gs::deal_edges(nb->indptr, nb->n_parents, nb->n_child, nb->n_edges, lanes);
    static const int64_t ragged = 0;                // any address: the rows' lists are ragged
    p.rows = nb->ids ? gs::deal_edges(&ragged, nb->n_rows, 0, n_inv, lanes)
                     : gs::deal_edges(nullptr, nb->n_rows, 1, nb->n_rows, lanes);
    size_t off = gs::align256((size_t)nb->n_parents * heads * sizeof(float));        // delta
    p.off_parent = off;
    if (nb->indptr) off += gs::align256((size_t)nb->n_edges * sizeof(int32_t));
    p.off_piece = off;
    size_t piece = 0;
    if (p.parents.pieces) piece = (size_t)p.parents.workers * 2 * heads * dim * sizeof(float);
    if (p.rows.pieces) {
        const size_t r = (size_t)p.rows.workers * 4 * kv_heads * dim * sizeof(float);
        if (r > piece) piece = r;
    }
    p.total = off + piece;
    return p;
}

template <class T>
int run_bwd(BwdArgs a, const Plan &p, int lanes, bool aligned, hipStream_t stream) {
    a.chunk = (int)p.parents.chunk;
    if (p.parents.workers) {
        GS_BY_LANES(launch_parents, a, p.parents.workers, stream);
        if (int rc = gs::check_launch("gs_neighbor_attention_bwd (parents)")) return rc;
    }
    if (a.g_q && a.nb.n_parents && p.parents.pieces) {
        attn_bwd_join_kernel<T><<<dim3((unsigned)((a.nb.n_parents + 63) / 64), (unsigned)a.heads), gs::kJoinWaves * 64, 0, stream>>>(
            a.nb, a.piece, a.heads, 1, a.dim, a.chunk, 64 / lanes, static_cast<T *>(a.g_q), (T *)nullptr);
        if (int rc = gs::check_launch("gs_neighbor_attention_bwd (parents' join)")) return rc;
    }
    if (!a.g_k && !a.g_v) return GS_OK;
    a.chunk = (int)p.rows.chunk;
    if (p.rows.workers) {
        GS_BY_LANES(launch_rows, a, p.rows.workers, stream);
        if (int rc = gs::check_launch("gs_neighbor_attention_bwd (rows)")) return rc;
    }
    if (a.inv_indptr && a.nb.n_rows) {
        Neighbors rows = a.nb;
        rows.indptr = a.inv_indptr;
        rows.n_parents = a.nb.n_rows;
        rows.n_edges = a.n_inv;
        attn_bwd_join_kernel<T><<<dim3((unsigned)((a.nb.n_rows + 63) / 64), (unsigned)a.kv_heads), gs::kJoinWaves * 64, 0, stream>>>(
            rows, a.piece, a.kv_heads, 2, a.dim, a.chunk, 64 / lanes, static_cast<T *>(a.g_k), static_cast<T *>(a.g_v));
        return gs::check_launch("gs_neighbor_attention_bwd (rows' join)");
    }
    return GS_OK;
}

}  // namespace

extern "C" size_t gs_neighbor_attention_bwd_workspace(const gs_neighbors *nb, int heads, int kv_heads, int dim, int dtype,
                                                      int64_t n_inv) {
    if (gs::check_neighbors("gs_neighbor_attention_bwd_workspace", nb, heads, kv_heads, dim, dtype)) return 0;
    if (n_inv < 0) { gs::fail(GS_EINVAL, "gs_neighbor_attention_bwd_workspace: n_inv=%lld", (long long)n_inv); return 0; }
    return make_plan(nb, heads, kv_heads, dim, dtype, n_inv).total;
}

extern "C" int gs_neighbor_attention_bwd(const void *q, const void *k, const void *v, const gs_neighbors *nb, int heads,
                                         int kv_heads, int dim, int dtype, float scale, const void *out, const float *lse,
                                         const void *g_out, const int64_t *inv_indptr, const int32_t *inv_edges,
                                         int64_t n_inv, void *g_q, void *g_k, void *g_v, void *workspace,
                                         size_t workspace_bytes, void *stream) {
    const char *what = "gs_neighbor_attention_bwd";
    if (int rc = gs::check_neighbors(what, nb, heads, kv_heads, dim, dtype)) return rc;
    if (!v) g_v = nullptr;
    if (!g_q && !g_k && !g_v) return GS_OK;
    const bool rows = g_k || g_v;
    const int size = gs::dtype_size(dtype), lanes = gs::lanes_for(dim, size);
    if (nb->n_parents && (!q || !out || !lse || !g_out)) return gs::fail(GS_EINVAL, "%s: null pointer argument", what);
    if (nb->n_edges && nb->n_rows && !k) return gs::fail(GS_EINVAL, "%s: null pointer argument", what);
    if (rows && nb->ids && (!inv_indptr || n_inv < 0 || n_inv > nb->n_edges || (n_inv && !inv_edges)))
        return gs::fail(GS_EINVAL, "%s: rows read by id need the inverse lists (n_inv=%lld of %lld edges)", what,
                        (long long)n_inv, (long long)nb->n_edges);
    const uintptr_t all = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)g_out | (uintptr_t)g_q |
                          (uintptr_t)g_k | (uintptr_t)g_v;
    if (all & (size - 1)) return gs::fail(GS_EINVAL, "%s: pointer not aligned to its element", what);
    const Plan p = make_plan(nb, heads, kv_heads, dim, dtype, nb->ids ? n_inv : 0);
    if (workspace_bytes < p.total || (p.total && (!workspace || ((uintptr_t)workspace & 15))))
        return gs::fail(GS_EINVAL, "%s: aligned workspace of %zu bytes needed, %zu given", what, p.total, workspace_bytes);
    if (nb->n_parents == 0 && (!rows || nb->n_rows == 0 || !nb->ids)) return GS_OK;
    BwdArgs a;
    a.nb = Neighbors{nb->indptr, nb->ids, nb->n_parents, nb->id_offset, nb->n_rows, (uint32_t)(nb->indptr ? 0 : nb->n_child), (uint32_t)nb->n_edges};
    a.q = q; a.k = k; a.v = v; a.out = out; a.g_out = g_out; a.lse = lse;
    a.g_q = g_q; a.g_k = g_k; a.g_v = g_v;
    char *ws = static_cast<char *>(workspace);
    a.delta = reinterpret_cast<float *>(ws);
    a.edge_parent = nb->indptr ? reinterpret_cast<int32_t *>(ws + p.off_parent) : nullptr;
    a.piece = reinterpret_cast<float *>(ws + p.off_piece);
    a.inv_indptr = nb->ids ? inv_indptr : nullptr;
    a.inv_edges = nb->ids ? inv_edges : nullptr;
    a.n_inv = (uint32_t)(nb->ids ? n_inv : nb->n_rows);
    a.scale = scale;
    a.heads = heads; a.kv_heads = kv_heads; a.dim = dim; a.chunk = 0; a.parts = 1;
    const bool aligned = (dim * size) % 16 == 0 && (all & 15) == 0;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == GS_F32) return run_bwd<float>(a, p, lanes, aligned, s);
    if (dtype == GS_BF16) return run_bwd<__bf16>(a, p, lanes, aligned, s);
    return run_bwd<_Float16>(a, p, lanes, aligned, s);
}
