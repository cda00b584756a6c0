// Gradients of the attention over neighbors (the dealing of edges: attention.h).
//
// With P = exp(s - lse), recomputed edge by edge, and delta = <g_out, out> (which is sum_e P_e <g_out, v_e>):
//     ds_e = P_e (<g_out, v_e> - delta) scale      g_q = sum over a parent's edges of ds_e k_e
//     g_k[row] = sum over the edges that read it of ds_e q,    g_v[row] = the same sum of P_e g_out
// Two walks.  The parents' walk is the forward's, with sums in place of the running softmax; it also leaves delta and, for
// ragged neighborhoods read by id, the parent of every edge.  Dense rows have one reader each: their gradients are written
// as they pass.  For rows read by id the rows' walk is the same with the roles exchanged: the row's keys and values
// stay in registers and the queries and g_out of the edges that read it arrive, so a row's gradient is summed in registers
// in the order of its list, and no atomics are needed.
//
// 8192 dense lists of 25 rows of 32 fp32, four heads: 25 us (the forward 13 us), one wave per SIMD, whose vector ALU is busy 43% of the
// time (48%) and which waits for loads 41% of it (43%).  226 000 ragged edges into 3700 rows of 2 x 33 fp16: parents 40 us, rows 31 us,
// each with a join of 7 to 9 us; nine in ten requests hit L2, the vector ALU is busy 55 to 60% of the time and waves wait 44 to
// 52% of theirs: the work per list (3700 to 6040 lists of 40 to 60 edges) and its latency bound both walks.
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
    float *dense_part;                              // [parts][n_rows][kv_heads][2][dim], dense rows of more heads than one wave takes
    float *piece;                                   // parents: [waves][2][heads][dim]; rows: [waves][2][kv_heads][2][dim]
    float scale;
    int heads, kv_heads, dim, chunk, parts;
    uint32_t n_inv;
};

// What the lanes of a row group keep of a parent: queries and g_out of G heads, delta, lse and the sums of g_q.
template <class T, int L, int G, bool SHARED> struct ParentState {
    static constexpr int E = gs::Pack<T>::E;
    RowPart<T> q[G], go[G], q_next[G], go_next[G], out_next[G];
    float acc[G * E], delta[G], lse2[G], lse_next[G];

    __device__ __forceinline__ void fetch(const BwdArgs &a, int64_t p, int h0, int n_heads, const gs::Place<T, L> &at) {
#pragma unroll
        for (int g = 0; g < G; ++g) {               // (heads past the last one repeat it)
            const int64_t of = p * a.heads + h0 + min(g, n_heads - 1);
            q_next[g].load(static_cast<const T *>(a.q) + of * a.dim, at);
            go_next[g].load(static_cast<const T *>(a.g_out) + of * a.dim, at);
            out_next[g].load(static_cast<const T *>(a.out) + of * a.dim, at);
            lse_next[g] = a.lse[of];
        }
    }
    // `writes`: the lane that leaves delta (every wave that has a part of the list leaves the same bits)
    __device__ __forceinline__ void begin(const BwdArgs &a, int64_t p, int h0, int n_heads, const gs::Place<T, L> &at, bool writes) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            q[g] = q_next[g];
            go[g] = go_next[g];
            q[g].own(at);
            go[g].own(at);
            if (g >= n_heads) { q[g].zero(); go[g].zero(); }           // their part of dense rows' gradients: nothing
            lse2[g] = lse_next[g] * gs::kLog2e;
#pragma unroll
            for (int i = 0; i < E; ++i) acc[g * E + i] = 0.f;
            delta[g] = gs::lanes_sum<L>(gs::dot(go[g], out_next[g]));
            if (g < n_heads && writes) a.delta[p * a.heads + h0 + g] = delta[g];
        }
    }
    // U rows at once; a negative one is none.  Dense rows: nobody else reads them, their gradients are written (`live`).
    template <int U>
    __device__ __forceinline__ void rows(const BwdArgs &a, const int32_t (&row)[U], bool gaps, bool dense, bool live, int j, const T *K,
                                         const T *V, int64_t stride, const gs::Place<T, L> &at) {
        const float scale2 = a.scale * gs::kLog2e;
        RowPart<T> kr[U], vr[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t to = (int64_t)max(row[u], 0) * stride;       // (what is no neighbor reads row 0 and forgets it)
            kr[u].load(K + to, at);
            if (!SHARED) vr[u].load(V + to, at);
        }
        if (gaps)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                kr[u].zero_if(row[u] < 0);
                if (!SHARED) vr[u].zero_if(row[u] < 0);
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float gk[E], gv[E];
#pragma unroll
            for (int i = 0; i < E; ++i) gk[i] = gv[i] = 0.f;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const float s = gs::lanes_sum<L>(gs::dot(q[g], kr[u])) * scale2;
                const float dp = gs::lanes_sum<L>(gs::dot(go[g], SHARED ? kr[u] : vr[u]));
                const float pr = row[u] >= 0 && lse2[g] != -INFINITY ? gs::fast_exp2(s - lse2[g]) : 0.f;
                const float ds = pr * (dp - delta[g]) * a.scale;
#pragma unroll
                for (int i = 0; i < E; ++i) acc[g * E + i] += ds * kr[u].at(i);
                if (dense)
#pragma unroll
                    for (int i = 0; i < E; ++i) { gk[i] += ds * q[g].at(i); gv[i] += pr * go[g].at(i); }
            }
            if (dense && live && row[u] >= 0) {
                if (SHARED)
#pragma unroll
                    for (int i = 0; i < E; ++i) gk[i] += gv[i];
                const int64_t to = (int64_t)row[u] * stride + (int64_t)j * a.dim;
                if (a.parts > 1) {
                    float *part = a.dense_part + ((int64_t)(blockIdx.y % a.parts) * a.nb.n_rows * stride + to) * 2;
                    gs::store_part<E>(part, at, 0, gk);
                    if (!SHARED) gs::store_part<E>(part + a.dim, at, 0, gv);
                } else {
                    if (a.g_k) gs::store_part<E>(static_cast<T *>(a.g_k) + to, at, 0, gk);
                    if (!SHARED && a.g_v) gs::store_part<E>(static_cast<T *>(a.g_v) + to, at, 0, gv);
                }
            }
        }
    }
};

// The parents' walk.  Two rows at a time for four heads, as in the forward pass (300 lists of 2000, four heads of 128 bf16, the whole
// backward pass: 251 us, 326 with four rows).
template <class T, int L, int G, bool SHARED>
__global__ __launch_bounds__(gs::kAttnThreads)
void attn_bwd_parents_kernel(BwdArgs a) {
    constexpr int E = gs::Pack<T>::E, W = 64 / L, U = L == 2 || G == 4 ? 2 : gs::kAttnRows;
    const int lane64 = threadIdx.x & 63, lane = lane64 & (L - 1), group = lane64 / L;
    const int share = a.heads / a.kv_heads;
    const int j = blockIdx.y / a.parts, h0 = j * share + (blockIdx.y % a.parts) * G;
    const int n_heads = min(G, (j + 1) * share - h0);
    const T *K = static_cast<const T *>(a.k) + (int64_t)j * a.dim, *V = SHARED ? nullptr : static_cast<const T *>(a.v) + (int64_t)j * a.dim;
    const int64_t stride = (int64_t)a.kv_heads * a.dim;
    const gs::Place<T, L> at(lane, a.dim);
    const bool dense = !a.nb.ids && (a.g_k || a.g_v);

    gs::Walk walk(a.nb, gs::this_wave(), a.chunk);
    if (a.edge_parent && blockIdx.y == 0) {         // edges before the first list and behind the last have no parent
        const int64_t first = a.nb.offset(0), last = a.nb.offset(a.nb.n_parents);
        if (walk.e0 < first || walk.e1 > last)
            for (uint32_t e = walk.e0 + lane64; e < walk.e1; e += 64)
                if (e < first || e >= last) a.edge_parent[e] = -1;
    }
    bool have = walk.next();
    if (!have) return;
    gs::Unit cur = walk.u;
    int32_t entry = a.nb.entry(cur.e + lane64);
    ParentState<T, L, G, SHARED> st;
    st.fetch(a, cur.p, h0, n_heads, at);
    while (have) {
        if (a.edge_parent && blockIdx.y == 0 && lane64 < cur.n) a.edge_parent[cur.e + lane64] = (int32_t)cur.p;
        if (cur.first) st.begin(a, cur.p, h0, n_heads, at, lane64 == 0);
        const int32_t rows = lane64 < cur.n ? a.nb.row_of(entry) : -1;
        const bool gaps = __any(rows < 0 && lane64 < cur.n) || cur.n % (W * U);
        have = walk.next();
        if (have) {
            entry = a.nb.entry(walk.u.e + lane64);
            if (walk.u.first) st.fetch(a, walk.u.p, h0, n_heads, at);
        }
        for (uint32_t b = 0; b < cur.n; b += W * U) {
            int32_t row[U];
#pragma unroll
            for (int u = 0; u < U; ++u) row[u] = __shfl(rows, b + u * W + group, 64);
            st.template rows<U>(a, row, gaps, dense, true, j, K, V, stride, at);
        }
        if (cur.last && a.g_q) {
            gs::Scatter<G * E, L> mine;
            mine.run(st.acc, lane64);
            constexpr int N = gs::Scatter<G * E, L>::kKept, S = N < E ? N : E;
#pragma unroll
            for (int x = 0; x < N; x += S) {
                const int g = (mine.start + x) / E, start = (mine.start + x) % E;
                if (g >= n_heads || mine.dup) continue;
                if (cur.complete) gs::store_part<S>(static_cast<T *>(a.g_q) + (cur.p * a.heads + h0 + g) * a.dim, at, start, st.acc + x);
                else gs::store_part<S>(a.piece + ((size_t)cur.place * a.heads + h0 + g) * a.dim, at, start, st.acc + x);
            }
        }
        cur = walk.u;
    }
}

// Short lists of one length: L lanes take a parent each.
template <class T, int L, int G, bool SHARED>
__global__ __launch_bounds__(gs::kAttnThreads)
void attn_bwd_short_kernel(BwdArgs a) {
    constexpr int E = gs::Pack<T>::E, W = 64 / L, U = L == 2 ? 2 : gs::kAttnRows;
    const int lane64 = threadIdx.x & 63, lane = lane64 & (L - 1), group0 = lane64 & ~(L - 1);
    const int share = a.heads / a.kv_heads;
    const int j = blockIdx.y / a.parts, h0 = j * share + (blockIdx.y % a.parts) * G;
    const int n_heads = min(G, (j + 1) * share - h0);
    const T *K = static_cast<const T *>(a.k) + (int64_t)j * a.dim, *V = SHARED ? nullptr : static_cast<const T *>(a.v) + (int64_t)j * a.dim;
    const int64_t stride = (int64_t)a.kv_heads * a.dim;
    const gs::Place<T, L> at(lane, a.dim);
    const bool dense = !a.nb.ids && (a.g_k || a.g_v);
    const uint32_t n = a.nb.n_child, n_lists = (uint32_t)a.nb.n_parents, waves = gridDim.x * (gs::kAttnThreads / 64);

    uint32_t base = gs::this_wave() * W;            // of the wave; lists past the last one repeat it
    if (base >= n_lists) return;
    uint32_t p = min(base + lane64 / L, n_lists - 1);
    int32_t entry = a.nb.entry(p * n + lane);
    ParentState<T, L, G, SHARED> st;
    st.fetch(a, p, h0, n_heads, at);
    for (;;) {
        const uint32_t cur = p;
        const bool mine = base + lane64 / L < n_lists;
        st.begin(a, cur, h0, n_heads, at, lane == 0 && mine);
        base += waves * W;
        const bool more = base < n_lists;
        for (uint32_t c = 0; c < n; c += L) {
            const int32_t rows = c + lane < n ? a.nb.row_of(entry) : -1;
            const uint32_t here = min(n - c, (uint32_t)L);
            const bool gaps = __any(rows < 0 && (uint32_t)lane < here) || here % U;
            if (c + L < n) entry = a.nb.entry(p * n + c + L + lane);
            else if (more) {
                p = min(base + lane64 / L, n_lists - 1);
                entry = a.nb.entry(p * n + lane);
                st.fetch(a, p, h0, n_heads, at);
            }
            for (uint32_t b = 0; b < here; b += U) {
                int32_t row[U];
#pragma unroll
                for (int u = 0; u < U; ++u) row[u] = __shfl(rows, group0 + b + u, 64);
                st.template rows<U>(a, row, gaps, dense, mine, j, K, V, stride, at);
            }
        }
        if (mine && a.g_q)
#pragma unroll
            for (int g = 0; g < G; ++g)
                if (g < n_heads) gs::store_part<E>(static_cast<T *>(a.g_q) + ((int64_t)cur * a.heads + h0 + g) * a.dim, at, 0, st.acc + g * E);
        if (!more) return;
    }
}

// The rows' walk, for rows that are read by id: list entry x of row r is edge inv_edges[x].
template <class T, int L, int G, bool SHARED>
__global__ __launch_bounds__(gs::kAttnThreads)
void attn_bwd_rows_kernel(BwdArgs a) {
    constexpr int E = gs::Pack<T>::E, W = 64 / L;
    constexpr int U = G == 1 && L != 2 ? 4 : G <= 2 ? 2 : 1;
    const int lane64 = threadIdx.x & 63, lane = lane64 & (L - 1), group = lane64 / L;
    const int share = a.heads / a.kv_heads, j = blockIdx.y;
    Neighbors lists;                                // the lists of the rows, walked as the parents' are
    lists.indptr = a.inv_indptr;
    lists.ids = nullptr;
    lists.n_parents = lists.n_rows = a.nb.n_rows;
    lists.id_offset = 0;
    lists.n_child = 1;
    lists.n_edges = a.n_inv;
    const T *Q = static_cast<const T *>(a.q), *GO = static_cast<const T *>(a.g_out);
    const int64_t stride = (int64_t)a.kv_heads * a.dim;
    const float scale2 = a.scale * gs::kLog2e;
    const gs::Place<T, L> at(lane, a.dim);
    // an entry's edge, the edge's parent: three steps, each a load (or none) that can be on its way for a while
    const auto edge_at = [&](uint32_t e) { return (uint32_t)a.inv_edges[min(e, a.n_inv - 1)]; };
    const auto parent_at = [&](uint32_t x) { return a.nb.indptr ? a.edge_parent[min(x, a.nb.n_edges - 1)] : (int32_t)(x / a.nb.n_child); };
    const auto checked = [&](uint32_t x, int32_t p) {
        return x < a.nb.n_edges && (uint64_t)(int64_t)p < (uint64_t)a.nb.n_parents ? p : -1;
    };

    gs::Walk walk(lists, gs::this_wave(), a.chunk);
    bool have = walk.next();
    if (!have) return;
    gs::Unit cur = walk.u;
    uint32_t edge = edge_at(cur.e + lane64);
    int32_t parent = parent_at(edge);
    RowPart<T> key, val, key_next, val_next;
    const auto fetch = [&](int64_t r) {
        key_next.load(static_cast<const T *>(a.k) + r * stride + (int64_t)j * a.dim, at);
        if (!SHARED) val_next.load(static_cast<const T *>(a.v) + r * stride + (int64_t)j * a.dim, at);
    };
    fetch(cur.p);
    float sum[2 * E];                               // g_k, g_v
    while (have) {
        if (cur.first) {
            key = key_next;
            key.own(at);
            if (!SHARED) { val = val_next; val.own(at); }
#pragma unroll
            for (int i = 0; i < 2 * E; ++i) sum[i] = 0.f;
        }
        const int32_t parents = lane64 < cur.n ? checked(edge, parent) : -1;
        have = walk.next();
        if (have) {
            edge = edge_at(walk.u.e + lane64);
            if (walk.u.first) fetch(walk.u.p);
        }
        for (uint32_t b = 0; b < cur.n; b += W * U) {
            int32_t p[U];
#pragma unroll
            for (int u = 0; u < U; ++u) p[u] = __shfl(parents, b + u * W + group, 64);
            for (int h0 = j * share; h0 < (j + 1) * share; h0 += G) {
                RowPart<T> qr[U][G], gr[U][G];
                float lse2[U][G], delta[U][G];
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int g = 0; g < G; ++g) {   // (what is no neighbor, and heads past the last one, read another and forget it)
                        const int64_t of = (int64_t)max(p[u], 0) * a.heads + min(h0 + g, (j + 1) * share - 1);
                        qr[u][g].load(Q + of * a.dim, at);
                        gr[u][g].load(GO + of * a.dim, at);
                        lse2[u][g] = a.lse[of] * gs::kLog2e;
                        delta[u][g] = a.delta[of];
                    }
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const bool none = p[u] < 0 || h0 + g >= (j + 1) * share || lse2[u][g] == -INFINITY;
                        qr[u][g].zero_if(none);
                        gr[u][g].zero_if(none);
                        lse2[u][g] = none ? -INFINITY : lse2[u][g];
                        delta[u][g] = none ? 0.f : delta[u][g];
                    }
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const float s = gs::lanes_sum<L>(gs::dot(key, qr[u][g])) * scale2;
                        const float dp = gs::lanes_sum<L>(gs::dot(SHARED ? key : val, gr[u][g]));
                        const float pr = lse2[u][g] != -INFINITY ? gs::fast_exp2(s - lse2[u][g]) : 0.f;
                        const float ds = pr * (dp - delta[u][g]) * a.scale;
#pragma unroll
                        for (int i = 0; i < E; ++i) { sum[i] += ds * qr[u][g].at(i); sum[E + i] += pr * gr[u][g].at(i); }
                    }
            }
        }
        if (have) parent = parent_at(edge);
        if (cur.last) {
            if (SHARED)
#pragma unroll
                for (int i = 0; i < E; ++i) sum[i] += sum[E + i];
            gs::Scatter<2 * E, L> mine;
            mine.run(sum, lane64);
            constexpr int N = gs::Scatter<2 * E, L>::kKept, S = N < E ? N : E;
#pragma unroll
            for (int x = 0; x < N; x += S) {
                const int set = (mine.start + x) / E, start = (mine.start + x) % E;
                T *out = static_cast<T *>(set ? a.g_v : a.g_k);
                if (!out || mine.dup) continue;
                if (cur.complete) gs::store_part<S>(out + cur.p * stride + (int64_t)j * a.dim, at, start, sum + x);
                else gs::store_part<S>(a.piece + (((size_t)cur.place * a.kv_heads + j) * 2 + set) * a.dim, at, start, sum + x);
            }
        }
        cur = walk.u;
    }
}

// The rows' walk where the lists are short on the mean: every L lanes take `chunk` entries of their own by the same rule
// (lists that begin there, and parts of longer ones).  Which row an entry belongs to is what child_ids say, so nothing is
// searched, and every entry's loads (the row's key and value again and again, they are near) are known before its turn.
template <class T, int L, int G, bool SHARED>
__global__ __launch_bounds__(gs::kAttnThreads)
void attn_bwd_rows_short_kernel(BwdArgs a) {
    constexpr int E = gs::Pack<T>::E, W = 64 / L;
    constexpr int U = L == 2 ? 1 : G == 1 && E == 4 ? 4 : G <= 2 ? 2 : 1;             // (divides L)
    const int lane64 = threadIdx.x & 63, lane = lane64 & (L - 1), group0 = lane64 & ~(L - 1);
    const int share = a.heads / a.kv_heads, j = blockIdx.y;
    Neighbors lists = a.nb;
    lists.indptr = a.inv_indptr;
    lists.n_edges = a.n_inv;
    const T *Q = static_cast<const T *>(a.q), *GO = static_cast<const T *>(a.g_out);
    const T *K = static_cast<const T *>(a.k) + (int64_t)j * a.dim, *V = SHARED ? nullptr : static_cast<const T *>(a.v) + (int64_t)j * a.dim;
    const int64_t stride = (int64_t)a.kv_heads * a.dim;
    const float scale2 = a.scale * gs::kLog2e;
    const gs::Place<T, L> at(lane, a.dim);
    const uint32_t chunk = (uint32_t)a.chunk, most = 4 * chunk, run = gs::this_wave() * W + lane64 / L;
    const uint32_t e0 = (uint32_t)min((uint64_t)run * chunk, (uint64_t)a.n_inv), e1 = min(e0 + chunk, a.n_inv);

    struct Entry { int32_t row, parent; uint32_t begin, end; };        // what a lane knows of entry e
    const auto entry_at = [&](uint32_t e) {
        Entry t;
        const uint32_t edge = (uint32_t)a.inv_edges[min(e, a.n_inv - 1)];
        const int32_t id = a.nb.ids[min(edge, a.nb.n_edges - 1)];
        const int32_t p = a.nb.indptr ? a.edge_parent[min(edge, a.nb.n_edges - 1)] : (int32_t)(edge / a.nb.n_child);
        t.row = edge < a.nb.n_edges ? a.nb.row_of(id) : -1;
        t.parent = t.row >= 0 && (uint64_t)(int64_t)p < (uint64_t)a.nb.n_parents ? p : -1;
        lists.range(max(t.row, 0), t.begin, t.end);
        if (t.row < 0 || e < t.begin || e >= t.end) { t.row = t.parent = -1; t.begin = e; t.end = e + 1; }    // (in no row's list)
        return t;
    };
    // from the end of a list that another has begun and keeps, to the end of the last one that begins here
    Entry t = entry_at(e0 + lane);
    uint32_t start = e0, stop = e0;
    {
        const uint32_t f_begin = __shfl(t.begin, group0, 64), f_end = __shfl(t.end, group0, 64);
        const int back = (int)min(chunk, (uint32_t)L) - 1;
        Entry l;
        l.begin = __shfl(t.begin, group0 + back, 64);
        l.end = __shfl(t.end, group0 + back, 64);
        if (chunk > L || e1 - e0 < chunk) l = entry_at(e1 - 1);
        if (e0 < e1) {
            if (f_begin < e0 && f_end - f_begin <= most) start = f_end;
            stop = l.end - l.begin > most ? e1 : min(l.end, e1 + most);
        }
    }
    float sum[2 * E];
#pragma unroll
    for (int i = 0; i < 2 * E; ++i) sum[i] = 0.f;
    for (uint32_t at_e = e0; __any(at_e < stop && start < stop); at_e += L) {
        const uint32_t mine = at_e + lane;
        if (at_e != e0) t = entry_at(mine);
        const bool cut = t.end - t.begin > most, in = mine >= start && mine < stop;
        // 1: the list's last entry here, 2: a piece of it, 4: the piece's place
        const int flags = in && t.row >= 0 && mine + 1 == (cut ? min(t.end, e1) : t.end) ? 1 | (cut ? 2 : 0) | (t.begin > e0 ? 4 : 0) : 0;
        const int32_t parent = in ? t.parent : -1;
        const unsigned long long some = __ballot(parent >= 0 || flags);
        for (int x = 0; x < L; x += U) {
            unsigned long long turn = 0;                               // the entries of this turn, in all groups
#pragma unroll
            for (int g = 0; g < 64; g += L) turn |= ((1ull << U) - 1) << (g + x);
            if (!(some & turn)) continue;
            int32_t row[U], p[U];
            int fl[U];
            RowPart<T> key[U], val[U];
            float c[U][2 * E];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                row[u] = __shfl(t.row, group0 + x + u, 64);
                p[u] = __shfl(parent, group0 + x + u, 64);
                fl[u] = __shfl(flags, group0 + x + u, 64);
                const int64_t to = (int64_t)max(row[u], 0) * stride;
                key[u].load(K + to, at);
                if (!SHARED) val[u].load(V + to, at);
#pragma unroll
                for (int i = 0; i < 2 * E; ++i) c[u][i] = 0.f;
            }
            for (int h0 = j * share; h0 < (j + 1) * share; h0 += G) {
                RowPart<T> qr[U][G], gr[U][G];
                float lse2[U][G], delta[U][G];
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int g = 0; g < G; ++g) {   // (what is no neighbor, and heads past the last one, read another and forget it)
                        const int64_t of = (int64_t)max(p[u], 0) * a.heads + min(h0 + g, (j + 1) * share - 1);
                        qr[u][g].load(Q + of * a.dim, at);
                        gr[u][g].load(GO + of * a.dim, at);
                        lse2[u][g] = a.lse[of] * gs::kLog2e;
                        delta[u][g] = a.delta[of];
                    }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    RowPart<T> own_key = key[u], own_val = val[u];
                    own_key.own(at);
                    if (!SHARED) own_val.own(at);
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const bool none = p[u] < 0 || h0 + g >= (j + 1) * share || lse2[u][g] == -INFINITY;
                        qr[u][g].zero_if(none);
                        gr[u][g].zero_if(none);
                        const float s = gs::lanes_sum<L>(gs::dot(own_key, qr[u][g])) * scale2;
                        const float dp = gs::lanes_sum<L>(gs::dot(SHARED ? own_key : own_val, gr[u][g]));
                        const float pr = none ? 0.f : gs::fast_exp2(s - lse2[u][g]);
                        const float ds = none ? 0.f : pr * (dp - delta[u][g]) * a.scale;
#pragma unroll
                        for (int i = 0; i < E; ++i) { c[u][i] += ds * qr[u][g].at(i); c[u][E + i] += pr * gr[u][g].at(i); }
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int i = 0; i < 2 * E; ++i) sum[i] += c[u][i];
                if (!(fl[u] & 1)) continue;
                if (SHARED)
#pragma unroll
                    for (int i = 0; i < E; ++i) sum[i] += sum[E + i];
                const int64_t to = (int64_t)row[u] * stride + (int64_t)j * a.dim;
                if (fl[u] & 2) {
                    float *piece = a.piece + ((size_t)(run * 2 + (fl[u] >> 2)) * a.kv_heads + j) * 2 * a.dim;
                    gs::store_part<E>(piece, at, 0, sum);
                    if (!SHARED) gs::store_part<E>(piece + a.dim, at, 0, sum + E);
                } else {
                    if (a.g_k) gs::store_part<E>(static_cast<T *>(a.g_k) + to, at, 0, sum);
                    if (!SHARED && a.g_v) gs::store_part<E>(static_cast<T *>(a.g_v) + to, at, 0, sum + E);
                }
#pragma unroll
                for (int i = 0; i < 2 * E; ++i) sum[i] = 0.f;
            }
        }
    }
}

// Adds the pieces of the lists that were cut, and writes zeros for empty ones.  `sets` vectors of dim floats per head: the
// parents' walk has one per (list, head), the rows' two per (list, key head).  Few pieces: one wave alone.
constexpr uint32_t kFewPieces = 16;

template <class T>
__global__ __launch_bounds__(gs::kJoinWaves * 64)
void attn_bwd_join_kernel(Neighbors seg, const float *piece, int per_slot, int sets, int dim, uint32_t chunk, T *out0, T *out1) {
    constexpr int N = gs::kJoinWaves;
    __shared__ float part[N][64];
    __shared__ gs::LongLists longs;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, y = blockIdx.y / sets, set = blockIdx.y % sets;
    T *out = set ? out1 : out0;
    if (!out) return;
    const gs::JoinLanes l(lane, dim, blockIdx.z);
    const int64_t mine = gs::join_list(wave, lane);
    uint32_t b = 0, e = 0;
    if (mine < seg.n_parents) seg.range(mine, b, e);
    const bool mine_todo = mine < seg.n_parents && gs::needs_join(b, e, chunk);
    const bool many = mine_todo && e > b && (e - 1) / chunk - b / chunk >= kFewPieces;
    unsigned long long few = __ballot(mine_todo && !many);
    const auto add = [&](uint32_t sb, uint32_t se, uint32_t first, uint32_t step) {
        const uint32_t n = (se - 1) / chunk - sb / chunk + 1;
        float acc = 0.f;
        for (uint32_t i = first; i < n; i += gs::kJoinFlight * step) {
            float x[gs::kJoinFlight];
#pragma unroll
            for (int k = 0; k < gs::kJoinFlight; ++k)
                x[k] = piece[((gs::piece_place(sb, chunk, min(i + k * step, n - 1)) * per_slot + y) * sets + set) * dim + l.d];
#pragma unroll
            for (int k = 0; k < gs::kJoinFlight; ++k) acc += i + k * step < n ? x[k] : 0.f;
        }
        for (int o = l.width; o < 64; o *= 2) acc += __shfl_xor(acc, o, 64);
        return acc;
    };
    const auto write = [&](int64_t p, float v) {
        if (l.sub == 0 && l.in) out[(p * per_slot + y) * dim + l.d] = (T)v;
    };
    for (; few; few &= few - 1) {
        const int src = __builtin_ctzll(few);
        const uint32_t sb = __shfl(b, src, 64), se = __shfl(e, src, 64);
        write(gs::join_list(wave, src), se > sb ? add(sb, se, l.sub, l.subs) : 0.f);
    }
    if (!__syncthreads_or(many)) return;
    if (threadIdx.x == 0) longs.n = 0;
    __syncthreads();
    if (many) {
        const int i = atomicAdd(&longs.n, 1);
        longs.slot[i] = threadIdx.x; longs.b[i] = b; longs.e[i] = e;
    }
    __syncthreads();
    for (int i = 0; i < longs.n; ++i) {
        const float own = add(longs.b[i], longs.e[i], wave * l.subs + l.sub, N * l.subs);
        __syncthreads();                            // the last list's parts are read
        part[wave][lane] = own;
        __syncthreads();
        if (wave) continue;
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < N; ++k) sum += part[k][lane];
        write(gs::join_list(longs.slot[i] >> 6, longs.slot[i] & 63), sum);
    }
}

// Adds the head groups' parts of dense rows' gradients.
template <class T>
__global__ __launch_bounds__(256)
void attn_bwd_dense_kernel(BwdArgs a) {
    const int64_t n = a.nb.n_rows * a.kv_heads * a.dim;
    const int64_t first = a.nb.indptr ? a.nb.indptr[0] : 0, last = a.nb.indptr ? a.nb.indptr[a.nb.n_parents] : (int64_t)a.nb.n_edges;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / ((int64_t)a.kv_heads * a.dim), vec = i / a.dim;
        if (row < first || row >= last) continue;   // belongs to no parent: left as it is
        float k = 0.f, v = 0.f;
        for (int p = 0; p < a.parts; ++p) {
            const float *part = a.dense_part + ((int64_t)p * n + vec * a.dim) * 2 + i % a.dim;
            k += part[0];
            if (a.v) v += part[a.dim];
        }
        if (a.g_k) static_cast<T *>(a.g_k)[i] = (T)k;
        if (a.g_v) static_cast<T *>(a.g_v)[i] = (T)v;
    }
}

template <class T, int L, bool SHARED>
void launch_parents(const BwdArgs &a, const gs::Deal &d, hipStream_t stream) {
    const int g = gs::heads_per_wave(a.heads / a.kv_heads);
    const dim3 grid((unsigned)((d.waves + gs::kAttnThreads / 64 - 1) / (gs::kAttnThreads / 64)), (unsigned)(a.kv_heads * a.parts));
    if (d.is_short) {
        if (g == 1) attn_bwd_short_kernel<T, L, 1, SHARED><<<grid, gs::kAttnThreads, 0, stream>>>(a);
        else if (g == 2) attn_bwd_short_kernel<T, L, 2, SHARED><<<grid, gs::kAttnThreads, 0, stream>>>(a);
        else attn_bwd_short_kernel<T, L, 4, SHARED><<<grid, gs::kAttnThreads, 0, stream>>>(a);
    } else if (g == 1) attn_bwd_parents_kernel<T, L, 1, SHARED><<<grid, gs::kAttnThreads, 0, stream>>>(a);
    else if (g == 2) attn_bwd_parents_kernel<T, L, 2, SHARED><<<grid, gs::kAttnThreads, 0, stream>>>(a);
    else attn_bwd_parents_kernel<T, L, 4, SHARED><<<grid, gs::kAttnThreads, 0, stream>>>(a);
}

template <class T, int L, bool SHARED>
void launch_rows(const BwdArgs &a, const gs::Deal &d, hipStream_t stream) {
    const int g = gs::heads_per_wave(a.heads / a.kv_heads);
    const int64_t waves = d.is_short ? (d.waves + 64 / L - 1) / (64 / L) : d.waves;
    const dim3 grid((unsigned)((waves + gs::kAttnThreads / 64 - 1) / (gs::kAttnThreads / 64)), (unsigned)a.kv_heads);
    if (d.is_short) {
        if (g == 1) attn_bwd_rows_short_kernel<T, L, 1, SHARED><<<grid, gs::kAttnThreads, 0, stream>>>(a);
        else if (g == 2) attn_bwd_rows_short_kernel<T, L, 2, SHARED><<<grid, gs::kAttnThreads, 0, stream>>>(a);
        else attn_bwd_rows_short_kernel<T, L, 4, SHARED><<<grid, gs::kAttnThreads, 0, stream>>>(a);
    } else if (g == 1) attn_bwd_rows_kernel<T, L, 1, SHARED><<<grid, gs::kAttnThreads, 0, stream>>>(a);
    else if (g == 2) attn_bwd_rows_kernel<T, L, 2, SHARED><<<grid, gs::kAttnThreads, 0, stream>>>(a);
    else attn_bwd_rows_kernel<T, L, 4, SHARED><<<grid, gs::kAttnThreads, 0, stream>>>(a);
}

struct Plan {
    gs::Deal parents, rows;
    int parts;
    size_t off_parent, off_dense, off_piece, total;
};

// Rows whose lists are this long on the mean, or shorter, are taken by L lanes a run of entries, which pays the longer the fewer
// heads a wave has at once (the backward pass without g_q, rows of 64, a list per wave against this: 10 000 fp32 rows, one head,
// mean 4 26 us and 22, 8 28 and 32; 100 000 bf16 rows, one head, mean 8 159 us and 109, 12 176 and 160; two heads, 4 142 us and 93,
// 8 165 and 165; four heads, 4 160 us and 153; 10 000 bf16 rows, four heads, 4 35 us and 37, 6 37 and 45).
constexpr int64_t short_mean(int heads_at_once) { return heads_at_once == 1 ? 8 : heads_at_once == 2 ? 6 : 4; }

gs::Deal deal_rows(int64_t n_rows, int64_t n_inv, int lanes, int heads_at_once) {
    static const int64_t ragged = 0;                // any address: the rows' lists are ragged
    gs::Deal d = gs::deal_edges(&ragged, n_rows, 0, n_inv, lanes);
    d.is_short = n_inv && n_inv <= short_mean(heads_at_once) * n_rows;
    if (d.is_short) {
        // runs for two waves per SIMD, of 2 to 16 entries (7600 entries of 16 fp32: 22 us with 8, 9 with 2; 96000 of 64: 19 us with 8,
        // 16 with 16; 360 000 of 256 bf16: 104 and 87), 131072 runs at most (each may leave two pieces)
        d.chunk = n_inv / (2048 * (64 / lanes));
        d.chunk = d.chunk < 2 ? 2 : d.chunk > 16 ? 16 : d.chunk;
        if (d.chunk < (n_inv + 131071) / 131072) d.chunk = (n_inv + 131071) / 131072;
        d.waves = (n_inv + d.chunk - 1) / d.chunk;  // runs, here
    }
    return d;
}

// The pieces of both walks share a region: the second walk starts when the first one's pieces are joined.
Plan make_plan(const gs_neighbors *nb, int heads, int kv_heads, int dim, int dtype, int64_t n_inv) {
    Plan p;
    const int lanes = gs::lanes_for(dim, gs::dtype_size(dtype)), share = heads / kv_heads;
    p.parts = (share + gs::heads_per_wave(share) - 1) / gs::heads_per_wave(share);
    p.parents = gs::deal_edges(nb, lanes);
    p.rows = deal_rows(nb->n_rows, nb->ids && nb->n_rows && nb->n_parents ? n_inv : 0, lanes, gs::heads_per_wave(share));
    size_t off = gs::align256((size_t)nb->n_parents * heads * sizeof(float));        // delta
    p.off_parent = off;
    if (nb->indptr && nb->ids) off += gs::align256((size_t)nb->n_edges * sizeof(int32_t));
    p.off_dense = off;
    if (!nb->ids && p.parts > 1) off += gs::align256((size_t)p.parts * nb->n_rows * kv_heads * 2 * dim * sizeof(float));
    p.off_piece = off;
    size_t piece = 0;
    if (p.parents.pieces) piece = (size_t)p.parents.waves * 2 * heads * dim * sizeof(float);
    const size_t r = (size_t)p.rows.waves * 4 * kv_heads * dim * sizeof(float);
    p.total = off + (r > piece ? r : piece);
    return p;
}

template <class T>
int run_bwd(BwdArgs a, const Plan &p, int lanes, hipStream_t stream) {
    a.chunk = (int)p.parents.chunk;
    if (p.parents.waves) {
        GS_BY_LANES(launch_parents, a.v == nullptr, a, p.parents, stream);
        if (int rc = gs::check_launch("gs_neighbor_attention_bwd (parents)")) return rc;
    }
    if (a.g_q && a.nb.n_parents && p.parents.pieces) {
        attn_bwd_join_kernel<T><<<gs::join_grid(a.nb.n_parents, a.heads, a.dim), gs::kJoinWaves * 64, 0, stream>>>(
            a.nb, a.piece, a.heads, 1, a.dim, a.chunk, static_cast<T *>(a.g_q), (T *)nullptr);
        if (int rc = gs::check_launch("gs_neighbor_attention_bwd (parents' join)")) return rc;
    }
    if (!a.g_k && !a.g_v) return GS_OK;
    if (!a.nb.ids) {
        if (a.parts == 1 || !a.nb.n_rows || !p.parents.waves) return GS_OK;
        const int64_t blocks = (a.nb.n_rows * a.kv_heads * a.dim + 255) / 256;
        attn_bwd_dense_kernel<T><<<dim3((unsigned)(blocks < 1 << 20 ? blocks : 1 << 20)), 256, 0, stream>>>(a);
        return gs::check_launch("gs_neighbor_attention_bwd (dense rows)");
    }
    a.chunk = (int)p.rows.chunk;
    if (p.rows.waves) {
        GS_BY_LANES(launch_rows, a.v == nullptr, a, p.rows, stream);
        if (int rc = gs::check_launch("gs_neighbor_attention_bwd (rows)")) return rc;
    }
    if (!a.nb.n_rows) return GS_OK;
    Neighbors rows = a.nb;
    rows.indptr = a.nb.n_parents ? a.inv_indptr : nullptr;             // (without parents every row's list is empty)
    rows.n_child = 0;
    rows.n_parents = a.nb.n_rows;
    rows.n_edges = a.n_inv;
    attn_bwd_join_kernel<T><<<gs::join_grid(a.nb.n_rows, a.kv_heads * 2, a.dim), gs::kJoinWaves * 64, 0, stream>>>(
        rows, a.piece, a.kv_heads, 2, a.dim, a.chunk, static_cast<T *>(a.g_k), static_cast<T *>(a.g_v));
    return gs::check_launch("gs_neighbor_attention_bwd (rows' join)");
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
    a.nb = gs::device_neighbors(nb);
    a.q = q; a.k = k; a.v = v; a.out = out; a.g_out = g_out; a.lse = lse;
    a.g_q = g_q; a.g_k = g_k; a.g_v = g_v;
    char *ws = static_cast<char *>(workspace);
    a.delta = reinterpret_cast<float *>(ws);
    a.edge_parent = nb->indptr && nb->ids ? reinterpret_cast<int32_t *>(ws + p.off_parent) : nullptr;
    a.dense_part = reinterpret_cast<float *>(ws + p.off_dense);
    a.piece = reinterpret_cast<float *>(ws + p.off_piece);
    a.inv_indptr = nb->ids ? inv_indptr : nullptr;
    a.inv_edges = nb->ids ? inv_edges : nullptr;
    a.n_inv = (uint32_t)(nb->ids ? n_inv : 0);
    a.scale = scale;
    a.heads = heads; a.kv_heads = kv_heads; a.dim = dim; a.chunk = 0; a.parts = p.parts;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == GS_F32) return run_bwd<float>(a, p, lanes, s);
    if (dtype == GS_BF16) return run_bwd<__bf16>(a, p, lanes, s);
    return run_bwd<_Float16>(a, p, lanes, s);
}
