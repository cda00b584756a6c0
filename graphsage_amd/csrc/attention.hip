// Attention of every parent over its neighbors, forward (the dealing of edges: attention.h).
//
// An edge costs one row of dim elements (two with separate values) and, per head, dim multiply-adds for the score and as
// many for the sum.  One head is bound by the row gathers: 1 024 000 rows of 64 fp32 in lists of 10 take 37 us, 7.0 TB/s out of
// the caches (their mean, which gathers the same rows, 34 us).  Four heads a key head are bound by the vector ALU: 2M ragged edges of
// eight heads of 64 bf16, 4M row pairs, take 308 us, 94% of them busy with 140M instructions, a part of which repeats in the lanes of a
// row group (the softmax step of a score) or ends a list.  Scores are kept in units of log 2 (scale * log2 e goes into the query), so
// an exponential is one instruction.
#include "attention.h"

namespace gs {

int check_neighbors(const char *what, const gs_neighbors *nb, int heads, int kv_heads, int dim, int dtype) {
    if (!nb) return fail(GS_EINVAL, "%s: null pointer argument", what);
    if (!dtype_size(dtype)) return fail(GS_EINVAL, "%s: dtype %d", what, dtype);
    if (nb->n_parents < 0 || nb->n_edges < 0 || nb->n_rows < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || dim < 1)
        return fail(GS_EINVAL, "%s: parents=%lld edges=%lld rows=%lld heads=%d kv_heads=%d dim=%d", what,
                    (long long)nb->n_parents, (long long)nb->n_edges, (long long)nb->n_rows, heads, kv_heads, dim);
    if (dim > 256 || heads > 1024) return fail(GS_ELIMIT, "%s: dim=%d (at most 256), heads=%d (at most 1024)", what, dim, heads);
    if (nb->n_edges >= (int64_t)1 << 31 || nb->n_parents >= (int64_t)1 << 31 || nb->n_rows >= (int64_t)1 << 31)
        return fail(GS_ELIMIT, "%s: %lld edges, %lld parents, %lld rows (less than 2^31)", what, (long long)nb->n_edges,
                    (long long)nb->n_parents, (long long)nb->n_rows);
    if (!nb->indptr && (nb->n_child < 0 || nb->n_child >= (int64_t)1 << 31 || nb->n_parents * nb->n_child != nb->n_edges))
        return fail(GS_EINVAL, "%s: %lld edges for %lld parents of %lld", what, (long long)nb->n_edges, (long long)nb->n_parents,
                    (long long)nb->n_child);
    return GS_OK;
}

}  // namespace gs

namespace {

using gs::Neighbors;
using gs::RowPart;

struct FwdArgs {
    Neighbors nb;
    const void *q, *k, *v;
    void *out;
    float *lse;
    float2 *piece_ms;                               // [waves][2][heads]: maximum (log 2), sum
    float *piece_acc;                               // [waves][2][heads][dim]
    float scale2;                                   // scale * log2 e
    int heads, kv_heads, dim, chunk, parts;         // parts: head groups per key head
};

// What the lanes of a row group keep of a list: the queries of G heads, their running maxima (units of log 2), sums and
// weighted rows.
template <class T, int L, int G, bool SHARED> struct FwdState {
    static constexpr int E = gs::Pack<T>::E;
    RowPart<T> q[G];
    float acc[G * E], m[G], s[G];

    __device__ __forceinline__ void begin(const RowPart<T> *queries, const gs::Place<T, L> &at) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            m[g] = -INFINITY;
            s[g] = 0.f;
            q[g] = queries[g];
            q[g].own(at);
#pragma unroll
            for (int i = 0; i < E; ++i) acc[g * E + i] = 0.f;
        }
    }
    // U rows at once; a negative one is none
    template <int U>
    __device__ __forceinline__ void rows(const int32_t (&row)[U], bool gaps, const T *K, const T *V, int64_t stride, float scale2,
                                         const gs::Place<T, L> &at) {
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
        for (int g = 0; g < G; ++g) {
            float sc[U], top = m[g];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float d = gs::lanes_sum<L>(gs::dot(q[g], kr[u])) * scale2;
                sc[u] = row[u] >= 0 ? d : -INFINITY;
                top = fmaxf(top, sc[u]);
            }
            const float ref = top == -INFINITY ? 0.f : top;            // nothing yet: exponentials of -inf, zeros
            const float keep = gs::fast_exp2(m[g] - ref);
            m[g] = top;
            s[g] *= keep;
#pragma unroll
            for (int i = 0; i < E; ++i) acc[g * E + i] *= keep;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float pr = gs::fast_exp2(sc[u] - ref);
                s[g] += pr;
#pragma unroll
                for (int i = 0; i < E; ++i) acc[g * E + i] += pr * (SHARED ? kr[u].at(i) : vr[u].at(i));
            }
        }
    }
};

// 1 / s; nothing to divide by: zeros; a NaN stays one
__device__ __forceinline__ float inverse_of(float s) { return s > 0.f ? __builtin_amdgcn_rcpf(s) : s == 0.f ? 0.f : s; }

// Two rows at a time for four heads, which have enough to do (2M edges of eight heads of 64 bf16, two a key head: 313 us, 342 with four
// rows, of which a list's end leaves more unused).
template <class T, int L, int G, bool SHARED>
__global__ __launch_bounds__(gs::kAttnThreads)
void attn_fwd_kernel(FwdArgs a) {
    constexpr int E = gs::Pack<T>::E, W = 64 / L, U = L == 2 || G == 4 ? 2 : gs::kAttnRows;
    const int lane64 = threadIdx.x & 63, lane = lane64 & (L - 1), group = lane64 / L;
    const int share = a.heads / a.kv_heads;
    const int j = blockIdx.y / a.parts, h0 = j * share + (blockIdx.y % a.parts) * G;
    const int n_heads = min(G, (j + 1) * share - h0);
    const T *Q = static_cast<const T *>(a.q);
    const T *K = static_cast<const T *>(a.k) + (int64_t)j * a.dim, *V = SHARED ? nullptr : static_cast<const T *>(a.v) + (int64_t)j * a.dim;
    const int64_t stride = (int64_t)a.kv_heads * a.dim;
    const gs::Place<T, L> at(lane, a.dim);

    gs::Walk walk(a.nb, gs::this_wave(), a.chunk);
    bool have = walk.next();
    if (!have) return;
    gs::Unit cur = walk.u;
    int32_t entry = a.nb.entry(cur.e + lane64);
    RowPart<T> q_next[G];
#pragma unroll
    for (int g = 0; g < G; ++g)                     // (heads past the last one repeat it)
        q_next[g].load(Q + (cur.p * a.heads + h0 + min(g, n_heads - 1)) * a.dim, at);
    FwdState<T, L, G, SHARED> st;
    while (have) {
        if (cur.first) st.begin(q_next, at);
        const int32_t rows = lane64 < cur.n ? a.nb.row_of(entry) : -1;
        const bool gaps = __any(rows < 0 && lane64 < cur.n) || cur.n % (W * U);
        // the next unit's entries and queries are on their way while this one's rows are used
        have = walk.next();
        if (have) {
            entry = a.nb.entry(walk.u.e + lane64);
            if (walk.u.first)
#pragma unroll
                for (int g = 0; g < G; ++g) q_next[g].load(Q + (walk.u.p * a.heads + h0 + min(g, n_heads - 1)) * a.dim, at);
        }
        for (uint32_t b = 0; b < cur.n; b += W * U) {
            int32_t row[U];
#pragma unroll
            for (int u = 0; u < U; ++u) row[u] = __shfl(rows, b + u * W + group, 64);     // (-1 behind the last entry)
            st.template rows<U>(row, gaps, K, V, stride, a.scale2, at);
        }
        if (cur.last) {
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const float top = gs::groups_max<L>(st.m[g]), ref = top == -INFINITY ? 0.f : top;
                const float keep = gs::fast_exp2(st.m[g] - ref);
                st.m[g] = top;
                st.s[g] = gs::groups_sum<L>(st.s[g] * keep);
                const float f = cur.complete ? keep * inverse_of(st.s[g]) : keep;
#pragma unroll
                for (int i = 0; i < E; ++i) st.acc[g * E + i] *= f;
            }
            gs::Scatter<G * E, L> mine;
            mine.run(st.acc, lane64);
            constexpr int N = gs::Scatter<G * E, L>::kKept, S = N < E ? N : E;
#pragma unroll
            for (int x = 0; x < N; x += S) {
                const int g = (mine.start + x) / E, start = (mine.start + x) % E;
                if (g >= n_heads || mine.dup) continue;
                const int64_t o = cur.p * a.heads + h0 + g;
                if (cur.complete) gs::store_part<S>(static_cast<T *>(a.out) + o * a.dim, at, start, st.acc + x);
                else gs::store_part<S>(a.piece_acc + ((size_t)cur.place * a.heads + h0 + g) * a.dim, at, start, st.acc + x);
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
                if (lane64 != 0 || g >= n_heads) continue;
                if (cur.complete) a.lse[cur.p * a.heads + h0 + g] = (st.m[g] + gs::fast_log2(st.s[g])) * gs::kLn2;
                else a.piece_ms[(size_t)cur.place * a.heads + h0 + g] = make_float2(st.m[g], st.s[g]);
            }
        }
        cur = walk.u;
    }
}

// Short lists of one length: L lanes take a list each.  Entries come L at a time, one a lane, one load ahead.
template <class T, int L, int G, bool SHARED>
__global__ __launch_bounds__(gs::kAttnThreads)
void attn_fwd_short_kernel(FwdArgs a) {
    constexpr int E = gs::Pack<T>::E, W = 64 / L, U = L == 2 ? 2 : gs::kAttnRows;
    const int lane64 = threadIdx.x & 63, lane = lane64 & (L - 1), group0 = lane64 & ~(L - 1);
    const int share = a.heads / a.kv_heads;
    const int j = blockIdx.y / a.parts, h0 = j * share + (blockIdx.y % a.parts) * G;
    const int n_heads = min(G, (j + 1) * share - h0);
    const T *Q = static_cast<const T *>(a.q);
    const T *K = static_cast<const T *>(a.k) + (int64_t)j * a.dim, *V = SHARED ? nullptr : static_cast<const T *>(a.v) + (int64_t)j * a.dim;
    const int64_t stride = (int64_t)a.kv_heads * a.dim;
    const gs::Place<T, L> at(lane, a.dim);
    const uint32_t n = a.nb.n_child, n_lists = (uint32_t)a.nb.n_parents, waves = gridDim.x * (gs::kAttnThreads / 64);

    uint32_t base = gs::this_wave() * W;            // of the wave; lists past the last one repeat it
    if (base >= n_lists) return;
    uint32_t p = min(base + lane64 / L, n_lists - 1);
    int32_t entry = a.nb.entry(p * n + lane);
    RowPart<T> q_next[G];
#pragma unroll
    for (int g = 0; g < G; ++g) q_next[g].load(Q + ((int64_t)p * a.heads + h0 + min(g, n_heads - 1)) * a.dim, at);
    FwdState<T, L, G, SHARED> st;
    for (;;) {
        st.begin(q_next, at);
        const uint32_t cur = p;
        const bool mine = base + lane64 / L < n_lists;
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
#pragma unroll
                for (int g = 0; g < G; ++g) q_next[g].load(Q + ((int64_t)p * a.heads + h0 + min(g, n_heads - 1)) * a.dim, at);
            }
            for (uint32_t b = 0; b < here; b += U) {
                int32_t row[U];
#pragma unroll
                for (int u = 0; u < U; ++u) row[u] = __shfl(rows, group0 + b + u, 64);
                st.template rows<U>(row, gaps, K, V, stride, a.scale2, at);
            }
        }
        if (mine)
#pragma unroll
            for (int g = 0; g < G; ++g) {
                if (g >= n_heads) continue;
                const float f = inverse_of(st.s[g]);
#pragma unroll
                for (int i = 0; i < E; ++i) st.acc[g * E + i] *= f;
                const int64_t o = (int64_t)cur * a.heads + h0 + g;
                gs::store_part<E>(static_cast<T *>(a.out) + o * a.dim, at, 0, st.acc + g * E);
                if (lane == 0) a.lse[o] = (st.m[g] + gs::fast_log2(st.s[g])) * gs::kLn2;
            }
        if (!more) return;
    }
}

// Joins the pieces of the lists that were cut and writes the parents without edges, for one head and 64 elements.  A wave
// joins a list of a few pieces by itself; of a long one every wave takes its share (one list of 20000 rows of 64, four heads: 17 us
// with the walk, 38 with one wave; 2000 lists of 2000, 9 pieces each: 133 us, 143 with every wave).
constexpr uint32_t kFewPieces = 16;

struct Joined {
    float m, s, acc;
    __device__ __forceinline__ void add(float mo, float so, float ao) {
        const float top = fmaxf(m, mo), ref = top == -INFINITY ? 0.f : top;
        const float ka = gs::fast_exp2(m - ref), kb = gs::fast_exp2(mo - ref);
        m = top;
        s = s * ka + so * kb;
        acc = acc * ka + ao * kb;
    }
};

// Pieces first, first + step, ... of list [b, e); then joined across the pieces a wave holds at a time.
__device__ __forceinline__ Joined join_pieces(const FwdArgs &a, uint32_t b, uint32_t e, uint32_t first, uint32_t step, int h, const gs::JoinLanes &l) {
    const uint32_t n = (e - 1) / a.chunk - b / a.chunk + 1;
    Joined j{-INFINITY, 0.f, 0.f};
    for (uint32_t i = first; i < n; i += gs::kJoinFlight * step) {
        float2 ms[gs::kJoinFlight];
        float x[gs::kJoinFlight];
#pragma unroll
        for (int k = 0; k < gs::kJoinFlight; ++k) {
            const size_t at = gs::piece_place(b, a.chunk, min(i + k * step, n - 1)) * a.heads + h;
            ms[k] = a.piece_ms[at];
            x[k] = a.piece_acc[at * a.dim + l.d];
        }
        float top = j.m;
#pragma unroll
        for (int k = 0; k < gs::kJoinFlight; ++k) {
            if (i + k * step >= n) { ms[k] = make_float2(-INFINITY, 0.f); x[k] = 0.f; }
            top = fmaxf(top, ms[k].x);
        }
        const float ref = top == -INFINITY ? 0.f : top, ko = gs::fast_exp2(j.m - ref);
        j.m = top;
        j.s *= ko;
        j.acc *= ko;
#pragma unroll
        for (int k = 0; k < gs::kJoinFlight; ++k) {
            const float kn = gs::fast_exp2(ms[k].x - ref);
            j.s += ms[k].y * kn;
            j.acc += x[k] * kn;
        }
    }
    for (int o = l.width; o < 64; o *= 2) j.add(__shfl_xor(j.m, o, 64), __shfl_xor(j.s, o, 64), __shfl_xor(j.acc, o, 64));
    return j;
}

template <class T>
__global__ __launch_bounds__(gs::kJoinWaves * 64)
void attn_join_kernel(FwdArgs a) {
    constexpr int N = gs::kJoinWaves;
    __shared__ Joined part[N][64];
    __shared__ gs::LongLists longs;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = blockIdx.y;
    const gs::JoinLanes l(lane, a.dim, blockIdx.z);
    const int64_t mine = gs::join_list(wave, lane);
    uint32_t b = 0, e = 0;
    if (mine < a.nb.n_parents) a.nb.range(mine, b, e);
    const bool mine_todo = mine < a.nb.n_parents && gs::needs_join(b, e, a.chunk);
    const bool many = mine_todo && e > b && (e - 1) / a.chunk - b / a.chunk >= kFewPieces;
    unsigned long long few = __ballot(mine_todo && !many);
    const auto write = [&](int64_t list, const Joined &j) {
        const int64_t at = list * a.heads + h;
        if (l.sub == 0 && l.in) static_cast<T *>(a.out)[at * a.dim + l.d] = (T)(j.acc * inverse_of(j.s));
        if (lane == 0 && blockIdx.z == 0) a.lse[at] = (j.m + gs::fast_log2(j.s)) * gs::kLn2;
    };
    for (; few; few &= few - 1) {
        const int src = __builtin_ctzll(few);
        const uint32_t sb = __shfl(b, src, 64), se = __shfl(e, src, 64);
        Joined j{-INFINITY, 0.f, 0.f};
        if (se > sb) j = join_pieces(a, sb, se, l.sub, l.subs, h, l);
        write(gs::join_list(wave, src), j);
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
        const Joined own = join_pieces(a, longs.b[i], longs.e[i], wave * l.subs + l.sub, N * l.subs, h, l);
        __syncthreads();                            // the last list's parts are read
        part[wave][lane] = own;
        __syncthreads();
        if (wave) continue;
        Joined j = part[0][lane];
        for (int k = 1; k < N; ++k) j.add(part[k][lane].m, part[k][lane].s, part[k][lane].acc);
        write(gs::join_list(longs.slot[i] >> 6, longs.slot[i] & 63), j);
    }
}

template <class T, int L, bool SHARED>
void launch_fwd(const FwdArgs &a, const gs::Deal &d, hipStream_t stream) {
    const int share = a.heads / a.kv_heads;
    FwdArgs b = a;
    const int g = gs::heads_per_wave(share);
    b.parts = (share + g - 1) / g;
    const dim3 grid((unsigned)((d.waves + gs::kAttnThreads / 64 - 1) / (gs::kAttnThreads / 64)), (unsigned)(a.kv_heads * b.parts));
    if (d.is_short) {
        if (g == 1) attn_fwd_short_kernel<T, L, 1, SHARED><<<grid, gs::kAttnThreads, 0, stream>>>(b);
        else if (g == 2) attn_fwd_short_kernel<T, L, 2, SHARED><<<grid, gs::kAttnThreads, 0, stream>>>(b);
        else attn_fwd_short_kernel<T, L, 4, SHARED><<<grid, gs::kAttnThreads, 0, stream>>>(b);
    } else if (g == 1) attn_fwd_kernel<T, L, 1, SHARED><<<grid, gs::kAttnThreads, 0, stream>>>(b);
    else if (g == 2) attn_fwd_kernel<T, L, 2, SHARED><<<grid, gs::kAttnThreads, 0, stream>>>(b);
    else attn_fwd_kernel<T, L, 4, SHARED><<<grid, gs::kAttnThreads, 0, stream>>>(b);
}

template <class T>
int run_fwd(const FwdArgs &a, const gs::Deal &d, int lanes, hipStream_t stream) {
    if (d.waves) {
        GS_BY_LANES(launch_fwd, a.v == nullptr, a, d, stream);
        if (int rc = gs::check_launch("gs_neighbor_attention_fwd")) return rc;
    }
    if (d.pieces) {
        attn_join_kernel<T><<<gs::join_grid(a.nb.n_parents, a.heads, a.dim), gs::kJoinWaves * 64, 0, stream>>>(a);
        return gs::check_launch("gs_neighbor_attention_fwd (join)");
    }
    return GS_OK;
}

size_t pieces_bytes(const gs::Deal &d, int heads, int dim, size_t *off_acc) {
    if (!d.pieces || !d.waves) { if (off_acc) *off_acc = 0; return 0; }
    const size_t ms = gs::align256((size_t)d.waves * 2 * heads * sizeof(float2));
    if (off_acc) *off_acc = ms;
    return ms + (size_t)d.waves * 2 * heads * dim * sizeof(float);
}

}  // namespace

extern "C" size_t gs_neighbor_attention_workspace(const gs_neighbors *nb, int heads, int kv_heads, int dim, int dtype) {
    if (gs::check_neighbors("gs_neighbor_attention_workspace", nb, heads, kv_heads, dim, dtype)) return 0;
    const gs::Deal d = gs::deal_edges(nb, gs::lanes_for(dim, gs::dtype_size(dtype)));
    return pieces_bytes(d, heads, dim, nullptr);
}

extern "C" int gs_neighbor_attention_fwd(const void *q, const void *k, const void *v, const gs_neighbors *nb, int heads,
                                         int kv_heads, int dim, int dtype, float scale, void *out, float *lse,
                                         void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = gs::check_neighbors("gs_neighbor_attention_fwd", nb, heads, kv_heads, dim, dtype)) return rc;
    if (nb->n_parents == 0) return GS_OK;
    if (!q || !out || !lse || (nb->n_edges && nb->n_rows && !k)) return gs::fail(GS_EINVAL, "gs_neighbor_attention_fwd: null pointer argument");
    const int size = gs::dtype_size(dtype), lanes = gs::lanes_for(dim, size);
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & (size - 1))
        return gs::fail(GS_EINVAL, "gs_neighbor_attention_fwd: pointer not aligned to its element");
    const gs::Deal d = gs::deal_edges(nb, lanes);
    size_t off_acc = 0;
    const size_t need = pieces_bytes(d, heads, dim, &off_acc);
    if (workspace_bytes < need || (need && (!workspace || ((uintptr_t)workspace & 15))))
        return gs::fail(GS_EINVAL, "gs_neighbor_attention_fwd: aligned workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    FwdArgs a;
    a.nb = gs::device_neighbors(nb);
    a.q = q; a.k = k; a.v = v; a.out = out; a.lse = lse;
    a.piece_ms = need ? static_cast<float2 *>(workspace) : nullptr;
    a.piece_acc = need ? reinterpret_cast<float *>(static_cast<char *>(workspace) + off_acc) : nullptr;
    a.scale2 = scale * gs::kLog2e;
    a.heads = heads; a.kv_heads = kv_heads; a.dim = dim; a.chunk = (int)d.chunk; a.parts = 1;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == GS_F32) return run_fwd<float>(a, d, lanes, s);
    if (dtype == GS_BF16) return run_fwd<__bf16>(a, d, lanes, s);
    return run_fwd<_Float16>(a, d, lanes, s);
}
