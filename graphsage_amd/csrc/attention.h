// Attention over neighbors: how the edges are dealt to the lanes, shared by the forward and the backward kernels.
//
// A row of dim elements is covered by a "worker" of L lanes, 16 bytes each (L = the power of two >= dim / (elements in
// 16 bytes)); a dot product is a few multiply-adds per lane and a sum over the worker's lanes, the running softmax
// (maximum, sum, weighted row) lives in the worker's registers, and the row is read once, whatever the number of
// heads that share it.  Tables whose rows do not start on 16 bytes are read element by element: lane l then holds
// elements l, l + L, ...; nothing else depends on which element sits where.
//
// Edges are dealt by count, not by parent: worker w takes the parents whose edges begin in [w C, (w + 1) C), so short
// lists cost no idle lanes, and of a list longer than 4 C the part that lies in there: a popular parent's list is spread
// over the chip.  Every worker leaves a piece (maximum, sum, unnormalised row) of such a list in the workspace and a second
// launch joins them in worker order; a wave that lies inside one list joins its workers' pieces in registers first and
// leaves one.  Where no list is that long there is no second launch.  The result depends on C, which depends on the
// sizes only.
#pragma once

#include "ops_common.h"

namespace gs {

constexpr int kAttnThreads = 256;
constexpr int kAttnRows = 8;                        // rows a worker has in flight, at most

struct Neighbors {
    const int64_t *indptr;
    const int32_t *ids;
    int64_t n_parents, id_offset, n_rows;
    uint32_t n_child, n_edges;

    // [begin, end) of parent p, inside [0, n_edges] whatever indptr holds
    __device__ __forceinline__ void range(int64_t p, uint32_t &b, uint32_t &e) const {
        if (!indptr) { b = (uint32_t)p * n_child; e = b + n_child; return; }
        const int64_t x = indptr[p], y = indptr[p + 1];
        b = (uint32_t)(x < 0 ? 0 : x > n_edges ? n_edges : x);
        e = (uint32_t)(y < 0 ? 0 : y > n_edges ? n_edges : y);
        if (e < b) e = b;
    }
    // the first parent from p on whose range ends behind edge e; n_parents if there is none.  Steps grow from one: the
    // answer is near unless many parents without neighbors lie between.
    __device__ __forceinline__ int64_t seek(uint32_t e, int64_t p) const {
        if (!indptr) return e / n_child;
        int64_t step = 1, lo = p, hi = p;
        while (hi < n_parents && indptr[hi + 1] <= (int64_t)e) { lo = hi + 1; hi += step; step *= 2; }
        if (hi > n_parents) hi = n_parents;
        while (lo < hi) {
            const int64_t mid = (lo + hi) >> 1;
            if (indptr[mid + 1] > (int64_t)e) hi = mid; else lo = mid + 1;
        }
        return lo;
    }
    // the same from 0 on, by all lanes of a wave: 64 probes a round
    __device__ __forceinline__ int64_t seek_wave(uint32_t e) const {
        if (!indptr) return n_child ? e / n_child : 0;
        int64_t lo = 0, hi = n_parents;
        while (lo < hi) {
            const int64_t step = (hi - lo + 63) / 64, at = lo + (threadIdx.x & 63) * step;
            const unsigned long long found = __ballot(at < hi && indptr[at + 1] > (int64_t)e);
            // the answer lies behind the last probe that has not passed e and not behind the first that has
            const int64_t last = (hi - 1 - lo) / step;                 // the last probe inside
            const int64_t first = found ? __builtin_ctzll(found) : last + 1;
            if (first == 0) break;
            if (found) hi = lo + first * step;
            lo = lo + (first - 1) * step + 1;
        }
        return lo;
    }
    // table row of edge e, or -1
    __device__ __forceinline__ int32_t row_of(uint32_t e) const {
        const int64_t r = ids ? (int64_t)ids[e] - id_offset : (int64_t)e;
        return (uint64_t)r < (uint64_t)n_rows ? (int32_t)r : -1;
    }
};

// A worker's way through its edges, list by list.
struct Walk {
    const Neighbors &nb;
    uint32_t e, e0, e1, most;
    int64_t p_next;
    // the piece at hand: parent p with edges [sb, se), of which [begin, end) are this worker's
    int64_t p;
    uint32_t sb, se, begin, end;

    __device__ __forceinline__ Walk(const Neighbors &n, uint32_t w, uint32_t chunk, int lanes) : nb(n), most(4 * chunk) {
        e0 = (uint32_t)min((uint64_t)w * chunk, (uint64_t)nb.n_edges);
        e1 = (uint32_t)min((uint64_t)e0 + chunk, (uint64_t)nb.n_edges);
        e = e0;
        const uint32_t first = w & ~(uint32_t)(64 / lanes - 1);
        const uint32_t ef = (uint32_t)min((uint64_t)first * chunk, (uint64_t)nb.n_edges);
        p_next = nb.n_parents;
        if (ef < nb.n_edges) p_next = nb.seek_wave(ef);                // (the same for all lanes)
        if (e < e1 && p_next < nb.n_parents) p_next = nb.seek(e, p_next);
    }
    __device__ __forceinline__ bool next() {
        while (e < e1 && p_next < nb.n_parents) {
            nb.range(p_next, sb, se);
            if (se <= e) { p_next = nb.seek(e, p_next + 1); continue; }
            const bool cut = se - sb > most;
            if (!cut && sb < e0) { e = se; ++p_next; continue; }       // begins before this worker's edges: another's
            if (sb > e) { e = sb; if (e >= e1) return false; }
            begin = e;
            end = cut ? min(se, e1) : se;
            e = end;
            p = p_next++;
            return true;
        }
        return false;
    }
    __device__ __forceinline__ bool complete() const { return begin == sb && end == se; }
    // whether the whole wave lies inside this list; the same in all its lanes
    __device__ __forceinline__ bool inside(uint32_t w, uint32_t chunk, uint32_t per_wave) const {
        const uint32_t b = w / per_wave * per_wave * chunk;
        return per_wave > 1 && se - sb > most && sb <= b && se >= b + per_wave * chunk;
    }
    // place (worker * 2 + 0 or 1) of this piece
    __device__ __forceinline__ size_t place(uint32_t w) const { return (size_t)w * 2 + (begin == e0 ? 0 : 1); }
};

// The pieces of a parent with edges [b, e), more than 4 C, in order: the workers of a wave that is only
// partly inside, one piece for each wave that lies inside (left by its first worker), the workers of the last wave.
struct PieceList {
    uint32_t first, n_head, n_full, full0, n_tail, tail0, cut;
    __device__ __forceinline__ PieceList(uint32_t b, uint32_t e, uint32_t chunk, uint32_t per_wave) {
        const uint32_t span = chunk * per_wave, a = (b + span - 1) / span, z = e / span;
        first = b / chunk;
        cut = b % chunk;                            // not 0: the first piece lies in its worker's second place
        if (z > a && per_wave > 1) {
            n_head = a * per_wave - first;
            n_full = z - a;
            full0 = a * per_wave;
            tail0 = z * per_wave;
            n_tail = e > z * span ? (e - 1) / chunk - tail0 + 1 : 0;
        } else { n_head = (e - 1) / chunk - first + 1; n_full = n_tail = full0 = tail0 = 0; }
        step = per_wave;
    }
    uint32_t step;
    __device__ __forceinline__ uint32_t count() const { return n_head + n_full + n_tail; }
    // place (worker * 2 + 0 or 1) of piece i
    __device__ __forceinline__ size_t place(uint32_t i) const {
        if (i < n_head) return (size_t)(first + i) * 2 + (i == 0 && cut ? 1 : 0);
        if (i < n_head + n_full) return (size_t)(full0 + (i - n_head) * step) * 2;
        return (size_t)(tail0 + (i - n_head - n_full)) * 2;
    }
};

constexpr int kJoinWaves = 8;

// 16 bytes of a row per lane, as they arrive.
template <class T, int L, bool ALIGNED> struct RowPart {
    static constexpr int E = Pack<T>::E;
    T x[E];
    __device__ __forceinline__ void load(const T *row, int lane, int dim) {
        if (ALIGNED) {
            if (lane * E < dim) *reinterpret_cast<uint4 *>(x) = reinterpret_cast<const uint4 *>(row)[lane];
            else *reinterpret_cast<uint4 *>(x) = make_uint4(0, 0, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] = lane + i * L < dim ? row[lane + i * L] : (T)0.f;
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = (T)0.f;
    }
    __device__ __forceinline__ float at(int i) const { return (float)x[i]; }
};

template <class T, int L, bool ALIGNED>
__device__ __forceinline__ void store_row(T *row, int lane, int dim, const float *v) {
    constexpr int E = Pack<T>::E;
    if (ALIGNED) {
        if (lane * E < dim) {
            alignas(16) T x[E];
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] = (T)v[i];
            reinterpret_cast<uint4 *>(row)[lane] = *reinterpret_cast<const uint4 *>(x);
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (lane + i * L < dim) row[lane + i * L] = (T)v[i];
    }
}

// Element index of part i of a lane, for the fp32 pieces in the workspace.
template <class T, int L, bool ALIGNED> __device__ __forceinline__ int element_of(int lane, int i) {
    return ALIGNED ? lane * Pack<T>::E + i : lane + i * L;
}

// Lanes per row: enough for dim elements at 16 bytes a lane.
inline int lanes_for(int dim, int size) {
    const int per = 16 / size;
    int l = 4;
    while (l * per < dim) l *= 2;
    return l;
}

// Edges per worker, and whether any list may be cut.
struct Deal {
    int64_t chunk, workers;
    bool pieces;
};

inline Deal deal_edges(const int64_t *indptr, int64_t n_parents, int64_t n_child, int64_t n_edges, int lanes) {
    Deal d;
    const int64_t per_wave = 64 / lanes;
    if (!indptr && n_child > 0 && (n_child <= 4 * kAttnRows || n_parents >= 4096 * per_wave)) {
        // lists of one length, short or many: whole lists, several where they are shorter than a round of loads
        const int64_t group = n_child < kAttnRows && n_parents >= 32768 * per_wave ? (kAttnRows + n_child - 1) / n_child : 1;
        d.chunk = group * n_child;
    } else {
        // one round of loads at least, then as many edges as leave 8192 waves (eight per SIMD), at most 128
        int64_t c = n_edges / (8192 * per_wave);
        c = (c + kAttnRows - 1) / kAttnRows * kAttnRows;
        d.chunk = c < kAttnRows ? kAttnRows : c > 128 ? 128 : c;
    }
    d.pieces = indptr || n_child > 4 * d.chunk || n_child == 0;
    d.workers = n_edges ? (n_edges + d.chunk - 1) / d.chunk : 0;
    return d;
}

// Whether the second launch has something to do for a list: it is empty, or was cut.
__device__ __forceinline__ bool needs_join(uint32_t b, uint32_t e, uint32_t chunk) { return b == e || e - b > 4 * chunk; }

// Checks a gs_neighbors; 0 or the error.
int check_neighbors(const char *what, const gs_neighbors *nb, int heads, int kv_heads, int dim, int dtype);

}  // namespace gs
