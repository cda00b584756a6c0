// Attention over neighbors: how the edges are dealt to the waves, shared by the forward and the backward kernels.
//
// A row of dim elements is covered by L lanes, 16 bytes each (L = the power of two >= dim / (elements in 16 bytes)), so
// a wave holds 64 / L rows at a time and keeps kAttnRows such groups in flight.  A dot product is a few multiply-adds per
// lane (16-bit types: two products per instruction, straight from the packed row) and a sum over L lanes; a row is read
// once, whatever the number of heads that share it.  Loads ask for the alignment of an element only, which the hardware
// serves at 16 bytes a lane; where dim is not a multiple of those, the last lane takes the last 16 bytes of the row and
// the elements it shares with its neighbor count there alone.
//
// A wave works on one list (the neighbors of one parent) at a time: control flow and list bounds are scalar, lists of any
// length leave no lane waiting for another lane's list (2M ragged edges of eight heads: 840 us with a list per L lanes, 528 us
// with the first form of this), and the running softmax of each of the 64 / L row groups is joined at the end of the list by
// half-wave and quarter-wave swaps that leave every lane the results it stores.  Entries come 64 at a time, one a lane,
// one load ahead: the next list's ids are on their way while this list's rows are used.
//
// Short lists of one length (a sampled batch) are the exception: there every L lanes take a list of their own, one row
// after the other, and nothing has to be joined (short_lists below).
//
// Lists are dealt by edges: wave w takes the lists that begin in edges [w C, (w + 1) C) and, of a list longer than 4 C, the
// part that lies in there, so that a popular parent's list is spread over the chip.  Every wave leaves a piece (maximum,
// sum, unnormalised row) of such a list in the workspace and a second launch joins them in wave order.  Where no list is
// that long there is no second launch.  The result depends on C, which depends on the sizes only.
#pragma once

#include "ops_common.h"

namespace gs {

constexpr int kAttnThreads = 256;
constexpr int kAttnRows = 4;                        // rows in flight per L lanes (L = 2: two, 64 in a wave)

// Offsets are read with scalar loads: they do not change while a kernel runs.
using ConstOffsets = const __attribute__((address_space(4))) int64_t *;

struct Neighbors {
    const int64_t *indptr;
    __device__ __forceinline__ int64_t offset(int64_t i) const { return ((ConstOffsets)(uintptr_t)indptr)[i]; }
    const int32_t *ids;
    int64_t n_parents, id_offset, n_rows;
    uint32_t n_child, n_edges;

    // [begin, end) of parent p, inside [0, n_edges] whatever indptr holds
    // (scalar: p is the same in all lanes)
    __device__ __forceinline__ void range(int64_t p, uint32_t &b, uint32_t &e, bool scalar = false) const {
        if (!indptr) { b = (uint32_t)p * n_child; e = b + n_child; return; }
        const int64_t x = scalar ? offset(p) : indptr[p], y = scalar ? offset(p + 1) : indptr[p + 1];
        b = (uint32_t)(x < 0 ? 0 : x > n_edges ? n_edges : x);
        e = (uint32_t)(y < 0 ? 0 : y > n_edges ? n_edges : y);
        if (e < b) e = b;
    }
    // the first parent from p on whose range ends behind edge e; n_parents if there is none.  Steps grow from one: the
    // answer is near unless many parents without neighbors lie between.
    __device__ __forceinline__ int64_t seek(uint32_t e, int64_t p) const {
        if (!indptr) return e / n_child;
        int64_t step = 1, lo = p, hi = p;
        while (hi < n_parents && offset(hi + 1) <= (int64_t)e) { lo = hi + 1; hi += step; step *= 2; }
        if (hi > n_parents) hi = n_parents;
        while (lo < hi) {
            const int64_t mid = (lo + hi) >> 1;
            if (offset(mid + 1) > (int64_t)e) hi = mid; else lo = mid + 1;
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
    // Entry e of the lists as it stands in memory, and the table row it means, or -1: two steps, so that a load can be
    // on its way for a while.
    __device__ __forceinline__ int32_t entry(uint32_t e) const { return ids ? ids[min(e, n_edges - 1)] : (int32_t)e; }
    __device__ __forceinline__ int32_t row_of(int32_t entry) const {
        const int64_t r = ids ? (int64_t)entry - id_offset : (int64_t)entry;
        return (uint64_t)r < (uint64_t)n_rows ? (int32_t)r : -1;
    }
};

// A wave's way through its edges, list by list, in units of at most 64 entries.  All of it is the same in every lane.
struct Unit {
    int64_t p;                                      // the list
    uint32_t e, n;                                  // entries e .. e + n - 1
    bool first, last;                               // of this wave's part of the list
    bool complete;                                  // the part is the list
    uint32_t place;                                 // wave * 2 + 0 or 1: where a piece goes
};

struct Walk {
    Neighbors nb;
    uint32_t e, e0, e1, most, w, left;              // left: entries of the list at hand that no unit has yet
    int64_t p_next;
    Unit u;

    __device__ __forceinline__ Walk(const Neighbors &n, uint32_t wave, uint32_t chunk) : nb(n), most(4 * chunk), w(wave), left(0) {
        e0 = (uint32_t)min((uint64_t)w * chunk, (uint64_t)nb.n_edges);
        e1 = (uint32_t)min((uint64_t)e0 + chunk, (uint64_t)nb.n_edges);
        e = e0;
        p_next = e < e1 ? nb.seek_wave(e) : nb.n_parents;
    }
    __device__ __forceinline__ bool next() {
        if (left) {
            u.e += u.n;
            u.n = min(left, 64u);
            left -= u.n;
            u.first = false;
            u.last = left == 0;
            return true;
        }
        while (e < e1 && p_next < nb.n_parents) {
            uint32_t sb, se;
            nb.range(p_next, sb, se, true);
            if (se <= e) { p_next = nb.seek(e, p_next + 1); continue; }
            const bool cut = se - sb > most;
            if (!cut && sb < e0) { e = se; ++p_next; continue; }       // begins before this wave's edges: another's
            if (sb > e) { e = sb; if (e >= e1) return false; }
            const uint32_t end = cut ? min(se, e1) : se;
            u.p = p_next++;
            u.e = e;
            u.n = min(end - e, 64u);
            left = end - e - u.n;
            u.first = true;
            u.last = left == 0;
            u.complete = !cut;
            u.place = w * 2 + (e == e0 ? 0 : 1);
            e = end;
            return true;
        }
        return false;
    }
};

// Pieces of a list [b, e) that was cut: the first lies in its wave's second place unless the list begins there.
__device__ __forceinline__ size_t piece_place(uint32_t b, uint32_t chunk, uint32_t i) {
    return (size_t)(b / chunk + i) * 2 + (i == 0 && b % chunk ? 1 : 0);
}

// Joins across the 64 / L row groups of a wave.  other<O>: the value of lane ^ O (or, for 8, of the lane half a row of 16
// away, which is the same lane).
template <int O> __device__ __forceinline__ float other(float v) {
    if (O == 4) return __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(v), (4 << 10) | 0x1F));
    if (O == 2) return dpp<0x4E>(v);                // quad_perm 2 3 0 1
    if (O == 8) return dpp<0x128>(v);               // row_ror 8
    return __shfl_xor(v, O, 64);
}
template <int L> __device__ __forceinline__ float groups_max(float v) {
    if (L <= 32) {
        auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
        v = fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
    }
    if (L <= 16) {
        auto r = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
        v = fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
    }
    if (L <= 8) v = fmaxf(v, other<8>(v));
    if (L <= 4) v = fmaxf(v, other<4>(v));
    if (L <= 2) v = fmaxf(v, other<2>(v));
    return v;
}
template <int L> __device__ __forceinline__ float groups_sum(float v) {
    if (L <= 32) {
        auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
        v = __int_as_float(r[0]) + __int_as_float(r[1]);
    }
    if (L <= 16) {
        auto r = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
        v = __int_as_float(r[0]) + __int_as_float(r[1]);
    }
    if (L <= 8) v += other<8>(v);
    if (L <= 4) v += other<4>(v);
    if (L <= 2) v += other<2>(v);
    return v;
}

// Sums N values per lane over the row groups, halving what a lane keeps at every step: x[0 .. kept) are then the sums of
// values start .. start + kept - 1 of its element lane.  Lanes with dup set hold copies of another's.
template <int N, int L> struct Scatter {
    static constexpr int kGroups = 64 / L, kKept = N > kGroups ? N / kGroups : 1;
    int start;
    bool dup;
    template <int C, int O> __device__ __forceinline__ void step(float *x, int lane64) {
        if constexpr (O >= L) {
            const bool up = lane64 & O;
            if constexpr (C > 1) {
                constexpr int H = C / 2;
#pragma unroll
                for (int i = 0; i < H; ++i) {
                    if constexpr (O == 32) {
                        auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(x[i]), __float_as_int(x[i + H]), false, false);
                        x[i] = __int_as_float(r[0]) + __int_as_float(r[1]);
                    } else if constexpr (O == 16) {
                        auto r = __builtin_amdgcn_permlane16_swap(__float_as_int(x[i]), __float_as_int(x[i + H]), false, false);
                        x[i] = __int_as_float(r[0]) + __int_as_float(r[1]);
                    } else {
                        const float a = x[i] + other<O>(x[i]), b = x[i + H] + other<O>(x[i + H]);
                        x[i] = up ? b : a;
                    }
                }
                if (up) start += H;
            } else {
                x[0] += other<O>(x[0]);
                if (up) dup = true;
            }
            step<(C > 1 ? C / 2 : 1), O / 2>(x, lane64);
        }
    }
    __device__ __forceinline__ void run(float *x, int lane64) {
        start = 0;
        dup = false;
        step<N, 32>(x, lane64);
    }
};

constexpr int kJoinWaves = 16;

// Where a lane's 16 bytes of a row begin, and how many of its elements belong to the lane before it (E or more: all).
// L = 2 stands for rows shorter than 16 bytes, read element by element.
template <class T, int L> struct Place {
    static constexpr int E = Pack<T>::E;
    int off, skip, dim;
    __device__ __forceinline__ Place(int lane, int d) {
        off = L == 2 ? 0 : min(lane * E, d - E);
        skip = lane * E - off;
        dim = d;
    }
};

// 16 bytes of a row, as they arrive.
template <class T> struct RowPart {
    static constexpr int E = Pack<T>::E;
    T x[E];
    __device__ __forceinline__ void zero() {
        const uint4 z = make_uint4(0, 0, 0, 0);
        __builtin_memcpy(x, &z, 16);
    }
    __device__ __forceinline__ void zero_if(bool c) {
        uint4 v;
        __builtin_memcpy(&v, x, 16);
        v.x = c ? 0 : v.x; v.y = c ? 0 : v.y; v.z = c ? 0 : v.z; v.w = c ? 0 : v.w;
        __builtin_memcpy(x, &v, 16);
    }
    template <int L> __device__ __forceinline__ void load(const T *row, const Place<T, L> &at) {
        if (L != 2) __builtin_memcpy(x, row + at.off, 16);
        else
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] = i < at.dim ? row[i] : (T)0.f;
    }
    // zeros in place of the elements that count in another lane: for one side of every dot product
    template <int L> __device__ __forceinline__ void own(const Place<T, L> &at) {
        if (L == 2 || at.dim % E)
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] = i < at.skip ? (T)0.f : x[i];
        else zero_if(at.skip > 0);
    }
    __device__ __forceinline__ float at(int i) const { return (float)x[i]; }
};

__device__ __forceinline__ float dot(const RowPart<float> &a, const RowPart<float> &b) {
    float d = a.x[0] * b.x[0];
#pragma unroll
    for (int i = 1; i < 4; ++i) d = __builtin_fmaf(a.x[i], b.x[i], d);
    return d;
}
__device__ __forceinline__ float dot(const RowPart<__bf16> &a, const RowPart<__bf16> &b) {
    using V = __attribute__((ext_vector_type(2))) __bf16;
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) d = __builtin_amdgcn_fdot2_f32_bf16(V{a.x[i], a.x[i + 1]}, V{b.x[i], b.x[i + 1]}, d, false);
    return d;
}
__device__ __forceinline__ float dot(const RowPart<_Float16> &a, const RowPart<_Float16> &b) {
    using V = __attribute__((ext_vector_type(2))) _Float16;
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) d = __builtin_amdgcn_fdot2(V{a.x[i], a.x[i + 1]}, V{b.x[i], b.x[i + 1]}, d, false);
    return d;
}

// Stores values start .. start + N - 1 of a lane's part of a row, those that count in this lane.
template <int N, class T, int L, class O>
__device__ __forceinline__ void store_part(O *row, const Place<T, L> &at, int start, const float *v) {
    if (L != 2 && at.skip <= 0) {
        O x[N];
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = (O)v[i];
        __builtin_memcpy(row + at.off + start, x, N * sizeof(O));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (start + i >= at.skip && at.off + start + i < at.dim) row[at.off + start + i] = (O)v[i];
    }
}

// Lanes per row: enough for dim elements at 16 bytes a lane.
inline int lanes_for(int dim, int size) {
    const int per = 16 / size;
    if (dim < per) return 2;
    int l = 4;
    while (l * per < dim) l *= 2;
    return l;
}

// Heads of one key head that a wave takes at once (a share of three fills four: 20000 lists of 10, gradients 139 us, 192 by twos).
inline int heads_per_wave(int share) { return share >= 3 ? 4 : share; }

// Lists of one length that L lanes take each.  Up to 12 entries always (lists of 12 rows of 64 fp32, four heads, forward and backward,
// this against a list per wave: 64 lists 16 us and 19, 4096 lists 20 and 27; one head, 64 lists 11 and 12); up to 32 where
// the lists fill a wave for each of the chip's 1024 SIMDs, at which the crossing lies for any number of lanes:
//   8 lanes, four heads, 25 rows   4096 lists 32 us and 27, 8192 lists 36 and 43, 16384 lists 50 and 69
//   16 lanes, one head, 20 rows    2048 lists 16 us and 13, 4096 lists 18 and 18, 8192 lists 27 and 31
//   64 lanes, four heads, 25 rows  1024 lists 44 us and 56, 4096 lists 110 and 157
// (4 lanes cross earlier, one head, 20 rows: 8192 lists 17 us and 20).
inline bool short_lists(int64_t n_lists, int64_t n_child, int lanes) {
    return n_child <= 12 || (n_lists * lanes >= 1024 * 64 && n_child <= 32);
}

// Edges per wave, and whether any list may be cut.  Short: lists of one length, a list per `lanes` lanes.
struct Deal {
    int64_t chunk, waves;
    bool pieces, is_short;
};

inline Deal deal_edges(const int64_t *indptr, int64_t n_lists, int64_t n_child, int64_t n_edges, int lanes) {
    Deal d;
    d.is_short = !indptr && n_child > 0 && short_lists(n_lists, n_child, lanes);
    if (d.is_short) {
        // eight lists a group, if that leaves enough waves
        const int64_t lists = n_edges / n_child, groups = 64 / lanes;
        d.chunk = n_child;
        d.pieces = false;
        d.waves = (lists + groups - 1) / groups;
        if (d.waves > 16384) d.waves = d.waves / 8 > 16384 ? (d.waves + 7) / 8 : 16384;
        return d;
    }
    // two rounds of row loads, but no more than two lists of the mean length: a wave takes them one after the other
    // (1450 edges of 13000 lists, 32 a wave: 112 us); as many edges as leave 16384 waves (two rounds of eight per SIMD: a
    // little more than one round leaves a few waves for the second), at most 512; and a list of the mean length
    // leaves at most 256 pieces (three lists of 39000: 4900 pieces each took 270 us to join)
    const int64_t mean = n_lists ? n_edges / n_lists : 0;
    int64_t c = 2 * kAttnRows * (64 / lanes);
    if (c > 2 * mean) c = 2 * mean > 2 ? 2 * mean : 2;
    if (c < n_edges / 16384) c = n_edges / 16384 < 512 ? n_edges / 16384 : 512;
    if (c < mean / 256) c = mean / 256;
    // lists of one length that are no longer than that: whole lists
    if (!indptr && n_child > 0 && n_child <= c) c = c / n_child * n_child;
    d.chunk = c;
    d.pieces = indptr || n_child > 4 * c || n_child == 0;
    d.waves = n_edges ? (n_edges + c - 1) / c : 0;
    return d;
}

// A table without rows leaves every parent without neighbors.
inline Deal deal_edges(const gs_neighbors *nb, int lanes) {
    return nb->n_rows ? deal_edges(nb->indptr, nb->n_parents, nb->n_child, nb->n_edges, lanes) : deal_edges(nullptr, 0, 0, 0, lanes);
}
inline Neighbors device_neighbors(const gs_neighbors *nb) {
    if (!nb->n_rows) return Neighbors{nullptr, nb->ids, nb->n_parents, 0, 0, 0, 0};
    return Neighbors{nb->indptr, nb->ids, nb->n_parents, nb->id_offset, nb->n_rows, (uint32_t)(nb->indptr ? 0 : nb->n_child),
                     (uint32_t)nb->n_edges};
}

// Whether the second launch has something to do for a list: it is empty, or was cut.
__device__ __forceinline__ bool needs_join(uint32_t b, uint32_t e, uint32_t chunk) { return b == e || e - b > 4 * chunk; }

// How the lanes of a joining wave share the pieces of a list: 64 / width pieces at a time, width lanes each, for the
// elements that blockIdx.z stands for (64 of them, or the row where it is shorter).
struct JoinLanes {
    int width, sub, subs, d;
    bool in;
    __device__ __forceinline__ JoinLanes(int lane, int dim, int column) {
        width = 64;
        while (width / 2 >= dim) width /= 2;
        sub = lane / width;
        subs = 64 / width;
        d = column * 64 + lane % width;
        in = d < dim;
        if (!in) d = dim - 1;
    }
};
constexpr int kJoinFlight = 8;                      // pieces of a lane on their way
// A joining launch: y a vector, z 64 elements of it.  List x of block b is x * blocks + b (popular lists tend to be neighbors),
// and wave x % kJoinWaves looks after it: one list a block while there are few, then about 2048 blocks in all, 512 for a vector at
// most, until a lane has one each (100 000 lists, most of them empty: 8 us, 32 us in blocks of 64 lists; 1053 lists for twelve
// heads of 200: 67 us with 512 for each of the 48).
inline dim3 join_grid(int64_t lists, int vectors, int dim) {
    const int columns = (dim + 63) / 64;
    const int64_t full = (lists + 64 * kJoinWaves - 1) / (64 * kJoinWaves);
    int64_t few = 2048 / ((int64_t)vectors * columns);
    few = few < 16 ? 16 : few > 512 ? 512 : few;
    if (few > lists) few = lists;
    return dim3((unsigned)(full > few ? full : few), (unsigned)vectors, (unsigned)columns);
}
__device__ __forceinline__ int64_t join_list(int wave, int lane) { return (int64_t)(lane * kJoinWaves + wave) * gridDim.x + blockIdx.x; }
// The lists of a block that take all its waves, in any order.
struct LongLists {
    int n;
    uint32_t slot[64 * kJoinWaves], b[64 * kJoinWaves], e[64 * kJoinWaves];
};

__device__ __forceinline__ uint32_t this_wave() {
    return __builtin_amdgcn_readfirstlane(blockIdx.x * (kAttnThreads / 64) + (threadIdx.x >> 6));
}

// f<T, lanes, flag>(...)
#define GS_BY_LANES(f, flag, ...)                                          \
    do {                                                                   \
        if (flag) {                                                        \
            if (lanes == 2) f<T, 2, true>(__VA_ARGS__);                    \
            else if (lanes == 4) f<T, 4, true>(__VA_ARGS__);               \
            else if (lanes == 8) f<T, 8, true>(__VA_ARGS__);               \
            else if (lanes == 16) f<T, 16, true>(__VA_ARGS__);             \
            else if (lanes == 32) f<T, 32, true>(__VA_ARGS__);             \
            else f<T, 64, true>(__VA_ARGS__);                              \
        } else {                                                           \
            if (lanes == 2) f<T, 2, false>(__VA_ARGS__);                   \
            else if (lanes == 4) f<T, 4, false>(__VA_ARGS__);              \
            else if (lanes == 8) f<T, 8, false>(__VA_ARGS__);              \
            else if (lanes == 16) f<T, 16, false>(__VA_ARGS__);            \
            else if (lanes == 32) f<T, 32, false>(__VA_ARGS__);            \
            else f<T, 64, false>(__VA_ARGS__);                             \
        }                                                                  \
    } while (0)

// Checks a gs_neighbors; 0 or the error.
int check_neighbors(const char *what, const gs_neighbors *nb, int heads, int kv_heads, int dim, int dtype);

}  // namespace gs
