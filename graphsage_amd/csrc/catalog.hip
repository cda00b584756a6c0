// Log probabilities, entropy and best items of users over a catalog (layout and tile product: catalog.h).
//
// A wave keeps the fragments of 32 or 64 users in registers and streams the tiles of its share of the items; per tile the
// matrix cores give it 32 scores per user, sixteen in each of two lanes, and each lane runs the softmax over its own:
// a running maximum m, sum s = sum 2^(z - m) and w = sum 2^(z - m) (z - m), z in units of log 2 (scale log2 e goes into one
// multiply-add).  The shares' (m, s, w) are joined by a second launch: lse = m + log s, entropy = log s - w / s.
// The score of the target is picked up as its tile passes, so that log_prob is exactly 0 for a catalog of one item.
//
// Best items: the first launch also writes the largest score of every group of 4 or 32 items.  The k best items lie in groups
// whose largest score is among the k largest (each of k better groups would hold a better item), so only about k groups of a
// user are scored again, in 64 bits, from the tables themselves; groups within the rounding error of the first product
// count as candidates too.  The list is then a function of the tables alone, whatever the product's order of additions.
//
// 4096 users, 100 000 items of 64 bf16: 126 to 146 us for 52 GFLOP, bound by the vector ALU, which is busy 87% of the time (the
// exponential and about ten more instructions a score; the product alone would take 47 us at a large product's rate).  512 users of
// fp32, 20 best: 14 us to lay the tables out, 52 us (matrix cores busy 43%, vector ALU 41% of the time), 38 us for the best items,
// whose waves wait two thirds of theirs: phases with barriers between them.
#include "catalog.h"

#include <algorithm>

namespace gs {

int check_catalog(const char *what, int64_t n_users, int64_t n_items, int dim, int dtype, float scale) {
    if (!dtype_size(dtype)) return fail(GS_EINVAL, "%s: dtype %d", what, dtype);
    if (n_users < 0 || n_items < 0 || dim < 1) return fail(GS_EINVAL, "%s: users=%lld items=%lld dim=%d", what, (long long)n_users, (long long)n_items, dim);
    if (dim > 256) return fail(GS_ELIMIT, "%s: dim=%d (at most 256)", what, dim);
    if (n_items >= ((int64_t)1 << 31) - 512 || n_users >= ((int64_t)1 << 31) - 512)
        return fail(GS_ELIMIT, "%s: %lld users, %lld items (less than 2^31 - 512)", what, (long long)n_users, (long long)n_items);
    if (!(scale > 0.f) || !(scale < INFINITY)) return fail(GS_EINVAL, "%s: scale %g", what, scale);
    return GS_OK;
}

namespace {

// One block per tile of 32 rows, which lie one behind the other in memory: they are read whole, in 16-byte pieces where
// the table starts on one, into LDS as fp32, and leave in fragment order.
constexpr int kLdsPad = 4;

template <class T>
__global__ __launch_bounds__(kCatThreads)
void layout_kernel(Layout first, Layout second, int first_tiles, int block0, int dim, int blocks, uint32_t magic, int vector) {
    constexpr int P = Pieces<T>::P, E = 16 / sizeof(T);
    extern __shared__ float buf[];                  // [32][blocks * 32 + kLdsPad]
    __shared__ int on[32];
    __shared__ float tops[kCatThreads / 64];
    const int block = block0 + (int)blockIdx.x;
    const bool is_first = block < first_tiles;
    const Layout &l = is_first ? first : second;
    const int64_t tile = is_first ? block : block - first_tiles, row0 = tile * 32;
    const int rows = (int)min((int64_t)32, l.n_rows - row0), width = blocks * 32, ld = width + kLdsPad, tid = threadIdx.x;
    if (tid < 32) {
        const bool offered = tid < rows && !(l.bias && l.bias[row0 + tid] < kOffer);
        on[tid] = offered;
        if (l.bias2) l.bias2[row0 + tid] = !offered ? kMasked : l.bias ? l.bias[row0 + tid] * kLog2e : 0.f;
        if (l.stats) {
            // lse2 = 1e14 silences a user: padding, or one for whom nothing is on offer
            const int64_t n = row0 + tid;
            float lse2 = 1e14f, ca = 0.f, cb = 0.f, g = 0.f;
            int32_t t = -1;
            if (tid < rows && l.from.lse[n] != -INFINITY) {
                lse2 = l.from.lse[n] * kLog2e;
                if (l.from.targets && l.from.g_log_prob && l.from.targets[n] >= 0 && l.from.targets[n] < l.from.n_items) {
                    t = l.from.targets[n];
                    g = l.from.g_log_prob[n];
                }
                const float ge = l.from.g_entropy ? l.from.g_entropy[n] : 0.f;
                ca = -(g + (l.from.g_entropy ? ge * l.from.entropy[n] : 0.f));
                cb = -ge * kLn2;
            }
            Stats &st = l.stats[tile];
            st.lse2[tid] = lse2; st.a[tid] = ca; st.b2[tid] = cb; st.g[tid] = g; st.target[tid] = t;
        }
    }
    __syncthreads();
    const T *X = static_cast<const T *>(l.x) + row0 * dim;
    const int n = rows * dim;
    const auto put = [&](int i, float v) {
        const int r = dim == 1 ? i : (int)__umulhi((uint32_t)i, magic), d = i - r * dim;
        buf[r * ld + d] = on[r] ? v : 0.f;
    };
    int i = tid * E;
    if (vector)
        for (; i + E <= n; i += kCatThreads * E) {
            T v[E];
            *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(X + i);
#pragma unroll
            for (int k = 0; k < E; ++k) put(i + k, (float)v[k]);
        }
    for (; i < n; i += kCatThreads * E)
        for (int k = 0; k < E && i + k < n; ++k) put(i + k, (float)X[i + k]);
    // zeros behind the rows' ends and behind the last row
    for (int r = tid >> 5; r < 32; r += kCatThreads / 32)
        for (int d = (r < rows ? dim : 0) + (tid & 31); d < width; d += 32) buf[r * ld + d] = 0.f;
    __syncthreads();

    const int kcs = blocks * 2, lane = tid & 63;
    float top = 0.f;
    for (int f = tid >> 6; f < kcs; f += kCatThreads / 64) {
        if (l.rows) {
            float v[8];
            const float *src = buf + (lane & 31) * ld + f * 16 + (lane >> 5) * 8;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[k] = src[k];
                top = fmaxf(top, v[k] == v[k] ? fabsf(v[k]) : INFINITY);
            }
            uint4 *out = l.rows + ((size_t)tile * kcs + f) * P * 64 + lane;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] = next_piece(v[2 * k], v[2 * k + 1]);
                out[(size_t)p * 64] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        if (l.cols) {
            float v[8];
            const int t = f / blocks, db = f % blocks;
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = buf[(t * 16 + 8 * (k >> 2) + 4 * (lane >> 5) + (k & 3)) * ld + db * 32 + (lane & 31)];
            uint4 *out = l.cols + ((size_t)tile * kcs + f) * P * 64 + lane;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] = next_piece(v[2 * k], v[2 * k + 1]);
                out[(size_t)p * 64] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
    if (l.tile_abs) {
#pragma unroll
        for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        if (lane == 0) tops[tid >> 6] = top;
        __syncthreads();
        if (tid == 0) {
#pragma unroll
            for (int k = 1; k < kCatThreads / 64; ++k) top = fmaxf(top, tops[k]);
            l.tile_abs[tile] = top;
        }
    }
}

template <class T>
int launch_layouts_of(const Layout &first, const Layout &second, int dim, hipStream_t stream) {
    const int64_t t0 = tiles_of(first.n_rows), t1 = tiles_of(second.n_rows);
    if (t0 + t1 == 0) return GS_OK;
    const int blocks = blocks_of(dim);
    const size_t lds = (size_t)32 * (blocks * 32 + kLdsPad) * sizeof(float);
    // i / dim for i < 2^13: exact with the rounded-up reciprocal
    const uint32_t magic = dim == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + dim - 1) / dim);
    const int vector = (((uintptr_t)first.x | (uintptr_t)second.x) & 15) == 0;
    constexpr int64_t most = kMostThreads / kCatThreads;
    for (int64_t b = 0; b < t0 + t1; b += most) {
        layout_kernel<T><<<dim3((unsigned)std::min(most, t0 + t1 - b)), kCatThreads, lds, stream>>>(first, second, (int)t0, (int)b, dim, blocks, magic, vector);
        if (int rc = check_launch("gs_catalog (layout)")) return rc;
    }
    return GS_OK;
}

}  // namespace

int launch_layouts(const Layout &first, const Layout &second, int dim, int dtype, hipStream_t stream) {
    if (dtype == GS_F32) return launch_layouts_of<float>(first, second, dim, stream);
    if (dtype == GS_BF16) return launch_layouts_of<__bf16>(first, second, dim, stream);
    return launch_layouts_of<_Float16>(first, second, dim, stream);
}

}  // namespace gs

namespace {

using namespace gs;

constexpr int kMaxTop = 64;

struct FwdArgs {
    const uint4 *user, *item;                       // rows layouts
    const float *bias2;
    const int32_t *targets;
    float4 *part;                                   // [users][shares]: m, s, w, target's score
    float *group_max;                               // [users][group_stride], with TOP: of every TOP consecutive items
    int64_t group_stride;
    int64_t n_users, n_items;
    int user_tiles, item_tiles, group_blocks, shares, tiles_per_share;
    float scale2;
};

// (m, s, w, target's score) of two sets of items.
__device__ __forceinline__ float4 join_sums(float4 a, float4 b) {
    const float m = fmaxf(a.x, b.x), da = a.x - m, db = b.x - m, fa = fast_exp2(da), fb = fast_exp2(db);
    return make_float4(m, a.y * fa + b.y * fb, fa * (a.z + a.y * da) + fb * (b.z + b.y * db), fmaxf(a.w, b.w));
}

template <int N> __device__ __forceinline__ float4 join_lanes(float4 q) {
#pragma unroll
    for (int o = N / 2; o; o >>= 1)
        q = join_sums(q, make_float4(__shfl_xor(q.x, o, 64), __shfl_xor(q.y, o, 64), __shfl_xor(q.z, o, 64), __shfl_xor(q.w, o, 64)));
    return q;
}

template <int P, int DB, int OF, int TOP>
__global__ __launch_bounds__(kCatThreads, waves_for(8 * DB * P * OF + 16 * OF + 24))
void catalog_fwd_kernel(FwdArgs a) {
    constexpr int KC = 2 * DB, F = KC * P, ST = tiles_per_stage(F), W = kCatThreads / 64;
    extern __shared__ uint4 stage[];                // [2][ST][F][64]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t lds = __builtin_amdgcn_readfirstlane((uint32_t)reinterpret_cast<uintptr_t>(stage));
    const int group = (int)(blockIdx.x % (uint32_t)a.group_blocks) * W + wave, share = (int)(blockIdx.x / (uint32_t)a.group_blocks);
    const int t0 = share * a.tiles_per_share, t1 = min(t0 + a.tiles_per_share, a.item_tiles);
    const auto issue = [&](int t, int half) {
#pragma unroll
        for (int k = 0; k < ST; ++k)
            if (t + k < t1)
#pragma unroll
                for (int i = 0; i < (F + W - 1) / W; ++i)
                    if (i * W + wave < F)
                        fragment_to_lds(a.item + ((size_t)(t + k) * F + i * W + wave) * 64, lane, lds + ((half * ST + k) * F + i * W + wave) * 1024);
    };
    issue(t0, 0);

    Fragment<P> own[OF][KC];
    float m[OF], s[OF], w[OF], hit[OF];
    int target[OF];
#pragma unroll
    for (int f = 0; f < OF; ++f) {
        const int tile = min(group * OF + f, a.user_tiles - 1);            // (a tile past the end repeats the last one)
        const uint4 *src = a.user + (size_t)tile * KC * P * 64;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) own[f][kc] = load_fragment<P>(src, kc, lane);
        const int64_t n = (int64_t)tile * 32 + (lane & 31);
        target[f] = a.targets && n < a.n_users ? a.targets[n] : -1;
        if (target[f] >= a.n_items) target[f] = -1;
        m[f] = kFloor;
        s[f] = w[f] = 0.f;
        hit[f] = -INFINITY;
    }
    float tops[OF][4];
    for (int t = t0; t < t1; ++t) {
        const int at = (t - t0) % ST, half = (t - t0) / ST % 2;
        if (at == 0) {
            stage_ready();
            if (t + ST < t1) issue(t + ST, half ^ 1);
        }
        const uint4 *src = stage + (half * ST + at) * F * 64;
        f32x16 acc[OF];
#pragma unroll
        for (int f = 0; f < OF; ++f)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[f][r] = 0.f;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
            const Fragment<P> it = load_fragment<P>(src, kc, lane);
#pragma unroll
            for (int f = 0; f < OF; ++f) multiply<P, P, 2>(acc[f], it.p, own[f][kc].p);
        }
        float b[16];
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<float4 *>(b + 4 * g) = *reinterpret_cast<const float4 *>(a.bias2 + (size_t)t * 32 + 8 * g + 4 * (lane >> 5));
#pragma unroll
        for (int f = 0; f < OF; ++f) {
            float z[16], top = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                z[r] = __builtin_fmaf(acc[f][r], a.scale2, b[r]);
                top = fmaxf(top, z[r]);
            }
            const int local = target[f] - t * 32;
            if (__any(target[f] >= 0 && (unsigned)local < 32u))
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (target[f] >= 0 && local == row_of_reg(r, lane)) hit[f] = z[r];
            const int64_t n = ((int64_t)group * OF + f) * 32 + (lane & 31);
            if (TOP == 32) {
                // four tiles' largest scores leave together
                tops[f][t & 3] = half_max(top);
                if (((t & 3) == 3 || t + 1 == t1) && lane < 32 && n < a.n_users)
                    *reinterpret_cast<float4 *>(a.group_max + n * a.group_stride + (t & ~3)) = make_float4(tops[f][0], tops[f][1], tops[f][2], tops[f][3]);
            } else if (TOP == 4) {
                // registers 4 q .. 4 q + 3 are items 8 q + 4 (lane / 32) and on of the tile
                if (n < a.n_users)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        a.group_max[n * a.group_stride + t * 8 + 2 * q + (lane >> 5)] =
                            fmaxf(fmaxf(z[4 * q], z[4 * q + 1]), fmaxf(z[4 * q + 2], z[4 * q + 3]));
            }
            if (__any(top > m[f])) {
                const float m1 = fmaxf(m[f], top), step = m[f] - m1, keep = fast_exp2(step);
                w[f] = keep * (w[f] + s[f] * step);
                s[f] *= keep;
                m[f] = m1;
            }
            // a tile's terms first, in four chains: hundreds one by one would cost digits
            float sp[4] = {0.f, 0.f, 0.f, 0.f}, wp[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float d = z[r] - m[f], p = fast_exp2(d);
                sp[r & 3] += p;
                wp[r & 3] = __builtin_fmaf(p, d, wp[r & 3]);
            }
            s[f] += (sp[0] + sp[1]) + (sp[2] + sp[3]);
            w[f] += (wp[0] + wp[1]) + (wp[2] + wp[3]);
        }
    }
#pragma unroll
    for (int f = 0; f < OF; ++f) {
        const int tile = group * OF + f;
        // the two lanes of a user
        const float m1 = half_max(m[f]), step = m[f] - m1, keep = fast_exp2(step);
        const float s1 = s[f] * keep, w1 = keep * (w[f] + s[f] * step);
        const float s2 = s1 + __shfl_xor(s1, 32, 64), w2 = w1 + __shfl_xor(w1, 32, 64);
        const float hit1 = half_max(hit[f]);
        const int64_t n = (int64_t)tile * 32 + lane;
        if (lane < 32 && tile < a.user_tiles && n < a.n_users) a.part[(size_t)n * a.shares + share] = make_float4(m1, s2, w2, hit1);
    }
}

// A few users: a block has them all, 32 a wave, so an item row is used by few waves and laying the table out would cost more than
// that saves.  The waves read the rows as they are, eight elements a lane, and cut them into pieces in registers (one user, 100 000
// items of 32 fp32: 10.5 us; 12 us to lay the items out and 11 us for their product else).  With less than 33 users the four
// waves take a tile of items each, with less than 65 two, else all the same one.
struct FewArgs {
    const void *user, *item;
    const float *bias;
    const int32_t *targets;
    float4 *part;                                   // [users][blocks]
    float *group_max, *tile_abs;                    // tile_abs: [blocks], the largest |element| of their tiles
    int64_t group_stride, n_items;
    int n_users, dim, item_tiles;
    float scale2;
};

// Elements 16 kc + 8 half + 0 .. 7 of a row for all kc, zeros for those past its end: the last eight lie elsewhere among the eight,
// but in the same places for every row.  All loads leave before the first is used: four of them share a line that other waves
// would drive out of the first cache (5 users, 73 000 items of 256 bf16, if taken so: 46 us, 61 one after the other).
template <class T, int KC> struct RawRow {
    T x[KC][8];
    __device__ __forceinline__ void load(const T *row, int half, int dim) {
        if (dim >= 8) {
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) __builtin_memcpy(x[kc], row + min(16 * kc + 8 * half, dim - 8), sizeof(x[kc]));
        } else {
#pragma unroll
            for (int kc = 0; kc < KC; ++kc)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[kc][i] = row[min(16 * kc + 8 * half + i, dim - 1)];
        }
    }
    // element i of the eight, or a zero
    __device__ __forceinline__ float at(int kc, int i, int half, int dim) const {
        const int e0 = 16 * kc + 8 * half;
        const bool there = dim >= 8 ? i >= e0 - min(e0, dim - 8) : e0 + i < dim;
        return there ? (float)x[kc][i] : 0.f;
    }
};

template <class T, int DB, int TOP>
__global__ __launch_bounds__(kCatThreads, waves_for(8 * DB * Pieces<T>::P + 16 * DB + 80))
void catalog_few_kernel(FewArgs a) {
    constexpr int P = Pieces<T>::P, KC = 2 * DB, W = kCatThreads / 64;
    __shared__ float4 sums[W][32];
    __shared__ float tops[W];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 31, half = lane >> 5;
    const int user_tiles = (a.n_users + 31) / 32, at_once = max(W / user_tiles, 1);        // tiles of items a block has at once
    const int n = wave % user_tiles * 32 + r;       // the user of this lane
    Fragment<P> own[KC];
    const T *U = static_cast<const T *>(a.user) + (int64_t)min(n, a.n_users - 1) * a.dim;
    RawRow<T, KC> raw;
    raw.load(U, half, a.dim);
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = n < a.n_users ? raw.at(kc, i, half, a.dim) : 0.f;
        cut_pieces<P>(v, own[kc].p);
    }
    int target = a.targets && n < a.n_users ? a.targets[n] : -1;
    if (target >= a.n_items) target = -1;
    float m = kFloor, s = 0.f, w = 0.f, hit = -INFINITY, most_abs = 0.f;
    const int first = wave < at_once * user_tiles ? blockIdx.x * at_once + wave / user_tiles : a.item_tiles;
    for (int t = first; t < a.item_tiles; t += gridDim.x * at_once) {
        const int64_t row = min((int64_t)t * 32 + r, a.n_items - 1);
        raw.load(static_cast<const T *>(a.item) + row * a.dim, half, a.dim);
        const bool on = !(a.bias && a.bias[row] < kOffer);
        float b[16];
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t j = (int64_t)t * 32 + 8 * g + 4 * half + i;
                const float x = a.bias ? a.bias[min(j, a.n_items - 1)] : 0.f;
                b[4 * g + i] = j >= a.n_items || x < kOffer ? kMasked : x * kLog2e;
            }
        f32x16 acc;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] = 0.f;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[i] = on ? raw.at(kc, i, half, a.dim) : 0.f;
                if (TOP) most_abs = fmaxf(most_abs, fabsf(v[i]));
            }
            Fragment<P> it;
            cut_pieces<P>(v, it.p);
            multiply<P, P, 2>(acc, it.p, own[kc].p);
        }
        float z[16], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            z[i] = __builtin_fmaf(acc[i], a.scale2, b[i]);
            top = fmaxf(top, z[i]);
        }
        const int local = target - t * 32;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (target >= 0 && local == row_of_reg(i, lane)) hit = z[i];
        if (TOP == 32) {
            const float most = half_max(top);
            if (lane < 32 && n < a.n_users) a.group_max[n * a.group_stride + t] = most;
        } else if (TOP == 4) {
            if (n < a.n_users)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    a.group_max[n * a.group_stride + (int64_t)t * 8 + 2 * q + half] =
                        fmaxf(fmaxf(z[4 * q], z[4 * q + 1]), fmaxf(z[4 * q + 2], z[4 * q + 3]));
        }
        const float m1 = fmaxf(m, top), step = m - m1, keep = fast_exp2(step);
        w = keep * (w + s * step);
        s *= keep;
        m = m1;
        float sp[4] = {0.f, 0.f, 0.f, 0.f}, wp[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float d = z[i] - m, p = fast_exp2(d);
            sp[i & 3] += p;
            wp[i & 3] = __builtin_fmaf(p, d, wp[i & 3]);
        }
        s += (sp[0] + sp[1]) + (sp[2] + sp[3]);
        w += (wp[0] + wp[1]) + (wp[2] + wp[3]);
    }
    // the two lanes of a user, then the waves that have it
    const float m1 = half_max(m), step = m - m1, keep = fast_exp2(step);
    const float s1 = s * keep, w1 = keep * (w + s * step);
    const float s2 = s1 + __shfl_xor(s1, 32, 64), w2 = w1 + __shfl_xor(w1, 32, 64);
    const float hit1 = half_max(hit);
    if (lane < 32) sums[wave][r] = make_float4(m1, s2, w2, hit1);
    if (TOP) {
#pragma unroll
        for (int o = 32; o; o >>= 1) most_abs = fmaxf(most_abs, __shfl_xor(most_abs, o, 64));
        if (lane == 0) tops[wave] = most_abs;
    }
    __syncthreads();
    if (threadIdx.x >= a.n_users) return;
    const int mine = threadIdx.x;
    float4 q = sums[mine >> 5][mine & 31];
    for (int k = 1; k < at_once; ++k) q = join_sums(q, sums[k * user_tiles + (mine >> 5)][mine & 31]);
    a.part[(size_t)mine * gridDim.x + blockIdx.x] = q;
    if (TOP && mine == 0) a.tile_abs[blockIdx.x] = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
}

// What the shares of a user leave, and where it goes (nullable, one entry a user).
struct JoinArgs {
    const float4 *part;
    int shares;
    int64_t n_items;
    const int32_t *targets;
    float *log_prob, *entropy, *lse;
};

// N threads join the shares of user n, thread t of them the ones t, t + N, ...; a wave's part of it, in every lane.
template <int N> __device__ __forceinline__ float4 join_shares(const JoinArgs &a, int64_t n, int t) {
    const float4 none = make_float4(kFloor, 0.f, 0.f, -INFINITY);
    float4 q = none;
    for (int i = t; i < a.shares; i += 4 * N) {
        float4 x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = a.part[(size_t)n * a.shares + min(i + N * k, a.shares - 1)];
#pragma unroll
        for (int k = 0; k < 4; ++k) q = join_sums(q, i + N * k < a.shares ? x[k] : none);
    }
    return join_lanes<64>(q);
}

// The results of user n; log sum exp.  The target's distance to the largest score first: where it is the largest, what is left of
// 1 - p is log s alone, however far from zero the scores lie.
__device__ __forceinline__ float finish_user(const JoinArgs &a, int64_t n, float4 q, bool writes) {
    const float top = q.x, s = q.y, w = q.z, hit = q.w;
    const float l2 = fast_log2(s);                  // s 0: nothing on offer
    const float lse = s == 0.f ? -INFINITY : (top + l2) * kLn2;
    if (writes) {
        if (a.lse) a.lse[n] = lse;
        if (a.entropy) a.entropy[n] = s == 0.f ? 0.f : (l2 - w / s) * kLn2;
        if (a.log_prob) {
            const bool there = a.targets && a.targets[n] >= 0 && a.targets[n] < a.n_items;
            a.log_prob[n] = !there ? 0.f : s != s ? s : hit < kFloor ? -INFINITY : ((hit - top) - l2) * kLn2;
        }
    }
    return lse;
}

// A wave per user.
__global__ __launch_bounds__(kCatThreads)
void catalog_join_kernel(JoinArgs a, int64_t first_user, int64_t n_users) {
    const int64_t n = first_user + (int64_t)blockIdx.x * (kCatThreads / 64) + (threadIdx.x >> 6);
    if (n < n_users) finish_user(a, n, join_shares<64>(a, n, threadIdx.x & 63), (threadIdx.x & 63) == 0);
}

struct TopArgs {
    const void *user, *item;
    const float *bias, *group_max, *tile_abs;
    int64_t n_users, n_items, group_stride;
    int dim, n_abs, groups, log2_items, k, vector;  // log2_items: of a group
    float scale;
    float *top_log_prob;
    int32_t *top_ids;
};

// One block of N threads per user, which first joins the user's shares.  Thresholds and candidates: see the head of the file.
// Four lanes score an item.
template <class T, int N>
__global__ __launch_bounds__(N)
void catalog_top_kernel(TopArgs a, JoinArgs join) {
    constexpr int kBuf = 1024, kChunk = 4096, E = 16 / sizeof(T), kSets = 256, kPasses = 2048 / N;
    __shared__ double user[256];
    __shared__ double val[kBuf];
    __shared__ int32_t id[kBuf];
    __shared__ double best_val[kMaxTop];
    __shared__ int32_t best_id[kMaxTop];
    __shared__ __align__(16) float group_max[kSets];
    __shared__ float group_abs[kSets];
    __shared__ uint16_t cand[kChunk];
    __shared__ int n_val, n_cand;
    __shared__ float low, lse;
    __shared__ float4 joined[N / 64];
    const int tid = threadIdx.x, quad = tid >> 2, part = tid & 3;
    const int64_t n = blockIdx.x;
    const float *gm = a.group_max + n * a.group_stride;
    const int items = 1 << a.log2_items, at_once = (N / 4) >> a.log2_items;     // a pass scores N / 4 items
    const T *U = static_cast<const T *>(a.user) + n * a.dim, *I = static_cast<const T *>(a.item);
    for (int d = tid; d < a.dim; d += N) user[d] = (double)(float)U[d];
    float top = -INFINITY, most_abs = 0.f;
#pragma unroll 4
    for (int t = tid; t < a.groups; t += N) top = fmaxf(top, gm[t]);
#pragma unroll 4
    for (int t = tid; t < a.n_abs; t += N) most_abs = fmaxf(most_abs, a.tile_abs[t]);
#pragma unroll
    for (int o = 1; o < N / kSets; o *= 2) {
        top = fmaxf(top, __shfl_xor(top, o, 64));
        most_abs = fmaxf(most_abs, __shfl_xor(most_abs, o, 64));
    }
    if (tid % (N / kSets) == 0) { group_max[tid / (N / kSets)] = top; group_abs[tid / (N / kSets)] = most_abs; }
    if (tid == 0) { n_val = 0; n_cand = 0; low = -INFINITY; }
    const float4 share = join_shares<N>(join, n, tid);
    if (tid % 64 == 0) joined[tid / 64] = share;
    __syncthreads();
    if (tid >= N - 64) {
        const float l = finish_user(join, n, join_lanes<N / 64>(joined[tid % (N / 64)]), tid == N - 1);
        if (tid == N - 1) lse = l;
    }
    // the k-th largest of the maxima of 256 sets of groups: at least k groups reach it
    if (tid < kSets) {
        int rank = 0;
        top = group_max[tid];
#pragma unroll 8
        for (int i = 0; i < kSets; i += 4) {
            const float4 o = *reinterpret_cast<const float4 *>(group_max + i);
            rank += (o.x > top || (o.x == top && i < tid)) + (o.y > top || (o.y == top && i + 1 < tid)) +
                    (o.z > top || (o.z == top && i + 2 < tid)) + (o.w > top || (o.w == top && i + 3 < tid));
        }
        if (rank == a.k - 1) low = top;
    }
    // |user|, and the largest |element| of an item, by every wave for itself
    double norm = 0.0;
    for (int d = tid & 63; d < a.dim; d += 64) norm += user[d] * user[d];
    most_abs = fmaxf(fmaxf(group_abs[tid & 63], group_abs[(tid & 63) + 64]), fmaxf(group_abs[(tid & 63) + 128], group_abs[(tid & 63) + 192]));
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        norm += __shfl_xor(norm, o, 64);
        most_abs = fmaxf(most_abs, __shfl_xor(most_abs, o, 64));
    }
    __syncthreads();
    // |z - its product in the matrix cores| <= (terms) 2^-23 sum |user| |item|, sum |user| |item| <= |user| sqrt(dim) max |item|
    const double most = sqrt(norm) * sqrt((double)a.dim) * (double)most_abs * (double)a.scale;
    const double z_low = (double)low * (double)kLn2;
    const double margin = (6.0 * 256 + 16) * 0x1p-23 * most + 0x1p-20 * (fabs(z_low) + most);
    double thr = low > kFloor ? z_low - margin : -INFINITY;
    if (thr != thr) thr = -INFINITY;

    const auto better = [](double v, int32_t i, double w, int32_t j) { return v > w || (v == w && i < j); };
    // keeps the k best of the buffer, in order: by rank where there are few, by a bitonic sort else (6 users, the 64 best of 1082
    // items of 64 bf16: 114 us by rank)
    const auto compress = [&]() {
        __syncthreads();
        const int c = n_val;
        if (c <= 128) {
            for (int i = tid; i < c; i += N) {
                const double v = val[i];
                const int32_t at = id[i];
                int r = 0;
#pragma unroll 4
                for (int j = 0; j < c; ++j) r += better(val[j], id[j], v, at);
                if (r < a.k) { best_val[r] = v; best_id[r] = at; }
            }
        } else {
            int p = 256;
            while (p < c) p *= 2;                   // at most kBuf
            for (int i = c + tid; i < p; i += N) { val[i] = -INFINITY; id[i] = 0x7fffffff; }
            __syncthreads();
            for (int size = 2; size <= p; size *= 2)
                for (int step = size / 2; step; step /= 2) {
                    for (int t = tid; t < p / 2; t += N) {
                        const int i = 2 * t - (t & (step - 1)), j = i + step;
                        const double v = val[i], w = val[j];
                        const int32_t vi = id[i], wi = id[j];
                        if ((i & size) ? better(v, vi, w, wi) : better(w, wi, v, vi)) { val[i] = w; id[i] = wi; val[j] = v; id[j] = vi; }
                    }
                    __syncthreads();
                }
            if (tid < a.k) { best_val[tid] = val[tid]; best_id[tid] = id[tid]; }       // (k <= 64 < c)
        }
        __syncthreads();
        const int kept = min(c, a.k);
        if (tid < kept) { val[tid] = best_val[tid]; id[tid] = best_id[tid]; }
        if (tid == 0) n_val = kept;
        __syncthreads();
        if (kept == a.k && val[a.k - 1] > thr) thr = val[a.k - 1];
    };
    const float thr_tile = (float)(thr * (1.0 / (double)kLn2));
    const float thr_down = thr == -INFINITY ? -INFINITY : thr_tile - fabsf(thr_tile) * 0x1p-20f;
    for (int t0 = 0; t0 < a.groups; t0 += kChunk) {
        const int t1 = min(t0 + kChunk, a.groups);
#pragma unroll 4
        for (int t = t0 + tid; t < t1; t += N)
            if (!(gm[t] < thr_down)) cand[atomicAdd(&n_cand, 1)] = (uint16_t)(t - t0);
        __syncthreads();
        const int count = n_cand;
        // the buffer takes 512 items between two looks at it
        for (int c0 = 0; c0 < count; c0 += kPasses * at_once) {
            for (int c = c0 + (quad >> a.log2_items); c < min(c0 + kPasses * at_once, count); c += at_once) {
                const int64_t j = (((int64_t)t0 + cand[c]) << a.log2_items) + (quad & (items - 1));
                const float b = j < a.n_items && a.bias ? a.bias[j] : 0.f;
                const bool in = j < a.n_items && !(b < kOffer);
                const T *row = I + (in ? j : 0) * a.dim;
                double dot = 0.0;
                int d = part * E;
                if (a.vector)
                    for (; d < a.dim; d += 8 * E) {                    // (whole pieces of 16 bytes; two are on their way at once)
                        const bool more = d + 4 * E < a.dim;
                        const int d2 = more ? d + 4 * E : d;
                        T v[E], w[E];
                        __builtin_memcpy(v, row + d, 16);
                        __builtin_memcpy(w, row + d2, 16);
                        double second = 0.0;
#pragma unroll
                        for (int k = 0; k < E; ++k) {
                            dot += user[d + k] * (double)(float)v[k];
                            second += user[d2 + k] * (double)(float)w[k];
                        }
                        if (more) dot += second;
                    }
                for (; d < a.dim; d += 4 * E)
                    for (int k = 0; k < E && d + k < a.dim; ++k) dot += user[d + k] * (double)(float)row[d + k];
                dot += __shfl_xor(dot, 1, 64);
                dot += __shfl_xor(dot, 2, 64);
                const double z = dot * (double)a.scale + (double)b;
                if (part == 0 && in && z >= thr && z > -INFINITY) {
                    const int at = atomicAdd(&n_val, 1);
                    val[at] = z;
                    id[at] = (int32_t)j;
                }
            }
            __syncthreads();
            const bool full = n_val > kBuf - 512;
            __syncthreads();                        // everybody has looked before anybody adds
            if (full) compress();
        }
        __syncthreads();
        if (tid == 0) n_cand = 0;
        __syncthreads();
    }
    compress();
    if (tid < a.k) {
        const bool has = tid < n_val;
        a.top_log_prob[n * a.k + tid] = has ? (float)(val[tid] - (double)lse) : -INFINITY;
        a.top_ids[n * a.k + tid] = has ? id[tid] : -1;
    }
}

// Groups of a user, to a multiple of four.
int64_t group_stride_of(int64_t n_items, int top) { return (tiles_of(n_items) * (32 / top) + 3) / 4 * 4; }

constexpr int64_t kBlocks = 1024;                   // blocks a launch is cut into: four waves per SIMD

// Whether a block has all users at once and the tables stay as they are (this against laid-out tables; the border of users lies at
// two tiles of them, for up to 16384 items at the four that a block's waves hold): rows of 32 fp32, 64 users 9.3 us and 12.7 for 16 000
// items, 11.5 and 14.6 for 32 000, 128 users 11.8 and 12.8, 17.8 and 14.7; rows of 64 bf16, 64 users 9.8 and 11.9, 12.2 and 13.4, 128 users
// 12.6 and 12.1, 19.5 and 13.6.  Wide rows are fetched in pieces of lines and pay only for few users where fp32 would be laid out as
// three pieces (32 000 items of 128 fp32: 32 users 16.4 us and 25.9, 64 users 28.0 and 26.6; 73 000 of 200: 5 users 60 and 75; of 256
// bf16: 46 and 37).
inline bool few_users(int64_t n_users, int64_t n_items, int dim, int dtype) {
    if (dim > 64) return n_users <= 32 && dtype == GS_F32;
    return n_users <= 64 || (n_users <= 128 && n_items <= 16384);
}

// How a call is cut: users in slices that bound the table of tile maxima, a slice in waves.
struct Cut {
    int64_t slice;                                  // users per slice
    int of, top;                                    // top: items per group whose largest score is kept, 0 for none
};

Cut cut_of(int64_t n_users, int64_t n_items, int dim, int dtype, int top_k) {
    Cut c;
    const int regs = pieces_of(dtype) * blocks_of(dim);                   // registers of a fragment row: 8 each
    // two tiles of users a wave halve the reads of the items where the pairs still fill the chip (4096 users, 100 000 items of
    // 64 bf16: 126 us, 133 with one; 512 users of fp32: 64 us, 68) and leave it idle where they do not (1024 users and items: 17 us,
    // 14 with one; 64 users: 30 us, 26)
    constexpr int W = gs::kCatThreads / 64;
    c.of = regs <= 8 && tiles_of(n_users) / (2 * W) * (tiles_of(n_items) / 4) >= kBlocks ? 2 : 1;
    c.slice = n_users;
    c.top = 0;
    if (top_k > 0) {
        // What a user costs beside the product: the groups' maxima, written and read, and about k groups of rows read again
        // (out of L2: half the price).  Groups of 4 for few items, wide rows or long lists (3196 users, 4036 items of 200 fp32, 64
        // best: 185 us, 540 with groups of 32), of 32 else (512 users, 100 000 items of 64 fp32, 20 best: 100 us, 142 with groups of 4).
        const auto cost = [&](double group) { return 8.0 * n_items / group + 0.5 * top_k * group * dim * dtype_size(dtype); };
        c.top = cost(4) < cost(32) ? 4 : 32;
        const int64_t most = ((int64_t)1 << 26) / (group_stride_of(n_items, c.top) + 1) / 256 * 256;
        // (256 threads a user in the launch of the best items)
        c.slice = std::min({n_users, std::max<int64_t>(most, 256), gs::kMostThreads / 256});
    }
    return c;
}

void shares_of(int64_t users, int64_t n_items, int of, int *group_blocks, int *shares, int *per_share) {
    constexpr int W = gs::kCatThreads / 64;
    const int64_t ut = tiles_of(users), it = tiles_of(n_items);
    *group_blocks = (int)((ut + of * W - 1) / (of * W));
    int64_t sh = kBlocks / *group_blocks;
    if (sh > (it + 3) / 4) sh = (it + 3) / 4;
    if (sh < 1) sh = 1;
    *per_share = it ? (int)((it + sh - 1) / sh + 3) / 4 * 4 : 4;       // (tile maxima leave by fours)
    *shares = (int)((it + *per_share - 1) / *per_share);
}

struct Space {
    size_t user, item, bias2, part, tile_abs, group_max, total;
};

Space space_of(int64_t n_users, int64_t n_items, int dim, int dtype, int top_k) {
    Space s;
    const Cut c = cut_of(n_users, n_items, dim, dtype, top_k);
    int blocks, shares, per;
    shares_of(c.slice, n_items, c.of, &blocks, &shares, &per);
    size_t off = 0;
    const bool few = few_users(n_users, n_items, dim, dtype);        // lays nothing out
    s.user = off; off += few ? 0 : align256(layout_bytes(c.slice, dim, dtype));
    s.item = off; off += few ? 0 : align256(layout_bytes(n_items, dim, dtype));
    s.bias2 = off; off += few ? 0 : align256((size_t)tiles_of(n_items) * 32 * sizeof(float));
    s.part = off;
    // the last slice may be smaller and have more shares: the product of both is bounded by the blocks' users
    off += align256((few ? (size_t)(n_users * kBlocks) : (size_t)(c.slice * (int64_t)shares + kBlocks * 256)) * sizeof(float4));
    s.tile_abs = off;
    if (top_k > 0) off += align256((size_t)tiles_of(n_items) * sizeof(float));
    s.group_max = off;
    if (top_k > 0) off += (size_t)c.slice * group_stride_of(n_items, c.top) * sizeof(float);
    s.total = off;
    return s;
}

template <int P, int DB, int OF, int TOP>
int launch_one(const FwdArgs &a, hipStream_t stream) {
    constexpr int F = 2 * DB * P, lds = 2 * F * gs::tiles_per_stage(F) * 1024;
    static_assert(gs::fits_lds(F), "a tile does not fit");
    const auto kernel = catalog_fwd_kernel<P, DB, OF, TOP>;
    if (lds > 64 * 1024) {
        const hipError_t e = gs::raise_lds_limit(reinterpret_cast<const void *>(kernel), lds);
        if (e != hipSuccess) return gs::fail(GS_ELAUNCH, "gs_catalog_fwd: LDS limit: %s", hipGetErrorString(e));
    }
    kernel<<<dim3((unsigned)((int64_t)a.group_blocks * a.shares)), kCatThreads, lds, stream>>>(a);
    return gs::check_launch("gs_catalog_fwd");
}

template <int P, int DB, int OF>
int launch_tile(const FwdArgs &a, int top, hipStream_t stream) {
    return top == 32 ? launch_one<P, DB, OF, 32>(a, stream) : top == 4 ? launch_one<P, DB, OF, 4>(a, stream) : launch_one<P, DB, OF, 0>(a, stream);
}

template <int P>
int launch_fwd(const FwdArgs &a, int blocks, int of, int top, hipStream_t stream) {
    if (of == 2) {
        if (blocks == 1) return launch_tile<P, 1, 2>(a, top, stream);
        if (blocks == 2) return launch_tile<P, 2, 2>(a, top, stream);
        if constexpr (P * 4 <= 8) {
            if (blocks == 4) return launch_tile<P, 4, 2>(a, top, stream);
        }
        if constexpr (P == 1) return launch_tile<P, 8, 2>(a, top, stream);
    }
    if (blocks == 1) return launch_tile<P, 1, 1>(a, top, stream);
    if (blocks == 2) return launch_tile<P, 2, 1>(a, top, stream);
    if (blocks == 4) return launch_tile<P, 4, 1>(a, top, stream);
    return launch_tile<P, 8, 1>(a, top, stream);
}

template <class T, int TOP>
int launch_few(const FewArgs &a, int shares, hipStream_t stream) {
    const int blocks = gs::blocks_of(a.dim);
    const dim3 grid((unsigned)shares);
    if (blocks == 1) catalog_few_kernel<T, 1, TOP><<<grid, kCatThreads, 0, stream>>>(a);
    else if (blocks == 2) catalog_few_kernel<T, 2, TOP><<<grid, kCatThreads, 0, stream>>>(a);
    if constexpr (Pieces<T>::P == 3) {              // (wider rows: few_users)
        if (blocks == 4) catalog_few_kernel<T, 4, TOP><<<grid, kCatThreads, 0, stream>>>(a);
        else if (blocks == 8) catalog_few_kernel<T, 8, TOP><<<grid, kCatThreads, 0, stream>>>(a);
    }
    return gs::check_launch("gs_catalog_fwd");
}

template <class T>
int run_few(const FewArgs &a, int shares, int top, hipStream_t stream) {
    return top == 32 ? launch_few<T, 32>(a, shares, stream) : top == 4 ? launch_few<T, 4>(a, shares, stream) : launch_few<T, 0>(a, shares, stream);
}

// 1024 threads a user while there is a block for every compute unit (256 users, 100 000 items of 64 fp32, 20 best: 67 us, 75 with 256),
// 256 else (512 users: 94 us, 104 with 1024; 2000 users, 20 000 items of bf16: 101 us, 180).
template <class T>
int run_top(const TopArgs &t, const JoinArgs &j, hipStream_t stream) {
    if (t.n_users <= 256) catalog_top_kernel<T, 1024><<<dim3((unsigned)t.n_users), 1024, 0, stream>>>(t, j);
    else catalog_top_kernel<T, 256><<<dim3((unsigned)t.n_users), 256, 0, stream>>>(t, j);
    return gs::check_launch("gs_catalog_fwd (best items)");
}

}  // namespace

extern "C" size_t gs_catalog_workspace(int64_t n_users, int64_t n_items, int dim, int dtype, int top_k) {
    if (gs::check_catalog("gs_catalog_workspace", n_users, n_items, dim, dtype, 1.f)) return 0;
    if (top_k < 0 || top_k > kMaxTop) { gs::fail(GS_ELIMIT, "gs_catalog_workspace: top_k=%d (at most %d)", top_k, kMaxTop); return 0; }
    if (n_users == 0) return 0;
    return space_of(n_users, n_items, dim, dtype, top_k).total;
}

extern "C" int gs_catalog_fwd(const void *user, int64_t n_users, const void *item, int64_t n_items, int dim, int dtype,
                              const float *bias, float scale, const int32_t *targets, float *log_prob, float *entropy,
                              float *lse, int top_k, float *top_log_prob, int32_t *top_ids, void *workspace,
                              size_t workspace_bytes, void *stream) {
    const char *what = "gs_catalog_fwd";
    if (int rc = gs::check_catalog(what, n_users, n_items, dim, dtype, scale)) return rc;
    if (top_k < 0) return gs::fail(GS_EINVAL, "%s: top_k=%d", what, top_k);
    if (top_k > kMaxTop) return gs::fail(GS_ELIMIT, "%s: top_k=%d (at most %d)", what, top_k, kMaxTop);
    if (n_users == 0) return GS_OK;
    if (!user || (n_items && !item) || (top_k && (!top_log_prob || !top_ids)))
        return gs::fail(GS_EINVAL, "%s: null pointer argument", what);
    const int size = gs::dtype_size(dtype);
    if (((uintptr_t)user | (uintptr_t)item) & (size - 1)) return gs::fail(GS_EINVAL, "%s: pointer not aligned to its element", what);
    const Space sp = space_of(n_users, n_items, dim, dtype, top_k);
    if (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < sp.total)
        return gs::fail(GS_EINVAL, "%s: 256-byte aligned workspace of %zu bytes needed, %zu given", what, sp.total, workspace_bytes);
    const Cut cut = cut_of(n_users, n_items, dim, dtype, top_k);
    char *ws = static_cast<char *>(workspace);
    hipStream_t s = (hipStream_t)stream;
    const int blocks = gs::blocks_of(dim), pieces = gs::pieces_of(dtype);
    float *tile_abs = top_k ? reinterpret_cast<float *>(ws + sp.tile_abs) : nullptr;
    const int vector = ((uintptr_t)item & 15) == 0 && (dim * size) % 16 == 0;
    for (int64_t u0 = 0; u0 < n_users; u0 += cut.slice) {
        const int64_t nu = n_users - u0 < cut.slice ? n_users - u0 : cut.slice;
        const void *users = static_cast<const char *>(user) + (size_t)u0 * dim * size;
        const int32_t *aims = targets ? targets + u0 : nullptr;
        float4 *part = reinterpret_cast<float4 *>(ws + sp.part);
        float *group_max = top_k ? reinterpret_cast<float *>(ws + sp.group_max) : nullptr;
        const int64_t group_stride = top_k ? group_stride_of(n_items, cut.top) : 0;
        const int item_tiles = (int)gs::tiles_of(n_items);
        int shares = 0, n_abs = item_tiles;
        if (few_users(n_users, n_items, dim, dtype)) {
            const int user_tiles = (int)gs::tiles_of(nu), at_once = user_tiles == 1 ? 4 : user_tiles == 2 ? 2 : 1;
            const int all = (item_tiles + at_once - 1) / at_once;
            shares = all < kBlocks ? all : (int)kBlocks;
            n_abs = shares;
            const FewArgs f{users, item, bias, aims, part, group_max, tile_abs, group_stride, n_items, (int)nu, dim, item_tiles, scale * gs::kLog2e};
            if (shares)
                if (int rc = dtype == GS_F32 ? run_few<float>(f, shares, cut.top, s) : dtype == GS_BF16 ? run_few<__bf16>(f, shares, cut.top, s)
                                                                                     : run_few<_Float16>(f, shares, cut.top, s))
                    return rc;
        } else {
            gs::Layout lu{}, li{};
            lu.x = users;
            lu.n_rows = nu;
            lu.rows = reinterpret_cast<uint4 *>(ws + sp.user);
            if (u0 == 0) {
                li.x = item; li.n_rows = n_items; li.bias = bias;
                li.rows = reinterpret_cast<uint4 *>(ws + sp.item);
                li.bias2 = reinterpret_cast<float *>(ws + sp.bias2);
                li.tile_abs = tile_abs;
            }
            if (int rc = gs::launch_layouts(lu, li, dim, dtype, s)) return rc;
            FwdArgs a;
            a.user = lu.rows;
            a.item = reinterpret_cast<const uint4 *>(ws + sp.item);
            a.bias2 = reinterpret_cast<const float *>(ws + sp.bias2);
            a.targets = aims;
            a.part = part;
            a.group_max = group_max;
            a.group_stride = group_stride;
            a.n_users = nu; a.n_items = n_items;
            a.user_tiles = (int)gs::tiles_of(nu); a.item_tiles = item_tiles;
            shares_of(nu, n_items, cut.of, &a.group_blocks, &a.shares, &a.tiles_per_share);
            a.scale2 = scale * gs::kLog2e;
            if (n_items) {
                shares = a.shares;
                if (int rc = pieces == 1 ? launch_fwd<1>(a, blocks, cut.of, cut.top, s) : pieces == 2 ? launch_fwd<2>(a, blocks, cut.of, cut.top, s)
                                                                                            : launch_fwd<3>(a, blocks, cut.of, cut.top, s))
                    return rc;
            }
        }
        const JoinArgs j{part, shares, n_items, aims, log_prob ? log_prob + u0 : nullptr, entropy ? entropy + u0 : nullptr, lse ? lse + u0 : nullptr};
        if (!top_k) {
            constexpr int64_t most = gs::kMostThreads / 64;
            for (int64_t n = 0; n < nu; n += most) {
                const int64_t users_now = std::min(most, nu - n);
                catalog_join_kernel<<<dim3((unsigned)((users_now + 3) / 4)), gs::kCatThreads, 0, s>>>(j, n, nu);
                if (int rc = gs::check_launch("gs_catalog_fwd (join)")) return rc;
            }
            continue;
        }
        TopArgs t;
        t.user = users; t.item = item; t.bias = bias; t.group_max = group_max; t.tile_abs = tile_abs;
        t.n_users = nu; t.n_items = n_items; t.group_stride = group_stride; t.dim = dim; t.n_abs = n_abs;
        t.groups = item_tiles * (32 / cut.top); t.log2_items = cut.top == 4 ? 2 : 5; t.k = top_k;
        t.vector = vector;
        t.scale = scale; t.top_log_prob = top_log_prob + u0 * top_k; t.top_ids = top_ids + u0 * top_k;
        if (int rc = dtype == GS_F32 ? run_top<float>(t, j, s) : dtype == GS_BF16 ? run_top<__bf16>(t, j, s) : run_top<_Float16>(t, j, s))
            return rc;
    }
    return GS_OK;
}
