// Users against a catalog of items: operand layout and tile product, shared by the forward and backward kernels.
//
// The scores z = scale <user, item> + bias are a matrix product whose result is only ever reduced, so it stays in
// registers.  All table types run on the bf16 matrix instruction (v_mfma_f32_32x32x16_bf16, fp32 accumulators): an element
// is cut into pieces, each the bf16 nearest to what the ones before leave, whose sum it is exactly -- one piece for bf16,
// two for fp16, three for fp32 -- and the products (exact in fp32) of pieces i and k with i + k <= 2 are added, smallest
// first.  Piece i is at most 2^-8i of the element, so what is left out is below 2^-23 of |user| |item|, the size of
// one fp32 rounding.
//
// Operands are laid out once per call in the order in which lanes use them (one kilobyte per fragment, 16 bytes a
// lane), rows padded to 32, elements to a multiple of 32, with zeros:
//   rows layout   fragment (tile, kc, piece): lane l holds row 32 tile + (l & 31), elements 16 kc + 8 (l >> 5) + 0..7
//   cols layout   fragment (tile, t, db, piece): lane l holds element 32 db + (l & 31) of rows
//                 32 tile + 16 t + 8 (i >> 2) + 4 (l >> 5) + (i & 3), i = 0..7
// The product of two row fragments puts the wave's own row (l & 31) in the lane and the streamed row 8 (r >> 2) +
// 4 (l >> 5) + (r & 3) in register r: a lane keeps its own row's running maximum and sum without talking to other lanes, and
// eight registers of it ARE the operand of the next product (gradient times streamed rows) whose other operand is a
// cols fragment -- that is the order of rows inside one.
//
// An item whose bias is below kOffer is not on offer: its row is laid out as zeros (whatever it holds) and its score
// becomes kMasked, far below kFloor where every running maximum starts, so that its exponential is an exact zero.
#pragma once

#include "ops_common.h"

namespace gs {

constexpr float kOffer = -1e10f;
constexpr float kFloor = -1e12f;                    // in units of log 2, as all scores in the kernels
constexpr float kMasked = -1e14f;
constexpr int kCatThreads = 256;
// A dispatch has fewer than 2^32 threads along x: kernels of a block per few rows or elements are started in parts.
constexpr int64_t kMostThreads = (int64_t)1 << 31;

using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f32x16 = __attribute__((ext_vector_type(16))) float;

template <class T> struct Pieces;
template <> struct Pieces<__bf16>   { static constexpr int P = 1; };
template <> struct Pieces<_Float16> { static constexpr int P = 2; };
template <> struct Pieces<float>    { static constexpr int P = 3; };
inline int pieces_of(int dtype) { return dtype == GS_F32 ? 3 : dtype == GS_F16 ? 2 : 1; }

// Blocks of 32 elements a row is padded to: 1, 2, 4 or 8.
inline int blocks_of(int dim) { return dim <= 32 ? 1 : dim <= 64 ? 2 : dim <= 128 ? 4 : 8; }
inline int64_t tiles_of(int64_t rows) { return (rows + 31) / 32; }
inline size_t layout_bytes(int64_t rows, int dim, int dtype) { return (size_t)tiles_of(rows) * 2 * blocks_of(dim) * pieces_of(dtype) * 1024; }

// Row in a tile of register r of a lane.
__device__ __forceinline__ int row_of_reg(int r, int lane) { return 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3); }

using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;

// The bf16 nearest to lo (lower half) and hi; both become what it leaves of them.
__device__ __forceinline__ uint32_t next_piece(float &lo, float &hi) {
    const bf16x2 v = {(__bf16)lo, (__bf16)hi};
    const uint32_t w = __builtin_bit_cast(uint32_t, v);
    lo -= __uint_as_float(w << 16);
    hi -= __uint_as_float(w & 0xFFFF0000u);
    return w;
}

// Eight floats cut into NZ pieces.
template <int NZ> __device__ __forceinline__ void cut_pieces(float *v, bf16x8 *z) {
#pragma unroll
    for (int p = 0; p < NZ; ++p) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = next_piece(v[2 * i], v[2 * i + 1]);
        z[p] = __builtin_bit_cast(bf16x8, *reinterpret_cast<uint4 *>(w));
    }
}

template <int P> struct Fragment { bf16x8 p[P]; };

// Waves per SIMD a kernel is compiled for: two where its operands leave room in 256 registers (the matrix results then
// stay in the registers the vector ALU reads), else one.
constexpr int waves_for(int registers) { return registers <= 160 ? 2 : 1; }

// The four waves of a block own neighboring rows and stream the same tiles, which therefore pass through LDS: loads that
// write LDS directly fill one half of it while the waves work on the other (a wave reading its fragments itself was
// measured at 626 us for 4096 users and 100 000 items of 64 bf16, forward and backward, bound by 7 TB/s out of L2).
// `fragments`: kilobytes of a tile; tiles per half so that a barrier is worth it.
constexpr int tiles_per_stage(int fragments) { return fragments <= 4 ? 4 : fragments <= 12 ? 2 : 1; }
constexpr bool fits_lds(int fragments) { return 2 * fragments * tiles_per_stage(fragments) <= 152; }

// One fragment into LDS at byte offset dst; both the same in all lanes.  Done when vmcnt says so.
__device__ __forceinline__ void fragment_to_lds(const uint4 *src, int lane, uint32_t dst) {
    const unsigned long long from = reinterpret_cast<unsigned long long>(src + lane);
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(from), "s"(dst) : "memory");
}
// This wave's loads into LDS have arrived, and then everybody's.
__device__ __forceinline__ void stage_ready() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// frag: the first fragment of a tile, the same in all lanes.
template <int P>
__device__ __forceinline__ Fragment<P> load_fragment(const uint4 *frag, int index, int lane) {
    Fragment<P> f;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const uint4 v = frag[(index * P + i) * 64 + lane];
        f.p[i] = *reinterpret_cast<const bf16x8 *>(&v);
    }
    return f;
}

// acc += a b over the pieces whose product counts.
template <int PA, int PB, int MOST>
__device__ __forceinline__ void multiply(f32x16 &acc, const bf16x8 *a, const bf16x8 *b) {
#pragma unroll
    for (int w = MOST; w >= 0; --w)
#pragma unroll
        for (int i = PA - 1; i >= 0; --i)
            if (w - i >= 0 && w - i < PB) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[w - i], acc, 0, 0, 0);
}

__device__ __forceinline__ float half_max(float v) {           // the larger of lane l's and lane l ^ 32's
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    return fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
}

// What the backward kernels need of 32 users, as one more fragment of their tile (catalog_bwd.hip).
struct alignas(16) Stats {
    float lse2[32], a[32], b2[32], g[32];
    int32_t target[32];
    float unused[96];                               // (a fragment is a kilobyte)
};
struct StatsFrom {
    int64_t n_items;
    const int32_t *targets;
    const float *lse, *entropy, *g_log_prob, *g_entropy;
};

struct Layout {                                     // one table to lay out
    const void *x;
    int64_t n_rows;
    const float *bias;                              // nullable
    uint4 *rows, *cols;                             // nullable
    float *bias2;                                   // nullable: bias in units of log 2, or kMasked
    float *tile_abs;                                // nullable: the largest |element| of every tile
    Stats *stats;                                   // nullable
    StatsFrom from;
};

// Lays out two tables in one launch.
int launch_layouts(const Layout &first, const Layout &second, int dim, int dtype, hipStream_t stream);
int check_catalog(const char *what, int64_t n_users, int64_t n_items, int dim, int dtype, float scale);

}  // namespace gs
