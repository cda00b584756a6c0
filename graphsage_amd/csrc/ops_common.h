// Element types of the operators in gsage_ops.h, and small cross-lane helpers.
#pragma once

#include "gs_common.h"
#include "gsage_ops.h"

namespace gs {

template <class T> struct Pack;                     // 16 bytes of a table row
template <> struct Pack<float>    { static constexpr int E = 4; };
template <> struct Pack<__bf16>   { static constexpr int E = 8; };
template <> struct Pack<_Float16> { static constexpr int E = 8; };

inline int dtype_size(int dtype) { return dtype == GS_F32 ? 4 : dtype == GS_BF16 || dtype == GS_F16 ? 2 : 0; }

// Sum over the L lanes (a power of two, aligned in the wave) that share a row; every lane gets it, the same bits in
// each.  The first four steps are data-parallel primitives of the vector ALU, the last two the half- and quarter-wave
// swaps: none goes through LDS.
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
template <int L> __device__ __forceinline__ float lanes_sum(float v) {
    if (L > 1) v += dpp<0xB1>(v);                   // quad_perm 1 0 3 2
    if (L > 2) v += dpp<0x4E>(v);                   // quad_perm 2 3 0 1
    if (L > 4) v += dpp<0x141>(v);                  // row_half_mirror
    if (L > 8) v += dpp<0x140>(v);                  // row_mirror
    if (L > 16) {
        auto r = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
        v = __int_as_float(r[0]) + __int_as_float(r[1]);
    }
    if (L > 32) {
        auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
        v = __int_as_float(r[0]) + __int_as_float(r[1]);
    }
    return v;
}

// exp2 and log2 of the hardware (1 ulp; results below 2^-126 are zeros).
__device__ __forceinline__ float fast_exp2(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float fast_log2(float v) { return __builtin_amdgcn_logf(v); }
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

inline size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

}  // namespace gs
