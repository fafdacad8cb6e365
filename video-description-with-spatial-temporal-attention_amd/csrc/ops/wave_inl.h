// Reductions and scans over a wave of 64 on the vector pipe.  Lanes meet by DPP moves, a few cycles a step; by LDS permutes, a dependent
// one (two for 64 bits) a step, the sum of a 64-bit value took longer than reading and adding 512 words.
#pragma once
#include <hip/hip_runtime.h>

namespace stattn {

// `v` as DPP moves it; lanes without a source, and rows outside the mask ROWS, get `old`
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_move(float old, float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, old), __builtin_bit_cast(int, v), CTRL, ROWS, 0xF, false));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_move(double old, double v) {
    const int2 o = __builtin_bit_cast(int2, old), x = __builtin_bit_cast(int2, v);
    return __builtin_bit_cast(double, make_int2(__builtin_amdgcn_update_dpp(o.x, x.x, CTRL, ROWS, 0xF, false), __builtin_amdgcn_update_dpp(o.y, x.y, CTRL, ROWS, 0xF, false)));
}
// lane `from`'s value in every lane; `from` is the same in all of them
__device__ __forceinline__ float from_lane(float v, int from) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), from)); }
__device__ __forceinline__ int from_lane(int v, int from) { return __builtin_amdgcn_readlane(v, from); }
template <class T>
__device__ __forceinline__ T from_lane(T v, int from) {
    static_assert(sizeof(T) == 8, "four or eight bytes");
    const int2 x = __builtin_bit_cast(int2, v);
    return __builtin_bit_cast(T, make_int2(__builtin_amdgcn_readlane(x.x, from), __builtin_amdgcn_readlane(x.y, from)));
}

// join(v of all lanes), in all lanes; `none` joins as nothing (0 of a sum, -inf of a maximum).  All lanes take part.
template <class T, class F>
__device__ __forceinline__ T wave_join(T v, T none, F join) {
    v = join(v, dpp_move<0xB1, 0xF>(v, v));         // quad_perm [1, 0, 3, 2]
    v = join(v, dpp_move<0x4E, 0xF>(v, v));         // quad_perm [2, 3, 0, 1]
    v = join(v, dpp_move<0x141, 0xF>(v, v));        // row_half_mirror: every lane has its eight
    v = join(v, dpp_move<0x140, 0xF>(v, v));        // row_mirror: its row of sixteen
    v = join(v, dpp_move<0x142, 0xA>(none, v));     // row_bcast 15: rows 1 and 3 add the row before
    v = join(v, dpp_move<0x143, 0xC>(none, v));     // row_bcast 31: row 3 adds the first half; lane 63 has all
    return from_lane(v, 63);
}
template <class T>
__device__ __forceinline__ T wave_sum(T v) { return wave_join(v, (T)0, [](T a, T b) { return a + b; }); }
__device__ __forceinline__ float wave_max(float v) { return wave_join(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); }); }
// sum over the lanes up to and with this one.  All lanes take part.
__device__ __forceinline__ double wave_scan(double v) {
    v += dpp_move<0x111, 0xF>(0.0, v);              // row_shr 1, 2, 4, 8: within the row of sixteen
    v += dpp_move<0x112, 0xF>(0.0, v);
    v += dpp_move<0x114, 0xF>(0.0, v);
    v += dpp_move<0x118, 0xF>(0.0, v);
    v += dpp_move<0x142, 0xA>(0.0, v);              // the rows' totals, as above
    v += dpp_move<0x143, 0xC>(0.0, v);
    return v;
}

}  // namespace stattn
