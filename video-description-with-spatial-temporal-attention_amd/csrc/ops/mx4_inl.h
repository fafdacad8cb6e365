// Device pieces of the 4-bit operators: element types, the block scale, the code conversions of gfx950.
#pragma once
#include "ops.h"

#if defined(__HIP_DEVICE_COMPILE__) && !defined(__gfx950__)
#error "libstattn is written for gfx950 (MI355X / CDNA4) only"
#endif

namespace stattn {

typedef int i32x4v __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef float f32x16v __attribute__((ext_vector_type(16)));

template <OpType T> struct Elem;
template <> struct Elem<OP_F32> { typedef float type; };
template <> struct Elem<OP_BF16> { typedef __bf16 type; };
template <> struct Elem<OP_F16> { typedef _Float16 type; };

__device__ __forceinline__ unsigned abs_bits(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

// Scale byte of a block whose largest magnitude has the fp32 bits `a` (compared as integers a NaN is the largest of all):
// floor(log2) is the exponent field, the largest code's exponent is 2.  2^-126 is the smallest scale, 255 (NaN) marks a block that
// holds an infinity or NaN, a block of zeros gets 1.
__device__ __forceinline__ unsigned mx4_scale_byte(unsigned a) {
    const unsigned e = a >> 23;
    return e == 255u ? 255u : a == 0u ? 127u : e > 3u ? e - 2u : 1u;
}
// eight values -> eight codes in one word.  v_cvt_scalef32_pk_fp4_f32 divides by the scale's power of two, rounds to nearest even and
// saturates at 6; a NaN block is written as zeros under its NaN scale.
__device__ __forceinline__ unsigned mx4_codes8(const float* v, unsigned byte) {
    const float s = __builtin_bit_cast(float, byte << 23);
    unsigned c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], s, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], s, 3);
    return byte == 255u ? 0u : c;
}
// the largest of four neighbouring lanes (a quad), in each of them
__device__ __forceinline__ unsigned quad_max(unsigned v) {
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));     // quad_perm [1, 0, 3, 2]
    return max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));  // quad_perm [2, 3, 0, 1]
}
__device__ __forceinline__ unsigned top8(const float* v) {
    unsigned t = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) t = max(t, abs_bits(v[j]));
    return t;
}
// Eight neighbouring elements as they lie in memory: `take` requests them and `put` turns them into floats, so that a caller can have
// several requests on their way.  Elements from number n on are not there and become 0.  Any address will do: 16-byte loads need no more
// than an element's alignment here (a row of odd length costs what an even one does); only a row's last, partial eight go one by one.
template <OpType T>
struct Eight {
    typedef typename Elem<T>::type E;
    typedef E vec __attribute__((ext_vector_type(16 / sizeof(E)), aligned(sizeof(E))));
    static constexpr int PARTS = sizeof(E) / 2, PER = 16 / sizeof(E);
    vec raw[PARTS];
    __device__ __forceinline__ void take(const E* x, int n) {
        if (n >= 8) {
#pragma unroll
            for (int j = 0; j < PARTS; ++j) raw[j] = reinterpret_cast<const vec*>(x)[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) raw[j / PER][j % PER] = j < n ? x[j] : (E)0.f;
        }
    }
    __device__ __forceinline__ void put(float* v) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)raw[j / PER][j % PER];
    }
};
// the fp32 value of a scale byte (0 is 2^-127, a subnormal; 255 is NaN)
__device__ __forceinline__ float mx4_scale(unsigned byte) {
    return __builtin_bit_cast(float, byte == 255u ? 0x7fc00000u : byte == 0u ? 0x00400000u : byte << 23);
}

}  // namespace stattn
