// Writing matrices in microscaled 4 bits and reading them back.  Both are bound by memory: 4 (2) bytes an element on one side, 17 / 32 on
// the other.  13312 x 4096 in bf16, 138 MB: written in 21.5 us, read back in 22.6 (6.4 and 6.1 TB/s, the 4-bit side staying in the caches; a
// 1 GiB copy reaches 5.1); in fp32, 247 MB, 37.6 and 38.8.
#include "mx4_inl.h"

namespace stattn {

// x row-major.  A lane takes eight columns (one or two 16-byte loads) and writes the word of their codes, so a wave reads and writes
// whole lines; the four lanes of a block find its scale by two moves inside the quad.  (A lane per block, 32 columns each, read lines in
// eight or four pieces: 13312 x 4096 in bf16 took 125 us.)
template <OpType T>
__global__ __launch_bounds__(256) void mx4_quantize_rows_kernel(Mx4QuantArgs a, unsigned words, int64_t n) {
    typedef typename Elem<T>::type E;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {      // n and the steps are multiples of 4
        const int64_t r = n >> 32 ? i / words : (int64_t)((unsigned)i / words);
        const int c = (int)(i - r * words) * 8;
        Eight<T> x;
        float v[8];
        x.take(static_cast<const E*>(a.x) + r * a.row_stride + c, (int)(a.cols - c));
        x.put(v);
        const unsigned byte = mx4_scale_byte(quad_max(top8(v)));
        reinterpret_cast<unsigned*>(a.codes)[i] = mx4_codes8(v, byte);
        if ((threadIdx.x & 3) == 0) a.scales[i >> 2] = (uint8_t)byte;
    }
}

// x column-major (the rows of the form are neighbours in memory), and any other pair of strides.  A workgroup takes 64 rows x 128 columns
// of the form: a lane reads the 32 values of a block down its row, 64 lanes side by side; the 16-byte blocks meet in LDS, from where each
// row's 64 bytes leave together.  A 512 x 12000 weight in fp32: 4.9 us.
// Where neither stride is 1, neighbouring lanes read different lines (every second column of 13312 x 8192: 154 us in fp32, 116 in bf16, a copy
// into rows and its form 152 and 77; every second column of 512 x 24000, rows as here: 9.9 and 6.5).
template <OpType T>
__global__ __launch_bounds__(256) void mx4_quantize_cols_kernel(Mx4QuantArgs a, unsigned row_tiles, unsigned kp128) {
    typedef typename Elem<T>::type E;
    __shared__ uint4 code[64][5];                    // a row's four blocks, one slot apart from the next row's banks
    __shared__ unsigned scale[64];                   // a row's four scale bytes
    const int lane = threadIdx.x & 63, blk = threadIdx.x >> 6;
    for (int64_t t = blockIdx.x; t < (int64_t)row_tiles * kp128; t += gridDim.x) {
        const int64_t r0 = t % row_tiles * 64, c0 = t / row_tiles * 128, r = r0 + lane, c = c0 + blk * 32;
        float v[32];
        const E* x = static_cast<const E*>(a.x) + r * a.row_stride + c * a.col_stride;
        const int here = r < a.rows ? (int)max(min(a.cols - c, (int64_t)32), (int64_t)0) : 0;
        if (here == 32) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = (float)x[j * a.col_stride];
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = j < here ? (float)x[j * a.col_stride] : 0.f;
        }
        const unsigned byte = mx4_scale_byte(max(max(top8(v), top8(v + 8)), max(top8(v + 16), top8(v + 24))));
        code[lane][blk] = make_uint4(mx4_codes8(v, byte), mx4_codes8(v + 8, byte), mx4_codes8(v + 16, byte), mx4_codes8(v + 24, byte));
        reinterpret_cast<uint8_t*>(&scale[lane])[blk] = (uint8_t)byte;
        __syncthreads();
        const int64_t ro = r0 + (threadIdx.x >> 2);
        if (ro < a.rows) {
            const int64_t at = ro * kp128 * 4 + c0 / 32;
            reinterpret_cast<uint4*>(a.codes)[at + (threadIdx.x & 3)] = code[threadIdx.x >> 2][threadIdx.x & 3];
            if ((threadIdx.x & 3) == 0) *reinterpret_cast<unsigned*>(a.scales + at) = scale[threadIdx.x >> 2];
        }
        __syncthreads();
    }
}

constexpr int64_t FULL = 256 * 16;      // workgroups that keep the chip busy; more elements are walked by the same ones

template <OpType T>
static hipError_t quantize(hipStream_t s, const Mx4QuantArgs& a) {
    const int64_t kp = mx4_kp(a.cols);
    if (a.col_stride == 1 || a.cols == 1) {
        const int64_t n = a.rows * (kp / 8);
        mx4_quantize_rows_kernel<T><<<dim3((unsigned)std::min((n + 255) / 256, FULL)), 256, 0, s>>>(a, (unsigned)(kp / 8), n);
    } else {
        const int64_t rt = (a.rows + 63) / 64;
        mx4_quantize_cols_kernel<T><<<dim3((unsigned)std::min(rt * (kp / 128), FULL)), 256, 0, s>>>(a, (unsigned)rt, (unsigned)(kp / 128));
    }
    return hipGetLastError();
}

hipError_t launch_mx4_quantize(hipStream_t s, const Mx4QuantArgs& a) {
    return a.type == OP_F32 ? quantize<OP_F32>(s, a) : a.type == OP_BF16 ? quantize<OP_BF16>(s, a) : quantize<OP_F16>(s, a);
}

// A lane takes as many columns as make a 16-byte store (4 of fp32, 8 of 16 bits), so a wave's stores are whole lines.  The code is turned
// into its number first and multiplied by the scale after, so that the smallest scales (2^-127 is subnormal) and NaN need no case of
// their own.
template <OpType T>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(Mx4View q, typename Elem<T>::type* out, int64_t ld, unsigned parts, int64_t n) {
    typedef typename Elem<T>::type E;
    constexpr int C = 16 / sizeof(E);
    typedef E vec __attribute__((ext_vector_type(C), aligned(sizeof(E))));       // (16-byte stores to any element's address)
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t r = n >> 32 ? i / parts : (int64_t)((unsigned)i / parts);
        const int c = (int)(i - r * parts) * C;
        if (c >= q.cols) continue;
        const unsigned w = C == 8 ? reinterpret_cast<const unsigned*>(q.codes)[i] : reinterpret_cast<const unsigned short*>(q.codes)[i];
        const float s = mx4_scale(q.scales[i / (32 / C)]);
        vec v;
        auto put = [&](int at, auto two) { v[at] = (E)(two[0] * s); v[at + 1] = (E)(two[1] * s); };
        put(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0));
        put(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1));
        if constexpr (C == 8) {
            put(4, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2));
            put(6, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3));
        }
        E* o = out + r * ld + c;
        if (c + C <= q.cols) {
            *reinterpret_cast<vec*>(o) = v;
        } else {
#pragma unroll
            for (int j = 0; j < C; ++j)
                if (c + j < q.cols) o[j] = v[j];
        }
    }
}

template <OpType T>
static hipError_t dequantize(hipStream_t s, const Mx4View& q, void* out, int64_t ld) {
    typedef typename Elem<T>::type E;
    const int64_t parts = mx4_kp(q.cols) * (int64_t)sizeof(E) / 16, n = q.rows * parts;
    mx4_dequantize_kernel<T><<<dim3((unsigned)std::min((n + 255) / 256, FULL)), 256, 0, s>>>(q, static_cast<E*>(out), ld, (unsigned)parts, n);
    return hipGetLastError();
}

hipError_t launch_mx4_dequantize(hipStream_t s, const Mx4View& q, void* out, OpType type, int64_t ld) {
    return type == OP_F32 ? dequantize<OP_F32>(s, q, out, ld) : type == OP_BF16 ? dequantize<OP_BF16>(s, q, out, ld) : dequantize<OP_F16>(s, q, out, ld);
}

}  // namespace stattn
