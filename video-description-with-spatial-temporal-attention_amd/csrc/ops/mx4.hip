// Writing matrices in microscaled 4 bits and reading them back.
#include "mx4_inl.h"

namespace stattn {

// One thread per block of 32 columns.
template <OpType T>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(Mx4QuantArgs a, int64_t kb, int64_t nblk) {
    typedef typename Elem<T>::type E;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= nblk) return;
    const int64_t r = i / kb, b = i % kb;
    const E* x = static_cast<const E*>(a.x) + r * a.row_stride;
    float v[32];
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        const int64_t c = b * 32 + j;
        v[j] = c < a.cols ? (float)x[c * a.col_stride] : 0.f;
        top = max(top, abs_bits(v[j]));
    }
    const unsigned byte = mx4_scale_byte(top);
    uint4 o;
    o.x = mx4_codes8(v, byte); o.y = mx4_codes8(v + 8, byte); o.z = mx4_codes8(v + 16, byte); o.w = mx4_codes8(v + 24, byte);
    *reinterpret_cast<uint4*>(a.codes + i * 16) = o;
    a.scales[i] = (uint8_t)byte;
}

hipError_t launch_mx4_quantize(hipStream_t s, const Mx4QuantArgs& a) {
    const int64_t kb = mx4_kp(a.cols) / 32, n = a.rows * kb;
    const dim3 grid((unsigned)((n + 255) / 256));
    switch (a.type) {
        case OP_F32: mx4_quantize_kernel<OP_F32><<<grid, 256, 0, s>>>(a, kb, n); break;
        case OP_BF16: mx4_quantize_kernel<OP_BF16><<<grid, 256, 0, s>>>(a, kb, n); break;
        case OP_F16: mx4_quantize_kernel<OP_F16><<<grid, 256, 0, s>>>(a, kb, n); break;
    }
    return hipGetLastError();
}

// One thread per eight columns: a word of codes, the block's scale, eight values.  The code is turned into its number first and
// multiplied by the scale after, so that the smallest scales (2^-127 is subnormal) and NaN need no case of their own.
template <OpType T>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(Mx4View q, typename Elem<T>::type* out, int64_t ld, int64_t w8, int64_t n) {
    typedef typename Elem<T>::type E;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int64_t r = i / w8, c = i % w8;
    const unsigned w = reinterpret_cast<const unsigned*>(q.codes)[i];
    const float s = mx4_scale(q.scales[i >> 2]);
    float v[8];
    auto put = [&](int at, auto two) { v[at] = two[0] * s; v[at + 1] = two[1] * s; };
    put(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0));
    put(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1));
    put(4, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2));
    put(6, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3));
    E* o = out + r * ld + c * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (c * 8 + j < q.cols) o[j] = (E)v[j];
}

hipError_t launch_mx4_dequantize(hipStream_t s, const Mx4View& q, void* out, OpType type, int64_t ld) {
    const int64_t w8 = mx4_kp(q.cols) / 8, n = q.rows * w8;
    const dim3 grid((unsigned)((n + 255) / 256));
    switch (type) {
        case OP_F32: mx4_dequantize_kernel<OP_F32><<<grid, 256, 0, s>>>(q, static_cast<float*>(out), ld, w8, n); break;
        case OP_BF16: mx4_dequantize_kernel<OP_BF16><<<grid, 256, 0, s>>>(q, static_cast<__bf16*>(out), ld, w8, n); break;
        case OP_F16: mx4_dequantize_kernel<OP_F16><<<grid, 256, 0, s>>>(q, static_cast<_Float16*>(out), ld, w8, n); break;
    }
    return hipGetLastError();
}

}  // namespace stattn
