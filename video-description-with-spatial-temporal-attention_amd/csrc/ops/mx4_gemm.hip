// Products of two matrices in microscaled 4 bits on the matrix cores: v_mfma_scale_f32_32x32x64_f8f6f4 multiplies 32 x 64 codes by
// 64 x 32 codes under their block scales and adds in fp32.  Lane l of the wave holds row l % 32 and the block l / 32 of an operand:
// exactly one 16-byte block of the row-major form and its scale byte, so operands go from memory to registers as they are.
#include "mx4_inl.h"

namespace stattn {

__device__ __forceinline__ i32x8 frag4(uint4 v) { return i32x8{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0}; }

// One wave per 32 x 32 tile of y, operands straight from memory.
template <OpType T>
__global__ __launch_bounds__(64) void mx4_gemm_wave_kernel(Mx4GemmArgs p, int64_t kb, unsigned nt) {
    typedef typename Elem<T>::type E;
    const int l = threadIdx.x, r = l & 31, g = l >> 5;
    const int64_t m0 = (int64_t)(blockIdx.x / nt) * 32, n0 = (int64_t)(blockIdx.x % nt) * 32;
    const int64_t ma = min(m0 + r, p.a.rows - 1), nw = min(n0 + r, p.w.rows - 1);
    const uint4* ca = reinterpret_cast<const uint4*>(p.a.codes) + ma * kb + g;
    const uint4* cw = reinterpret_cast<const uint4*>(p.w.codes) + nw * kb + g;
    const uint8_t* sa = p.a.scales + ma * kb + g;
    const uint8_t* sw = p.w.scales + nw * kb + g;
    f32x16v acc;
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.f;
    for (int64_t k = 0; k < kb; k += 2)
        acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(frag4(ca[k]), frag4(cw[k]), acc, 4, 4, 0, (int)sa[k], 0, (int)sw[k]);
    const int64_t n = n0 + r;
    if (n >= p.w.rows) return;
    const float b = p.bias ? p.bias[n] : 0.f;
    E* y = static_cast<E*>(p.y) + n;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int64_t m = m0 + (i >> 2) * 8 + g * 4 + (i & 3);
        if (m < p.a.rows) y[m * p.ldy] = (E)(acc[i] + b);
    }
}

template <OpType T>
static hipError_t run(hipStream_t s, const Mx4GemmArgs& g) {
    const int64_t kb = mx4_kp(g.a.cols) / 32, mt = (g.a.rows + 31) / 32, nt = (g.w.rows + 31) / 32;
    mx4_gemm_wave_kernel<T><<<dim3((unsigned)(mt * nt)), 64, 0, s>>>(g, kb, (unsigned)nt);
    return hipGetLastError();
}

hipError_t launch_mx4_matmul(hipStream_t s, const Mx4GemmArgs& g) {
    return g.type == OP_F32 ? run<OP_F32>(s, g) : g.type == OP_BF16 ? run<OP_BF16>(s, g) : run<OP_F16>(s, g);
}

}  // namespace stattn
