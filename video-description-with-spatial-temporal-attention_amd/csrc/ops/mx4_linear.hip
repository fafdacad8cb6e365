// y = x w^T + bias for few rows of x: x is brought into 4 bits inside the launch, w (n, k) in 4 bits is read once.
// What bounds it is reading w, 17/32 byte an element, and below some megabytes the latency of doing so: 1 x 12000 x 512 (3.3 MB) takes
// 3.5 us, 5 x 20000 x 1024 (11 MB) 6.5, 64 x 12000 x 512 9.1 -- there every workgroup's rounding of x counts.  With 32 or 64 rows of w a
// wave instead of 16, so that fewer workgroups round x, 160 x 12000 x 512 took 12.0 and 17.3 us instead of 14.6; two launches (the
// form of x written once, then mx4_gemm.hip) take 7.6 and are used from there on.
#include "mx4_inl.h"

#include <type_traits>

namespace stattn {

// v_mfma_scale_f32_16x16x128_f8f6f4: lane l holds row l % 16 and block l / 16 of four of an operand.  The workgroup's 16 MT rows of x are
// rounded into LDS once, KC columns at a time, in that layout (row after row, 16 bytes further each, so that the sixteen lanes of a
// read meet sixteen slots of four banks).  A wave owns 16 rows of w and streams them from memory into registers, as they are, U steps
// of 128 columns ahead, the first of them asked for behind the first values of x and on their way while those are rounded (asked for in
// front of them, they had to arrive first, since loads come back in order: 5 x 20000 x 1024 took 7.1 us instead of 6.5).  KS = 4: the
// four waves share 16 rows of w, every fourth step each, and add up through LDS: for heads with few rows, where a wave a group would
// leave most of the chip without one.
constexpr int U = 8;

template <OpType T, int MT, int KS>
__global__ __launch_bounds__(256) void mx4_linear_kernel(Mx4LinearArgs p) {
    typedef typename Elem<T>::type E;
    constexpr int BM = 16 * MT, KC = 4096 / MT;                      // 32 KB of codes
    constexpr unsigned RS = KC / 2 + 16, SS = KC / 32 + 4;          // bytes from a row to the next: codes, scales
    __shared__ __attribute__((aligned(16))) unsigned char xc[BM * RS];
    __shared__ __attribute__((aligned(16))) unsigned char xs[BM * SS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g = lane >> 4;
    const int64_t n0 = ((int64_t)blockIdx.x * (KS == 1 ? 4 : 1) + (KS == 1 ? wave : 0)) * 16, m0 = (int64_t)blockIdx.y * BM;
    const int64_t kp = mx4_kp(p.w.cols), kb = kp / 32;
    const int steps = (int)(kp / 128);
    const int64_t nw = min(n0 + r, p.w.rows - 1);                   // rows behind the last one repeat it; their results are not stored
    const uint4* wc = reinterpret_cast<const uint4*>(p.w.codes) + nw * kb + g;
    const uint8_t* ws = p.w.scales + nw * kb + g;
    const int rows = (int)min(p.m - m0, (int64_t)BM);

    f32x4v acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;

    uint4 wr[U];
    int sr[U];
    auto fetch = [&](int s0) {                                      // this wave's steps s0, s0 + KS, ...
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t s = min(s0 + u * KS, steps - 1);
            wr[u] = wc[s * 4];
            sr[u] = ws[s * 4];
        }
    };
    const int first = KS == 1 ? 0 : wave;
    for (int c0 = 0; c0 < steps; c0 += KC / 128) {                  // KC columns of x
        const int cs = min(steps - c0, KC / 128);
        if (c0) __syncthreads();
        const int words = cs * 16, total = rows * words;            // eight columns each; all counts are multiples of 4, so a quad is whole
        auto round_x = [&](auto requests) {                         // that many requests of a lane on their way
            constexpr int Q = decltype(requests)::value;
            auto some = [&](int i0, auto meanwhile) {
                Eight<T> x[Q];
                int at[Q], row[Q];
#pragma unroll
                for (int q = 0; q < Q; ++q) {                       // (behind the end: the last words once more)
                    const int i = min(i0 + 256 * q, total - 4 + (tid & 3));
                    row[q] = (unsigned)i / (unsigned)words;
                    at[q] = i - row[q] * words;
                    const int64_t c = (int64_t)c0 * 128 + at[q] * 8;
                    x[q].take(static_cast<const E*>(p.x) + (m0 + row[q]) * p.ldx + c, (int)(p.w.cols - c));
                }
                __builtin_amdgcn_sched_barrier(0);
                meanwhile();
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    float v[8];
                    x[q].put(v);
                    const unsigned byte = mx4_scale_byte(quad_max(top8(v)));
                    *reinterpret_cast<unsigned*>(xc + row[q] * RS + at[q] * 4) = mx4_codes8(v, byte);
                    if ((at[q] & 3) == 0) xs[row[q] * SS + (at[q] >> 2)] = (uint8_t)byte;
                }
            };
            some(tid, [&]() { fetch(c0 + first); });
            for (int i0 = tid + 256 * Q; i0 - tid < total; i0 += 256 * Q) some(i0, []() {});
        };
        if (total <= 256) round_x(std::integral_constant<int, 1>());
        else if (MT == 1 && total <= 1024) round_x(std::integral_constant<int, 4>());
        else round_x(std::integral_constant<int, 8>());
        __syncthreads();
        for (int s0 = first; s0 < cs; s0 += U * KS) {
            if (s0 != first) fetch(c0 + s0);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int s = s0 + u * KS;
                if (s >= cs) break;                                 // (the same for all lanes of the wave)
                const i32x8 fw = {(int)wr[u].x, (int)wr[u].y, (int)wr[u].z, (int)wr[u].w, 0, 0, 0, 0};
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    const uint4 v = *reinterpret_cast<const uint4*>(xc + (16 * t + r) * RS + (s * 4 + g) * 16);
                    const i32x8 fx = {(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
                    acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fx, fw, acc[t], 4, 4, 0, (int)xs[(16 * t + r) * SS + s * 4 + g], 0, sr[u]);
                }
            }
        }
    }
    // The products mix lanes, and the compiler moves them freely: the empty statement keeps them in front of the lane-dependent branches
    // below.  Rows of x that do not exist were never written to LDS: whatever stood there reached only their own results.
#pragma unroll
    for (int t = 0; t < MT; ++t) asm volatile("" : "+v"(acc[t]));
    if (KS > 1) {
        __syncthreads();
        float* part = reinterpret_cast<float*>(xc);                 // [wave][t][e][lane]
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[((wave * MT + t) * 4 + e) * 64 + lane] = acc[t][e];
        __syncthreads();
        // wave w adds row group(s) e = w of every tile, in the order of the waves
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) v += part[((w * MT + t) * 4 + wave) * 64 + lane];
            const int m = 16 * t + 4 * g + wave;
            const int64_t n = n0 + r;
            if (m < rows && n < p.w.rows) static_cast<E*>(p.y)[(m0 + m) * p.ldy + n] = (E)(v + (p.bias ? p.bias[n] : 0.f));
        }
        return;
    }
    const int64_t n = n0 + r;
    if (n >= p.w.rows) return;
    const float b = p.bias ? p.bias[n] : 0.f;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int m = 16 * t + 4 * g + e;
            if (m < rows) static_cast<E*>(p.y)[(m0 + m) * p.ldy + n] = (E)(acc[t][e] + b);
        }
}

template <OpType T, int MT>
static hipError_t run(hipStream_t s, const Mx4LinearArgs& a) {
    const unsigned gm = (unsigned)((a.m + 16 * MT - 1) / (16 * MT)), gn = (unsigned)((a.w.rows + 15) / 16);
    if ((int64_t)gm * gn < 4 * 128 && a.w.cols > 128) mx4_linear_kernel<T, MT, 4><<<dim3(gn, gm), 256, 0, s>>>(a);
    else mx4_linear_kernel<T, MT, 1><<<dim3((gn + 3) / 4, gm), 256, 0, s>>>(a);
    return hipGetLastError();
}

template <OpType T>
static hipError_t run_rows(hipStream_t s, const Mx4LinearArgs& a) {
    return a.m <= 16 ? run<T, 1>(s, a) : a.m <= 32 ? run<T, 2>(s, a) : run<T, 4>(s, a);
}

hipError_t launch_mx4_linear_few(hipStream_t s, const Mx4LinearArgs& a) {
    return a.type == OP_F32 ? run_rows<OP_F32>(s, a) : a.type == OP_BF16 ? run_rows<OP_BF16>(s, a) : run_rows<OP_F16>(s, a);
}

}  // namespace stattn
