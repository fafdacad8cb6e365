// Drafted words against the decoder's own distribution.  For one caption with drafted words d_0 .. d_{len-1}, the target's
// probabilities p_j (one more row than words) and the proposal's q_j they were drawn from:
//     d_j is kept while u_j q_j(d_j) < p_j(d_j);  n = the first j that is not, or len;
//     the word at n is drawn from  max(p_n - q_n, 0)  (normalised) after a refusal, from p_n itself after len kept words,
// which makes the kept words and the drawn one a sample of the target's distribution whatever the proposal is.
// Products and sums are in 64 bits: u q is then exact for 32-bit inputs, and a word next to a border of the running sum does not
// depend on the order of 32-bit roundings.
#include "mx4_inl.h"

namespace stattn {

constexpr int VF_THREADS = 1024;

template <OpType T>
__device__ __forceinline__ double prob(const void* base, int64_t i) { return (double)(float)static_cast<const typename Elem<T>::type*>(base)[i]; }

__device__ __forceinline__ double weight(double p, double q) { const double w = p - q; return w > 0.0 ? w : 0.0; }

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// one workgroup per caption
template <OpType T>
__global__ __launch_bounds__(VF_THREADS) void verify_kernel(VerifyArgs a) {
    __shared__ double part[VF_THREADS / 64];
    __shared__ int s_n;
    __shared__ long long s_word;
    const int64_t i = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int len = a.lens ? min(max(a.lens[i], 0), a.j) : a.j;
    if (tid == 0) {
        int n = 0;
        for (; n < len; ++n) {
            const int64_t d = a.draft[i * a.draft_ld + n];
            if (d < 0 || d >= a.v) break;
            const double p = prob<T>(a.target, i * a.target_b + n * a.target_j + d);
            const double q = a.proposal ? prob<T>(a.proposal, i * a.proposal_b + n * a.proposal_j + d) : 1.0;
            if (!((double)a.accept_u[i * a.accept_ld + n] * q < p)) break;
        }
        s_n = n;
        s_word = -1;
    }
    __syncthreads();
    const int n = s_n;
    const int64_t pt = i * a.target_b + n * a.target_j, pq = i * a.proposal_b + n * a.proposal_j;
    const int64_t refused = n < len ? a.draft[i * a.draft_ld + n] : -1;
    bool rest = n < len;
    auto w = [&](int64_t v) {
        const double p = prob<T>(a.target, pt + v);
        const double q = !rest ? 0.0 : a.proposal ? prob<T>(a.proposal, pq + v) : v == refused ? 1.0 : 0.0;
        return weight(p, q);
    };
    const int64_t per = (a.v + VF_THREADS - 1) / VF_THREADS, lo = min(tid * per, a.v), hi = min(lo + per, a.v);
    for (int turn = 0; turn < 2; ++turn) {
        double mine = 0.0;
        for (int64_t v = lo; v < hi; ++v) mine += w(v);
        double incl = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) { const double t = __shfl_up(incl, o, 64); if (lane >= o) incl += t; }
        if (lane == 63) part[wave] = incl;
        __syncthreads();
        double base = 0.0, total = 0.0;
        for (int k = 0; k < VF_THREADS / 64; ++k) { if (k < wave) base += part[k]; total += part[k]; }
        if (total > 0.0) {
            const double t = (double)a.draw_u[i] * total;
            double c = base + incl - mine;
            int64_t word = -1;
            for (int64_t v = lo; v < hi && word < 0; ++v) { const double x = w(v); c += x; if (x > 0.0 && c > t) word = v; }
            // first crossing over the whole row: the smallest word any thread reports
            unsigned long long best = word < 0 ? ~0ull : (unsigned long long)word;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) best = min(best, __shfl_xor(best, o, 64));
            __syncthreads();
            if (lane == 0) part[wave] = __builtin_bit_cast(double, best);
            __syncthreads();
            if (tid == 0) {
                for (int k = 0; k < VF_THREADS / 64; ++k) best = min(best, __builtin_bit_cast(unsigned long long, part[k]));
                s_word = best == ~0ull ? a.v - 1 : (long long)best;
            }
            break;
        }
        if (!rest) break;
        rest = false;              // p <= q everywhere: nothing is left over, the draw is from p itself
        __syncthreads();
    }
    __syncthreads();
    for (int k = tid; k <= a.j; k += VF_THREADS)
        a.words[i * a.words_ld + k] = k < n ? a.draft[i * a.draft_ld + k] : k == n ? s_word : -1;
    if (tid == 0) a.accepted[i] = n;
}

hipError_t launch_verify_draft(hipStream_t s, const VerifyArgs& a) {
    const dim3 grid((unsigned)a.b);
    switch (a.type) {
        case OP_F32: verify_kernel<OP_F32><<<grid, VF_THREADS, 0, s>>>(a); break;
        case OP_BF16: verify_kernel<OP_BF16><<<grid, VF_THREADS, 0, s>>>(a); break;
        case OP_F16: verify_kernel<OP_F16><<<grid, VF_THREADS, 0, s>>>(a); break;
    }
    return hipGetLastError();
}

}  // namespace stattn
