// Drafted words against the decoder's own distribution.  For one caption with drafted words d_0 .. d_{len-1}, the target's
// probabilities p_j (one more row than words) and the proposal's q_j they were drawn from:
//     d_j is kept while u_j q_j(d_j) < p_j(d_j);  n = the first j that is not, or len;
//     the word at n is drawn from  max(p_n - q_n, 0)  (normalised) after a refusal, from p_n itself after len kept words,
// which makes the kept words and the drawn one a sample of the target's distribution whatever the proposal is.
// Products and sums are in 64 bits: u q is then exact for 32-bit inputs, and a word next to a border of the running sum does not
// depend on the order of 32-bit roundings.
// 1 caption x 12000 words 7 us, 64 x 20000 in fp32 7.9, 128 x 128000 in bf16 18 (66 MB, 3.7 TB/s), 128 x 250000 28 (4.6 TB/s).
#include "mx4_inl.h"
#include "wave_inl.h"

namespace stattn {

template <OpType T>
__device__ __forceinline__ double prob(const void* base, int64_t i) { return (double)(float)static_cast<const typename Elem<T>::type*>(base)[i]; }

// One caption's weights over a stretch of the vocabulary: p alone, p without the one word that a certain proposal has all its mass on, or
// p over q.
template <OpType T>
struct Weights {
    typedef typename Elem<T>::type E;
    const E* p;
    const E* q;                     // or null
    int64_t certain;                // or -1

    // a > b is decided in 32 bits, where it is exact (and false for a NaN); the difference is one operation in 64
    static __device__ __forceinline__ double over(float a, float b) {
        const bool more = a > b;
        return (double)(more ? a : 0.f) - (double)(more ? b : 0.f);
    }
    static __device__ __forceinline__ double over(float a) { return (double)(a > 0.f ? a : 0.f); }
    __device__ __forceinline__ double at(int64_t i) const { return q ? over((float)p[i], (float)q[i]) : i == certain ? over((float)p[i], 1.f) : over((float)p[i]); }

    // Sum of the weights from `from` to `to`, this lane's share of the wave's walk; K requests on their way.  The lanes take eight
    // neighbours each.
    template <bool Q>
    __device__ __forceinline__ double walk(int64_t from, int64_t to, int lane) const {
        constexpr int K = 2;            // (stretches of 1024 words are the most frequent here; with 4, 128 x 250000 in bf16 took 41 us instead of 28)
        double sum = 0.0;
        for (int64_t c0 = from; c0 < to; c0 += 512 * K) {
            Eight<T> a[K], b[K];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int64_t c = c0 + 512 * k + 8 * lane;
                const int here = (int)min(to - c, (int64_t)8);
                a[k].take(p + c, here);
                if (Q) b[k].take(q + c, here);
            }
#pragma unroll
            for (int k = 0; k < K; ++k) {
                float x[8], y[8];
                a[k].put(x);
                if (Q) b[k].put(y);
#pragma unroll
                for (int j = 0; j < 8; ++j) sum += Q ? over(x[j], y[j]) : over(x[j]);
            }
        }
        return sum;
    }
    // The sums of stretches k, k + stride, ... of `n` stretches of 512 words into all[]; K of them on their way.
    template <bool Q>
    __device__ __forceinline__ void chunks(int k0, int stride, int n, int64_t v, int lane, double* all) const {
        constexpr int K = 2;
        for (; k0 < n; k0 += K * stride) {
            Eight<T> a[K], b[K];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int64_t c = (int64_t)(k0 + k * stride) * 512 + 8 * lane;
                const int here = (int)min(v - c, (int64_t)8);
                a[k].take(p + c, here);
                if (Q) b[k].take(q + c, here);
            }
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int at_ = k0 + k * stride;
                if (at_ >= n) break;
                float x[8], y[8];
                a[k].put(x);
                if (Q) b[k].put(y);
                double s = 0.0;
#pragma unroll
                for (int j = 0; j < 8; ++j) s += Q ? over(x[j], y[j]) : over(x[j]);
                if (!Q && certain >= (int64_t)at_ * 512 && certain < (int64_t)at_ * 512 + 512) {     // (the same for the wave, and rare)
                    const int64_t c = (int64_t)at_ * 512 + 8 * lane;
                    s = 0.0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) s += c + j == certain ? over(x[j], 1.f) : over(x[j]);
                }
                s = wave_sum(s);
                if (lane == 0) all[at_] = s;
            }
        }
    }
    __device__ __forceinline__ double sum(int64_t from, int64_t to, int lane) const {
        if (q) return wave_sum(walk<true>(from, to, lane));
        if (certain < from || certain >= to) return wave_sum(walk<false>(from, to, lane));
        // A certain proposal's word weighs p - 1 (0 unless p is over 1), not p.  Taken back from the sum it would leave a rounding behind,
        // so the 512 words around it are summed without it.
        const int64_t c0 = from + ((certain - from) & ~(int64_t)511), c1 = min(c0 + 512, to);
        double s = walk<false>(from, c0, lane) + walk<false>(c1, to, lane);
        for (int64_t c = c0 + lane; c < c1; c += 64) s += at(c);
        return wave_sum(s);
    }
};

// The first word of caption i's draft that is refused, or its length; every wave finds it for itself, a lane a word.  Words are read
// whether they count or not, so that the length need not be there first.
template <OpType T>
__device__ __forceinline__ int first_refused(const VerifyArgs& a, int64_t i, int& len, int lane) {
    len = a.lens ? min(max(a.lens[i], 0), a.j) : a.j;
    for (int j0 = 0; j0 < a.j; j0 += 64) {
        const int j = j0 + lane;
        bool kept = true;
        if (j < a.j) {
            const int64_t d = a.draft[i * a.draft_b + j * a.draft_j];
            kept = d >= 0 && d < a.v;
            if (kept) {
                const double p = prob<T>(a.target, i * a.target_b + j * a.target_j + d);
                const double q = a.proposal ? prob<T>(a.proposal, i * a.proposal_b + j * a.proposal_j + d) : 1.0;
                kept = (double)a.accept_u[i * a.accept_b + j * a.accept_j] * q < p;
            }
        }
        const unsigned long long refused = __ballot(!kept);
        if (refused) return min(__builtin_amdgcn_readfirstlane(j0 + __builtin_ctzll(refused)), len);
        if (j0 + 64 >= len) break;
    }
    return len;
}
template <OpType T>
__device__ __forceinline__ Weights<T> weights_at(const VerifyArgs& a, int64_t i, int n, int len) {
    typedef typename Elem<T>::type E;
    Weights<T> w;
    w.p = static_cast<const E*>(a.target) + i * a.target_b + n * a.target_j;
    w.q = n < len && a.proposal ? static_cast<const E*>(a.proposal) + i * a.proposal_b + n * a.proposal_j : nullptr;
    w.certain = n < len && !a.proposal ? a.draft[i * a.draft_b + n * a.draft_j] : -1;
    return w;
}
// The length of at most `n` stretches of the vocabulary: multiples of 512 words, as many as 64 lanes take at a time.
__device__ __forceinline__ int64_t stretch(int64_t v, int n) { return ((v + n - 1) / n + 511) & ~(int64_t)511; }
constexpr int STRETCHES = 256, NW16 = 16;
// This wave's share (every `stride`-th) of the sums of all stretches.
template <OpType T>
__device__ __forceinline__ void sum_stretches(const Weights<T>& w, int64_t v, int k0, int stride, int lane, double* all) {
    const int64_t step = stretch(v, STRETCHES);
    const int n = (int)((v + step - 1) / step);
    if (step == 512) {
        if (w.q) w.template chunks<true>(k0, stride, n, v, lane, all);
        else w.template chunks<false>(k0, stride, n, v, lane, all);
        return;
    }
    for (int k = k0; k < n; k += stride) {
        const double s = w.sum(k * step, min((k + 1) * step, v), lane);
        if (lane == 0) all[k] = s;
    }
}
// Running sums of the stretches, four neighbours a lane (a loop over them, one dependent read and addition after the other, took longer
// than reading the rows).
struct Running {
    double x[4], incl;              // this lane's stretches; the sum up to and with them
    __device__ __forceinline__ Running(const double* all, int n, int lane) {
        double own = 0.0;
#pragma unroll
        for (int j = 0; j < 4; ++j) { x[j] = 4 * lane + j < n ? all[4 * lane + j] : 0.0; own += x[j]; }
        incl = wave_scan(own);
    }
    __device__ __forceinline__ double total() const { return from_lane(incl, 63); }
    // The stretch in which the running sum from `base` on passes t, and (in `base`) the sum in front of it; where roundings leave none,
    // the last with any weight.
    __device__ __forceinline__ int passes(double t, double& base, int lane) const {
        int first = -1, some = -1;
        double run = base + (incl - ((x[0] + x[1]) + (x[2] + x[3]))), at_first = 0.0, at_some = 0.0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const double next = run + x[j];
            if (x[j] > 0.0) {
                some = 4 * lane + j; at_some = run;
                if (next > t && first < 0) { first = 4 * lane + j; at_first = run; }
            }
            run = next;
        }
        const unsigned long long over = __ballot(first >= 0), with = __ballot(some >= 0);
        const int from = over ? __builtin_ctzll(over) : with ? 63 - __builtin_clzll(with) : 0;
        base = from_lane(over ? at_first : at_some, from);
        return from_lane(over ? first : some, from);
    }
};

// The stretches' sums of long rows by several workgroups a caption (blockIdx.x of gridDim.x), for verify_kernel to go on from.
template <OpType T>
__global__ __launch_bounds__(64 * NW16) void verify_sums_kernel(VerifyArgs a) {
    const int64_t i = blockIdx.y;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int len;
    const int n = first_refused<T>(a, i, len, lane);
    sum_stretches<T>(weights_at<T>(a, i, n, len), a.v, blockIdx.x * NW16 + wave, gridDim.x * NW16, lane, a.sums + i * STRETCHES);
}

// One workgroup of NW waves a caption.  The vocabulary is cut into stretches of 512 words (longer ones from 131072 words on: 256 at most),
// whose sums the waves share out (or verify_sums_kernel has left); in the stretch that the draw falls into one wave goes word by word.
// That reads the rows once and one stretch again, and no sum's order depends on anything but v, so results repeat.  Bound: at one
// caption the chain of dependent reads (draft -> probabilities -> rows -> stretch), at many reading two rows each.
template <OpType T, int NW>
__global__ __launch_bounds__(64 * NW) void verify_kernel(VerifyArgs a) {
    __shared__ double all[2][STRETCHES];    // [turn]: never written again while a wave may still read it
    __shared__ double part[2][NW];
    const int64_t i = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const double u = (double)a.draw_u[i];
    int len;
    const int n = first_refused<T>(a, i, len, lane);
    Weights<T> w = weights_at<T>(a, i, n, len);

    int64_t word = -1;
    for (int turn = 0; turn < 2; ++turn) {
        int64_t step = stretch(a.v, STRETCHES);
        const int ns = (int)((a.v + step - 1) / step);
        if (turn == 0 && a.split > 1) {
            if (tid < ns) all[0][tid] = a.sums[i * STRETCHES + tid];
        } else {
            sum_stretches<T>(w, a.v, wave, NW, lane, all[turn]);
        }
        __syncthreads();
        const Running run(all[turn], ns, lane);
        const double total = run.total(), t = u * total;
        double base = 0.0;
        const bool any = total > 0.0;
        if (any) {
            int64_t from = min(run.passes(t, base, lane) * step, a.v), to = min(from + step, a.v);
            if (step > 2048) {               // a long stretch is cut once more
                step = stretch(to - from, NW);
                const int64_t lo = min(from + wave * step, to), hi = min(lo + step, to);
                const double mine = lo < hi ? w.sum(lo, hi, lane) : 0.0;
                if (lane == 0) part[turn][wave] = mine;
                __syncthreads();
                from = min(from + max(Running(part[turn], NW, lane).passes(t, base, lane), 0) * step, to);
                to = min(from + step, to);
            }
            if (wave == 0) {                 // word by word: eight neighbours a lane, 512 at a time
                for (int64_t c0 = from; c0 < to; c0 += 512) {
                    const int64_t c = c0 + 8 * lane;
                    double x[8], mine = 0.0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) { x[j] = c + j < to ? w.at(c + j) : 0.0; mine += x[j]; }
                    const double incl = wave_scan(mine);
                    double run = base + (incl - mine);
                    int64_t first = -1, some = -1;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        run += x[j];
                        if (x[j] > 0.0) { some = c + j; if (run > t && first < 0) first = c + j; }
                    }
                    const unsigned long long over = __ballot(first >= 0), with = __ballot(some >= 0);
                    if (over) { word = from_lane(first, __builtin_ctzll(over)); break; }
                    if (with) word = from_lane(some, 63 - __builtin_clzll(with));        // the last with weight, should roundings leave none over t
                    base += from_lane(incl, 63);
                }
            }
            break;
        }
        if (w.q == nullptr && w.certain < 0) break;
        w.q = nullptr; w.certain = -1;       // nothing is left over a proposal that is nowhere smaller: the draw is from p itself
    }
    if (wave == 0)
        for (int k = lane; k <= a.j; k += 64) a.words[i * a.words_ld + k] = k < n ? a.draft[i * a.draft_b + k * a.draft_j] : k == n ? word : -1;
    if (tid == 0) a.accepted[i] = n;
}

template <OpType T>
static hipError_t run(hipStream_t s, const VerifyArgs& a) {
    if (a.split > 1) verify_sums_kernel<T><<<dim3((unsigned)a.split, (unsigned)a.b), 64 * NW16, 0, s>>>(a);
    if (a.v <= 4 * 512) verify_kernel<T, 4><<<dim3((unsigned)a.b), 64 * 4, 0, s>>>(a);
    else verify_kernel<T, NW16><<<dim3((unsigned)a.b), 64 * NW16, 0, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_verify_draft(hipStream_t s, const VerifyArgs& a) {
    return a.type == OP_F32 ? run<OP_F32>(s, a) : a.type == OP_BF16 ? run<OP_BF16>(s, a) : run<OP_F16>(s, a);
}

}  // namespace stattn
