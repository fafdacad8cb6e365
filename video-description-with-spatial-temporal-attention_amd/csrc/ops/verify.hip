// Drafted words against the decoder's own distribution.  For one caption with drafted words d_0 .. d_{len-1}, the target's
// probabilities p_j (one more row than words) and the proposal's q_j they were drawn from:
//     d_j is kept while u_j q_j(d_j) < p_j(d_j);  n = the first j that is not, or len;
//     the word at n is drawn from  max(p_n - q_n, 0)  (normalised) after a refusal, from p_n itself after len kept words,
// which makes the kept words and the drawn one a sample of the target's distribution whatever the proposal is.
// Products and sums are in 64 bits: u q is then exact for 32-bit inputs, and a word next to a border of the running sum does not
// depend on the order of 32-bit roundings.
#include "mx4_inl.h"

namespace stattn {

template <OpType T>
__device__ __forceinline__ double prob(const void* base, int64_t i) { return (double)(float)static_cast<const typename Elem<T>::type*>(base)[i]; }

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// One caption's weights over a stretch of the vocabulary.  q null: p alone, or p without the refused word (a certain proposal).
template <OpType T, bool WIDE>
struct Weights {
    typedef typename Elem<T>::type E;
    const E* p;
    const E* q;
    int64_t v, certain;             // vocabulary; the word that a certain proposal has all its mass on, or -1

    // p > q is decided in 32 bits, where it is exact (and false for a NaN); the difference is one operation in 64
    __device__ __forceinline__ double of(float a, float b) const {
        const bool over = a > b;
        return (double)(over ? a : 0.f) - (double)(over ? b : 0.f);
    }
    __device__ __forceinline__ double at(int64_t i) const { return of((float)p[i], q ? (float)q[i] : i == certain ? 1.f : 0.f); }

    // Sum of the weights from `from` to `to`, this lane's share of the wave's walk; K requests on their way.  The lanes take eight
    // neighbours each where those are 16-byte loads, else every 64th word.
    template <bool Q>
    __device__ __forceinline__ double walk(int64_t from, int64_t to, int lane) const {
        constexpr int K = sizeof(E) == 4 ? 2 : 4;       // (sixteen waves leave 128 registers each)
        double sum = 0.0;
        for (int64_t c0 = from; c0 < to; c0 += 512 * K) {
            if constexpr (WIDE) {
                Eight<T, true> a[K], b[K];
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const int64_t c = c0 + 512 * k + 8 * lane;
                    a[k].take(p, c, c < to ? 8 : 0);
                    if (Q) b[k].take(q, c, c < to ? 8 : 0);
                }
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const int64_t c = c0 + 512 * k + 8 * lane;
                    float x[8], y[8];
                    a[k].put(x, c < to ? 8 : 0);
                    if (Q) b[k].put(y, c < to ? 8 : 0);
#pragma unroll
                    for (int j = 0; j < 8; ++j) sum += of(x[j], Q ? y[j] : c + j == certain ? 1.f : 0.f);
                }
            } else {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    E a[8], b[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int64_t c = c0 + 512 * k + 64 * j + lane;
                        a[j] = p[c < to ? c : from];
                        if (Q) b[j] = q[c < to ? c : from];
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int64_t c = c0 + 512 * k + 64 * j + lane;
                        const double w = of((float)a[j], Q ? (float)b[j] : c == certain ? 1.f : 0.f);
                        sum += c < to ? w : 0.0;
                    }
                }
            }
        }
        return sum;
    }
    __device__ __forceinline__ double sum(int64_t from, int64_t to, int lane) const {
        return wave_sum64(q ? walk<true>(from, to, lane) : walk<false>(from, to, lane));
    }
};

// One workgroup of NW waves a caption.  The vocabulary is cut into NW stretches, a wave sums one; the stretch that the draw falls into is
// cut again if it is long, and one wave walks the rest word by word.  That reads the rows once and a sixteenth (a 256th) of them again,
// and no sum's order depends on anything but v, so results repeat.  Bound: at one caption the chain of dependent reads (draft ->
// probabilities -> rows -> stretch), at many reading two rows each.
template <OpType T, int NW, bool WIDE>
__global__ __launch_bounds__(64 * NW) void verify_kernel(VerifyArgs a) {
    typedef typename Elem<T>::type E;
    __shared__ double part[2][2][NW];       // [turn][level]: never written again while a wave may still read it
    const int64_t i = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t* drafts = a.draft + i * a.draft_b;
    auto draft = [&](int j) { return drafts[j * a.draft_j]; };
    // every wave finds the first refused word for itself, a lane a word
    const int len = a.lens ? min(max(a.lens[i], 0), a.j) : a.j;
    int n = len;
    for (int j0 = 0; j0 < len; j0 += 64) {
        const int j = j0 + lane;
        bool kept = true;
        if (j < len) {
            const int64_t d = draft(j);
            kept = d >= 0 && d < a.v;
            if (kept) {
                const double p = prob<T>(a.target, i * a.target_b + j * a.target_j + d);
                const double q = a.proposal ? prob<T>(a.proposal, i * a.proposal_b + j * a.proposal_j + d) : 1.0;
                kept = (double)a.accept_u[i * a.accept_b + j * a.accept_j] * q < p;
            }
        }
        const unsigned long long refused = __ballot(!kept);
        if (refused) { n = j0 + __builtin_ctzll(refused); break; }
    }
    n = __builtin_amdgcn_readfirstlane(n);
    Weights<T, WIDE> w;
    w.v = a.v;
    w.p = static_cast<const E*>(a.target) + i * a.target_b + n * a.target_j;
    w.q = n < len && a.proposal ? static_cast<const E*>(a.proposal) + i * a.proposal_b + n * a.proposal_j : nullptr;
    w.certain = n < len && !a.proposal ? draft(n) : -1;
    const double u = (double)a.draw_u[i];

    int64_t word = -1;
    for (int turn = 0; turn < 2; ++turn) {
        // a stretch of the vocabulary for each wave: multiples of 512 words, as many as 64 lanes take at a time
        int64_t from = 0, to = a.v, step = ((a.v + NW - 1) / NW + 511) & ~(int64_t)511;
        double base = 0.0, t = 0.0;
        bool any = false;
        for (int level = 0; level < 2; ++level) {
            const int64_t lo = min(from + wave * step, to), hi = min(lo + step, to);
            const double mine = lo < hi ? w.sum(lo, hi, lane) : 0.0;
            if (lane == 0) part[turn][level][wave] = mine;
            __syncthreads();
            const double* all = part[turn][level];
            if (level == 0) {
                double total = 0.0;
                for (int k = 0; k < NW; ++k) total += all[k];
                any = total > 0.0;
                if (!any) break;
                t = u * total;
            }
            // the stretch in which the running sum passes t; where roundings leave none, the last with any weight
            int hit = -1, last = 0;
            double before = base, c = base;
            for (int k = 0; k < NW; ++k) {
                if (all[k] > 0.0 && hit < 0) {
                    last = k; before = c;
                    if (c + all[k] > t) hit = k;
                }
                c += all[k];
            }
            base = before;
            from = min(from + last * step, to);
            to = min(from + step, to);
            if (step <= 2048) break;
            step = ((to - from + NW - 1) / NW + 511) & ~(int64_t)511;
        }
        if (any) {
            if (wave == 0) {                 // word by word: eight neighbours a lane, 512 at a time
                for (int64_t c0 = from; c0 < to; c0 += 512) {
                    const int64_t c = c0 + 8 * lane;
                    double x[8], mine = 0.0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) { x[j] = c + j < to ? w.at(c + j) : 0.0; mine += x[j]; }
                    double incl = mine;
#pragma unroll
                    for (int o = 1; o < 64; o <<= 1) { const double y = __shfl_up(incl, o, 64); if (lane >= o) incl += y; }
                    double run = base + (incl - mine);
                    int64_t first = -1, some = -1;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        run += x[j];
                        if (x[j] > 0.0) { some = c + j; if (run > t && first < 0) first = c + j; }
                    }
                    const unsigned long long over = __ballot(first >= 0), with = __ballot(some >= 0);
                    if (over) { word = __shfl(first, __builtin_ctzll(over), 64); break; }
                    if (with) word = __shfl(some, 63 - __builtin_clzll(with), 64);        // the last with weight, should roundings leave none over t
                    base += __shfl(incl, 63, 64);
                }
            }
            break;
        }
        if (w.q == nullptr && w.certain < 0) break;
        w.q = nullptr; w.certain = -1;       // nothing is left over a proposal that is nowhere smaller: the draw is from p itself
    }
    if (wave == 0)
        for (int k = lane; k <= a.j; k += 64) a.words[i * a.words_ld + k] = k < n ? draft(k) : k == n ? word : -1;
    if (tid == 0) a.accepted[i] = n;
}

template <OpType T, int NW>
static hipError_t run(hipStream_t s, const VerifyArgs& a) {
    constexpr size_t size = sizeof(typename Elem<T>::type);
    const bool wide = eights_are_wide(a.target, a.target_b, a.v, size) && a.target_j * (int64_t)size % 16 == 0 &&
                      (!a.proposal || (eights_are_wide(a.proposal, a.proposal_b, a.v, size) && a.proposal_j * (int64_t)size % 16 == 0));
    if (wide) verify_kernel<T, NW, true><<<dim3((unsigned)a.b), 64 * NW, 0, s>>>(a);
    else verify_kernel<T, NW, false><<<dim3((unsigned)a.b), 64 * NW, 0, s>>>(a);
    return hipGetLastError();
}

template <OpType T>
static hipError_t run(hipStream_t s, const VerifyArgs& a) { return a.v <= 4 * 512 ? run<T, 4>(s, a) : run<T, 16>(s, a); }

hipError_t launch_verify_draft(hipStream_t s, const VerifyArgs& a) {
    return a.type == OP_F32 ? run<OP_F32>(s, a) : a.type == OP_BF16 ? run<OP_BF16>(s, a) : run<OP_F16>(s, a);
}

}  // namespace stattn
