// Kernels of drafted sampling (api_draft.cpp): distributions and draws of the drafts, and per caption the state behind the kept words, the
// words, the next round's numbers.
#include "mx4_inl.h"
#include "wave_inl.h"

namespace stattn {

// One workgroup of 16 waves a row, a stretch of the row (a multiple of 512 words) for each wave, eight neighbours a lane.  Three walks of
// it, the second and third from the caches: the largest logit, the sum, the probabilities -- whose own sums over the stretches (in 64 bits)
// then say where a draw falls, and the first wave looks there word by word.  A row of 20000 words is 20 values a lane: what counts is the
// chain of reads (8.6 us; the 256-lane softmax of the other paths takes 41 us for such a row, and the draw was another launch).
__global__ __launch_bounds__(1024) void softmax_draw_kernel(DrawArgs a) {
    constexpr int NW = 16;
    __shared__ float top[NW], sums[NW];
    __shared__ double part[NW];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const float* x = a.logits + (int64_t)blockIdx.x * a.ld;
    float* p = a.p + (int64_t)blockIdx.x * a.ld;
    const int step = ((a.v + NW - 1) / NW + 511) & ~511, lo = min(wave * step, a.v), hi = min(lo + step, a.v);
    auto walk = [&](auto each) {                       // each(first column, eight logits): -inf behind the row's end (in the row's padding)
        for (int c = lo + 8 * lane; c < hi; c += 512) {
            const float4 u = reinterpret_cast<const float4*>(x + c)[0], w = reinterpret_cast<const float4*>(x + c)[1];
            float v[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j >= hi) v[j] = -INFINITY;
            each(c, v);
        }
    };
    float m = -INFINITY;
    walk([&](int, const float* v) {
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, v[j]);
    });
    m = wave_max(m);
    if (lane == 0) top[wave] = m;
    __syncthreads();
    for (int k = 0; k < NW; ++k) m = fmaxf(m, top[k]);
    float sum = 0.f;
    walk([&](int, const float* v) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += __expf(v[j] - m);
    });
    sum = wave_sum(sum);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    sum = 0.f;
    for (int k = 0; k < NW; ++k) sum += sums[k];
    const float inv = 1.0f / sum;
    double mine = 0.0;
    walk([&](int c, const float* v) {
        float e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) { e[j] = __expf(v[j] - m) * inv; mine += (double)e[j]; }
        reinterpret_cast<float4*>(p + c)[0] = make_float4(e[0], e[1], e[2], e[3]);     // (0 behind the row's end)
        reinterpret_cast<float4*>(p + c)[1] = make_float4(e[4], e[5], e[6], e[7]);
    });
    if (!a.u) return;
    mine = wave_sum(mine);
    if (lane == 0) part[wave] = mine;
    __syncthreads();
    if (wave) return;
    // the stretch that the draw falls into: a lane a stretch
    const double own = lane < NW ? part[lane] : 0.0;
    const double upto = wave_scan(own);
    const double t = (double)a.u[blockIdx.x] * from_lane(upto, NW - 1);
    const unsigned long long over16 = __ballot(lane < NW && own > 0.0 && upto > t), with16 = __ballot(own > 0.0);
    const int last = over16 ? __builtin_ctzll(over16) : with16 ? 63 - __builtin_clzll(with16) : 0;
    double base = from_lane(upto - own, last);
    const int from = min(last * step, a.v), to = min(from + step, a.v);
    int word = 0;                                       // (a row of NaNs draws word 0)
    for (int c0 = from; c0 < to; c0 += 512) {
        const int i = c0 + 8 * lane;
        float e[8];
        double eight = 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) { e[j] = i + j < to ? p[i + j] : 0.f; eight += (double)e[j]; }
        const double incl = wave_scan(eight);
        double run = base + (incl - eight);
        int first = -1, some = -1;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            run += (double)e[j];
            if (e[j] > 0.f) { some = i + j; if (run > t && first < 0) first = i + j; }
        }
        const unsigned long long over = __ballot(first >= 0), with = __ballot(some >= 0);
        if (over) { word = from_lane(first, __builtin_ctzll(over)); break; }
        if (with) word = from_lane(some, 63 - __builtin_clzll(with));
        base += from_lane(incl, 63);
    }
    if (lane == 0) a.words[blockIdx.x] = word;
    for (int i = lane; i < a.dim / 4; i += 64)
        reinterpret_cast<float4*>(a.emb + (int64_t)blockIdx.x * a.dim)[i] = reinterpret_cast<const float4*>(a.Wemb + (int64_t)word * a.dim)[i];
}

hipError_t launch_softmax_draw(hipStream_t s, const DrawArgs& a) {
    softmax_draw_kernel<<<dim3((unsigned)a.rows), 1024, 0, s>>>(a);
    return hipGetLastError();
}

// A caption's share of the next round's uniform numbers: row r of a round holds one number a caption
__device__ __forceinline__ void next_numbers(const DraftState& d, int m, int round, int lane) {
    const int rows = 2 * d.k + 1;
    for (int r = lane; r < rows && round < d.maxlen; r += 64) d.u[r * d.M + m] = d.uniforms[((int64_t)round * rows + r) * d.M + m];
}

__global__ __launch_bounds__(256) void draft_begin_kernel(DraftState d, const float* h0, const float* c0) {
    const int m = blockIdx.x;
    for (int i = threadIdx.x; i < d.D; i += 256) { d.h[(int64_t)m * d.D + i] = h0[(int64_t)m * d.D + i]; d.c[(int64_t)m * d.D + i] = c0[(int64_t)m * d.D + i]; }
    for (int i = threadIdx.x; i < d.maxlen; i += 256) d.tokens[(int64_t)m * d.maxlen + i] = -1;
    if (threadIdx.x == 0) {
        d.x[m] = -1;
        d.info[m] = DraftInfo{0, 0, 0, 0, 0, 0.f};
    }
    if (threadIdx.x < 64) next_numbers(d, m, 0, threadIdx.x);
}

// words row m: n = accepted[m] kept drafts, then the drawn word.  hs / cs (and projs, 8 D wide) hold the states behind each of the round's
// k + 1 inputs (the last word, then the drafts), p the target's rows in front of each word.
__global__ __launch_bounds__(1024) void draft_commit_kernel(DraftState d, const int64_t* words, const int32_t* accepted, const float* hs, const float* cs,
                                                            const float* projs, const float* p, int64_t ldp) {
    const int m = blockIdx.x, t = threadIdx.x;
    DraftInfo f = d.info[m];
    const int n = accepted[m];
    __syncthreads();                       // (the first wave writes it below)
    if (f.done) return;
    const int64_t from = (int64_t)n * d.M + m;
    for (int i = t; i < d.D; i += 1024) { d.h[(int64_t)m * d.D + i] = hs[from * d.D + i]; d.c[(int64_t)m * d.D + i] = cs[from * d.D + i]; }
    if (projs)
        for (int i = t; i < 2 * d.D; i += 1024)
            reinterpret_cast<float4*>(d.proj)[(int64_t)m * 2 * d.D + i] = reinterpret_cast<const float4*>(projs)[from * 2 * d.D + i];
    if (t < 64) next_numbers(d, m, f.rounds + 1, t);
    if (t >= 64) return;
    // one wave: lane j has word j of the round (at most 8 drafts and the drawn one) and its probability
    const int64_t w = t <= n ? words[(int64_t)m * (d.k + 1) + t] : -1;
    const float pw = w >= 0 ? p[((int64_t)t * d.M + m) * ldp + w] : 0.f;
    // the caption takes words up to its first <eos>, its length's end, or the first that could not be drawn (a model of NaNs)
    const unsigned long long ends = __ballot(t <= n && w <= 0), bad = __ballot(t <= n && w < 0);
    const int stop = ends ? __builtin_ctzll(ends) : n;
    int take = min(stop + 1, d.maxlen - f.len);
    if (bad && __builtin_ctzll(bad) < take) take = __builtin_ctzll(bad);
    if (t < take) d.tokens[(int64_t)m * d.maxlen + f.len + t] = w;
    float score = f.score;
    for (int j = 0; j < take; ++j) score += from_lane(pw, j);
    const int64_t last = from_lane(w, n);
    if (t == 0) {
        f.drafted += d.k; f.kept += n; ++f.rounds;
        f.len += take; f.score = score;
        f.done = ends != 0 || f.len == d.maxlen;
        d.x[m] = last < 0 ? 0 : last;
        d.info[m] = f;
    }
}

hipError_t launch_draft_begin(hipStream_t s, const DraftState& d, const float* h0, const float* c0) {
    draft_begin_kernel<<<dim3((unsigned)d.M), 256, 0, s>>>(d, h0, c0);
    return hipGetLastError();
}
hipError_t launch_draft_commit(hipStream_t s, const DraftState& d, const int64_t* words, const int32_t* accepted, const float* hs, const float* cs,
                               const float* projs, const float* p, int64_t ldp) {
    draft_commit_kernel<<<dim3((unsigned)d.M), 1024, 0, s>>>(d, words, accepted, hs, cs, projs, p, ldp);
    return hipGetLastError();
}

}  // namespace stattn
