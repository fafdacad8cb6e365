// Bookkeeping of drafted sampling (api_draft.cpp): per caption the state behind the kept words, the words, the next round's numbers.
#include "ops.h"

namespace stattn {

// A caption's share of the next round's uniform numbers: row r of a round holds one number a caption
__device__ __forceinline__ void next_numbers(const DraftState& d, int m, int round) {
    const int rows = 2 * d.k + 1;
    for (int r = threadIdx.x; r < rows && round < d.maxlen; r += blockDim.x) d.u[r * d.M + m] = d.uniforms[((int64_t)round * rows + r) * d.M + m];
}

__global__ __launch_bounds__(256) void draft_begin_kernel(DraftState d, const float* h0, const float* c0) {
    const int m = blockIdx.x;
    for (int i = threadIdx.x; i < d.D; i += 256) { d.h[(int64_t)m * d.D + i] = h0[(int64_t)m * d.D + i]; d.c[(int64_t)m * d.D + i] = c0[(int64_t)m * d.D + i]; }
    for (int i = threadIdx.x; i < d.maxlen; i += 256) d.tokens[(int64_t)m * d.maxlen + i] = -1;
    if (threadIdx.x == 0) {
        d.x[m] = -1;
        d.info[m] = DraftInfo{0, 0, 0, 0, 0, 0.f};
    }
    next_numbers(d, m, 0);
}

// words row m: n = accepted[m] kept drafts, then the drawn word.  hs / cs hold the states behind each of the round's k + 1 inputs (the
// last word, then the drafts), p the target's rows in front of each word.
__global__ __launch_bounds__(256) void draft_commit_kernel(DraftState d, const int64_t* words, const int32_t* accepted, const float* hs, const float* cs,
                                                           const float* p, int64_t ldp) {
    const int m = blockIdx.x;
    DraftInfo f = d.info[m];
    __syncthreads();                       // (thread 0 writes it below)
    if (f.done) return;
    const int n = accepted[m];
    const float* h = hs + ((int64_t)n * d.M + m) * d.D;
    const float* c = cs + ((int64_t)n * d.M + m) * d.D;
    for (int i = threadIdx.x; i < d.D; i += 256) { d.h[(int64_t)m * d.D + i] = h[i]; d.c[(int64_t)m * d.D + i] = c[i]; }
    if (threadIdx.x == 0) {
        f.drafted += d.k; f.kept += n;
        int64_t w = 0;
        for (int j = 0; j <= n && !f.done; ++j) {
            w = words[(int64_t)m * (d.k + 1) + j];
            if (w < 0) { f.done = 1; break; }                       // no word can be drawn (a model of NaNs): the caption ends here
            d.tokens[(int64_t)m * d.maxlen + f.len++] = w;
            f.score += p[((int64_t)j * d.M + m) * ldp + w];
            f.done = w == 0 || f.len == d.maxlen;
        }
        d.x[m] = w < 0 ? 0 : w;
        ++f.rounds;
        d.info[m] = f;
    }
    next_numbers(d, m, f.rounds + (threadIdx.x ? 1 : 0));          // thread 0 has counted the round already
}

hipError_t launch_draft_begin(hipStream_t s, const DraftState& d, const float* h0, const float* c0) {
    draft_begin_kernel<<<dim3((unsigned)d.M), 256, 0, s>>>(d, h0, c0);
    return hipGetLastError();
}
hipError_t launch_draft_commit(hipStream_t s, const DraftState& d, const int64_t* words, const int32_t* accepted, const float* hs, const float* cs,
                               const float* p, int64_t ldp) {
    draft_commit_kernel<<<dim3((unsigned)d.M), 256, 0, s>>>(d, words, accepted, hs, cs, p, ldp);
    return hipGetLastError();
}

}  // namespace stattn
