// Launchers of the device-memory operators (csrc/api_ops.cpp checks the arguments, these trust them).
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

namespace stattn {

enum OpType { OP_F32 = 0, OP_BF16 = 1, OP_F16 = 2 };

// The 4-bit form of a (rows, cols) matrix: codes [rows][kp / 2] bytes (even column in the low half), scales [rows][kp / 32] bytes,
// kp = cols rounded up to 128.  Codes are 16-byte, scales 4-byte aligned.
struct Mx4View { const uint8_t* codes; const uint8_t* scales; int64_t rows; int64_t cols; };
__host__ __device__ inline int64_t mx4_kp(int64_t cols) { return (cols + 127) / 128 * 128; }

struct Mx4QuantArgs {
    const void* x; OpType type; int64_t rows, cols, row_stride, col_stride;      // element (r, c) at x[r * row_stride + c * col_stride]
    uint8_t* codes; uint8_t* scales;
};
hipError_t launch_mx4_quantize(hipStream_t s, const Mx4QuantArgs& a);
hipError_t launch_mx4_dequantize(hipStream_t s, const Mx4View& q, void* out, OpType type, int64_t ld);

struct Mx4GemmArgs {
    Mx4View a, w;                        // y[m][n] = sum_k a[m][k] w[n][k] + bias[n]
    const float* bias;                   // or null
    void* y; OpType type; int64_t ldy;
};
hipError_t launch_mx4_matmul(hipStream_t s, const Mx4GemmArgs& g);

// The same with x (m, k) of `type`, brought into the 4-bit form inside the launch: for few rows, where one launch and no trip of x's 4-bit
// form through memory are what counts (api_ops.cpp has the rule).
struct Mx4LinearArgs {
    const void* x; OpType type; int64_t m, ldx;
    Mx4View w;
    const float* bias;
    void* y; int64_t ldy;
};
hipError_t launch_mx4_linear_few(hipStream_t s, const Mx4LinearArgs& a);

struct VerifyArgs {
    const int64_t* draft; int64_t draft_b, draft_j;          // strides as below
    const void* target; int64_t target_b, target_j;          // strides of the caption and of the position, in elements
    const void* proposal; int64_t proposal_b, proposal_j;    // or null: every drafted word was certain
    OpType type;
    const float* accept_u; int64_t accept_b, accept_j;
    const float* draw_u;
    const int32_t* lens;                                     // or null: every draft has j words
    int64_t b; int j; int64_t v;
    int64_t* words; int64_t words_ld; int32_t* accepted;
    int split; double* sums;                                 // workgroups that sum a caption's rows, and [b][256] sums; 1: none
};
// Long rows of few captions: several workgroups a caption, one a CU in all.  (1 x 128000 words: 12 us instead of 18, 64 x 128000 in bf16 14
// instead of 21; 1 x 64000 11.9 and 12.5, of which a caller has 13.8 and 12.2, a launch more taking 3.5 us of its time.)  With 128
// captions in 16 bits half the CUs are bound by arithmetic and two workgroups help (128 x 128000: 18 us instead of 21); in 32 bits they
// wait for memory either way (24.4 and 23.5).
inline int verify_split(int64_t b, int64_t v, OpType type) {
    if (v < 98304 || b > (type == OP_F32 ? 64 : 128)) return 1;
    int n = 1;
    while (n < 16 && b * n < 256) n *= 2;
    return n;
}
hipError_t launch_verify_draft(hipStream_t s, const VerifyArgs& a);

// drafted sampling (api_draft.cpp): what is kept of each caption between rounds of k drafted words
struct DraftInfo { int len, done, rounds, drafted, kept; float score; };
struct DraftState {
    int M, D, k, maxlen;
    float* h; float* c; int64_t* x;      // state and last word in front of the next round
    float* proj;                         // [M][8 D] projections of h, or null
    DraftInfo* info;
    int64_t* tokens;                     // [M][maxlen]
    const float* uniforms;               // [maxlen][2 k + 1][M]: draws of the drafts, checks, draw of the last word
    float* u;                            // [2 k + 1][M] of the round to come
};
hipError_t launch_draft_begin(hipStream_t s, const DraftState& d, const float* h0, const float* c0);
hipError_t launch_draft_commit(hipStream_t s, const DraftState& d, const int64_t* words, const int32_t* accepted, const float* hs, const float* cs,
                               const float* projs, const float* p, int64_t ldp);
// Rows of probabilities p = softmax(logits); with `u` also a word drawn from each (the first whose running sum exceeds u * total) and its
// embedding, `dim` floats.  ld: row stride of logits and p, a multiple of 8.
struct DrawArgs {
    const float* logits; float* p; int64_t ld; int v, rows;
    const float* u; int64_t* words; const float* Wemb; float* emb; int dim;
};
hipError_t launch_softmax_draw(hipStream_t s, const DrawArgs& a);

}  // namespace stattn
