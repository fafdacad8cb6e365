// C ABI of libstattn.so: the operators on device memory (include/stattn.h).  Arguments are checked here, before anything is launched.
#include "../../include/stattn.h"
#include "ops/ops.h"

#include <cstdarg>
#include <cstdio>

using namespace stattn;

namespace {

thread_local char op_error[512] = "";

int refuse(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(op_error, sizeof op_error, fmt, ap);
    va_end(ap);
    return code;
}

// The stream's device is current while kernels are launched on it, and the caller's is again afterwards.
struct OnDevice {
    int before = -1, dev;
    hipError_t err;
    explicit OnDevice(int d) : dev(d) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != d) err = hipSetDevice(d);
    }
    ~OnDevice() { if (before >= 0 && before != dev) (void)hipSetDevice(before); }
};

constexpr int64_t MAX_ROWS = (int64_t)1 << 31, MAX_COLS = (int64_t)1 << 24;

bool type_ok(int t) { return t == STATTN_F32 || t == STATTN_BF16 || t == STATTN_F16; }
bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// |stride| * (n - 1) stays far from the end of 64 bits
bool stride_ok(int64_t s) { return s > -((int64_t)1 << 40) && s < ((int64_t)1 << 40); }

int form_ok(const char* who, const void* codes, const void* scales, int64_t rows, int64_t cols) {
    if (rows < 0 || rows >= MAX_ROWS || cols < 1 || cols > MAX_COLS)
        return refuse(STATTN_EINVAL, "%s: a matrix of %lld x %lld is outside 0 .. 2^31 - 1 rows and 1 .. 2^24 columns", who, (long long)rows, (long long)cols);
    if (rows && (!codes || !scales)) return refuse(STATTN_EINVAL, "%s: null codes or scales", who);
    if (!al16(codes) || (reinterpret_cast<uintptr_t>(scales) & 3)) return refuse(STATTN_EINVAL, "%s: codes must be 16-byte aligned, scales 4-byte aligned", who);
    return STATTN_OK;
}

int launched(const char* who, hipError_t e) {
    return e == hipSuccess ? STATTN_OK : refuse(STATTN_EHIP, "%s: %s", who, hipGetErrorString(e));
}

}  // namespace

#define OPCHK(expr) do { const int rc_ = (expr); if (rc_ != STATTN_OK) return rc_; } while (0)

extern "C" {

const char* stattn_op_error(void) { return op_error; }

int stattn_mx4_quantize(int device, void* stream, const void* x, int dtype, int64_t rows, int64_t cols, int64_t row_stride,
                        int64_t col_stride, void* codes, void* scales) {
    OPCHK(form_ok("mx4_quantize", codes, scales, rows, cols));
    if (!type_ok(dtype)) return refuse(STATTN_EINVAL, "mx4_quantize: dtype %d is none of STATTN_F32, STATTN_BF16, STATTN_F16", dtype);
    if (!stride_ok(row_stride) || !stride_ok(col_stride)) return refuse(STATTN_EINVAL, "mx4_quantize: strides must stay under 2^40 elements");
    if (!rows) return STATTN_OK;
    if (!x) return refuse(STATTN_EINVAL, "mx4_quantize: null x");
    const OnDevice on(device);
    if (on.err != hipSuccess) return launched("mx4_quantize", on.err);
    Mx4QuantArgs a{x, (OpType)dtype, rows, cols, row_stride, col_stride, static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales)};
    return launched("mx4_quantize", launch_mx4_quantize(static_cast<hipStream_t>(stream), a));
}

int stattn_mx4_dequantize(int device, void* stream, const void* codes, const void* scales, int64_t rows, int64_t cols, void* out,
                          int dtype, int64_t ld_out) {
    OPCHK(form_ok("mx4_dequantize", codes, scales, rows, cols));
    if (!type_ok(dtype)) return refuse(STATTN_EINVAL, "mx4_dequantize: dtype %d is none of STATTN_F32, STATTN_BF16, STATTN_F16", dtype);
    if (ld_out < cols || !stride_ok(ld_out)) return refuse(STATTN_EINVAL, "mx4_dequantize: ld_out (%lld) must be at least cols (%lld)", (long long)ld_out, (long long)cols);
    if (!rows) return STATTN_OK;
    if (!out) return refuse(STATTN_EINVAL, "mx4_dequantize: null out");
    const OnDevice on(device);
    if (on.err != hipSuccess) return launched("mx4_dequantize", on.err);
    const Mx4View q{static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), rows, cols};
    return launched("mx4_dequantize", launch_mx4_dequantize(static_cast<hipStream_t>(stream), q, out, (OpType)dtype, ld_out));
}

static int product_ok(const char* who, int64_t m, int64_t n, int64_t k, const void* y, int dtype, int64_t ld_y) {
    if (!type_ok(dtype)) return refuse(STATTN_EINVAL, "%s: dtype %d is none of STATTN_F32, STATTN_BF16, STATTN_F16", who, dtype);
    if (ld_y < n || ld_y >= (int64_t)1 << 22) return refuse(STATTN_EINVAL, "%s: ld_y (%lld) must be at least n (%lld) and under 2^22", who, (long long)ld_y, (long long)n);
    if (m && n && !y) return refuse(STATTN_EINVAL, "%s: null y", who);
    // tiles are 64 x 64 at least, so a launch stays under 2^24 workgroups
    if ((m + 31) / 32 * ((n + 31) / 32) >= (int64_t)1 << 24) return refuse(STATTN_EINVAL, "%s: a product of %lld x %lld is too large for one call", who, (long long)m, (long long)n);
    (void)k;
    return STATTN_OK;
}

int stattn_mx4_matmul(int device, void* stream, const void* a_codes, const void* a_scales, const void* w_codes, const void* w_scales,
                      int64_t m, int64_t n, int64_t k, const float* bias, void* y, int dtype, int64_t ld_y) {
    OPCHK(form_ok("mx4_matmul (a)", a_codes, a_scales, m, k));
    OPCHK(form_ok("mx4_matmul (w)", w_codes, w_scales, n, k));
    OPCHK(product_ok("mx4_matmul", m, n, k, y, dtype, ld_y));
    if (!m || !n) return STATTN_OK;
    const OnDevice on(device);
    if (on.err != hipSuccess) return launched("mx4_matmul", on.err);
    const Mx4GemmArgs g{{static_cast<const uint8_t*>(a_codes), static_cast<const uint8_t*>(a_scales), m, k},
                        {static_cast<const uint8_t*>(w_codes), static_cast<const uint8_t*>(w_scales), n, k}, bias, y, (OpType)dtype, ld_y};
    return launched("mx4_matmul", launch_mx4_matmul(static_cast<hipStream_t>(stream), g));
}

// Few rows: one launch in which every workgroup rounds x for itself, instead of two with x's 4-bit form between them.  Up to 32768
// values of x that takes the GPU little longer (1 x 12000 x 512: 3.5 us against 5.1; 32: 6.0 against 5.6; 64: 9.1 against 5.8; beyond,
// 64 x 20000 x 1024: 18.5 against 7.4) and saves the caller a launch and a workspace, 4.5 us of its time.  Rows whose last eight are
// partial load one by one in between (64 x 12000 x 511: 12): up to 16384.  The rule is the eager caller's: replayed in a graph, where a
// launch and a workspace cost nothing more, two launches are the faster way from about 32 rows of 512 on (64 x 12000 x 512: 9.1 against 5.8).
static bool few_rows(int64_t m, int64_t k) { return m <= 64 && m * k <= (k % 8 ? 16384 : 32768); }

size_t stattn_mx4_linear_workspace(int64_t m, int64_t n, int64_t k) {
    (void)n;
    return m <= 0 || k <= 0 || few_rows(m, k) ? 0 : (size_t)(((m * mx4_kp(k) / 2 + 15) & ~(int64_t)15) + ((m * mx4_kp(k) / 32 + 15) & ~(int64_t)15));
}

int stattn_mx4_linear(int device, void* stream, const void* x, int dtype, int64_t ld_x, const void* w_codes, const void* w_scales,
                      int64_t m, int64_t n, int64_t k, const float* bias, void* y, int64_t ld_y, void* workspace, size_t workspace_bytes) {
    OPCHK(form_ok("mx4_linear (w)", w_codes, w_scales, n, k));
    if (m < 0 || m >= MAX_ROWS) return refuse(STATTN_EINVAL, "mx4_linear: %lld rows are outside 0 .. 2^31 - 1", (long long)m);
    OPCHK(product_ok("mx4_linear", m, n, k, y, dtype, ld_y));
    if (ld_x < k || !stride_ok(ld_x)) return refuse(STATTN_EINVAL, "mx4_linear: ld_x (%lld) must be at least k (%lld)", (long long)ld_x, (long long)k);
    if (!m || !n) return STATTN_OK;
    if (!x) return refuse(STATTN_EINVAL, "mx4_linear: null x");
    const size_t need = stattn_mx4_linear_workspace(m, n, k);
    if (need && (!workspace || !al16(workspace) || workspace_bytes < need))
        return refuse(STATTN_EINVAL, "mx4_linear: a 16-byte aligned workspace of %zu bytes is needed (got %zu)", need, workspace ? workspace_bytes : (size_t)0);
    const OnDevice on(device);
    if (on.err != hipSuccess) return launched("mx4_linear", on.err);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const Mx4View w{static_cast<const uint8_t*>(w_codes), static_cast<const uint8_t*>(w_scales), n, k};
    if (few_rows(m, k)) {
        const Mx4LinearArgs a{x, (OpType)dtype, m, ld_x, w, bias, y, ld_y};
        return launched("mx4_linear", launch_mx4_linear_few(s, a));
    }
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    uint8_t* scales = codes + ((m * mx4_kp(k) / 2 + 15) & ~(int64_t)15);
    const Mx4QuantArgs qa{x, (OpType)dtype, m, k, ld_x, 1, codes, scales};
    OPCHK(launched("mx4_linear", launch_mx4_quantize(s, qa)));
    const Mx4GemmArgs g{{codes, scales, m, k}, w, bias, y, (OpType)dtype, ld_y};
    return launched("mx4_linear", launch_mx4_matmul(s, g));
}

size_t stattn_verify_draft_workspace(int64_t b, int64_t j, int64_t v) {
    (void)j;
    const int n = b > 0 ? verify_split(b, v, OP_BF16) : 1;      // (32 bits are split for fewer captions)
    return n > 1 ? (size_t)b * 256 * sizeof(double) : 0;
}

int stattn_verify_draft(int device, void* stream, const int64_t* draft, int64_t draft_ld, const void* target, int64_t target_b,
                        int64_t target_j, const void* proposal, int64_t proposal_b, int64_t proposal_j, int dtype, const float* accept_u,
                        int64_t accept_ld, const float* draw_u, const int32_t* lens, int64_t b, int64_t j, int64_t v, int64_t* words,
                        int64_t words_ld, int32_t* accepted, void* workspace, size_t workspace_bytes) {
    if (!type_ok(dtype)) return refuse(STATTN_EINVAL, "verify_draft: dtype %d is none of STATTN_F32, STATTN_BF16, STATTN_F16", dtype);
    if (b < 0 || b >= ((int64_t)1 << 22) || j < 0 || j > 65535 || v < 1 || v >= MAX_ROWS)
        return refuse(STATTN_EINVAL, "verify_draft: b = %lld, j = %lld, v = %lld are outside b < 2^22, 0 <= j < 2^16, 1 <= v < 2^31", (long long)b, (long long)j, (long long)v);
    for (int64_t s : {draft_ld, target_b, target_j, proposal_b, proposal_j, accept_ld, words_ld})
        if (!stride_ok(s)) return refuse(STATTN_EINVAL, "verify_draft: strides must stay under 2^40 elements");
    if (words_ld < j + 1) return refuse(STATTN_EINVAL, "verify_draft: words_ld (%lld) must be at least j + 1", (long long)words_ld);
    if (!b) return STATTN_OK;
    if (!target || !draw_u || !words || !accepted || (j && (!draft || !accept_u))) return refuse(STATTN_EINVAL, "verify_draft: null argument");
    const size_t need = stattn_verify_draft_workspace(b, j, v);
    if (need && (!workspace || !al16(workspace) || workspace_bytes < need))
        return refuse(STATTN_EINVAL, "verify_draft: a 16-byte aligned workspace of %zu bytes is needed (got %zu)", need, workspace ? workspace_bytes : (size_t)0);
    const OnDevice on(device);
    if (on.err != hipSuccess) return launched("verify_draft", on.err);
    const VerifyArgs a{draft, draft_ld, 1, target, target_b, target_j, proposal, proposal_b, proposal_j, (OpType)dtype, accept_u, accept_ld, 1,
                       draw_u, lens, b, (int)j, v, words, words_ld, accepted, verify_split(b, v, (OpType)dtype), static_cast<double*>(workspace)};
    return launched("verify_draft", launch_verify_draft(static_cast<hipStream_t>(stream), a));
}

}  // extern "C"
