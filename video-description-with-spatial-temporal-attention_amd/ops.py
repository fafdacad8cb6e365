"""Operators on device memory (torch tensors): matrices in microscaled 4 bits, and drafted words checked against the decoder's own
next-word distribution -- the pieces of `Decoder.sample_drafted`, for programs that keep their tensors on the GPU.

    head = mx4_quantize(W, axis=0)                 # ff_logit_W (dim_word, n_words) -> a 4-bit head, one row per word
    logits = mx4_linear(x, head, bias=b)           # x (m, dim_word) float32 / bfloat16 / float16 -> (m, n_words) of the same type
    words, accepted = verify_draft(draft, target, proposal, accept_u, draw_u)

Every call forwards to one entry point of include/stattn.h, which states what is computed.  Work is enqueued on the current stream of
the tensors' device (which need not be the current device); results are new tensors.  Arguments of a wrong type raise TypeError, of a
wrong size or place ValueError; there is no CPU fallback."""
import torch

try:
    from . import _native
except ImportError:
    import _native

_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)


def _fail(rc):
    msg = _native.load_library().stattn_op_error().decode()
    raise ValueError(msg) if rc == -1 else _native.NativeError("libstattn error %d: %s" % (rc, msg))


def _float(t, name):
    if t.dtype not in _DTYPE:
        raise TypeError("%s must be float32, bfloat16 or float16 (got %s)" % (name, t.dtype))
    return _DTYPE[t.dtype]


def _place(device, **more):
    """The GPU index of `device`, after checking that every other tensor lives there too."""
    if device.type != "cuda":
        raise ValueError("the operators run on a GPU (got a tensor on %s)" % device)
    for name, t in more.items():
        if t is not None and t.device != device:
            raise ValueError("%s is on %s, not on %s" % (name, t.device, device))
    return device.index


class MX4(object):
    """A (rows, cols) matrix in microscaled 4 bits: `codes` (rows, kp / 2) and `scales` (rows, kp / 32), uint8, kp = cols rounded up to
    128.  Built by mx4_quantize, or from the two tensors of a matrix that was saved in this form."""
    __slots__ = ("codes", "scales", "cols")

    def __init__(self, codes, scales, cols):
        kp = -(-cols // 128) * 128
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("codes and scales must be uint8")
        if codes.dim() != 2 or codes.shape[1] * 2 != kp or tuple(scales.shape) != (codes.shape[0], kp // 32):
            raise ValueError("codes %s and scales %s do not hold %d columns: (rows, %d) and (rows, %d) are wanted"
                             % (tuple(codes.shape), tuple(scales.shape), cols, kp // 2, kp // 32))
        if not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError("codes and scales must be contiguous")
        self.codes, self.scales, self.cols = codes, scales, cols

    @property
    def rows(self):
        return self.codes.shape[0]

    @property
    def device(self):
        return self.codes.device

    def __repr__(self):
        return "MX4(%d x %d on %s)" % (self.rows, self.cols, self.device)


def mx4_quantize(x, axis=-1):
    """`x` (two dimensions, any strides) in 4 bits, blocks along `axis`: axis 1 keeps its rows, axis 0 gives a row per column of x (the
    form in which a weight stored (inputs, outputs) is multiplied)."""
    if x.dim() != 2:
        raise ValueError("x must have two dimensions")
    dtype, dev = _float(x, "x"), _place(x.device)
    if axis not in (-2, -1, 0, 1):
        raise ValueError("axis must be 0 or 1")
    (rows, cols), (rs, cs) = x.shape, x.stride()
    if axis in (0, -2):
        rows, cols, rs, cs = cols, rows, cs, rs
    kp = -(-cols // 128) * 128
    codes = torch.empty((rows, kp // 2), dtype=torch.uint8, device=x.device)
    scales = torch.empty((rows, kp // 32), dtype=torch.uint8, device=x.device)
    rc = _native.load_library().stattn_mx4_quantize(dev, _raw_stream(dev), x.data_ptr(), dtype, rows, cols, rs, cs, codes.data_ptr(), scales.data_ptr())
    if rc:
        _fail(rc)
    return MX4(codes, scales, cols)


def mx4_dequantize(q, dtype=torch.float32):
    """The numbers `q` stands for, (rows, cols) of `dtype`."""
    if dtype not in _DTYPE:
        raise TypeError("dtype must be float32, bfloat16 or float16 (got %s)" % dtype)
    dev = _place(q.codes.device, scales=q.scales)
    out = torch.empty((q.rows, q.cols), dtype=dtype, device=q.codes.device)
    rc = _native.load_library().stattn_mx4_dequantize(dev, _raw_stream(dev), q.codes.data_ptr(), q.scales.data_ptr(), q.rows, q.cols,
                                                      out.data_ptr(), _DTYPE[dtype], q.cols)
    if rc:
        _fail(rc)
    return out


def _bias(bias, n, device):
    if bias is None:
        return None
    if bias.dtype != torch.float32:
        raise TypeError("bias must be float32 (got %s)" % bias.dtype)
    if bias.dim() != 1 or bias.shape[0] != n or not bias.is_contiguous():
        raise ValueError("bias must be a contiguous vector of %d values" % n)
    if bias.device != device:
        raise ValueError("bias is on %s, not on %s" % (bias.device, device))
    return bias.data_ptr()


def mx4_matmul(a, w, bias=None, dtype=torch.float32):
    """a (m, k) times w (n, k) transposed, both MX4, plus bias (n,) float32: (m, n) of `dtype`."""
    if dtype not in _DTYPE:
        raise TypeError("dtype must be float32, bfloat16 or float16 (got %s)" % dtype)
    if a.cols != w.cols:
        raise ValueError("inner dimensions differ: %d and %d" % (a.cols, w.cols))
    device = a.codes.device
    dev = _place(device, a_scales=a.scales, w=w.codes, w_scales=w.scales)
    m, n = a.codes.shape[0], w.codes.shape[0]
    b = _bias(bias, n, device)
    y = torch.empty((m, n), dtype=dtype, device=device)
    rc = _native.load_library().stattn_mx4_matmul(dev, _raw_stream(dev), a.codes.data_ptr(), a.scales.data_ptr(), w.codes.data_ptr(),
                                                  w.scales.data_ptr(), m, n, a.cols, b, y.data_ptr(), _DTYPE[dtype], n)
    if rc:
        _fail(rc)
    return y


def mx4_linear(x, w, bias=None):
    """x (m, k) -- its rows may be strided, its columns not -- rounded to 4 bits on the way, times w (n, k) MX4 transposed, plus bias
    (n,) float32: (m, n) of x's type."""
    dtype = _float(x, "x")
    if x.dim() != 2 or x.shape[1] != w.cols:
        raise ValueError("x must be (m, %d), got %s" % (w.cols, tuple(x.shape)))
    m, k = x.shape
    ld = x.stride(0) if m > 1 else k
    if (k > 1 and x.stride(1) != 1) or ld < k:
        raise ValueError("the columns of x must be contiguous and its rows must not overlap")
    device = x.device
    dev = _place(device, w=w.codes, w_scales=w.scales)
    n = w.codes.shape[0]
    b = _bias(bias, n, device)
    lib = _native.load_library()
    y = torch.empty((m, n), dtype=x.dtype, device=device)
    need = lib.stattn_mx4_linear_workspace(m, n, k)
    work = torch.empty((need,), dtype=torch.uint8, device=device) if need else None
    rc = lib.stattn_mx4_linear(dev, _raw_stream(dev), x.data_ptr(), dtype, ld, w.codes.data_ptr(), w.scales.data_ptr(), m, n, k, b,
                               y.data_ptr(), n, work.data_ptr() if need else None, need)
    if rc:
        _fail(rc)
    return y


def verify_draft(draft, target, proposal, accept_u, draw_u, lens=None):
    """(words, accepted) of b captions with up to j drafted words each (stattn_verify_draft): draft (b, j) int64, target (b, j + 1, v) and
    proposal (b, j, v) -- None for arg-max drafts -- probabilities of one floating type with contiguous words, accept_u (b, j) and
    draw_u (b,) float32 in [0, 1), lens (b,) int32 or None.  words (b, j + 1) int64: the kept words, the drawn one, then -1;
    accepted (b,) int32: how many were kept."""
    dtype = _float(target, "target")
    if target.dim() != 3 or target.shape[1] < 1:
        raise ValueError("target must be (b, j + 1, v)")
    b, j, v = target.shape
    j -= 1
    if draft.dtype != torch.int64 or accept_u.dtype != torch.float32 or draw_u.dtype != torch.float32:
        raise TypeError("draft must be int64, accept_u and draw_u float32")
    if draft.shape != (b, j) or accept_u.shape != (b, j) or draw_u.shape != (b,):
        raise ValueError("draft and accept_u must be (%d, %d), draw_u (%d,)" % (b, j, b))
    if v > 1 and target.stride(2) != 1 or j > 1 and (draft.stride(1) != 1 or accept_u.stride(1) != 1) or b > 1 and draw_u.stride(0) != 1:
        raise ValueError("the last dimension of target, draft, accept_u and draw_u must be contiguous")
    pp = pb = pj = 0
    if proposal is not None:
        if proposal.dtype != target.dtype:
            raise TypeError("proposal must have target's type (%s), got %s" % (target.dtype, proposal.dtype))
        if proposal.shape != (b, j, v) or (v > 1 and proposal.stride(2) != 1):
            raise ValueError("proposal must be (%d, %d, %d) with contiguous words" % (b, j, v))
        pp, pb, pj = proposal.data_ptr(), proposal.stride(0), proposal.stride(1)
    if lens is not None and (lens.dtype != torch.int32 or lens.shape != (b,) or (b > 1 and lens.stride(0) != 1)):
        raise ValueError("lens must be a contiguous int32 vector of %d values" % b)
    device = target.device
    dev = _place(device, draft=draft, proposal=proposal, accept_u=accept_u, draw_u=draw_u, lens=lens)
    lib = _native.load_library()
    words = torch.empty((b, j + 1), dtype=torch.int64, device=device)
    accepted = torch.empty((b,), dtype=torch.int32, device=device)
    need = lib.stattn_verify_draft_workspace(b, j, v)
    work = torch.empty((need,), dtype=torch.uint8, device=device) if need else None
    rc = lib.stattn_verify_draft(dev, _raw_stream(dev), draft.data_ptr(), draft.stride(0), target.data_ptr(), target.stride(0),
                                 target.stride(1), pp, pb, pj, dtype, accept_u.data_ptr(), accept_u.stride(0), draw_u.data_ptr(),
                                 None if lens is None else lens.data_ptr(), b, j, v, words.data_ptr(), j + 1, accepted.data_ptr(),
                                 work.data_ptr() if need else None, need)
    if rc:
        _fail(rc)
    return words, accepted
