"""Operators on device memory (torch tensors): matrices in microscaled 4 bits, and drafted words checked against the decoder's own
next-word distribution -- the pieces of `Decoder.sample_drafted`, for programs that keep their tensors on the GPU.

    head = mx4_quantize(W, axis=0)                 # ff_logit_W (dim_word, n_words) -> a 4-bit head, one row per word
    logits = mx4_linear(x, head, bias=b)           # x (m, dim_word) float32 / bfloat16 / float16 -> (m, n_words) of the same type
    words, accepted = verify_draft(draft, target, proposal, accept_u, draw_u)

Every call forwards to one entry point of include/stattn.h, which states what is computed.  Work is enqueued on the current stream of
the tensors' device (which need not be the current device); results are new tensors.  Arguments of a wrong type raise TypeError, of a
wrong size or place ValueError; there is no CPU fallback.  A view whose sign torch keeps beside the memory (is_neg(): z.conj().imag) is
written out first.

These are operators of decoding: none has a gradient.  A product of tensors that record one (x or bias with requires_grad, outside
torch.no_grad()) is computed all the same, and its backward raises RuntimeError; forward-mode tangents raise at the call.  The 4-bit form
and the words of verify_draft are whole numbers, through which nothing is differentiated, as through any cast to integers in torch."""
import torch
from torch.autograd import forward_ad

try:
    from . import _native
except ImportError:
    import _native

_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)
_U8, _F32, _I32, _I64 = torch.uint8, torch.float32, torch.int32, torch.int64
# The checks below are written out, plain comparisons on the way of a good call: of the 7 us that a small product takes a caller, 3.5 are
# the launch and 1.7 the result's allocation.


def _fail(rc):
    msg = _native.load_library().stattn_op_error().decode()
    raise ValueError(msg) if rc == -1 else _native.NativeError("libstattn error %d: %s" % (rc, msg))


def _wrong_type(name, t):
    raise TypeError("%s must be float32, bfloat16 or float16 (got %s)" % (name, t))


def _wrong_place(dev, **tensors):
    """Names the tensor that is not on GPU number `dev` (-1: not on a GPU)."""
    if dev < 0:
        raise ValueError("the operators run on a GPU (got tensors on the host)")
    for name, t in tensors.items():
        if t is not None and t.get_device() != dev:
            raise ValueError("%s is on %s, not on cuda:%d" % (name, t.device, dev))


class _NoGradient(torch.autograd.Function):
    """The tensor in `box` as it is, on the record of those it was computed from: a backward pass through it fails instead of leaving them
    out.  (In a box, since an input that is handed back would be a view, and could not be written in place.)"""

    @staticmethod
    def forward(ctx, box, name, *inputs):
        ctx.name = name
        return box[0]

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("%s has no gradient: call it under torch.no_grad() or on detached tensors" % ctx.name)


def _tangent(name, *tensors):
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("%s has no derivative (an argument carries a forward-mode tangent)" % name)


class MX4(object):
    """A (rows, cols) matrix in microscaled 4 bits: `codes` (rows, kp / 2) and `scales` (rows, kp / 32), uint8, kp = cols rounded up to
    128.  Built by mx4_quantize, or from the two tensors of a matrix that was saved in this form."""
    __slots__ = ("codes", "scales", "cols")

    def __init__(self, codes, scales, cols):
        kb = (cols + 127) // 128 * 4
        shape = codes.shape
        if codes.dtype != _U8 or scales.dtype != _U8:
            raise TypeError("codes and scales must be uint8")
        if len(shape) != 2 or cols < 1 or shape[1] != 16 * kb or scales.shape != (shape[0], kb):
            raise ValueError("codes %s and scales %s do not hold %d columns: (rows, %d) and (rows, %d) are wanted"
                             % (tuple(shape), tuple(scales.shape), cols, 16 * kb, kb))
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


def _made(codes, scales, cols):         # an MX4 of tensors made here
    q = MX4.__new__(MX4)
    q.codes, q.scales, q.cols = codes, scales, cols
    return q


def mx4_quantize(x, axis=-1):
    """`x` (two dimensions, any strides) in 4 bits, blocks along `axis`: axis 1 keeps its rows, axis 0 gives a row per column of x (the
    form in which a weight stored (inputs, outputs) is multiplied)."""
    dtype = _DTYPE.get(x.dtype)
    if dtype is None:
        _wrong_type("x", x.dtype)
    if x.dim() != 2:
        raise ValueError("x must have two dimensions")
    if axis not in (-2, -1, 0, 1):
        raise ValueError("axis must be 0 or 1")
    if x.is_neg():
        x = x.resolve_neg()
    dev = x.get_device()
    if dev < 0:
        _wrong_place(dev)
    (rows, cols), (rs, cs) = x.shape, x.stride()
    if axis in (0, -2):
        rows, cols, rs, cs = cols, rows, cs, rs
    kb = (cols + 127) // 128 * 4
    codes = x.new_empty((rows, 16 * kb), dtype=_U8)
    scales = codes.new_empty((rows, kb))
    rc = _native.load_library().stattn_mx4_quantize(dev, _raw_stream(dev), x.data_ptr(), dtype, rows, cols, rs, cs, codes.data_ptr(), scales.data_ptr())
    if rc:
        _fail(rc)
    return _made(codes, scales, cols)


def mx4_dequantize(q, dtype=torch.float32):
    """The numbers `q` stands for, (rows, cols) of `dtype`."""
    t = _DTYPE.get(dtype)
    if t is None:
        _wrong_type("dtype", dtype)
    codes, scales, cols = q.codes, q.scales, q.cols
    dev = codes.get_device()
    if dev < 0 or scales.get_device() != dev:
        _wrong_place(dev, scales=scales)
    rows = codes.shape[0]
    out = codes.new_empty((rows, cols), dtype=dtype)
    rc = _native.load_library().stattn_mx4_dequantize(dev, _raw_stream(dev), codes.data_ptr(), scales.data_ptr(), rows, cols, out.data_ptr(), t, cols)
    if rc:
        _fail(rc)
    return out


def _check_bias(bias, n, dev):
    if bias.dtype != _F32:
        raise TypeError("bias must be float32 (got %s)" % bias.dtype)
    if bias.shape != (n,) or not bias.is_contiguous():
        raise ValueError("bias must be a contiguous vector of %d values" % n)
    if bias.get_device() != dev:
        _wrong_place(dev, bias=bias)
    return bias.resolve_neg()           # itself, unless is_neg()


def mx4_matmul(a, w, bias=None, dtype=torch.float32):
    """a (m, k) times w (n, k) transposed, both MX4, plus bias (n,) float32: (m, n) of `dtype`."""
    t = _DTYPE.get(dtype)
    if t is None:
        _wrong_type("dtype", dtype)
    k = a.cols
    if k != w.cols:
        raise ValueError("inner dimensions differ: %d and %d" % (k, w.cols))
    ac, as_, wc, ws = a.codes, a.scales, w.codes, w.scales
    dev = ac.get_device()
    if dev < 0 or as_.get_device() != dev or wc.get_device() != dev or ws.get_device() != dev:
        _wrong_place(dev, a_scales=as_, w=wc, w_scales=ws)
    m, n = ac.shape[0], wc.shape[0]
    if bias is not None:
        bias = _check_bias(bias, n, dev)
    if forward_ad._current_level >= 0:
        _tangent("mx4_matmul", bias)
    y = ac.new_empty((m, n), dtype=dtype)
    rc = _native.load_library().stattn_mx4_matmul(dev, _raw_stream(dev), ac.data_ptr(), as_.data_ptr(), wc.data_ptr(), ws.data_ptr(), m, n, k,
                                                  None if bias is None else bias.data_ptr(), y.data_ptr(), t, n)
    if rc:
        _fail(rc)
    if bias is not None and bias.requires_grad and torch.is_grad_enabled():
        return _NoGradient.apply([y], "mx4_matmul", bias)
    return y


def mx4_linear(x, w, bias=None):
    """x (m, k) -- its rows may be strided, its columns not -- rounded to 4 bits on the way, times w (n, k) MX4 transposed, plus bias
    (n,) float32: (m, n) of x's type."""
    dtype = _DTYPE.get(x.dtype)
    if dtype is None:
        _wrong_type("x", x.dtype)
    shape, k = x.shape, w.cols
    if len(shape) != 2 or shape[1] != k:
        raise ValueError("x must be (m, %d), got %s" % (k, tuple(shape)))
    if x.is_neg():
        x = x.resolve_neg()
    m = shape[0]
    ld, one = x.stride()
    if m <= 1:
        ld = k
    if (k > 1 and one != 1) or ld < k:
        raise ValueError("the columns of x must be contiguous and its rows must not overlap")
    wc, ws = w.codes, w.scales
    dev = x.get_device()
    if dev < 0 or wc.get_device() != dev or ws.get_device() != dev:
        _wrong_place(dev, w=wc, w_scales=ws)
    n = wc.shape[0]
    if bias is not None:
        bias = _check_bias(bias, n, dev)
    if forward_ad._current_level >= 0:
        _tangent("mx4_linear", x, bias)
    lib = _native.load_library()
    y = x.new_empty((m, n))
    need = lib.stattn_mx4_linear_workspace(m, n, k)
    work = x.new_empty((need,), dtype=_U8) if need else None        # alive until the launches are enqueued
    rc = lib.stattn_mx4_linear(dev, _raw_stream(dev), x.data_ptr(), dtype, ld, wc.data_ptr(), ws.data_ptr(), m, n, k,
                               None if bias is None else bias.data_ptr(), y.data_ptr(), n, work.data_ptr() if need else None, need)
    if rc:
        _fail(rc)
    if (x.requires_grad or bias is not None and bias.requires_grad) and torch.is_grad_enabled():
        return _NoGradient.apply([y], "mx4_linear", x, bias)
    return y


def verify_draft(draft, target, proposal, accept_u, draw_u, lens=None):
    """(words, accepted) of b captions with up to j drafted words each (stattn_verify_draft): draft (b, j) int64, target (b, j + 1, v) and
    proposal (b, j, v) -- None for arg-max drafts -- probabilities of one floating type with contiguous words, accept_u (b, j) and
    draw_u (b,) float32 in [0, 1), lens (b,) int32 or None.  words (b, j + 1) int64: the kept words, the drawn one, then -1;
    accepted (b,) int32: how many were kept.  (lens of another type or size: ValueError.)"""
    dtype = _DTYPE.get(target.dtype)
    if dtype is None:
        _wrong_type("target", target.dtype)
    shape = target.shape
    if len(shape) != 3 or shape[1] < 1:
        raise ValueError("target must be (b, j + 1, v)")
    b, j, v = shape
    j -= 1
    if draft.dtype != _I64 or accept_u.dtype != _F32 or draw_u.dtype != _F32:
        raise TypeError("draft must be int64, accept_u and draw_u float32")
    if draft.shape != (b, j) or accept_u.shape != (b, j) or draw_u.shape != (b,):
        raise ValueError("draft and accept_u must be (%d, %d), draw_u (%d,)" % (b, j, b))
    if target.is_neg() or accept_u.is_neg() or draw_u.is_neg():
        target, accept_u, draw_u = target.resolve_neg(), accept_u.resolve_neg(), draw_u.resolve_neg()
    tb, tj, tv = target.stride()
    db, dj = draft.stride()
    ub, uj = accept_u.stride()
    if v > 1 and tv != 1 or j > 1 and (dj != 1 or uj != 1) or b > 1 and draw_u.stride(0) != 1:
        raise ValueError("the last dimension of target, draft, accept_u and draw_u must be contiguous")
    pp, pb, pj = None, 0, 0
    dev = target.get_device()
    wrong = dev < 0 or draft.get_device() != dev or accept_u.get_device() != dev or draw_u.get_device() != dev
    if proposal is not None:
        if proposal.dtype != target.dtype:
            raise TypeError("proposal must have target's type (%s), got %s" % (target.dtype, proposal.dtype))
        if proposal.is_neg():
            proposal = proposal.resolve_neg()
        pb, pj, pv = proposal.stride() if proposal.dim() == 3 else (0, 0, 0)
        if proposal.shape != (b, j, v) or (v > 1 and pv != 1):
            raise ValueError("proposal must be (%d, %d, %d) with contiguous words" % (b, j, v))
        pp = proposal.data_ptr()
        wrong = wrong or proposal.get_device() != dev
    pl = None
    if lens is not None:
        if lens.dtype != _I32 or lens.shape != (b,) or (b > 1 and lens.stride(0) != 1):
            raise ValueError("lens must be a contiguous int32 vector of %d values" % b)
        pl = lens.data_ptr()
        wrong = wrong or lens.get_device() != dev
    if wrong:
        _wrong_place(dev, draft=draft, proposal=proposal, accept_u=accept_u, draw_u=draw_u, lens=lens)
    words = draft.new_empty((b, j + 1))
    accepted = draft.new_empty((b,), dtype=_I32)
    lib = _native.load_library()
    need = lib.stattn_verify_draft_workspace(b, j, v)
    work = draft.new_empty((need,), dtype=_U8) if need else None        # alive until the launches are enqueued
    rc = lib.stattn_verify_draft(dev, _raw_stream(dev), draft.data_ptr(), db, target.data_ptr(), tb, tj, pp, pb, pj, dtype, accept_u.data_ptr(), ub,
                                 draw_u.data_ptr(), pl, b, j, v, words.data_ptr(), j + 1, accepted.data_ptr(), work.data_ptr() if need else None, need)
    if rc:
        _fail(rc)
    return words, accepted
