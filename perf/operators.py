"""Cases and plain forms of the device-memory operators of the caption sampler (stattn.ops): microscaled 4-bit numbers -- written,
read back, multiplied -- and the check of drafted words against the decoder's own next-word probabilities.

The number format (OCP microscaling, MXFP4): a row is cut into blocks of 32 columns; a block holds 32 four-bit codes (sign, two bits
of exponent, one of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6) and one byte s, the power of two 2^(s - 127) that its values share.  The
scale of a block whose largest magnitude is a is 2^(floor(log2 a) - 2); values are rounded to the nearest code, ties to the even code,
magnitudes beyond 6 to 6.  In memory: codes (rows, Kp / 2) bytes, the even column in the low half, scales (rows, Kp / 32) bytes, Kp the
columns rounded up to 128; columns behind the last one hold code 0."""
import math

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # the decoder's vocabulary projection ff_logit_W (512 x 12000, stored input-major) turned into a 4-bit head and read back
        dict(name="readback_head_f32", op="readback", rows=12000, cols=512, axis=0, dtype="float32"),
        # region features of a batch (64 videos x 26 frames x 8 regions, 4096 features) as activations
        dict(name="readback_regions_bf16", op="readback", rows=13312, cols=4096, axis=1, dtype="bfloat16"),
        # one word of one caption through the 4-bit vocabulary head: the smallest call, all latency
        dict(name="linear_word_f32", op="linear", m=1, n=12000, k=512, dtype="float32", bias=True),
        # a beam of five hypotheses, hidden size 1024, the 20000-word vocabulary
        dict(name="linear_beam5_bf16", op="linear", m=5, n=20000, k=1024, dtype="bfloat16", bias=True),
        # 32 videos x beam 5, one word
        dict(name="linear_beams160_f32", op="linear", m=160, n=12000, k=512, dtype="float32", bias=True),
        # a batch's region features projected 4096 -> 1024
        dict(name="linear_regions_bf16", op="linear", m=13312, n=1024, k=4096, dtype="bfloat16", bias=True),
        # odd sizes: a tail in every dimension
        dict(name="product_odd_f16", op="product", m=1001, n=1777, k=1111, dtype="float16", bias=False),
        # readout of a whole batch of captions (64 x 30 rows), both sides already in 4 bits, logits in fp32
        dict(name="product_readout_f32", op="product", m=1920, n=12000, k=512, dtype="float32", bias=True),
        # the largest product
        dict(name="product_large_bf16", op="product", m=8192, n=8192, k=8192, dtype="bfloat16", bias=False),
        # one caption, four drafted words
        dict(name="verify_one_f32", op="verify", b=1, j=4, v=12000, dtype="float32"),
        # the captions of a batch, drafts of unequal length
        dict(name="verify_batch_f32", op="verify", b=64, j=5, v=20000, dtype="float32"),
        # many sequences, a large vocabulary, probabilities kept in bf16
        dict(name="verify_wide_bf16", op="verify", b=128, j=7, v=128000, dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("readback", "linear", "linear", "product", "product", "verify", "verify"))
    dtype = rng.choice(sorted(DTYPES))
    if op == "readback":
        rows, cols = _log(rng, 1, 16384), _log(rng, 1, 8192)
        return dict(op=op, rows=min(rows, max(1, 13312 * 4096 // cols)), cols=cols, axis=rng.randrange(2), dtype=dtype)
    if op == "verify":
        b, j, v = _log(rng, 1, 128), rng.randrange(0, 9), _log(rng, 50, 128000)
        return dict(op=op, b=b, j=min(j, max(0, (1 << 26) // (b * v) - 1)), v=v, dtype=dtype)
    if op == "linear":      # as in decoding: few rows as often as many
        m, n, k = _log(rng, 1, 32) if rng.random() < 0.5 else _log(rng, 17, 13000), _log(rng, 16, 20000), _log(rng, 16, 8192)
        most = 13312 * 1024 * 4096
    else:
        m, n, k = _log(rng, 1, 8192), _log(rng, 16, 20000), _log(rng, 16, 8192)
        most = 1 << 38
    m = max(1, min(m, most // (n * k), (1 << 27) // n))
    return dict(op=op, m=m, n=n, k=k, dtype=dtype, bias=rng.random() < 0.5)


def _codes(x):
    """(codes, scales) of the rows of a float32 tensor, in the layout above."""
    rows, cols = x.shape
    kp = -(-cols // 128) * 128
    b = torch.zeros(rows, kp, device=x.device)
    b[:, :cols] = x
    b = b.view(rows, kp // 32, 32)
    e = torch.frexp(b.abs().amax(2))[1] - 3                    # frexp gives [0.5, 1): floor(log2 a) is one less than its exponent
    e = torch.where(b.abs().amax(2) > 0, e, torch.zeros_like(e)).clamp(-126, 127)
    q = torch.ldexp(b, -e[:, :, None])
    mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device)
    mag = torch.bucketize(q.abs(), mid, right=False)           # a midpoint goes to the lower code ...
    tie = (q.abs() == mid[mag.clamp(max=6)]) & (mag % 2 == 1)  # ... unless that is the odd one
    c = (mag + tie + 8 * torch.signbit(q)).to(torch.uint8).view(rows, kp)
    return (c[:, 0::2] | (c[:, 1::2] << 4)).contiguous(), (e + 127).to(torch.uint8)


def _values(codes, scales, cols, f=torch.float32):
    """The numbers that (codes, scales) stand for: (rows, cols) in f."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), dtype=f, device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), 2).view(codes.shape[0], -1)
    v = grid[c.long()].view(codes.shape[0], -1, 32)
    return torch.ldexp(v, scales.int()[:, :, None] - 127).reshape(codes.shape[0], -1)[:, :cols]


def _rounded(x):
    """Rows of a float32 tensor rounded to the format: what writing and reading back gives."""
    rows, cols = x.shape
    b = torch.nn.functional.pad(x, (0, -cols % 32)).view(rows, -1, 32)
    a = b.abs().amax(2, keepdim=True)
    e = torch.where(a > 0, torch.frexp(a)[1] - 3, 0).clamp(-126, 127)
    q = torch.ldexp(b, -e)
    m = q.abs()
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    m = (torch.round(m / step) * step).clamp(max=6.0)          # round() takes ties to even, which is the even code
    return torch.ldexp(torch.copysign(m, q), e).view(rows, -1)[:, :cols]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = dict(case=case)
    if case["op"] == "readback":
        rows, cols = case["rows"], case["cols"]
        x = normal(rows, cols) * torch.exp2(3 * normal(rows, 1))          # rows of unequal scale
        s["x"] = (x.t() if case["axis"] == 0 else x).to(dt).contiguous()
        return s
    if case["op"] in ("linear", "product"):
        m, n, k = case["m"], case["n"], case["k"]
        x = torch.tanh(normal(m, k)) * torch.exp2(normal(m, 1))
        s["w"] = _codes(normal(n, k) * k ** -0.5)                         # weights laid out once, as a program keeps them
        s["x"] = x.to(dt) if case["op"] == "linear" else _codes(x)
        s["bias"] = normal(n) if case["bias"] else None
        return s
    b, j, v = case["b"], case["j"], case["v"]
    logit = 3 * normal(b, j + 1, v)
    draft = logit[:, :j] + 0.7 * normal(b, j, v)                          # the draft is near the target, not equal to it
    target, proposal = torch.softmax(logit, 2), torch.softmax(draft, 2)
    noise = -torch.log(-torch.log(uniform(b, j, v).clamp(1e-20, 1 - 1e-7)))
    s["draft"] = (draft + noise).argmax(2) if j else torch.zeros(b, 0, dtype=torch.int64, device="cuda")
    s["target"], s["proposal"] = target.to(dt), proposal.to(dt)
    s["accept_u"], s["draw_u"] = uniform(b, j), uniform(b)
    s["lens"] = torch.randint(0, j + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    s["lens"][0] = j
    return s


def _plain_verify(s):
    target, proposal, draft, lens = s["target"], s["proposal"], s["draft"], s["lens"].long()
    b, j1, v = target.shape
    j = j1 - 1
    rows = torch.arange(b, device=target.device)
    n = torch.zeros_like(lens)
    if j:
        p = target[:, :j].gather(2, draft[:, :, None])[:, :, 0].double()
        q = proposal.gather(2, draft[:, :, None])[:, :, 0].double()
        live = torch.arange(j, device=target.device) < lens[:, None]
        n = ((s["accept_u"].double() * q < p) & live).long().cumprod(1).sum(1)
    p = target[rows, n].double()
    w = p
    if j:
        rest = (p - proposal[rows, n.clamp(max=j - 1)].double()).clamp(min=0)
        rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, p)
        w = torch.where((n < lens)[:, None], rest, p)
    c = w.cumsum(1)
    word = torch.searchsorted(c, (s["draw_u"].double() * c[:, -1])[:, None], right=True)[:, 0].clamp(max=v - 1)
    at = torch.arange(j1, device=target.device)
    kept = torch.cat((draft, draft.new_zeros(b, 1)), 1)
    words = torch.where(at < n[:, None], kept, torch.where(at == n[:, None], word[:, None], -1))
    return {"words": words, "accepted": n.int()}


def run(s):
    case = s["case"]
    op, dt = case["op"], DTYPES[case["dtype"]]
    if own:
        from stattn import ops
        if op == "readback":
            return ops.mx4_dequantize(ops.mx4_quantize(s["x"], axis=case["axis"]), dtype=dt)
        if op == "linear":
            return ops.mx4_linear(s["x"], ops.MX4(*s["w"], case["k"]), bias=s["bias"])
        if op == "product":
            return ops.mx4_matmul(ops.MX4(*s["x"], case["k"]), ops.MX4(*s["w"], case["k"]), bias=s["bias"], dtype=dt)
        words, accepted = ops.verify_draft(s["draft"], s["target"], s["proposal"], s["accept_u"], s["draw_u"], lens=s["lens"])
        return {"words": words, "accepted": accepted}
    if op == "readback":
        x = s["x"].t() if case["axis"] == 0 else s["x"]
        return _rounded(x.float()).to(dt)
    if op == "verify":
        return _plain_verify(s)
    x = _rounded(s["x"].float()) if op == "linear" else _values(*s["x"], case["k"])
    y = x @ _values(*s["w"], case["k"]).t()
    return (y + s["bias"] if s["bias"] is not None else y).to(dt)


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "readback":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (2 * e + 2 * (0.5 + 1 / 32)), "flops": 4 * n}       # values in and out, the 4-bit form written and read
    if case["op"] == "verify":
        b, j, v = case["b"], case["j"], case["v"]
        # one row of the target a sequence, one of the proposal as well where a word was refused, the drafted words' own probabilities
        return {"bytes": b * (v * e * (2 if j else 1) + j * (8 + 2 * e + 4) + 8 * (j + 1) + 12), "flops": b * v * 3}
    m, n, k = case["m"], case["n"], case["k"]
    side = k * (0.5 + 1 / 32)
    return {"bytes": m * (k * e if case["op"] == "linear" else side) + n * side + m * n * e + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}


def _exact_rounded(x):
    """Rounding to the format by the nearest of the sixteen numbers of each block, in 64 bits."""
    rows, cols = x.shape
    b = torch.zeros(rows, -(-cols // 32) * 32, dtype=torch.float64, device=x.device)
    b[:, :cols] = x
    b = b.view(rows, -1, 32)
    scale = torch.exp2((torch.floor(torch.log2(b.abs().amax(2, keepdim=True).clamp(min=1e-300))) - 2).clamp(-126, 127))
    m = b.abs() / scale
    # a midpoint goes to the even one of its two codes: past it for the lower one, from it on for the upper one
    near = 0.5 * ((m > 0.25).double() + (m >= 0.75) + (m > 1.25) + (m >= 1.75)) + (m > 2.5).double() + (m >= 3.5) + 2 * (m > 5)
    return (torch.sign(b) * near * scale).view(rows, -1)[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "readback":
        x = s["x"].double()
        return _exact_rounded(x.t() if case["axis"] == 0 else x)
    if case["op"] in ("linear", "product"):
        if case["op"] == "linear":
            x = _exact_rounded(s["x"].double())
        else:
            x = _exact_read(*s["x"], case["k"])
        y = x @ _exact_read(*s["w"], case["k"]).t().contiguous()
        return y if s["bias"] is None else y + s["bias"].double()
    # a caption at a time: walk the draft, then walk the weights of the word behind it
    words, accepted = [], []
    t = {k: (v.double() if v.is_floating_point() else v).cpu().numpy() for k, v in s.items() if k in ("draft", "accept_u", "draw_u", "lens")}
    for i in range(case["b"]):
        p, q = s["target"][i].double().cpu().numpy(), s["proposal"][i].double().cpu().numpy()
        n = 0
        while n < t["lens"][i] and t["accept_u"][i, n] * q[n, t["draft"][i, n]] < p[n, t["draft"][i, n]]:
            n += 1
        w = p[n]
        if n < t["lens"][i]:
            rest = np.maximum(p[n] - q[n], 0.0)
            w = rest if rest.any() else w
        c = np.add.accumulate(w.astype(np.longdouble))
        word = min(int(np.count_nonzero(c <= t["draw_u"][i] * c[-1])), case["v"] - 1)
        words.append(list(t["draft"][i, :n]) + [word] + [-1] * (case["j"] - n))
        accepted.append(n)
    return {"words": torch.tensor(np.array(words, np.int64)), "accepted": torch.tensor(accepted, dtype=torch.int32)}


def _exact_read(codes, scales, cols):
    """The numbers of (codes, scales) in 64 bits, from the bits of a code: (-1)^s 2^(e - 1) (1 + m / 2), or (-1)^s m / 2 where e = 0."""
    c = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    c[:, 0::2], c[:, 1::2] = (codes % 16).double(), torch.div(codes, 16, rounding_mode="floor").double()
    neg = c >= 8
    c = c - 8 * neg
    e, m = torch.floor(c / 2), c % 2
    mag = torch.where(e > 0, torch.exp2(e - 1) * (1 + m / 2), m / 2)
    scale = torch.exp2(scales.double() - 127).repeat_interleave(32, 1)
    return (torch.where(neg, -mag, mag) * scale)[:, :cols]
