"""Plain implementations in 64 bits of the device-memory operators (stattn.ops), and the inputs their tests share."""
import numpy as np
import torch

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# a value rounded to the type is off by at most this, relative to itself
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def np64(t):
    return t.detach().double().cpu().numpy()


def quantize(x):
    """(codes as numbers 0..15 (rows, kp), scale bytes (rows, kp / 32)) of a float64 matrix, a block and a value at a time in numpy."""
    rows, cols = x.shape
    kp = -(-cols // 128) * 128
    pad = np.zeros((rows, kp))
    pad[:, :cols] = x
    b = pad.reshape(rows, kp // 32, 32)
    top = np.abs(b).max(2)
    bad = ~np.isfinite(b).all(2)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.floor(np.log2(np.where(bad | (top == 0), 1.0, top)))
    # log2 of a number just under a power of two may round up to it
    e -= (np.exp2(e) > np.where(bad | (top == 0), 1.0, top))
    byte = np.where(top == 0, 127, np.clip(e - 2, -126, 127) + 127)
    byte = np.where(bad, 255, byte).astype(np.int64)
    q = np.where(bad[:, :, None], 0.0, b) / np.exp2(np.where(bad, 0, byte - 127.0))[:, :, None]
    d = np.abs(np.abs(q)[..., None] - GRID)
    d[..., 1::2] += 1e-9 * (d[..., 1::2] > 0) * (np.abs(d[..., 1::2] - d.min(-1, keepdims=True)) == 0)   # ties to the even code
    code = d.argmin(-1) + 8 * np.signbit(q)
    code = np.where(bad[:, :, None], 0, code)
    return code.reshape(rows, kp), byte


def unpack(codes):
    c = codes.cpu().numpy().astype(np.int64)
    return np.stack((c & 15, c >> 4), 2).reshape(c.shape[0], -1)


def pack(code):
    return torch.from_numpy((code[:, 0::2] | code[:, 1::2] << 4).astype(np.uint8))


def values(code, byte, cols):
    """The numbers a (rows, kp) code array stands for."""
    v = np.where(code >= 8, -1.0, 1.0) * GRID[code & 7]
    s = np.where(byte == 255, np.nan, np.exp2(byte - 127.0))
    return (v.reshape(v.shape[0], -1, 32) * s[:, :, None]).reshape(v.shape[0], -1)[:, :cols]


def verify(draft, target, proposal, accept_u, draw_u, lens):
    """One caption after the other, one word after the other."""
    b, j1, v = target.shape
    words = np.full((b, j1), -1, np.int64)
    accepted = np.zeros(b, np.int32)
    for i in range(b):
        n, ln = 0, j1 - 1 if lens is None else min(max(int(lens[i]), 0), j1 - 1)
        while n < ln:
            d = int(draft[i, n])
            if not 0 <= d < v:
                break
            q = 1.0 if proposal is None else proposal[i, n, d]
            if not accept_u[i, n] * q < target[i, n, d]:
                break
            words[i, n] = d
            n += 1
        p = target[i, n]
        w = np.where(p > 0, p, 0.0)
        if n < ln:
            q = np.zeros(v) if proposal is None else proposal[i, n]
            if proposal is None and 0 <= int(draft[i, n]) < v:
                q[int(draft[i, n])] = 1.0
            with np.errstate(invalid="ignore"):
                rest = p - q
            rest = np.where(rest > 0, rest, 0.0)
            w = rest if rest.sum() > 0 else w
        c = np.cumsum(w.astype(np.longdouble))
        accepted[i] = n
        if c[-1] > 0:
            over = np.nonzero((c > np.longdouble(draw_u[i]) * c[-1]) & (w > 0))[0]
            words[i, n] = over[0] if len(over) else v - 1
    return words, accepted
