"""The device-memory operators on a box without a GPU: every call that an entry point must refuse is refused before anything is
launched, and the plain implementations the GPU tests compare with are right."""
import ctypes as C
import itertools

import numpy as np
import pytest
import torch

from stattn import _native, ops
import ops_reference as R

A = 1 << 20        # a pointer that is aligned and never followed: each call below is refused before it would be


def lib():
    return _native.load_library()


def refused(rc, *words):
    msg = lib().stattn_op_error().decode()
    assert rc == -1, (rc, msg)
    for w in words:
        assert w in msg, msg


def test_quantize_refusals():
    f = lib().stattn_mx4_quantize
    refused(f(0, None, A, 3, 4, 32, 32, 1, A, A), "dtype")
    refused(f(0, None, A, 0, -1, 32, 32, 1, A, A), "rows")
    refused(f(0, None, A, 0, 4, 0, 32, 1, A, A), "columns")
    refused(f(0, None, A, 0, 4, (1 << 24) + 1, 32, 1, A, A), "columns")
    refused(f(0, None, A, 0, 4, 32, 32, 1, None, A), "null")
    refused(f(0, None, A, 0, 4, 32, 32, 1, A, None), "null")
    refused(f(0, None, None, 0, 4, 32, 32, 1, A, A), "null x")
    refused(f(0, None, A, 0, 4, 32, 32, 1, A + 8, A), "aligned")
    refused(f(0, None, A, 0, 4, 32, 1 << 41, 1, A, A), "strides")
    assert f(0, None, None, 0, 0, 32, 32, 1, None, None) == 0          # no rows: nothing to do


def test_dequantize_refusals():
    f = lib().stattn_mx4_dequantize
    refused(f(0, None, A, A, 4, 33, A, 0, 32), "ld_out")
    refused(f(0, None, A, A, 4, 32, None, 0, 32), "null out")
    refused(f(0, None, A, A, 4, 32, A, -1, 32), "dtype")
    refused(f(0, None, None, A, 4, 32, A, 0, 32), "null")
    assert f(0, None, None, None, 0, 32, None, 0, 32) == 0


def test_matmul_and_linear_refusals():
    f = lib().stattn_mx4_matmul
    refused(f(0, None, A, A, A, A, 4, 8, 32, None, A, 0, 7), "ld_y")
    refused(f(0, None, A, A, A, A, 4, 8, 32, None, A, 0, 1 << 22), "ld_y")
    refused(f(0, None, A, A, A, A, 4, 8, 32, None, A, 9, 8), "dtype")
    refused(f(0, None, A, A, A, A, 4, 8, 32, None, None, 0, 8), "null y")
    refused(f(0, None, A, A, A, A + 2, 4, 8, 32, None, A, 0, 8), "aligned")
    refused(f(0, None, A, A, A + 8, A, 4, 8, 32, None, A, 0, 8), "aligned")
    refused(f(0, None, A, A, A, A, 1 << 20, 1 << 20, 32, None, A, 0, 1 << 20), "too large")
    refused(f(0, None, None, A, A, A, 4, 8, 32, None, A, 0, 8), "null")
    assert f(0, None, None, None, A, A, 0, 8, 32, None, None, 0, 8) == 0
    g, need = lib().stattn_mx4_linear, lib().stattn_mx4_linear_workspace
    assert need(0, 8, 32) == 0
    n = need(300, 1024, 4096)
    refused(g(0, None, A, 0, 31, A, A, 300, 1024, 32, None, A, 1024, A, 1 << 30), "ld_x")
    if n:
        refused(g(0, None, A, 0, 4096, A, A, 300, 1024, 4096, None, A, 1024, A, n - 1), "workspace")
        refused(g(0, None, A, 0, 4096, A, A, 300, 1024, 4096, None, A, 1024, None, n), "workspace")
        refused(g(0, None, A, 0, 4096, A, A, 300, 1024, 4096, None, A, 1024, A + 8, n), "workspace")
    refused(g(0, None, None, 0, 32, A, A, 300, 1024, 32, None, A, 1024, A, 1 << 30), "null x")
    refused(g(0, None, A, 0, 32, A, A, -1, 1024, 32, None, A, 1024, A, 1 << 30), "rows")


def test_verify_refusals():
    f = lib().stattn_verify_draft

    def call(b=2, j=3, v=10, dtype=0, draft=A, target=A, proposal=A, au=A, du=A, words=A, ld=4, acc=A, ws=A, nws=1 << 30):
        return f(0, None, draft, j, target, (j + 1) * v, v, proposal, j * v, v, dtype, au, j, du, None, b, j, v, words, ld, acc, ws, nws)
    refused(call(dtype=5), "dtype")
    refused(call(v=0), "v = 0")
    refused(call(j=-1), "j = -1")
    refused(call(j=1 << 16, ld=1 << 20), "j = ")
    refused(call(b=-1), "b = -1")
    refused(call(ld=3), "words_ld")
    for name in ("draft", "target", "au", "du", "words", "acc"):
        refused(call(**{name: None}), "null")
    need = lib().stattn_verify_draft_workspace(2, 3, 200000)
    assert need and not lib().stattn_verify_draft_workspace(2, 3, 20000)
    refused(call(v=200000, nws=need - 1), "workspace")
    refused(call(v=200000, ws=None), "workspace")
    refused(call(v=200000, ws=A + 4), "workspace")
    assert call(b=0) == 0


def test_python_refusals():
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="GPU"):
        ops.mx4_quantize(x)
    with pytest.raises(TypeError):
        ops.mx4_quantize(x.double())
    with pytest.raises(ValueError, match="dimensions"):
        ops.mx4_quantize(x[0])
    c, s = torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8)
    q = ops.MX4(c, s, 100)
    assert q.rows == 4 and q.cols == 100
    for bad in ((c, s, 129), (c, s, 0), (c[:, :32], s, 100), (c, s[:3], 100), (c.t(), s, 100)):
        with pytest.raises(ValueError):
            ops.MX4(*bad)
    with pytest.raises(TypeError):
        ops.MX4(c.int(), s, 100)
    with pytest.raises(TypeError):
        ops.mx4_dequantize(q, torch.float64)
    with pytest.raises(ValueError, match="GPU"):
        ops.mx4_dequantize(q)
    with pytest.raises(ValueError, match="inner"):
        ops.mx4_matmul(q, ops.MX4(c, s, 99))
    with pytest.raises(ValueError, match="GPU"):
        ops.mx4_matmul(q, q)
    with pytest.raises(ValueError, match="must be"):
        ops.mx4_linear(torch.zeros(3, 99), q)
    t, p = torch.zeros(2, 4, 10), torch.zeros(2, 3, 10)
    d, u, r = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3), torch.zeros(2)
    for bad in ((d.int(), t, p, u, r), (d, t.double(), p, u, r), (d, t, p.half(), u, r), (d, t, p, u.double(), r)):
        with pytest.raises(TypeError):
            ops.verify_draft(*bad)
    for bad in ((d[:, :2], t, p, u, r), (d, t[:, :3], p, u, r), (d, t, p[:1], u, r), (d, t, p, u, r[:1]), (d, t, p, u, r),
                (d, t.transpose(1, 2).contiguous().transpose(1, 2), p, u, r)):
        with pytest.raises(ValueError):
            ops.verify_draft(*bad)
    with pytest.raises(ValueError, match="lens"):
        ops.verify_draft(d, t, p, u, r, lens=torch.zeros(2))


def test_reference_rounds_to_the_nearest_code():
    grid = np.concatenate([R.GRID, -R.GRID])
    x = np.array([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9] * 4, [0.26, 0.74, 1.26, 1.74, 2.6, 3.4, 5.1, -4.9] * 4])
    code, byte = R.quantize(x)
    assert (byte[:, 0] == 127).all()
    assert R.values(code, byte, 8).tolist() == [[0, 1, 1, 2, 2, 4, 4, 6], [0.5, 0.5, 1.5, 1.5, 3, 3, 6, -4]]
    rng = np.random.RandomState(0)
    x = rng.standard_normal((50, 96)) * np.exp2(rng.randint(-40, 40, (50, 1)))
    code, byte = R.quantize(x)
    v = R.values(code, byte, 96)
    for i, k in itertools.product(range(50), range(3)):
        s = np.exp2(byte[i, k] - 127.0)
        b = x[i, 32 * k:32 * k + 32]
        assert 4 * s <= np.abs(b).max() < 8 * s                          # the largest magnitude's exponent is the largest code's
        best = np.abs(np.clip(b, -6 * s, 6 * s)[:, None] - grid * s).min(1)
        np.testing.assert_array_equal(np.abs(np.clip(b, -6 * s, 6 * s) - v[i, 32 * k:32 * k + 32]), best)


def test_reference_check_samples_the_target():
    """Kept words and the drawn one are distributed as the target says, whatever the proposal: chi-square of the first word of 20000
    drafts (each uniform number drawn afresh), 7 degrees of freedom; 40 is passed by 1 in 10^6 at most."""
    rng = np.random.RandomState(3)
    p, q = rng.dirichlet(np.ones(8)), rng.dirichlet(np.ones(8))
    n = 20000
    d = rng.choice(8, (n, 1), p=q)
    t = np.broadcast_to(p, (n, 2, 8))
    words, acc = R.verify(d, t, np.broadcast_to(q, (n, 1, 8)), rng.random_sample((n, 1)), rng.random_sample(n), None)
    count = np.bincount(words[:, 0], minlength=8)
    assert ((count - n * p) ** 2 / (n * p)).sum() < 40
    assert 0 < acc.mean() < 1
