"""Products over the whole range of scale bytes.  A product of two codes has 4 significant bits; under its scales it is exact in fp32
while it lies between 2^-126 and 2^128, infinite beyond, and rounded to a multiple of 2^-149 below."""
import numpy as np
import pytest
import torch

import ops_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from stattn import ops
    return ops


@pytest.mark.parametrize("code,value", [(1, 0.5), (2, 1.0), (3, 1.5), (7, 6.0), (13, -3.0)])
def test_every_pair_of_scales(ops, code, value):
    """255 x 255 products of one code under each pair of scale bytes: the number itself, rounded to fp32."""
    codes = torch.zeros(255, 64, dtype=torch.uint8)
    codes[:, 16] = code                                                    # column 32: the second block
    scales = torch.full((255, 4), 200, dtype=torch.uint8)                  # (the other blocks hold zeros)
    scales[:, 1] = torch.arange(255, dtype=torch.uint8)
    q = ops.MX4(codes.to(DEV), scales.to(DEV), 100)
    e = np.arange(255)[:, None] + np.arange(255) - 254
    with np.errstate(over="ignore"):
        want = np.ldexp(value * value, e).astype(np.float32)
    assert np.isinf(want).any() and (want == 0).any()
    np.testing.assert_array_equal(ops.mx4_matmul(q, q).cpu().numpy(), want)
    # x of one fp32 number a row, whose block gets the scale byte e - 2
    for rows in (16, 64):
        ex = np.linspace(-126, 127, 64).round().astype(int)[-rows:]
        x = torch.zeros(rows, 100)
        x[:, 40] = torch.ldexp(torch.ones(rows), torch.tensor(ex, dtype=torch.int32))
        scales[:, 1] = torch.arange(255, dtype=torch.uint8)
        w = codes.clone()
        w[:, 16], w[:, 20] = 0, code                                       # column 40
        with np.errstate(over="ignore"):
            want = np.ldexp(value, ex[:, None] + np.arange(255) - 127).astype(np.float32)
        np.testing.assert_array_equal(ops.mx4_linear(x.to(DEV), ops.MX4(w.to(DEV), scales.to(DEV), 100)).cpu().numpy(), want)


@pytest.mark.parametrize("m,n,k", [(1, 300, 513), (200, 255, 96), (2049, 2100, 300), (2050, 3900, 1200)])
def test_sums_under_scales_of_the_whole_range(ops, m, n, k):
    """A row has one scale, rows have any: y is a whole number of quarters (under 2^24 of them, exact in fp32) times a power of two, so y
    is that number where all sums lie in fp32's normal range.  Below, each of the k additions is off by at most a step of 2^-149."""
    g = torch.Generator().manual_seed(m + k)

    def form(rows):
        code = torch.randint(0, 16, (rows, k), generator=g)
        byte = torch.randint(0, 255, (rows, 1), generator=g)
        pad = torch.zeros(rows, -(-k // 128) * 128, dtype=torch.int64)
        pad[:, :k] = code
        grid = torch.from_numpy(np.concatenate([R.GRID, -R.GRID]))
        return (ops.MX4(R.pack(pad.numpy()).to(DEV), byte.expand(rows, pad.shape[1] // 32).to(torch.uint8).contiguous().to(DEV), k),
                grid[code].to(DEV), byte.double().to(DEV) - 127)
    a, va, ea = form(m)
    w, vw, ew = form(n)
    scale = torch.exp2(ea + ew.t())
    want, mag = (va @ vw.t().contiguous()) * scale, (va.abs() @ vw.abs().t().contiguous()) * scale
    y = ops.mx4_matmul(a, w).double()
    held = mag < 2.0 ** 127
    tol = torch.where(scale * 0.25 >= 2.0 ** -149, 0.0, k * 2.0 ** -149)
    assert 0.3 < float(held.double().mean()) < 1.0
    assert bool(((y - want).abs()[held] <= tol[held]).all())
