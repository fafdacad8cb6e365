"""Matrices in microscaled 4 bits on the GPU: written, read back and multiplied, against numpy in 64 bits.  Writing and reading back are
exact operations (one rounding each), so codes, scales and values have to be equal.  A product of two codes under their scales has at
most 4 significant bits and is exact in fp32; a sum of k of them in any order in fp32, each addition off by at most one step
(2^-23, a matrix core may cut instead of rounding), is off by at most k 2^-23 sum |a w|; bias and the rounding to the type add a half
step of the result each."""
import numpy as np
import pytest
import torch

import ops_reference as R
from ops_reference import DTYPES, HALF_STEP, np64

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from stattn import ops
    return ops


def wild(rows, cols, dtype, seed):
    """Values of many scales, ties, zeros of both signs, whole blocks of zeros, the type's largest and smallest."""
    rng = np.random.RandomState(seed)
    span = 12 if dtype == torch.float16 else 100
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.uniform(-span, span, (rows, 1)))
    if dtype == torch.float16:
        x = np.clip(x, -65000, 65000)
    tie = rng.random_sample((rows, cols)) < 0.3
    x = np.where(tie, np.exp2(rng.randint(-9, 9, (rows, 1))) * rng.randint(-32, 33, (rows, cols)) / 4, x)
    x[rng.random_sample((rows, cols)) < 0.05] = 0.0
    x[rng.random_sample((rows, cols)) < 0.02] = -0.0
    t = torch.from_numpy(x).to(dtype)
    f = torch.finfo(dtype)
    if rows > 2:
        t[1, : min(cols, 40)] = 0
        t[2, 0] = f.max
        t[0, -1] = f.tiny
        t[0, max(0, cols - 32):] *= 0
        t[0, -1] = f.smallest_normal / 2
    return t


def forms_equal(q, x64):
    code, byte = R.quantize(x64)
    np.testing.assert_array_equal(q.scales.cpu().numpy().astype(np.int64), byte)
    np.testing.assert_array_equal(R.unpack(q.codes), code)
    return code, byte


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 31), (5, 33), (7, 128), (4, 129), (33, 260), (65, 511), (300, 1000), (2, 4097), (1030, 96)])
@pytest.mark.parametrize("axis", [0, 1])
def test_write_and_read_back(ops, dt, rows, cols, axis):
    dtype = DTYPES[dt]
    x = wild(rows, cols, dtype, rows + 7 * cols + axis)
    given = (x.t().contiguous() if axis == 0 else x).to(DEV)
    q = ops.mx4_quantize(given, axis=axis)
    code, byte = forms_equal(q, np64(x))
    want = R.values(code, byte, cols)
    for out in DTYPES.values():
        got = ops.mx4_dequantize(q, out)
        assert got.dtype == out and got.shape == (rows, cols)
        ref = torch.from_numpy(want).to(out)                              # one rounding from 64 bits
        torch.testing.assert_close(got.cpu(), ref, rtol=0, atol=0, equal_nan=True)


def test_strides_and_offsets(ops):
    """Row strides, column strides, both, odd starting addresses: the same forms as of the contiguous copy."""
    base = wild(70, 700, torch.float32, 5).to(DEV)
    for dtype in DTYPES.values():
        b = base.clamp(-6e4, 6e4).to(dtype)
        for v in (b[:, 3:300], b[1::2, :], b[:, ::2], b[5:60:3, 7:500:5], b.t()[10:200, 1:50], b[:, 1:129], b[::7].t()):
            for axis in (0, 1):
                q, w = ops.mx4_quantize(v, axis=axis), ops.mx4_quantize(v.contiguous(), axis=axis)
                assert torch.equal(q.codes, w.codes) and torch.equal(q.scales, w.scales)
    e = b[:1].expand(9, 700)                                               # the same row nine times
    q = ops.mx4_quantize(e)
    assert torch.equal(q.codes, q.codes[:1].expand_as(q.codes))


@pytest.mark.parametrize("axis", [0, 1])
def test_infinities_and_nan_make_their_block_nan_and_no_other(ops, axis):
    x = wild(40, 300, torch.float32, 9)
    x[3, 5], x[4, 70], x[5, 299], x[39, 0] = float("inf"), float("nan"), -float("inf"), float("nan")
    q = ops.mx4_quantize((x.t().contiguous() if axis == 0 else x).to(DEV), axis=axis)
    code, byte = forms_equal(q, np64(x))
    got = ops.mx4_dequantize(q).cpu()
    bad = torch.zeros(40, 300, dtype=torch.bool)
    bad[3, 0:32] = bad[4, 64:96] = bad[5, 288:300] = bad[39, 0:32] = True
    assert torch.equal(torch.isnan(got), bad)
    w = ops.mx4_quantize(torch.randn(50, 300, device=DEV))
    for y in (ops.mx4_matmul(q, w), ops.mx4_matmul(w, q).t()):
        rows = torch.zeros(40, dtype=torch.bool)
        rows[[3, 4, 5, 39]] = True
        assert torch.equal(torch.isnan(y).all(1).cpu(), rows) and torch.equal(torch.isnan(y).any(1).cpu(), rows)


def test_every_scale_byte_is_read(ops):
    rng = np.random.RandomState(2)
    code = rng.randint(0, 16, (256, 128))
    byte = np.arange(256)[:, None].repeat(4, 1)
    q = ops.MX4(R.pack(code).to(DEV), torch.from_numpy(byte.astype(np.uint8)).to(DEV), 128)
    with np.errstate(over="ignore"):
        ref = torch.from_numpy(R.values(code, byte, 128)).float()
    torch.testing.assert_close(ops.mx4_dequantize(q).cpu(), ref, rtol=0, atol=0, equal_nan=True)


def check_product(y, a, w, bias, k, out):
    """y against the 64-bit product of the values a (m, k) and w (n, k)."""
    ref, mag = a @ w.T, np.abs(a) @ np.abs(w).T
    if bias is not None:
        ref = ref + bias
    with np.errstate(over="ignore"):
        tol = k * 2.0 ** -23 * mag
        tol = tol + 2.0 ** -24 * (np.abs(ref) + tol)                        # the bias is added in fp32
        tol = tol + HALF_STEP[out] * (np.abs(ref) + tol) + float(torch.finfo(out).smallest_normal) * HALF_STEP[out]
    err = np.abs(np64(y) - ref)
    assert y.dtype == out and (err <= tol).all(), (err - tol).max()


# (the last four: 128 x 128 tiles, twice, and 256 x 256 tiles; the last stage of 256 columns is half there in the first and third)
SHAPES = [(1, 1, 1), (1, 33, 128), (2, 16, 31), (5, 100, 129), (16, 64, 256), (17, 129, 511), (31, 255, 640), (33, 32, 1024), (64, 700, 96),
          (65, 66, 2050), (129, 257, 300), (255, 300, 1300), (257, 513, 257), (300, 40, 4096), (1, 5000, 513), (700, 1, 384), (12, 12, 12000),
          (513, 2049, 128), (1000, 1300, 160), (260, 2100, 4100),
          (2100, 2100, 300), (2050, 2300, 700), (3000, 2900, 1030), (2950, 3100, 1200)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(ops, dt, m, n, k):
    dtype = DTYPES[dt]
    rng = np.random.RandomState(m + 3 * n + 5 * k)
    x = torch.from_numpy(rng.standard_normal((m, k)) * np.exp2(rng.uniform(-3, 3, (m, 1)))).float().to(DEV)
    w = torch.from_numpy(rng.standard_normal((n, k)) * k ** -0.5).float().to(DEV)
    bias = torch.from_numpy(rng.standard_normal(n)).float().to(DEV) if (m + n) % 2 else None
    qx, qw = ops.mx4_quantize(x), ops.mx4_quantize(w)
    y = ops.mx4_matmul(qx, qw, bias=bias, dtype=dtype)
    check_product(y, np64(ops.mx4_dequantize(qx)), np64(ops.mx4_dequantize(qw)), None if bias is None else np64(bias), k, dtype)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_is_write_then_product(ops, dt, m, n, k):
    dtype = DTYPES[dt]
    rng = np.random.RandomState(2 * m + n + k)
    x = torch.from_numpy(np.tanh(rng.standard_normal((m, k)))).to(dtype).to(DEV)
    qw = ops.mx4_quantize(torch.from_numpy(rng.standard_normal((k, n))).float().to(DEV), axis=0)
    bias = torch.from_numpy(rng.standard_normal(n)).float().to(DEV) if (m + k) % 2 else None
    y = ops.mx4_linear(x, qw, bias=bias)
    code, byte = R.quantize(np64(x))
    check_product(y, R.values(code, byte, k), np64(ops.mx4_dequantize(qw)), None if bias is None else np64(bias), k, dtype)


@pytest.mark.parametrize("m,n,k", [(1, 70, 64), (16, 200, 640), (40, 90, 2100), (300, 500, 1000), (600, 1100, 1500)])
def test_products_of_whole_numbers_are_exact(ops, m, n, k):
    """Codes 0, 1, 2, 3, 4, 6 under one scale: every partial sum is a whole number under 2^24 (36 x 2100 < 2^17), exact in fp32."""
    g = torch.Generator().manual_seed(m)
    pick = torch.tensor([0., 1, 2, 3, 4, 6, -1, -2, -3, -4, -6])
    a, w = pick[torch.randint(0, 11, (m, k), generator=g)], pick[torch.randint(0, 11, (n, k), generator=g)]
    a[:, ::32], w[:, ::32] = 4, -6                                          # every block has the scale 1
    want = (a.double() @ w.double().t()).float()
    qa, qw = ops.mx4_quantize(a.to(DEV)), ops.mx4_quantize(w.to(DEV))
    assert torch.equal(ops.mx4_dequantize(qa).cpu(), a)
    assert torch.equal(ops.mx4_matmul(qa, qw).cpu(), want)
    assert torch.equal(ops.mx4_linear(a.to(DEV), qw).cpu(), want)


def test_linear_of_strided_rows_and_odd_addresses(ops):
    qw = ops.mx4_quantize(torch.randn(300, 200, device=DEV))
    for dtype in DTYPES.values():
        base = torch.randn(90, 700, device=DEV).to(dtype)
        for v in (base[:3, 1:201], base[:, 7:207], base[::9, 500:700], base[4:5, 3:203], base[:40, 8:208], base[:70:2, 16:216]):
            assert torch.equal(ops.mx4_linear(v, qw), ops.mx4_linear(v.contiguous(), qw))
        with pytest.raises(ValueError):
            ops.mx4_linear(base[:, ::3][:, :200], qw)


@pytest.mark.parametrize("k", [100, 300, 640])
def test_a_run_of_rows_is_a_matrix_too(ops, k):
    """Rows 7 .. 64 of a form, whose scales start at any multiple of four bytes."""
    q, x = ops.mx4_quantize(torch.randn(90, k, device=DEV)), torch.randn(33, k, device=DEV)
    part = ops.MX4(q.codes[7:64], q.scales[7:64], k)
    assert torch.equal(ops.mx4_dequantize(part), ops.mx4_dequantize(q)[7:64])
    assert torch.equal(ops.mx4_linear(x, part), ops.mx4_linear(x, q)[:, 7:64])
    assert torch.equal(ops.mx4_matmul(part, q), ops.mx4_matmul(q, q)[7:64])
    assert torch.equal(ops.mx4_matmul(q, part), ops.mx4_matmul(q, q)[:, 7:64])


def test_rows_behind_the_last_and_columns_beside_are_left_alone(ops):
    """Through the C entry: y inside a larger buffer, every tile size, both types of store; nothing beside it is touched."""
    from stattn import _native
    lib = _native.load_library()
    for m, n, k, dtype, code in [(5, 33, 64, torch.float32, 0), (70, 130, 300, torch.bfloat16, 1), (1100, 1000, 256, torch.float16, 2), (2100, 3900, 1200, torch.bfloat16, 1)]:
        a, w = ops.mx4_quantize(torch.randn(m, k, device=DEV)), ops.mx4_quantize(torch.randn(n, k, device=DEV))
        big = torch.full((m + 5, n + 37), 7.0, dtype=dtype, device=DEV)
        y = big[2:2 + m, 3:3 + n]
        rc = lib.stattn_mx4_matmul(0, torch.cuda.current_stream().cuda_stream, a.codes.data_ptr(), a.scales.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(),
                                   m, n, k, None, y.data_ptr(), code, n + 37)
        assert rc == 0
        assert torch.equal(y, ops.mx4_matmul(a, w, dtype=dtype))
        big[2:2 + m, 3:3 + n] = 7.0
        assert bool((big == 7.0).all())


def test_no_rows_no_outputs(ops):
    q = ops.mx4_quantize(torch.zeros(0, 100, device=DEV))
    w = ops.mx4_quantize(torch.ones(7, 100, device=DEV))
    assert ops.mx4_dequantize(q).shape == (0, 100)
    assert ops.mx4_matmul(q, w).shape == (0, 7) and ops.mx4_matmul(w, q).shape == (7, 0)
    assert ops.mx4_linear(torch.zeros(0, 100, device=DEV), w).shape == (0, 7)
    with pytest.raises(ValueError):
        ops.mx4_quantize(torch.zeros(3, 0, device=DEV))


def test_the_same_operand_twice_and_other_streams(ops):
    x = torch.randn(333, 500, device=DEV)
    q = ops.mx4_quantize(x)
    v = np64(ops.mx4_dequantize(q))
    check_product(ops.mx4_matmul(q, q), v, v, None, 500, torch.float32)
    want = ops.mx4_linear(x, q)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(ops.mx4_linear(x, q))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("m", [1, 5, 40, 300])
def test_captured_and_replayed(ops, m):
    w = ops.mx4_quantize(torch.randn(512, 900, device=DEV), axis=0)
    x = torch.randn(m, 512, device=DEV)
    ops.mx4_linear(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.mx4_linear(x, w)
        z = ops.mx4_dequantize(ops.mx4_quantize(y))
    for k in range(4):
        x.copy_(torch.randn(m, 512, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        want = ops.mx4_linear(x, w)
        assert torch.equal(y, want) and torch.equal(z, ops.mx4_dequantize(ops.mx4_quantize(want)))


def test_offsets_past_32_bits(ops):
    """2^20 + 5 rows of 8192: values, codes and results that lie more than 2^32 bytes or elements behind the first.  Values -1, 0, 1 are
    exact in the form, sums of 8192 products of them are whole numbers under 2^24."""
    rows, k = 2 ** 20 + 5, 8192
    x = torch.randint(-1, 2, (rows, k), dtype=torch.int8, device=DEV).to(torch.bfloat16)
    q = ops.mx4_quantize(x)
    assert x.numel() > 2 ** 32 and q.codes.numel() > 2 ** 32
    back = ops.mx4_dequantize(q, torch.bfloat16)
    assert all(torch.equal(back[r:r + 65536], x[r:r + 65536]) for r in range(0, rows, 65536))
    del back
    ends = torch.cat([torch.arange(7), torch.arange(rows // 2 - 3, rows // 2 + 3), torch.arange(rows - 40, rows)]).to(DEV)
    few = x[rows // 3:rows // 3 + 4].float()
    want = few.double() @ x[ends].double().t()
    assert torch.equal(ops.mx4_linear(few, q)[:, ends].double(), want)                  # one launch
    many = few.repeat(25, 1)
    assert torch.equal(ops.mx4_linear(many, q)[:, ends].double(), want.repeat(25, 1))   # two launches, w past 32 bits
    right = x[1000:4000].float()
    y = ops.mx4_matmul(q, ops.mx4_quantize(right))                                      # y past 32 bits
    assert y.numel() * 4 > 2 ** 33
    assert torch.equal(y[ends].double(), x[ends].double() @ right.double().t())
    del y
    tall = x[:, :4100].t()                                                              # (4100, rows): rows neighbours in memory
    qt = ops.mx4_quantize(tall[:, rows - 70000:])
    assert torch.equal(ops.mx4_dequantize(qt, torch.bfloat16), tall[:, rows - 70000:])
    x = q = tall = qt = None
    torch.cuda.empty_cache()
