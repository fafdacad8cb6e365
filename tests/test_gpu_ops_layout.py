"""Results of the device-memory operators inside larger buffers, through the C entries: rows of any stride, and a whole tile's worth of
memory around them -- behind the last row and column, in front of the first -- that has to stay as it was."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [(torch.float32, 0), (torch.bfloat16, 1), (torch.float16, 2)]
EDGE = 260                                                                  # rows and columns around a result: more than the largest tile


@pytest.fixture(scope="module")
def ops():
    from stattn import ops
    return ops


@pytest.fixture(scope="module")
def lib():
    from stattn import _native
    return _native.load_library()


def framed(rows, cols, dtype, fill=7):
    """(buffer, the (rows, cols) view in its middle, whose row stride is the buffer's)"""
    big = torch.full((rows + 2 * EDGE, cols + 2 * EDGE + 3), fill, dtype=dtype, device=DEV)
    return big, big[EDGE:EDGE + rows, EDGE + 1:EDGE + 1 + cols]


def untouched(big, view, fill=7):
    view.fill_(fill)
    return bool((big == fill).all())


def stream():
    return torch.cuda.current_stream().cuda_stream


def tile(m, n, k):
    """The edge of the product's tiles for these sizes (the rule of ops/mx4_gemm.hip): this file has to meet all three."""
    def tiles(e):
        return -(-m // e) * -(-n // e)
    return 64 if tiles(64) < 1024 else 256 if tiles(256) >= 128 and k > 1024 else 128


# last tiles with one row, with one column, with all but one, and whole ones
@pytest.mark.parametrize("dtype,code", TYPES)
@pytest.mark.parametrize("edge,m,n,k", [(64, 1, 1, 64), (64, 5, 33, 64), (64, 65, 191, 300), (64, 128, 64, 128), (64, 63, 129, 513),
                                        (128, 2049, 2177, 160), (128, 2175, 2047, 700), (128, 2048, 2176, 129),
                                        (256, 2049, 3841, 1030), (256, 2303, 3839, 1200), (256, 2048, 4096, 1153)])
def test_product_in_a_frame(ops, lib, edge, m, n, k, dtype, code):
    assert tile(m, n, k) == edge
    a, w, bias = ops.mx4_quantize(torch.randn(m, k, device=DEV)), ops.mx4_quantize(torch.randn(n, k, device=DEV)), torch.randn(n, device=DEV)
    big, y = framed(m, n, dtype)
    rc = lib.stattn_mx4_matmul(0, stream(), a.codes.data_ptr(), a.scales.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), m, n, k, bias.data_ptr(),
                               y.data_ptr(), code, big.stride(0))
    assert rc == 0
    assert torch.equal(y, ops.mx4_matmul(a, w, bias=bias, dtype=dtype)) and untouched(big, y)


@pytest.mark.parametrize("dtype,code", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 5, 64), (3, 4001, 200), (16, 70, 1000), (17, 129, 640), (33, 1000, 320), (64, 35, 511), (65, 130, 300), (300, 500, 2000)])
def test_linear_in_a_frame(ops, lib, m, n, k, dtype, code):
    """One launch (up to 64 rows of these lengths) and two; x is a frame's middle too, with infinities around it."""
    xbig, x = framed(m, k, dtype, float("inf"))
    x.copy_(torch.randn(m, k, device=DEV))
    w, bias = ops.mx4_quantize(torch.randn(n, k, device=DEV)), torch.randn(n, device=DEV)
    big, y = framed(m, n, dtype)
    need = lib.stattn_mx4_linear_workspace(m, n, k)
    work = torch.full((need + 512,), 9, dtype=torch.uint8, device=DEV)
    rc = lib.stattn_mx4_linear(0, stream(), x.data_ptr(), code, xbig.stride(0), w.codes.data_ptr(), w.scales.data_ptr(), m, n, k, bias.data_ptr(),
                               y.data_ptr(), big.stride(0), work.data_ptr(), need)
    assert rc == 0
    assert torch.equal(y, ops.mx4_linear(x.contiguous(), w, bias=bias)) and bool(torch.isfinite(y).all())
    assert untouched(big, y) and bool((work[need:] == 9).all())


@pytest.mark.parametrize("dtype,code", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 33), (70, 127), (33, 128), (4, 1001)])
def test_read_back_and_written_in_a_frame(ops, lib, rows, cols, dtype, code):
    q = ops.mx4_quantize(torch.randn(rows, cols, device=DEV))
    big, out = framed(rows, cols, dtype)
    assert lib.stattn_mx4_dequantize(0, stream(), q.codes.data_ptr(), q.scales.data_ptr(), rows, cols, out.data_ptr(), code, big.stride(0)) == 0
    assert torch.equal(out, ops.mx4_dequantize(q, dtype)) and untouched(big, out)
    # the form itself: as many bytes as its rows have, none in front of or behind them
    for axis in (0, 1):
        xbig, x = framed(cols, rows, dtype, float("nan")) if axis == 0 else framed(rows, cols, dtype, float("nan"))
        x.copy_(torch.randn(x.shape, device=DEV))
        kb = -(-cols // 128) * 4
        codes, scales = (torch.full((rows * n + 8192,), 201, dtype=torch.uint8, device=DEV) for n in (16 * kb, kb))
        rs, cs = (1, xbig.stride(0)) if axis == 0 else (xbig.stride(0), 1)
        assert lib.stattn_mx4_quantize(0, stream(), x.data_ptr(), code, rows, cols, rs, cs, codes.data_ptr() + 4096, scales.data_ptr() + 4096) == 0
        want = ops.mx4_quantize(x.contiguous(), axis=axis)
        for got, ref in ((codes, want.codes), (scales, want.scales)):
            assert torch.equal(got[4096:-4096], ref.flatten()) and bool((got[:4096] == 201).all()) and bool((got[-4096:] == 201).all())


@pytest.mark.parametrize("b,j,v", [(1, 0, 30), (5, 3, 700), (3, 70, 200), (2, 2, 98304)])
def test_check_in_a_frame(ops, lib, b, j, v):
    """words with a row stride of their own; behind its j + 1 words a row stays as it was, and so does what lies behind the workspace."""
    g = torch.Generator().manual_seed(b + v)
    t = torch.softmax(2 * torch.randn(b, j + 1, v, generator=g), 2).to(DEV)
    p = torch.softmax(2 * torch.randn(b, j, v, generator=g), 2).to(DEV)
    d, au, du = torch.randint(0, v, (b, j), generator=g).to(DEV), torch.rand(b, j, generator=g).to(DEV), torch.rand(b, generator=g).to(DEV)
    big, words = framed(b, j + 1, torch.int64, 99)
    acc = torch.full((b + 64,), 99, dtype=torch.int32, device=DEV)
    need = lib.stattn_verify_draft_workspace(b, j, v)
    work = torch.full((need + 512,), 9, dtype=torch.uint8, device=DEV)
    rc = lib.stattn_verify_draft(0, stream(), d.data_ptr(), j, t.data_ptr(), (j + 1) * v, v, p.data_ptr(), j * v, v, 0, au.data_ptr(), j, du.data_ptr(), None,
                                 b, j, v, words.data_ptr(), big.stride(0), acc.data_ptr(), work.data_ptr(), need)
    assert rc == 0
    want = ops.verify_draft(d, t, p, au, du)
    assert torch.equal(words, want[0]) and torch.equal(acc[:b], want[1])
    assert untouched(big, words, 99) and bool((acc[b:] == 99).all()) and bool((work[need:] == 9).all())


@pytest.mark.parametrize("dtype,code", TYPES[:2])
def test_the_largest_row_stride(ops, lib, dtype, code):
    """Row strides of 2^22 - 1 elements, the largest that is accepted: the last row of a 256-row tile in fp32 ends just under 2^32 bytes
    behind its first.  Between the rows, and in the columns beside the result, nothing is written."""
    m, n, k, ld = 2047, 4095, 1030, 2 ** 22 - 1
    assert tile(m, n, k) == 256
    a, w = ops.mx4_quantize(torch.randn(m, k, device=DEV)), ops.mx4_quantize(torch.randn(n, k, device=DEV))
    big = torch.full((m + 1, ld), 7, dtype=dtype, device=DEV)
    y = big[:m, 5:5 + n]
    assert lib.stattn_mx4_matmul(0, stream(), a.codes.data_ptr(), a.scales.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), m, n, k, None,
                                 y.data_ptr(), code, ld) == 0
    assert torch.equal(y, ops.mx4_matmul(a, w, dtype=dtype))
    y.fill_(7)
    assert all(bool((big[r:r + 64] == 7).all()) for r in range(0, m + 1, 64))
    big = y = None
    torch.cuda.empty_cache()
