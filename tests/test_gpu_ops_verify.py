"""Drafted words checked on the GPU against a walk through the draft in 64 bits (numpy).  Words and counts are whole numbers: they have
to be equal.  u q is exact in 64 bits for inputs of 32 bits or fewer; the running sums differ in their order only, by 2^-53 v of the total
at most, and the uniform numbers are drawn so that none lies that near a border."""
import numpy as np
import pytest
import torch

import ops_reference as R
from ops_reference import DTYPES, np64

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from stattn import ops
    return ops


def make(b, j, v, dtype, seed, near=0.7, sharp=3.0):
    g = torch.Generator().manual_seed(seed)
    logit = sharp * torch.randn(b, j + 1, v, generator=g)
    target = torch.softmax(logit, 2).to(dtype)
    proposal = torch.softmax(logit[:, :j] + near * torch.randn(b, j, v, generator=g), 2)
    draft = torch.multinomial(proposal.reshape(b * j, v), 1, generator=g).view(b, j) if j else torch.zeros(b, 0, dtype=torch.int64)
    return [t.to(DEV) for t in (draft, target, proposal.to(dtype), torch.rand(b, j, generator=g), torch.rand(b, generator=g))]


def check(ops, args, lens=None):
    words, accepted = ops.verify_draft(*args, lens=lens)
    draft, target, proposal, au, du = args
    want, n = R.verify(draft.cpu().numpy(), np64(target), None if proposal is None else np64(proposal), np64(au), np64(du),
                       None if lens is None else lens.cpu().numpy())
    assert words.dtype == torch.int64 and accepted.dtype == torch.int32
    np.testing.assert_array_equal(accepted.cpu().numpy(), n)
    np.testing.assert_array_equal(words.cpu().numpy(), want)
    return n


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("b,j,v", [(1, 0, 1), (1, 1, 1), (1, 1, 2), (3, 2, 7), (1, 4, 63), (5, 5, 64), (2, 3, 1000), (64, 5, 1025), (1, 4, 12000), (7, 8, 4099),
                                   (33, 1, 20000), (3, 70, 500), (2, 2, 50257), (1, 3, 128000), (300, 2, 37), (4, 3, 200001), (70, 1, 98304)])
def test_words_and_counts(ops, dt, b, j, v):
    args = make(b, j, v, DTYPES[dt], b + 3 * j + 7 * v)
    check(ops, args)
    lens = torch.randint(0, j + 1, (b,), generator=torch.Generator().manual_seed(v), dtype=torch.int32).to(DEV)
    check(ops, args, lens)
    check(ops, [args[0], args[1], None, args[3], args[4]], lens)           # arg-max drafts: the proposal was certain


def test_all_kept_none_kept(ops):
    d, t, p, au, du = make(40, 4, 999, torch.float32, 1)
    assert (check(ops, [d, t, p, torch.zeros_like(au), du]) == 4).all()
    certain = torch.zeros_like(p).scatter_(2, d[:, :, None], 1.0)           # each word certain, and the target all but excludes it
    low = t.clone()
    low[:, :4].scatter_(2, d[:, :, None], 1e-30)
    assert (check(ops, [d, low, certain, au.clamp(min=0.01), du]) == 0).all()


def test_draw_at_the_ends(ops):
    """draw_u of 0 takes the first word with any weight, the largest under 1 the last; words without weight are never drawn."""
    d, t, p, au, du = make(6, 2, 3001, torch.float32, 2)
    t[:, :, :1500] = 0
    t[:, :, 2900:] = 0
    lens = torch.zeros(6, dtype=torch.int32, device=DEV)
    for u in (0.0, 1 - 2.0 ** -24, 0.5):
        check(ops, [d, t, p, au, torch.full_like(du, u)], lens)
    only = torch.zeros_like(t)
    only[:, :, 2999] = 1e-38
    words, _ = ops.verify_draft(d, only, p, au, du, lens=lens)
    assert (words[:, 0] == 2999).all()


def test_nothing_left_over_and_rows_without_weight(ops):
    """p <= q everywhere: the refused word is replaced by a draw from p.  A target row of zeros (or of NaN) draws -1."""
    d, t, p, au, du = make(5, 3, 700, torch.float32, 3)
    q = t[:, :3] * 1.5
    n = check(ops, [d, t, q, torch.full_like(au, 0.9), du])
    assert (n == 0).all()
    zero = t.clone()
    zero[1], zero[3] = 0, float("nan")
    words, acc = ops.verify_draft(d, zero, p, au, du)
    check(ops, [d, zero, p, au, du])
    assert words[1, 0] == -1 and words[3, 0] == -1 and acc[1] == 0 and acc[3] == 0


def test_nan_and_words_outside_the_vocabulary(ops):
    d, t, p, au, du = make(8, 4, 333, torch.float32, 4)
    t[0, 0, 5] = float("nan")
    p[1, 0, 7] = float("nan")
    t[2, 1, int(d[2, 1])] = float("nan")
    d[3, 0], d[4, 1], d[5, 3], d[6, 2] = -1, 333, 1 << 40, -(1 << 62)
    check(ops, [d, t, p, au * 0.01, du])
    check(ops, [d, t, None, au * 0.01, du])


def test_lens_outside_the_draft_are_the_nearer_end(ops):
    args = make(4, 3, 100, torch.bfloat16, 5)
    check(ops, args, torch.tensor([-5, 9, 2, 3], dtype=torch.int32, device=DEV))


def test_strided_inputs(ops):
    d, t, p, au, du = make(9, 4, 1200, torch.float32, 6)
    big = torch.full((9, 7, 1300), float("nan"), device=DEV)
    big[:, 1:6, 3:1203] = t
    pig = torch.full((4, 9, 1201), float("nan"), device=DEV)
    pig[:, :, 1:] = p.transpose(0, 1)
    dd = torch.full((9, 11), -7, dtype=torch.int64, device=DEV)
    dd[:, 2:6] = d
    uu = torch.full((9, 6), 2.0, device=DEV)
    uu[:, 1:5] = au
    got = ops.verify_draft(dd[:, 2:6], big[:, 1:6, 3:1203], pig[:, :, 1:].transpose(0, 1), uu[:, 1:5], du)
    want = ops.verify_draft(d, t, p, au, du)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    check(ops, [dd[:, 2:6], big[:, 1:6, 3:1203], pig[:, :, 1:].transpose(0, 1), uu[:, 1:5], du])
    row = t[:1].expand(9, 5, 1200)                                          # one target for all captions
    check(ops, [d, row, p, au, du])


def test_no_captions(ops):
    d, t, p, au, du = make(1, 3, 10, torch.float32, 7)
    words, acc = ops.verify_draft(d[:0], t[:0], p[:0], au[:0], du[:0])
    assert words.shape == (0, 4) and acc.shape == (0,)


@pytest.mark.parametrize("b,j,v", [(1, 4, 300), (4, 3, 60000), (2, 2, 98305)])
def test_captured_and_replayed_and_on_other_streams(ops, b, j, v):
    args = make(b, j, v, torch.float32, 8)
    ops.verify_draft(*args)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(ops.verify_draft(*args))
    for k in range(4):
        fresh = make(b, j, v, torch.float32, 20 + k)
        for t, f in zip(args, fresh):
            t.copy_(f)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = ops.verify_draft(*fresh)
        for o in outs:
            assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])
        check(ops, fresh)
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(ops.verify_draft(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(g[0], want[0]) for g in got)


def test_captions_follow_the_target(ops):
    """The first word of 200000 drafts from another distribution is distributed as the target: chi-square over 40 words, 39 degrees of
    freedom, 110 is passed by fewer than 1 in 10^7."""
    g = torch.Generator().manual_seed(9)
    n, v = 200000, 40
    p, q = torch.softmax(torch.randn(v, generator=g), 0), torch.softmax(torch.randn(v, generator=g), 0)
    d = torch.multinomial(q, n, replacement=True, generator=g)[:, None]
    words, acc = ops.verify_draft(d.to(DEV), p.to(DEV).expand(n, 2, v), q.to(DEV).expand(n, 1, v), torch.rand(n, 1, generator=g).to(DEV),
                                  torch.rand(n, generator=g).to(DEV))
    count = torch.bincount(words[:, 0].cpu(), minlength=v).double()
    e = n * p.double() / p.double().sum()
    assert float(((count - e) ** 2 / e).sum()) < 110 and 0 < float(acc.float().mean()) < 1


def test_offsets_past_32_bits(ops):
    """Captions 2^31 + 24 elements apart."""
    d, t, p, au, du = make(3, 2, 1000, torch.bfloat16, 21)
    step = 2 ** 31 + 24
    far = torch.empty(2 * step + 3000, dtype=torch.bfloat16, device=DEV)
    ft, fp = far.as_strided((3, 3, 1000), (step, 1000, 1)), torch.empty_like(far).as_strided((3, 2, 1000), (step, 1000, 1))
    ft.copy_(t)
    fp.copy_(p)
    check(ops, [d, ft, fp, au, du])
    far = ft = fp = None
    torch.cuda.empty_cache()
