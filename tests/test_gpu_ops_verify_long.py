"""The check of drafted words on vocabularies of more than 131072 words, where the 256 stretches of the running sum grow beyond 512 words,
and of more than 524288, where the stretch that a draw falls into is cut once more.

Weights of one half each on some words: every sum is a multiple of 1/2 and exact, so a draw_u of i / n, n = 1024 words with weight, takes
word number i of them, to the word.  The words lie at the ends of stretches, of their sub-stretches and of the eights a lane reads."""
import numpy as np
import pytest
import torch

import ops_reference as R
from ops_reference import DTYPES, np64
from test_gpu_ops_verify import check, make, ops      # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu
DEV = "cuda"
N = 1024


def borders(v, seed):
    """N words of a vocabulary of v in ascending order, most of them at a border, the first and the last among them."""
    up = lambda a, b: -(-a // b) * b
    step = up(up(v, 256) // 256, 512)
    sub = up(up(min(step, v), 16) // 16, 512)
    rng = np.random.RandomState(seed)
    at = [0, v - 1]
    for s in (step, sub, 512):
        edge = s * rng.randint(1, v // s + 1, 170)
        at += list(edge) + list(edge - 1)
    at = np.unique([a for a in at if 0 <= a < v])
    more = np.setdiff1d(rng.randint(0, v, 2 * N), at)
    return np.sort(np.concatenate([at, rng.permutation(more)[:N - len(at)]]))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("v", [131072, 131073, 200001, 524288, 524289, 1100003, 2 ** 24 + 3])
def test_draws_at_every_border(ops, dt, v):      # noqa: F811
    """In groups of 64 (several workgroups a caption) and 1024 (one): without a draft, behind a refusal with a proposal, and behind a
    refused word that was certain."""
    at = borders(v, v)
    assert len(at) == N
    row = torch.zeros(v, dtype=DTYPES[dt], device=DEV)
    row[torch.from_numpy(at).to(DEV)] = 0.5
    want = torch.from_numpy(at).to(DEV)
    du = torch.arange(N, device=DEV, dtype=torch.float32) / N
    none = torch.zeros(N, 0, device=DEV)
    free = int(np.setdiff1d(np.arange(at[-2]), at)[-1])                     # a word without weight, behind nearly all of them
    refused = torch.full((N, 1), free, device=DEV)
    other = torch.zeros(v, dtype=DTYPES[dt], device=DEV)
    other[torch.from_numpy(np.setdiff1d(np.arange(0, v, 1001), at)).to(DEV)] = 0.25     # a proposal beside the target: p - q is p
    with_certain = row.clone()
    with_certain[free] = 0.5                                                # half of 1: refused at 0.75, and nothing of it left over
    au = torch.full((N, 1), 0.75, device=DEV)
    for b in (64, N) if v < 2 ** 24 else (64, 130):
        for i in range(0, N, b):
            s = slice(i, min(i + b, N))
            n = s.stop - s.start
            words, acc = ops.verify_draft(none[s].long(), row.expand(n, 1, v), None, none[s], du[s])
            assert torch.equal(words[:, 0], want[s]) and not acc.any()
            words, acc = ops.verify_draft(refused[s], row.expand(n, 2, v), other.expand(n, 1, v), au[s], du[s])
            assert torch.equal(words[:, 0], want[s]) and not acc.any() and bool((words[:, 1] == -1).all())
            words, acc = ops.verify_draft(refused[s], with_certain.expand(n, 2, v), None, au[s], du[s])
            assert torch.equal(words[:, 0], want[s]) and not acc.any()


@pytest.mark.parametrize("v", [524289, 1100003, 2 ** 24 + 3])
def test_weight_in_one_sub_stretch(ops, v):      # noqa: F811
    """All weight within 512 words, at the first, a middle and the last of the cut; draws from one end of it to the other."""
    for lo in (0, 512 * 9, v // 2 // 512 * 512, (v - 1) // 512 * 512):
        hi = min(lo + 512, v)
        row = torch.zeros(v, device=DEV)
        row[lo:hi] = torch.rand(hi - lo, generator=torch.Generator().manual_seed(lo)).to(DEV) + 0.01
        c = np.cumsum(np64(row[lo:hi]).astype(np.longdouble))
        u = np.concatenate([[0.0, 1 - 2.0 ** -24], np.random.RandomState(1).random_sample(38)]).astype(np.float32)
        t = np.asarray(u, np.longdouble) * c[-1]
        assert (np.abs(c[:-1, None] - t[None]) > 2.0 ** -42 * c[-1]).all()  # no draw next to a border: sums in 64 bits are 2^-44 off at most
        want = lo + (c[:, None] <= t).sum(0)
        du = torch.from_numpy(u).to(DEV)
        words, _ = ops.verify_draft(torch.zeros(40, 0, dtype=torch.int64, device=DEV), row.expand(40, 1, v), None, torch.zeros(40, 0, device=DEV), du)
        np.testing.assert_array_equal(words[:, 0].cpu().numpy(), want)


def clear_of_borders(draft, target, proposal, au, du, lens):
    """No draw lies within 2^-52 v of the total of a border of its running sum, nor a product u q next to its p."""
    draft, target, proposal, au, du = draft.numpy(), np64(target), None if proposal is None else np64(proposal), np64(au), np64(du)
    words, acc = R.verify(draft, target, None if proposal is None else proposal.copy(), au, du, lens)
    v = target.shape[2]
    for i in range(len(du)):
        n, ln = acc[i], target.shape[1] - 1 if lens is None else lens[i]
        w = target[i, n]
        if n < ln:
            q = np.zeros(v) if proposal is None else proposal[i, n]
            if proposal is None:
                q[draft[i, n]] = 1
            rest = np.maximum(w - q, 0)
            w = rest if rest.any() else w
        c = np.cumsum(w.astype(np.longdouble))
        if not (np.abs(c - np.longdouble(du[i]) * c[-1]) > 2.0 ** -52 * v * c[-1]).all():
            return False
    return True


CASES = [("f32", 1, 2, 524288, 1), ("f32", 2, 2, 524289, 2), ("f32", 66, 1, 524289, 3), ("bf16", 130, 1, 524291, 4), ("f16", 3, 1, 1100003, 5)]


@pytest.mark.parametrize("dt,b,j,v,seed", CASES)
def test_words_and_counts_of_long_rows(ops, dt, b, j, v, seed):      # noqa: F811
    args = make(b, j, v, DTYPES[dt], seed)
    lens = torch.randint(0, j + 1, (b,), generator=torch.Generator().manual_seed(v), dtype=torch.int32)
    host = [a.cpu() for a in args]
    for p, ln in ((host[2], None), (host[2], lens), (None, lens)):
        assert clear_of_borders(host[0], host[1], p, host[3], host[4], None if ln is None else ln.numpy())
    check(ops, args)
    check(ops, args, lens.to(DEV))
    check(ops, [args[0], args[1], None, args[3], args[4]], lens.to(DEV))


def test_the_longest_rows(ops):      # noqa: F811
    """2^31 - 1 words: the eight draws fall on the first word, the last, and next to 2^30 and 2^31 - 2."""
    v = 2 ** 31 - 1
    row = torch.zeros(v, dtype=torch.bfloat16, device=DEV)
    at = torch.tensor([0, 511, 2 ** 30 - 1, 2 ** 30, 2 ** 30 + 1, v - 513, v - 2, v - 1], device=DEV)
    row[at] = 0.5
    du = torch.arange(8, device=DEV, dtype=torch.float32) / 8
    words, _ = ops.verify_draft(torch.zeros(8, 0, dtype=torch.int64, device=DEV), row.expand(8, 1, v), None, torch.zeros(8, 0, device=DEV), du)
    assert torch.equal(words[:, 0], at)
    draft = at[[1, 7, 7, 7]][:, None].contiguous()                          # certain words: the target's half refuses them at 0.75, keeps them at 0.25
    au = torch.tensor([[0.25], [0.75], [0.75], [0.25]], device=DEV)
    words, acc = ops.verify_draft(draft, row.expand(4, 2, v), None, au, torch.tensor([0.99, 0.99, 0.0, 0.0], device=DEV))
    assert acc.tolist() == [1, 0, 0, 1] and words.tolist() == [[511, v - 1], [v - 2, -1], [0, -1], [v - 1, 0]]
    row = words = None
    torch.cuda.empty_cache()
