"""Drafted sampling (stattn_sample_drafted): words drafted by a 4-bit copy of the vocabulary projection, checked by the full-precision one.
The captions have to be samples of the full-precision decoder whatever the draft is worth, so the checks need no number of the draft:
scores against the float64 oracle's teacher-forced probabilities, distributions of the first two words against its exact ones, and
captions of a decoder whose distributions are all but certain against the greedy ones of the beam search."""
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
TOL = 1e-4


@pytest.fixture(scope="module")
def O():
    from oracle import stattn_oracle
    return stattn_oracle


@pytest.fixture(scope="module")
def stattn_mod():
    import stattn
    return stattn


def small(O, sharpen=6.0):
    opt = O.default_options(dim=64, dim_word=64, n_words=37, ctxg_dim=64, ctxl_dim=32, ctxm_dim=32, ctxglm_dim=64)
    gold = os.path.join(os.path.dirname(os.path.abspath(__file__)), 'golden')
    P = dict(np.load(os.path.join(gold, 'params.npz')))
    P['ff_logit_W'] = P['ff_logit_W'] * np.float32(sharpen)
    P['ff_logit_b'] = P['ff_logit_b'].copy()
    P['ff_logit_b'][0] += np.float32(1.0)
    return opt, P


def decoder(stattn_mod, opt, P, **kw):
    dec = stattn_mod.Decoder(opt, **kw)
    dec.set_params(P)
    return dec


def features(b, sl=slice(None)):
    return b['ctxg'][sl], b['mask_ctxg'][sl], b['ctxl'][sl], b['ctxm'][sl]


def teacher_forced(O, P, opt, b, v, words):
    fi, fn = O.sampler_closures(O.cast_params(P, np.float64), opt, np.float64)
    args = (b['ctxg'][v].astype(np.float64), b['mask_ctxg'][v], b['ctxl'][v].astype(np.float64), None, b['ctxm'][v].astype(np.float64), None)
    _, h, c = fi(args[0], args[1])
    h, c, x, out = h[None], c[None], np.array([-1], np.int64), []
    for w in words:
        p, _, h, c = fn(x, *args, h, c)
        out.append(p[0, w])
        x = np.array([w], np.int64)
    return np.array(out)


@pytest.mark.parametrize("lt_mode", [0, 1])
@pytest.mark.parametrize("nvid,draft,maxlen", [(1, 1, 1), (1, 4, 12), (3, 2, 7), (4, 8, 12), (16, 5, 20), (16, 8, 3), (13, 3, 30)])
def test_captions_and_scores(stattn_mod, O, lt_mode, nvid, draft, maxlen):
    opt, P = small(O)
    b = O.synthetic_batch(opt, B=nvid, T=5, K=3, t=3, seed=70 + nvid)
    dec = decoder(stattn_mod, opt, P, lt_mode=lt_mode)
    u = np.random.RandomState(draft).random_sample((maxlen, 2 * draft + 1, nvid)).astype(np.float32)
    u = np.minimum(u, np.float32(1 - 2.0 ** -24))
    got = dec.sample_drafted(*features(b), draft=draft, maxlen=maxlen, uniforms=u)
    drafted, kept = dec.draft_counts
    assert ((0 <= kept) & (kept <= drafted) & (drafted % draft == 0) & (drafted > 0)).all()
    for v, (words, score) in enumerate(got):
        assert 1 <= len(words) <= maxlen and all(0 <= w < 37 for w in words)
        assert 0 not in words[:-1] and (len(words) == maxlen or words[-1] == 0)
        p = teacher_forced(O, P, opt, b, v, words)
        assert (p > 0).all()
        np.testing.assert_allclose(score, p.sum(), rtol=0, atol=TOL * len(words))
    # the same numbers give the same captions, replayed, launched plainly, and from staged features
    again = dec.sample_drafted(draft=draft, maxlen=maxlen, uniforms=u, resident=True)
    assert again == got
    os.environ['STATTN_BEAM_NOGRAPH'] = '1'
    try:
        assert dec.sample_drafted(draft=draft, maxlen=maxlen, uniforms=u, resident=True) == got
    finally:
        del os.environ['STATTN_BEAM_NOGRAPH']
    # checks of 0 keep every draft that the target does not exclude
    u[:, draft:2 * draft] = 0
    dec.sample_drafted(draft=draft, maxlen=maxlen, uniforms=u, resident=True)
    assert (dec.draft_counts[0] == dec.draft_counts[1]).all()


@pytest.mark.parametrize("precision", ["fp32", "split", "bf16"])
def test_all_but_certain_distributions_give_the_greedy_captions(stattn_mod, O, precision):
    """ff_logit_W a few hundred times as large: where the most probable word leaves under 1e-4 to all others, a number in [1e-3, 1 - 1e-3]
    can neither keep nor draw another one, so the captions have to be the greedy ones, over several rounds, and after a new matrix (the
    4-bit copy follows it)."""
    opt, P = small(O, 6.0)
    b = O.synthetic_batch(opt, B=6, T=5, K=3, t=3, seed=7)
    dec = decoder(stattn_mod, opt, P, precision=precision)
    rng = np.random.RandomState(1)
    compared = 0
    for scale in (600.0, 900.0, 700.0):
        Q = dict(P)
        Q['ff_logit_W'] = P['ff_logit_W'] * np.float32(scale / 6.0)
        if scale == 900.0:
            Q['ff_logit_W'] = Q['ff_logit_W'][:, ::-1].copy()               # other words altogether
        dec.set_params(Q)
        greedy = dec.beam_search(*features(b), k=1, maxlen=14)
        for draft in (1, 3, 4, 8):
            u = rng.uniform(1e-3, 1 - 1e-3, (14, 2 * draft + 1, 6)).astype(np.float32)
            got = dec.sample_drafted(draft=draft, maxlen=14, uniforms=u, resident=True)
            for v, (words, _) in enumerate(got):
                want = greedy[v][0][0]
                p = teacher_forced(O, Q, opt, b, v, want)
                sure = int(np.argmax(np.append(p < 1 - 1e-4, True)))        # from the first word that is less than certain on, captions may differ
                assert words[:sure] == want[:sure], (scale, draft, v, p)
                compared += sure
    assert compared > 200


def test_first_two_words_are_distributed_as_the_decoder_says(stattn_mod, O):
    """4000 captions of one video, a coarse draft: the pairs' first word and second word against the oracle's exact distributions, by
    total variation.  For n draws over k words its expectation is at most sqrt(k / n) / 2 = 0.048 (37 words, 4000 draws), its standard
    deviation at most 1 / (2 sqrt(n)) = 0.008: 0.08 is four of them away."""
    opt, P = small(O, 3.0)
    b = O.synthetic_batch(opt, B=1, T=5, K=3, t=3, seed=70)
    dec = decoder(stattn_mod, opt, P)
    dec.set_seed(3)
    dec.beam_stage(*(np.repeat(x, 16, 0) for x in features(b)))
    first, second = np.zeros(37), np.zeros(38)                              # second[37]: the caption ended with its first word
    kept = drafted = 0
    for _ in range(250):
        for words, _ in dec.sample_drafted(draft=3, maxlen=2, resident=True):
            first[words[0]] += 1
            second[words[1] if len(words) > 1 else 37] += 1
        drafted += dec.draft_counts[0].sum()
        kept += dec.draft_counts[1].sum()
    assert 0 < kept < drafted
    fi, fn = O.sampler_closures(O.cast_params(P, np.float64), opt, np.float64)
    args = (b['ctxg'][0].astype(np.float64), b['mask_ctxg'][0], b['ctxl'][0].astype(np.float64), None, b['ctxm'][0].astype(np.float64), None)
    _, h, c = fi(args[0], args[1])
    p1, _, h, c = fn(np.array([-1], np.int64), *args, h[None], c[None])
    p2 = fn(np.arange(37), *args, np.repeat(h, 37, 0), np.repeat(c, 37, 0))[0]
    want = np.append((p1[0, 1:, None] * p2[1:]).sum(0), p1[0, 0])
    assert 0.5 * np.abs(first / first.sum() - p1[0]).sum() < 0.08
    assert 0.5 * np.abs(second / second.sum() - want).sum() < 0.08


def test_seed_and_surface(stattn_mod, O):
    opt, P = small(O)
    b = O.synthetic_batch(opt, B=18, T=5, K=3, t=3, seed=71)
    model = stattn_mod.Attention()
    tparams = model.init_tparams(P)
    out = model.gen_sample_drafted(tparams, opt, *features(b), draft=4, maxlen=9)           # two groups of videos
    assert len(out) == 18
    for v in (0, 17):
        np.testing.assert_allclose(out[v][1], teacher_forced(O, P, opt, b, v, out[v][0]).sum(), rtol=0, atol=TOL * 9)
    dec = tparams.decoder
    few = features(b, slice(0, 4))
    dec.set_seed(5)
    one = dec.sample_drafted(*few, maxlen=9)
    two = dec.sample_drafted(*few, maxlen=9)
    dec.set_seed(5)
    assert dec.sample_drafted(*few, maxlen=9) == one and one != two
    other = decoder(stattn_mod, opt, P)
    other.set_seed(5)
    assert other.sample_drafted(*few, maxlen=9) == one
    # the other searches go on as before, with their own results, and a beam search's final states stay readable
    want = other.beam_search(*few, k=3, maxlen=9)
    states = other.beam_final_state()
    other.sample_drafted(*few, maxlen=9)
    for (h, c), (h2, c2) in zip(states, other.beam_final_state()):
        assert np.array_equal(h, h2) and np.array_equal(c, c2)
    got = dec.beam_search(*few, k=3, maxlen=9)
    assert [w for w, _ in got] == [w for w, _ in want]


def test_refusals(stattn_mod, O):
    opt, P = small(O)
    b = O.synthetic_batch(opt, B=17, T=5, K=3, t=3, seed=72)
    dec = decoder(stattn_mod, opt, P)
    with pytest.raises(ValueError, match="nvid"):
        dec.sample_drafted(*features(b))
    two = features(b, slice(0, 2))
    for kw in (dict(draft=0), dict(draft=9), dict(maxlen=0), dict(maxlen=65537)):
        with pytest.raises(ValueError):
            dec.sample_drafted(*two, **kw)
    with pytest.raises(ValueError):
        dec.sample_drafted(*two, draft=2, maxlen=3, uniforms=np.zeros((3, 5, 3), np.float32))
    with pytest.raises(TypeError):
        dec.sample_drafted(*two, draft=2, maxlen=3, uniforms=np.zeros((3, 5, 2)))
    fresh = decoder(stattn_mod, opt, P)
    with pytest.raises(ValueError, match="beam_stage"):
        fresh.sample_drafted(resident=True)
