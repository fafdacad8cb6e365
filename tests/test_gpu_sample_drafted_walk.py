"""Drafted sampling against a walk in 64 bits (drafted_walk.py) with the same uniform numbers: the words, the counts of drafted and kept
words and the scores.  Vocabularies from one stretch of the draws to all sixteen with tails of every kind, one and several workgroups in
the check (98305 words), vocabulary heads of up to 512 columns, one to sixteen captions, 3 to 144 rows in the full-precision product.

Small vocabularies also by the distribution of what comes out, with a draft that is far from the target."""
import numpy as np
import pytest

import drafted_walk as D
from test_gpu_sample_drafted import O, decoder, features, small, stattn_mod      # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


def states_are_close(O, P, opt, dec, b):      # noqa: F811
    """The premise of the comparison, on the first video: states within D.STATES of the oracle's and logits within D.LOGITS, over words
    that follow one another on either side's own states."""
    P64 = O.cast_params(P, np.float64)
    g, gm, l, m = (np.asarray(b[k][0]) for k in ('ctxg', 'mask_ctxg', 'ctxl', 'ctxm'))
    wide = [a.astype(np.float64) for a in (g, gm, l, m)]
    _, h64, c64 = O.sampler_closures(P64, opt, np.float64)[0](wide[0], wide[1])
    h, c = (a.astype(np.float32)[None] for a in (h64, c64))
    h64, c64 = h64[None], c64[None]
    for x in (-1, 1, opt['n_words'] - 1, 2, 0, opt['n_words'] // 2):
        x = np.array([x], np.int64)
        (_, _, h, c), ex = dec.f_next(x, g, gm, l, None, m, None, h, c, extras=True)
        (_, _, h64, c64), r = O.f_next(P64, opt, x, wide[0], wide[1], wide[2], None, wide[3], None, h64, c64, extras=True)
        assert np.abs(h - h64).max() <= D.STATES and np.abs(c - c64).max() <= D.STATES
        assert np.abs(ex['logit'] - r['logit']).max() <= D.LOGITS


@pytest.mark.parametrize("precision", ["fp32", "split"])
@pytest.mark.parametrize("n_words,dim_word,nvid,draft,maxlen,seed,options", D.CASES)
def test_words_counts_and_scores(stattn_mod, O, n_words, dim_word, nvid, draft, maxlen, seed, options, precision):      # noqa: F811
    opt, P, b = D.case(O, n_words, dim_word, nvid, seed, **options)
    u = D.uniforms(draft, maxlen, nvid, seed)
    dec = decoder(stattn_mod, opt, P, precision=precision)
    states_are_close(O, P, opt, dec, b)
    got = dec.sample_drafted(*features(b), draft=draft, maxlen=maxlen, uniforms=u)
    drafted, kept = dec.draft_counts
    walk = D.Walk(O, P, opt)
    compared = 0
    for v in range(nvid):
        want = walk.caption(b, v, u, draft, maxlen)
        n = len(want['words'])
        assert got[v][0][:n] == want['words'], v
        if want['whole']:
            assert len(got[v][0]) == n, v
            np.testing.assert_allclose(got[v][1], want['score'], rtol=np.expm1(2 * D.LOGITS), atol=1e-6 * n)
        if want['kept'] is not None:
            assert (int(drafted[v]), int(kept[v])) == (want['drafted'], want['kept']), v
        compared += n
    assert compared >= (8 if nvid == 1 else 37)


def test_a_coarse_draft_leaves_the_decoders_distribution(stattn_mod, O):      # noqa: F811
    """4000 captions of two words of one video, the logits wide enough that the draft is 0.2 and more (total variation) away from the
    target: the first word's and the second's distribution against the oracle's.  For n draws over k words the total variation's mean is
    at most sqrt(k / n) / 2 = 0.048 and its standard deviation at most 1 / (2 sqrt(n)) = 0.008; 0.08 is four of them away, and far under
    what words that nobody checked would show."""
    opt, P = small(O, 50.0)
    b = O.synthetic_batch(opt, B=1, T=5, K=3, t=3, seed=70)
    walk = D.Walk(O, P, opt)
    g, gm, l, m = (np.asarray(b[k][0], np.float64) for k in ('ctxg', 'mask_ctxg', 'ctxl', 'ctxm'))
    walk.video, walk.cached = (g, gm, l, None, m, None), O.project_video(walk.P, opt, g, l, m)
    _, h, c = O.sampler_closures(walk.P, opt, np.float64)[0](g, gm)
    h, c, a = walk.state(-1, h[None], c[None])
    p1, q1 = walk.target(a)[0], walk.proposal(a)[0]
    p2, q2 = np.zeros((37, 37)), np.zeros((37, 37))
    for w in range(37):
        a = walk.state(w, h, c)[2]
        p2[w], q2[w] = walk.target(a)[0], walk.proposal(a)[0]
    want = np.append(p1[1:] @ p2[1:], p1[0])                                # [37]: the caption ended with its first word
    unchecked = np.append(q1[1:] @ q2[1:], q1[0])
    assert 0.5 * np.abs(p1 - q1).sum() > 0.2 and 0.5 * np.abs(want - unchecked).sum() > 0.2
    shared = np.minimum(p1, q1)                                             # a refused word drawn from the target itself would show as well
    assert 0.5 * np.abs(shared + (1 - shared.sum()) * p1 - p1).sum() > 0.15
    dec = decoder(stattn_mod, opt, P)
    dec.set_seed(3)
    dec.beam_stage(*(np.repeat(x, 16, 0) for x in features(b)))
    first, second = np.zeros(37), np.zeros(38)
    for _ in range(250):
        for words, _ in dec.sample_drafted(draft=3, maxlen=2, resident=True):
            first[words[0]] += 1
            second[words[1] if len(words) > 1 else 37] += 1
    assert 0.5 * np.abs(first / first.sum() - p1).sum() < 0.08
    assert 0.5 * np.abs(second / second.sum() - want).sum() < 0.08
