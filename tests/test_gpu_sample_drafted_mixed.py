"""Drafted sampling between other calls: shapes that change from call to call (its buffers are kept), other searches and
training steps on the same handle.  A handle's results are those of a new one."""
import numpy as np
import pytest

from test_gpu_sample_drafted import O, decoder, features, small, stattn_mod      # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu
SHAPES = [(3, 5, 3, 2, 9), (3, 7, 3, 2, 9), (3, 5, 3, 4, 9), (1, 5, 4, 2, 12), (16, 9, 6, 8, 5), (3, 5, 3, 2, 9), (1, 5, 4, 2, 9), (3, 7, 3, 2, 9)]


def calls(O, opt):      # noqa: F811
    for i, (nvid, T, K, draft, maxlen) in enumerate(SHAPES):
        b = O.synthetic_batch(opt, B=nvid, T=T, K=K, t=4, seed=90 + i)
        u = np.random.RandomState(i).random_sample((maxlen, 2 * draft + 1, nvid)).astype(np.float32)
        yield b, dict(draft=draft, maxlen=maxlen, uniforms=np.minimum(u, np.float32(1 - 2.0 ** -24)))


@pytest.mark.parametrize("precision", ["fp32", "bf16"])
def test_one_handle_many_shapes(stattn_mod, O, precision):      # noqa: F811
    opt, P = small(O)
    dec = decoder(stattn_mod, opt, P, precision=precision)
    for b, kw in calls(O, opt):
        want = decoder(stattn_mod, opt, P, precision=precision).sample_drafted(*features(b), **kw)
        assert dec.sample_drafted(*features(b), **kw) == want
        assert dec.sample_drafted(resident=True, **kw) == want


def test_between_searches_and_training_steps(stattn_mod, O):      # noqa: F811
    opt, P = small(O)
    dec, other = decoder(stattn_mod, opt, P), decoder(stattn_mod, opt, P)
    train = O.synthetic_batch(opt, B=6, T=5, K=3, t=6, seed=80)
    for b, kw in calls(O, opt):
        for d in (dec, other):
            d.set_batch(**train)
            d.forward_train()
            d.backward()
            d.update()
            d.sync()
        fresh = decoder(stattn_mod, opt, {k: dec.get_param(k) for k in P})
        want = fresh.sample_drafted(*features(b), **kw)
        beams = other.beam_search(*features(b), k=2, maxlen=7)
        got = dec.sample_drafted(*features(b), **kw)
        assert got == want
        for (words, scores), (words2, scores2) in zip(dec.beam_search(k=2, maxlen=7, resident=True), beams):
            assert words == words2                                              # as on a handle that never drafted
            np.testing.assert_array_equal(scores, scores2)
        assert dec.sample_drafted(resident=True, **kw) == want
    for k in P:                                                                 # nor do its training steps differ
        np.testing.assert_array_equal(dec.get_param(k), other.get_param(k))
