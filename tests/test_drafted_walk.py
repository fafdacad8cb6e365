"""The walk that the GPU tests of drafted sampling compare with (drafted_walk.py): its rounding is the format's, and the comparison would
see a sampler that keeps every draft or draws a refused word's place from the target itself."""
import numpy as np
import pytest

import drafted_walk as D
import ops_reference as R
from oracle import stattn_oracle as O


def test_rounding():
    rng = np.random.RandomState(0)
    x = rng.standard_normal((40, 111)) * np.exp2(rng.randint(-30, 30, (40, 1)))
    x[3], x[4, :7] = np.arange(111) / 4, 0
    np.testing.assert_array_equal(D.rounded(x), R.values(*R.quantize(x), 111))


@pytest.mark.parametrize("n_words,dim_word,nvid,draft,maxlen,seed,options", [c for c in D.CASES if c[0] <= 20000 and c[2] > 1])
def test_mistakes_are_seen(n_words, dim_word, nvid, draft, maxlen, seed, options):
    opt, P, b = D.case(O, n_words, dim_word, nvid, seed, **options)
    u = D.uniforms(draft, maxlen, nvid, seed)
    walk = D.Walk(O, P, opt)
    right = [walk.caption(b, v, u, draft, maxlen) for v in range(nvid)]
    assert sum(len(r['words']) for r in right) >= 40 and any(r['whole'] for r in right)
    for mistake in ({'always_keep': True}, {'redraw_from_target': True}):
        walk = D.Walk(O, P, opt, **mistake)
        wrong = [walk.caption(b, v, u, draft, maxlen) for v in range(nvid)]
        assert any(a != z for r, w in zip(right, wrong) for a, z in zip(r['words'], w['words'])), mistake
