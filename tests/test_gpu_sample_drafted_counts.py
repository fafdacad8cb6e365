"""The words drafted and kept that drafted sampling reports: a pair for every caption, of whole rounds."""
import numpy as np
import pytest

from test_gpu_sample_drafted import O, decoder, features, small, stattn_mod      # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


def test_every_video_of_several_groups_has_its_counts(stattn_mod, O):            # noqa: F811
    opt, P = small(O)
    b = O.synthetic_batch(opt, B=35, T=5, K=3, t=3, seed=73)
    u = np.random.RandomState(4).random_sample((9, 7, 35)).astype(np.float32)
    u = np.minimum(u, np.float32(1 - 2.0 ** -24))
    model = stattn_mod.Attention()
    tparams = model.init_tparams(P)
    model.gen_sample_drafted(tparams, opt, *features(b), draft=3, maxlen=9, uniforms=u)
    drafted, kept = tparams.decoder.draft_counts
    assert drafted.shape == kept.shape == (35,) and drafted.dtype == kept.dtype == np.int32
    dec = decoder(stattn_mod, opt, P)
    for v in (0, 15, 16, 33, 34):                                                # the counts of the call with this video alone
        dec.sample_drafted(*features(b, slice(v, v + 1)), draft=3, maxlen=9, uniforms=np.ascontiguousarray(u[:, :, v:v + 1]))
        assert (int(drafted[v]), int(kept[v])) == (int(dec.draft_counts[0][0]), int(dec.draft_counts[1][0])), v
    assert model.gen_sample_drafted(tparams, opt, *features(b, slice(0, 0)), draft=3, maxlen=9) == []
    assert all(c.shape == (0,) for c in tparams.decoder.draft_counts)


def test_counts_are_of_whole_rounds(stattn_mod, O):                              # noqa: F811
    """Checks of 0 keep every draft: a caption of maxlen = 1 counts all eight words of its one round."""
    opt, P = small(O)
    b = O.synthetic_batch(opt, B=4, T=5, K=3, t=3, seed=74)
    u = np.full((1, 17, 4), 0.5, np.float32)
    u[:, 8:16] = 0
    dec = decoder(stattn_mod, opt, P)
    got = dec.sample_drafted(*features(b), draft=8, maxlen=1, uniforms=u)
    assert [len(w) for w, _ in got] == [1] * 4
    assert dec.draft_counts[0].tolist() == [8] * 4 and dec.draft_counts[1].tolist() == [8] * 4
