"""Drafted sampling walked through in 64 bits, one caption after the other: what stattn_sample_drafted returns for given uniform numbers.

Only decisions that no rounding of the device can turn are taken.  Its logits lie within LOGITS of the oracle's, so a probability is off
by a factor of e^(2 LOGITS) at most; the draft's logits are products of rounded values, so what counts there is whether an activation,
off by STATES at most, may round to another code: where it may, the words' logits are taken to be off by what that changes.  A number
nearer to a border than these bounds allow ends the comparison of its caption.  LOGITS is the bar of the parity tests; STATES is a tenth
of theirs, since a state is a sum of at most 1024 products of numbers of about 1 (2^-24 each, a few of them in the same direction), and
is checked on the device before a walk is compared."""
import numpy as np

LOGITS, STATES = 1e-4, 1e-5


def rounded(x):
    """A float64 matrix rounded to the 4-bit form, along its rows: steps of 1/2, 1 and 2 under the block's scale, up to 6."""
    rows, cols = x.shape
    b = np.pad(x, ((0, 0), (0, -cols % 32))).reshape(rows, -1, 32)
    top = np.abs(b).max(2, keepdims=True)
    scale = np.exp2(np.clip(np.frexp(top)[1] - 3.0, -126, 127))
    m = np.abs(b) / scale
    step = np.where(m < 2, 0.5, np.where(m < 4, 1.0, 2.0))
    v = np.minimum(np.round(m / step) * step, 6.0)
    return (np.copysign(v, b) * scale).reshape(rows, -1)[:, :cols]


def softmax(x):
    e = np.exp(x - x.max())
    return e / e.sum()


def draw(w, u, off):
    """The first word whose running sum exceeds u times the total, or None if that depends on sums that are off by `off`."""
    c = np.cumsum(w)
    t, some = u * c[-1], np.flatnonzero(w > 0)
    word = int(min(np.searchsorted(c, t, side="right"), some[-1]))
    if word > some[0] and t - (c[word] - w[word]) <= 2 * off:
        return None
    if word < some[-1] and c[word] - t <= 2 * off:
        return None
    return word


class Walk(object):
    """`always_keep` and `redraw_from_target` are mistakes, for showing that the comparison would see them."""

    def __init__(self, O, P, opt, always_keep=False, redraw_from_target=False):
        self.O, self.opt, self.P = O, opt, O.cast_params(P, np.float64)
        head = np.asarray(P['ff_logit_W'], np.float64)
        self.head = rounded(np.ascontiguousarray(head.T)).T.copy()          # (dim_word, n_words)
        self.mag = np.abs(self.head)
        self.always_keep, self.redraw_from_target = always_keep, redraw_from_target

    def state(self, x, h, c):
        """One step from word x: (h, c, readout activations (E,))."""
        O, P, opt, v = self.O, self.P, self.opt, self.video
        x = np.array([x], np.int64)
        _, r = O.f_next(P, opt, x, *v, h, c, extras=True, cached=self.cached)
        E = P['Wemb'].shape[1]
        emb = np.where((x < 0)[:, None], np.zeros((1, E)), P['Wemb'][np.maximum(x, 0)])
        _, z = O.readout(P, opt, r['h'], emb, r['ctx'], 0.5, 0.5)
        return r['h'], r['c'], 0.5 * np.tanh(z[0])

    def proposal(self, a):
        """(q, the factor - 1 by which its entries may be off)"""
        here = rounded(a[None])[0]
        apart = np.maximum(np.abs(rounded(a[None] + STATES)[0] - here), np.abs(rounded(a[None] - STATES)[0] - here))
        q = softmax(here @ self.head + self.P['ff_logit_b'])
        return q, float(np.expm1(2 * (1e-5 + (apart @ self.mag).max())))

    def target(self, a):
        return softmax(a @ self.P['ff_logit_W'] + self.P['ff_logit_b']), float(np.expm1(2 * LOGITS))

    def caption(self, batch, v, uniforms, draft, maxlen):
        """dict(words: as far as they are certain; whole: all of them; score; drafted, kept: None unless every round is certain)"""
        g, gm, l, m = (np.asarray(batch[k][v], np.float64) for k in ('ctxg', 'mask_ctxg', 'ctxl', 'ctxm'))
        self.video = (g, gm, l, None, m, None)
        self.cached = self.O.project_video(self.P, self.opt, g, l, m)
        _, h, c = self.O.sampler_closures(self.P, self.opt, np.float64)[0](g, gm)
        h, c, x = h[None], c[None], -1
        words, score, drafted, kept = [], 0.0, 0, 0
        for r in range(maxlen):
            u = uniforms[r, :, v].astype(np.float64)
            states, d, n, word = [], [], 0, None
            xs, hj, cj = x, h, c
            while True:                                                     # one position after the other, as far as the check goes
                hj, cj, a = self.state(xs, hj, cj)
                states.append((hj, cj))
                p, ep = self.target(a)
                if n == draft:
                    word = draw(p, u[2 * draft], ep)
                    break
                q, eq = self.proposal(a)
                dn = draw(q, u[n], eq)
                if dn is None:
                    break
                uq, pd = u[draft + n] * q[dn], p[dn]
                if abs(uq - pd) <= eq * uq + ep * pd:
                    break
                if not uq < pd and not self.always_keep:
                    rest, off = np.maximum(p - q, 0), ep + eq
                    if self.redraw_from_target:
                        rest, off = p, ep
                    if rest.sum() > 2 * off:
                        word = draw(rest, u[2 * draft], off)
                    break
                d.append((dn, pd))
                n, xs = n + 1, dn
            new = d + ([] if word is None else [(word, p[word])])
            for w, pw in new:
                words.append(w)
                score += pw
                if w == 0 or len(words) == maxlen:
                    if word is None:
                        drafted = kept = None
                    elif drafted is not None:
                        drafted, kept = drafted + draft, kept + n
                    return dict(words=words, whole=True, score=score, drafted=drafted, kept=kept)
            if word is None:
                return dict(words=words, whole=False, score=None, drafted=None, kept=None)
            drafted, kept = drafted + draft, kept + n
            x, (h, c) = word, states[n]


def stretch(v):
    """Words of a row that a wave of the softmax takes."""
    return ((v + 15) // 16 + 511) // 512 * 512


def case(O, n_words, dim_word, nvid, seed, sharp=3.0, **options):
    """(options, parameters, features): a decoder whose words at the ends of the stretches have most of the probability, so that draws
    fall there and seldom near a border, and whose logits are wide enough for the 4-bit head to be a coarse draft."""
    opt = O.default_options(dim=64, dim_word=dim_word, n_words=n_words, ctxg_dim=64, ctxl_dim=32, ctxm_dim=32, ctxglm_dim=64, **options)
    P = O.random_params(opt, seed=seed, dtype=np.float32)
    b = O.synthetic_batch(opt, B=nvid, T=5, K=3, t=3, seed=seed + 1)
    P['ff_logit_W'] = P['ff_logit_W'] * np.float32(sharp * 3)              # (activations of about a third)
    ends = {0, 1, n_words - 1}
    for s in (stretch(n_words), 512):
        for k in range(1, 17):
            ends |= {e for e in (s * k - 1, s * k, n_words // 512 * 512 - s * k) if 0 <= e < n_words}
    ends = sorted(ends)
    bias = np.zeros(n_words)
    bias[ends] = np.log(n_words * 2.0 / len(ends)) + 2 * sharp
    bias[0] -= 1.0
    P['ff_logit_b'] = bias.astype(np.float32)
    return opt, P, b


def uniforms(draft, maxlen, nvid, seed):
    """Random numbers; the second caption's drafts are drawn by 0 in its first round, the third's words all by the largest number under 1,
    the fourth keeps every draft."""
    u = np.random.RandomState(seed).random_sample((maxlen, 2 * draft + 1, nvid)).astype(np.float32)
    u = np.minimum(u, np.float32(1 - 2.0 ** -24))
    if nvid > 3:
        u[0, :draft, 1] = 0
        u[:, :draft, 2] = u[:, 2 * draft, 2] = 1 - 2.0 ** -24
        u[:, draft:2 * draft, 3] = 0
    return u


CASES = [  # n_words, dim_word, nvid, draft, maxlen, seed, options
    (37, 64, 16, 4, 12, 11, {}),
    (513, 64, 16, 3, 10, 12, {}),
    (513, 192, 16, 5, 8, 13, dict(prev2out=False)),
    (8193, 192, 16, 8, 10, 14, {}),
    (8192, 128, 1, 2, 20, 22, dict(ctx2out=False)),
    (12001, 512, 12, 4, 10, 16, {}),
    (20000, 192, 13, 3, 8, 17, dict(selector=False)),
    (98303, 64, 8, 4, 6, 18, {}),
    (98305, 192, 9, 6, 8, 19, {}),
]
