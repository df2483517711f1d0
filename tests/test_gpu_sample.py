"""Sampling (ak_sample) on the GPU, against 64 bits (numpy, test infrastructure).

Tokens are compared exactly except where a decision of the 64-bit evaluation lies within 1e-5 of its threshold; the log
probabilities within 2^-20 of 1 + |log p| per unit of (largest logit difference / temperature): a logit difference is exact in
fp32, its quotient and exponential are rounded."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

from _lib import check, Dev, f2bf_array, bf2f_array
from _ops import Stream, Graph
from _step import step, sample64

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))


class Rows:
    """b rows of logits and their settings (None: the argument is left out)."""

    def __init__(self, bits, temp=None, top_k=None, top_p=None, min_p=None, u=None, pad=0):
        self.bits = bits
        self.b, self.vocab = bits.shape
        self.ld = self.vocab + pad
        mem = np.full((self.b, self.ld), 0x7F7F, dtype=np.uint16)  # between the rows: never to be chosen
        mem[:, :self.vocab] = bits
        full = lambda v, t: None if v is None else np.broadcast_to(np.asarray(v, dtype=t), (self.b,)).copy()  # noqa: E731
        self.temp, self.top_k = full(temp, np.float32), full(top_k, np.int32)
        self.top_p, self.min_p = full(top_p, np.float32), full(min_p, np.float32)
        self.u = full(0.5 if u is None else u, np.float32)
        dev = lambda v: None if v is None else Dev.of(v)  # noqa: E731
        self.L = Dev.of(mem)
        self.d = [dev(v) for v in (self.temp, self.top_k, self.top_p, self.min_p, self.u)]
        self.tok, self.lp = Dev.of(np.full(self.b + 1, 99, dtype=np.int32)), Dev.of(np.full(self.b + 1, 99, dtype=np.float32))

    def call(self, stream=None, logp=True):
        return step().ak_sample(self.L.p, self.ld, *[x.p if x else None for x in self.d], self.b, self.vocab, self.tok.p,
                                self.lp.p if logp else None, stream)

    def got(self):
        check(step().ak_synchronize())
        t, l = self.tok.get(np.int32, self.b + 1), self.lp.get(np.float32, self.b + 1)
        assert t[self.b] == 99 and l[self.b] == 99
        return t[:self.b], l[:self.b]

    def run(self):
        check(self.call())
        return self.got()

    def compare(self, got, least=0.9, tol=1e-5):
        tok, lp = got
        sure = 0
        for i in range(self.b):
            v = lambda x, off: off if x is None else x[i]  # noqa: E731
            heat = min(float(v(self.temp, 1.0)), 1.44e30)  # (more counts as that, and less than fp32's normal numbers as their first)
            heat = max(heat, 2.0 ** -126) if heat > 0 else heat
            want, wl, near = sample64(self.bits[i], heat, int(v(self.top_k, 0)), float(v(self.top_p, 1.0)),
                                      float(v(self.min_p, 0.0)), float(self.u[i]), tol)
            if near:
                continue
            sure += 1
            assert tok[i] == want, (i, tok[i], want, heat, v(self.top_k, 0), v(self.top_p, 1), v(self.min_p, 0), self.u[i])
            l = bf2f_array(self.bits[i]).astype(np.float64)
            spread = np.ptp(l[np.isfinite(l)]) / (heat if heat > 0 else 1.0) if np.isfinite(l).any() else 0.0
            assert abs(lp[i] - wl) <= 2.0 ** -20 * (1 + abs(wl)) * (1 + spread)
        assert sure >= int(least * self.b)


def logits(rng, b, vocab, spread=2.0, peaks=8):
    x = rng.standard_normal((b, vocab)) * spread
    for r in x:
        r[rng.integers(0, vocab, peaks)] += 6 + 6 * rng.random(peaks)
    return f2bf_array(x.astype(np.float32).ravel()).reshape(b, vocab)


def settings(rng, b, vocab):
    pick = lambda p, x, off: np.where(rng.random(b) < p, x, off)  # noqa: E731
    return dict(temp=pick(0.9, 0.2 + 1.5 * rng.random(b), 0.0), top_k=pick(0.5, np.exp(rng.random(b) * np.log(vocab + 1)), 0).astype(int),
                top_p=pick(0.6, rng.random(b), 1.0), min_p=pick(0.4, 10.0 ** -(4 * rng.random(b)), 0.0), u=rng.random(b))


@pytest.mark.parametrize("peaks", [0, 8])
@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 1000, 1003, 4099, 16384, 16385, 33000, 152064])
def test_against_64_bits(vocab, peaks):
    rng = np.random.default_rng(vocab + peaks)
    b = 12 if vocab > 20000 else 60
    x = Rows(logits(rng, b, vocab, peaks=min(peaks, vocab)), pad=vocab % 5, **settings(rng, b, vocab))
    x.compare(x.run(), least=0.7)


@pytest.mark.parametrize("vocab", [253951, 253953, 262144, 1048576])
def test_large_vocabularies(vocab):
    """Where the chunks' windows fit into LDS and where they do not, up to the limit."""
    rng = np.random.default_rng(vocab)
    b = 10
    s = settings(rng, b, vocab)
    s["temp"] = np.full(b, 0.8)
    s["top_k"][:4] = [50, 1, 400, 0]
    x = Rows(logits(rng, b, vocab, peaks=30), pad=3, **s)
    # 4e-6 n of the draws without a filter are too near where all n tokens weigh the same; the peaks weigh e^7 and more of the rest
    x.compare(x.run(), least=0.3, tol=2e-6)


@pytest.mark.parametrize("one", ["top_k", "top_p", "min_p", None])
def test_each_filter_alone(one):
    rng = np.random.default_rng(7)
    b, vocab = 40, 5000
    s = settings(rng, b, vocab)
    s = {"u": s["u"], **({one: dict(top_k=rng.integers(1, 300, b), top_p=0.3 + 0.6 * rng.random(b),
                                    min_p=0.2 * rng.random(b))[one]} if one else {})}
    x = Rows(logits(rng, b, vocab), **s)
    x.compare(x.run())


def test_flat_rows_whose_border_is_far_down():
    """Logits around 0 of either sign: what is kept reaches keys far below the largest's."""
    rng = np.random.default_rng(9)
    b, vocab = 48, 40000
    x = f2bf_array((rng.standard_normal((b, vocab)) * 0.7).astype(np.float32).ravel()).reshape(b, vocab)
    top_k = np.where(np.arange(b) % 3 == 0, rng.integers(10000, 40000, b), 0)
    top_p = np.where(np.arange(b) % 3 == 1, 0.9 + 0.0999 * rng.random(b), 1.0)
    min_p = np.where(np.arange(b) % 3 == 2, 0.01 * rng.random(b), 0.0)
    r = Rows(x, None, top_k, top_p, min_p, rng.random(b))
    # exponents below 16 are off by 2^-20 at most, weights and their sums by 2^-20 ln 2 and a step: 8e-7.  (Decisions are 1 / 40000
    # apart: 1e-5 on either side would leave the half of them out.)
    r.compare(r.run(), least=0.7, tol=2e-6)


def far_borders(rng, b, vocab):
    """Top-k or top-p of each row, never both, that keeps a large part of a flat row."""
    ks = np.arange(b) % 2 == 0
    return np.where(ks, rng.integers(vocab // 10, vocab - vocab // 50, b), 0), np.where(ks, 1.0, 0.5 + 0.4999 * rng.random(b))


@pytest.mark.parametrize("zeros", [0.0, 0.2])
@pytest.mark.parametrize("vocab", [8191, 8192, 8199, 16385, 100277])
def test_long_flat_rows(vocab, zeros):
    """One border far down, which a sample of the row finds: also among zeros of either sign, and with min-p's around it."""
    rng = np.random.default_rng(vocab)
    b = 20
    x = rng.standard_normal((b, vocab)) * (0.5 + 0.5 * rng.random((b, 1)))
    x = np.where(rng.random((b, vocab)) < zeros, np.where(rng.random((b, vocab)) < 0.5, 0.0, -0.0), x)
    bits = f2bf_array(x.astype(np.float32).ravel()).reshape(b, vocab)
    top_k, top_p = far_borders(rng, b, vocab)
    min_p = np.where(np.arange(b) % 5 == 1, 1e-6, np.where(np.arange(b) % 5 > 2, 0.003 + 0.04 * rng.random(b), 0.0))
    r = Rows(bits, None, top_k, top_p, min_p, rng.random(b))
    # (as above.  A draw is within 2e-6 of one of n tokens' ends with a chance of 4e-6 n, 0.40 of 100277 and 0.07 of 16385; top-p's
    # border, in the half of the rows, is so with about twice that.  Of the most, 0.6 (0.5 + 0.5 0.5) = 0.45 of 20 rows are left,
    # give or take 0.11 a standard deviation; of 16385 0.87 0.93 = 0.8.)
    r.compare(r.run(), least=0.15 if vocab > 20000 else 0.5, tol=2e-6)


@pytest.mark.parametrize("vocab", [1000, 2617, 8199, 40000])
def test_borders_behind_all_weights(vocab):
    """Cold rows: what weighs anything ends within the keys that are counted first, the border of top-k (or of a top-p of all but
    nothing) is far behind."""
    rng = np.random.default_rng(vocab)
    b = 60
    kind = np.arange(b) % 4
    top_k = np.where(kind < 3, rng.integers(vocab // 2, vocab, b), 0)
    top_p = np.where(kind < 2, 0.3 + 0.69 * rng.random(b), np.where(kind == 2, 1.0, np.float32(1 - 2.0 ** -24)))
    min_p = np.where(kind == 1, 0.01, 0.0)
    x = logits(rng, b, vocab, peaks=40)
    x[kind == 2, vocab // 3:] = 0xFF80  # fewer tokens than top-k keeps
    r = Rows(x, 0.1 + 0.4 * rng.random(b), top_k, top_p, min_p, rng.random(b))
    r.compare(r.run(), least=0.7, tol=2e-6)


def test_top_k_of_more_than_there_are_far_below_zero():
    """Logits at the lowest finite numbers, below which there are fewer keys than are counted first."""
    rng = np.random.default_rng(23)
    b, vocab = 12, 700
    x = rng.integers(0xFF00, 0xFF80, (b, vocab)).astype(np.uint16)
    x[:, 50:] = 0xFF80
    r = Rows(x, 1e37, np.where(np.arange(b) % 2 == 0, 300, 0), np.where(np.arange(b) % 3 == 0, 1.0, 0.7), None, rng.random(b))
    r.compare(r.run(), least=0.7, tol=2e-6)


@pytest.mark.parametrize("kind", ["ascending", "descending", "blocks", "masked", "nan", "equal", "shifted"])
@pytest.mark.parametrize("vocab", [16384, 65536])
def test_long_rows_that_a_sample_misjudges(kind, vocab):
    rng = np.random.default_rng(vocab)
    b = 16
    x = rng.standard_normal((b, vocab)) * 0.8
    # every (vocab / 8192)th eight logits are those that a sample of 8192 in eights takes
    eights = np.arange(vocab) // 8 % (vocab // 8192) == 0
    if kind in ("ascending", "descending"):
        x = np.sort(x, axis=1)[:, :: 1 if kind == "ascending" else -1]
    elif kind == "blocks":
        x[:, eights] -= 4.0
    elif kind == "masked":
        x[:, eights] = -np.inf
    elif kind == "nan":
        x[:, eights] = np.nan
    elif kind == "equal":
        x[:, ~eights] = -0.25
    else:
        x[:, eights] += 0.5
    bits = f2bf_array(x.astype(np.float32).ravel()).reshape(b, vocab)
    top_k, top_p = far_borders(rng, b, vocab)
    r = Rows(bits, None, top_k, top_p, None, rng.random(b))
    r.compare(r.run(), least=0.5, tol=2e-6)


@pytest.mark.parametrize("tiny", [0.0, 1e-6, 1e-15, 1e-30])
@pytest.mark.parametrize("shift", [0.0, -1.0, 3.0])
def test_borders_among_zeros_and_tiny_values(tiny, shift):
    """Many logits of 0, -0 and magnitudes far below the largest: borders fall among them, where keys are far apart."""
    rng = np.random.default_rng(19)
    b, vocab = 40, 9000
    x = rng.standard_normal((b, vocab)) + np.where(rng.random((b, vocab)) < 0.2, shift, 0.0)
    kind = rng.random((b, vocab))
    x = np.where(kind < 0.4, tiny * rng.standard_normal((b, vocab)), x)
    bits = f2bf_array(x.astype(np.float32).ravel()).reshape(b, vocab)
    bits[(kind > 0.4) & (kind < 0.45)] = 0x0000
    bits[(kind > 0.45) & (kind < 0.5)] = 0x8000
    bits[::7] |= 0x8000  # no positive logit
    top_k = np.where(np.arange(b) % 3 == 0, rng.integers(1000, 8000, b), 0)
    top_p = np.where(np.arange(b) % 3 != 0, 0.3 + 0.69 * rng.random(b), 1.0)
    top_p[::4] = 0.9
    min_p = np.where(np.arange(b) % 5 == 2, 0.03, 0.0)
    r = Rows(bits, 0.5 + rng.random(b), top_k, top_p, min_p, rng.random(b))
    # weights of |d / T| below 16: 8e-7 (as above)
    r.compare(r.run(), least=0.7, tol=2e-6)


@pytest.mark.parametrize("zero", list(range(506, 518)) + list(range(1018, 1030)) + list(range(8186, 8198)) + [16382, 16384])
def test_zeros_at_a_windows_end(zero):
    """0 and -0 at every place around the last of the keys that are counted first."""
    rng = np.random.default_rng(zero)
    x = np.full((4, 600), 0xC000, dtype=np.uint16)
    x[:, 300] = zero  # (the key of the largest logit is this far above 0's)
    x[:, 301:340] = rng.integers(1, zero + 1, 39)
    x[:, 100:200:2], x[:, 101:200:2] = 0x8000, 0x0000
    r = Rows(x, 1e-38, [60, 0, 139, 140], [1.0, 0.8, 0.999, 0.6], None, rng.random(4))
    r.compare(r.run(), least=0.5, tol=2e-6)


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 1.0, 1e30])
def test_rows_of_any_size(scale):
    rng = np.random.default_rng(3)
    b, vocab = 24, 3001
    x = f2bf_array((rng.standard_normal((b, vocab)) * scale).astype(np.float32).ravel()).reshape(b, vocab)
    x[::2] |= 0x8000  # all below 0
    s = settings(rng, b, vocab)
    s["temp"] = s["temp"] * scale
    r = Rows(x, **s)
    r.compare(r.run(), least=0.7)


def test_equal_logits():
    """All weights alike: sums are exact, so the token is known to the last one.  The lowest tokens are kept."""
    vocab, b = 20000, 9
    x = np.full((b, vocab), f2bf_array(np.array([-3.0], dtype=np.float32))[0])
    top_k = [0, 1, 777, 777, 0, 0, 0, 0, 777]
    top_p = [1, 1, 1, 0.5, 0.25, 0.0, 1, 1, 1]
    min_p = [0, 0, 0, 0, 0, 0, 1.0, 0.5, 0.0]
    u = np.float32([0.75, 0.99, 0.5, 0.5, 0.5, 0.99, 0.25, 1 - 2.0 ** -24, 1 - 2.0 ** -24])
    tok, lp = Rows(x, None, top_k, top_p, min_p, u).run()
    # kept: all, 1, 777, 389 (388.5 of 777 reached), 5000, 1, all, all, 777
    assert tok.tolist() == [15000, 0, 388, 194, 2500, 0, 5000, 19999, 776]  # (u times 20000 is 0.0012 below it)
    assert np.allclose(lp, -np.log(vocab), atol=1e-6)


def test_zeros_of_either_sign_are_equal():
    x = np.full((3, 400), f2bf_array(np.array([-9.0], dtype=np.float32))[0])
    x[:, 10:20:2], x[:, 11:20:2] = 0x8000, 0x0000
    tok, _ = Rows(x, [0.0, 1.0, 1.0], [0, 3, 3], None, None, [0.5, 0.5, 0.99]).run()
    assert tok.tolist() == [10, 11, 12]


def test_masked_infinite_and_empty_rows():
    rng = np.random.default_rng(6)
    vocab = 30000
    x = logits(rng, 9, vocab)
    x[0] = 0xFF80                      # nothing above -inf
    x[1] = 0x7FC0                      # NaN alone
    x[2], x[2, 17] = 0xFF80, 0xC000    # one token left
    x[3, 100], x[3, 29000] = 0x7F80, 0x7F80   # +inf twice
    x[4, ::2] = 0x7FC1                 # NaN counts as -inf
    x[5] = 0xFF80
    x[5, 5:40] = f2bf_array(np.arange(35).astype(np.float32) * 0.1)
    x[6] = 0xFF7F                      # the type's lowest value
    x[7], x[7, 29999] = 0xFF7F, 0x7F7F
    x[8] = 0xFF80
    x[8, 3], x[8, 4] = 0xFF7F, 0xFF7E
    for k, p, m in ((0, 1.0, 0.0), (5, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.1), (28000, 0.999, 1e-6)):
        r = Rows(x, 0.8, k, p, m, 0.6)
        with np.errstate(over="ignore"):
            tok, lp = r.run()
        assert tok[0] == -1 and tok[1] == -1 and lp[0] == 0 and lp[1] == 0
        assert tok[2] == 17 and lp[2] == 0
        assert tok[3] == (29000 if k != 1 else 100) and abs(lp[3] + np.log(2)) < 1e-6
        assert tok[4] % 2 == 1 and 5 <= tok[5] < 40 and tok[7] == 29999 and tok[8] in (3, 4)
        for i in (4, 5):
            want, wl, near = sample64(x[i], float(np.float32(0.8)), k, p, m, 0.6)
            assert near or (tok[i] == want and abs(lp[i] - wl) < 1e-4)
    tok, _ = Rows(x, 0.0, 3, 0.5, 0.1, 0.6).run()
    assert tok[:4].tolist() == [-1, -1, 17, 100] and tok[6] == 0


@pytest.mark.parametrize("nan", [0x7F81, 0x7FFF, 0xFF81, 0xFFFF])
@pytest.mark.parametrize("top", [0x7F80, 0x7F7F, 0x4000])
def test_nan_next_to_the_largest(nan, top):
    """The bits of a NaN are neighbours of an infinity's: it is never counted, let alone drawn."""
    rng = np.random.default_rng(21)
    x = f2bf_array(rng.standard_normal(6 * 9000).astype(np.float32)).reshape(6, 9000)
    x[:, 40::9] = nan
    x[:, 4500] = top
    r = Rows(x, 1.0, [1, 0, 3, 0, 8999, 0], [1.0, 0.4, 0.9, 1.0, 0.9999, 1.0], [0, 0, 0, 0.5, 0, 0], [0.0, 0.99, 0.5, 0.3, 0.7, 0.5])
    tok, lp = r.run()
    assert all(t < 40 or (t - 40) % 9 for t in tok)
    if top != 0x4000:  # (2: others are larger)
        assert (tok == 4500).all() and (lp == 0).all()
    else:
        r.compare((tok, lp), least=0.5)


@pytest.mark.parametrize("u", [1.0, float("nan"), 2.0, -1.0])
def test_numbers_that_are_none(u):
    """u outside [0, 1): one of the tokens that are kept."""
    rng = np.random.default_rng(22)
    x = logits(rng, 3, 5000)
    tok, _ = Rows(x, 1.0, [0, 10, 0], [1.0, 1.0, 0.5], None, u).run()
    l = bf2f_array(x).astype(np.float64)
    assert ((tok >= 0) & (tok < 5000)).all() and l[1, tok[1]] >= np.sort(l[1])[-10] and l[2, tok[2]] >= np.sort(l[2])[-2000]


def test_settings_out_of_their_ranges():
    """NaN and what is beyond a filter's range: off, or the most it can do."""
    rng = np.random.default_rng(8)
    nan, inf = float("nan"), float("inf")
    x = logits(rng, 1, 900).repeat(12, 0)
    r = Rows(x, [1, 1, 1, 1, 1, 1, 1, 1, nan, -1, 1e-45, 3e38], [-5, 900, 2 ** 31 - 1, 0, 0, 0, 0, 0, 0, 0, 0, 0],
             [nan, inf, 2, -1, 1, 1, 1, 1, 1, 1, 1, 1], [0, 0, 0, 0, nan, -1, 2, inf, 0, 0, 0, 0], 0.7)
    tok, _ = r.run()
    free, best = sample64(x[0], 1.0, 0, 1.0, 0.0, 0.7)[0], int(bf2f_array(x[0]).argmax())
    assert tok.tolist()[:11] == [free, free, free, best, free, free, best, best, best, best, best]
    assert abs(tok[11] - 630) <= 1  # all tokens alike


def test_draws_follow_the_distribution():
    """Over a grid of u the tokens come as often as their renormalised weights say, to one grid step."""
    rng = np.random.default_rng(10)
    n = 2000
    row = logits(rng, 1, 50, spread=1.0, peaks=0)
    x = Rows(row.repeat(n, 0), 0.7, 20, 0.95, 0.02, (np.arange(n) + 0.5) / n)
    tok, _ = x.run()
    l = bf2f_array(row[0]).astype(np.float64)
    p = np.exp((l - l.max()) / np.float32(0.7))
    p /= p.sum()
    order = np.argsort(-l, kind="stable")[:20]
    upto = np.cumsum(p[order])
    order = order[:int((upto < np.float32(0.95) * upto[-1]).sum()) + 1]
    order = order[p[order] >= np.float32(0.02) * p.max()]
    w = np.zeros(50)
    w[order] = p[order] / p[order].sum()
    assert np.abs(np.bincount(tok, minlength=50) / n - w).max() <= 1.01 / n


def test_without_filters_as_verification_draws():
    rng = np.random.default_rng(11)
    b, vocab = 32, 152064
    x = Rows(logits(rng, b, vocab, peaks=30), 0.5 + rng.random(b), u=rng.random(b))
    tok, lp = x.run()
    T, A, LP = Dev(4 * b), Dev(4 * b), Dev(4 * b)
    check(step().ak_spec_verify(x.L.p, x.ld, None, 0, None, None, x.d[4].p, x.d[0].p, b, 0, vocab, T.p, A.p, LP.p, None))
    check(step().ak_synchronize())
    assert np.array_equal(tok, T.get(np.int32, b)) and np.allclose(lp, LP.get(np.float32, b), atol=1e-5)


def test_many_rows_unaligned_and_without_logp():
    """More rows than a launch's scratch holds; rows at odd addresses."""
    rng = np.random.default_rng(12)
    b, vocab = 33000, 33
    x = Rows(logits(rng, b, vocab, peaks=3), pad=2, **settings(rng, b, vocab))
    tok, lp = x.run()
    for i in rng.integers(0, b, 300):
        want, wl, near = sample64(x.bits[i], float(x.temp[i]), int(x.top_k[i]), float(x.top_p[i]), float(x.min_p[i]), float(x.u[i]))
        assert near or tok[i] == want
    check(x.call(logp=False))
    assert np.array_equal(x.got()[0], tok)


def test_a_row_gives_the_same_alone():
    rng = np.random.default_rng(13)
    b, vocab = 20, 60001
    s = settings(rng, b, vocab)
    bits = logits(rng, b, vocab, peaks=0)
    tok, lp = Rows(bits, **s).run()
    for i in range(0, b, 3):
        t, l = Rows(bits[i:i + 1], **{k: v[i:i + 1] for k, v in s.items()}).run()
        assert t[0] == tok[i] and l[0] == lp[i]


def captured_before_any_call():
    """In a process of its own, whose library has no scratch: the form without it, then the form with it."""
    rng = np.random.default_rng(14)
    x = [Rows(logits(rng, 40, v, peaks=p), **settings(rng, 40, v)) for v, p in ((3000, 8), (50001, 0), (50001, 20))]
    s = Stream()
    graphs = [Graph(s, r.call) for r in x]
    plain = []
    for g in graphs:
        g.launch()
    s.sync()
    plain = [r.got() for r in x]
    for r, (t, l) in zip(x, plain):
        t2, l2 = r.run()
        assert np.array_equal(t, t2) and np.array_equal(l, l2)
        r.compare((t, l), least=0.7)
    graphs = [Graph(s, r.call) for r in x]
    for _ in range(3):
        for r, g, (t, l) in zip(x, graphs, plain):
            check(step().ak_memcpy_h2d(r.tok.p, ctypes.c_void_p(np.full(40, 5, dtype=np.int32).ctypes.data), 160))
            g.launch()
            s.sync()
            t2, l2 = r.got()
            assert np.array_equal(t, t2) and np.array_equal(l, l2)
            check(r.call())
    print("captured: the same")


def test_captured_without_and_with_scratch():
    r = subprocess.run([sys.executable, "-c", "import test_gpu_sample as t; t.captured_before_any_call()"], cwd=HERE,
                       capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "the same" in r.stdout, r.stdout + r.stderr


def faint_tokens(vocab):
    """Rows of a token that weighs 2^-45 of the largest at either end, the largest, and, in every other row, one of 2^-39.5 beside
    it, with u at either end and each filter; the tokens drawn."""
    faint, some, top = f2bf_array(np.array([8.8125, 12.625, 40.0], dtype=np.float32))
    filters = [(5, 1.0, 0.0), (0, 1 - 2.0 ** -24, 0.0), (0, 1.0, 1e-20), (vocab - 1, 0.9999999, 1e-25), (0, 1.0, 0.0)]
    x, at = np.full((4 * len(filters), vocab), 0xFF80, dtype=np.uint16), vocab // 2
    x[:, 0], x[:, -1], x[:, at] = faint, faint, top
    x[1::2, at - 1] = some
    k, p, m = (np.repeat(v, 4) for v in zip(*filters))
    u = np.tile(np.float32([0, 0, 1 - 2.0 ** -24, 1 - 2.0 ** -24]), len(filters))
    # (top-p's front, all but 2^-24 of the weights, is the largest alone)
    return Rows(x, None, k, p, m, u), [t for f in filters[:-1] for t in (at, at if f[1] < 1 else at - 1, at, at)] + [0, 0, at, at]


@pytest.mark.parametrize("vocab", [10, 1000, 4097, 9000, 300001])
def test_tokens_below_a_unit_are_not_drawn_where_a_filter_is_on(vocab):
    """Below 2^-40 of the largest weight, whether the token shares a chunk with heavier ones or not.  Without a filter u = 0 draws it."""
    r, want = faint_tokens(vocab)
    assert r.run()[0].tolist() == want


def faint_tokens_before_any_call():
    for vocab in (1000, 9000, 300001):
        r, want = faint_tokens(vocab)
        s = Stream()
        g = Graph(s, r.call)
        g.launch()
        s.sync()
        assert r.got()[0].tolist() == want, vocab
    print("captured: the same")


def test_tokens_below_a_unit_without_scratch():
    r = subprocess.run([sys.executable, "-c", "import test_gpu_sample as t; t.faint_tokens_before_any_call()"], cwd=HERE,
                       capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "the same" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("step", range(-3, 4))
@pytest.mark.parametrize("top_k", [700, 2500])
def test_zeros_where_the_bins_of_the_least_keys_begin(step, top_k):
    """Logits and temperatures so small that all keys do not fit the bins, 4096 keys and more between the largest and 0, and the
    keys around -0 the first of the bins of the least: borders among zeros of either sign."""
    rng = np.random.default_rng(24)
    vocab = 4000
    x = np.full(vocab, 0x9000, dtype=np.uint16)  # (-2^-95, 0 but for one in 2^44)
    x[10:3000] = np.where(rng.random(2990) < 0.5, 0x8000, 0x0000)
    x[5] = 0x1020
    top, least = bf2f_array(x[5:6])[0].astype(np.float64), 0x0FFD + step
    temp = np.float32((top + bf2f_array(np.uint16([least]))[0] * (1 + 2.0 ** -9)) / 31)
    # zeros weigh e^-17.3 of the largest each, their kept ones (top_k - 1) times that; u is a multiple of 2^-24, two of them
    w = np.exp(-top / np.float64(temp))
    u = np.float32([1 - f * (top_k - 1) * w for f in (0.9, 0.77, 0.6, 0.47, 0.34, 0.2, 0.1, 0.04)] + [0.1])
    b = len(u)
    r = Rows(np.tile(x, (b, 1)), temp, top_k, np.where(np.arange(b) % 4 == 1, 1 - 2.0 ** -24, 1.0), None, u)
    # weights lose less than a unit of 2^-40 each: 2500 of them 2.3e-9, a tenth of a token
    r.compare(r.run(), least=0.5, tol=3e-9)


@pytest.mark.parametrize("vocab", [8192, 33000, 100277])
def test_top_k_behind_min_p_in_flat_rows(vocab):
    """min-p's border beyond the keys counted first, and top-k's further down, or beside it: a sample says which may come first."""
    rng = np.random.default_rng(vocab + 1)
    b = 16
    bits = f2bf_array((rng.standard_normal(b * vocab) * 0.5).astype(np.float32)).reshape(b, vocab)
    min_p = 0.1 + 0.1 * rng.random(b)
    l = np.sort(bf2f_array(bits).reshape(b, vocab), axis=1)[:, ::-1]
    left = (l >= l[:, :1] + np.log(min_p)[:, None]).sum(1)
    assert (left > vocab // 20).all() and (left < vocab - 1500).all()
    top_k = left + np.where(np.arange(b) % 2 == 0, 1500, [-40, -3, -1, 0, 1, 3, 40, 400] * (b // 8))
    r = Rows(bits, None, top_k, None, min_p, rng.random(b))
    # (as of other flat rows: 4e-6 n of the draws are too near)
    r.compare(r.run(), least=0.3, tol=2e-6)
