"""Verification of drafts (ak_spec_verify) on the GPU, against 64 bits (numpy, test infrastructure).

Tokens and counts are compared exactly except where a decision of the 64-bit evaluation lies within 1e-5 of its threshold;
the log probabilities within 2^-20 of 1 + |log p| per unit of (largest logit difference / temperature): a logit difference
is exact in fp32, its quotient and exponential are rounded."""
import ctypes

import numpy as np
import pytest

from _lib import check, Dev, f2bf_array, bf2f_array
from _ops import ops, verify64, Stream, Graph

pytestmark = pytest.mark.gpu


def logits(rng, shape, spread=2.0, peaks=8):
    x = rng.standard_normal(shape) * spread
    v = shape[-1]
    flat = x.reshape(-1, v)
    for r in flat:
        r[rng.integers(0, v, peaks)] += 6 + 6 * rng.random(peaks)
    return f2bf_array(x.astype(np.float32).ravel()).reshape(shape)


def run(target, draft, ids, counts, u, temp, b, t, vocab, pad=0, stream=None, logp=True):
    def rows(x, n):
        out = np.full((b, n, vocab + pad), 0x7F7F, dtype=np.uint16)  # between the rows: never to be chosen
        out[..., :vocab] = x
        return Dev.of(out)
    T = rows(target, t + 1)
    D = rows(draft, t) if draft is not None else None
    I = Dev.of(np.asarray(ids, dtype=np.int32)) if t else None
    C = Dev.of(np.asarray(counts, dtype=np.int32)) if counts is not None else None
    U, H = Dev.of(np.asarray(u, dtype=np.float32)), Dev.of(np.asarray(temp, dtype=np.float32)) if temp is not None else None
    tok, acc, lp = Dev.of(np.full(b * (t + 1), 99, dtype=np.int32)), Dev(4 * b), Dev(4 * b * (t + 1))
    check(ops().ak_spec_verify(T.p, vocab + pad, D.p if D else None, vocab + pad, I.p if I else None, C.p if C else None,
                               U.p, H.p if H else None, b, t, vocab, tok.p, acc.p, lp.p if logp else None, stream))
    check(ops().ak_synchronize())
    return (tok.get(np.int32, b * (t + 1)).reshape(b, t + 1), acc.get(np.int32, b),
            lp.get(np.float32, b * (t + 1)).reshape(b, t + 1))


def compare(got, target, draft, ids, counts, u, temp, b, t, least=0.9):
    tok, acc, lp = got
    sure = 0
    for i in range(b):
        heat = 1.0 if temp is None else float(np.float32(temp[i]))
        n = t if counts is None else int(counts[i])
        wt, wa, wl, near = verify64(target[i], None if draft is None else draft[i], ids[i] if t else [], n,
                                    np.asarray(u[i], dtype=np.float32), heat, t)
        if near:
            continue
        sure += 1
        assert acc[i] == wa and np.array_equal(tok[i], wt), (i, tok[i], wt)
        l = bf2f_array(target[i]).astype(np.float64)
        spread = np.ptp(l[np.isfinite(l)]) / (heat if heat > 0 else 1.0) if np.isfinite(l).any() else 0.0
        assert (np.abs(lp[i] - wl) <= 2.0 ** -20 * (1 + np.abs(wl)) * (1 + spread)).all()
    assert sure >= int(least * b)


@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 1000, 1003, 4099, 33000, 152064])
@pytest.mark.parametrize("t,drafted", [(0, False), (1, True), (4, True), (3, False), (8, True)])
def test_against_64_bits(vocab, t, drafted):
    rng = np.random.default_rng(vocab * 10 + t)
    b = 3 if vocab > 20000 else 12
    target = logits(rng, (b, t + 1, vocab), peaks=min(8, vocab))
    near = bf2f_array(target[:, :t]) + 0.5 * rng.standard_normal((b, t, vocab)).astype(np.float32)
    draft = f2bf_array(near.ravel()).reshape(b, t, vocab)
    temp = 0.5 + 0.7 * rng.random(b)
    temp[::3] = 0.0
    noise = rng.gumbel(size=(b, t, vocab))
    ids = (bf2f_array(draft) / np.maximum(temp, 0.05)[:, None, None] + noise).argmax(-1)
    counts = rng.integers(0, t + 1, b)
    counts[:2] = t
    u = rng.random((b, t + 1))
    args = (target, draft if drafted else None, ids, counts, u, temp, b, t)
    compare(run(*args[:6], b, t, vocab, pad=vocab % 5), *args, least=0.7)


def test_all_accepted_and_first_rejected():
    """A draft model equal to the target is always accepted; one that is certain of an impossible token never."""
    rng = np.random.default_rng(3)
    b, t, vocab = 6, 5, 500
    target = logits(rng, (b, t + 1, vocab))
    ids = rng.integers(0, vocab, (b, t))
    u = rng.random((b, t + 1))
    u[0, :t] = np.nextafter(np.float32(1), np.float32(0))
    tok, acc, _ = run(target, target[:, :t], ids, None, u, None, b, t, vocab)
    assert (acc == t).all() and np.array_equal(tok[:, :t], ids)
    target[np.arange(b), 0, ids[:, 0]] = 0xFF80
    args = (target, None, ids, None, u, None, b, t)
    got = run(*args[:6], b, t, vocab)
    assert (got[1] == 0).all() and (got[0][:, 1:] == -1).all()
    compare(got, *args)


def test_greedy_ties_take_the_lowest_token():
    b, t, vocab = 4, 2, 5000
    target = f2bf_array(np.zeros(b * (t + 1) * vocab, dtype=np.float32)).reshape(b, t + 1, vocab)
    top = f2bf_array(np.array([3.0], dtype=np.float32))[0]
    for j, places in enumerate(([4097, 4096, 70], [4999, 17], [0, 4999])):
        target[:, j, places] = top
    ids = np.array([[70, 17], [70, 4999], [4096, 17], [-1, 17]])
    tok, acc, lp = run(target, None, ids, None, np.full((b, t + 1), 0.5), np.array([0.0, -1.0, 0.0, 0.0]), b, t, vocab)
    assert list(acc) == [2, 1, 0, 0]
    assert tok.tolist() == [[70, 17, 0], [70, 17, -1], [70, -1, -1], [70, -1, -1]]
    assert np.allclose(lp[0, 0], 3 - np.log(3 * np.exp(3) + vocab - 3), atol=1e-4)


def test_uniform_numbers_at_their_ends():
    """u = 0 takes the first token with any weight, u just below 1 the last one."""
    vocab = 5000
    target = np.full((2, 1, vocab), 0xFF80, dtype=np.uint16)
    target[:, 0, [33, 2000, 4990]] = f2bf_array(np.array([1.0, -3.0, -9.0], dtype=np.float32))
    u = np.array([[0.0], [np.nextafter(np.float32(1), np.float32(0))]])
    tok, acc, lp = run(target, None, None, None, u, None, 2, 0, vocab)
    assert tok.ravel().tolist() == [33, 4990] and (acc == 0).all()


@pytest.mark.parametrize("temp", [0.0, 1.0])
def test_masked_and_non_finite_logits(temp):
    """NaN counts as -inf, a row of +inf shares its weight among them, a row of nothing emits -1."""
    vocab, t, b = 300, 1, 7
    rng = np.random.default_rng(4)
    target = logits(rng, (b, t + 1, vocab))
    target[0, 0] = 0x7FC0
    target[1, 0] = 0xFF80
    target[2, 0, 100:] = 0xFFC0
    target[2, 0, :99] = 0xFF7F  # the type's lowest value, but for one token
    target[3, 0, [5, 9]] = 0x7F80
    target[4, 1] = 0xFF80
    target[5, 0] = 0xFF7F  # nothing but the lowest value: uniform
    target[6, 0, ::2] = 0x7FC1
    ids = np.array([[3], [3], [99], [9], [int(bf2f_array(target[4, 0]).argmax())], [7], [2]])
    u = np.array([[.5, .5], [.5, .5], [.5, .5], [.7, .3], [0., .5], [.5, .25], [.5, .5]])
    temps = np.full(b, temp)
    args = (target, None, ids, None, u, temps, b, t)
    got = run(*args[:6], b, t, vocab)
    assert got[0][0].tolist() == [-1, -1] and got[0][1].tolist() == [-1, -1]
    assert got[0][2, 0] == 99 and got[0][4].tolist() == [int(ids[4, 0]), -1]
    compare(got, *args)


def test_drafts_out_of_range_and_counts():
    rng = np.random.default_rng(6)
    b, t, vocab = 6, 3, 700
    target = logits(rng, (b, t + 1, vocab))
    draft = logits(rng, (b, t, vocab))
    ids = rng.integers(0, vocab, (b, t))
    ids[0, 0], ids[1, 0] = -3, vocab
    counts = np.array([3, 3, -2, 9, 0, 1])
    u = rng.random((b, t + 1))
    for d in (draft, None):
        args = (target, d, ids, counts, u, np.full(b, 0.8), b, t)
        compare(run(*args[:6], b, t, vocab), *args, least=0.6)


def test_emits_the_targets_distribution():
    """20000 sequences of one draft drawn from q: the first token's frequencies are p within 5 standard deviations."""
    rng = np.random.default_rng(7)
    b, t, vocab = 20000, 1, 12
    lp, lq = (f2bf_array((rng.standard_normal(vocab) * 1.5).astype(np.float32)) for _ in range(2))
    p, q = (np.exp(bf2f_array(x).astype(np.float64)) for x in (lp, lq))
    p, q = p / p.sum(), q / q.sum()
    ids = rng.choice(vocab, size=(b, t), p=q)
    target, draft = np.broadcast_to(lp, (b, t + 1, vocab)), np.broadcast_to(lq, (b, t, vocab))
    tok, acc, _ = run(target, draft, ids, None, rng.random((b, t + 1)), None, b, t, vocab, logp=False)
    freq = np.bincount(tok[:, 0], minlength=vocab) / b
    assert (np.abs(freq - p) <= 5 * np.sqrt(p * (1 - p) / b)).all()
    assert abs(acc.mean() - np.minimum(p, q).sum()) < 5 * 0.5 / b ** 0.5


def test_rows_do_not_depend_on_the_batch():
    rng = np.random.default_rng(8)
    b, t, vocab = 40, 4, 30011
    target = logits(rng, (b, t + 1, vocab))
    draft = f2bf_array((bf2f_array(target[:, :t]) + 0.3).ravel()).reshape(b, t, vocab)
    ids = (bf2f_array(draft) + rng.gumbel(size=draft.shape)).argmax(-1)
    u, temp = rng.random((b, t + 1)), 0.5 + rng.random(b)
    tok, acc, lp = run(target, draft, ids, None, u, temp, b, t, vocab)
    for i in (0, 17, 39):
        s = slice(i, i + 1)
        tok1, acc1, lp1 = run(target[s], draft[s], ids[s], None, u[s], temp[s], 1, t, vocab)
        assert np.array_equal(tok1[0], tok[i]) and acc1[0] == acc[i] and np.array_equal(lp1[0], lp[i])


def test_graph_replays():
    rng = np.random.default_rng(9)
    b, t, vocab = 3, 3, 20001
    T, D = Dev.of(logits(rng, (b, t + 1, vocab))), Dev.of(logits(rng, (b, t, vocab)))
    I = Dev.of(rng.integers(0, vocab, (b, t)).astype(np.int32))
    U, H = Dev(4 * b * (t + 1)), Dev.of(np.array([0.7, 0.0, 1.0], dtype=np.float32))
    outs = tok, acc, lp = Dev(4 * b * (t + 1)), Dev(4 * b), Dev(4 * b * (t + 1))
    s = Stream()

    def call(stream):
        return ops().ak_spec_verify(T.p, vocab, D.p, vocab, I.p, None, U.p, H.p, b, t, vocab, tok.p, acc.p, lp.p, stream)

    def put(dev, arr):
        check(ops().ak_memcpy_h2d(dev.p, ctypes.c_void_p(arr.ctypes.data), arr.nbytes))

    def take():
        s.sync()
        out = [x.get(np.int32, x.nbytes // 4) for x in outs]
        for x in outs:
            put(x, np.full(x.nbytes // 4, 99, dtype=np.int32))
        return out
    put(U, rng.random((b, t + 1)).astype(np.float32))
    assert call(s.h) == 0
    take()
    g = Graph(s, call)
    for step in range(4):
        put(U, rng.random((b, t + 1)).astype(np.float32))
        put(T, logits(rng, (b, t + 1, vocab)))
        g.launch()
        got = take()
        assert call(s.h) == 0
        assert all(np.array_equal(x, y) for x, y in zip(got, take()))


def test_no_sequences():
    assert ops().ak_spec_verify(None, 8, None, 8, None, None, None, None, 0, 0, 8, None, None, None, None) == 0
