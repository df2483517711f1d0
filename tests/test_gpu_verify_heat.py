"""Verification of drafts at temperatures of every size, on the GPU, against 64 bits.

Tolerances: tokens and counts as in test_gpu_spec_verify; a log probability that the definition puts above -50 within 1e-5 of
1 + |log p|, since the weights that count are fp32's exp2 of exponents above -150 (150 * 2^-24 of the exponent's rounding)."""
import numpy as np
import pytest

from _lib import f2bf_array, bf2f_array
from _ops import verify64
from test_gpu_spec_verify import logits, run, compare

pytestmark = pytest.mark.gpu

COLD = [1e-38, 3e-37, 1e-36, 1e-33, 1e-30, 1e-25, 1e-20, 1e-12, 1e-11, 1e-10, 1e-9, 1e-8, 4e-8]  # below 2^-24 / log2(e)
ORDINARY = [1e-7, 1e-6, 1e-4, 1e-3, 0.02, 0.05, 0.1, 0.2, 0.3, 0.45]


def rounding(temp):
    """What fp32 loses of log2(e) / T."""
    scale = 1.44269504088896340736 / float(np.float32(temp))
    return scale - float(np.float32(scale))


def test_temperatures_cover_both_roundings():
    signs = [rounding(t) < 0 for t in COLD if abs(rounding(t)) > 1]
    assert any(signs) and not all(signs)


def scene(vocab, temps, seed, masks):
    rng = np.random.default_rng(seed)
    b, t = len(temps), 2
    target = logits(rng, (b, t + 1, vocab), peaks=min(8, vocab))
    if masks:
        target[:, :, ::5] = 0xFF80  # -inf
        target[:, :, 1::10] = 0x7FC0  # NaN
        target[:, :, 2::10] = 0xFF7F  # the type's lowest value
        target[:, :, 3::20] = f2bf_array(np.array([-1e30], dtype=np.float32))[0]
    best = np.where(np.isfinite(bf2f_array(target)), bf2f_array(target), -np.inf).argmax(-1)
    ids = best[:, :t].copy()
    ids[::2, 1] = rng.integers(0, vocab, len(ids[::2]))  # every other one's second draft is any token
    draft = f2bf_array((bf2f_array(target[:, :t]) + 0.25 * rng.standard_normal((b, t, vocab)).astype(np.float32)).ravel())
    draft = draft.reshape(b, t, vocab)
    return target, draft, ids, rng.random((b, t + 1)) * 0.99, np.array(temps), b, t


@pytest.mark.parametrize("masks", [False, True])
@pytest.mark.parametrize("vocab", [300, 4096, 8193, 100277])
@pytest.mark.parametrize("drafted", [True, False])
def test_cold(vocab, drafted, masks):
    """Nothing weighs anything but the largest logits: what is emitted is greedy's, with log probabilities to match."""
    target, draft, ids, u, temp, b, t = scene(vocab, COLD, 5, masks)
    got = run(target, draft if drafted else None, ids, None, u, temp, b, t, vocab)
    with np.errstate(over="ignore"):
        for i in range(b):
            tok, acc, lp, near = verify64(target[i], draft[i] if drafted else None, ids[i], t, np.float32(u[i]),
                                          float(np.float32(temp[i])), t)
            assert not near
            assert got[1][i] == acc and np.array_equal(got[0][i], tok), temp[i]
            assert (np.abs(got[2][i] - lp) <= 1e-5).all(), temp[i]


@pytest.mark.parametrize("masks", [False, True])
@pytest.mark.parametrize("vocab", [300, 8193])
@pytest.mark.parametrize("drafted", [True, False])
def test_low(vocab, drafted, masks):
    target, draft, ids, u, temp, b, t = scene(vocab, ORDINARY, 6, masks)
    args = (target, draft if drafted else None, ids, None, u, temp, b, t)
    got = run(*args[:6], b, t, vocab)
    compare(got, *args, least=0.8)
    for i in range(b):
        tok, acc, lp, near = verify64(target[i], args[1][i] if drafted else None, ids[i], t, np.float32(u[i]),
                                      float(np.float32(temp[i])), t)
        if not near:
            assert (np.abs(got[2][i] - lp) <= 1e-5 * (1 + np.abs(lp)))[lp > -50].all(), temp[i]


def test_small_logits_and_a_small_temperature():
    """The weights are those of (l - largest) / T, however small both are."""
    rng = np.random.default_rng(7)
    b, t, vocab = 8, 0, 1000
    size = np.array([1e-3, 1e-8, 1e-10, 1e-12, 1e-20, 1e-28, 1e-33, 1e-36])
    target = f2bf_array((2.0 * rng.standard_normal((b, 1, vocab)) * size[:, None, None]).astype(np.float32).ravel())
    args = (target.reshape(b, 1, vocab), None, None, None, rng.random((b, 1)), size, b, t)
    compare(run(*args[:6], b, t, vocab), *args, least=0.8)


@pytest.mark.parametrize("drafted", [True, False])
def test_a_large_temperature(drafted):
    """Every token weighs nearly the same, masked ones nothing."""
    target, draft, ids, u, temp, b, t = scene(300, [10.0, 1e3, 1e10, 1e20], 8, False)
    target[:, :, ::3] = 0xFF80
    args = (target, draft if drafted else None, ids, None, u, temp, b, t)
    got = run(*args[:6], b, t, 300)
    compare(got, *args, least=0.7)
    assert not np.isin(got[0], np.arange(0, 300, 3)).any()
