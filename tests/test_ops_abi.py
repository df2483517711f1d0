"""CPU checks of the cache, attention and verification entry points: sizes and refusals, before any device call."""
import ctypes

import numpy as np
import pytest

from _ops import ops, page_bytes, quantise, held, bf16_rn, verify64, attention64
from _lib import f2bf_array, bf2f_array

P = ctypes.c_void_p(1 << 20)  # an aligned address that no refused call may touch
ODD = ctypes.c_void_p((1 << 20) + 8)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("page,heads,dim", [(16, 1, 64), (32, 8, 128), (256, 3, 256), (64, 256, 128)])
def test_page_bytes(bits, page, heads, dim):
    assert ops().ak_kv_page_bytes(bits, page, heads, dim) == page_bytes(bits, page, heads, dim)


BAD_SHAPES = [(3, 16, 8, 128), (16, 8, 8, 128), (16, 24, 8, 128), (16, 512, 8, 128), (16, 16, 0, 128), (16, 16, 257, 128),
              (16, 16, 8, 96), (16, 16, 8, 0), (0, 16, 8, 128), (16, -16, 8, 128)]


@pytest.mark.parametrize("bits,page,heads,dim", BAD_SHAPES)
def test_bad_shapes_are_refused(bits, page, heads, dim):
    K = ops()
    assert K.ak_kv_page_bytes(bits, page, heads, dim) == 0
    assert K.ak_kv_write(bits, P, P, 1, 4096, 4096, P, P, 4, page, heads, dim, None) == 1
    assert K.ak_kv_read(bits, P, 4, page, heads, dim, P, 1, P, P, 4096, 4096, None) == 1
    assert K.ak_paged_attn(bits, P, 1, 8192, P, 4, page, heads, heads, dim, 1, None, P, P, 4, 1.0, P, 8192, None, None) == 1


def test_cache_refusals():
    K = ops()
    w = lambda **o: K.ak_kv_write(*[o.get(n, v) for n, v in dict(  # noqa: E731
        bits=8, k=P, v=P, m=2, ldk=1024, ldv=1024, slots=P, pool=P, npages=4, page=16, heads=8, dim=128, stream=None).items()])
    r = lambda **o: K.ak_kv_read(*[o.get(n, v) for n, v in dict(  # noqa: E731
        bits=8, pool=P, npages=4, page=16, heads=8, dim=128, slots=P, m=2, k=P, v=P, ldk=1024, ldv=1024,
        stream=None).items()])
    for f in (w, r):
        for bad in (dict(k=None), dict(v=None), dict(slots=None), dict(pool=None), dict(k=ODD), dict(v=ODD), dict(pool=ODD),
                    dict(ldk=1020), dict(ldv=1028), dict(ldk=-1024), dict(m=-1), dict(npages=0)):
            assert f(**bad) == 1, bad
        assert f(m=0, k=None, v=None) == 0
    assert r(ldk=1016) == 1  # the rows written would overlap


def test_attention_refusals():
    K = ops()
    f = lambda **o: K.ak_paged_attn(*[o.get(n, v) for n, v in dict(  # noqa: E731
        bits=8, q=P, m=4, ldq=5120, pool=P, npages=4, page=16, heads=40, kv_heads=8, dim=128, b=2, qstart=None, lens=P,
        table=P, ldt=3, scale=0.1, y=P, ldy=5120, lse=None, stream=None).items()])
    for bad in (dict(q=None), dict(pool=None), dict(lens=None), dict(table=None), dict(y=None), dict(q=ODD), dict(y=ODD),
                dict(pool=ODD), dict(heads=12), dict(heads=0), dict(ldq=5124), dict(ldy=5124), dict(ldy=5112), dict(ldq=-8),
                dict(m=-1), dict(m=3), dict(b=0), dict(b=-1), dict(b=4097, m=4097), dict(ldt=0), dict(npages=0),
                dict(scale=float("nan")), dict(scale=float("inf"))):
        assert f(**bad) == 1, bad
    assert f(m=0, q=None, y=None) == 0
    assert f(m=0, b=0, q=None, y=None, lens=None, table=None) == 0


def test_verify_refusals():
    K = ops()
    f = lambda **o: K.ak_spec_verify(*[o.get(n, v) for n, v in dict(  # noqa: E731
        target=P, ldt=1000, draft=P, ldd=1000, ids=P, counts=P, u=P, temp=P, b=2, t=3, vocab=1000, tokens=P, accepted=P,
        logp=P, stream=None).items()])
    for bad in (dict(target=None), dict(ids=None), dict(u=None), dict(tokens=None), dict(accepted=None), dict(b=-1),
                dict(t=-1), dict(t=128), dict(vocab=0), dict(ldt=999), dict(ldd=999)):
        assert f(**bad) == 1, bad
    assert f(b=0, target=None) == 0


def test_limits():
    K = ops()
    assert K.ak_spec_verify(P, 1 << 21, None, 0, None, None, P, None, 1, 0, (1 << 20) + 1, P, P, None, None) == 1
    # 1025 sequences; rows of 256 heads whose numbers do not divide exactly
    assert K.ak_paged_attn(8, P, 1025, 128, P, 4, 16, 1, 1, 128, 1025, None, P, P, 1, 1.0, P, 128, None, None) == 1
    assert K.ak_paged_attn(8, P, 65536, 32768, P, 4, 16, 256, 1, 128, 1, None, P, P, 1, 1.0, P, 32768, None, None) == 1


# ------------------------------------------------------------------------------------------------ the oracle itself
def test_quantise_definition():
    x = f2bf_array(np.array([[127.0, 2.5, 3.5, -0.5] + [0.0] * 4, [7.0, 1.0, -3.0, 0.25] + [0.0] * 4], dtype=np.float32))
    c, s = quantise(x[:1], 8)
    assert bf2f_array(s)[0] == 1.0 and list(c[0, :4].astype(int) - 128) == [127, 2, 4, 0]  # halves to even
    c, s = quantise(x[1:], 4)
    assert bf2f_array(s)[0] == 1.0 and list(c[0, :4].astype(int) - 8) == [7, 1, -3, 0]
    tiny = np.array([[0x0001] * 8], dtype=np.uint16)
    assert (held(tiny, 8) == 0).all()
    bad = f2bf_array(np.ones((1, 8), dtype=np.float32))
    bad[0, 3] = 0x7F80
    assert np.isnan(held(bad, 4)).all()
    assert bf16_rn(1 + 2.0 ** -8) == 0x3F80 and bf16_rn(1 + 2.0 ** -8 + 2.0 ** -40) == 0x3F81


def test_attention_oracle_of_one_key():
    rng = np.random.default_rng(0)
    q = f2bf_array(rng.standard_normal((1, 2, 64)).astype(np.float32))
    k, v = rng.standard_normal((1, 1, 64)), rng.standard_normal((1, 1, 64))
    y, lse, _, _ = attention64(q, [(0, 1, k, v, np.array([True]))], 2, 1, 64, 0.5)
    assert np.allclose(y[0], v[0]) and np.allclose(lse[0], bf2f_array(q)[0].astype(np.float64) @ k[0, 0] * 0.5)


def test_verify_oracle_emits_the_targets_distribution():
    """Speculative sampling leaves the target's distribution unchanged: over a grid of uniform numbers the first token's
    frequencies are p, whatever the draft."""
    target = f2bf_array(np.log(np.array([[0.5, 0.25, 0.15, 0.1]] * 2, dtype=np.float32)))
    draft = f2bf_array(np.log(np.array([[0.1, 0.2, 0.3, 0.4]], dtype=np.float32)))
    p, q = softmax64_pair(target[0]), softmax64_pair(draft[0])
    hits, grid = np.zeros(4), (np.arange(60) + 0.5) / 60
    for x in range(4):  # a draft x occurs with probability q[x]
        for a in grid:
            for b in grid:
                hits[verify64(target, draft, [x], 1, [a, b], 1.0, 1)[0][0]] += q[x] / len(grid) ** 2
    assert np.abs(hits - p).max() < 0.01


def softmax64_pair(bits):
    e = np.exp(bf2f_array(bits).astype(np.float64))
    return e / e.sum()
