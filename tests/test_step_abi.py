"""CPU checks of the entry points of a batched step: sizes, refusals before any device call, frequencies on the host."""
import ctypes

import numpy as np
import pytest

from _lib import ptr, f2bf_array
from _step import step, freqs64, plan64, sample64, rope64

P = ctypes.c_void_p(1 << 20)  # an aligned address that no refused call may touch
ODD = ctypes.c_void_p((1 << 20) + 8)
ARR = (ctypes.c_void_p * 4)(1 << 20, 1 << 20, 1 << 20, 1 << 20)
HOLE = (ctypes.c_void_p * 4)(1 << 20, None, 1 << 20, 1 << 20)
CROOKED = (ctypes.c_void_p * 4)(1 << 20, (1 << 20) + 2, 1 << 20, 1 << 20)


def caller(f, **given):
    return lambda **o: f(*[o.get(n, v) for n, v in given.items()])


def test_plan_refusals():
    f = caller(step().ak_kv_plan, b=2, m=8, counts=P, drop=P, cached=P, held=P, free_count=P, free_pages=P, npages=10, page=16,
               table=P, ldt=4, lens=P, held_out=P, free_out=P, qstart=P, pos=P, slots=P, refused=P, stream=None)
    for bad in (dict(b=-1), dict(b=1025), dict(m=-1), dict(m=(1 << 20) + 1), dict(page=8), dict(page=24), dict(page=512),
                dict(npages=0), dict(npages=1 << 27), dict(ldt=0), dict(ldt=1 << 30), dict(counts=None), dict(cached=None),
                dict(held=None), dict(free_count=None), dict(table=None), dict(lens=None), dict(held_out=None),
                dict(free_out=None), dict(qstart=None), dict(pos=None), dict(slots=None), dict(refused=None)):
        assert f(**bad) == 1, bad


def test_rope_refusals():
    K = step()
    f = caller(K.ak_rope, x=P, ldx=1024, y=P, ldy=1024, m=2, heads=8, dim=128, pos=P, freqs=P, rot=128, interleaved=0, mag=1.0,
               stream=None)
    turn = (dict(pos=None), dict(freqs=None), dict(rot=0), dict(rot=3), dict(rot=130), dict(rot=-2), dict(interleaved=2),
            dict(mag=float("nan")), dict(mag=float("inf")))
    for bad in turn + (dict(x=None), dict(y=None), dict(x=ODD), dict(y=ODD), dict(ldx=1020), dict(ldx=-1024), dict(ldy=1016),
                       dict(ldx=2048), dict(m=-1), dict(heads=0), dict(heads=4097), dict(dim=4), dict(dim=100),
                       dict(dim=520)):
        assert f(**bad) == 1, bad
    assert f(m=0, x=None) == 0
    g = caller(K.ak_rope_kv_write, bits=8, q=P, ldq=6144, k=P, ldk=6144, v=P, ldv=6144, y=P, ldy=6144, m=2, heads=32, pos=P,
               freqs=P, rot=128, interleaved=0, mag=1.0, slots=P, pool=P, npages=4, page=16, kv_heads=8, dim=128, stream=None)
    for bad in turn + (dict(bits=3), dict(q=None), dict(k=None), dict(v=None), dict(y=None), dict(slots=None), dict(pool=None),
                       dict(pool=ODD), dict(k=ODD), dict(v=ODD), dict(ldk=4), dict(ldv=-8), dict(ldy=4088), dict(m=-1),
                       dict(heads=0), dict(kv_heads=0), dict(kv_heads=257), dict(dim=96), dict(page=12), dict(npages=0)):
        assert g(**bad) == 1, bad
    assert g(m=0, q=None) == 0


def test_sample_refusals():
    f = caller(step().ak_sample, logits=P, ld=1000, temperature=P, top_k=P, top_p=P, min_p=P, u=P, b=2, vocab=1000, tokens=P,
               logp=P, stream=None)
    for bad in (dict(logits=None), dict(u=None), dict(tokens=None), dict(b=-1), dict(vocab=0), dict(ld=999),
                dict(vocab=(1 << 20) + 1, ld=1 << 21)):
        assert f(**bad) == 1, bad
    assert f(b=0, logits=None) == 0


def test_lora_refusals():
    K = step()
    ns, ld = (ctypes.c_int * 4)(64, 40, 8, 8), (ctypes.c_int * 4)(64, 40, 8, 8)
    f = caller(K.ak_lora_add, plan=P, x=P, m=3, ldx=256, k=256, adapters=2, rank=16, a=P, scale=P, nseg=2, b=ARR, base=ARR,
               y=ARR, n=ns, ldy=ld, stream=None)
    for bad in (dict(plan=None), dict(plan=ODD), dict(x=None), dict(x=ODD), dict(a=None), dict(a=ODD), dict(ldx=252), dict(ldx=-256),
                dict(k=0), dict(k=100), dict(k=(1 << 24) + 8), dict(m=-1), dict(m=(1 << 20) + 1), dict(adapters=0),
                dict(adapters=4097), dict(rank=0), dict(rank=12), dict(rank=136), dict(nseg=0), dict(nseg=5), dict(b=None),
                dict(b=HOLE), dict(b=CROOKED), dict(y=None), dict(y=HOLE), dict(base=HOLE), dict(n=None),
                dict(n=(ctypes.c_int * 4)(64, 0, 8, 8)), dict(ldy=(ctypes.c_int * 4)(64, 39, 8, 8))):
        assert f(**bad) == 1, bad
    assert f(m=0, x=None) == 0
    g = caller(K.ak_lora_plan, ids=P, m=3, adapters=2, plan=P, stream=None)
    for bad in (dict(ids=None), dict(m=-1), dict(m=(1 << 20) + 1), dict(adapters=0), dict(adapters=4097), dict(plan=None),
                dict(plan=ODD)):
        assert g(**bad) == 1, bad
    for bad in ((-1, 2, 16, 256), (3, 0, 16, 256), (3, 4097, 16, 256), (3, 2, 0, 256), (3, 2, 12, 256), (3, 2, 520, 256),
                (3, 2, 16, 0), (3, 2, 16, 100)):
        assert K.ak_lora_plan_bytes(*bad) == 0, bad
    assert K.ak_lora_plan_bytes(3, 2, 16, 256) > 0
    assert K.ak_lora_plan_bytes(1 << 20, 4096, 512, 65536) > 1 << 33  # (counted in 64 bits)


@pytest.mark.parametrize("theta,rot,scaling,factor,trained", [(1e4, 128, 0, 1.0, 0), (1e6, 2, 0, 1.0, 0), (5e5, 64, 1, 4.0, 0),
                                                              (1e4, 96, 2, 8.0, 0), (1e6, 128, 3, 4.0, 32768),
                                                              (1e4, 30, 3, 1.0, 4096)])
def test_rope_freqs(theta, rot, scaling, factor, trained):
    f, mag = np.zeros(rot // 2), ctypes.c_float(0)
    assert step().ak_rope_freqs(theta, rot, scaling, factor, trained, 1.0, 32.0, ptr(f), ctypes.byref(mag)) == 0
    want, wmag = freqs64(theta, rot, scaling, factor, trained)
    assert np.abs(f / want - 1).max() < 2.0 ** -46 and abs(mag.value - wmag) < 1e-6  # (pow of 64 bits, a few of its steps)


def test_rope_freqs_refusals():
    K, f, mag = step(), np.zeros(64), ctypes.c_float(0)
    g = caller(K.ak_rope_freqs, theta=1e4, rot=128, scaling=3, factor=2.0, trained=4096, slow=1.0, fast=32.0, freqs=ptr(f),
               mag=ctypes.byref(mag))
    for bad in (dict(theta=0.0), dict(theta=float("nan")), dict(theta=float("inf")), dict(rot=0), dict(rot=5), dict(scaling=-1),
                dict(scaling=4), dict(factor=0.5), dict(factor=float("nan")), dict(factor=float("inf")), dict(trained=0),
                dict(slow=-1.0), dict(fast=1.0), dict(fast=float("inf")), dict(freqs=None), dict(mag=None),
                dict(scaling=2, rot=2)):
        assert g(**bad) == 1, bad


# ------------------------------------------------------------------------------------------------ the oracles themselves
def test_plan_oracle():
    table = np.array([[7, 3, -1], [5, -1, -1], [9, 8, -1]], dtype=np.int32)
    free = np.array([0, 1, 2, -1, -1, -1, -1, -1, -1, -1], dtype=np.int32)
    r = plan64([1, 18, 0], [0, 0, 1], [32, 14, 20], [2, 1, 2], table, free, 3, 16, 10, 24)
    # row 2 gives 9 and 8 back; the pages taken are the last ones: 8, then 9
    assert r["table"].tolist() == [[7, 3, 8], [5, 9, -1], [9, 8, -1]] and r["nfree"][0] == 3
    assert r["lens"].tolist() == [33, 32, 0] and r["held"].tolist() == [3, 2, 0] and r["refused"].tolist() == [0, 0, 0]
    assert r["slots"][:4].tolist() == [128, 94, 95, 144] and r["pos"][19:].tolist() == [-1] * 5


def test_sample_oracle():
    bits = f2bf_array(np.log(np.array([0.1, 0.4, 0.1, 0.4], dtype=np.float32)))
    pick = lambda u, k=0, p=1.0, m=0.0: sample64(bits, 1.0, k, p, m, u)[0]  # noqa: E731
    assert [pick(u) for u in (0.05, 0.3, 0.55, 0.9)] == [0, 1, 2, 3]
    assert [pick(u, k=1) for u in (0.0, 0.99)] == [1, 1] and [pick(u, k=3) for u in (0.05, 0.3, 0.9)] == [0, 1, 3]
    assert [pick(u, p=0.3) for u in (0.0, 0.99)] == [1, 1] and pick(0.9, p=0.79) == 3
    assert [pick(u, m=0.5) for u in (0.05, 0.9)] == [1, 3]


def test_rope_oracle_of_a_quarter_turn():
    x = f2bf_array(np.array([1, 2, 3, 4], dtype=np.float32)).reshape(1, 1, 4)
    f = [np.pi / 2, np.pi]
    assert np.allclose(rope64(x, [1], f, 4, 0, 1.0)[0, 0], [-3, -2, 1, -4]) and \
        np.allclose(rope64(x, [1], f, 4, 1, 2.0)[0, 0], [-4, 2, -6, -8])
