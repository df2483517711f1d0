"""The ways of the cache's attention and of draft verification that ordinary sizes do not take, on the GPU: sums that fit no
scratch, captures without any, more sequences than a launch holds, and scores' scales of either sign."""
import ctypes
import subprocess
import sys
import os

import numpy as np
import pytest

from _lib import check, Dev, f2bf_array
from _ops import ops, Stream, Graph, page_bytes
from test_gpu_paged_attn import Batch
import test_gpu_spec_verify as sv

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))


def test_more_sums_than_scratch_holds():
    """64 new tokens of 256 heads over 65000 cached ones: their rows have the bits of one-token calls."""
    bits, page, heads, kv, dim, t, n = 4, 256, 256, 16, 64, 64, 65000
    rng = np.random.default_rng(1)
    npages = (n + page - 1) // page
    pool = rng.integers(0, 256, (npages, page_bytes(bits, page, kv, dim)), dtype=np.uint8)
    at = 2 * kv * page * dim // 2  # scales: bf16 between 2^-3 and 2^0
    pool[:, at:at + 4 * kv * page] = (0x3E00 + rng.integers(0, 0x180, (npages, 2 * kv * page))).astype(np.uint16).view(np.uint8)
    q = f2bf_array(0.3 * rng.standard_normal(t * heads * dim).astype(np.float32)).reshape(t, heads * dim)
    P, T = Dev.of(pool), Dev.of(rng.permutation(npages).astype(np.int32))

    def run(q, length):
        m = len(q)
        Q, Y, E = Dev.of(q), Dev(q.nbytes), Dev(m * heads * 4)
        L = Dev.of(np.array([length], dtype=np.int32))
        check(ops().ak_paged_attn(bits, Q.p, m, heads * dim, P.p, npages, page, heads, kv, dim, 1, None, L.p, T.p, npages,
                                  dim ** -0.5, Y.p, heads * dim, E.p, None))
        check(ops().ak_synchronize())
        return Y.get(np.uint16, m * heads * dim).reshape(m, -1), E.get(np.float32, m * heads).reshape(m, heads)
    y, e = run(q, n)
    assert np.isfinite(e).all()
    for i in (0, 30, 63):
        y1, e1 = run(q[i:i + 1], n - t + i + 1)
        assert np.array_equal(y1[0], y[i]) and np.array_equal(e1[0], e[i])


def first_captures():
    """In a process of its own: both operators' first calls are captured, so no scratch is there yet."""
    b = Batch(3, 8, 16, 40, 8, 128, [2500, 20, 700], [2, 1, 3]).device()
    w = 40 * 128
    s = Stream()
    Q, Y, E = Dev.of(b.q), Dev(b.m * w * 2), Dev(b.m * 40 * 4)

    def attend(stream):
        return ops().ak_paged_attn(8, Q.p, b.m, w, b.P.p, b.npages, 16, 40, 8, 128, 3, b.F.p, b.L.p, b.T.p, b.ldt, b.scale,
                                   Y.p, w, E.p, stream)
    rng = np.random.default_rng(4)
    n, t, vocab = 5, 3, 20001
    target, draft = sv.logits(rng, (n, t + 1, vocab)), sv.logits(rng, (n, t, vocab))
    ids = rng.integers(0, vocab, (n, t)).astype(np.int32)
    ids[::2] = draft[::2].view(np.int16).argmax(-1)
    target[0, :t] = draft[0]
    u, temp = rng.random((n, t + 1)).astype(np.float32), np.array([0.7, 0, 1, 1.3, 0], dtype=np.float32)
    T, D, I, U, H = (Dev.of(x) for x in (target, draft, ids, u, temp))
    outs = Dev(4 * n * (t + 1)), Dev(4 * n), Dev(4 * n * (t + 1))
    results = []
    for drafted in (True, False):
        def verify(stream):
            return ops().ak_spec_verify(T.p, vocab, D.p if drafted else None, vocab, I.p, None, U.p, H.p, n, t, vocab,
                                        *(x.p for x in outs), stream)
        g = Graph(s, verify)
        for _ in range(2):
            g.launch()
            s.sync()
            results.append([x.get(np.int32, x.nbytes // 4) for x in outs])
    g = Graph(s, attend)
    for _ in range(2):
        g.launch()
        s.sync()
        results.append([Y.get(np.uint16, b.m * w), E.get(np.int32, b.m * 40)])
    # the same with scratch
    for k, drafted in enumerate((True, False)):
        assert ops().ak_spec_verify(T.p, vocab, D.p if drafted else None, vocab, I.p, None, U.p, H.p, n, t, vocab,
                                    *(x.p for x in outs), None) == 0
        check(ops().ak_synchronize())
        for r in results[2 * k:2 * k + 2]:
            assert all(np.array_equal(a, x.get(np.int32, x.nbytes // 4)) for a, x in zip(r, outs))
    y, e = b.run()
    for r in results[4:]:
        assert np.array_equal(r[0], y.ravel()) and np.array_equal(r[1].view(np.float32), e.ravel())
    print("same bits")


def test_first_calls_captured():
    r = subprocess.run([sys.executable, "-u", "-c", "import test_gpu_serving_paths as t; t.first_captures()"], cwd=HERE,
                       capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "same bits" in r.stdout, r.stdout + r.stderr


def test_more_sequences_than_a_launch_holds():
    rng = np.random.default_rng(5)
    b, t, vocab = 20000, 127, 2
    target, draft = sv.logits(rng, (b, t + 1, vocab)), sv.logits(rng, (b, t, vocab))
    ids = rng.integers(0, vocab, (b, t)).astype(np.int32)
    counts = rng.integers(0, t + 1, b).astype(np.int32)
    u, temp = rng.random((b, t + 1)), rng.random(b) + 0.5
    temp[::3] = 0
    tok, acc, lp = sv.run(target, draft, ids, counts, u, temp, b, t, vocab)
    for a in (0, 9000, 19900):
        s = slice(a, a + 100)
        tok1, acc1, lp1 = sv.run(target[s], draft[s], ids[s], counts[s], u[s], temp[s], 100, t, vocab)
        assert np.array_equal(tok1, tok[s]) and np.array_equal(acc1, acc[s]) and np.array_equal(lp1, lp[s])


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("times", [-1.0, 0.0, 1e-3])
def test_scales(bits, times):
    """A scale of another sign than the usual one, none at all (the mean of the values), and one that is not a power of two."""
    b = Batch(6, bits, 16, 10, 2, 128, [300, 1, 37], [3, 1, 2])
    b.scale *= times
    want = b.want
    b.want = lambda: [np.abs(x) if i == 3 else x for i, x in enumerate(want())]  # (sum |q k| times the scale)
    b.check()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** 60])
def test_queries_of_any_size(bits, size):
    """Queries far from 1 give the scores that the scale makes of them."""
    b = Batch(7, bits, 16, 10, 2, 128, [300, 1, 37], [3, 1, 2])
    y, e = b.device().run()
    b.q = f2bf_array((np.asarray(b.q, dtype=np.uint32) << 16).view(np.float32).ravel() * np.float32(size)).reshape(b.q.shape)
    b.scale /= size
    y2, e2 = b.device().run()
    assert np.array_equal(y, y2) and np.array_equal(e, e2)


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_small_queries_without_a_scale(bits):
    """Scores too small for any number: the mean of the values that a row sees."""
    b = Batch(8, bits, 16, 10, 2, 128, [300, 5], [3, 2])
    b.q = f2bf_array((np.asarray(b.q, dtype=np.uint32) << 16).view(np.float32).ravel() * np.float32(2.0 ** -100)).reshape(b.q.shape)
    b.scale = 0.0
    b.check()
