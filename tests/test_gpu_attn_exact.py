"""Attention over the paged cache (ak_paged_attn) on the GPU against 64 bits, under _attn's tolerance: each key's own error by its
share of the row.  Small queries make every token weigh the same, so that a lost one shows in lse and the outputs."""
import os
import subprocess
import sys

import numpy as np
import pytest

from _attn import Scene, bf16
from _lib import check, Dev, bf2f_array
from _ops import ops, Stream, Graph

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))
SHAPES = [(16, 10, 2, 128), (32, 5, 1, 128), (64, 4, 4, 64), (16, 6, 2, 256), (256, 16, 1, 64)]


@pytest.mark.parametrize("sharp", [0.02, 1.0])
@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("page,heads,kv,dim", SHAPES)
def test_one_token_each(bits, page, heads, kv, dim, sharp):
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, page + 1, 300, 511, 513, 700]
    Scene(bits + page, bits, page, heads, kv, dim, lens, [1] * len(lens), sharp).check(ragged=False)


@pytest.mark.parametrize("sharp", [0.02, 1.0])
@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_contexts_around_blocks(bits, dim, sharp):
    lens = [1023, 1024, 1025, 2047, 2048, 3000, 4097, 5003]
    Scene(3, bits, 32, 5, 1, dim, lens, [1] * len(lens), sharp).check(ragged=False)


@pytest.mark.parametrize("bits,dim", [(16, 64), (16, 128), (8, 64), (8, 128), (8, 256), (4, 64), (4, 128)])
def test_contexts_around_groups_of_blocks(bits, dim):
    """Groups of 16 blocks: two and three of them, alone and in a batch."""
    lens = [16383, 16385, 35000, 32768]
    Scene(4, bits, 64, 2, 1, dim, lens, [1] * 4, 0.02).check(ragged=False)
    Scene(5, bits, 64, 2, 1, dim, [17001], [2], 0.02).check(ragged=False)


@pytest.mark.parametrize("sharp", [0.02, 1.0])
@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("page,heads,kv,dim", SHAPES[:4])
def test_drafts(bits, page, heads, kv, dim, sharp):
    lens, counts = [8, 70, 513, 5, 0, 1030, 40, 9], [8, 1, 7, 9, 3, 16, 0, 2]
    Scene(11 + bits, bits, page, heads, kv, dim, lens, counts, sharp).check()


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompts(bits, dim):
    Scene(2, bits, 16, 4, 2, dim, [200, 1300, 333], [200, 150, 333], 0.5).check()


def first_captures():
    """In a process of its own: nothing has scratch yet, so a wave takes a sequence's head.  All nine kernels, with a NaN in a
    late draft's key and value (unseen by the earlier ones) and a page that is not there."""
    s = Stream()
    graphs = []
    for bits in (16, 8, 4):
        for dim in (64, 128, 256):
            a = Scene(31, bits, 32, 6, 2, dim, [2500, 20, 700, 17500], [2, 1, 5, 1], 0.02)
            for x in (a.k[2], a.v[2]):
                x[698, :, 3:5] = 0x7FC0
                x[699, :, 9] = 0xFF80
            a.fill()
            a.table[0, 3], a.present[0][96:128] = -1, False
            a.device()
            w = 6 * dim
            Q, Y, E = Dev.of(a.q), Dev(a.m * w * 2), Dev(a.m * 6 * 4)

            def call(stream, a=a, w=w, Q=Q, Y=Y, E=E):
                return ops().ak_paged_attn(a.bits, Q.p, a.m, w, a.P.p, a.npages, 32, 6, 2, a.dim, 4, a.F.p, a.L.p, a.T.p,
                                           a.ldt, a.scale, Y.p, w, E.p, stream)
            graphs.append((a, Graph(s, call), Q, Y, E))
    kept = []
    for a, g, Q, Y, E in graphs:
        for _ in range(2):
            g.launch()
            s.sync()
            y = Y.get(np.uint16, a.m * 6 * a.dim).reshape(a.m, 6, a.dim)
            e = E.get(np.float32, a.m * 6).reshape(a.m, 6)
            a.x = a.k[2], a.v[2]
            clean = [0, 1, 2, 3, 4, 5, 8]  # rows 6 and 7 see the NaN
            for x in a.x:
                x[698:] = 0
            a.compare(y, e, clean)
            assert not np.isfinite(bf2f_array(y[6:8])).all()
        kept.append((y, e))
    for (a, *_), (y, e) in zip(graphs, kept):  # the same bits with scratch
        y2, e2 = a.run()
        rows = [0, 1, 2, 3, 4, 5, 8]
        assert np.array_equal(y[rows], y2[rows]) and np.array_equal(e[rows], e2[rows])
        assert np.array_equal(np.isnan(bf2f_array(y)), np.isnan(bf2f_array(y2)))
    print("all forms")


def test_a_wave_for_a_head():
    r = subprocess.run([sys.executable, "-u", "-c", "import test_gpu_attn_exact as t; t.first_captures()"], cwd=HERE,
                       capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "all forms" in r.stdout, r.stdout + r.stderr


def test_many_items_a_wave():
    """1024 sequences of 256 heads with room for long contexts: more work items than a wave's table holds at once."""
    a = Scene(6, 4, 16, 256, 256, 64, [40], [1], 0.5)
    b, w = 1024, 256 * 64
    lens = np.arange(b, dtype=np.int32) * 7 % 41
    table = np.full((b, 70), -1, dtype=np.int32)
    table[:, :3] = a.table[0, :3]
    a.device()
    rng = np.random.default_rng(7)
    q = bf16(rng.standard_normal((b, w), dtype=np.float32) * 0.5)
    Q, Y, E, L, T = Dev.of(q), Dev(b * w * 2), Dev(b * 256 * 4), Dev.of(lens), Dev.of(table)

    def call(first, n):
        check(ops().ak_paged_attn(4, Q.addr(2 * w * first), n, w, a.P.p, a.npages, 16, 256, 256, 64, n, None, L.addr(4 * first),
                                  T.addr(4 * 70 * first), 70, a.scale, Y.addr(2 * w * first), w, E.addr(4 * 256 * first), None))
        check(ops().ak_synchronize())
        return Y.get(np.uint16, b * w).reshape(b, w), E.get(np.float32, b * 256).reshape(b, 256)
    y, e = call(0, b)
    for i in range(0, b, 64):
        y2, e2 = call(i, 64)
    assert np.array_equal(y, y2) and np.array_equal(e, e2)
    for i in (0, 1, 500, 1023):
        a.lens, a.q = [int(lens[i])], q[i:i + 1].reshape(1, 256, 64)
        a.compare(y[i:i + 1].reshape(1, 256, 64), e[i:i + 1])


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("n", [600, 4096])
def test_tail_behind_one_heavy_token(bits, n):
    """One token has nearly all the weight, and zeros in half of its values: there the others' sum is the result."""
    a = Scene(8, bits, 32, 1, 1, 128, [n], [1], 1.0)
    q = bf2f_array(a.q)[0, 0].astype(np.float64)
    a.k[0][5, 0] = bf16(q * (21.0 / (a.scale * (q @ q))))  # some 2^-30 for each of the others
    a.v[0][5, 0, ::2] = 0
    a.fill()
    a.check()


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("first,then", [(100, -40), (110, -60), (-40, 100), (-100, -120), (60, 60)])
def test_values_of_any_size(bits, first, then):
    """Large values of no weight before, and after, small ones that have it all."""
    a = Scene(9, bits, 32, 5, 1, 128, [300], [1], 1.0, vsize=lambda i, n: np.where(np.arange(n) < 64, 2.0 ** first, 2.0 ** then))
    q = bf2f_array(a.q)[0].astype(np.float64).mean(0)
    late = bf2f_array(a.k[0])
    late[64:] = late[64:] * 0.1 + (q * 600 / (a.scale * (q @ q)))[None, None]
    a.k[0] = bf16(late)
    a.fill()
    y, e = a.device().run()
    assert np.isfinite(bf2f_array(y)).all()
    wy, ty, wl, tl = a.expect()
    off = np.abs(bf2f_array(y).astype(np.float64) - wy)
    assert (off <= ty + 2.0 ** (max(first, then) - 120)).all()  # (below 2^-120 of the largest value's scale: fp32's range)
    assert (np.abs(e - wl) <= tl).all()


# (in bf16 q . k is summed before the scale, and leaves fp32 at 2^123 times these queries)
@pytest.mark.parametrize("bits,power", [(b, p) for b in (16, 8, 4) for p in (-110, 100, 118, 119, 120, 123) if b < 16 or p < 123])
def test_queries_and_scales_far_from_one(bits, power):
    """Queries times a power of two with a scale divided by it: the same scores."""
    a = Scene(12, bits, 16, 5, 1, 128, [300, 37], [2, 1], 1.0).device()
    y, e = a.run()
    a.q = bf16(bf2f_array(a.q) * np.float32(2.0 ** power))
    assert np.isfinite(bf2f_array(a.q)).all()
    a.scale /= 2.0 ** power
    y2, e2 = a.run()
    assert np.array_equal(y, y2) and np.array_equal(e, e2)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("power,scale", [(124, 0.088), (-10, 3.0e38), (0, 1e30)])
def test_scores_at_the_end_of_fp32(bits, power, scale):
    """A row whose best score leads by far, up to where scores leave fp32: that token's value."""
    a = Scene(13, bits, 16, 1, 1, 128, [100], [1], 1.0)
    q = np.where(np.arange(128) % 2, 1.0, -1.0) * 2.0 ** power
    a.q = bf16(q).reshape(1, 1, 128)
    a.k[0] = bf16(np.full((100, 1, 128), 0.0))
    a.k[0][41, 0, :4] = bf16(q[:4] * 2.0 ** -power * 2.0 ** -9)
    a.scale = scale
    a.fill()
    y, _ = a.device().run()
    from _ops import held
    assert np.array_equal(y[0, 0], bf16(held(a.v[0], bits)[41, 0]))


@pytest.mark.parametrize("drafts", [1, 3])
def test_infinite_values(drafts):
    """In bf16 an infinite value of a token that a row sees makes that output infinite, both signs nothing."""
    a = Scene(10, 16, 16, 4, 1, 128, [200, 1400, 30], [drafts] * 3, 1.0)
    for i, n in enumerate(a.lens):
        v = a.v[i]
        v[n - drafts, 0, 3], v[3, 0, 9], v[5, 0, 9] = 0x7F80, 0xFF80, 0x7F80
        v[n - drafts - 1, 0, 20], v[0, 0, 127] = 0xFF80, 0x7FC0
    a.fill()
    y, e = a.device().run()
    f = bf2f_array(y)
    assert (f[..., 3] == np.inf).all() and (f[..., 20] == -np.inf).all()
    assert np.isnan(f[..., 9]).all() and np.isnan(f[..., 127]).all()
    for i in range(3):
        a.v[i][~np.isfinite(bf2f_array(a.v[i]))] = 0
    y[..., [3, 9, 20, 127]] = 0
    wy, ty, wl, tl = a.expect()
    rest = [c for c in range(128) if c not in (3, 9, 20, 127)]
    assert (np.abs(bf2f_array(y) - wy) <= ty)[..., rest].all() and (np.abs(e - wl) <= tl).all()
