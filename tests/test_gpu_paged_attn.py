"""Attention over the paged cache (ak_paged_attn) on the GPU, against 64 bits (numpy, test infrastructure).

Tolerance of an output: its own rounding to bf16 (2^-8 of it at most), the rounding of the softmax weights to bf16 before
they meet the values (2^-8 of sum p |v|), and the scores' error dz, which changes a weight by the factor exp(dz): a score
is an fp32 sum of dim products whose terms are at most |q| (|k| + the code's offset), so dz is below (dim + 8) * 2^-24 times
scale * sum |q| |k|, the offset making that at most 130 times as large for a code near zero.  lse: dz, and fp32's own
rounding."""
import ctypes

import numpy as np
import pytest

from _lib import check, Dev, f2bf_array, bf2f_array
from _ops import ops, Pool, held, attention64, page_bytes, Stream, Graph

pytestmark = pytest.mark.gpu


def bits16(x):
    x = np.asarray(x, dtype=np.float32)
    return f2bf_array(x.ravel()).reshape(x.shape)


class Batch:
    """Sequences with their pages: contexts `lens`, `counts` new tokens each."""

    def __init__(self, seed, bits, page, heads, kv, dim, lens, counts, sharp=1.5, spare=3, fill=0xFF):
        rng = self.rng = np.random.default_rng(seed)
        self.bits, self.page, self.heads, self.kv, self.dim = bits, page, heads, kv, dim
        self.lens, self.counts = list(lens), list(counts)
        self.m, self.b = sum(counts), len(lens)
        need = [(n + page - 1) // page for n in lens]
        self.npages = sum(need) + spare
        self.pool = Pool(bits, page, kv, dim, self.npages, fill)
        self.ldt = max(need + [1]) + 1
        self.table = np.full((self.b, self.ldt), -7, dtype=np.int32)
        order, at = rng.permutation(self.npages), 0
        self.k, self.v, self.present = [], [], []
        for i, n in enumerate(lens):
            pages = order[at:at + need[i]]
            at += need[i]
            self.table[i, :need[i]] = pages
            k, v = (bits16(rng.standard_normal((n, kv, dim)) * np.exp(0.3 * rng.standard_normal((n, kv, 1))))
                    for _ in range(2))
            self.k.append(k)
            self.v.append(v)
            self.present.append(np.ones(n, dtype=bool))
            if n:
                self.pool.put(pages[np.arange(n) // page] * page + np.arange(n) % page, k, v)
        self.q = bits16(rng.standard_normal((self.m, heads, dim)) * sharp)
        self.scale = dim ** -0.5
        self.first = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)

    def want(self):
        seqs = [(self.first[i], self.counts[i], held(self.k[i], self.bits), held(self.v[i], self.bits), self.present[i])
                for i in range(self.b)]
        return attention64(self.q, seqs, self.heads, self.kv, self.dim, self.scale)

    def device(self):
        self.P, self.T = Dev.of(self.pool.mem), Dev.of(self.table)
        self.L, self.F = Dev.of(np.asarray(self.lens, dtype=np.int32)), Dev.of(self.first)
        return self

    def run(self, ragged=True, padq=0, pady=0, stream=None, sync=True, table=None):
        w = self.heads * self.dim
        q = np.full((max(self.m, 1), w + padq), 0x7FC0, dtype=np.uint16)
        q[:self.m, :w] = self.q.reshape(self.m, w)
        Q = Dev.of(q)
        self.Y = Dev.of(np.full((max(self.m, 1), w + pady), 0x1234, dtype=np.uint16))
        self.E = Dev.of(np.full((max(self.m, 1), self.heads), 77.0, dtype=np.float32))
        check(ops().ak_paged_attn(self.bits, Q.p, self.m, w + padq, self.P.p, self.npages, self.page, self.heads, self.kv,
                                  self.dim, self.b, self.F.p if ragged else None, self.L.p, (table or self.T).p, self.ldt,
                                  self.scale, self.Y.p, w + pady, self.E.p, stream), "ak_paged_attn")
        check(ops().ak_synchronize())
        y = self.Y.get(np.uint16, self.m * (w + pady)).reshape(self.m, w + pady)
        assert (y[:, w:] == 0x1234).all()
        return y[:, :w].reshape(self.m, self.heads, self.dim), self.E.get(np.float32, self.m * self.heads).reshape(
            self.m, self.heads)

    def check(self, **kw):
        y, e = self.device().run(**kw)
        self.compare(y, e)
        return y, e

    def compare(self, y, e, rows=slice(None)):
        wy, we, mag, zabs = self.want()
        dz = (self.dim + 8) * 2.0 ** -24 * zabs * (1 if self.bits == 16 else 130)
        got = bf2f_array(y).astype(np.float64)
        tol = 2.0 ** -8 * np.abs(wy) + (2.0 ** -8 + 2 * dz[..., None]) * mag + 1e-30
        bad = ~(np.abs(got - wy) <= tol)[rows]
        assert not bad.any(), f"{bad.sum()} of {bad.size} outputs, worst {(np.abs(got - wy) / tol)[rows].max():.2f}"
        empty = np.isneginf(we)
        assert np.array_equal(np.isneginf(e)[rows], empty[rows]) and not y[empty].any()
        ok = np.abs(e - we, where=~empty, out=np.zeros_like(we)) <= dz + 2.0 ** -20 * (1 + np.abs(np.where(empty, 0, we)))
        assert ok[rows].all()


SHAPES = [  # page, heads, kv, dim
    (16, 40, 8, 128), (32, 5, 1, 128), (64, 8, 8, 64), (16, 6, 2, 256), (256, 4, 4, 128), (128, 16, 1, 64), (32, 24, 1, 128)]


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("page,heads,kv,dim", SHAPES)
def test_one_token_each(bits, page, heads, kv, dim):
    """Contexts from nothing to a few pages, ends inside and at the edges of pages and tiles."""
    lens = [0, 1, 2, 15, 16, 17, 31, 33, 64, 65, 100, page, page + 1, 300]
    Batch(bits + page, bits, page, heads, kv, dim, lens, [1] * len(lens)).check(ragged=False)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("lens", [[511], [512], [513], [1024, 1025], [2047, 3], [5003], [4096, 4097, 1]])
def test_split_contexts(bits, lens):
    Batch(3, bits, 32, 5, 1, 128, lens, [1] * len(lens)).check(ragged=False)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("page,heads,kv,dim", SHAPES[:4])
def test_drafts(bits, page, heads, kv, dim):
    """Several new tokens a sequence, causal at the cache's end, more of them than the cache holds, none at all."""
    lens, counts = [8, 70, 513, 5, 0, 1030, 40, 9], [8, 1, 7, 9, 3, 16, 0, 2]
    Batch(11 + bits, bits, page, heads, kv, dim, lens, counts).check()


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_many_rows(bits):
    """A prompt's worth of new tokens on a few heads."""
    Batch(2, bits, 16, 8, 2, 128, [150, 700], [131, 40]).check()


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_uniform_counts_without_ranges(bits):
    b = Batch(4, bits, 16, 10, 2, 128, [37, 600, 4], [4, 4, 4])
    y, e = b.check(ragged=False)
    y2, e2 = b.run(ragged=True)
    assert np.array_equal(y, y2) and np.array_equal(e, e2)


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_strides(bits):
    Batch(5, bits, 16, 5, 1, 128, [20, 333], [3, 2]).check(padq=24, pady=8)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("page", [16, 64])
def test_absent_pages(bits, page):
    """Pages that are not held (negative, or past the pool) are as if their tokens were not there; a row may lose all."""
    b = Batch(6, bits, page, 5, 1, 128, [700, 90, 64, 1300], [1, 3, 2, 5])
    for i, gone in ((0, [0, 2, 10]), (1, [0]), (2, list(range(64 // page))), (3, [0, 1, 5, 6, 7, 8, 9, 10])):
        for p in gone:
            if p * page < b.lens[i]:
                b.table[i, p] = -1 if p % 2 else b.npages + p
                b.present[i][p * page:(p + 1) * page] = False
    b.check()


def test_lengths_past_the_table_and_bad_ranges():
    """Lengths end at the table's last page, token ranges at the tokens there are; what is in no range is left alone."""
    b = Batch(7, 8, 16, 5, 1, 128, [48, 32], [2, 1]).device()
    b.m += 2  # two tokens in nobody's range
    b.q = np.concatenate([b.q, b.q[:2]])
    y, e = b.run()
    long = np.array([1 << 30, 32], dtype=np.int32)
    b.ldt = 3
    b.table = np.ascontiguousarray(b.table[:, :3])
    b.T, b.L = Dev.of(b.table), Dev.of(long)
    y2, e2 = b.run()
    assert np.array_equal(y[:3], y2[:3]) and np.array_equal(e[:3], e2[:3])
    for a in (y, y2):
        assert (a[3:] == 0x1234).all()
    b.F = Dev.of(np.array([2, 1, 1 << 30], dtype=np.int32))  # ends before it begins; past the tokens
    y3, e3 = b.run()
    assert (y3[:1] == 0x1234).all() and (e3[:1] == 77.0).all()
    b.L = Dev.of(np.array([-5, 32], dtype=np.int32))
    b.F = Dev.of(b.first)
    y4, e4 = b.run()
    assert not y4[:2].any() and np.isneginf(e4[:2]).all() and np.array_equal(y4[2], y[2])


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("bad", ["nan", "inf"])
def test_rows_do_not_see_later_tokens(bits, bad):
    """NaN or Inf in the keys and values of a later draft leave the earlier rows as they are."""
    lens, counts = [300, 40, 6], [5, 4, 6]
    clean = Batch(9, bits, 16, 5, 1, 128, lens, counts)
    y, e = clean.device().run()
    dirty = Batch(9, bits, 16, 5, 1, 128, lens, counts)
    for i, n in enumerate(lens):
        for x in (dirty.k[i], dirty.v[i]):
            x[n - 2, 0, 7:9] = 0x7FC0 if bad == "nan" else 0x7F80  # the last but one
        pages = dirty.table[i, :(n + 15) // 16]
        dirty.pool.put(pages[np.arange(n) // 16] * 16 + np.arange(n) % 16, dirty.k[i], dirty.v[i])
    y2, e2 = dirty.device().run()
    for i in range(3):
        a, z = clean.first[i], clean.first[i + 1]
        assert np.array_equal(y[a:z - 2], y2[a:z - 2]) and np.array_equal(e[a:z - 2], e2[a:z - 2])
        assert not np.isfinite(bf2f_array(y2[z - 2:z])).all()


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_slots_past_the_end_have_no_effect(bits):
    a = Batch(10, bits, 64, 5, 1, 128, [70, 1, 530], [2, 1, 3], fill=0xFF)
    z = Batch(10, bits, 64, 5, 1, 128, [70, 1, 530], [2, 1, 3], fill=0x00)
    for (y, e), (y2, e2) in [(a.device().run(), z.device().run())]:
        assert np.array_equal(y, y2) and np.array_equal(e, e2)


def test_infinite_scores_and_large_ones():
    """Scores of both signs far apart, and a key of -inf direction: the other keys' softmax."""
    b = Batch(12, 16, 16, 4, 1, 128, [200], [1], sharp=60.0)
    b.k[0][17, 0] = 0
    b.k[0][17, 0, 0] = 0xFF80  # score -inf or +inf by the sign of q
    b.q[0, :, 0] = bits16(np.array([2.0]))[0]
    pages = b.table[0, :13]
    b.pool.put(pages[np.arange(200) // 16] * 16 + np.arange(200) % 16, b.k[0], b.v[0])
    b.present[0][17] = False  # exp(-inf) = 0
    y, e = b.device().run()
    b.k[0][17] = 0
    b.compare(y, e)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("heads,kv,dim", [(5, 1, 128), (8, 8, 64), (16, 2, 256)])
def test_rows_do_not_depend_on_the_call(bits, heads, kv, dim):
    """A verify of T drafts gives, bit for bit, what T one-token calls give, alone or in a batch."""
    lens, counts = [1100, 65, 530, 4500], [6, 3, 9, 8]
    b = Batch(13, bits, 16, heads, kv, dim, lens, counts)
    y, e = b.device().run()
    for i in range(4):
        for t in (0, counts[i] // 2, counts[i] - 1):
            one = Batch.__new__(Batch)
            one.__dict__.update(b.__dict__)
            one.lens, one.counts, one.b, one.m = [lens[i] - counts[i] + t + 1], [1], 1, 1
            one.q, one.table = b.q[b.first[i] + t:b.first[i] + t + 1], np.ascontiguousarray(b.table[i:i + 1])
            one.first = np.array([0, 1], dtype=np.int32)
            y1, e1 = one.device().run()
            assert np.array_equal(y1[0], y[b.first[i] + t]) and np.array_equal(e1[0], e[b.first[i] + t])


def test_many_sequences():
    """More (sequence, head) pairs than one launch joins."""
    lens = [(37 * i) % 90 + 1 for i in range(300)]
    lens[7], lens[200] = 1700, 2600
    Batch(14, 8, 16, 8, 8, 64, lens, [1] * 300).check(ragged=False)


def test_pool_past_4_gib():
    bits, page, heads, dim = 8, 256, 8, 128
    pb = page_bytes(bits, page, heads, dim)
    npages = (5 << 30) // pb
    b = Batch(15, bits, page, 40, 8, dim, [300], [1]).device()
    big = Dev(npages * pb)
    top = npages - 1
    for i, p in enumerate(b.table[0, :2]):
        src = np.ascontiguousarray(b.pool.mem[p])
        check(ops().ak_memcpy_h2d(big.addr((top - i) * pb), ctypes.c_void_p(src.ctypes.data), pb))
    b.P, b.npages = big, npages
    b.table[0, :2] = [top, top - 1]
    b.T = Dev.of(b.table)
    b.compare(*b.run())


def put(dev, arr):
    arr = np.ascontiguousarray(arr)
    check(ops().ak_memcpy_h2d(dev.p, ctypes.c_void_p(arr.ctypes.data), arr.nbytes))


@pytest.mark.parametrize("first", ["eager", "captured"])
def test_streams_and_graph_replays(first):
    """A call on another stream, and a captured one whose lengths change between the replays, with eager calls on the same
    stream in between; also where the capture is the first call on its stream."""
    b = Batch(16, 8, 16, 40, 8, 128, [1500, 20, 700], [1, 1, 1]).device()
    y0, e0 = b.run(ragged=False)
    w, n = 40 * 128, 3 * 40
    s = Stream()
    Q, Y, E = Dev.of(b.q), Dev(3 * w * 2), Dev(n * 4)

    def call(stream):
        return ops().ak_paged_attn(8, Q.p, 3, w, b.P.p, b.npages, 16, 40, 8, 128, 3, None, b.L.p, b.T.p, b.ldt, b.scale, Y.p,
                                   w, E.p, stream)

    def take():
        s.sync()
        out = Y.get(np.uint16, 3 * w).reshape(y0.shape), E.get(np.float32, n).reshape(e0.shape)
        put(Y, np.full(3 * w, 0x7FC1, dtype=np.uint16))
        return out
    if first == "eager":
        assert call(s.h) == 0
        y, e = take()
        assert np.array_equal(y, y0) and np.array_equal(e, e0)
    g = Graph(s, call)
    for step in range(4):
        put(b.L, np.array([1500 - 400 * step, 20 - step, 700 - 3 * step], dtype=np.int32))
        g.launch()
        y, e = take()
        assert call(s.h) == 0
        y2, e2 = take()
        assert np.array_equal(y, y2) and np.array_equal(e, e2)
        if step == 0:
            assert np.array_equal(y, y0) and np.array_equal(e, e0)


def test_no_tokens():
    assert ops().ak_paged_attn(8, None, 0, 0, None, 1, 16, 8, 8, 128, 0, None, None, None, 1, 1.0, None, 0, None, None) == 0
