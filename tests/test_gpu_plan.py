"""Pages, slots and positions of a batch (ak_kv_plan) on the GPU, number for number against the definition."""
import numpy as np
import pytest

from _lib import check, Dev
from _ops import Stream, Graph
from _step import step, plan64, i32

pytestmark = pytest.mark.gpu

GUARD = 77


class Batch:
    def __init__(self, seed, b, page, ldt, longest, short=0, drops=0.2, spare=5):
        rng = np.random.default_rng(seed)
        self.b, self.page, self.ldt = b, page, ldt
        self.cached = rng.integers(0, ldt * page + 1, b)
        self.counts = np.minimum(rng.integers(0, longest + 1, b), ldt * page - self.cached)
        self.drop = (rng.random(b) < drops).astype(np.int32)
        self.held = -(-self.cached // page)
        more = rng.random(b) < 0.2  # pages kept from rejected drafts
        self.held = np.minimum(self.held + more, ldt)
        need = np.maximum(-(-(self.cached + self.counts) // page) - self.held, 0).sum() + (self.drop * 3).sum()
        total = int(self.held.sum() + need) + 7
        self.npages = total
        ids = rng.permutation(total)
        self.table = np.full((b, ldt), -1, dtype=np.int32)
        at = 0
        for i, h in enumerate(self.held):
            self.table[i, :h] = ids[at:at + h]
            at += h
        self.free = np.full(total, -1, dtype=np.int32)
        self.nfree = total - at
        self.free[:self.nfree] = ids[at:]
        self.nfree = max(self.nfree - short, 0)
        self.m = int(self.counts.sum()) + spare

    def want(self, drop=True, alloc=True):
        return plan64(self.counts, self.drop if drop else None, self.cached, self.held, self.table, self.free, self.nfree,
                      self.page, self.npages, self.m, alloc)

    def device(self, in_place=False):
        b, m = self.b, self.m
        d = {n: Dev.of(i32(getattr(self, n))) for n in ("counts", "drop", "cached", "held", "table", "free")}
        d["nfree"] = Dev.of(i32([self.nfree]))
        new = lambda n: Dev.of(np.full(n + 1, GUARD, dtype=np.int32))  # noqa: E731
        out = {"lens": d["cached"], "held_out": d["held"], "nfree_out": d["nfree"]} if in_place else \
            {"lens": new(b), "held_out": new(b), "nfree_out": new(1)}
        out.update(qstart=new(b + 1), pos=new(m), slots=new(m), refused=new(b))
        self.d, self.out, self.in_place = d, out, in_place
        return self

    def call(self, stream=None, drop=True, alloc=True, m=None):
        d, o = self.d, self.out
        p = lambda x: x.p if alloc else None  # noqa: E731
        return step().ak_kv_plan(self.b, self.m if m is None else m, d["counts"].p, d["drop"].p if drop else None, d["cached"].p,
                                 p(d["held"]), p(d["nfree"]), p(d["free"]), self.npages, self.page, d["table"].p, self.ldt,
                                 o["lens"].p, p(o["held_out"]), p(o["nfree_out"]), o["qstart"].p, o["pos"].p, o["slots"].p,
                                 o["refused"].p, stream)

    def got(self, alloc=True):
        check(step().ak_synchronize())
        b, m, o, d = self.b, self.m, self.out, self.d
        r = {}
        for name, src, n in (("lens", "lens", b), ("held", "held_out", b), ("nfree", "nfree_out", 1), ("qstart", "qstart", b + 1),
                             ("pos", "pos", m), ("slots", "slots", m), ("refused", "refused", b)):
            if not alloc and name in ("held", "nfree"):
                continue
            own = self.in_place and name in ("lens", "held", "nfree")
            a = o[src].get(np.int32, n if own else n + 1)
            assert own or a[n] == GUARD
            r[name] = a[:n]
        r["table"] = d["table"].get(np.int32, b * self.ldt).reshape(b, self.ldt)
        r["free"] = d["free"].get(np.int32, self.npages)
        return r


def same(got, want):
    for k, v in got.items():
        assert np.array_equal(v, want[k]), (k, v, want[k])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("b,page,ldt,longest", [(1, 16, 4, 1), (1, 256, 1, 300), (3, 16, 300, 900), (64, 32, 40, 1), (65, 16, 20, 0),
                                                (257, 64, 9, 40), (1024, 16, 33, 7), (1024, 128, 5, 60), (200, 16, 256, 700)])
def test_against_the_definition(b, page, ldt, longest, in_place):
    x = Batch(b * 7 + page + longest, b, page, ldt, longest).device(in_place)
    check(x.call())
    same(x.got(), x.want())


@pytest.mark.parametrize("short", [1, 3, 10, 60, 10 ** 6])
@pytest.mark.parametrize("b,longest", [(5, 100), (40, 30), (300, 90)])
def test_too_few_pages(b, longest, short):
    x = Batch(b + short % 100, b, 16, 50, longest, short=short, drops=0.05).device()
    check(x.call())
    w = x.want()
    assert short < 10 ** 6 or b == 5 or w["refused"].any()
    same(x.got(), w)


def test_refusals_of_sequences():
    """A full row, a range past m, counts that are negative or beyond all bounds; the others get theirs."""
    x = Batch(5, 8, 16, 4, 5, drops=0.0)
    x.cached[:] = [0, 60, 64, 3, 10, 2, 1, 0]
    x.counts[:] = [3, 5, 1, 2, -4, 2 ** 31 - 1, 3, 0]
    x.held[:] = [0, 4, 4, 1, 1, 1, 1, 0]
    x.table[:] = np.arange(32).reshape(8, 4)
    x.npages, x.free, x.nfree, x.m = 64, np.arange(64).astype(np.int32), 64, 40
    w = x.want()
    assert w["refused"].tolist() == [0, 1, 1, 0, 0, 1, 1, 1]  # (after the sixth every range is past m)
    x.device()
    check(x.call())
    same(x.got(), w)


def test_bad_numbers_stay_in_bounds():
    """Held pages, lengths and a free count outside their arrays, pages outside the pool: no fault, slots of -1."""
    x = Batch(6, 6, 16, 5, 3, drops=0.0)
    x.cached[:] = [-5, 7, 2 ** 31 - 1, 20, 33, 79]
    x.held[:] = [-1, 9, 5, 1, 2, 5]
    x.table[:] = [[-1] * 5, [10 ** 9] * 5, [1] * 5, [-7] * 5, [2 ** 31 - 1] * 5, [3] * 5]
    x.drop[:] = [0, 0, 1, 0, 0, 0]
    x.counts[:] = [2, 1, 1, 1, 1, 1]
    x.npages, x.free, x.nfree, x.m = 9, np.arange(9).astype(np.int32), 6, 12
    x.device()
    check(x.call())
    same(x.got(), x.want())
    x.nfree = 10 ** 6
    x.device()
    check(x.call())
    assert x.got()["nfree"][0] <= 9


@pytest.mark.parametrize("b,longest", [(4, 9), (50, 300)])
def test_table_as_it_is(b, longest):
    x = Batch(9, b, 32, 30, longest, drops=0.0)
    x.table[:] = np.random.default_rng(1).integers(0, x.npages, x.table.shape)
    x.table[0, :] = -1
    x.device()
    check(x.call(drop=False, alloc=False))
    w = x.want(drop=False, alloc=False)
    g = x.got(alloc=False)
    assert (g["slots"][:w["qstart"][1]] == -1).all()
    same(g, w)


def test_lengths_end_at_31_bits():
    """Room for more than 2^31 tokens: a sequence that would pass them is refused, its neighbour is not."""
    x = Batch(8, 2, 256, 8, 3, drops=0.0)
    x.ldt = (1 << 23) + 5
    x.cached, x.counts = np.array([2 ** 31 - 3, 2 ** 31 - 6]), np.array([3, 5])
    x.table = np.zeros((2, x.ldt), dtype=np.int32)
    x.m = 10
    x.device()
    check(x.call(drop=False, alloc=False))
    g = x.got(alloc=False)
    assert g["refused"].tolist() == [1, 0] and g["lens"].tolist() == [2 ** 31 - 3, 2 ** 31 - 1]
    assert g["pos"][3:8].tolist() == [2 ** 31 - 6 + j for j in range(5)] and (g["pos"][:3] == -1).all()


def test_no_sequences_and_no_tokens():
    x = Batch(3, 1, 16, 4, 0)
    x.m = 6
    x.device()
    x.b = 0
    check(x.call())
    check(step().ak_synchronize())
    assert x.out["qstart"].get(np.int32, 1)[0] == 0 and (x.out["pos"].get(np.int32, 6) == -1).all()
    x = Batch(4, 7, 16, 9, 0, spare=0).device()
    assert x.m == 0
    check(x.call())
    same(x.got(), x.want())


def test_captured_steps_follow_the_device():
    """A decode loop as a graph: every replay takes one token more of each sequence, in place."""
    x = Batch(11, 20, 16, 12, 1, drops=0.0)
    x.cached[:] = np.arange(20) * 3
    x.held[:] = -(-x.cached // 16)
    x.counts[:] = 1
    x.m = 20
    ids = np.random.default_rng(0).permutation(400)
    x.table[:] = -1
    at = 0
    for i, h in enumerate(x.held):
        x.table[i, :h] = ids[at:at + h]
        at += h
    x.npages, x.nfree = 400, 400 - at
    x.free = np.concatenate([ids[at:], np.full(at, -1)]).astype(np.int32)
    x.device(in_place=True)
    s = Stream()
    g = Graph(s, lambda st: x.call(st))
    for _ in range(40):
        w = x.want()
        g.launch()
        s.sync()
        same(x.got(), w)
        x.cached, x.held, x.table, x.free, x.nfree = w["lens"], w["held"], w["table"], w["free"], w["nfree"][0]


@pytest.mark.parametrize("drop", [False, True])
@pytest.mark.parametrize("b,page,ldt,longest", [(1, 16, 700, 11000), (3, 16, 400, 6000), (20, 16, 90, 1400), (64, 32, 60, 1800),
                                                (64, 16, 300, 4700), (5, 256, 100, 25000)])
def test_few_sequences_with_long_prompts(b, page, ldt, longest, drop):
    """More tokens than one launch writes, fewer pages than 1024 and more, and those that ended sequences give back."""
    x = Batch(b + page, b, page, ldt, longest, drops=0.3 if drop else 0.0)
    x.cached = np.where(np.arange(b) % 3 == 1, x.cached, x.cached % 50)
    x.held = np.maximum(-(-x.cached // page), np.minimum(x.held, 5))
    x.counts = np.random.default_rng(b).integers(longest // 2, longest, b)
    x.counts = np.minimum(x.counts, ldt * page - x.cached)
    ids = np.random.default_rng(page).permutation(x.b * ldt + 9)
    x.npages, x.free, at = len(ids), np.full(len(ids), -1, dtype=np.int32), int(x.held.sum())
    x.table = np.full((b, ldt), -1, dtype=np.int32)
    x.table[np.arange(ldt)[None] < x.held[:, None]] = ids[:at]
    x.nfree = len(ids) - at
    x.free[:x.nfree] = ids[at:]
    x.m = int(x.counts.sum()) + 3
    assert x.m > 4096
    x.device()
    check(x.call(drop=drop))
    w = x.want(drop=drop)
    assert (w["nfree"][0] < x.nfree or drop) and not w["refused"].any()
    same(x.got(), w)
