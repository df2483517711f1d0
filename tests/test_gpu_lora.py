"""Low-rank adapters (ak_lora_plan, ak_lora_add) on the GPU, against 64 bits (numpy, test infrastructure).

Tolerance of an output y with M = scale * sum |B| sum |x A|: half a bf16 step of y; (k / 8 + rank / 8 + 64) fp32 roundings of
M for the sums (products of a matrix instruction may be added one after another); 2^-17 M for A x held in two bf16."""
import numpy as np
import pytest

from _lib import check, Dev, f2bf_array, bf2f_array, ptr_array, int_array
from _ops import Stream, Graph
from _step import step, lora64, i32

pytestmark = pytest.mark.gpu

FILL = 0x1234


def bf(rng, *shape, scale=1.0):
    return f2bf_array((rng.standard_normal(shape) * scale).astype(np.float32).ravel()).reshape(shape)


class Job:
    def __init__(self, seed, m, adapters, rank, k, ns, ids=None, pad=0, scale=True, in_place=False):
        rng = np.random.default_rng(seed)
        self.__dict__.update(m=m, adapters=adapters, rank=rank, k=k, ns=ns, in_place=in_place)
        self.ids = i32(rng.integers(-1, adapters, m) if ids is None else ids)
        self.x = bf(rng, m, k)
        self.a, self.b = bf(rng, adapters, len(ns) * rank, k, scale=k ** -0.5), [bf(rng, adapters, n, rank, scale=rank ** -0.5) for n in ns]
        self.base = [bf(rng, m, n) for n in ns]
        self.scale = rng.standard_normal(adapters).astype(np.float32) if scale else None
        self.ldx, self.ldy = k + 8 * pad, [n + pad for n in ns]
        xs = np.full((m, self.ldx), 0x7FC1, dtype=np.uint16)
        xs[:, :k] = self.x
        self.I, self.X, self.A = Dev.of(self.ids), Dev.of(xs), Dev.of(self.a)
        self.B, self.S = [Dev.of(v) for v in self.b], Dev.of(self.scale) if scale else None
        self.Z = []
        for v, ld in zip(self.base, self.ldy):
            z = np.full((m, ld), FILL, dtype=np.uint16)
            z[:, :v.shape[1]] = v
            self.Z.append(Dev.of(z))
        self.fresh()
        size = step().ak_lora_plan_bytes(m, adapters, len(ns) * rank, k)
        self.size = size
        self.P = Dev.of(np.full(size + 64, 0xA5, dtype=np.uint8))

    def fresh(self):
        self.Y = []
        for v, ld in zip(self.base, self.ldy):
            z = np.full((self.m, ld), FILL, dtype=np.uint16)
            if self.in_place:
                z[:, :v.shape[1]] = v
            self.Y.append(Dev.of(z))

    def plan(self, stream=None):
        return step().ak_lora_plan(self.I.p, self.m, self.adapters, self.P.p, stream)

    def add(self, stream=None, m=None, adapters=None):
        return step().ak_lora_add(self.P.p, self.X.p, m or self.m, self.ldx, self.k, adapters or self.adapters, self.rank,
                                  self.A.p, self.S.p if self.S else None, len(self.ns), ptr_array([v.p for v in self.B]),
                                  None if self.in_place else ptr_array([v.p for v in self.Z]), ptr_array([v.p for v in self.Y]),
                                  int_array(self.ns), int_array(self.ldy), stream)

    def run(self):
        check(self.plan())
        check(self.add())
        return self.got()

    def got(self):
        check(step().ak_synchronize())
        assert (self.P.get(np.uint8, self.size + 64)[self.size:] == 0xA5).all()
        out = []
        for Y, n, ld in zip(self.Y, self.ns, self.ldy):
            y = Y.get(np.uint16, self.m * ld).reshape(self.m, ld)
            assert (y[:, n:] == FILL).all()  # between the rows
            out.append(y[:, :n])
        return out

    def compare(self, got):
        want, mag = lora64(self.x, self.ids, self.a, self.b, self.scale, self.base, self.rank)
        none = (self.ids < 0) | (self.ids >= self.adapters)
        for y, w, g, z in zip(got, want, mag, self.base):
            assert np.array_equal(y[none], z[none])
            err = np.abs(bf2f_array(y).astype(np.float64).reshape(y.shape) - w)
            tol = 2.0 ** -8 * np.abs(w) + g * ((self.k / 8 + self.rank / 8 + 64) * 2.0 ** -24 * 1.01 + 2.0 ** -17)
            assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("m,adapters,rank,k,ns", [
    (1, 1, 8, 8, [1]), (1, 4, 16, 5120, [5120]), (2, 3, 24, 520, [17]), (17, 5, 64, 1000, [300, 33]), (64, 32, 16, 5120, [5120, 1024, 1024]),
    (100, 2, 128, 264, [257, 64, 1, 100]), (130, 1, 32, 4104, [64]), (333, 40, 8, 512, [129]), (700, 3, 48, 9000, [70]),
    (5, 4096, 16, 64, [40]), (1500, 7, 16, 640, [2055]), (900, 3, 64, 9000, [70, 64]), (1000, 2, 128, 8200, [40]),
    (3400, 5, 16, 520, [72])])
def test_against_64_bits(m, adapters, rank, k, ns):
    j = Job(m + k, m, adapters, rank, k, ns, pad=m % 3)
    j.compare(j.run())


@pytest.mark.parametrize("m,adapters,rank,k,ns", [(1800, 3, 64, 9000, [70, 64]), (2600, 2, 40, 9000, [33]), (700, 5, 72, 27648, [17, 1, 80])])
def test_sums_of_many_tokens_and_parts(m, adapters, rank, k, ns):
    """Parts that are added up once, ahead of the second product: segments, ranks of no multiple of 32, odd outputs."""
    j = Job(m + rank, m, adapters, rank, k, ns, pad=m % 3)
    j.compare(j.run())


@pytest.mark.parametrize("pad", [0, 1, 8])
def test_in_place_and_without_scales(pad):
    j = Job(5, 90, 4, 16, 1024, [500, 40], pad=pad, scale=False, in_place=True)
    j.compare(j.run())


@pytest.mark.parametrize("ids", [[-1] * 70, [0] * 70, [3] * 64 + [1] * 6, [9, -7, 2 ** 31 - 1, -2 ** 31] + [2] * 66,
                                 list(range(4)) * 17 + [3, 3], [-1] * 69 + [0]])
@pytest.mark.parametrize("in_place", [False, True])
def test_groups_of_every_kind(ids, in_place):
    j = Job(6, 70, 4, 16, 256, [100], ids=ids, in_place=in_place)
    j.compare(j.run())


@pytest.mark.parametrize("rank", [16, 64])
def test_tokens_do_not_depend_on_the_call(rank):
    """Alone, in small batches and in large ones that take other launches: the same bits."""
    rng = np.random.default_rng(1)
    big = Job(7, 2600, 3, rank, 9224, [96], ids=rng.integers(-1, 3, 2600))
    y = big.run()[0]
    for some in ([0], [5, 9], list(range(100, 140)), list(rng.integers(0, 2600, 300))):
        j = Job(7, len(some), 3, rank, 9224, [96], ids=big.ids[some])
        j.x, j.a, j.b, j.scale = big.x[some], big.a, big.b, big.scale
        j.X, j.A, j.B, j.S = Dev.of(j.x), big.A, big.B, big.S
        j.Z = [Dev.of(big.base[0][some])]
        j.base = [big.base[0][some]]
        assert np.array_equal(j.run()[0], y[some])


def test_non_finite_values_stay_in_their_rows():
    j = Job(8, 40, 2, 16, 512, [64])
    x = j.x.copy()
    j.ids[:] = np.arange(40) % 2
    x[3, 5], x[6, 7], x[9, 0] = 0x7F80, 0x7FC0, 0x7F7F
    j.X, j.I = Dev.of(x), Dev.of(j.ids)
    y = j.run()[0]
    bad = [i for i in range(40) if not np.isfinite(bf2f_array(y[i])).all()]
    assert set(bad) <= {3, 6, 9} and {3, 6} <= set(bad)
    keep = [i for i in range(40) if i not in (3, 6, 9)]
    j.x = x
    want, _ = lora64(x[keep], j.ids[keep], j.a, j.b, j.scale, [j.base[0][keep]], 16)
    assert np.allclose(bf2f_array(y[keep]).reshape(len(keep), 64), want[0], rtol=2.0 ** -7, atol=1e-2)


def test_an_infinite_sum_is_infinite():
    """With weights of one sign no infinities meet: the output is infinite, as the formula's (of several signs it is NaN)."""
    j = Job(8, 20, 1, 16, 512, [64], ids=[0] * 20, scale=False)
    x = j.x.copy()
    x[3, 5], x[4, 6] = 0x7F80, 0xFF80
    j.X, j.A, j.B = Dev.of(x), Dev.of(j.a & 0x7FFF), [Dev.of(j.b[0] & 0x7FFF)]
    y = bf2f_array(j.run()[0]).reshape(20, 64)
    assert (y[3] == np.inf).all() and (y[4] == -np.inf).all() and np.isfinite(np.delete(y, [3, 4], 0)).all()


def test_one_plan_for_linears_of_other_shapes():
    """The plan is made once; a linear with fewer inputs and rows runs in the same memory."""
    a, b = Job(9, 50, 6, 32, 2048, [200]), Job(10, 50, 6, 16, 512, [90, 30])
    b.ids, b.P, b.size = a.ids, a.P, a.size
    check(a.plan())
    check(a.add())
    check(b.add())
    check(a.add())
    a.compare(a.got())
    b.compare(b.got())


def test_a_plan_of_another_call_changes_nothing():
    j = Job(11, 30, 4, 16, 256, [64])
    check(j.plan())
    check(j.add(m=29))
    check(j.add(adapters=3))
    assert (j.got()[0] == FILL).all()
    assert step().ak_lora_add(j.P.p, None, 0, 8, 8, 4, 16, None, None, 1, ptr_array([0]), None, ptr_array([0]), int_array([1]), None,
                              None) == 0


def test_captured_plan_follows_the_ids():
    rng = np.random.default_rng(2)
    j = Job(12, 48, 8, 16, 1024, [300, 64])
    s = Stream()
    g = Graph(s, lambda st: j.plan(st) or j.add(st))
    for _ in range(4):
        j.ids = i32(rng.integers(-1, 8, 48))
        check(step().ak_memcpy_h2d(j.I.p, j.ids.ctypes.data, j.ids.nbytes))
        g.launch()
        s.sync()
        j.compare(j.got())


def test_two_streams_with_plans_of_their_own():
    jobs = [Job(20 + i, 60, 5, 16, 2048, [500]) for i in range(2)]
    s = [Stream(), Stream()]
    for _ in range(20):
        for j, st in zip(jobs, s):
            check(j.plan(st.h))
            check(j.add(st.h))
    for j in jobs:
        j.compare(j.got())


@pytest.mark.parametrize("m,rank,k", [(1, 16, 64), (3, 16, 5120), (70, 8, 1024), (700, 32, 9224), (700, 64, 9224), (1800, 64, 9000),
                                      (1800, 72, 9000), (3700, 64, 5120)])
def test_sums_enter_the_second_product_with_24_bits(m, rank, k):
    """A sum s = p0 + p1 + p2 of three bf16, from which the second product takes p1 and the base takes p0: p2 is left, which lies
    below the 16 bits of two bf16.  All of it is exact in fp32 but for the last sums' order: four roundings of s at most."""
    rng = np.random.default_rng(m + rank)
    s = (np.float32(1) + rng.random(m).astype(np.float32) * np.float32(0.9)) * np.float32(2) ** rng.integers(-20, 20, m).astype(np.float32)
    part, left = [], s
    for _ in range(3):
        part.append(f2bf_array(left))
        left = left - bf2f_array(part[-1])
    assert (left == 0).all() and (np.abs(bf2f_array(part[2])) > 8 * 2.0 ** -24 * s).any()
    j = Job(30, m, 2, rank, k, [9], ids=[t % 2 for t in range(m)], scale=False)
    x, a, b = np.zeros((m, k), dtype=np.uint16), np.zeros((2, rank, k), dtype=np.uint16), np.zeros((2, 9, rank), dtype=np.uint16)
    one, at = 0x3F80, [0, k // 3, k // 2, k - 1]
    for i, p in zip(at, part + [part[1] ^ 0x8000]):
        x[:, i] = p
    a[:, 0, at[:3]], a[:, rank - 1, at[3]] = one, one
    b[:, :, 0], b[:, :, rank - 1] = one, one
    base = np.repeat((part[0] ^ 0x8000)[:, None], 9, axis=1)
    j.X, j.A, j.B, j.Z = Dev.of(x), Dev.of(a), [Dev.of(b)], [Dev.of(base)]
    y = bf2f_array(j.run()[0]).astype(np.float64).reshape(m, 9)
    want = bf2f_array(part[2]).astype(np.float64)[:, None]
    assert (np.abs(y - want) <= 4 * 2.0 ** -24 * s[:, None]).all()


@pytest.mark.parametrize("m,adapters", [(40, 3), (1, 3), (0, 3), (1799, 3), (1801, 3), (1800, 2), (1800, 600), (3000, 3)])
@pytest.mark.parametrize("calls", [(1800, 64, 9000), (700, 16, 9224), (30, 16, 256)])
def test_memory_past_a_plan_of_other_sizes_stays(m, adapters, calls):
    """A plan of m tokens and `adapters`, and a call of other sizes in all of its launches' forms (joined sums, many tokens, few):
    the outputs stay, and so does all behind the plan's own memory, which here goes on for the call's needs."""
    n, rank, k = calls
    j = Job(40, n, 3, rank, k, [70])
    own = step().ak_lora_plan_bytes(m, adapters, rank, k)
    room = max(own, j.size) + 64
    j.P = Dev.of(np.full(room, 0xA5, dtype=np.uint8))
    ids = Dev.of(i32(np.arange(max(m, 1)) % adapters))
    check(step().ak_lora_plan(ids.p, m, adapters, j.P.p, None))
    check(step().ak_synchronize())
    before = j.P.get(np.uint8, room)
    assert (before[own:] == 0xA5).all()
    check(j.add())
    check(step().ak_synchronize())
    assert np.array_equal(j.P.get(np.uint8, room), before)
    assert (j.Y[0].get(np.uint16, n * j.ldy[0]) == FILL).all()


@pytest.mark.parametrize("m,adapters,used,rank,ns,in_place", [(4200, 4096, 3, 8, [700, 70], False), (4200, 4096, 3, 8, [700, 70], True),
                                                              (2000, 2000, 2000, 8, [1300], False), (8192, 3, 3, 64, [5120], True),
                                                              (300, 600, 40, 40, [2055, 1030], False)])
def test_many_output_rows_of_a_workgroup(m, adapters, used, rank, ns, in_place):
    """512 and 1024 output rows a workgroup, full tiles and tiles of a token, rows that end within a turn."""
    ids = np.random.default_rng(m).integers(-1, used, m)
    j = Job(50 + m, m, adapters, rank, 64, ns, ids=ids, in_place=in_place)
    j.compare(j.run())


@pytest.mark.parametrize("m", [40, 1800])
def test_infinite_weights_of_the_second_product_stay_in_their_output(m):
    j = Job(60, m, 2, 64, 9000, [70], ids=np.arange(m) % 2)
    want = j.run()[0]
    b = j.b[0].copy()
    b[1, 33, 5], b[1, 64, 9] = 0x7F80, 0xFF80
    j.B = [Dev.of(b)]
    y = j.run()[0]
    bad = np.zeros(y.shape, dtype=bool)
    bad[1::2, [33, 64]] = True
    assert np.array_equal(y[~bad], want[~bad]) and not np.isfinite(bf2f_array(y[bad])).any()
