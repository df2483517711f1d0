"""Rotary positions (ak_rope, ak_rope_kv_write) on the GPU, bit for bit against the definition in 64 bits rounded once.

The kernels' angles and products are 64 bits, off by some 2^-52 of a value, and the oracle's likewise: a bf16 border lies
between the two for one value in 2^40 or so."""
import numpy as np
import pytest

from _lib import check, Dev, f2bf_array, bf2f_array
from _ops import Pool, bf16_rn, Stream, Graph
from _step import step, rope64, freqs64, i32

pytestmark = pytest.mark.gpu

FILL = 0x1234


def rows(rng, m, heads, dim):
    x = rng.standard_normal((m, heads, dim)) * np.exp(2 * rng.standard_normal((m, heads, 1)))
    return f2bf_array(x.astype(np.float32).ravel()).reshape(m, heads, dim)


def want(x, pos, freqs, rot, interleaved, mag, old):
    y = x.copy()
    r = bf16_rn(rope64(x, np.maximum(pos, 0), freqs, rot, interleaved, mag))
    y[..., :rot] = r[..., :rot]
    return np.where((np.asarray(pos) < 0)[:, None, None], old, y)


def rotate(x, pos, freqs, rot, interleaved, mag=1.0, pad_in=0, pad_out=0, in_place=False, stream=None):
    m, heads, dim = x.shape
    w = heads * dim
    src = np.full((m, w + pad_in), 0x7FC1, dtype=np.uint16)
    src[:, :w] = x.reshape(m, w)
    X, P, F = Dev.of(src), Dev.of(i32(pos)), Dev.of(np.asarray(freqs, dtype=np.float64))
    ldy = w + (pad_in if in_place else pad_out)
    Y = X if in_place else Dev.of(np.full((m, ldy), FILL, dtype=np.uint16))
    check(step().ak_rope(X.p, w + pad_in, Y.p, ldy, m, heads, dim, P.p, F.p, rot, interleaved, mag, stream), "ak_rope")
    check(step().ak_synchronize())
    y = Y.get(np.uint16, m * ldy).reshape(m, ldy)
    assert (y[:, w:] == (0x7FC1 if in_place else FILL)).all()  # between the rows
    return y[:, :w].reshape(m, heads, dim)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("m,heads,dim,rot", [(1, 48, 128, 128), (5, 3, 64, 64), (37, 2, 256, 64), (9, 5, 80, 20), (3, 1, 96, 96),
                                             (2, 7, 8, 2), (4, 2, 8, 8), (3, 3, 512, 512), (130, 1, 128, 126), (6, 2, 72, 70),
                                             (33, 12, 128, 34)])
def test_against_64_bits(m, heads, dim, rot, interleaved, in_place):
    rng = np.random.default_rng(m * 1000 + dim + rot)
    x = rows(rng, m, heads, dim)
    pos = rng.integers(0, 1 << 20, m)
    pos[0] = 0
    if m > 4:
        pos[2], pos[3] = -1, (1 << 20) + 1
    f, _ = freqs64(1e4, rot)
    got = rotate(x, pos, f, rot, interleaved, 1.25, pad_in=8 * (m % 3), pad_out=16, in_place=in_place)
    old = x if in_place else np.full_like(x, FILL)
    assert np.array_equal(got, want(x, pos, f, rot, interleaved, np.float32(1.25), old))


@pytest.mark.parametrize("scaling", [0, 1, 2, 3])
def test_far_positions_and_scaled_frequencies(scaling):
    rng = np.random.default_rng(scaling)
    x = rows(rng, 64, 2, 128)
    f, mag = freqs64(1e6, 128, scaling, 8.0, 8192)
    pos = np.concatenate([[0, 1, 2 ** 31 - 1, 2 ** 30 + 12345, 10 ** 9], rng.integers(0, 2 ** 31, 59)])
    assert np.array_equal(rotate(x, pos, f, 128, 0, float(np.float32(mag))), want(x, pos, f, 128, 0, np.float32(mag), x))


def test_turning_back():
    """Negative frequencies undo a rotation to within two roundings of a pair's length."""
    rng = np.random.default_rng(2)
    x = rows(rng, 20, 4, 128)
    f, _ = freqs64(1e4, 128)
    pos = rng.integers(0, 100000, 20)
    back = rotate(rotate(x, pos, f, 128, 0), pos, -f, 128, 0)
    a, b = (bf2f_array(v).astype(np.float64).reshape(x.shape) for v in (x, back))
    length = np.hypot(a[..., :64], a[..., 64:])
    # half a step is 2^-8 of a value at most: the first rounding moves the pair by 2^-8 of its length, the second each coordinate
    # by 2^-8 of the length and a little
    assert (np.abs(a - b) / np.concatenate([length, length], -1)).max() <= 2.0 ** -7 * (1 + 2.0 ** -8)


def test_special_values():
    """Infinities and NaN stay within their pair; the values beyond rot keep every bit; tiny and huge values."""
    x = f2bf_array(np.linspace(-2, 2, 3 * 2 * 64).astype(np.float32)).reshape(3, 2, 64)
    x[0, 0, 3], x[1, 1, 40], x[2, 0, 63], x[2, 1, 62] = 0x7F80, 0xFFC1, 0x7FA5, 0x0001
    x[1, 0, :4] = [0x7F7F, 0xFF7F, 0x0001, 0x8001]
    f, _ = freqs64(1e4, 32)
    for interleaved in (0, 1):
        got = rotate(x, [5, 6, 7], f, 32, interleaved)
        with np.errstate(invalid="ignore", over="ignore"):
            w = want(x, [5, 6, 7], f, 32, interleaved, 1.0, x)
        nan = lambda v: (v & 0x7FFF) > 0x7F80  # noqa: E731
        a, b = got[..., :32], w[..., :32]
        assert np.array_equal(nan(a), nan(b)) and np.array_equal(a[~nan(a)], b[~nan(b)])
        assert np.array_equal(got[..., 32:], x[..., 32:])


def test_many_tokens_and_frequencies_of_zero():
    rng = np.random.default_rng(4)
    m = 3000
    x = rows(rng, m, 6, 64)
    f, _ = freqs64(1e4, 64)
    f[5:] = 0.0
    pos = rng.integers(-2, 1 << 17, m)
    old = np.full_like(x, FILL)
    assert np.array_equal(rotate(x, pos, f, 64, 0), want(x, pos, f, 64, 0, 1.0, old))


def test_one_row_for_all_tokens():
    """Rows of x may be one (ldx 0)."""
    rng = np.random.default_rng(5)
    x = rows(rng, 1, 2, 128)
    f, _ = freqs64(1e4, 128)
    X, P, F, Y = Dev.of(x), Dev.of(i32([4, 5, 6])), Dev.of(f), Dev(3 * 512)
    check(step().ak_rope(X.p, 0, Y.p, 256, 3, 2, 128, P.p, F.p, 128, 0, 1.0, None))
    check(step().ak_synchronize())
    assert np.array_equal(Y.get(np.uint16, 768).reshape(3, 2, 128), want(np.repeat(x, 3, 0), np.array([4, 5, 6]), f, 128, 0, 1.0, x))


# ------------------------------------------------------------------------------------------------ into the cache
class Merged:
    """A merged projection's rows [q | k | v] and all that the calls take."""

    def __init__(self, seed, bits, m, heads, kv, dim, rot, interleaved, page, pad=0):
        rng = np.random.default_rng(seed)
        self.__dict__.update(bits=bits, m=m, heads=heads, kv=kv, dim=dim, rot=rot, interleaved=interleaved, page=page)
        self.w = (heads + 2 * kv) * dim + pad
        x = rows(rng, m, heads + 2 * kv, dim).reshape(m, -1)
        self.x = np.concatenate([x, np.full((m, pad), 0x7FC1, dtype=np.uint16)], 1)
        self.npages = (m + page - 1) // page + 2
        self.slots = rng.permutation(self.npages * page)[:m]
        self.pos = rng.integers(0, 1 << 18, m)
        if m > 6:
            self.pos[3], self.slots[5], self.slots[6] = -1, -1, self.npages * page
        self.f, _ = freqs64(1e4, rot)
        self.mag = 1.5
        self.pool = Pool(bits, page, kv, dim, self.npages, fill=0x5A)
        self.X, self.P, self.F, self.S = Dev.of(self.x), Dev.of(i32(self.pos)), Dev.of(self.f), Dev.of(i32(self.slots))

    def fused(self, Y, ldy, D, stream=None, X=None):
        h, d = self.heads, self.dim
        X = X or self.X
        return step().ak_rope_kv_write(self.bits, X.p, self.w, X.addr(2 * h * d), self.w, X.addr(2 * (h + self.kv) * d), self.w,
                                       Y.p, ldy, self.m, h, self.P.p, self.F.p, self.rot, self.interleaved, self.mag, self.S.p,
                                       D.p, self.npages, self.page, self.kv, d, stream)

    def apart(self):
        """ak_rope of q and of k, then ak_kv_write (tokens without a position: not written)."""
        h, d, kv, m = self.heads, self.dim, self.kv, self.m
        Q, K, D = Dev.of(np.full((m, h * d), FILL, dtype=np.uint16)), Dev(m * kv * d * 2), Dev.of(self.pool.mem)
        slots = Dev.of(i32(np.where(self.pos < 0, -1, self.slots)))
        turn = (self.P.p, self.F.p, self.rot, self.interleaved, self.mag, None)
        check(step().ak_rope(self.X.p, self.w, Q.p, h * d, m, h, d, *turn))
        check(step().ak_rope(self.X.addr(2 * h * d), self.w, K.p, kv * d, m, kv, d, *turn))
        check(step().ak_kv_write(self.bits, K.p, self.X.addr(2 * (h + kv) * d), m, kv * d, self.w, slots.p, D.p, self.npages,
                                 self.page, kv, d, None))
        check(step().ak_synchronize())
        return Q.get(np.uint16, m * h * d), D.get(np.uint8, self.pool.mem.size)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("m,heads,kv,dim,rot,interleaved,page", [
    (1, 40, 8, 128, 128, 0, 16), (48, 40, 8, 128, 128, 1, 16), (7, 5, 1, 128, 64, 0, 32), (19, 4, 2, 64, 64, 0, 256),
    (33, 3, 3, 256, 256, 0, 64), (20, 8, 4, 64, 36, 1, 16), (20, 8, 4, 256, 100, 0, 16), (300, 2, 1, 64, 64, 1, 128)])
def test_into_the_cache_as_the_calls_apart(bits, m, heads, kv, dim, rot, interleaved, page):
    a = Merged(m + dim + bits, bits, m, heads, kv, dim, rot, interleaved, page, pad=8 * (m % 2))
    Y, D = Dev.of(np.full((m, heads * dim), FILL, dtype=np.uint16)), Dev.of(a.pool.mem)
    check(a.fused(Y, heads * dim, D))
    check(step().ak_synchronize())
    q, pool = a.apart()
    assert np.array_equal(Y.get(np.uint16, m * heads * dim), q)
    assert np.array_equal(D.get(np.uint8, a.pool.mem.size), pool)
    # and by the definition
    x = a.x[:, :(heads + 2 * kv) * dim].reshape(m, heads + 2 * kv, dim)
    k = want(x[:, heads:heads + kv], a.pos, a.f, rot, interleaved, a.mag, x[:, heads:heads + kv])
    ok = (a.pos >= 0) & (a.slots >= 0) & (a.slots < a.npages * page)
    a.pool.put(a.slots[ok], k[ok], x[ok, heads + kv:])
    assert np.array_equal(pool, a.pool.mem.ravel())


def test_queries_in_place_and_captured():
    a = Merged(8, 8, 30, 8, 2, 128, 128, 0, 16)
    want_q, want_pool = a.apart()
    X, D = Dev.of(a.x), Dev.of(a.pool.mem)
    check(a.fused(X, a.w, D, X=X))
    check(step().ak_synchronize())
    got = X.get(np.uint16, a.x.size).reshape(a.x.shape)
    q = np.where((a.pos < 0)[:, None], a.x[:, :1024], want_q.reshape(30, 1024))
    assert np.array_equal(got[:, :1024], q) and np.array_equal(got[:, 1024:], a.x[:, 1024:])
    assert np.array_equal(D.get(np.uint8, a.pool.mem.size), want_pool)
    s, Y, D = Stream(), Dev.of(np.full((30, 1024), FILL, dtype=np.uint16)), Dev.of(a.pool.mem)
    g = Graph(s, lambda st: a.fused(Y, 1024, D, st))
    for _ in range(3):
        g.launch()
        s.sync()
        assert np.array_equal(Y.get(np.uint16, 30 * 1024), want_q) and np.array_equal(D.get(np.uint8, a.pool.mem.size), want_pool)


@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("rot", [64, 60])
def test_results_below_the_normal_numbers_are_rounded_once(rot, interleaved):
    """Products a little above, at and below the middles between bf16's numbers below 2^-126, which fp32 has not the bits to tell."""
    rng = np.random.default_rng(9)
    x = np.zeros((24, 4, 64), dtype=np.uint16)
    x[:] = f2bf_array((rng.integers(1, 256, x.size) * 2.0 ** rng.integers(-18, 2, x.size)).astype(np.float32)).reshape(x.shape)
    x |= (rng.random(x.shape) < 0.5).astype(np.uint16) << 15
    f, _ = freqs64(1e4, rot)
    for part in (1.0, 1 + 2.0 ** -23, 1 - 2.0 ** -24):
        mag = np.float32(2.0 ** -125 * part)
        for pos in (np.zeros(24, dtype=int), rng.integers(0, 1000, 24)):
            got = rotate(x, pos, f, rot, interleaved, float(mag))
            w = want(x, pos, f, rot, interleaved, mag, x)
            assert np.array_equal(got, w), (part, (got != w).sum())


# ------------------------------------------------------------------------------------------------ prompts
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("m,heads,dim,rot,interleaved", [(530, 48, 128, 128, 0), (530, 48, 128, 120, 0), (530, 48, 128, 64, 1),
                                                         (517, 20, 256, 250, 0), (520, 40, 80, 80, 1), (8500, 6, 64, 64, 0),
                                                         (9800, 5, 64, 36, 0), (8500, 6, 64, 64, 1)])
def test_prompts(m, heads, dim, rot, interleaved, in_place):
    """512 workgroups and more: each turns several times, the next heads' values on their way before these are stored."""
    rng = np.random.default_rng(m + dim + rot)
    x = rows(rng, m, heads, dim)
    pos = rng.integers(-1, 1 << 20, m)
    f, _ = freqs64(1e4, rot)
    got = rotate(x, pos, f, rot, interleaved, 0.75, pad_in=8 * (heads % 3), pad_out=24, in_place=in_place)
    assert np.array_equal(got, want(x, pos, f, rot, interleaved, np.float32(0.75), x if in_place else np.full_like(x, FILL)))


PROMPTS = [(530, 40, 8, 128, 128, 0, 16), (530, 40, 8, 128, 128, 1, 64), (530, 40, 8, 128, 100, 0, 256), (520, 16, 4, 256, 256, 0, 32),
           (3100, 9, 3, 64, 64, 0, 128), (1030, 30, 9, 64, 44, 0, 16)]


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("m,heads,kv,dim,rot,interleaved,page", PROMPTS)
def test_prompts_into_the_cache(bits, m, heads, kv, dim, rot, interleaved, page):
    test_into_the_cache_as_the_calls_apart(bits, m, heads, kv, dim, rot, interleaved, page)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("m,heads,kv,dim,rot,interleaved,page", PROMPTS)
def test_prompts_into_the_cache_with_queries_in_place(bits, m, heads, kv, dim, rot, interleaved, page):
    a = Merged(m + bits, bits, m, heads, kv, dim, rot, interleaved, page, pad=8)
    q, pool = a.apart()
    X, D, w = Dev.of(a.x), Dev.of(a.pool.mem), heads * dim
    check(a.fused(X, a.w, D, X=X))
    check(step().ak_synchronize())
    got = X.get(np.uint16, a.x.size).reshape(a.x.shape)
    assert np.array_equal(got[:, :w], np.where((a.pos < 0)[:, None], a.x[:, :w], q.reshape(m, w)))
    assert np.array_equal(got[:, w:], a.x[:, w:]) and np.array_equal(D.get(np.uint8, a.pool.mem.size), pool)
