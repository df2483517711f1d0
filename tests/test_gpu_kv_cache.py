"""The paged key-value cache (ak_kv_write, ak_kv_read) on the GPU, bit for bit against the definition in 64 bits."""
import ctypes

import numpy as np
import pytest

from _lib import check, Dev, f2bf_array, bf2f_array
from _ops import ops, Pool, held, bf16_rn, page_bytes

pytestmark = pytest.mark.gpu


def rows(rng, m, heads, dim, spread=2.0):
    x = rng.standard_normal((m, heads, dim)) * np.exp(spread * rng.standard_normal((m, heads, 1)))
    return f2bf_array(x.astype(np.float32).ravel()).reshape(m, heads, dim)


def write(pool, dev, slots, k, v, ldk=None, ldv=None, stream=None):
    m, w = len(slots), pool.heads * pool.dim
    K, V, S = Dev.of(k), Dev.of(v), Dev.of(np.asarray(slots, dtype=np.int32))
    check(ops().ak_kv_write(pool.bits, K.p, V.p, m, ldk or w, ldv or w, S.p, dev.p, pool.npages, pool.page, pool.heads,
                            pool.dim, stream), "ak_kv_write")
    check(ops().ak_synchronize())


def read(pool, dev, slots, pad=0):
    m, w = len(slots), pool.heads * pool.dim
    ld = w + pad
    K, V = (Dev.of(np.full(m * ld, 0x1234, dtype=np.uint16)) for _ in range(2))
    S = Dev.of(np.asarray(slots, dtype=np.int32))
    check(ops().ak_kv_read(pool.bits, dev.p, pool.npages, pool.page, pool.heads, pool.dim, S.p, m, K.p, V.p, ld, ld, None),
          "ak_kv_read")
    check(ops().ak_synchronize())
    out = []
    for X in (K, V):
        a = X.get(np.uint16, m * ld).reshape(m, ld)
        assert (a[:, w:] == 0x1234).all()  # between the rows
        out.append(a[:, :w].reshape(m, pool.heads, pool.dim))
    return out


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("m,heads,dim,page", [(1, 8, 128, 16), (37, 3, 64, 32), (130, 8, 128, 64), (19, 1, 256, 256),
                                              (700, 2, 128, 16)])
def test_write_and_read_back(bits, m, heads, dim, page):
    rng = np.random.default_rng(m + bits)
    pool = Pool(bits, page, heads, dim, (m + page - 1) // page + 3, fill=0x5A)
    k, v = rows(rng, m, heads, dim), rows(rng, m, heads, dim)
    slots = rng.permutation(pool.npages * page)[:m]
    dev = Dev.of(pool.mem)
    write(pool, dev, slots, k, v)
    pool.put(slots, k, v)
    got = dev.get(np.uint8, pool.mem.size).reshape(pool.mem.shape)
    assert np.array_equal(got, pool.mem)  # the layout, and nothing else touched
    for x, y in zip((k, v), read(pool, dev, slots, pad=8)):
        assert np.array_equal(y, bf16_rn(held(x, bits)))


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_special_rows(bits):
    """Zeros, halves (exact ties), one large value, the smallest and largest magnitudes, and non-finite rows."""
    heads, dim, page = 2, 128, 16
    rng = np.random.default_rng(5)
    x = rows(rng, 10, heads, dim)
    x[0] = 0
    x[1] = 0x8000
    q = 127 if bits == 8 else 7
    x[2] = f2bf_array((np.arange(heads * dim) % (2 * q) / 2 - q / 2).astype(np.float32)).reshape(heads, dim)
    x[2, :, 0] = f2bf_array(np.array([q], dtype=np.float32))[0]  # scale 1: every other value is a tie
    x[3, 0, 5] = 0x7F7F  # the largest finite
    x[4] = x[4] & 0x80FF  # subnormals and the smallest normals
    x[5] = 0x0001
    x[6, 0, 3] = 0x7F80
    x[7, 1, 77] = 0xFFC1
    x[8, 1, 127] = 0xFF80
    x[9] = f2bf_array((3.0 * (np.arange(heads * dim) % 11 - 5)).astype(np.float32)).reshape(heads, dim)
    pool = Pool(bits, page, heads, dim, 2, fill=0)
    slots = np.arange(10)[::-1].copy()
    dev = Dev.of(pool.mem)
    write(pool, dev, slots, x, x)
    pool.put(slots, x, x)
    got = dev.get(np.uint8, pool.mem.size).reshape(pool.mem.shape)
    assert np.array_equal(got, pool.mem)
    for y in read(pool, dev, slots):
        if bits == 16:
            assert np.array_equal(y, x)
            continue
        want = held(x, bits)
        nan = np.isnan(want)
        assert np.isnan(bf2f_array(y[nan])).all() and nan.sum() == 3 * dim
        assert np.array_equal(y[~nan], bf16_rn(want[~nan]))


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_strided_rows_of_a_merged_projection(bits):
    """Keys and values as slices of one q, k, v row."""
    m, heads, dim, page, qw = 9, 4, 128, 16, 640
    rng = np.random.default_rng(8)
    w = heads * dim
    qkv = rows(rng, m, 1, qw + 2 * w + 8)[:, 0]
    X, S = Dev.of(qkv), Dev.of(np.arange(m, dtype=np.int32) * 3)
    pool = Pool(bits, page, heads, dim, 2, fill=0)
    dev = Dev.of(pool.mem)
    ld = qkv.shape[1]
    check(ops().ak_kv_write(bits, X.addr(2 * qw), X.addr(2 * (qw + w)), m, ld, ld, S.p, dev.p, 2, page, heads, dim, None))
    check(ops().ak_synchronize())
    pool.put(np.arange(m) * 3, np.ascontiguousarray(qkv[:, qw:qw + w]).reshape(m, heads, dim),
             np.ascontiguousarray(qkv[:, qw + w:qw + 2 * w]).reshape(m, heads, dim))
    assert np.array_equal(dev.get(np.uint8, pool.mem.size).reshape(pool.mem.shape), pool.mem)


@pytest.mark.parametrize("bits", [16, 4])
def test_slots_outside_the_pool(bits):
    heads, dim, page, npages = 2, 64, 16, 3
    rng = np.random.default_rng(1)
    k, v = rows(rng, 5, heads, dim), rows(rng, 5, heads, dim)
    pool = Pool(bits, page, heads, dim, npages, fill=0x11)
    dev = Dev.of(pool.mem)
    slots = [-1, 47, 48, 2 ** 31 - 1, -2 ** 31]
    write(pool, dev, slots, k, v)
    pool.put([47], k[1:2], v[1:2])
    assert np.array_equal(dev.get(np.uint8, pool.mem.size).reshape(pool.mem.shape), pool.mem)
    a, b = read(pool, dev, slots)
    for t in (0, 2, 3, 4):
        assert not a[t].any() and not b[t].any()
    assert np.array_equal(a[1], bf16_rn(held(k[1], bits)))


def test_pool_past_4_gib():
    """Pages whose byte offsets need more than 32 bits."""
    bits, page, heads, dim = 16, 256, 8, 128
    pb = page_bytes(bits, page, heads, dim)
    npages = (5 << 30) // pb
    dev = Dev(npages * pb)
    rng = np.random.default_rng(2)
    k, v = rows(rng, 3, heads, dim), rows(rng, 3, heads, dim)
    top = npages * page - 1
    pool = Pool(bits, page, heads, dim, 1)
    pool.npages = npages
    slots = [top, top - page, top // 2]
    write(pool, dev, slots, k, v)
    a, b = read(pool, dev, slots)
    assert np.array_equal(a, k) and np.array_equal(b, v)


def test_no_tokens():
    assert ops().ak_kv_write(8, None, None, 0, 0, 0, None, None, 1, 16, 1, 64, None) == 0
    assert ops().ak_kv_read(8, None, 1, 16, 1, 64, None, 0, None, None, 0, 0, None) == 0
