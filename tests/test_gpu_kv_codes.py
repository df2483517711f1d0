"""Codes of the cache (ak_kv_write) are those of exact division: every bf16 mantissa by every mantissa of a row's largest value, over
the exponents whose codes are not all zero, in ranges of magnitude up to both ends of bf16, against 64 bits."""
import numpy as np
import pytest

from _lib import check, Dev
from _ops import ops, page_bytes, quantise

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("exponent", [254, 250, 127, 64, 63, 60, 20, 10, 8, 5])
def test_every_mantissa(bits, exponent):
    """exponent: of the largest values, as bf16 holds it."""
    dim, page = 128, 256
    mantissas = np.arange(128, dtype=np.int64)
    down = np.arange(10 if bits == 8 else 6, dtype=np.int64)
    x = ((np.maximum(exponent - down, 0)[:, None] << 7) + mantissas).ravel()  # every value but the sign
    x = np.concatenate([x, np.zeros(-len(x) % (dim - 1), dtype=np.int64)])
    each = len(x) // (dim - 1)  # rows of a largest value
    rows = np.empty((128, each, dim), dtype=np.uint16)
    most = (exponent << 7) + mantissas
    rows[..., 0] = most[:, None]
    rows[..., 1:] = np.minimum(x.reshape(1, each, dim - 1), most[:, None, None])
    rows[:, :, 1::2] |= 0x8000
    rows = rows.reshape(-1, 1, dim)
    m = len(rows)
    npages = (m + page - 1) // page
    K, V, S = Dev.of(rows), Dev.of(rows[::-1].copy()), Dev.of(np.arange(m, dtype=np.int32))
    pb = page_bytes(bits, page, 1, dim)
    P = Dev.of(np.zeros((npages, pb), dtype=np.uint8))
    check(ops().ak_kv_write(bits, K.p, V.p, m, dim, dim, S.p, P.p, npages, page, 1, dim, None))
    check(ops().ak_synchronize())
    mem = P.get(np.uint8, npages * pb).reshape(npages, pb)
    rb = dim * bits // 8
    held = mem[:, :2 * page * rb].reshape(npages, 2, page, rb)
    scales = np.ascontiguousarray(mem[:, 2 * page * rb:2 * page * rb + 4 * page]).view(np.uint16).reshape(npages * page, 2)
    codes, s = quantise(rows[:, 0], bits)
    raw = codes if bits == 8 else codes[:, 0::2] | (codes[:, 1::2] << 4)
    for part in range(2):
        got = held[:, part].reshape(npages * page, rb)[:m]
        assert np.array_equal(got, raw if part == 0 else raw[::-1])
        assert np.array_equal(scales[:m, part], s if part == 0 else s[::-1])
