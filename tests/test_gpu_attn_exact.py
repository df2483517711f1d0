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
