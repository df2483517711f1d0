"""The comparison of attention with 64 bits sees a lost or doubled token, a chunk, a part and coarser weights (CPU)."""
import numpy as np
import pytest

from _attn import Scene, bf16
from _lib import bf2f_array


def outputs(s, drop=()):
    """What an exact attention without the tokens `drop` gives, rounded."""
    for i in range(s.b):
        s.present[i][list(drop)] = False
    y, _, lse, _ = s.expect()
    for i in range(s.b):
        s.present[i][list(drop)] = True
    return bf16(y), lse.astype(np.float32)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("n", [300, 513, 1024, 1025, 5003, 17000])
def test_lost_tokens_are_seen(bits, n):
    s = Scene(1, bits, 32, 2, 1, 64, [n], [1], sharp=0.02)
    s.compare(*outputs(s))
    for drop in ([0], [n - 1], [n // 2], [128], [127], range(16, 32), range(64, 128), range(128, 256)):
        with pytest.raises(AssertionError):
            s.compare(*outputs(s, drop))


@pytest.mark.parametrize("bits,keep", [(16, 8), (8, 8), (4, 8), (8, 11), (4, 11)])
def test_coarser_weights_are_seen(bits, keep):
    """Weights of 8 bits (bf16) or 11 (f16) beside the values."""
    s = Scene(2, bits, 16, 8, 2, 64, list(range(2, 40)), [1] * 38, sharp=0.05)
    wy, _, wl, _ = s.expect()
    y = np.zeros_like(wy)
    from _attn import Held
    q = bf2f_array(s.q).astype(np.float64)
    for i in range(s.b):
        k, v = Held(s.k[i], bits).x, Held(s.v[i], bits)
        unit = 1 if bits == 16 else np.abs(v.most).max(-1) / (255 if bits == 8 else 15)  # codes: the scale is in the weight
        for a in range(8):
            z = k[:, a // 4] @ q[i, a] * s.scale
            p = np.exp(z - z.max())
            w = p * (unit if bits == 16 else unit[:, a // 4])
            f, e = np.frexp(w)
            w = np.ldexp(np.round(f * 2.0 ** keep), e - keep)
            y[i, a] = (w / (1 if bits == 16 else unit[:, a // 4])) @ v.x[:, a // 4] / p.sum()
    s.compare(bf16(wy), wl.astype(np.float32))
    with pytest.raises(AssertionError):
        s.compare(bf16(y), wl.astype(np.float32))
