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
