"""Draws whose uniform number falls between two tokens' weights, closer than the sums' last bit, on the GPU.

At this temperature log2(e) / T rounds to 1, so a token whose logit is -n weighs 2^-n.  Token A's weight is 3 * 2^-54 and B's 1.
In 64 bits their sum is 1 + 2^-52, from which B's weight leaves 2^-52: more than A's.  u = 0.875 * 2^-52 lies in that gap, beyond
A's weight, so the definition draws B."""
import numpy as np
import pytest

from _lib import f2bf_array
from test_gpu_spec_verify import run

pytestmark = pytest.mark.gpu

HEAT = np.float32(1.44269504088896340736)
GAP = 0.875 * 2.0 ** -52
OFF, TOP, LOW = 0xFF80, 0x0000, f2bf_array(np.array([-54.0], dtype=np.float32))[0]


def row(vocab, low, top):
    x = np.full(vocab, OFF, dtype=np.uint16)
    x[low], x[top] = LOW, TOP
    return x


# three tokens of A and one of B: in two chunks of a row, in two threads of a chunk, two waves, in chunks of two waves
PLACES = [(10000, [5, 6, 7], 4096 + 100), (500, [3, 4, 5], 70), (500, [3, 4, 5], 16), (4096, [1021, 1022, 1023], 1024),
          (66 * 4096, [64 * 4096 - 3, 64 * 4096 - 2, 64 * 4096 - 1], 64 * 4096)]


@pytest.mark.parametrize("vocab,low,top", PLACES)
def test_draw_between_two_weights(vocab, low, top):
    target = row(vocab, low, top).reshape(1, 1, vocab)
    tok, acc, lp = run(target, None, None, None, [[GAP]], [HEAT], 1, 0, vocab)
    assert tok[0, 0] == top and abs(lp[0, 0]) < 1e-6


@pytest.mark.parametrize("vocab,low,top", PLACES)
@pytest.mark.parametrize("drafted", [True, False])
def test_draw_after_a_rejected_draft(vocab, low, top, drafted):
    """The rejected draft itself, as heavy as B and before it, is not what is emitted."""
    x = low[-1] + 1 if low[-1] + 1 != top else low[0] - 1
    target = row(vocab, low, top)
    target[x] = TOP
    draft = np.full(vocab, OFF, dtype=np.uint16)
    draft[x] = TOP
    tok, acc, _ = run(np.stack([target, target])[None], draft[None, None] if drafted else None, [[x]], None, [[0.9, GAP]],
                      [HEAT], 1, 1, vocab)
    assert acc[0] == 0 and tok[0].tolist() == [top, -1]


@pytest.mark.parametrize("vocab,low,top", PLACES)
def test_draws_beside_the_edge(vocab, low, top):
    """Below A's weight its tokens are drawn, at u = 0 the first of them."""
    target = row(vocab, low, top)
    u = np.array([0.0, 0.2, 0.3, 0.6, 0.9, 1.5, 2.0 ** 30, 0.5 * 2.0 ** 54]) * 2.0 ** -54 * [1, 1, 1, 3, 3, 3, 1, 1]
    want = [low[0], low[0], low[0], low[1], low[2], top, top, top]
    b = len(u)
    tok, _, _ = run(np.broadcast_to(target, (b, 1, vocab)), None, None, None, u[:, None], np.full(b, HEAT), b, 0, vocab)
    assert tok.ravel().tolist() == want
