"""Paged attention and the append to its cache where they can go wrong beside the sizes and masks of
test_gpu_encoder_ops.py, whose helpers and count of roundings are used here."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_encoder_ops import BF16, F32, U, Paged, attention_want, close, g, randn  # noqa: E402, F401


# --- a row's maximum that keeps rising ------------------------------------------------------------

def rising(b, heads, rise, seed):
    """Queries and a cache whose scores rise by `rise` (of a base-2 exponent, for the first head of a group; by one and a
    half times that for the second; they fall for a third) from each 128 keys to the next, over values that shrink
    as much, so that all keys count alike in the first head's output and the last ones in the second's."""
    D = b.k.shape[3]
    along = torch.full((D,), D ** -0.5, device="cuda")
    gain = torch.tensor([8.0, 12.0, -8.0], device="cuda")[torch.arange(heads, device="cuda") % 3]
    q = (gain[:, None] * along + randn(b.rows, heads, D, seed=seed, scale=0.2)).to(BF16)
    step = rise * math.log(2.0) / (8.0 * D ** -0.5)
    for s, (n, p) in enumerate(zip(b.new, b.past)):
        at = b.places(s, 0, n + p)
        tile = torch.arange(n + p, device="cuda")[:, None, None] // 128
        hk = b.k.shape[2]
        b.k[at] = (tile * step * along + randn(n + p, hk, D, seed=seed + 2 * s + 1, scale=0.2)).to(BF16)
        b.v[at] = (randn(n + p, hk, D, seed=seed + 2 * s + 2) * torch.exp2(-rise * tile)).to(BF16)
    return q


@pytest.mark.parametrize("D", [64, 72, 128, 136, 192, 256])
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("new, past", [([70] * 40, [700] * 40), ([150], [620])])
@pytest.mark.parametrize("window", [0, 300])
def test_a_maximum_that_rises_from_tile_to_tile(g, D, page, new, past, window):
    """Every key tile moves every row's reference over an output that is not zero. Two roundings of the probabilities
    count, of the numerator's and of the divisor's; the other terms are attention_want's."""
    b = Paged(new, past, 2, D, page, BF16, seed=D, fill=0.0)
    q = rising(b, 6, 9.0, seed=D + window % 7)
    want, tol = attention_want(b, q, D ** -0.5, window, 0, 0.0)
    first = None
    for _ in range(3):
        got = g.paged_attention_device(q, b.k, b.v, *b.args(), b.max_kv, window=window)
        g.synchronize()
        close(got, want, tol + want.abs() * 2 * U[BF16], (D, window))
        assert first is None or torch.equal(got, first)
        first = got


# --- few rows -------------------------------------------------------------------------------------

@pytest.mark.parametrize("D, G", [(64, 4), (128, 8), (256, 2), (136, 1)])
@pytest.mark.parametrize("page", [1, 5, 24, 16])
def test_single_tokens_over_any_pages_repeat_themselves(g, D, G, page):
    """One warp to a group of keys: what its lanes copy and look up for one another is there before it is read. The same
    bits each time, beside other work, and the 64-bit result."""
    b = Paged([1, 2, 1, 1], [3000, 130, 15, 700], 2, D, page, BF16, seed=D + page).fill(3)
    q = randn(b.rows, 2 * G, D, seed=4, dtype=BF16, scale=2.0)
    want, tol = attention_want(b, q, D ** -0.5, 0, 0, 0.0)
    got = [g.paged_attention_device(q, b.k, b.v, *b.args(), b.max_kv) for _ in range(20)]
    g.synchronize()
    close(got[0], want, tol + want.abs() * 2 * U[BF16])
    assert all(torch.equal(x, got[0]) for x in got[1:])
