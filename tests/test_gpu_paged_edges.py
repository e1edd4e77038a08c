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


# --- soft caps of any size ------------------------------------------------------------------------

def capped_want(b, q, scale, cap):
    """attention_want with an error of the cap that does not grow with it. The cheap form, used up to a cap of 1024, is off
    by at most 3.5 2^-23 of the base-2 exponent's cap (the exponential's, the sum's and the quotient's roundings, twice, and the
    last one's): 2^-21 of the cap in the score. Any other is off by that at a quarter of the cap or more, 2^-19 of the
    score, or by a few roundings of the score (attention_want's eight)."""
    heads, hk, D = q.shape[1], b.k.shape[2], q.shape[2]
    want, tol = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    row = 0
    for s, (n, p) in enumerate(zip(b.new, b.past)):
        at = b.places(s, 0, n + p)
        k, v = (t[at].double().repeat_interleave(heads // hk, 1).transpose(0, 1) for t in (b.k, b.v))
        qq = q[row:row + n].double().transpose(0, 1)
        t = cap * torch.tanh(qq @ k.transpose(1, 2) * scale / cap)
        size = qq.abs() @ k.abs().transpose(1, 2) * scale
        hidden = torch.arange(n + p, device="cuda") > torch.arange(p, p + n, device="cuda")[:, None]
        prob = torch.softmax(t.masked_fill(hidden, -math.inf), -1)
        e = (D / 8 + 16) * 2.0 ** -24 * size + (2.0 ** -21 * cap if cap <= 1024 else 2.0 ** -19 * t.abs()) + 2.0 ** -20
        e = e.masked_fill(hidden, 0).amax(-1, keepdim=True)
        p_round = U[BF16] if q.dtype == BF16 else 0.0
        want[row:row + n] = (prob @ v).transpose(0, 1)
        tol[row:row + n] = ((prob @ v.abs()) * (2 * e * 1.01 + p_round + (n + p) / 16 * 2.0 ** -24)).transpose(0, 1)
        row += n
    return want, tol + want.abs() * (2 if q.dtype == BF16 else 1) * U[q.dtype]


@pytest.mark.parametrize("cap", [0.5, 50.0, 1000.0, 1025.0, 1e4, 1e5, 1e6, 1e7, 1e30])
@pytest.mark.parametrize("dtype, D", [(BF16, 64), (BF16, 128), (BF16, 256), (F32, 64)])
@pytest.mark.parametrize("new, past", [([1, 1], [40, 600]), ([150, 9], [70, 300])])
def test_caps_large_against_the_scores(g, cap, dtype, D, new, past):
    b = Paged(new, past, 2, D, 16, dtype, seed=D).fill(8)
    q = randn(b.rows, 4, D, seed=9, dtype=dtype, scale=3.0)
    want, tol = capped_want(b, q, D ** -0.5, cap)
    got = g.paged_attention_device(q, b.k, b.v, *b.args(), b.max_kv, softcap=cap)
    g.synchronize()
    close(got, want, tol)


# --- the append leaves out what attention leaves out ----------------------------------------------

@pytest.mark.parametrize("starts, lens, max_new, max_kv, left_out", [
    ([0, 2, 5], [8, 5], 2, 64, [1]),        # more new tokens than max_new
    ([0, 2, 5], [8, 2], 3, 64, [1]),        # fewer tokens than new ones: none of them, not the first alone
    ([0, 2, 5], [1, 5], 3, 64, [0]),
    ([0, 2, 5], [8, 5], 3, 7, [0]),         # longer than max_kv
    ([-1, 2, 5], [8, 5], 3, 64, [0]),       # begins in front of the rows
    ([0, 2, 7], [8, 5], 9, 64, [1]),        # ends behind them
    ([0, 2, 5, 8], [8, 5, 3], 3, 64, [2]),  # lies behind them
    ([0, 2, 5, 5], [8, 5, -1], 3, 64, []),  # no new token, and a length that cannot be
])
@pytest.mark.parametrize("turned", [False, True])
def test_append_leaves_out_whole_sequences(g, starts, lens, max_new, max_kv, left_out, turned):
    """A sequence out of bounds is recorded, and none of its rows is written, as the header says."""
    b = Paged([2, 3], [6, 2], 2, 64, 4, BF16, seed=1, fill=7.0)
    table = torch.cat([b.table, b.table[:1]])[:len(lens)]
    q, k, v = (randn(5, n, 64, seed=i, dtype=BF16) for i, n in enumerate((4, 2, 2)))
    freq = torch.full((32,), 0.5, dtype=torch.float64, device="cuda") if turned else None
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    keep = q.clone()
    out = g.rotary_append_device(q, k, v, freq, b.k, b.v, i32(starts), i32(lens), table, max_new, inplace=True, max_kv=max_kv)
    with pytest.raises(ValueError, match="kv_len|row_start"):
        g.synchronize()
    g.synchronize()  # once
    written = 0
    for s, (n, p) in enumerate(zip(b.new, b.past)):
        rows = slice(2 * s, 2 * s + n)
        if s in left_out:
            assert torch.equal(out[rows], keep[rows])
            continue
        assert torch.equal(b.v[b.places(s, p, p + n)], v[rows])
        assert not turned or not torch.equal(out[rows], keep[rows])
        written += n
    assert (b.v != 7.0).any(-1).any(-1).sum().item() == written


@pytest.mark.parametrize("dtype, max_new", [(BF16, 1), (BF16, 200), (F32, 1)])
def test_nothing_cached(g, dtype, max_new):
    """A padded batch whose sequences are all empty, max_new its fixed bound: nothing is written or recorded. A token with
    a length of 0 is recorded."""
    b = Paged([0, 0, 0], [0, 0, 0], 2, 64, 16, dtype, seed=0)
    q = randn(4, 4, 64, seed=1, dtype=dtype)
    out = torch.full_like(q, 3.0)
    g.paged_attention_device(q, b.k, b.v, b.row_start, b.kv_len, b.table, max_new, 0, out=out)
    g.synchronize()
    b.row_start[1:] = 1
    g.paged_attention_device(q, b.k, b.v, b.row_start, b.kv_len, b.table, max_new, 0, out=out)
    with pytest.raises(ValueError, match="kv_len"):
        g.synchronize()
    assert (out == 3.0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("max_kv", [0, 64])
def test_no_new_tokens_allowed(g, dtype, max_kv):
    """max_new 0: sequences without new tokens are left alone, others are recorded and left out, by both operators."""
    b = Paged([2, 0], [6, 2], 2, 64, 16, dtype, seed=0, fill=7.0)
    q, k = randn(2, 4, 64, seed=1, dtype=dtype), randn(2, 2, 64, seed=2, dtype=dtype)
    out = torch.full_like(q, 3.0)
    for starts in ([0, 0, 0], [0, 2, 2]):
        row_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
        for call in (lambda: g.paged_attention_device(q, b.k, b.v, row_start, b.kv_len, b.table, 0, max_kv, out=out),
                     lambda: g.rotary_append_device(None, k, k, None, b.k, b.v, row_start, b.kv_len, b.table, 0, max_kv=max_kv)):
            call()
            if starts[1] or max_kv == 0:
                # (the second sequence's length is above a max_kv of 0: either of the two may be recorded first)
                with pytest.raises(ValueError, match="row_start" if max_kv else "row_start|kv_len"):
                    g.synchronize()
            g.synchronize()
    assert (out == 3.0).all() and (b.k == 7.0).all() and (b.v == 7.0).all()


# --- a chunk and single tokens in one batch -------------------------------------------------------

@pytest.mark.parametrize("dtype, D", [(BF16, 64), (BF16, 128), (BF16, 256), (F32, 64)])
@pytest.mark.parametrize("new, past", [([300, 1], [10, 3000]), ([1, 1, 40, 1], [2500, 900, 0, 17]), ([1, 130, 1], [4000, 70, 1300])])
@pytest.mark.parametrize("window, sinks", [(0, 0), (700, 5)])
@pytest.mark.parametrize("page", [16, 24])
def test_chunks_and_single_tokens_in_one_batch(g, dtype, D, new, past, window, sinks, page):
    """One launch for all, whose tiles and splits are the longest ones': each row as it would be alone."""
    b = Paged(new, past, 2, D, page, dtype, seed=D).fill(3)
    q = randn(b.rows, 4, D, seed=9, dtype=dtype, scale=2.0)
    got = g.paged_attention_device(q, b.k, b.v, *b.args(), b.max_kv, window=window, sinks=sinks)
    g.synchronize()
    want, tol = attention_want(b, q, D ** -0.5, window, sinks, 0.0)
    close(got, want, tol + want.abs() * 2 * U[dtype])


def test_a_batch_in_two_calls(g):
    """Chunks and single tokens of one batch in a call each, over their parts of the same arrays: together all rows."""
    b = Paged([200, 30, 1, 1, 1], [10, 40, 3000, 500, 0], 2, 128, 16, BF16, seed=2, trailing=2).fill(3)
    q = randn(b.rows, 8, 128, seed=9, dtype=BF16, scale=2.0)
    out = torch.full_like(q, 5.0)
    for lo, hi, max_new, max_kv in ((0, 2, 200, 210), (2, 5, 1, 3001)):
        g.paged_attention_device(q, b.k, b.v, b.row_start[lo:hi + 1], b.kv_len[lo:hi], b.table[lo:hi], max_new, max_kv, out=out)
    g.synchronize()
    want, tol = attention_want(b, q, 128 ** -0.5, 0, 0, 0.0)
    close(out[:-2], want[:-2], (tol + want.abs() * 2 * U[BF16])[:-2])
    assert (out[-2:] == 5.0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_row_start_that_descends(g, dtype):
    """Recorded by both operators. The append writes no row at a place that is not its sequence's: a row is looked up by
    the ends, and the last sequence (rows 4 and 5) is not the one that holds rows 7 and 8."""
    b = Paged([2, 7, 0, 2], [6, 2, 3, 50], 2, 64, 16, dtype, seed=1, fill=7.0)
    starts = torch.tensor([0, 2, 9, 4, 6], dtype=torch.int32, device="cuda")
    q, k = randn(10, 4, 64, seed=1, dtype=dtype), randn(10, 2, 64, seed=2, dtype=dtype)
    out = torch.full_like(q, 3.0)
    g.rotary_append_device(None, k, k, None, b.k, b.v, starts, b.kv_len, b.table, 7, max_kv=64)
    with pytest.raises(ValueError, match="row_start"):
        g.synchronize()
    assert torch.equal(b.v[b.places(0, 6, 8)], k[:2])
    page, slot = b.places(3, 0, 64)  # the last sequence's page: its own two tokens at most
    kept = (b.v[page, slot] == 7.0).flatten(1).all(1)
    assert kept[:50].all() and kept[52:].all()
    b.v.fill_(0.0)
    b.k.fill_(0.0)
    g.paged_attention_device(q, b.k, b.v, starts, b.kv_len, b.table, 7, 64, out=out)
    with pytest.raises(ValueError, match="row_start"):
        g.synchronize()
    assert (out[9:] == 3.0).all()
