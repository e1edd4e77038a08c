"""The text encoder's operators on the GPU against plain restatements in 64 bits.

Tolerances count roundings. A value rounded to type t is off by at most half a step, u(t) =
finfo(t).eps / 2 relative (bf16 2^-8, e4m3 2^-4, fp32 2^-24). Sums of n fp32 terms are off by at
most n 2^-24 of the sum of their magnitudes; the kernels' trees do better, and n here is what a
thread adds up in sequence."""
import ctypes
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float8_e4m3fn: 2.0 ** -4}
vp = ctypes.c_void_p
F32, BF16, E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def g():
    from sana_b200 import SanaCuda
    g = SanaCuda(0)
    g.set_stream(1)  # CUDA's legacy stream, torch's default
    yield g
    g.close()


def randn(*shape, seed, dtype=F32, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def close(got, want, tol, what=""):
    """Every element within its tolerance; where the wanted value is not finite, the same value."""
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine), what
    assert torch.equal(torch.nan_to_num(got[~fine]), torch.nan_to_num(want[~fine])), what
    off = (got - want).abs()[fine] - (tol if isinstance(tol, float) else tol.expand_as(want)[fine])
    assert off.numel() == 0 or off.max().item() <= 0, (what, off.max().item())


# --- residual norm -----------------------------------------------------------------------------

def norm_want(x, r, w, offset, eps):
    h = x.double() if r is None else (x.double() + r.double()).to(r.dtype).double()
    n = h / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    return h, n if w is None else n * (w.double() + offset)


# y's relative error before its own rounding: the sum of squares (each thread's <= 16 elements, then 10
# halvings) 30 u, halved by the root; division, root, two products and the weight's sum 6 u more
NORM_U = (15 + 6) * 2.0 ** -24


def check_norm(g, x, r, w, offset, out, group, eps=1e-6):
    res = g.add_rms_norm_device(x, r, w, eps=eps, weight_offset=offset, out_dtype=out, group=group)
    res = res if isinstance(res, tuple) else (res,)
    h, y = norm_want(x, r, w, offset, eps)
    if r is not None:
        # fp32: the sum itself is rounded once; bf16: once in fp32 and once more, which may differ where the
        # first rounding lands on a border of the second
        close(res[-1], h, h.abs() * (0.0 if r.dtype == F32 else 2 * U[BF16]) + 1e-30, "sum")
        if r.dtype == BF16:  # the norm is that of the sum as it was stored
            y = norm_want(res[-1], None, w, offset, eps)[1]
    if out != E4M3:
        close(res[0], y, y.abs() * (U[out] + NORM_U) * 1.001 + 1e-37, "out")
        return res
    C = x.shape[1]
    gs = min(group or C, C)
    n = -(-C // gs)
    z = torch.nn.functional.pad(y, (0, n * gs - C)).view(-1, n, gs)
    scale = (z.abs().amax(-1) / 448.0).clamp(min=2.0 ** -100)
    close(res[1], scale, scale * (NORM_U + 2 * U[F32]) * 1.001, "scale")
    s = scale.repeat_interleave(gs, 1)[:, :C]
    # a normal value's half step, or the subnormals' (2^-10 of a scale)
    close(res[0].double() * s, y, (y.abs() * U[E4M3]).maximum(s * 2.0 ** -10) * 1.001 + y.abs() * 1e-5, "out * scale")
    return res


@pytest.mark.parametrize("rows, C", [(1, 1), (1, 2304), (3, 8), (5, 31), (2, 1153), (130, 2304), (7, 72), (2, 8192), (2, 8200),
                                     (3, 16384), (2, 5001), (1, 16383)])
@pytest.mark.parametrize("xt, rt, out", [(BF16, F32, BF16), (F32, F32, F32), (BF16, BF16, E4M3), (BF16, F32, E4M3),
                                         (F32, None, BF16), (BF16, None, F32), (F32, BF16, BF16)])
def test_norm_sizes_and_types(g, rows, C, xt, rt, out):
    x = randn(rows, C, seed=rows * 7 + C, dtype=xt)
    r = None if rt is None else randn(rows, C, seed=C, dtype=rt, scale=3.0)
    check_norm(g, x, r, randn(C, seed=2, scale=0.2), 1.0, out, 0)


@pytest.mark.parametrize("C, group", [(2304, 128), (2304, 64), (2304, 100), (1000, 128), (72, 8), (77, 10), (8200, 256), (64, 1),
                                      (24, 4096), (12288, 16),
                                      (16384, 1), (16384, 8), (64, 2 ** 31 - 1)])
def test_norm_groups(g, C, group):
    x, r = randn(9, C, seed=C, dtype=BF16), randn(9, C, seed=group % 1000, dtype=F32)
    x[:, :group] = 0
    r[:, :group] = 0  # a group of zeros has the smallest scale, and zeros
    res = check_norm(g, x, r, None, 0.0, E4M3, group)
    assert (res[1][:, 0] == 2.0 ** -100).all() and (res[0][:, :group].float() == 0).all()


def test_norm_strides_in_place_and_views(g):
    big = randn(6, 500, seed=1)
    x, r = big[:, 8:264].to(BF16), randn(6, 300, seed=2)[:, 4:260]
    want_h, want = norm_want(x, r, None, 0.0, 1e-5)
    buf = torch.zeros(6, 300, device="cuda")
    rr = buf[:, 3:259]  # unaligned rows
    rr.copy_(r)
    out, total = g.add_rms_norm_device(x, rr, eps=1e-5, out_dtype=F32, inplace=True)
    assert total.data_ptr() == rr.data_ptr()
    close(rr, want_h, want_h.abs() * 2.0 ** -24)
    close(out, want, want.abs() * (U[F32] + NORM_U) * 1.001)
    assert (buf[:, :3] == 0).all() and (buf[:, 259:] == 0).all()
    x2 = big[:, 11:240]  # rows 500 apart, 4-byte aligned
    close(g.add_rms_norm_device(x2), norm_want(x2, None, None, 0, 1e-6)[1], norm_want(x2, None, None, 0, 1e-6)[1].abs()
          * (U[F32] + NORM_U) * 1.001)


def test_norm_keeps_bad_rows_to_themselves(g):
    x, r = randn(4, 256, seed=3, dtype=BF16), randn(4, 256, seed=4)
    good = g.add_rms_norm_device(x, r, out_dtype=E4M3, group=64)
    x[1, 70] = math.nan
    r[2, 5] = math.inf
    x[3] = 0
    r[3] = 0
    out, scale, total = g.add_rms_norm_device(x, r, out_dtype=E4M3, group=64)
    assert torch.equal(out[0].view(torch.uint8), good[0][0].view(torch.uint8)) and torch.equal(scale[0], good[1][0])
    assert out[1].float().isnan().all() and scale[1].isnan().all()  # the root of a NaN mean reaches the whole row
    assert out[2].float()[5].isnan() and scale[2, 0].isnan() and (out[2].float()[64:] == 0).all()  # inf / inf, and x / inf
    assert (out[3].float() == 0).all() and torch.isfinite(scale[3]).all()
    assert g.add_rms_norm_device(x[:0], r[:0])[0].shape == (0, 256)


# --- rotary positions ----------------------------------------------------------------------------

def turn(x, pos, freq, interleaved, m=1.0):
    x = x.double().clone()
    half = freq.shape[0]
    i = torch.arange(half, device="cuda")
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    t = pos.double()[:, None, None] * freq
    xa, xb = x[..., a], x[..., b]
    x[..., a] = m * (xa * t.cos() - xb * t.sin())
    x[..., b] = m * (xb * t.cos() + xa * t.sin())
    return x


def turn_tol(x, freq, dtype, want, m=1.0):
    """The reduced angle is rounded once to fp32 (|angle| <= pi: 2^-24 pi), sine and cosine are good to 2 units
    (2^-22), the magnitude, two products and their sum round four times: 10 2^-22 of the pair's magnitudes cover them."""
    return want.abs() * (U[dtype] if dtype == BF16 else 2 * U[F32]) + 10 * 2.0 ** -22 * m * x.double().abs().amax(-1, keepdim=True)


@pytest.mark.parametrize("D, rotated", [(64, 64), (256, 256), (128, 64), (72, 72), (72, 16), (10, 6), (96, 48), (7, 2), (64, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rotary(g, D, rotated, interleaved, dtype):
    from sana_b200 import rotary_frequencies
    freq = torch.from_numpy(rotary_frequencies(rotated) if rotated else np.empty(0)).cuda()
    rows = 37
    fused = randn(rows, (5 + 2) * D, seed=D + rotated, dtype=dtype)  # one projection's rows: q | k
    q, k = fused[:, :5 * D].view(rows, 5, D), fused[:, 5 * D:].view(rows, 2, D)
    pos = torch.randint(-50, 200000, (rows,), device="cuda", dtype=torch.int32)
    pos[0], pos[1], pos[2] = 0, 2 ** 31 - 1, -2 ** 31
    qo, ko = g.rotary_device(q, k, pos, freq, interleaved=interleaved, magnitude=1.25)
    for x, got in ((q, qo), (k, ko)):
        want = turn(x, pos, freq, interleaved, 1.25)
        close(got, want, turn_tol(x, freq, dtype, want, 1.25))
        assert torch.equal(got[..., rotated:], x[..., rotated:])
    keep = fused.clone()
    qi = g.rotary_device(q, None, pos, freq, interleaved=interleaved, magnitude=1.25, inplace=True)
    assert qi.data_ptr() == q.data_ptr() and torch.equal(q, qo) and torch.equal(fused[:, 5 * D:], keep[:, 5 * D:])
    if dtype == F32 and rotated:  # turning back undoes it (position 0 is skipped by -pos = pos at the smallest int)
        back = g.rotary_device(q[3:], None, -pos[3:], freq, interleaved=interleaved, magnitude=0.8)
        close(back, keep[3:, :5 * D].reshape(-1, 5, D).double(), 40 * 2.0 ** -22 * keep.abs().max().double())


# --- the paged cache -------------------------------------------------------------------------------

class Paged:
    """A batch with lengths new[i] after past[i], in a pool with pages to spare filled with `fill`."""

    def __init__(self, new, past, hk, D, page, dtype, seed, fill=math.nan, layout="tokens", trailing=0, spare=3):
        self.new, self.past, self.page = new, past, page
        gen = torch.Generator().manual_seed(seed)
        need = [-(-(n + p) // page) for n, p in zip(new, past)]
        pages = sum(need) + spare
        shape = (pages, page, hk, D) if layout == "tokens" else (pages, hk, page, D)
        make = lambda: torch.full(shape, fill, dtype=dtype, device="cuda")  # noqa: E731
        self.k, self.v = make(), make()
        if layout == "heads":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        order = torch.randperm(pages, generator=gen).tolist()
        self.pages = [[order.pop() for _ in range(n)] for n in need]
        width = max(need + [1]) + 2
        table = torch.full((len(new), width), -7, dtype=torch.int32)  # entries behind the last page mean nothing
        for s, p in enumerate(self.pages):
            table[s, :len(p)] = torch.tensor(p, dtype=torch.int32)
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.rows = int(starts[-1]) + trailing
        self.row_start = torch.from_numpy(starts).cuda()
        self.kv_len = torch.tensor([n + p for n, p in zip(new, past)], dtype=torch.int32, device="cuda")
        self.table = table.cuda()
        self.max_new, self.max_kv = max(new), max(n + p for n, p in zip(new, past))

    def places(self, s, lo, hi):
        j = torch.arange(lo, hi)
        return torch.tensor(self.pages[s])[j // self.page].cuda(), (j % self.page).cuda()

    def fill(self, seed, scale=1.0):
        for s, (n, p) in enumerate(zip(self.new, self.past)):
            at = self.places(s, 0, n + p)
            hk, D = self.k.shape[2:]
            self.k[at] = randn(n + p, hk, D, seed=seed + 2 * s, dtype=self.k.dtype, scale=scale)
            self.v[at] = randn(n + p, hk, D, seed=seed + 2 * s + 1, dtype=self.k.dtype)
        return self

    def args(self):
        return self.row_start, self.kv_len, self.table, self.max_new


@pytest.mark.parametrize("dtype, D, rotated, page, layout", [(BF16, 128, 128, 16, "tokens"), (F32, 72, 36, 24, "tokens"),
                                                             (BF16, 256, 256, 1, "tokens"), (BF16, 64, 32, 7, "heads"),
                                                             (F32, 10, 4, 5, "heads"), (BF16, 96, 96, 1000, "tokens")])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_append(g, dtype, D, rotated, page, layout, interleaved):
    from sana_b200 import rotary_frequencies
    freq = torch.from_numpy(rotary_frequencies(rotated, scaling="linear", stretch=2.0)).cuda()
    b = Paged([3, 0, 1, 40], [5, 9, 0, 61], 2, D, page, dtype, seed=D, fill=7.0, layout=layout, trailing=4)
    q, k, v = (randn(b.rows, n, D, seed=i, dtype=dtype) for i, n in enumerate((6, 2, 2)))
    q_keep, kc, vc = q.clone(), b.k.clone(), b.v.clone()
    out = g.rotary_append_device(q, k, v, freq, b.k, b.v, *b.args(), interleaved=interleaved, inplace=True)
    row = 0
    for s, (n, p) in enumerate(zip(b.new, b.past)):
        pos = torch.arange(p, p + n, device="cuda")
        at = b.places(s, p, p + n)
        sl = slice(row, row + n)
        for x, got in ((q_keep[sl], out[sl]), (k[sl], b.k[at])):
            want = turn(x, pos, freq, interleaved)
            close(got, want, turn_tol(x, freq, dtype, want))
        assert torch.equal(b.v[at], v[sl])
        kc[at], vc[at] = b.k[at], v[sl]
        row += n
    assert torch.equal(out[row:], q_keep[row:])  # rows behind the last sequence
    assert torch.equal(b.k, kc) and torch.equal(b.v, vc)  # nothing else of the pool
    before = b.k.clone()
    g.rotary_append_device(None, k, v, None, b.k, b.v, *b.args())  # without turning
    at = b.places(3, 61, 101)
    assert torch.equal(b.k[at], k[4:44])
    assert not torch.equal(b.k, before)
    g.synchronize()  # nothing was recorded


def test_append_skips_and_records_bad_pages(g):
    b = Paged([2, 3], [6, 2], 2, 64, 4, BF16, seed=1, fill=7.0)
    k, v = (randn(5, 2, 64, seed=i, dtype=BF16) for i in (1, 2))
    for bad in (-1, b.k.shape[0], 2 ** 31 - 1):
        table = b.table.clone()
        table[0, 1] = bad  # where both new tokens of sequence 0 belong
        b.k.fill_(7.0)
        b.v.fill_(7.0)
        g.rotary_append_device(None, k, v, None, b.k, b.v, b.row_start, b.kv_len, table, 3)
        with pytest.raises(ValueError, match="page"):
            g.synchronize()
        g.synchronize()  # once
        at = b.places(1, 2, 5)
        assert torch.equal(b.k[at], k[2:]) and torch.equal(b.v[at], v[2:])
        assert (b.k == 7.0).sum().item() == b.k.numel() - 3 * 2 * 64
    for starts, lens in (([0, 2, 9], [8, 5]), ([0, 2, 5], [1, 5]), ([0, 2, 5], [-3, 5])):
        g.rotary_append_device(None, k, v, None, b.k, b.v, torch.tensor(starts, dtype=torch.int32, device="cuda"),
                               torch.tensor(lens, dtype=torch.int32, device="cuda"), b.table, 3)
        with pytest.raises(ValueError):
            g.synchronize()


# --- attention ---------------------------------------------------------------------------------------

def attention_want(b, q, scale, window, sinks, cap):
    """(outputs, tolerances before the output's rounding) of the batch's rows in 64 bits."""
    heads, hk, D = q.shape[1], b.k.shape[2], q.shape[2]
    G = heads // hk
    want = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(want)
    row = 0
    for s, (n, p) in enumerate(zip(b.new, b.past)):
        if n == 0:
            continue
        at = b.places(s, 0, n + p)
        k, v = (t[at].double().repeat_interleave(G, 1).transpose(0, 1) for t in (b.k, b.v))
        qq = q[row:row + n].double().transpose(0, 1)
        t = qq @ k.transpose(1, 2) * scale
        size = qq.abs() @ k.abs().transpose(1, 2) * abs(scale)
        if cap:
            t = cap * torch.tanh(t / cap)
        i, j = torch.arange(p, p + n, device="cuda")[:, None], torch.arange(n + p, device="cuda")
        hidden = j > i
        if window:
            hidden |= (j <= i - window) & (j >= sinks)
        t.masked_fill_(hidden, -math.inf)
        prob = torch.softmax(t, -1)
        vv = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
        o = prob @ vv
        # a value that is not finite reaches those who see it
        for h, jj, d in (~torch.isfinite(v)).nonzero().tolist():
            o[h, :, d] += torch.where(hidden[:, jj], 0.0, v[h, jj, d].item())
        want[row:row + n] = o.transpose(0, 1)
        # A score of D fp32 products is off by (D / 8 + 8) 2^-24 of its terms' magnitudes (the tensor cores add eight at a
        # time, a thread four), the scale, the base change and the cap by 8 roundings of the score (the cap by 2^-20 of
        # itself); its exponential by the same, relatively, and by 2^-21 of its own. Numerator and denominator both carry
        # it. The probabilities of the tensor cores are rounded once to bf16.
        e = ((D / 8 + 8) * 2.0 ** -24 * size + 8 * 2.0 ** -24 * size + (2.0 ** -20 * cap) + 2.0 ** -20).masked_fill(hidden, 0).amax(-1, keepdim=True)
        p_round = U[BF16] if q.dtype == BF16 else 0.0
        sums = (n + p) / 16 * 2.0 ** -24
        tol[row:row + n] = ((prob @ vv.abs()) * (2 * e * 1.01 + p_round + sums)).transpose(0, 1)
        row += n
    return want, tol


def check_attention(g, b, q, window=0, sinks=0, cap=0.0, scale=None, out=None):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    got = g.paged_attention_device(q, b.k, b.v, *b.args(), b.max_kv, scale=scale, window=window, sinks=sinks, softcap=cap, out=out)
    g.synchronize()  # nothing was recorded
    want, tol = attention_want(b, q, scale, window, sinks, cap)
    live = sum(b.new)
    close(got[:live], want[:live], (tol + want.abs() * U[q.dtype])[:live] + 1e-30, (window, sinks, cap))
    return got


LENGTHS = [([1], [0]), ([1, 1, 1], [0, 15, 300]), ([1], [4095]), ([2, 5, 1], [63, 64, 7]), ([0, 3, 0], [4, 0, 9]),
           ([17, 1, 33], [100, 0, 31]), ([130, 64, 1], [0, 64, 200]), ([300], [211]), ([257, 129], [511, 3])]


@pytest.mark.parametrize("new, past", LENGTHS)
@pytest.mark.parametrize("dtype, D, hk, G, page", [(BF16, 64, 2, 4, 16), (BF16, 128, 1, 8, 64), (BF16, 256, 2, 2, 16),
                                                   (BF16, 72, 3, 1, 24), (BF16, 128, 2, 3, 1), (F32, 72, 2, 3, 24),
                                                   (F32, 256, 1, 2, 16), (BF16, 100, 1, 5, 5), (F32, 3, 1, 1, 7)])
def test_attention_lengths(g, new, past, dtype, D, hk, G, page):
    b = Paged(new, past, hk, D, page, dtype, seed=D + len(new), trailing=2).fill(11)
    q = randn(b.rows, hk * G, D, seed=5, dtype=dtype, scale=2.0)
    out = torch.full_like(q, 5.0)
    check_attention(g, b, q, out=out)
    assert (out[sum(new):] == 5.0).all()  # rows behind the last sequence


@pytest.mark.parametrize("window, sinks", [(1, 0), (5, 0), (64, 4), (100, 1), (100, 150), (1000, 3), (16, 70), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("dtype, D, new, past", [(BF16, 128, [1, 1], [700, 3]), (BF16, 64, [40, 7], [300, 0]),
                                                 (BF16, 256, [200, 1], [350, 900]), (F32, 40, [33, 1], [200, 99]),
                                                 (BF16, 128, [400], [300])])
def test_attention_window_and_sinks(g, window, sinks, dtype, D, new, past):
    b = Paged(new, past, 2, D, 16, dtype, seed=window % 1000 + sinks % 1000).fill(3)
    check_attention(g, b, randn(b.rows, 4, D, seed=9, dtype=dtype, scale=2.0), window, sinks)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cap, scale", [(50.0, None), (3.0, 1.0), (0.0, -0.3), (0.0, 0.0), (1.0, 100.0)])
@pytest.mark.parametrize("new, past", [([1, 1], [40, 600]), ([150], [70])])
def test_attention_cap_and_scale(g, dtype, cap, scale, new, past):
    b = Paged(new, past, 2, 64, 32, dtype, seed=4).fill(8)
    check_attention(g, b, randn(b.rows, 4, 64, seed=9, dtype=dtype), cap=cap, scale=scale)


@pytest.mark.parametrize("layout, page", [("heads", 16), ("tokens", 4096), ("heads", 50)])
@pytest.mark.parametrize("new, past", [([1, 1], [40, 600]), ([150, 9], [70, 700])])
def test_attention_layouts(g, layout, page, new, past):
    """Heads before tokens in a page; one page per sequence (a contiguous cache); q as columns of a wider row."""
    b = Paged(new, past, 2, 128, page, BF16, seed=4, layout=layout).fill(8)
    wide = randn(b.rows, 10, 128, seed=9, dtype=BF16)
    check_attention(g, b, wide[:, 2:8])


@pytest.mark.parametrize("dtype, D", [(BF16, 128), (BF16, 256), (F32, 64), (BF16, 60)])
@pytest.mark.parametrize("new, past", [([1], [100]), ([70], [90]), ([300], [40])])
def test_what_is_not_seen_does_not_reach_the_output(g, dtype, D, new, past):
    """NaN and infinities in later tokens and outside the window: only the tokens that see them have them."""
    b = Paged(new, past, 1, D, 16, dtype, seed=6).fill(2)
    q = randn(b.rows, 2, D, seed=3, dtype=dtype)
    clean = check_attention(g, b, q, window=50, sinks=2).clone()
    n, p = new[0], past[0]
    bad = [0, 1, p + n - 1] if n > 1 else [20]
    if n > 1:
        for j, value in ((p + n - 1, math.nan), (p + n // 2, math.inf)):
            page, slot = b.places(0, j, j + 1)
            b.v[page, slot, :, 3] = value
        page, slot = b.places(0, p + n - 1, p + n)
        b.k[page, slot] = math.nan
    for j in ((20, 30) if p - 50 > 30 else ()):  # between the sinks and the first row's window
        page, slot = b.places(0, j, j + 1)
        b.k[page, slot] = math.nan
        b.v[page, slot] = math.inf
    got = g.paged_attention_device(q, b.k, b.v, *b.args(), b.max_kv, window=50, sinks=2)
    g.synchronize()
    seen_from = n // 2 if n > 1 else n
    assert torch.equal(got[:seen_from], clean[:seen_from])
    if n > 1:
        assert torch.isinf(got[seen_from:min(seen_from + 50, n - 1), :, 3]).all() and (got[seen_from:min(seen_from + 50, n - 1), :, 3] > 0).all()
        other = [d for d in range(D) if d != 3]
        assert torch.equal(got[:n - 1][:, :, other], clean[:n - 1][:, :, other])
        assert got[n - 1].isnan().all()  # it sees its own NaN key
    assert bad


def test_scores_that_overflow_and_empty_rows(g):
    """Scores of -inf and large ones; all of a row's keys on bad pages: zeros, recorded."""
    b = Paged([2, 3], [30, 0], 1, 64, 8, BF16, seed=6).fill(2)
    q = randn(5, 1, 64, seed=3, dtype=BF16, scale=1e4)
    check_attention(g, b, q, scale=1.0)
    table = b.table.clone()
    table[1, :] = b.k.shape[0]
    got = g.paged_attention_device(q, b.k, b.v, b.row_start, b.kv_len, table, 3, b.max_kv)
    with pytest.raises(ValueError, match="page"):
        g.synchronize()
    assert (got[2:] == 0).all() and torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_bad_pages_are_left_out(g, dtype):
    """A page outside the pool: its keys count as not there, the others as they would without it."""
    for new, past in (([1], [95]), ([90], [6])):
        b = Paged(new, past, 2, 64, 32, dtype, seed=1).fill(4)
        q = randn(b.rows, 4, 64, seed=2, dtype=dtype)
        table = b.table.clone()
        table[0, 0] = -5
        got = g.paged_attention_device(q, b.k, b.v, b.row_start, b.kv_len, table, b.max_new, b.max_kv)
        with pytest.raises(ValueError, match="page"):
            g.synchronize()
        want = g.paged_attention_device(q, b.k, b.v, b.row_start, b.kv_len, b.table, b.max_new, b.max_kv, window=10 ** 6)
        g.synchronize()
        # rows past the bad page: the 64-bit result over keys 32 .. p
        for r in range(max(0, 32 - past[0]), b.rows):
            p = past[0] + r
            at = b.places(0, 32, p + 1)
            k, v = b.k[at].double(), b.v[at].double()
            for h in range(4):
                pr = torch.softmax(q[r, h].double() @ k[:, h // 2].T / 8.0, -1)
                o, mag = pr @ v[:, h // 2], pr @ v[:, h // 2].abs()
                close(got[r, h], o, o.abs() * U[dtype] + mag * ((U[BF16] if dtype == BF16 else 0) + 1e-4))
        assert want.isfinite().all()


def test_bad_lengths_are_recorded(g):
    b = Paged([2, 3], [30, 5], 1, 64, 8, BF16, seed=6).fill(2)
    q = randn(5, 1, 64, seed=3, dtype=BF16)
    good = check_attention(g, b, q)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for starts, lens, max_new in (([0, 2, 5], [32, 2], 3), ([0, 2, 5], [32, 33], 3), ([0, 2, 5], [32, 8], 2),
                                  ([0, 2, 6], [32, 8], 9), ([0, 2, 1], [32, 8], 3), ([0, 2, 5], [32, -1], 3)):
        out = torch.full_like(q, 9.0)
        g.paged_attention_device(q, b.k, b.v, i32(starts), i32(lens), b.table, max_new, b.max_kv, out=out)
        with pytest.raises(ValueError):
            g.synchronize()
        assert torch.equal(out[:2], good[:2]) and (out[2:] == 9.0).all()


def test_offsets_beyond_32_bits(g):
    """A pool whose pages lie more than 2^31 elements apart."""
    step = 2 ** 31 + 64
    pool = torch.empty(step + 64 * 128, dtype=BF16, device="cuda")
    k = pool.as_strided((2, 16, 2, 64), (step, 256, 64, 1))
    v = pool.as_strided((2, 16, 2, 64), (step, 256, 64, 1), 128)  # between k's tokens
    new, past = randn(1, 2, 64, seed=1, dtype=BF16), 19
    b = Paged([1], [past], 2, 64, 16, BF16, seed=0, spare=0).fill(3)
    k[0], k[1], v[0], v[1] = b.k[b.pages[0][0]], b.k[b.pages[0][1]], b.v[b.pages[0][0]], b.v[b.pages[0][1]]
    b.k, b.v, b.pages = k, v, [[0, 1]]
    b.table = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    g.rotary_append_device(None, new, new, None, b.k, b.v, *b.args())
    assert torch.equal(k[1, 3], new[0]) and torch.equal(v[1, 3], new[0])
    check_attention(g, b, randn(1, 4, 64, seed=2, dtype=BF16))
    b.new, b.past, b.max_new, b.row_start = [18], [2], 18, torch.tensor([0, 18], dtype=torch.int32, device="cuda")
    check_attention(g, b, randn(18, 4, 64, seed=2, dtype=BF16))


@pytest.mark.parametrize("D", [8, 16, 40, 56, 88, 120, 136, 192, 200, 248])
@pytest.mark.parametrize("page", [8, 16, 32, 128, 256, 48, 4])
def test_attention_head_and_page_sizes(g, D, page):
    """Head sizes that end inside a slab, pages that divide a tile, that tiles divide, and others; few rows and many."""
    for new, past in (([1, 2], [200, 40]), ([70, 5], [130, 300])):
        b = Paged(new, past, 2, D, page, BF16, seed=D + page).fill(7)
        check_attention(g, b, randn(b.rows, 6, D, seed=1, dtype=BF16), window=150 if page != 16 else 0, sinks=3)


def test_rows_in_front_and_behind(g):
    """Rows before the first sequence, as behind the last, are nobody's."""
    b = Paged([3, 40], [20, 9], 1, 64, 16, BF16, seed=3, trailing=2).fill(5)
    starts = b.row_start + 4
    q = randn(b.rows + 4, 2, 64, seed=1, dtype=BF16)
    out, plain = torch.full_like(q, 3.0), check_attention(g, b, q[4:])
    g.paged_attention_device(q, b.k, b.v, starts, b.kv_len, b.table, b.max_new, b.max_kv, out=out)
    g.synchronize()
    assert torch.equal(out[4:47], plain[:43]) and (out[:4] == 3.0).all() and (out[47:] == 3.0).all()
    k, v = randn(b.rows + 4, 1, 64, seed=2, dtype=BF16), randn(b.rows + 4, 1, 64, seed=3, dtype=BF16)
    freq = torch.ones(32, dtype=torch.float64, device="cuda")
    keep = q.clone()
    got = g.rotary_append_device(q, k, v, freq, b.k, b.v, starts, b.kv_len, b.table, b.max_new, inplace=True)
    g.synchronize()
    assert torch.equal(got[:4], keep[:4]) and torch.equal(got[47:], keep[47:]) and not torch.equal(got[4:47], keep[4:47])
    assert torch.equal(b.v[b.places(1, 9, 49)], v[7:47])


def test_two_handles_at_once(g):
    """Two handles on two streams, each with a workspace of its own: the results of one at a time."""
    from sana_b200 import SanaCuda
    other = SanaCuda(0)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    bs = [Paged([1, 1, 1, 1], [3000, 64, 900, 10 + i], 2, 128, 16, BF16, seed=i).fill(5 + i) for i in range(2)]
    bs += [Paged([300], [700 + i], 2, 128, 16, BF16, seed=i).fill(9 + i) for i in range(2)]
    qs = [randn(b.rows, 8, 128, seed=i, dtype=BF16) for i, b in enumerate(bs)]
    want = [check_attention(g, b, q).clone() for b, q in zip(bs, qs)]
    torch.cuda.synchronize()
    got = [[], [], [], []]
    for _ in range(10):
        for h, st, pick in ((g, streams[0], (0, 2)), (other, streams[1], (1, 3))):
            with torch.cuda.stream(st):
                h.set_stream(st.cuda_stream)
                for i in pick:
                    got[i].append(h.paged_attention_device(qs[i], bs[i].k, bs[i].v, *bs[i].args(), bs[i].max_kv))
    torch.cuda.synchronize()
    g.set_stream(1)
    for w, all_ in zip(want, got):
        assert all(torch.equal(x, w) for x in all_)
    other.close()


def test_shared_prefix_pages(g):
    """Sequences whose first pages are the same: each as if it had its own copy."""
    b = Paged([9, 4, 12], [32, 32, 32], 2, 128, 16, BF16, seed=3).fill(5)
    for s in (1, 2):
        for i in range(2):
            b.pages[s][i] = b.pages[0][i]
            b.table[s, i] = b.pages[0][i]
    check_attention(g, b, randn(b.rows, 8, 128, seed=1, dtype=BF16))


def test_streams_graphs_and_workspaces(g):
    """A captured call replayed with other lengths and inputs; the same from another stream than torch's; a workspace
    that is too small is refused; results are the same bits every time."""
    b = Paged([1, 1, 1], [900, 64, 3000], 2, 128, 16, BF16, seed=3).fill(5)
    q = randn(3, 8, 128, seed=1, dtype=BF16)
    first = check_attention(g, b, q).clone()
    need = g.paged_attention_workspace(q, b.k, b.v, *b.args(), b.max_kv)
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError, match="workspace"):
        g.paged_attention_device(q, b.k, b.v, *b.args(), b.max_kv, workspace=ws[:need - 16])
    ws.fill_(255)
    assert torch.equal(g.paged_attention_device(q, b.k, b.v, *b.args(), b.max_kv, workspace=ws), first)

    from sana_b200 import SanaCuda
    other = SanaCuda(0)  # on its own stream
    for _ in range(3):
        x = randn(3, 8, 128, seed=1, dtype=BF16)  # freed and handed out again while the other stream works
        assert torch.equal(other.paged_attention_device(x, b.k, b.v, *b.args(), b.max_kv), first)
    other.synchronize()
    other.close()

    side = torch.cuda.Stream()
    out = torch.zeros_like(q)
    total = torch.zeros(3, 1024, device="cuda")
    w = randn(1024, seed=8)
    with torch.cuda.stream(side):
        g.set_stream(side.cuda_stream)
        g.paged_attention_device(q, b.k, b.v, *b.args(), b.max_kv, out=out, workspace=ws)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            g.paged_attention_device(q, b.k, b.v, *b.args(), b.max_kv, out=out, workspace=ws)
            y, _ = g.add_rms_norm_device(out.view(3, 1024), total, w, inplace=True)
    g.set_stream(1)
    torch.cuda.synchronize()
    total.zero_()
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first) and torch.equal(total, first.view(3, 1024).float())
    b.past = [17, 2000, 5]
    b.kv_len.copy_(torch.tensor([18, 2001, 6], dtype=torch.int32))
    b.pages = [[p for p in b.table[s].tolist()] for s in range(3)]
    # sequence 1 has too few pages for 2001 tokens: give it sequence 2's
    b.pages[1] = b.pages[2]
    b.table[1] = b.table[2]
    q.copy_(randn(3, 8, 128, seed=77, dtype=BF16))
    graph.replay()
    torch.cuda.synchronize()
    want, tol = attention_want(b, q, 128 ** -0.5, 0, 0, 0.0)
    close(out, want, tol + want.abs() * U[BF16])


def test_wrong_tensors_are_refused(g):
    b = Paged([1], [30], 1, 64, 8, BF16, seed=6).fill(2)
    q = randn(1, 2, 64, seed=3, dtype=BF16)
    for bad in (q.float(), q.cpu(), q[:, :, :32], q.half(), q[0], torch.cat([q, q], 2)[:, :, ::2]):
        with pytest.raises(ValueError):
            g.paged_attention_device(bad, b.k, b.v, *b.args(), b.max_kv)
    for change in (dict(row_start=b.row_start.long()), dict(kv_len=b.kv_len.float()), dict(page_table=b.table[0]),
                   dict(row_start=b.row_start[:1]), dict(page_table=b.table.cpu())):
        a = {**dict(row_start=b.row_start, kv_len=b.kv_len, page_table=b.table), **change}
        with pytest.raises(ValueError):
            g.paged_attention_device(q, b.k, b.v, max_new=1, max_kv=31, **a)
    with pytest.raises(ValueError):
        g.paged_attention_device(q, b.k, b.v[:1], *b.args(), b.max_kv)
    with pytest.raises(ValueError):
        g.add_rms_norm_device(q[0], torch.zeros(2, 32, device="cuda"))
    with pytest.raises(ValueError):
        g.rotary_device(q, None, torch.zeros(1, device="cuda", dtype=torch.int64), torch.ones(4, device="cuda").double())


# --- together ------------------------------------------------------------------------------------------

def test_an_encoder_block_over_a_shared_prefix(g):
    """The attention half of an encoder block, as a server of prompts runs it: residual norm, QKV product, rotary
    positions with the append, attention over the pages, output product onto the residual stream, norm in 8 bits. Two
    prompts whose instruction prefix is cached once; in one chunk, in two, and token by token. Each operator is held to
    the 64-bit result of what it was given, and the attended rows of all ways to one another."""
    from sana_b200 import rotary_frequencies
    heads, hk, D, page, prefix = 4, 2, 64, 16, 32
    C, W = heads * D, (heads + 2 * hk) * D
    w_qkv, w_o = randn(W, C, seed=1, dtype=BF16, scale=C ** -0.5), randn(C, C, seed=2, dtype=BF16, scale=C ** -0.5)
    w_n = randn(C, seed=3, scale=0.1)
    freq = torch.from_numpy(rotary_frequencies(D)).cuda()
    tokens = 24
    # the stream: the prefix's rows, then two prompts
    stream = randn(prefix + 2 * tokens, C, seed=4, scale=2.0)
    pages = torch.arange(8, dtype=torch.int32)
    table = torch.stack([torch.tensor([0, 1, 2, 3]), torch.tensor([0, 1, 4, 5])]).to(torch.int32).cuda()
    k_cache, v_cache = (torch.full((len(pages), page, hk, D), math.nan, dtype=BF16, device="cuda") for _ in range(2))

    def half_block(x, new, past, tab):
        rows = sum(new)
        zero = torch.zeros(rows, C, device="cuda", dtype=BF16)
        a, s = g.add_rms_norm_device(zero, x, w_n, weight_offset=1.0)
        h, y = norm_want(zero, x, w_n, 1.0, 1e-6)
        assert torch.equal(s, x)
        close(a, y, y.abs() * (U[BF16] + NORM_U) * 1.001)
        qkv = torch.empty(rows, W, device="cuda", dtype=BF16)
        g.gemm_device(a.data_ptr(), w_qkv.data_ptr(), rows, W, C, qkv.data_ptr())
        q, k, v = (qkv[:, lo * D:hi * D].unflatten(1, (-1, D)) for lo, hi in ((0, heads), (heads, heads + hk), (heads + hk, heads + 2 * hk)))
        starts = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
        lens = torch.tensor([n + p for n, p in zip(new, past)], dtype=torch.int32, device="cuda")
        qr = g.rotary_append_device(q, k, v, freq, k_cache, v_cache, starts, lens, tab, max(new))
        pos = torch.cat([torch.arange(p, p + n, device="cuda") for n, p in zip(new, past)])
        want = turn(q, pos, freq, False)
        close(qr, want, turn_tol(q, freq, BF16, want))
        o = g.paged_attention_device(qr, k_cache, v_cache, starts, lens, tab, max(new), max(lens.tolist()))
        b = Paged(new, past, hk, D, page, BF16, seed=0)
        b.k, b.v, b.pages = k_cache, v_cache, tab.tolist()
        want, tol = attention_want(b, qr, D ** -0.5, 0, 0, 0.0)
        close(o, want, tol + want.abs() * U[BF16])
        out = torch.empty(rows, C, device="cuda")
        g._call("sana_op_gemm_residual_device", vp(o.data_ptr()), vp(w_o.data_ptr()), rows, C, C, None, vp(x.data_ptr()),
                None, 1, vp(out.data_ptr()), None)
        want = x.double() + o.view(rows, C).double() @ w_o.double().T
        close(out, want, (C * 2.0 ** -24) * (o.view(rows, C).double().abs() @ w_o.double().abs().T) + want.abs() * 2.0 ** -23)
        check_norm(g, zero, out, w_n, 1.0, E4M3, 128)
        return o

    half_block(stream[:prefix], [prefix], [0], table[:1])  # once for both prompts
    ways = []
    for steps in ([24], [10, 14], [11, 1, 1, 11]):
        got, done = [[], []], 0
        for n in steps:
            x = torch.cat([stream[prefix + i * tokens + done:prefix + i * tokens + done + n] for i in range(2)])
            o = half_block(x.contiguous(), [n, n], [prefix + done] * 2, table)
            for i in range(2):
                got[i].append(o[i * n:(i + 1) * n])
            done += n
        g.synchronize()
        ways.append(torch.cat([torch.cat(x) for x in got]).double())
    # The projections of a row do not depend on the batch. The attention's probabilities round to bf16 against another
    # running maximum, and its output once: twice 2^-8 each, of magnitudes up to the values' largest.
    for w in ways[1:]:
        assert (w - ways[0]).abs().max() <= 4 * U[BF16] * v_cache[:6].float().nan_to_num().abs().max()
