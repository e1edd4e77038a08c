"""The text encoder's operators without a GPU: rotary frequencies (host only) against their
formulas, and what the entry points refuse. A handle that could not be created on this machine
still reports argument errors, which come before any use of the device."""
import ctypes
import math

import numpy as np
import pytest

import sana_b200
from sana_b200 import capi

INVALID, PTR = 1, 0x1000  # a non-NULL address; no refused call reads it


@pytest.fixture(scope="module")
def handle():
    lib = sana_b200.load_library()
    h = ctypes.c_void_p()
    rc = lib.sana_cuda_create(0, 0, ctypes.byref(h))
    yield lib, h, rc == 0
    lib.sana_cuda_destroy(h)


def message(lib, h):
    return lib.sana_cuda_last_error(h).decode()


@pytest.mark.parametrize("rotated", [2, 8, 64, 256])
def test_frequencies_follow_their_formulas(rotated):
    i = np.arange(rotated // 2)
    plain = 10000.0 ** (-2.0 * i / rotated)
    assert np.allclose(sana_b200.rotary_frequencies(rotated), plain, rtol=1e-14, atol=0)
    assert np.allclose(sana_b200.rotary_frequencies(rotated, scaling="linear", stretch=4.0), plain / 4, rtol=1e-14, atol=0)
    if rotated > 2:
        base = 500000.0 * 8.0 ** (rotated / (rotated - 2))
        got = sana_b200.rotary_frequencies(rotated, base=500000.0, scaling="base", stretch=8.0)
        assert np.allclose(got, base ** (-2.0 * i / rotated), rtol=1e-13, atol=0)
        # the slowest pair is slowed by the whole stretch, the fastest is left
        assert got[0] == 1.0
        assert np.isclose(got[-1], 500000.0 ** (-(rotated - 2) / rotated) / 8, rtol=1e-12)
    got = sana_b200.rotary_frequencies(rotated, scaling="parts", stretch=8.0, context=4096.0, slow=1.0, fast=32.0)
    for f, g in zip(plain, got):
        turns = 4096.0 * f / (2 * math.pi)
        want = f if turns >= 32 else f / 8 if turns <= 1 else f * (turns - 1) / 31 + f / 8 * (32 - turns) / 31
        assert math.isclose(g, want, rel_tol=1e-12)


@pytest.mark.parametrize("kw", [dict(rotated=3), dict(rotated=0), dict(rotated=-2), dict(rotated=8, base=0.0),
                                dict(rotated=8, stretch=0.5), dict(rotated=8, stretch=math.nan),
                                dict(rotated=2, scaling="base", stretch=2.0),
                                dict(rotated=8, scaling="parts", stretch=2.0, context=0.0),
                                dict(rotated=8, scaling="parts", stretch=2.0, context=4096.0, slow=4.0, fast=4.0),
                                dict(rotated=8, scaling="dynamic")])
def test_frequencies_refusals(kw):
    with pytest.raises(ValueError):
        sana_b200.rotary_frequencies(**kw)


NORM = dict(x=PTR, xt=0, ldx=64, r=PTR, rt=0, ldr=64, sum=PTR, w=PTR, off=0.0, eps=1e-6, rows=4, C=64, out=PTR, ot=0,
            ldo=64, scale=None, group=0)


@pytest.mark.parametrize("change, word", [
    (dict(x=None), "x"), (dict(out=None), "out"), (dict(ldx=63), "row stride"), (dict(ldo=0), "row stride"),
    (dict(ldr=1), "row stride"), (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(C=0), "C must"),
    (dict(C=16385, ldx=20000, ldr=20000, ldo=20000), "C must"), (dict(xt=2), "F32 or BF16"), (dict(rt=7), "F32 or BF16"),
    (dict(ot=3), "out must"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"), (dict(group=-1, ot=2, scale=PTR), "group"),
    (dict(group=32), "group"), (dict(ot=2), "scale"), (dict(r=None), "sum needs")])
def test_norm_refusals(handle, change, word):
    lib, h, _ = handle
    a = {**NORM, **change}
    assert lib.sana_op_add_rms_norm_device(h, *a.values()) == INVALID
    assert word in message(lib, h)


def batch(**kw):
    d = dict(sequences=2, rows=8, max_new=4, max_kv=64, row_start=PTR, kv_len=PTR, page_table=PTR, table_stride=4, table_width=4)
    return capi.sana_paged_batch(*{**d, **kw}.values())


def cache(**kw):
    d = dict(k=PTR, v=PTR, dtype=1, pages=8, page_size=16, kv_heads=2, head_dim=64, page_stride=2048, token_stride=128,
             head_stride=64)
    return capi.sana_paged_cache(*{**d, **kw}.values())


BAD_BATCH = [(dict(sequences=-1), "negative"), (dict(rows=-1), "negative"), (dict(max_kv=-5), "negative"),
             (dict(row_start=None), "NULL"), (dict(kv_len=None), "NULL"), (dict(page_table=None), "NULL"),
             (dict(table_stride=3), "table_stride")]
BAD_CACHE = [(dict(k=None), "NULL"), (dict(v=None), "NULL"), (dict(dtype=2), "dtype"), (dict(page_size=0), "sizes"),
             (dict(pages=-1), "sizes"), (dict(kv_heads=0), "sizes"), (dict(head_dim=0), "sizes"),
             (dict(page_stride=-1), "strides")]


def attend(lib, h, b=None, c=None, **kw):
    a = dict(q=PTR, ldq=512, heads=8, scale=0.125, window=0, sinks=0, cap=0.0, out=PTR, ldo=512, ws=None, n=0)
    b, c = b or batch(), c or cache()
    return lib.sana_op_paged_attention_device(h, ctypes.byref(b), ctypes.byref(c), *{**a, **kw}.values())


@pytest.mark.parametrize("change, word", BAD_BATCH)
def test_batch_refusals(handle, change, word):
    lib, h, _ = handle
    b, c = batch(**change), cache()
    assert attend(lib, h, b=b) == INVALID and word in message(lib, h)
    assert lib.sana_op_rotary_append_device(h, None, ctypes.byref(b), ctypes.byref(c), None, 0, 0, None, PTR, 128, PTR,
                                            128) == INVALID
    assert lib.sana_op_paged_attention_workspace(h, ctypes.byref(b), ctypes.byref(c), 8, 0, 0) == 0


@pytest.mark.parametrize("change, word", BAD_CACHE)
def test_cache_refusals(handle, change, word):
    lib, h, _ = handle
    b, c = batch(), cache(**change)
    assert attend(lib, h, c=c) == INVALID and word in message(lib, h)
    assert lib.sana_op_rotary_append_device(h, None, ctypes.byref(b), ctypes.byref(c), None, 0, 0, None, PTR, 128, PTR,
                                            128) == INVALID


@pytest.mark.parametrize("change, word", [
    (dict(q=None), "q must"), (dict(out=None), "out must"), (dict(ldq=511), "row stride"), (dict(ldo=0), "row stride"),
    (dict(heads=7), "multiple"), (dict(heads=0), "multiple"), (dict(window=-1), "window"), (dict(sinks=-1), "window"),
    (dict(scale=math.inf), "scale"), (dict(cap=-1.0), "softcap"), (dict(cap=math.nan), "softcap"), (dict(cap=1e-38), "softcap")])
def test_attention_refusals(handle, change, word):
    lib, h, _ = handle
    assert attend(lib, h, **change) == INVALID and word in message(lib, h)


def test_attention_refuses_large_heads_and_null_structs(handle):
    lib, h, _ = handle
    assert attend(lib, h, c=cache(head_dim=264), ldq=4096, ldo=4096) == INVALID and "head_dim" in message(lib, h)
    assert lib.sana_op_paged_attention_device(h, None, None, PTR, 512, 8, 0.1, 0, 0, 0.0, PTR, 512, None, 0) == INVALID
    assert lib.sana_op_rotary_append_device(h, None, None, None, None, 0, 0, None, PTR, 128, PTR, 128) == INVALID
    assert lib.sana_op_paged_attention_workspace(h, None, None, 8, 0, 0) == 0
    assert lib.sana_op_add_rms_norm_device(None, *NORM.values()) == INVALID  # no handle


ROT = dict(freq=PTR, rotated=64, interleaved=0, magnitude=1.0)


def rotate(lib, h, rot=ROT, **kw):
    a = dict(dtype=1, rows=4, D=64, pos=PTR, q=PTR, ldq=512, heads=8, qo=PTR, k=PTR, ldk=128, kv=2, ko=PTR)
    r = None if rot is None else ctypes.byref(capi.sana_rotary(*rot.values()))
    return lib.sana_op_rotary_device(h, r, *{**a, **kw}.values())


@pytest.mark.parametrize("change, word", [
    (dict(dtype=2), "dtype"), (dict(rows=-1), "sizes"), (dict(D=0), "sizes"), (dict(pos=None), "positions"),
    (dict(q=None), "q must"), (dict(qo=None), "q_out"), (dict(ko=None), "k_out"), (dict(ldq=500), "row stride"),
    (dict(ldk=100), "row stride"), (dict(rot=None), "rotary"), (dict(rot={**ROT, "rotated": 63}), "rotated"),
    (dict(rot={**ROT, "rotated": 66}), "rotated"), (dict(rot={**ROT, "freq": None}), "freq")])
def test_rotary_refusals(handle, change, word):
    lib, h, _ = handle
    assert rotate(lib, h, **change) == INVALID and word in message(lib, h)


def test_valid_calls_reach_the_device_check(handle):
    """Without a device the same calls, unchanged, fail for its absence and not for their arguments."""
    lib, h, created = handle
    if created:
        pytest.skip("a CUDA device is present")
    state = 4
    assert lib.sana_op_add_rms_norm_device(h, *NORM.values()) == state
    assert attend(lib, h) == state
    assert rotate(lib, h) == state
    b, c, r = batch(), cache(), capi.sana_rotary(*ROT.values())
    assert lib.sana_op_rotary_append_device(h, ctypes.byref(r), ctypes.byref(b), ctypes.byref(c), PTR, 512, 8, PTR, PTR, 128,
                                            PTR, 128) == state
