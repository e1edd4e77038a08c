"""More of what the text encoder's entry points refuse, without a GPU (see test_encoder_ops.py)."""
import ctypes

import pytest

from sana_b200 import capi
from test_encoder_ops import INVALID, NORM, PTR, ROT, attend, batch, cache, handle, message, rotate  # noqa: F401


@pytest.mark.parametrize("change, word", [
    (dict(x=PTR + 2), "x must be aligned"), (dict(x=PTR + 1, xt=1), "x must be aligned"), (dict(out=PTR + 2), "out must be aligned"),
    (dict(out=PTR + 1, ot=1), "out must be aligned"), (dict(r=PTR + 2), "residual must be aligned"), (dict(sum=PTR + 2), "sum must be aligned"),
    (dict(w=PTR + 1), "weight must be aligned"), (dict(ot=2, scale=PTR + 2), "scale must be aligned")])
def test_norm_refuses_misaligned_elements(handle, change, word):
    lib, h, _ = handle
    assert lib.sana_op_add_rms_norm_device(h, *{**NORM, **change}.values()) == INVALID and word in message(lib, h)


@pytest.mark.parametrize("change, word", [
    (dict(q=PTR + 1), "q must be"), (dict(qo=PTR + 1), "q_out must be"), (dict(k=PTR + 3), "k must be"), (dict(ko=PTR + 1), "k_out must be"),
    (dict(dtype=0, q=PTR + 2), "q must be"), (dict(pos=PTR + 2), "positions must be"), (dict(rot={**ROT, "freq": PTR + 4}), "freq must be")])
def test_rotary_refuses_misaligned_elements(handle, change, word):
    lib, h, _ = handle
    assert rotate(lib, h, **change) == INVALID and word in message(lib, h)


@pytest.mark.parametrize("b, c, kw, word", [
    ({}, {}, dict(q=PTR + 1), "q must be"), ({}, {}, dict(out=PTR + 1), "out must be"), ({}, dict(k=PTR + 1), {}, "k of the cache"),
    ({}, dict(v=PTR + 2, dtype=0), {}, "v of the cache"), (dict(row_start=PTR + 2), {}, {}, "row_start must be"),
    (dict(kv_len=PTR + 1), {}, {}, "kv_len must be"), (dict(page_table=PTR + 2), {}, {}, "page_table must be")])
def test_attention_and_append_refuse_misaligned_elements(handle, b, c, kw, word):
    lib, h, _ = handle
    bb, cc = batch(**b), cache(**c)
    assert attend(lib, h, b=bb, c=cc, **kw) == INVALID and word in message(lib, h)
    if not kw:
        assert lib.sana_op_rotary_append_device(h, None, ctypes.byref(bb), ctypes.byref(cc), None, 0, 0, None, PTR, 128, PTR,
                                                128) == INVALID and word in message(lib, h)


@pytest.mark.parametrize("change, word", [(dict(k=PTR + 1), "k must be"), (dict(v=PTR + 1), "v must be"), (dict(q=PTR + 1), "q must be"),
                                          (dict(qo=PTR + 1), "q_out must be")])
def test_append_refuses_misaligned_rows(handle, change, word):
    lib, h, _ = handle
    b, c, r = batch(), cache(), capi.sana_rotary(*ROT.values())
    a = {**dict(q=PTR, ldq=512, heads=8, qo=PTR, k=PTR, ldk=128, v=PTR, ldv=128), **change}
    assert lib.sana_op_rotary_append_device(h, ctypes.byref(r), ctypes.byref(b), ctypes.byref(c), *a.values()) == INVALID
    assert word in message(lib, h)


@pytest.mark.parametrize("change", [dict(ldx=72), dict(ldo=72), dict(ot=1), dict(ot=2, scale=PTR)])
def test_norm_in_place_needs_the_same_rows(handle, change):
    """Another row stride or element size would write rows that other blocks still read."""
    lib, h, created = handle
    assert lib.sana_op_add_rms_norm_device(h, *{**NORM, **change}.values()) == INVALID and "out may be x" in message(lib, h)
    if not created:  # a single row may: the argument check passes, and the missing device is reported
        assert lib.sana_op_add_rms_norm_device(h, *{**NORM, **change, "rows": 1}.values()) == 4
