"""CPU: prompt attention's host side - what the C entry points take, and where the HF backend sends what the kernels do not compute."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

OK, ARG = 0, -1


def desc(b=1024, h=128, t=128):
    from tq_local_b200.runtime.ffi import DenseDesc

    return C.byref(DenseDesc(4096, 1, b, h, t))


def test_strides_of_axes_with_one_element_are_not_looked_at():
    """No query or no sequence: strides are checked, nothing is launched."""
    from tq_local_b200.runtime import ffi

    plain = desc()
    call = lambda q=plain, k=plain, v=plain, out=plain, b=1, hq=1, hkv=1, n=0, m=1: ffi.lib().tq_prompt_attn(
        q, k, v, b, hq, hkv, n, m, None, 0.1, 1, None, 0, out, None)
    assert call() == OK
    for odd in (desc(b=3), desc(h=5), desc(t=7), desc(3, 5, 7)):
        for name in ("q", "k", "v", "out"):
            assert call(**{name: odd}) == OK
    for many, odd in ((dict(b=2), desc(b=3)), (dict(hq=2, hkv=2), desc(h=5)), (dict(m=2), desc(t=7))):
        for name in ("k", "v") if "m" in many else ("q", "k", "v", "out"):
            assert call(**many, **{name: odd}) == ARG
    assert call(hq=2, k=desc(h=5)) == OK and call(hq=2, q=desc(h=5)) == ARG
    packed = lambda d, n=0, total=8, h=2: ffi.lib().tq_prompt_attn_packed(d, d, d, n, total, h, h, 4096, 8, 0.1, 1, None, 0, d, None)
    assert packed(desc(b=3)) == OK and packed(desc(h=5)) == ARG and packed(desc(t=7)) == ARG
    assert packed(desc(h=5), h=1) == OK and packed(desc(t=7), total=1) == OK
