"""Argument checks of the FP8 KV cache's counts and steps, none of which reaches a device."""

from __future__ import annotations

import ctypes

from lumenrl_amd import _lib
from test_kv_cache_abi import FAKE, append, attend, cache


def test_append_looks_at_counts_that_are_aligned():
    assert append(c=cache(refs=0x50002)) == _lib.ERR_ALIGN
    assert append(c=cache(refs=0x50002), tokens=0) == 0


def test_resize_ready():
    old, wanted, new, new_len = (ctypes.c_void_p(x) for x in (0xB00000, 0xC00000, 0x900000, 0xA00000))

    def resize(ready=None, c=None, lengths=old, want=wanted, out_len=new_len, short=FAKE, ws=FAKE, wb=1 << 40):
        return _lib.lib().lrq_kv_resize_ready(cache() if c is None else c, FAKE, 4, 4, lengths, 3, want, new, out_len, ready, short, ws, wb, None)

    for bad in ({"ready": ctypes.c_void_p(0xB00004)}, {"ready": wanted}, {"ready": ctypes.c_void_p(0x9FFFF8)}, {"c": cache(refs=None)},
                {"lengths": None}, {"want": None}, {"out_len": None}, {"short": None}, {"out_len": old}):
        assert resize(**bad) == _lib.ERR_ARG, bad
    assert resize(ready=ctypes.c_void_p(0xD00002)) == _lib.ERR_ALIGN
    need = _lib.lib().lrq_kv_resize_workspace(3, 10)
    assert resize(ready=ctypes.c_void_p(0xD00000), wb=need - 1) == _lib.ERR_CAPACITY and resize(ws=None) == _lib.ERR_CAPACITY


def test_attend_takes_finite_scales():
    for scale in (float("nan"), float("inf"), -float("inf"), 3e38, -3e38):
        assert attend(scale=scale) == _lib.ERR_ARG, scale
    assert attend(tokens=0, scale=2.0 ** 127) == 0 and attend(tokens=0, scale=0.0) == 0
