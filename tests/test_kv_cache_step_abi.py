"""Argument checks of the FP8 KV cache's counts and steps, none of which reaches a device."""

from __future__ import annotations

from lumenrl_amd import _lib
from test_kv_cache_abi import append, cache


def test_append_looks_at_counts_that_are_aligned():
    assert append(c=cache(refs=0x50002)) == _lib.ERR_ALIGN
    assert append(c=cache(refs=0x50002), tokens=0) == 0
