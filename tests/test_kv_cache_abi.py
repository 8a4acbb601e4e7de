"""Argument checks of the FP8 KV cache, none of which reaches a device, and the rules that its GPU tests go by."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import kv_rules as R
from lumenrl_amd import _lib
from lumenrl_amd.quantization import FP8KVCache

FAKE, ODD, OFF4 = ctypes.c_void_p(0x10000), ctypes.c_void_p(0x10001), ctypes.c_void_p(0x10004)
CACHE = dict(k=0x10000, v=0x20000, k_scales=0x30000, v_scales=0x40000, refs=0x50000, layers=2, pages=10, kv_heads=2, page=64, dim=128,
             k_layer=163840, v_layer=163840, ks_layer=20, vs_layer=20, k_page=16384, v_page=16384, ks_page=2, vs_page=2)


def L():
    return _lib.lib()


def cache(**kw):
    return ctypes.byref(_lib.LrqKvCache(**{**CACHE, **kw}))


def append(c=None, layer=0, k=FAKE, kt=256, kh=128, v=FAKE, vt=256, vh=128, dt=0, tokens=5, table=FAKE, ld=4, width=4, lengths=FAKE,
           offsets=FAKE, seqs=3, ws=None, wb=0):
    return L().lrq_kv_append(cache() if c is None else c, layer, k, kt, kh, v, vt, vh, dt, tokens, table, ld, width, lengths, offsets, seqs, ws, wb,
                             None)


def attend(c=None, layer=0, q=FAKE, qt=1024, qh=128, dt=0, tokens=5, heads=8, table=FAKE, ld=4, width=4, lengths=FAKE, offsets=FAKE,
           seqs=3, scale=1.0, window=0, zero=1, out=FAKE, lse=None, ws=FAKE, wb=1 << 40):
    return L().lrq_kv_attend(cache() if c is None else c, layer, q, qt, qh, dt, tokens, heads, table, ld, width, lengths, offsets, seqs,
                             scale, window, zero, out, lse, ws, wb, None)


BAD_CACHES = [{"page": 48}, {"page": 8}, {"page": 512}, {"page": 0}, {"page": -64}, {"dim": 24}, {"dim": 272}, {"dim": 0}, {"kv_heads": 0},
              {"kv_heads": 257}, {"pages": 0}, {"pages": (1 << 28) + 1}, {"layers": -1}, {"layers": 65537}, {"k": None}, {"v": None},
              {"k_scales": None}, {"v_scales": None}]
FAR_CACHES = [{"k": 0x10008}, {"v": 0x10004}, {"k_scales": 0x30002}, {"k_page": 16385}, {"v_layer": 8}, {"k_page": -16384}, {"ks_page": -2},
              {"v_page": 1 << 60}]
BAD_SEQS = [{"layer": -1}, {"layer": 2}, {"tokens": -1}, {"tokens": (1 << 22) + 1}, {"seqs": -1}, {"seqs": (1 << 20) + 1, "offsets": None},
            {"width": -1}, {"width": 1 << 25}, {"ld": 3}, {"table": None}, {"lengths": None}, {"offsets": None, "seqs": 6}]


def test_append():
    assert append(tokens=0) == 0 and append(seqs=0) == 0 and append(width=0) == 0
    for bad in BAD_SEQS + [{"dt": 3}, {"dt": -1}, {"k": None}, {"v": None}, {"kt": -1}, {"vh": -128}, {"kt": 1 << 50},
                           {"tokens": 1 << 22, "seqs": 1 << 20, "c": cache(kv_heads=128, k_page=1 << 20, v_page=1 << 20)}]:
        assert append(**bad) == _lib.ERR_ARG, bad
    for bad in ({"k": ODD}, {"v": ODD}, {"table": ODD}, {"lengths": ODD}, {"offsets": ODD}, {"dt": 2, "k": ctypes.c_void_p(0x10002)}):
        assert append(**bad) == _lib.ERR_ALIGN, bad
    need = L().lrq_kv_append_workspace(257, 0)
    assert need > 0 and append(seqs=257, ws=FAKE, wb=need - 1) == _lib.ERR_CAPACITY and append(seqs=257) == _lib.ERR_CAPACITY
    assert append(seqs=257, ws=OFF4, wb=need) == _lib.ERR_ALIGN
    assert L().lrq_kv_append_workspace(256, 0) == 0 and L().lrq_kv_append_workspace(1000, 1) == 0 and L().lrq_kv_append_workspace(-1, 0) == 0
    for bad in BAD_CACHES:
        assert append(c=cache(**bad)) == _lib.ERR_ARG, bad
    for bad in FAR_CACHES:
        assert append(c=cache(**bad)) == _lib.ERR_ALIGN, bad
    assert append(c=ctypes.c_void_p(None)) == _lib.ERR_ARG


def test_attend():
    assert attend(tokens=0) == 0
    for bad in BAD_SEQS + [{"dt": 2}, {"dt": 3}, {"heads": 0}, {"heads": 7}, {"heads": 4098}, {"window": -1}, {"q": None}, {"out": None},
                           {"qt": -1}, {"qh": 1 << 50}]:
        assert attend(**bad) == _lib.ERR_ARG, bad
    for bad in ({"q": ODD}, {"out": OFF4}, {"lse": ODD}, {"table": ODD}, {"ws": OFF4}):
        assert attend(**bad) == _lib.ERR_ALIGN, bad
    need = L().lrq_kv_attend_workspace(5, 8, 2, 128, 3, 0)
    assert need > 0 and attend(ws=None) == _lib.ERR_CAPACITY and attend(wb=need - 1) == _lib.ERR_CAPACITY
    assert L().lrq_kv_attend_workspace(5, 8, 2, 300, 3, 0) == 0 and L().lrq_kv_attend_workspace(-1, 8, 2, 128, 3, 0) == 0
    for bad in BAD_CACHES:
        assert attend(c=cache(**bad)) == _lib.ERR_ARG, bad
    for bad in FAR_CACHES:
        assert attend(c=cache(**bad)) == _lib.ERR_ALIGN, bad


def test_upkeep():
    new, new_len, other = ctypes.c_void_p(0x900000), ctypes.c_void_p(0xA00000), ctypes.c_void_p(0xB00000)

    def fork(c=None, table=FAKE, ld=4, width=4, lengths=other, rows=3, parents=FAKE, out=new, out_len=new_len):
        return L().lrq_kv_fork(cache() if c is None else c, table, ld, width, lengths, rows, parents, out, out_len, None)

    def resize(c=None, table=FAKE, ld=4, width=4, lengths=other, rows=3, wanted=FAKE, out=new, out_len=new_len, short=FAKE, ws=FAKE, wb=1 << 40):
        return L().lrq_kv_resize(cache() if c is None else c, table, ld, width, lengths, rows, wanted, out, out_len, short, ws, wb, None)

    def compact(c=None, table=FAKE, ld=4, width=4, rows=3, out=new, count=FAKE, ws=FAKE, wb=1 << 40):
        return L().lrq_kv_compact(cache() if c is None else c, table, ld, width, rows, out, count, ws, wb, None)

    assert fork(rows=0) == 0
    common = [{"rows": -1}, {"rows": (1 << 20) + 1}, {"width": -1}, {"width": 1 << 25}, {"ld": 3}, {"table": None}, {"out": None},
              {"out": ctypes.c_void_p(0x10010)}, {"c": cache(refs=None)}]
    for bad in common + [{"lengths": None}, {"parents": None}, {"out_len": None}, {"out_len": other}]:
        assert fork(**bad) == _lib.ERR_ARG, bad
    for bad in common + [{"lengths": None}, {"wanted": None}, {"out_len": None}, {"out_len": ctypes.c_void_p(0xB00004)}, {"short": None}]:
        assert resize(**bad) == _lib.ERR_ARG, bad
    for bad in common + [{"count": None}]:
        assert compact(**bad) == _lib.ERR_ARG, bad
    for call, need in ((resize, L().lrq_kv_resize_workspace(3, 10)), (compact, L().lrq_kv_compact_workspace(10))):
        assert need > 0 and call(ws=None) == _lib.ERR_CAPACITY and call(wb=need - 1) == _lib.ERR_CAPACITY and call(ws=OFF4) == _lib.ERR_ALIGN
    for call in (fork, resize, compact):
        for bad in BAD_CACHES:
            assert call(c=cache(**bad)) == _lib.ERR_ARG, bad
        for bad in FAR_CACHES:
            assert call(c=cache(**bad)) == _lib.ERR_ALIGN, bad
        assert call(table=ODD) == _lib.ERR_ALIGN


def test_a_cache_is_on_a_device():
    k = torch.zeros(1, 4, 2, 16, 32, dtype=torch.uint8).view(R.E4M3)
    s = torch.ones(1, 4, 2)
    with pytest.raises(ValueError, match="HIP device"):
        FP8KVCache(k, k.view(1, 4, 2, 32, 16), s, s, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(TypeError):
        FP8KVCache(k, k.view(1, 4, 2, 32, 16), s.half(), s, torch.zeros(4, dtype=torch.int32))
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError):
            FP8KVCache.empty(1, 4, 2, 32)


def test_the_rules_grid_is_e4m3():
    codes = torch.arange(256, dtype=torch.uint8).view(R.E4M3).double()
    fin = codes[codes.isfinite()]
    assert torch.equal(R.grid(fin), fin)
    x = torch.linspace(-470, 470, 20001, dtype=torch.float64).float()
    got, want = R.grid(x.double()), x.to(R.E4M3).double()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("amax", [1.0, 448.0, 448.1, 447.9, 0.0, 3e38, 1e-40, 1.75, 1.7500001, 7.0, 2.0 ** -48])
def test_the_rules_scale(amax):
    s = R.scale_of(amax)
    assert math.frexp(s)[0] == 0.5 and 2.0 ** -48 <= s <= 2.0 ** 48
    assert s == 2.0 ** 48 or amax <= 448 * s
    assert s == 2.0 ** -48 or amax > 448 * s / 2


def test_the_rules_of_pages():
    class C:
        page = 16
        k = torch.zeros(1, 6, 1, 16, 16)
        v = torch.zeros(1, 6, 1, 16, 16)
        k_scales = v_scales = torch.zeros(1, 6, 1)
        refs = torch.tensor([1, 0, 2, 0, 0, 1], dtype=torch.int32)

    for p in range(6):
        C.k[0, p] = p
    c = R.Cache(C)
    table, lens = c.fork([[2, 5], [2, 0], [-1, -1]], [20, 30, 0], [0, 1, 0])
    assert table == [[2, 5], [2, 0], [2, 5]] and lens == [20, 30, 20] and c.refs == [1, 0, 3, 0, 0, 2]
    table, lens, short = c.resize(table, lens, [32, 0, 21])
    assert table == [[2, 0], [-1, -1], [2, 1]] and lens == [32, 0, 21] and short == 0 and c.refs == [1, 1, 2, 0, 0, 0]
    assert float(c.k[0, 0, 0, 0, 0]) == float(c.k[0, 1, 0, 0, 0]) == 5.0
    table, lens, short = c.resize(table, lens, [32, 32, 60])
    assert lens == [32, 32, 21] and short == 0  # three pages, of a table of two, are not looked for
    table, lens, short = c.resize([[2, 0], table[1], [2, 1]], [32, 0, 21], [32, 0, 16])
    table, n = c.compact(table)
    assert n == len([x for x in c.refs if x > 0])
