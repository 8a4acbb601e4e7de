"""Argument checks of the FP8 products, the router and the experts: none of them reaches a device."""

from __future__ import annotations

import ctypes

import pytest
import torch

from lumenrl_amd import _lib
from lumenrl_amd.quantization import fp8_block_linear, fp8_experts, fp8_matmul, route_experts

FAKE, ODD, OFF4 = ctypes.c_void_p(0x10000), ctypes.c_void_p(0x10001), ctypes.c_void_p(0x10004)


def L():
    return _lib.lib()


def test_fp8_matmul():
    def call(x=FAKE, xs=FAKE, rows=70, k=300, ld=300, codes=FAKE, scales=FAKE, n=64, bias=None, bdt=0, out=FAKE, dt=0, ws=None, wb=0):
        return L().lrq_fp8_matmul(x, xs, rows, k, ld, codes, scales, n, bias, bdt, out, dt, ws, wb, None)

    assert call(rows=0) == 0 and call(n=0) == 0
    for bad in ({"dt": 3}, {"dt": -1}, {"k": 0}, {"ld": 299}, {"rows": -1}, {"n": -1}, {"k": -1}, {"rows": (1 << 28) + 1},
                {"n": (1 << 26) + 1}, {"k": (1 << 22) + 1, "ld": 1 << 23}, {"ld": (1 << 22) + 1}, {"rows": 1 << 20, "n": (1 << 13) + 1},
                {"x": None}, {"xs": None}, {"codes": None}, {"scales": None}, {"out": None}, {"bias": FAKE, "bdt": 3}):
        assert call(**bad) == _lib.ERR_ARG, bad
    for bad in ({"xs": ODD}, {"scales": ODD}, {"out": ODD}, {"bias": ODD}, {"dt": 2, "out": ctypes.c_void_p(0x10002)}):
        assert call(**bad) == _lib.ERR_ALIGN, bad
    need = L().lrq_fp8_matmul_workspace(48, 4096, 4096)
    assert need == 4 * 48 * 4096 * 4  # four parts of K
    big = dict(rows=48, k=4096, ld=4096, n=4096)
    assert call(**big) == _lib.ERR_CAPACITY and call(**big, ws=FAKE, wb=need - 1) == _lib.ERR_CAPACITY
    assert call(**big, ws=OFF4, wb=need) == _lib.ERR_ALIGN


@pytest.mark.parametrize("rows,k,n,parts", [(4, 4096, 4096, 0), (5, 4096, 4096, 4), (64, 4096, 4096, 4), (65, 4096, 4096, 0),
                                            (48, 640, 64, 0), (48, 768, 64, 2), (48, 12288, 128, 32), (48, 4096, 12288, 0), (0, 4096, 64, 0)])
def test_parts_of_k_are_some_and_never_empty(rows, k, n, parts):
    assert L().lrq_fp8_matmul_workspace(rows, k, n) == 4 * parts * rows * n
    if parts:
        blocks = -(-k // 128)
        assert (parts - 1) * -(-blocks // parts) < blocks


def test_rows_that_are_not_aligned_are_copied_for_many_tokens():
    up = lambda v: -(-v // 256) * 256  # noqa: E731
    assert L().lrq_fp8_matmul_workspace(1536, 1041, 300) == up(300 * 1056) + up(1536 * 1056)
    assert L().lrq_fp8_matmul_workspace(1535, 1041, 300) == 0 and L().lrq_fp8_matmul_workspace(1536, 1044, 300) == 0
    assert L().lrq_fp8_block_linear_workspace(1536, 1041, 300) == up(1536 * 1056) + up(1536 * 9 * 4) + up(300 * 1056)
    assert L().lrq_fp8_matmul_workspace(1536, (1 << 22) - 1, 1 << 12) == 0  # more than 2 GiB of weight: as they are


def test_fp8_block_linear():
    def call(x=FAKE, dt=0, rows=70, k=300, ld=300, codes=FAKE, scales=FAKE, n=64, bias=None, bdt=0, out=FAKE, ws=FAKE, wb=1 << 30):
        return L().lrq_fp8_block_linear(x, dt, rows, k, ld, codes, scales, n, bias, bdt, out, ws, wb, None)

    assert call(rows=0) == 0 and call(n=0) == 0
    for bad in ({"dt": 3}, {"k": 0}, {"ld": 299}, {"rows": 1 << 27, "n": 1, "k": 2048, "ld": 2048}, {"rows": -1}, {"x": None}, {"codes": None}, {"scales": None}, {"out": None},
                {"bias": FAKE, "bdt": -1}, {"ld": (1 << 22) + 1}):
        assert call(**bad) == _lib.ERR_ARG, bad
    for bad in ({"x": ODD}, {"scales": ODD}, {"out": ODD}, {"bias": ODD}, {"ws": OFF4}):
        assert call(**bad) == _lib.ERR_ALIGN, bad
    need = L().lrq_fp8_block_linear_workspace(70, 300, 64)
    assert need == (70 * 304 + 255) // 256 * 256 + (70 * 3 * 4 + 255) // 256 * 256
    assert call(ws=None) == _lib.ERR_CAPACITY and call(wb=need - 1) == _lib.ERR_CAPACITY
    assert L().lrq_fp8_block_linear_workspace(4, 4096, 64) == 0 and L().lrq_fp8_block_linear_workspace(4, 1 << 20, 64) > 0


def test_route():
    def call(logits=FAKE, dt=0, tokens=8, experts=64, ld=64, bias=None, top_k=4, score=0, groups=1, top_groups=1, group_top=1,
             renorm=1, scale=1.0, weights=FAKE, ids=FAKE):
        return L().lrq_route(logits, dt, tokens, experts, ld, bias, top_k, score, groups, top_groups, group_top, renorm, scale,
                             weights, ids, None)

    assert call(tokens=0) == 0
    for bad in ({"dt": 3}, {"score": 2}, {"experts": 0, "ld": 0}, {"experts": 513, "ld": 513}, {"top_k": 0}, {"top_k": 65},
                {"top_k": 33, "experts": 32}, {"ld": 63}, {"tokens": -1}, {"groups": 0}, {"groups": 5}, {"groups": 32},
                {"groups": 4, "top_groups": 5}, {"groups": 4, "top_groups": 0}, {"groups": 16, "top_k": 5}, {"group_top": 0}, {"group_top": 3},
                {"logits": None}, {"weights": None}, {"ids": None}, {"ld": (1 << 31) + 1}):
        assert call(**bad) == _lib.ERR_ARG, bad
    for bad in ({"logits": ODD}, {"weights": ODD}, {"ids": ODD}, {"bias": ODD}):
        assert call(**bad) == _lib.ERR_ALIGN, bad


def test_route_grad():
    def call(logits=FAKE, dt=2, tokens=8, experts=64, ld=64, ids=FAKE, grad=FAKE, top_k=4, score=0, renorm=1, out=FAKE):
        return L().lrq_route_grad(logits, dt, tokens, experts, ld, ids, grad, top_k, score, renorm, 1.0, out, None)

    assert call(tokens=0) == 0
    for bad in ({"dt": 3}, {"score": -1}, {"experts": 513, "ld": 513}, {"top_k": 0}, {"top_k": 65}, {"ld": 63}, {"logits": None},
                {"ids": None}, {"grad": None}, {"out": None}):
        assert call(**bad) == _lib.ERR_ARG, bad
    for bad in ({"logits": ODD}, {"ids": ODD}, {"grad": ODD}, {"out": ODD}):
        assert call(**bad) == _lib.ERR_ALIGN, bad


def test_experts():
    def call(x=FAKE, dt=0, tokens=8, hidden=128, ld=128, ids=FAKE, weights=FAKE, top_k=2, gu=FAKE, gus=FAKE, dn=FAKE, dns=FAKE,
             experts=8, inter=64, out=FAKE, ws=FAKE, wb=1 << 40):
        return L().lrq_fp8_experts(x, dt, tokens, hidden, ld, ids, weights, top_k, gu, gus, dn, dns, experts, inter, out, ws, wb, None)

    assert call(tokens=0) == 0
    for bad in ({"dt": 2}, {"tokens": -1}, {"hidden": 120}, {"hidden": 0}, {"inter": 0}, {"inter": 65}, {"hidden": 1 << 15, "ld": 1 << 15, "inter": 1 << 15},
                {"experts": 0}, {"experts": 1025}, {"top_k": 0}, {"top_k": 65}, {"ld": 127}, {"x": None}, {"ids": None}, {"weights": None},
                {"gu": None}, {"gus": None}, {"dn": None}, {"dns": None}, {"out": None}):
        assert call(**bad) == _lib.ERR_ARG, bad
    for bad in ({"x": ODD}, {"ids": ODD}, {"weights": ODD}, {"gu": OFF4}, {"dn": OFF4}, {"gus": ODD}, {"dns": ODD}, {"out": OFF4}, {"ws": OFF4}):
        assert call(**bad) == _lib.ERR_ALIGN, bad
    assert call(ws=None) == _lib.ERR_CAPACITY and call(wb=0) == _lib.ERR_CAPACITY


@pytest.mark.parametrize("tokens", [1, 31, 32, 33, 5000, 300000])
def test_experts_workspace_grows_with_tokens_and_stays_bounded(tokens):
    """Passes hold at most 1 GiB of float32 results; the last one, of fewer tokens, may take other tiles."""
    ws = L().lrq_fp8_experts_workspace
    need = ws(tokens, 2048, 768, 128, 8)
    assert 0 < need < 2 << 30
    assert need >= ws(max(1, tokens // 2), 2048, 768, 128, 8)


def test_host_tensors_are_refused():
    w, s = torch.zeros(64, 128, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.ones(1, 1)
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    for call in (lambda: fp8_block_linear(x, w, s), lambda: fp8_matmul(w[:4], torch.ones(4, 1), w, s), lambda: route_experts(x, 4),
                 lambda: fp8_experts(x, torch.zeros(4, 2, dtype=torch.int32), torch.ones(4, 2), w[None], s[None], w[None], s[None])):
        with pytest.raises(ValueError, match="HIP device"):
            call()


@pytest.mark.parametrize("hidden,inter", [(16, 65536), (64, 16384), (256, 4096), (4096, 14336), (65536, 16)])
def test_experts_workspace_is_bounded_for_any_sizes(hidden, inter):
    """A pass holds at most 1 GiB of results and 1 GiB of hidden codes; their scales, x in codes and the pairs' order are no larger
    than those (a token's row of x is at most its pairs' results, blocks of 16 columns at least a quarter of their scale)."""
    ws = L().lrq_fp8_experts_workspace
    for tokens in (1 << 12, 1 << 16, 1 << 20, 1 << 28):
        assert 0 < ws(tokens, hidden, inter, 8, 2) < 4 << 30


def test_a_pass_of_the_experts_is_no_shorter_for_ordinary_sizes():
    """Up to an intermediate size of four times the hidden one, results alone bound it: 1 GiB of them."""
    ws = L().lrq_fp8_experts_workspace
    for hidden, inter in ((2048, 768), (4096, 14336), (2048, 8192)):
        tokens = (1 << 28) // (2 * hidden)
        assert ws(tokens, hidden, inter, 8, 2) > 1 << 30
        assert ws(4 * tokens, hidden, inter, 8, 2) == ws(tokens, hidden, inter, 8, 2)
