"""``FP8KVCache`` in the hands of its caller: derivatives that are asked for, and tensors whose memory moves."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import kv_rules as R
from test_gpu_kv_cache import close, ints, make, queries

pytestmark = pytest.mark.gpu


def test_tangents_are_refused_not_lost():
    c = make(1, 4, 1, 64, 16)
    table, lengths = ints([[0, 1]]), ints([20])
    k, q = queries(1, 1, 64, torch.bfloat16), queries(1, 2, 64, torch.bfloat16)
    kept = c.k.view(torch.uint8).clone(), c.v.view(torch.uint8).clone()
    plain = c.attend(0, q, table, lengths)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(k, torch.ones_like(k))
        for pair in ((dual, k), (k, dual)):
            with pytest.raises(RuntimeError, match="no gradient"):
                c.append(0, *pair, table, lengths)
            with torch.no_grad(), pytest.raises(RuntimeError, match="no gradient"):
                c.append(0, *pair, table, lengths)
        turned = forward_ad.make_dual(*(torch.ones(1, 64, 1, dtype=k.dtype, device=k.device) for _ in range(2)))
        with pytest.raises(RuntimeError, match="no gradient"):
            c.append(0, turned.transpose(1, 2), k, table, lengths)
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            c.attend(0, dual, table, lengths)
        with pytest.raises(RuntimeError, match="no gradient"):
            c.attend(0, dual, table, lengths, out=torch.empty_like(q))
        assert torch.equal(kept[0], c.k.view(torch.uint8)) and torch.equal(kept[1], c.v.view(torch.uint8))
        # tensors that have none are as good there as anywhere
        out = torch.empty_like(q)
        assert torch.equal(c.attend(0, q, table, lengths), plain) and torch.equal(c.attend(0, q, table, lengths, out=out), plain)
        c.append(0, k, k, table, lengths)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: c.append(0, x, x, table, lengths) or x, (k,), (torch.ones_like(k),))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: c.attend(0, x, table, lengths), (q,), (torch.ones_like(q),))


def test_memory_that_is_freed_and_put_back():
    c = make(1, 6, 2, 64, 16)
    table, lengths, wanted = ints([[0, 1, -1], [3, -1, -1]]), ints([20, 7]), ints([33, 8])
    c.refs.copy_(ints([1, 1, 0, 1, 0, 0]))
    k, q = queries(2, 2, 64, torch.bfloat16), queries(2, 4, 64, torch.bfloat16)

    def calls():
        return [lambda: c.append(0, k, k, table, lengths), lambda: c.attend(0, q, table, lengths), lambda: c.fork(table, lengths, lengths),
                lambda: c.resize(table, lengths, wanted), lambda: c.compact(table)]

    want = c.attend(0, q, table, lengths)
    for name in ("k", "v", "k_scales", "v_scales", "refs"):
        x = getattr(c, name)
        saved, size = x.view(torch.uint8).clone(), x.untyped_storage().nbytes()
        for left in (0, size // 2):
            x.untyped_storage().resize_(left)
            for call in calls():
                with pytest.raises(RuntimeError, match=f"memory of {name} has been freed"):
                    call()
        held = torch.empty(size, dtype=torch.uint8, device=x.device)  # what was freed is someone else's now
        x.untyped_storage().resize_(size)
        x.view(torch.uint8).copy_(saved)
        assert torch.equal(c.attend(0, q, table, lengths), want)
        # and memory of another tensor
        x.data = saved.clone().view(x.dtype)
        assert torch.equal(c.attend(0, q, table, lengths), want)
        assert torch.equal(saved, getattr(c, name).view(torch.uint8))
        del held
    # what is written goes where the tensors are
    old = c.k.data
    c.k.data = c.k.view(torch.uint8).clone().view(c.k.dtype)
    rules = R.Cache(c)
    c.append(0, k, k, table, lengths)
    rules.append(0, k, k, table.tolist(), lengths.tolist(), None)
    rules.same(c)
    assert not torch.equal(old.view(torch.uint8), c.k.view(torch.uint8))
    c.refs.data = ints([0, 1, 0, 1, 0, 0])
    t, n, short = c.resize(table, lengths, wanted)
    assert t.tolist() == [[0, 1, 0], [3, -1, -1]] and c.refs.tolist() == [1, 1, 0, 1, 0, 0]
    # tensors that do not fit any more are refused as they would be at first, until they do
    good = c.v.data
    c.v.data = good[:, :5].clone()
    for _ in range(2):
        with pytest.raises(ValueError, match="v must be"):
            c.attend(0, q, table, lengths)
    c.v.data = good
    c.attend(0, q, table, lengths)
    with pytest.raises(AttributeError):
        c.k = good


@pytest.mark.parametrize("tokens", [1, 400])  # 400: by tiles of many rows
def test_windows_and_scales_of_any_size(tokens):
    c = make(1, 40, 1, 64, 16)
    table, lengths, offsets = ints([list(range(40))]), ints([640]), ints([0, tokens])
    q = queries(tokens, 4, 64, torch.bfloat16)
    plain = c.attend(0, q, table, lengths, offsets)
    for window in (640, 1 << 30, (1 << 31) - 1, 1 << 32, (1 << 32) + 3, 1 << 63, (1 << 64) + 3, 1 << 90):
        assert torch.equal(c.attend(0, q, table, lengths, offsets, window=window), plain), window
    for window in (0, -1, -(1 << 64) + 3, 2.5, 64.0, "3"):
        with pytest.raises(ValueError, match="window"):
            c.attend(0, q, table, lengths, offsets, window=window)
    for scale in (float("nan"), float("inf"), -float("inf"), 1e300, -3e38):
        with pytest.raises(ValueError, match="scale"):
            c.attend(0, q, table, lengths, offsets, scale=scale)
    # the sign is the queries', and 0 takes the mean of what is seen
    want, bound, _ = R.attend(c, 0, -q, table.tolist(), [640], [0, tokens], 0.125, 0)
    got = c.attend(0, q, table, lengths, offsets, scale=-0.125)
    close(got, want, bound)
    want, bound, _ = R.attend(c, 0, q, table.tolist(), [640], [0, tokens], 0.0, 0)
    close(c.attend(0, q, table, lengths, offsets, scale=0.0), want, bound)


@pytest.mark.parametrize("page,dim,tokens", [(64, 128, 3), (16, 80, 3), (64, 128, 300), (32, 80, 300)])  # few rows and tiles, a page or less a unit
@pytest.mark.parametrize("kind", ["any", "large", "small", "range"])
def test_scales_of_a_callers_own(page, dim, tokens, kind):
    """Scales that are no powers of two, V's over all of the range in which they are taken; beyond it they are the nearest in it.

    Beside what the bound holds already, log2 of a scale and 2^ of it are approximate: 2^-22 of an exponent of up to 64, 2^-16 ln 2."""
    keys = 700
    pool = R.pages_of(keys, page) + 1
    c = make(1, pool, 1, dim, page, spread=0)
    g = torch.Generator(device="cuda").manual_seed(4)
    c.k_scales.copy_(0.004 + 0.006 * torch.rand(c.k_scales.shape, generator=g, device="cuda"))
    spread = torch.rand(c.v_scales.shape, generator=g, device="cuda", dtype=torch.float64)
    c.v_scales.copy_({"any": 0.01 + spread, "large": 2.0 ** (40 + 8 * spread), "small": 2.0 ** (-48 + 8 * spread),
                       "range": 2.0 ** (-48 + 96 * spread)}[kind])
    table = R.spread_table([keys], page, pool, pool, 2)
    q = queries(tokens, 4, dim, torch.bfloat16)
    out, lse = c.attend(0, q, ints(table), ints([keys]), ints([0, tokens]), return_lse=True)
    want, bound, wl = R.attend(c, 0, q, table, [keys], [0, tokens], dim ** -0.5, 0)
    size, _, _ = R.attend(_sizes(c), 0, q, table, [keys], [0, tokens], dim ** -0.5, 0)
    close(out, want, bound - 2.0 ** -32 + 2.0 ** -134 + 2.0 ** -16 * size)  # (half a step of the smallest number is fp16's there, bf16's here)
    assert bool(((lse.double() - wl).abs() <= 1e-4 + 2e-6 * wl.abs()).all())
    p = table[0]
    for inside, beyond in ((2.0 ** 48, 2.0 ** 90), (2.0 ** -48, 2.0 ** -100), (2.0 ** -48, 0.0)):
        c.v_scales[0, p[1]] = c.v_scales[0, p[2]] = inside
        want = c.attend(0, q, ints(table), ints([keys]), ints([0, tokens]))
        c.v_scales[0, p[1]] = c.v_scales[0, p[2]] = beyond
        assert torch.equal(c.attend(0, q, ints(table), ints([keys]), ints([0, tokens])), want), beyond


class _sizes:
    """A cache whose values are their sizes."""

    def __init__(self, c):
        self.__dict__.update({n: getattr(c, n) for n in ("k", "k_scales", "v_scales", "kv_heads", "page", "pages")})
        self.v = c.v.float().abs()


def test_a_caches_tensors_are_written_in_place():
    c = make(1, 4, 1, 64, 16)
    refs, scales = c.refs, c.k_scales.clone()
    c.refs += 1
    c.k_scales *= 2
    assert c.refs is refs and c.refs.tolist() == [1] * 4 and torch.equal(c.k_scales, scales * 2)
    for name in ("k", "v", "k_scales", "v_scales", "refs"):
        with pytest.raises(AttributeError):
            setattr(c, name, getattr(c, name).clone())
    assert c.refs is refs
