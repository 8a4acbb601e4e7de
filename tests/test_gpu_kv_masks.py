"""``FP8KVCache``: masked places, missing pages and NaN in every kernel's form, and forms that other tests pass by."""

from __future__ import annotations

import math

import pytest
import torch

import kv_rules as R
from test_gpu_kv_cache import DEV, batch, close, ints, make, queries

pytestmark = pytest.mark.gpu

# Sequences of up to 64 rows (tokens x query heads of a KV head) are the few-row kernel's, 4 and 24 of them in tiles of
# 16 and 32; calls of more than 1024 rows with longer ones take tiles of 128.  Pages of 64 and more, and heads
# of 64, 128, 192 and 256 channels, have forms of their own.
FORMS = [(64, 128), (64, 64), (64, 256), (64, 192), (128, 128), (256, 64), (128, 80), (32, 128)]


def lse_close(got, want):
    """The scores' error, and float32's own."""
    return bool(((got.double() - want).abs() <= 1e-4 + 2e-6 * want.abs()).logical_or(got.double() == want).all())


@pytest.mark.parametrize("page,dim", FORMS)
@pytest.mark.parametrize("new,window,prior", [(1, 0, 300), (1, 150, 300), (6, 0, 200), (6, 40, 300), (280, 0, 200), (280, 70, 300)])
def test_nan_reaches_only_those_who_see_it(page, dim, new, window, prior):
    kv, heads, pool = 2, 8, 48
    lengths, offsets, width = batch([new], [prior], page)
    n = lengths[0]
    c = make(1, pool, kv, dim, page, spread=0)
    table = R.spread_table(lengths, page, width, pool, 6)
    k, v = c.k.view(torch.uint8), c.v.view(torch.uint8)
    # everything that is not the sequence's is NaN, in codes and in scales
    others = [p for p in range(pool) if p not in table[0]]
    k[0, others], v[0, others] = 0x7F, 0xFF
    c.k_scales[0, others] = c.v_scales[0, others] = math.nan
    if n % page:
        last = table[0][(n - 1) // page]
        k[0, last, :, n % page:], v[0, last, :, :, n % page:] = 0x7F, 0xFF
    q = queries(new, heads, dim, torch.float16)
    call = (q, ints(table), ints(lengths), ints(offsets))
    want, bound, wl = R.attend(c, 0, q, table, lengths, offsets, dim ** -0.5, window)
    out, lse = c.attend(0, *call, window=window or None, return_lse=True)
    close(out, want, bound)
    assert lse_close(lse, wl)
    pos = torch.arange(n - new, n, device=DEV)
    for j in sorted({n - 1, n - 1 - new // 2, n - new, 190, max(0, n - new - window // 2)}):
        p, slot = table[0][j // page], j % page
        sees = (j <= pos) & (j > pos - window if window else pos >= 0)
        # of V: one channel of the second KV head's query heads
        kept = v[0, p, 1, 13, slot].clone()
        v[0, p, 1, 13, slot] = 0x7F if j % 2 else 0xFF
        out, lse = c.attend(0, *call, window=window or None, return_lse=True)
        v[0, p, 1, 13, slot] = kept
        assert torch.equal(out[:, 4:, 13].isnan(), sees[:, None].expand(-1, 4)), j
        close(torch.where(out.isnan(), want, out.double()), want, bound)
        assert int(out.isnan().sum()) == 4 * int(sees.sum()) and lse_close(lse, wl)
        # of K: those query heads' whole rows
        kept = k[0, p, 1, slot, 9].clone()
        k[0, p, 1, slot, 9] = 0x7F
        out = c.attend(0, *call, window=window or None)
        k[0, p, 1, slot, 9] = kept
        assert torch.equal(out.isnan(), (sees[:, None] & (torch.arange(heads, device=DEV) >= 4))[..., None].expand_as(out)), j
        close(torch.where(out.isnan(), want, out.double()), want, bound)
    # of a query: its own row
    q[new // 2, 3, 5] = math.nan
    out = c.attend(0, *call, window=window or None)
    assert bool(out[new // 2, 3].isnan().all()) and int(out.isnan().sum()) == dim
    close(torch.where(out.isnan(), want, out.double()), want, bound)


@pytest.mark.parametrize("page,dim", FORMS)
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [3, 5, 6, 1], [150, 290, 10, 200]])
@pytest.mark.parametrize("window", [0, 90])
def test_rows_that_see_nothing_and_missing_pages(page, dim, new, window):
    """More new tokens than the length, a length of 0, and entries that are no pages in the middle of a row, at its start and throughout."""
    kv, heads, pool = 2, 8, 60
    c = make(1, pool, kv, dim, page)
    width = max(-(-420 // page), 2) + 1
    first = [list(range(10 * i % 40, 10 * i % 40 + width)) for i in range(4)]
    table = [list(r) for r in first]
    table[1][1], table[2][0], table[3] = 2 ** 31 - 1, -7, [-1, pool] * width
    table[3] = table[3][:width]
    lengths = [max(0, new[0] - 60), 400, 410, 300]
    offsets = [sum(new[:i]) for i in range(5)]
    q = queries(sum(new), heads, dim, torch.bfloat16)
    out, lse = c.attend(0, q, ints(table), ints(lengths), ints(offsets), window=window or None, return_lse=True)
    want, bound, wl = R.attend(c, 0, q, table, lengths, offsets, dim ** -0.5, window)
    close(out, want, bound)
    assert lse_close(lse, wl)
    nothing = wl == -math.inf
    assert int(nothing.sum()) >= heads * (min(new[0], 60) + new[3])
    assert bool((out[nothing] == 0).all()) and bool((lse[nothing] == -math.inf).all())


@pytest.mark.parametrize("seqs", [256, 257, 1030])
@pytest.mark.parametrize("page,dim", [(64, 128), (16, 64)])
def test_drafts_of_many_sequences(seqs, page, dim):
    """Five tokens and four query heads a KV head are more than 16 rows a sequence, which go in tiles of 32."""
    new = [5 if i % 7 else 9 for i in range(seqs)]
    prior = [(11 * i) % 90 + (1500 if i % 301 == 5 else 0) for i in range(seqs)]
    lengths, offsets, width = batch(new, prior, page)
    pool = sum(R.pages_of(n, page) for n in lengths)
    c = make(1, pool, 1, dim, page)
    table = R.spread_table(lengths, page, width, pool, 4)
    q = queries(offsets[-1] + 2, 4, dim, torch.bfloat16)
    out, lse = c.attend(0, q, ints(table), ints(lengths), ints(offsets), return_lse=True)
    some = sorted({0, 1, 5, 254, 255, seqs // 2, seqs - 2, seqs - 1, *range(0, seqs, 37), *range(5, seqs, 301)})
    at = [t for i in some for t in range(offsets[i], offsets[i + 1])]
    few = [0]
    for i in some:
        few.append(few[-1] + new[i])
    want, bound, wl = R.attend(c, 0, q[at], [table[i] for i in some], [lengths[i] for i in some], few, dim ** -0.5, 0)
    close(out[at], want, bound)
    assert lse_close(lse[at], wl)
    assert bool((out[offsets[-1]:] == 0).all()) and bool((lse[offsets[-1]:] == -math.inf).all())
    assert bool((out[: offsets[-1]] != 0).any(-1).all()) and bool(lse[: offsets[-1]].isfinite().all())


@pytest.mark.parametrize("tokens,seqs", [(20, 3), (1200, 5)])
def test_the_sum_of_sequences_between_rows_of_none(tokens, seqs):
    """Rows before the first sequence and behind the last: the log-sum-exp of both kinds of row."""
    page, dim = 64, 128
    lead, tail = 4, 3
    ends = [lead + (tokens - lead - tail) * i // seqs for i in range(seqs + 1)]
    new = [b - a for a, b in zip(ends, ends[1:])]
    lengths = [n + 77 * i for i, n in enumerate(new)]
    width = max(R.pages_of(n, page) for n in lengths)
    pool = sum(R.pages_of(n, page) for n in lengths)
    c = make(1, pool, 1, dim, page)
    table = R.spread_table(lengths, page, width, pool, 1)
    q = queries(tokens, 2, dim, torch.bfloat16)
    out, lse = c.attend(0, q, ints(table), ints(lengths), ints(ends), return_lse=True)
    want, bound, wl = R.attend(c, 0, q, table, lengths, ends, dim ** -0.5, 0)
    close(out, want, bound)
    assert lse_close(lse, wl)
    assert int((wl == -math.inf).sum()) == 2 * (lead + tail) and bool((lse[:lead] == -math.inf).all()) and bool((lse[-tail:] == -math.inf).all())


@pytest.mark.parametrize("tokens", [1, 300])
def test_one_key_far_above_all_others(tokens):
    """Its score is 60 above every other in base e, so the result is its value to 2^-60 or so, however p is rounded."""
    page, dim, n, at = 64, 64, 3000, 1234
    pool = R.pages_of(n, page)
    c = make(1, pool, 1, dim, page, spread=0)
    table = [list(range(pool))]
    q = torch.ones(tokens, 4, dim, dtype=torch.bfloat16, device=DEV)
    c.k.copy_((c.k.float() / 8).clamp(-8, 8))  # sums of 64 of them, times a scale of 2^-4 and 1/8
    c.k[0, at // page, 0, at % page] = 224.0
    want, bound, wl = R.attend(c, 0, q, table, [n], [0, tokens], dim ** -0.5, 0)
    scores = (c.k[0].double() * c.k_scales[0].double()[..., None, None])[:, 0].reshape(-1, dim)[:n].sum(-1) * dim ** -0.5
    others = scores.clone()
    others[at] = -math.inf
    assert float(scores[at] - others.max()) > 60
    out, lse = c.attend(0, q, ints(table), ints([n]), ints([0, tokens]), return_lse=True)
    close(out, want, bound)
    assert lse_close(lse, wl)
    value = c.v[0, at // page, 0, :, at % page].float() * c.v_scales[0, at // page, 0]
    # e4m3 values times a power of two are bf16's own; p's part of the sum cancels to float32's error and fp16's rounding
    close(out, value.double().expand_as(out), value.double().abs() * (2.0 ** -8 + 2.0 ** -11) + 2.0 ** -60)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page,kv,dim", [(64, 8, 128), (16, 3, 48), (256, 1, 256), (32, 2, 16)])
def test_append_one_token_each(dtype, page, kv, dim):
    """Places at a page's first slot, inside it and at its last; values far above and below what the page holds, and none finite."""
    slots = [0, 1, page // 2, page - 1, page, 2 * page - 1, page + 3]
    rows = len(slots) + 2
    c = make(2, 2 * rows, kv, dim, page)
    want = R.Cache(c)
    table = R.spread_table([2 * page] * rows, page, 2, 2 * rows, 3)
    g = torch.Generator(device=DEV).manual_seed(8)
    k, v = (torch.randn(rows + 2, kv, dim, generator=g, device=DEV) * torch.randint(-12, 9, (rows + 2, kv, 1), generator=g, device=DEV).float().exp2()
            for _ in range(2))
    k[1, :, 3], v[2, :, 5], k[4], v[5] = math.inf, math.nan, 0.0, math.nan
    k[3, 0, 7], v[3, 0, 8] = 60000.0, -60000.0
    k, v = k.to(dtype), v.to(dtype)
    lengths = [s + 1 for s in slots] + [0, 2 * page + 9]  # no token, and one clamped to the table's last place
    c.append(1, k, v, ints(table), ints(lengths))
    want.append(1, k, v, table, lengths, None)
    want.same(c)
    c.append(0, v.transpose(0, 1).contiguous().transpose(0, 1), k, ints(table), ints(lengths))
    want.append(0, v, k, table, lengths, None)
    want.same(c)


def test_pages_of_no_row_stay_as_they_are():
    """Offsets that go back, on a pool of which every other page is no row's: what the claimed rows become is open, the other pages are not."""
    tokens, seqs, pool = 600, 2050, 600
    c = make(1, pool, 2, 64, 64)
    table = (torch.arange(seqs * 6, device=DEV, dtype=torch.int32) * 2 % pool).view(seqs, 6)
    rest = torch.ones(pool, dtype=torch.bool, device=DEV)
    rest[table.unique().long()] = False
    assert int(rest.sum()) == pool // 2
    kept = c.k.view(torch.uint8).clone(), c.v.view(torch.uint8).clone(), c.k_scales.clone(), c.v_scales.clone()
    lengths = torch.full((seqs,), 380, device=DEV, dtype=torch.int32)
    k = queries(tokens, 2, 64, torch.bfloat16)
    c.append(0, k, k, table, lengths, ints([tokens * (i % 2) for i in range(seqs + 1)]))
    now = c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scales, c.v_scales
    for a, b in zip(kept, now):
        assert torch.equal(a[:, rest], b[:, rest])
    assert not torch.equal(kept[0], now[0])
