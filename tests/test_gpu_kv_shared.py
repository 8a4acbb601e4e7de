"""``FP8KVCache`` where rows share pages and free ones run out: what other rows hold stays as it is."""

from __future__ import annotations

import ctypes
import random

import pytest
import torch

import kv_rules as R
from lumenrl_amd import _lib
from test_gpu_kv_cache import DEV, close, ints, make, queries

pytestmark = pytest.mark.gpu


class Rules(R.Cache):
    """The rules, where pages that more than one row holds are not written."""

    def append(self, layer, k, v, table, lengths, offsets):
        shared = {p for p, n in enumerate(self.refs) if n > 1}
        super().append(layer, k, v, [[-1 if p in shared else p for p in row] for row in table], lengths, offsets)

    def resize_ready(self, table, lengths, wanted):
        table, lengths, short = self.resize(table, lengths, wanted)
        return table, lengths, short, [n if n == w else 0 for n, w in zip(lengths, wanted)]


def tokens(n, kv, dim, dtype, seed, size=2.0 ** 6):
    """Keys or values far above what a cache of ``make`` holds, so that a page which they join has to be rounded again."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(n, kv, dim, generator=g, device=DEV) * size).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("page,kv,dim", [(16, 2, 48), (64, 3, 128), (256, 1, 256)])
def test_a_shared_page_is_not_written(dtype, page, kv, dim):
    c = make(2, 9, kv, dim, page)
    want = Rules(c)
    # rows 0 and 1 hold page 4 and end in it; 2 has it before one of its own; 3 has its own alone
    table = [[4, -1], [4, -1], [4, 7], [2, 8]]
    for x in (c.refs, want.refs):
        for p, n in ((4, 3), (7, 1), (2, 1), (8, 1)):
            x[p] = n
    k, v = tokens(4, kv, dim, dtype, 1), tokens(4, kv, dim, dtype, 2)
    lengths = [11, 11, page + 3, page + 1]
    c.append(1, k, v, ints(table), ints(lengths))
    want.append(1, k, v, table, lengths, None)
    want.same(c)
    # several tokens each: of row 2 two would be in the shared page, of row 3 five are in its first and three in its second
    offsets = [0, 3, 4, 10, 18]
    k, v = tokens(18, kv, dim, dtype, 3, 2.0 ** 9), tokens(18, kv, dim, dtype, 4, 2.0 ** 9)
    lengths = [13, 12, page + 4, page + 3]
    was = c.k.view(torch.uint8)[:, 4].clone(), c.v.view(torch.uint8)[:, 4].clone(), c.k_scales[:, 4].clone(), c.v_scales[:, 4].clone()
    c.append(1, k, v, ints(table), ints(lengths), ints(offsets))
    want.append(1, k, v, table, lengths, offsets)
    want.same(c)
    for a, b in zip(was, (c.k.view(torch.uint8)[:, 4], c.v.view(torch.uint8)[:, 4], c.k_scales[:, 4], c.v_scales[:, 4])):
        assert torch.equal(a, b)
    # held by one row alone, it is
    c.refs[4] = want.refs[4] = 1
    c.append(1, k[:1], v[:1], ints(table[:1]), ints([12]))
    want.append(1, k[:1], v[:1], table[:1], [12], None)
    want.same(c)
    assert not torch.equal(was[0], c.k.view(torch.uint8)[:, 4])


def test_a_cache_without_counts():
    """The C entry without refs has no shared pages."""
    c = make(1, 3, 1, 64, 16)
    c.refs.fill_(2)
    want = R.Cache(c)
    k = tokens(3, 1, 64, torch.bfloat16, 1)
    t, n, offsets = ints([[1], [2]]), ints([4, 9]), ints([0, 1, 3])
    desc = _lib.LrqKvCache.from_buffer_copy(c._desc)
    desc.refs = None
    for where in (offsets, None):
        rc = _lib.lib().lrq_kv_append(ctypes.byref(desc), 0, k.data_ptr(), 64, 64, k.data_ptr(), 64, 64, 0, 3, t.data_ptr(), 1, 1, n.data_ptr(),
                                      None if where is None else where.data_ptr(), 2, None, 0, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        want.append(0, k, k, t.tolist(), n.tolist(), None if where is None else where.tolist())
        want.same(c)


def test_a_shared_page_is_not_written_among_many_sequences():
    """More sequences than a work-group looks over: every third row holds the page before it as well."""
    page, kv, dim, rows = 16, 1, 32, 900
    c = make(1, rows, kv, dim, page)
    want = Rules(c)
    table = [[r - 1 if r % 3 == 2 else r] for r in range(rows)]
    want.refs = [[1, 2, 0][r % 3] for r in range(rows)]
    c.refs.copy_(ints(want.refs))
    new, lengths = [1 + r % 2 for r in range(rows)], [2 + r % 15 for r in range(rows)]
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    k, v = tokens(offsets[-1], kv, dim, torch.bfloat16, 1), tokens(offsets[-1], kv, dim, torch.bfloat16, 2)
    c.append(0, k, v, ints(table), ints(lengths), ints(offsets))
    want.append(0, k, v, table, lengths, offsets)
    want.same(c)


def whole(n, kv, dim, seed):
    """Keys or values that e4m3 holds exactly, in a page's scale and in any larger one that such values ask for."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(-15, 16, (n, kv, dim), generator=g, device=DEV).bfloat16()


def cached(c, codes, scales, layer, row, n):
    """The first n tokens of a row, [n, kv_heads, dim]."""
    idx = torch.tensor(row[: R.pages_of(n, c.page)], dtype=torch.long, device=DEV)
    x = codes[layer].view(torch.uint8)[idx].view(R.E4M3).float() * scales[layer][idx][..., None, None]
    if codes is c.v:
        x = x.transpose(2, 3)
    return x.transpose(1, 2).reshape(-1, c.kv_heads, c.dim)[:n]


@pytest.mark.parametrize("several", [False, True])
def test_a_refused_row_costs_no_one_a_token(several):
    """Four samples of a prompt, and pages for two of them to go on in: the others' new tokens are left out, everyone's old ones stay."""
    page, kv, dim, heads = 16, 2, 64, 4
    c = make(2, 5, kv, dim, page)
    c.refs.zero_()
    prompt = whole(40, kv, dim, 1)
    t, n, _, ready = c.resize(ints([[-1] * 4] * 4), ints([0] * 4), ints([40, 0, 0, 0]), return_ready=True)
    assert ready.tolist() == [40, 0, 0, 0]
    c.append(1, prompt, -prompt, t, ready, ints([0, 40, 40, 40, 40]))
    t, n = c.fork(t, n, ints([0] * 4))
    want = Rules(c)
    new = [2, 1, 3, 1] if several else [1] * 4
    offsets = [sum(new[:i]) for i in range(5)] if several else None
    wanted = [40 + x for x in new]
    table, lengths = t.tolist(), n.tolist()
    t, n, short, ready = c.resize(t, n, ints(wanted), return_ready=True)
    table, lengths, missing, now = want.resize_ready(table, lengths, wanted)
    assert t.tolist() == table and n.tolist() == lengths == [40 + new[0], 40 + new[1], 40, 40]
    assert int(short) == missing == 2 and ready.tolist() == now == [40 + new[0], 40 + new[1], 0, 0]
    k, v = tokens(sum(new), kv, dim, torch.bfloat16, 2), tokens(sum(new), kv, dim, torch.bfloat16, 3)
    c.append(1, k, v, t, ready, None if offsets is None else ints(offsets))
    want.append(1, k, v, table, now, offsets)
    want.same(c)
    for r in (2, 3):
        assert torch.equal(cached(c, c.k, c.k_scales, 1, table[r], 40), prompt.float())
        assert torch.equal(cached(c, c.v, c.v_scales, 1, table[r], 40), -prompt.float())
    q = queries(sum(new), heads, dim, torch.bfloat16)
    out, lse = c.attend(1, q, t, ready, None if offsets is None else ints(offsets), return_lse=True)
    exact, bound, _ = R.attend(c, 1, q, table, now, offsets, dim ** -0.5, 0)
    close(out, exact, bound)
    refused = slice(new[0] + new[1], None)
    assert bool((out[refused] == 0).all()) and bool((lse[refused] == -torch.inf).all()) and bool((out[: new[0] + new[1]] != 0).any(-1).all())
    # one ends, and there is room for the others
    t, n, short, ready = c.resize(t, n, ints([0, *wanted[1:]]), return_ready=True)
    table, lengths, missing, now = want.resize_ready(table, lengths, [0, *wanted[1:]])
    assert t.tolist() == table and n.tolist() == lengths and int(short) == missing and ready.tolist() == now


def test_a_row_as_long_as_the_table_is_wide():
    page, kv, dim = 16, 1, 32
    c = make(1, 9, kv, dim, page)
    c.refs.copy_(ints([1, 1, 1] + [0] * 6))
    want = Rules(c)
    t, n, short, ready = c.resize(ints([[0, 1], [2, -1]]), ints([32, 5]), ints([33, 6]), return_ready=True)
    assert t.tolist() == [[0, 1], [2, -1]] and n.tolist() == [32, 6] and int(short) == 0 and ready.tolist() == [0, 6]
    k = tokens(2, kv, dim, torch.bfloat16, 1)
    for offsets in (None, [0, 1, 2]):
        c.append(0, k, k, t, ready, None if offsets is None else ints(offsets))
        want.append(0, k, k, t.tolist(), [0, 6], offsets)
        want.same(c)
    t, n, short, ready = c.resize(t, n, ints([-3, 2 ** 31 - 1]), return_ready=True)
    assert n.tolist() == [0, 6] and ready.tolist() == [0, 0] and int(short) == 0
    t, n, short, ready = c.resize(t[:0], n[:0], ints([]), return_ready=True)
    assert ready.shape == (0,)


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("one_each", [False, True])
def test_steps_of_a_pool_that_runs_out(captured, one_each):
    """Samples decode until pages and the table's width run out, some end, others are forked from who is left.  Whatever was
    granted is in the cache, token for token, and nothing else has changed it."""
    page, kv, dim, heads, rows, width, pool = 16, 2, 32, 4, 8, 4, 13
    rnd = random.Random(3)
    c = make(1, pool, kv, dim, page)
    c.refs.zero_()
    most = rows if one_each else 3 * rows
    table, lengths, wanted = ints([[-1] * width] * rows), ints([0] * rows), ints([0] * rows)
    offsets = None if one_each else ints([0] * (rows + 1))
    k, v = (torch.zeros(most, kv, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q = queries(most, heads, dim, torch.bfloat16)

    def step():
        t, n, short, ready = c.resize(table, lengths, wanted, return_ready=True)
        c.append(0, k, v, t, ready, offsets)
        out = c.attend(0, q, t, ready, offsets)
        table.copy_(t), lengths.copy_(n)
        return short, ready, out

    if captured:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        c.refs.zero_(), table.fill_(-1), lengths.zero_()
    kept = [[torch.zeros(0, kv, dim, device=DEV)] * 2 for _ in range(rows)]
    refused = shorts = 0
    for i in range(60):
        if i % 9 == 8:  # half of them end, and are forked from the one after
            t, n, _ = c.resize(table, lengths, lengths * ints([(r + i // 9) % 2 for r in range(rows)]))
            parents = [r if (r + i // 9) % 2 else (r + 1) % rows for r in range(rows)]
            t, n = c.fork(t, n, ints(parents))
            table.copy_(t), lengths.copy_(n)
            kept = [kept[p] for p in parents]
        had = lengths.tolist()
        new = [1] * rows if one_each else [rnd.randrange(4) for _ in range(rows)]
        if i == 0 and not one_each:
            new = [3] * rows
        wanted.copy_(ints([a + b for a, b in zip(had, new)]))
        ends = [sum(new[:r]) for r in range(rows + 1)]
        if offsets is not None:
            offsets.copy_(ints(ends))
        k.copy_(whole(most, kv, dim, 2 * i)), v.copy_(whole(most, kv, dim, 2 * i + 1))
        if captured:
            graph.replay()
            short, ready, out = got
            if i % 5 == 0:
                torch.cuda.synchronize()
        else:
            short, ready, out = step()
        now, t, n = ready.tolist(), table.tolist(), lengths.tolist()
        shorts += int(short) > 0
        exact, bound, _ = R.attend(c, 0, q, t, now, None if one_each else ends, dim ** -0.5, 0)
        close(out, exact, bound)
        for r in range(rows):
            part = slice(ends[r], ends[r + 1])
            if had[r] + new[r] == n[r]:
                assert now[r] == n[r]
                kept[r] = [torch.cat([kept[r][0], k[part].float()]), torch.cat([kept[r][1], v[part].float()])]
            else:
                assert now[r] == 0 and n[r] == had[r]
                assert bool((out[part] == 0).all())
                refused += 1
            assert torch.equal(cached(c, c.k, c.k_scales, 0, t[r], n[r]), kept[r][0]), (i, r)
            assert torch.equal(cached(c, c.v, c.v_scales, 0, t[r], n[r]), kept[r][1]), (i, r)
    assert refused > 20 and shorts > 5
