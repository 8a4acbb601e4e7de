"""``FP8KVCache`` where rows share pages and free ones run out: what other rows hold stays as it is."""

from __future__ import annotations

import pytest
import torch

import kv_rules as R
from test_gpu_kv_cache import DEV, ints, make

pytestmark = pytest.mark.gpu


class Rules(R.Cache):
    """The rules, where pages that more than one row holds are not written."""

    def append(self, layer, k, v, table, lengths, offsets):
        shared = {p for p, n in enumerate(self.refs) if n > 1}
        super().append(layer, k, v, [[-1 if p in shared else p for p in row] for row in table], lengths, offsets)


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
