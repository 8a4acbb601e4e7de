"""``FP8KVCache`` in the hands of its caller: derivatives that are asked for, and tensors whose memory moves."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from test_gpu_kv_cache import ints, make, queries

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
