"""``route_experts`` against its definition in float64: the choice exactly, weights and gradients within float32's roundings."""

from __future__ import annotations

import math

import pytest
import torch

from lumenrl_amd.quantization import route_experts

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def scores(x, score):
    return torch.sigmoid(x) if score == "sigmoid" else torch.softmax(x, -1)


def choose(logits, top_k, score="softmax", bias=None, groups=1, top_groups=1, group_top=1, **_):
    """ids, row by row, from float64 picks on the host: NaN highest, then the value, then the lowest index."""
    x = logits.detach().double().cpu()
    pick = scores(x, score)
    if bias is not None:
        pick = pick + bias.double().cpu()
    elif groups == 1 or group_top == 1:
        pick = x
    out = []
    for xs, row in zip(x.tolist(), pick.tolist()):
        e = len(row)
        size = e // groups

        def rank(v):
            return (0, 0.0) if math.isnan(v) else (1, -v)

        def value(g):
            best = sorted(row[g * size: (g + 1) * size], key=rank)[:group_top]
            return sum(best)

        open_groups = sorted(range(groups), key=lambda g: (rank(value(g)), g))[:top_groups]
        cand = [i for g in open_groups for i in range(g * size, (g + 1) * size)]
        order = xs if bias is None else row
        out.append(sorted(cand, key=lambda i: (rank(order[i]), i))[:top_k])
    return torch.tensor(out, dtype=torch.int64).reshape(*x.shape[:-1], top_k)


def weigh(x, ids, score="softmax", renormalize=True, scale=1.0, **_):
    """float64 weights of chosen experts, differentiable."""
    if score == "softmax" and renormalize:
        return scale * torch.softmax(x.gather(-1, ids), -1)
    s = scores(x, score).gather(-1, ids)
    if renormalize:
        s = s / (s.sum(-1, keepdim=True) + 1e-20)
    return scale * s


def units(x):
    """Relative error in units of 2^-24: exp's argument carries a rounding of its own size; 10 for sums of up to 512
    by halves, 12 for exp, additions, divisions and the factor."""
    return (x.amax(-1, keepdim=True) - x.amin(-1, keepdim=True) + x.abs().amax(-1, keepdim=True) + 22) * 2.0 ** -24


def check(logits, top_k, **kw):
    w, ids = route_experts(logits, top_k, **kw)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32 and ids.shape == w.shape == (*logits.shape[:-1], top_k)
    flat = logits.detach().reshape(-1, logits.shape[-1])
    want_ids = choose(flat, top_k, **kw)
    assert torch.equal(ids.reshape(-1, top_k).long().cpu(), want_ids)
    x = flat.double().cpu()
    want = weigh(x, want_ids, **kw)
    off = (w.detach().reshape(-1, top_k).cpu().double() - want).abs()
    assert bool((off <= units(x) * want.abs() + 2.0 ** -140).all())
    return w, want_ids


CONFIGS = [
    dict(),
    dict(renormalize=False, scale=16.0),
    dict(score="sigmoid"),
    dict(score="sigmoid", renormalize=False, scale=0.5),
    dict(score="sigmoid", bias=True, groups=8, top_groups=4, group_top=2, scale=2.5),
    dict(score="softmax", bias=True),
    dict(score="softmax", bias=True, groups=4, top_groups=2, group_top=1),
    dict(score="softmax", groups=8, top_groups=3, group_top=1, renormalize=False),
    dict(score="softmax", groups=4, top_groups=3, group_top=2),
    dict(score="sigmoid", groups=8, top_groups=8, group_top=2),
]
EXPERTS = [(8, 1), (32, 4), (64, 6), (72, 3), (104, 12), (128, 8), (160, 6), (200, 17), (256, 8), (264, 9), (512, 64)]


def inputs(tokens, e, dtype, kw, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(tokens, e, generator=g, device=DEV) * 1.5 + torch.randn(e, generator=g, device=DEV) * 0.5).to(dtype)
    kw = dict(kw)
    if kw.get("bias"):
        kw["bias"] = torch.randn(e, generator=g, device=DEV) * 0.1
    return x, kw


@pytest.mark.parametrize("kw", CONFIGS, ids=lambda k: "-".join(str(v) for v in k.values()) or "plain")
@pytest.mark.parametrize("e,top_k", EXPERTS)
@pytest.mark.parametrize("dtype", TYPES)
def test_choice_and_weights(dtype, e, top_k, kw):
    top_k = min(top_k, e // kw.get("groups", 1) * kw.get("top_groups", 1))
    x, kw = inputs(37, e, dtype, kw, e)
    check(x, top_k, **kw)


@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 1000])
def test_token_counts(tokens):
    for kw in CONFIGS[::4]:
        x, kw = inputs(tokens, 64, torch.float32, kw, tokens)
        check(x, 4, **kw)


@pytest.mark.parametrize("kw", CONFIGS[4:7])
def test_near_ties_are_told_apart(kw):
    """Picks closer than float32 resolves: the same sums by other logits and biases, one unit apart."""
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(64, 128, generator=g, device=DEV)
    kw = dict(kw)
    # a bias that all but levels the scores of token 0, which other tokens share with noise of 1e-7
    kw["bias"] = (0.75 - scores(x[0].double(), kw["score"])).float()
    x[1:] = x[0] + torch.randn(63, 128, generator=g, device=DEV) * 1e-7
    check(x, 8, **kw)


@pytest.mark.parametrize("kw", [dict(), CONFIGS[2], CONFIGS[4], CONFIGS[6], CONFIGS[8]])
@pytest.mark.parametrize("dtype", TYPES)
def test_ties_go_to_the_lowest_index(dtype, kw):
    g = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randint(-2, 3, (50, 96), generator=g, device=DEV).to(dtype)
    x[0] = 0.0
    x[1, ::2] = -0.0
    x[1, 1::2] = 0.0
    kw = dict(kw)
    if kw.get("bias"):
        kw["bias"] = torch.zeros(96, device=DEV)
    check(x, 8, **kw)


@pytest.mark.parametrize("kw", [dict(), dict(renormalize=False), CONFIGS[2], CONFIGS[4], CONFIGS[5], CONFIGS[7], CONFIGS[8]])
@pytest.mark.parametrize("dtype", TYPES)
def test_inf_nan_and_masked_logits(dtype, kw):
    x, kw = inputs(12, 64, dtype, kw, 9)
    x[0, 5] = float("nan")
    x[1] = float("-inf")
    x[2, 3:] = float("-inf")
    x[3, 40] = float("inf")
    x[4, [1, 63]] = float("nan")
    x[5] = torch.finfo(dtype).min
    x[6] = torch.finfo(dtype).max
    x[7, 10:] = torch.finfo(dtype).min
    top_k = 4
    w, ids = route_experts(x, top_k, **kw)
    if kw.get("groups", 1) == 1 or kw.get("bias") is None:  # a masked expert's pick ties with nothing closed
        assert torch.equal(ids.long().cpu(), choose(x, top_k, **kw))
    assert bool(((ids >= 0) & (ids < 64)).all()) and all(len(set(r)) == top_k for r in ids.tolist())
    check(x[8:], top_k, **kw)
    if kw.get("score", "softmax") == "softmax":
        assert bool(w[0].isnan().all()) and bool(w[1].isnan().all())
    else:
        assert bool((w[1] == 0).all())
    assert bool(w[7].isfinite().all())


def test_strides_leading_dims_empty_and_none_of_it_copied_wrong():
    big = torch.randn(40, 3 * 64 + 5, device=DEV)
    for x in (big[:, 5:69], big[::2, 1:65], big[:, :128:2], big.t()[:40].t(), big[:1].expand(7, -1)[:, :64]):
        check(x, 6)
    check(torch.randn(3, 5, 64, device=DEV), 6)
    check(torch.randn(64, device=DEV), 6)
    w, ids = route_experts(torch.zeros(0, 64, device=DEV), 6)
    assert w.shape == ids.shape == (0, 6)
    x = torch.zeros(0, 64, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(route_experts(x, 6)[0].sum(), x)
    assert g.shape == (0, 64)


# ---------------------------------------------------------------------------
# gradient
# ---------------------------------------------------------------------------
def formula_grad(x, ids, grad, **kw):
    x = x.detach().double().cpu().requires_grad_()
    w = weigh(x, ids.cpu(), **{k: v for k, v in kw.items() if k != "bias"})
    (g,) = torch.autograd.grad(w, x, grad.double().cpu())
    return g


def check_grad(x, top_k, grad=None, **kw):
    x = x.detach().requires_grad_()
    w, ids = check(x, top_k, **kw)
    grad = torch.randn(w.shape, device=DEV) if grad is None else grad
    (got,) = torch.autograd.grad(w, x, grad)
    assert got.dtype == x.dtype and got.shape == x.shape
    want = formula_grad(x.reshape(-1, x.shape[-1]), ids, grad.reshape(-1, top_k), **kw)
    xd = x.detach().reshape(-1, x.shape[-1]).double().cpu()
    # every term of dx_i is a weight times at most (|g_i| + sum |g w| / scale); each with the weights' error, sums of top_k
    # more; 1 - s of sigmoid counts as the rest.  Then the rounding to x's type
    w64 = weigh(xd, ids, **{k: v for k, v in kw.items() if k != "bias"})
    g64 = grad.reshape(-1, top_k).double().cpu().abs()
    s = scores(xd, kw.get("score", "softmax")) if not kw.get("renormalize", True) else torch.zeros_like(xd).scatter(
        1, ids, w64 / kw.get("scale", 1.0))
    dense = torch.zeros_like(xd).scatter(1, ids, g64) * kw.get("scale", 1.0)
    size = s * (dense + (g64 * w64.abs()).sum(-1, keepdim=True))
    got = got.reshape(-1, x.shape[-1]).double().cpu()
    half = torch.finfo(x.dtype).eps / 2
    least = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -140}[x.dtype]
    bound = half * want.abs() * 1.01 + least + (3 * units(xd) + top_k * 2.0 ** -24) * size
    off = (got - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())
    return got


@pytest.mark.parametrize("kw", CONFIGS, ids=lambda k: "-".join(str(v) for v in k.values()) or "plain")
@pytest.mark.parametrize("e,top_k", [(8, 1), (72, 3), (128, 8), (160, 6), (264, 9), (512, 64)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_is_the_formulas(dtype, e, top_k, kw):
    top_k = min(top_k, e // kw.get("groups", 1) * kw.get("top_groups", 1))
    x, kw = inputs(35, e, dtype, kw, e + 1)
    check_grad(x, top_k, **kw)


@pytest.mark.parametrize("kw", [dict(), dict(renormalize=False, scale=2.0), dict(score="sigmoid"), dict(score="sigmoid", renormalize=False)])
def test_gradient_is_that_of_differences(kw):
    """Central differences of the float64 weights at step h: their own error is h^2 / 6 of a third derivative below 2 scale,
    and 2^-52 / h of rounding; the kernel's is float32's."""
    torch.manual_seed(5)
    x = torch.randn(3, 16, device=DEV, requires_grad=True)
    w, ids = route_experts(x, 4, **kw)
    c = torch.randn(w.shape, device=DEV)
    (got,) = torch.autograd.grad((w * c).sum(), x)
    xd, cd, idd, h = x.detach().double().cpu(), c.double().cpu(), ids.long().cpu(), 1e-4
    for t in range(3):
        for e in range(16):
            up, down = xd.clone(), xd.clone()
            up[t, e] += h
            down[t, e] -= h
            slope = ((weigh(up, idd, **kw) - weigh(down, idd, **kw)) * cd).sum() / (2 * h)
            scale = kw.get("scale", 1.0) * float(cd[t].abs().sum())
            assert abs(float(got[t, e]) - float(slope)) <= scale * (h * h + 2e-12 + 80 * 2.0 ** -24)


def test_gradient_of_broadcast_and_strided_gradients():
    x = torch.randn(20, 64, device=DEV)
    check_grad(x, 5, torch.ones(1, 1, device=DEV).expand(20, 5))
    check_grad(x, 5, torch.randn(5, 20, device=DEV).t(), score="sigmoid")
    wide = torch.randn(20, 70, device=DEV)
    check_grad(wide[:, 3:67], 5, renormalize=False)
    leaf = torch.randn(64, device=DEV, requires_grad=True)
    w, ids = route_experts(leaf.expand(9, 64), 5)
    c = torch.randn(9, 5, device=DEV)
    (got,) = torch.autograd.grad(w, leaf, c)
    want = formula_grad(leaf.expand(9, 64), ids.long(), c).sum(0)
    assert torch.allclose(got.double().cpu(), want, rtol=0, atol=9 * 80 * 2.0 ** -24 * float(c.abs().max()))


def test_the_choice_takes_no_gradient_and_no_graph_without_one():
    x = torch.randn(4, 32, device=DEV, requires_grad=True)
    bias = torch.zeros(32, device=DEV, requires_grad=True)
    w, ids = route_experts(x, 3, bias=bias)
    assert w.requires_grad and not ids.requires_grad
    assert torch.autograd.grad(w.sum(), [x, bias], allow_unused=True)[1] is None
    with torch.no_grad():
        assert not route_experts(x, 3)[0].requires_grad
    y = x * 1.0
    w, _ = route_experts(y, 3)
    (g,) = torch.autograd.grad(w[:, 0].sum(), x, create_graph=True)
    assert g.requires_grad
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    w, _ = route_experts(y, 3)
    y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        w.sum().backward()


def test_other_stream_and_graph():
    x = torch.randn(33, 128, device=DEV)
    want = route_experts(x, 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = route_experts(x, 8)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w, ids = route_experts(x, 8)
    for seed in range(3):
        x.copy_(torch.randn(33, 128, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV))
        graph.replay()
        want = route_experts(x, 8)
        assert torch.equal(w, want[0]) and torch.equal(ids, want[1])


def test_refusals():
    x = torch.zeros(4, 32, device=DEV)
    for kw, err in [(dict(top_k=0), ValueError), (dict(top_k=33), ValueError), (dict(top_k=4, score="relu"), ValueError),
                    (dict(top_k=4, groups=5), ValueError), (dict(top_k=4, groups=8, top_groups=9), ValueError),
                    (dict(top_k=5, groups=8, top_groups=1), ValueError), (dict(top_k=4, group_top=3), ValueError),
                    (dict(top_k=4, groups=32), ValueError), (dict(top_k=4, bias=torch.zeros(31, device=DEV)), ValueError),
                    (dict(top_k=4, bias=torch.zeros(32)), ValueError),
                    (dict(top_k=4, bias=torch.zeros(32, device=DEV, dtype=torch.bfloat16)), TypeError)]:
        with pytest.raises(err, match="route_experts"):
            route_experts(x, **kw)
    with pytest.raises(ValueError, match="512"):
        route_experts(torch.zeros(2, 513, device=DEV), 4)
    with pytest.raises(TypeError):
        route_experts(x.double(), 4)
    with pytest.raises(ValueError):
        route_experts(torch.zeros(4, 32), 4)


@pytest.mark.parametrize("kw", [dict(), dict(renormalize=False), dict(score="sigmoid")])
def test_forward_and_gradient_in_a_graph(kw):
    """Captured on leaves that no eager graph holds (torch ties a leaf's gradient to the stream of the graph that lives)."""
    x = torch.randn(40, 64, device=DEV, requires_grad=True)
    c = torch.randn(40, 4, device=DEV)

    def step():
        w, ids = route_experts(x, 4, **kw)
        return w.detach(), ids, torch.autograd.grad(w, x, c)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in range(3):
        x.data.copy_(torch.randn(40, 64, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_far_rows_and_wide_pitches():
    """Rows past 2^31 elements of the logits' storage."""
    big = torch.zeros((1 << 31) + 4096, dtype=torch.bfloat16, device=DEV)
    view = big.as_strided((5, 64), (1 << 29, 1))
    view.copy_(torch.randn(5, 64, device=DEV))
    check(view, 6)
    check_grad(view, 6, renormalize=False)


INF = float("inf")


@pytest.mark.parametrize("logits,bias,top_k", [
    ([0.0, -100.0, -100.0, -90.0], None, 2), ([0.0, -1e4, -1e4, -70.0], None, 2), ([0.0, -INF, -INF, -70.0], None, 2),
    ([1e-4, 1e-4, 1.01e-4], None, 1), ([0.0] * 100 + [1e-6] + [0.0] * 27, None, 1), ([5.0, -INF, -INF, -INF, -200.0, -INF], None, 2),
    ([3e38, 1.0, 1.0, 2.0], None, 2), ([0.0] * 300 + [2e-7, 1e-7], None, 2),
    ([0.0, 0.0, 0.0, 0.0], [0.0, -10.0, -10.0, -9.0], 2), ([0.0] * 4, [0.0, -INF, -INF, -9.0], 2),
    ([1.0] * 6, [0.5, 0.5, 0.5, 0.5 + 2.0 ** -24, 0.5, 0.5 + 2.0 ** -24], 1), ([20.0, 1.0, 1.0, 1.5, 1.0], [0.0] * 5, 2),
    ([20.0, -1.0, -1.0, -1.0, 2.0, 2.0, 2.5], [0.0] * 7, 3)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_a_tie_at_the_border_does_not_settle_it(logits, bias, top_k, score):
    """The last chosen and the next one are equal, and a higher one stands behind them, too near to them, or too far below the
    highest, for the words that order experts to tell."""
    x = torch.tensor([logits] * 3, device=DEV)
    kw = {"score": score}
    if bias is not None:
        kw["bias"] = torch.tensor(bias, device=DEV)
    _, ids = route_experts(x, top_k, **kw)
    assert torch.equal(ids.long().cpu(), choose(x, top_k, **kw))


@pytest.mark.parametrize("groups", [1, 4])
@pytest.mark.parametrize("kw", [dict(), dict(bias=0.0), dict(bias=1.0), dict(bias=30.0), dict(score="sigmoid", bias=0.0),
                                dict(score="sigmoid", bias=1.0), dict(score="sigmoid", bias=30.0)], ids=str)
@pytest.mark.parametrize("e,top_k", [(64, 2), (128, 8), (256, 8), (512, 20)])
def test_ties_among_near_neighbours(e, top_k, kw, groups):
    """Few distinct logits and biases, near one another or far below the highest, in every order: bf16 logits of a small spread
    widened to float32, confident experts above a crowd, masks of -inf and of large negative values with live experts below them."""
    g = torch.Generator(device=DEV).manual_seed(e + top_k)

    def some(values):
        return torch.tensor(values, device=DEV)[torch.randint(0, len(values), (64, e), generator=g, device=DEV)]

    rows = [(torch.randn(64, e, generator=g, device=DEV) * 1e-4).bfloat16().float(), some([1.0, 1.0 + 2.0 ** -22, 1.0 + 2.0 ** -23]),
            (torch.randn(64, e, generator=g, device=DEV) * 2).bfloat16().float(), some([-100.0, -90.0, -70.0, -1e4, -INF]),
            some([-100.0, -90.0, -70.0]), some([0.0, 1e-7, 2e-7, -1e-7])]
    for r in (2, 3, 4):  # confident experts above
        rows[r][torch.arange(64, device=DEV), torch.randint(0, e, (64,), generator=g, device=DEV)] = 20.0
    x = torch.cat(rows)
    kw = dict(kw, groups=groups, top_groups=(groups + 1) // 2, group_top=2 if groups > 1 else 1)
    if "bias" in kw:
        few = torch.tensor([0.0, -1.0, -1.0 + 2.0 ** -23, -0.5], device=DEV)
        kw["bias"] = few[torch.randint(0, 4, (e,), generator=g, device=DEV)] * kw["bias"]
    _, ids = route_experts(x, top_k, **kw)
    assert torch.equal(ids.long().cpu(), choose(x, top_k, **kw))


@pytest.mark.parametrize("kw", [k for k in CONFIGS if k.get("groups", 1) > 1], ids=str)
@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_groups_with_nan_infinite_and_masked_logits(dtype, zero, kw):
    """Every row against the definition: a group with a NaN is the highest, groups that are masked as a whole rank by their biases."""
    x, kw = inputs(12, 64, dtype, kw, 9)
    if zero and kw.get("bias") is not None:
        kw["bias"] = torch.zeros(64, device=DEV)
    x[0, 5] = float("nan")
    x[1] = -INF
    x[2, 3:] = -INF
    x[3, 40] = INF
    x[4, [1, 63]] = float("nan")
    x[5] = torch.finfo(dtype).min
    x[6] = torch.finfo(dtype).max
    x[7, 10:] = torch.finfo(dtype).min
    x[8, [3, 17, 33]] = INF
    x[9, 8:56] = -INF
    x[10, ::2] = torch.finfo(dtype).min
    _, ids = route_experts(x, 4, **kw)
    assert torch.equal(ids.long().cpu(), choose(x, 4, **kw))


def test_rows_more_than_2_31_elements_apart():
    big = torch.zeros(2 * ((1 << 31) + 8) + 64, dtype=torch.bfloat16, device=DEV)
    view = big.as_strided((3, 64), ((1 << 31) + 8, 1))
    view.copy_(torch.randn(3, 64, device=DEV))
    check(view, 6)
    check_grad(view, 6)


def test_more_tokens_than_a_launch_takes():
    """2^28 + 5 tokens of two experts; with 16 threads a token more than the 2^32 of one launch."""
    t = (1 << 28) + 5
    x = torch.randn(t, 2, dtype=torch.bfloat16, device=DEV).requires_grad_()
    w, ids = route_experts(x, 1, score="sigmoid", renormalize=False)
    second = x.detach()[:, 1] > x.detach()[:, 0]
    assert torch.equal(ids[:, 0] == 1, second)
    (g,) = torch.autograd.grad(w, x, torch.ones(1, 1, device=DEV).expand(t, 1))
    for rows in (slice(0, 1000), slice((1 << 27) - 500, (1 << 27) + 500), slice((1 << 28) - 995, None)):
        s = torch.sigmoid(x.detach()[rows].double()).gather(1, ids[rows].long())
        assert bool(((w[rows].double() - s).abs() <= 40 * 2.0 ** -24 * s).all())
        want = torch.zeros(len(s), 2, dtype=torch.float64, device=DEV).scatter(1, ids[rows].long(), s * (1 - s))
        assert bool(((g[rows].double() - want).abs() <= 1.01 * 2.0 ** -8 * want).all())
