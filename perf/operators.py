"""The FP8 rollout operators on 128x128-tile weights, and the expert router beside them.

``kind`` names the operator of a case:

* ``linear``   ``fp8_block_linear``: activations quantized to e4m3 in 1x128 blocks, times a
  weight in 128x128 tiles (the layout ``quantize_fp8_blockwise`` writes)
* ``matmul``   ``fp8_matmul``: the product alone, of codes and scales made earlier
* ``route``    ``route_experts``: scores, balance bias, groups, top-k, renormalised weights
* ``train``    the router in a training step: its weights and the gradient of the logits
* ``experts``  ``fp8_experts``: the chosen experts' SwiGLU MLPs and their weighted sum

Sizes are those of Qwen3-8B's linears and Qwen3-30B-A3B's experts, or generic ones of the
same range.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZES = {"bf16": 2, "f16": 2, "f32": 4}
_E4M3 = torch.float8_e4m3fn
_B = 128
_TINY = 2.0 ** -126
_MOST_MACS = 8192 * 4096 * 12288
_MOST_EXPERT_MACS = 4096 * 8 * 2048 * 768 * 3
_MOST_EXPERT_WEIGHTS = 128 * 2048 * 768 * 3


def _api():
    pkg = os.path.join(os.getcwd(), "lumen-rl_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import lumenrl_amd.quantization as q

    return q


def listed():
    return [
        # o_proj for the one token of a single decoding sequence: the smallest product, latency counts
        {"name": "linear_decode_1", "kind": "linear", "dtype": "bf16", "tokens": 1, "k": 4096, "n": 4096, "bias": False},
        # down_proj for a decoding step of 48 sequences, K three times as long as N is wide
        {"name": "linear_decode_48", "kind": "linear", "dtype": "bf16", "tokens": 48, "k": 12288, "n": 4096, "bias": False},
        # gate_proj over the prompts of a rollout batch: the largest product
        {"name": "linear_prefill_8192", "kind": "linear", "dtype": "bf16", "tokens": 8192, "k": 4096, "n": 12288, "bias": False},
        # no size a multiple of 16: ragged tokens, a cut weight, a last K block of 76, float32 out
        {"name": "matmul_odd", "kind": "matmul", "dtype": "f32", "tokens": 777, "k": 1100, "n": 1500, "bias": True},
        # q_proj over 2048 tokens whose codes serve q, k and v
        {"name": "matmul_prefill_2048", "kind": "matmul", "dtype": "bf16", "tokens": 2048, "k": 4096, "n": 4096, "bias": False},
        # routing of a decoding step of 64 sequences to 8 of 128 experts: launch latency
        {"name": "route_decode_64", "kind": "route", "dtype": "bf16", "tokens": 64, "experts": 128, "top_k": 8,
         "score": "softmax", "bias": False, "groups": 1, "top_groups": 1, "group_top": 1, "renormalize": True, "scale": 1.0},
        # a prompt batch through a grouped sigmoid router with a balance bias, float32 logits
        {"name": "route_groups_16384", "kind": "route", "dtype": "f32", "tokens": 16384, "experts": 256, "top_k": 8,
         "score": "sigmoid", "bias": True, "groups": 8, "top_groups": 4, "group_top": 2, "renormalize": True, "scale": 2.5},
        # the trainer's side of the first router: weights and the gradient of the logits
        {"name": "train_route_8192", "kind": "train", "dtype": "bf16", "tokens": 8192, "experts": 128, "top_k": 8,
         "score": "softmax", "bias": False, "groups": 1, "top_groups": 1, "group_top": 1, "renormalize": True, "scale": 1.0},
        # a router that keeps the softmax over all experts: a dense gradient, an expert count that 64 does not divide
        {"name": "train_route_odd", "kind": "train", "dtype": "f32", "tokens": 5001, "experts": 160, "top_k": 6,
         "score": "softmax", "bias": False, "groups": 8, "top_groups": 3, "group_top": 1, "renormalize": False, "scale": 16.0},
        # one token through 8 of 128 experts: their weights' bytes are all there is
        {"name": "experts_decode_1", "kind": "experts", "dtype": "bf16", "tokens": 1, "experts": 128, "hidden": 2048,
         "inter": 768, "top_k": 8},
        # a larger decoding batch on one rank of four: 768 cut to 192, tiles of 128 that end inside gate and up
        {"name": "experts_tp4_200", "kind": "experts", "dtype": "bf16", "tokens": 200, "experts": 128, "hidden": 2048,
         "inter": 192, "top_k": 8},
        # the prompts of a rollout batch: 256 pairs an expert
        {"name": "experts_prefill_4096", "kind": "experts", "dtype": "bf16", "tokens": 4096, "experts": 128, "hidden": 2048,
         "inter": 768, "top_k": 8},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "matmul", "matmul", "route", "train", "experts", "experts"])
    # an expert's hidden values are quantized from sums, so its outputs are 16 bits wide
    dtype = rng.choice(["bf16", "bf16", "f16"] + ([] if kind == "experts" else ["f32"]))
    if kind in ("linear", "matmul"):
        # half the widths whole tiles, half any number
        k, n = (128 * _log(rng, 2, 96) if rng.random() < 0.5 else _log(rng, 200, 12288) for _ in range(2))
        tokens = min(_log(rng, 1, 8192), _MOST_MACS // (k * n))
        return {"kind": kind, "dtype": dtype, "tokens": tokens, "k": k, "n": n, "bias": rng.random() < 0.25}
    if kind in ("route", "train"):
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * _log(rng, 4, 256 // groups)
        top_groups = 1 if groups == 1 else rng.randint(1, groups)
        return {"kind": kind, "dtype": dtype, "tokens": _log(rng, 1, 16384), "experts": experts,
                "top_k": rng.randint(1, min(12, experts // groups * top_groups)),
                "score": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.5, "groups": groups,
                "top_groups": top_groups, "group_top": rng.choice([1, 2]), "renormalize": rng.random() < 0.7,
                "scale": rng.choice([1.0, 2.5])}
    experts, hidden = _log(rng, 8, 128), 16 * _log(rng, 16, 256)
    inter = min(16 * _log(rng, 6, 128), _MOST_EXPERT_WEIGHTS // (3 * experts * hidden) // 16 * 16)
    top_k = rng.randint(1, 8)
    tokens = min(_log(rng, 1, 4096), _MOST_EXPERT_MACS // (3 * top_k * hidden * inter))
    return {"kind": kind, "dtype": dtype, "tokens": tokens, "experts": experts, "hidden": hidden, "inter": inter,
            "top_k": top_k}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _weight(gen, *shape):
    """Codes and float32 scales of N(0, 0.02) weights in 128x128 tiles."""
    *lead, n, k = shape
    codes = torch.empty(shape, dtype=_E4M3, device="cuda")
    scales = torch.empty((*lead, -(-n // _B), -(-k // _B)), dtype=torch.float32, device="cuda")
    for c, s in zip(codes.view(-1, n, k), scales.view(-1, *scales.shape[-2:])):
        w = torch.randn(n, k, generator=gen, device="cuda") * 0.02
        nb, kb = s.shape
        pad = torch.zeros(nb * _B, kb * _B, device="cuda")
        pad[:n, :k] = w
        tiles = pad.view(nb, _B, kb, _B)
        s.copy_(_scale(tiles.abs().amax((1, 3))))
        c.copy_((tiles / s[:, None, :, None]).view(nb * _B, kb * _B)[:n, :k])
    return codes, scales


def _acts(gen, tokens, k):
    """Activations of a decoder layer: unit normal, a few channels forty times as large."""
    x = torch.randn(tokens, k, generator=gen, device="cuda")
    x[:, torch.randint(0, k, (max(1, k // 500),), generator=gen, device="cuda")] *= 40.0
    return x


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dt = case["kind"], _DTYPES[case["dtype"]]
    st = {"case": case}
    if kind in ("linear", "matmul"):
        x = _acts(gen, case["tokens"], case["k"])
        st["codes"], st["scales"] = _weight(gen, case["n"], case["k"])
        st["bias"] = torch.randn(case["n"], generator=gen, device="cuda") if case["bias"] else None
        if kind == "linear":
            st["x"] = x.to(dt)
        else:
            q, s = _quant(x.to(torch.bfloat16).float())
            st["x_codes"], st["x_scales"] = q.to(_E4M3), s
    elif kind in ("route", "train"):
        t, e = case["tokens"], case["experts"]
        st["logits"] = (torch.randn(t, e, generator=gen, device="cuda") * 1.5
                        + torch.randn(e, generator=gen, device="cuda") * 0.5).to(dt)
        st["bias"] = torch.randn(e, generator=gen, device="cuda") * 0.1 if case["bias"] else None
        if kind == "train":
            st["logits"].requires_grad_()
            st["grad"] = torch.randn(t, case["top_k"], generator=gen, device="cuda")
    else:
        t, e, h, i, k = (case[n] for n in ("tokens", "experts", "hidden", "inter", "top_k"))
        st["x"] = _acts(gen, t, h).to(dt)
        st["gate_up"], st["gate_up_scales"] = _weight(gen, e, 2 * i, h)
        st["down"], st["down_scales"] = _weight(gen, e, h, i)
        # popular and unpopular experts, as a router has them
        score = torch.randn(t, e, generator=gen, device="cuda") + 0.5 * torch.randn(e, generator=gen, device="cuda")
        top = torch.topk(score, k)
        st["ids"], st["weights"] = top.indices.to(torch.int32), torch.softmax(top.values, -1)
    return st


# ---------------------------------------------------------------------------
# the operators in plain form
# ---------------------------------------------------------------------------
def _scale(amax):
    """amax / 448 by IEEE division (torch multiplies by the reciprocal of a plain number)."""
    return (amax / torch.full_like(amax, 448.0)).clamp_min(_TINY)


def _quant(x):
    """float32 [..., K] -> values of the e4m3 codes [..., K], scales [..., ceil(K/128)]."""
    k = x.shape[-1]
    kb = -(-k // _B)
    blocks = torch.zeros(*x.shape[:-1], kb * _B, device=x.device)
    blocks[..., :k] = x
    blocks = blocks.view(*x.shape[:-1], kb, _B)
    s = _scale(blocks.abs().amax(-1))
    q = (blocks / s[..., None]).to(_E4M3).float()
    return q.view(*x.shape[:-1], kb * _B)[..., :k], s


def _widen_rows(q, s):
    return q * s.repeat_interleave(_B, -1)[..., : q.shape[-1]]


def _widen_tiles(codes, s):
    n, k = codes.shape[-2:]
    return codes.float() * s.repeat_interleave(_B, -1)[..., :k].repeat_interleave(_B, -2)[..., :n, :]


def _score(logits, case):
    if case["score"] == "softmax":
        e = torch.exp(logits - logits.amax(-1, keepdim=True))
        return e / e.sum(-1, keepdim=True)
    return 1.0 / (1.0 + torch.exp(-logits))


def _select(logits, bias, case):
    """ids [T, k] by the scores plus the bias, in 64 bits (ranks next to each other); ties to the lowest index."""
    t, e = logits.shape
    pick = _score(logits.double(), case)
    if bias is not None:
        pick = pick + bias.double()
    elif case["group_top"] == 1 or case["groups"] == 1:
        pick = logits.double()  # the order of the scores
    g = case["groups"]
    if g > 1:
        per = pick.view(t, g, e // g).sort(-1, descending=True).values[..., : case["group_top"]].sum(-1)
        keep = per.sort(dim=-1, descending=True, stable=True).indices[:, : case["top_groups"]]
        allowed = torch.zeros(t, g, dtype=torch.bool, device=logits.device).scatter_(1, keep, True)
        pick = torch.where(allowed.repeat_interleave(e // g, 1), pick, -math.inf)
    return pick.sort(dim=-1, descending=True, stable=True).indices[:, : case["top_k"]]


def _route(st):
    case = st["case"]
    logits = st["logits"].detach().float()
    ids = _select(logits, st["bias"], case)
    score = _score(logits, case)
    w = score.gather(1, ids)
    if case["renormalize"]:
        w = w / (w.sum(-1, keepdim=True) + (1e-20 if case["score"] == "sigmoid" else 0.0))
    return logits, ids, score, w * case["scale"]


def _route_grad(case, ids, score, w, grad):
    """The gradient of the logits, from the formulas."""
    s, f = score.gather(1, ids), case["scale"]
    if case["renormalize"]:
        eps = 1e-20 if case["score"] == "sigmoid" else 0.0
        ds = f * (grad - (grad * w).sum(-1, keepdim=True) / f) / (s.sum(-1, keepdim=True) + eps)
    else:
        ds = f * grad
    if case["score"] == "sigmoid":
        return torch.zeros_like(score).scatter_(1, ids, ds * s * (1.0 - s))
    dp = torch.zeros_like(score).scatter_(1, ids, ds)
    return score * (dp - (ds * s).sum(-1, keepdim=True))


def _silu_mul(g, u):
    return g / (1.0 + torch.exp(-g)) * u


def _experts(st):
    x = _widen_rows(*_quant(st["x"].float()))
    ids, weights = st["ids"], st["weights"]
    t, k = ids.shape
    i = st["down"].shape[-1]
    if t * k <= 64:  # few pairs: each takes its expert's weights
        e = ids.reshape(-1).long()
        gu = _widen_tiles(st["gate_up"].view(torch.uint8)[e].view(_E4M3), st["gate_up_scales"][e])
        gu = (gu @ x.repeat_interleave(k, 0)[:, :, None])[..., 0]
        h = _widen_rows(*_quant(_silu_mul(gu[:, :i], gu[:, i:])))
        dn = _widen_tiles(st["down"].view(torch.uint8)[e].view(_E4M3), st["down_scales"][e])
        y = (dn @ h[:, :, None])[..., 0].view(t, k, -1)
        return (y * weights[..., None]).sum(1).to(st["x"].dtype)
    out = torch.zeros_like(x)
    for e in range(st["gate_up"].shape[0]):
        tok, slot = (ids == e).nonzero(as_tuple=True)
        gu = x[tok] @ _widen_tiles(st["gate_up"][e], st["gate_up_scales"][e]).t()
        h = _widen_rows(*_quant(_silu_mul(gu[:, :i], gu[:, i:])))
        y = h @ _widen_tiles(st["down"][e], st["down_scales"][e]).t()
        out.index_add_(0, tok, y * weights[tok, slot][:, None])
    return out.to(st["x"].dtype)


def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        q = _api()
        if kind == "linear":
            return q.fp8_block_linear(st["x"], st["codes"], st["scales"], st["bias"])
        if kind == "matmul":
            return q.fp8_matmul(st["x_codes"], st["x_scales"], st["codes"], st["scales"], st["bias"],
                                out_dtype=_DTYPES[case["dtype"]])
        if kind == "experts":
            return q.fp8_experts(st["x"], st["ids"], st["weights"], st["gate_up"], st["gate_up_scales"], st["down"],
                                 st["down_scales"])
        w, ids = q.route_experts(st["logits"], case["top_k"], score=case["score"], bias=st["bias"], groups=case["groups"],
                                 top_groups=case["top_groups"], group_top=case["group_top"],
                                 renormalize=case["renormalize"], scale=case["scale"])
        if kind == "route":
            return w, ids
        (grad,) = torch.autograd.grad(w, st["logits"], st["grad"])
        return w.detach(), ids, grad
    if kind in ("linear", "matmul"):
        xq, xs = _quant(st["x"].float()) if kind == "linear" else (st["x_codes"].float(), st["x_scales"])
        y = _widen_rows(xq, xs) @ _widen_tiles(st["codes"], st["scales"]).t()
        if st["bias"] is not None:
            y = y + st["bias"]
        return y.to(_DTYPES[case["dtype"]])
    if kind == "experts":
        return _experts(st)
    _, ids, score, w = _route(st)
    if kind == "route":
        return w, ids.to(torch.int32)
    return w, ids.to(torch.int32), _route_grad(case, ids, score, w, st["grad"]).to(st["logits"].dtype)


def work(case):
    kind, e = case["kind"], _SIZES[case["dtype"]]
    t = case["tokens"]
    if kind in ("linear", "matmul"):
        k, n = case["k"], case["n"]
        kb = -(-k // _B)
        nbytes = n * k + 4 * -(-n // _B) * kb + t * n * e + (4 * n if case["bias"] else 0)
        nbytes += t * k * e if kind == "linear" else t * (k + 4 * kb)
        return {"bytes": nbytes, "flops": 2 * t * n * k}
    if kind in ("route", "train"):
        ex, k = case["experts"], case["top_k"]
        nbytes = t * ex * e + 8 * t * k + (4 * ex if case["bias"] else 0)
        if kind == "train":  # the gradients in and out
            nbytes += 4 * t * k + t * ex * e
        return {"bytes": nbytes, "flops": 8 * t * ex}
    ex, h, i, k = (case[n] for n in ("experts", "hidden", "inter", "top_k"))
    used = ex * (1.0 - (1.0 - k / ex) ** t)  # experts that some token takes
    weights = 3 * h * i + 4 * (-(-2 * i // _B) * -(-h // _B) + -(-h // _B) * -(-i // _B))
    return {"bytes": int(used * weights) + 2 * t * h * e + 8 * t * k, "flops": 6 * t * k * h * i}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _e4m3_grid(v):
    """float64 -> the nearest e4m3 value, ties to even: steps of 2^(exponent - 3), 2^-9 at least."""
    _, exponent = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (exponent - 4).clamp_min(-9))
    return torch.round(v / step) * step


def _exact_quant(x):
    """The quantized image of float64 rows: float32 scales amax / 448 of 1x128 blocks, float32 quotients, e4m3."""
    out = torch.empty_like(x)
    for b in range(0, x.shape[-1], _B):
        blk = x[..., b: b + _B]
        s = (blk.abs().amax(-1, keepdim=True) / 448.0).float().double().clamp_min(_TINY)
        out[..., b: b + _B] = _e4m3_grid((blk / s).float().double()) * s
    return out


def _exact_tiles(codes, scales):
    n, k = codes.shape
    rows = torch.arange(n, device=codes.device) // _B
    cols = torch.arange(k, device=codes.device) // _B
    return codes.double() * scales.double()[rows][:, cols]


def _exact_route(st):
    case = st["case"]
    x = st["logits"].detach().double()
    t, e = x.shape
    top = x.max(1, keepdim=True).values
    p = torch.sigmoid(x) if case["score"] == "sigmoid" else torch.softmax(x - top, 1)
    choice = x if st["bias"] is None and (case["groups"] == 1 or case["group_top"] == 1) else p
    if st["bias"] is not None:
        choice = choice + st["bias"].double()
    if case["groups"] > 1:
        size = e // case["groups"]
        best = torch.stack([c.topk(min(case["group_top"], size), 1).values.sum(1) for c in choice.split(size, 1)], 1)
        # a group stays if fewer than top_groups others come before it (higher, or equal with a lower index)
        before = (best[:, None, :] > best[:, :, None]) | ((best[:, None, :] == best[:, :, None])
                                                          & torch.ones(best.shape[1], best.shape[1], device=x.device).tril(-1).bool())
        stays = before.sum(2) < case["top_groups"]
        choice = choice.masked_fill(~stays.repeat_interleave(size, 1), -math.inf)
    ids = torch.argsort(choice, dim=1, descending=True, stable=True)[:, : case["top_k"]]
    s = torch.gather(p, 1, ids)
    den = torch.ones(t, 1, dtype=x.dtype, device=x.device)
    if case["renormalize"]:
        den = s.sum(1, keepdim=True) + (1e-20 if case["score"] == "sigmoid" else 0.0)
    w = case["scale"] * s / den
    if case["kind"] == "route":
        return w, ids.to(torch.int32)
    # dw_j/dx_i through the scores' own derivatives
    g = st["grad"].double() * case["scale"] / den
    if case["renormalize"]:
        g = g - (g * s).sum(1, keepdim=True) / den
    full = torch.zeros_like(p).scatter(1, ids, g)
    if case["score"] == "sigmoid":
        dx = full * p * (1.0 - p)
    else:
        dx = p * full - p * (p * full).sum(1, keepdim=True)
    return w, ids.to(torch.int32), dx


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind in ("route", "train"):
        return _exact_route(st)
    if kind in ("linear", "matmul"):
        if kind == "linear":
            x = _exact_quant(st["x"].double())
        else:
            cols = torch.arange(case["k"], device="cuda") // _B
            x = st["x_codes"].double() * st["x_scales"].double()[:, cols]
        y = x @ _exact_tiles(st["codes"], st["scales"]).T
        return y if st["bias"] is None else y + st["bias"].double()
    x = _exact_quant(st["x"].double())
    ids, i = st["ids"].long(), case["inter"]
    out = torch.zeros_like(x)
    for e in torch.unique(ids).tolist():
        hit = ids == e
        tok = hit.any(1).nonzero()[:, 0]
        gu = x[tok] @ _exact_tiles(st["gate_up"][e], st["gate_up_scales"][e]).T
        h = _exact_quant(torch.nn.functional.silu(gu[:, :i]) * gu[:, i:])
        y = h @ _exact_tiles(st["down"][e], st["down_scales"][e]).T
        out[tok] += y * (st["weights"].double() * hit).sum(1)[tok][:, None]
    return out
