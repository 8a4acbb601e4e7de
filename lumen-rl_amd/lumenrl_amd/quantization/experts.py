"""Mixture-of-experts operators: the router, and the experts on FP8 weights.

``route_experts`` turns a router's logits into each token's experts and their
weights, with the gradient of the logits; ``fp8_experts`` runs those experts' MLPs
on the stacks that ``quantize_fp8_blockwise`` writes.  Every function launches on the
current stream of its operands' device and returns without synchronizing.
"""

from __future__ import annotations

import functools
from typing import Optional

import torch
from torch import Tensor
from torch.autograd import forward_ad

from lumenrl_amd import _lib
from lumenrl_amd.quantization.fp8_product import NoGradient, check_tiles
from lumenrl_amd.quantization.ops import _IN_DTYPES, _check_input, _dense, _on, _stream

_PITCH_MAX = 1 << 31  # rows further apart are copied
_SCORES = {"softmax": _lib.SCORE_SOFTMAX, "sigmoid": _lib.SCORE_SIGMOID}


def _rows(x: Tensor) -> tuple[Tensor, int, int]:
    """``x`` [..., E] as rows of unit stride: (tensor, rows, row pitch); a copy only where it has to be."""
    e = x.shape[-1]
    if x.is_contiguous():
        return x, x.numel() // e, e
    rows = x.numel() // e
    x = x.reshape(rows, e)
    ld = x.stride(0) if rows > 1 else e
    if (e > 1 and x.stride(1) != 1) or not e <= ld <= _PITCH_MAX:
        return x.contiguous(), rows, e
    return x, rows, ld


def _route(logits: Tensor, ids: Tensor, bias: Optional[Tensor], cfg: tuple) -> Tensor:
    top_k, score, groups, top_groups, group_top, renormalize, scale = cfg
    dev = logits.device
    x, rows, ld = _rows(logits)
    weights = _dense(ids.shape, torch.float32, dev)
    with _on(dev):
        rc = _lib.lib().lrq_route(x.data_ptr(), _IN_DTYPES[x.dtype], rows, logits.shape[-1], ld,
                                  bias.data_ptr() if bias is not None else None, top_k, score, groups, top_groups, group_top,
                                  renormalize, scale, weights.data_ptr(), ids.data_ptr(), _stream(dev))
    if rc:
        _lib.check(rc, "lrq_route")
    return weights


def _route_grad(ctx, grad: Tensor, *_):
    logits, ids = ctx.saved_tensors
    top_k, score, _, _, _, renormalize, scale = ctx.cfg
    dev = logits.device
    grad = grad.contiguous()
    x, rows, ld = _rows(logits)
    out = _dense(logits.shape, logits.dtype, dev)
    with _on(dev):
        rc = _lib.lib().lrq_route_grad(x.data_ptr(), _IN_DTYPES[x.dtype], rows, logits.shape[-1], ld, ids.data_ptr(),
                                       grad.data_ptr(), top_k, score, renormalize, scale, out.data_ptr(), _stream(dev))
    if rc:
        _lib.check(rc, "lrq_route_grad")
    return out, None, None, None


class _Route(torch.autograd.Function):
    """Weights of ``logits``; ``ids`` is filled on the way (as an input it costs autograd nothing)."""

    @staticmethod
    def forward(ctx, logits, ids, bias, cfg):
        ctx.save_for_backward(logits, ids)
        ctx.cfg = cfg
        return _route(logits, ids, bias, cfg)

    # the wrapper refuses a second derivative, also that by way of the logits; only for
    # backward passes that record one
    _recorded = staticmethod(torch.autograd.function.once_differentiable(_route_grad))

    @staticmethod
    def backward(ctx, grad):
        if torch.is_grad_enabled():
            return _Route._recorded(ctx, grad, ctx.saved_tensors[0])
        return _route_grad(ctx, grad)

    @staticmethod
    def jvp(ctx, *_):
        raise RuntimeError("route_experts has no forward-mode derivative")


def route_experts(logits: Tensor, top_k: int, *, score: str = "softmax", bias: Optional[Tensor] = None, groups: int = 1,
                  top_groups: int = 1, group_top: int = 1, renormalize: bool = True, scale: float = 1.0
                  ) -> tuple[Tensor, Tensor]:
    """Each token's experts: ``logits`` [..., E] -> (weights float32 [..., top_k], ids int32 [..., top_k]).

    Experts are chosen by their score (``"softmax"`` or ``"sigmoid"`` of the logits)
    plus ``bias`` [E] (float32; for balance: it moves the choice, not the weights,
    and takes no gradient), highest first, ties to the lowest index.  With
    ``groups`` > 1 only the ``top_groups`` runs of E / groups experts with the highest
    sum of their ``group_top`` (1 or 2) best are open.  Weights are the scores times
    ``scale``, divided by the chosen scores' sum if ``renormalize``.

    The choice is that of exact arithmetic; a NaN counts as the highest.  E is at
    most 512, ``top_k`` 64, ``groups`` 16.  The weights carry the gradient of the
    logits (once; not its own gradient).
    """
    _check_input(logits, "route_experts")
    if score not in _SCORES:
        raise ValueError(f"route_experts: score must be 'softmax' or 'sigmoid', got {score!r}")
    if logits.dim() < 1:
        raise ValueError("route_experts: logits must have a dimension of experts")
    e = logits.shape[-1]
    if bias is not None:
        if not isinstance(bias, Tensor) or bias.dtype != torch.float32:
            raise TypeError("route_experts: bias must be a float32 tensor")
        if bias.shape != (e,) or bias.device != logits.device:
            raise ValueError(f"route_experts: bias must be [{e}] on {logits.device}, got {tuple(bias.shape)} on {bias.device}")
        bias = bias.detach().contiguous()
    if not 1 <= e <= 512 or not 1 <= top_k <= min(e, 64):
        raise ValueError(f"route_experts: top_k {top_k} of {e} experts (at most 64 of 512)")
    if not 1 <= groups <= 16 or e % groups or not 1 <= top_groups <= groups or top_k > e // groups * top_groups:
        raise ValueError(f"route_experts: top_k {top_k} of {e} experts in {top_groups} of {groups} groups (at most 16)")
    if group_top not in (1, 2):
        raise ValueError(f"route_experts: group_top must be 1 or 2, got {group_top}")
    cfg = (top_k, _SCORES[score], groups, top_groups, group_top, int(renormalize), scale)
    ids = _dense((*logits.shape[:-1], top_k), torch.int32, logits.device)
    if (logits.requires_grad and torch.is_grad_enabled()) or forward_ad._current_level >= 0:
        return _Route.apply(logits, ids, bias, cfg), ids
    return _route(logits, ids, bias, cfg), ids


@functools.lru_cache(maxsize=4096)
def _experts_workspace(rows: int, hidden: int, inter: int, experts: int, top_k: int) -> int:
    return _lib.lib().lrq_fp8_experts_workspace(rows, hidden, inter, experts, top_k)


def fp8_experts(x: Tensor, ids: Tensor, weights: Tensor, gate_up: Tensor, gate_up_scales: Tensor, down: Tensor,
                down_scales: Tensor) -> Tensor:
    """The chosen experts' SwiGLU MLPs in FP8, and their weighted sum.

    ``x`` [..., H] (bf16 or fp16) with ``ids`` and float32 ``weights`` [..., k] (as
    ``route_experts`` gives them; int32, int64 ids are narrowed) -> [..., H] in x's
    dtype.  ``gate_up`` [E, 2 I, H] (gate's rows first) and ``down`` [E, H, I] are
    e4m3 codes with float32 scales of 128x128 tiles, as ``quantize_fp8_blockwise``
    writes them; H and I are multiples of 16 up to 65536.  x and the hidden values are
    quantized in 1x128 blocks; all else is float32, but that beyond some 64 pairs the
    second product's blocks of 128 are summed as ``fp8_matmul``'s for 16 bits.  A pair
    whose id is not one of 0 .. E - 1 is left out (a shard's other experts, say).  No
    gradient: a backward pass through the result raises.
    """
    what = "fp8_experts"
    _check_input(x, what)
    dev = x.device
    if x.dtype == torch.float32:
        raise TypeError(f"{what}: x must be bf16 or fp16")
    if not isinstance(ids, Tensor) or not isinstance(weights, Tensor):
        raise TypeError(f"{what}: ids and weights must be tensors")
    if ids.dtype not in (torch.int32, torch.int64) or weights.dtype != torch.float32:
        raise TypeError(f"{what}: ids must be int32 or int64 and weights float32, got {ids.dtype} and {weights.dtype}")
    gate_up, gate_up_scales = check_tiles(what, gate_up, gate_up_scales, dev)
    down, down_scales = check_tiles(what, down, down_scales, dev)
    if x.dim() < 1 or gate_up.dim() != 3 or down.dim() != 3:
        raise ValueError(f"{what}: x {tuple(x.shape)}, gate_up {tuple(gate_up.shape)} and down {tuple(down.shape)} do not fit")
    e, h, i = down.shape
    if gate_up.shape != (e, 2 * i, h) or x.shape[-1] != h:
        raise ValueError(f"{what}: x {tuple(x.shape)}, gate_up {tuple(gate_up.shape)} and down {tuple(down.shape)} do not fit")
    lead = x.shape[:-1]
    if ids.dim() != x.dim() or ids.shape[:-1] != lead or weights.shape != ids.shape:
        raise ValueError(f"{what}: ids {tuple(ids.shape)} and weights {tuple(weights.shape)} must be {(*lead, 'k')}")
    if ids.device != dev or weights.device != dev:
        raise ValueError(f"{what}: ids and weights must be on {dev}")
    k = ids.shape[-1]
    if (not 1 <= e <= 1024 or not 1 <= k <= 64 or h % 16 or i % 16 or not 0 < h <= 65536 or not 0 < i <= 65536
            or 2 * h * i >= 1 << 31):
        raise ValueError(f"{what}: {e} experts (at most 1024), top {k} (at most 64), H {h} and I {i} (multiples of 16 up to "
                         "65536, 2 H I below 2^31)")
    if forward_ad._current_level >= 0 or torch.is_grad_enabled() and (
            x.requires_grad or weights.requires_grad or gate_up.requires_grad or gate_up_scales.requires_grad
            or down.requires_grad or down_scales.requires_grad):
        return NoGradient.apply(what, _experts, x, ids, weights, gate_up, gate_up_scales, down, down_scales)
    return _experts(x, ids, weights, gate_up, gate_up_scales, down, down_scales)


def _experts(x: Tensor, ids: Tensor, weights: Tensor, gate_up: Tensor, gate_up_scales: Tensor, down: Tensor,
             down_scales: Tensor) -> Tensor:
    dev, lead, k = x.device, x.shape[:-1], ids.shape[-1]
    e, h, i = down.shape
    if ids.dtype == torch.int64:
        ids = ids.clamp(-1, e).to(torch.int32)
    x, rows, ld = _rows(x)
    gate_up, down = (w if w.data_ptr() % 16 == 0 else w.clone() for w in (gate_up, down))
    ids, weights = ids.contiguous(), weights.contiguous()
    out = _dense((*lead, h), x.dtype, dev)
    need = _experts_workspace(rows, h, i, e, k)
    work = _dense((need,), torch.uint8, dev)
    with _on(dev):
        rc = _lib.lib().lrq_fp8_experts(x.data_ptr(), _IN_DTYPES[x.dtype], rows, h, ld, ids.data_ptr(), weights.data_ptr(), k,
                                        gate_up.data_ptr(), gate_up_scales.data_ptr(), down.data_ptr(), down_scales.data_ptr(),
                                        e, i, out.data_ptr(), work.data_ptr(), need, _stream(dev))
    if rc:
        _lib.check(rc, "lrq_fp8_experts")
    return out
