"""FP8 products on weights in 128x128 tiles.

``quantize_fp8_blockwise`` writes a weight as e4m3 codes [N, K] with one float32
scale per 128x128 tile, the layout vLLM and ATOM load as ``weight_scale_inv``.
These are the products that consume it on this side: with activations that were
quantized earlier (``fp8_matmul``), or quantized on the way in
(``fp8_block_linear``).  Both return without synchronizing, on the current
stream of the operands' device.
"""

from __future__ import annotations

import functools
from typing import Optional

import torch
from torch import Tensor
from torch.autograd import forward_ad

from lumenrl_amd import _lib
from lumenrl_amd.quantization.ops import _IN_DTYPES, _check_input, _dense, _on, _prod, _stream

_BLOCK = 128
_PITCH_MAX = 1 << 22  # of the kernels' 32-bit offsets; rows further apart are copied


def check_tiles(what: str, codes: Tensor, scales: Tensor, device: torch.device) -> tuple[Tensor, Tensor]:
    """``codes`` [..., N, K] and their scales [..., ceil(N/128), ceil(K/128)], both dense on ``device``."""
    if not isinstance(codes, Tensor) or not isinstance(scales, Tensor):
        raise TypeError(f"{what}: codes and scales must be tensors")
    if codes.dtype != torch.float8_e4m3fn or scales.dtype != torch.float32:
        raise TypeError(f"{what}: codes must be float8_e4m3fn with float32 scales, got {codes.dtype} and {scales.dtype}")
    shape = codes.shape
    if len(shape) < 2:
        raise ValueError(f"{what}: codes must have rows and columns, got {tuple(shape)}")
    if scales.shape != (*shape[:-2], -(-shape[-2] // _BLOCK), -(-shape[-1] // _BLOCK)):
        raise ValueError(f"{what}: scales {tuple(scales.shape)} are not those of 128x128 tiles of {tuple(shape)}")
    if codes.device != device or scales.device != device:
        raise ValueError(f"{what}: codes and scales must be on {device}")
    return (codes if codes.is_contiguous() else codes.contiguous(),
            scales if scales.is_contiguous() else scales.contiguous())


def _check_bias(what: str, bias: Tensor, n: int, device: torch.device) -> None:
    if not isinstance(bias, Tensor):
        raise TypeError(f"{what}: bias must be a tensor, got {type(bias)!r}")
    if bias.shape != (n,) or bias.dtype not in _IN_DTYPES or bias.device != device or not bias.is_contiguous():
        raise ValueError(f"{what}: bias must be a contiguous [{n}] bf16, fp16 or fp32 tensor on {device}")


def _empty_sum(rows: int, n: int, bias: Optional[Tensor], dtype: torch.dtype, device: torch.device) -> Tensor:
    y = torch.zeros((rows, n), dtype=torch.float32, device=device)
    return (y if bias is None else y + bias).to(dtype)


class NoGradient(torch.autograd.Function):
    """An operator without a gradient, on inputs that want one: whoever asks for it is told, and not left without."""

    @staticmethod
    def forward(ctx, what, call, *args):
        ctx.what = what
        return call(*args)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.what} has no gradient")

    @staticmethod
    def jvp(ctx, *_):
        raise RuntimeError(f"{ctx.what} has no forward-mode derivative")


@functools.lru_cache(maxsize=4096)
def _matmul_workspace(rows: int, k: int, n: int) -> int:
    return _lib.lib().lrq_fp8_matmul_workspace(rows, k, n)


def fp8_matmul(x_codes: Tensor, x_scales: Tensor, codes: Tensor, scales: Tensor, bias: Optional[Tensor] = None, *,
               out_dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """``x`` [M, K] times the transpose of a weight [N, K], both e4m3.

    ``x_codes`` [M, K] with float32 ``x_scales`` [M, ceil(K/128)] (as
    ``fp8_block_quant(x, (1, 128))`` gives them; rows may be a view's),
    ``codes`` [N, K] with float32 ``scales`` [ceil(N/128), ceil(K/128)] ->
    [M, N] of ``out_dtype`` (bfloat16, float16 or float32).  Sums are float32; within
    a block of 128, 16-bit results of more than four rows take the matrix
    instructions' own, which drop what is below 2^-13 of the block's largest product
    (1.5e-5 of the result's norm with normal codes).  No gradient: a backward pass
    through the result raises.
    """
    if not isinstance(x_codes, Tensor) or not x_codes.is_cuda:
        raise ValueError("fp8_matmul: expected codes on a HIP device")
    if not isinstance(x_scales, Tensor):
        raise TypeError(f"fp8_matmul: x's scales must be a tensor, got {type(x_scales)!r}")
    if x_codes.dtype != torch.float8_e4m3fn or x_scales.dtype != torch.float32:
        raise TypeError(f"fp8_matmul: x must be float8_e4m3fn with float32 scales, got {x_codes.dtype} and {x_scales.dtype}")
    if out_dtype not in _IN_DTYPES:
        raise ValueError(f"fp8_matmul: out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
    dev = x_codes.device
    codes, scales = check_tiles("fp8_matmul", codes, scales, dev)
    if x_codes.dim() != 2 or codes.dim() != 2 or x_codes.shape[1] != codes.shape[1]:
        raise ValueError(f"fp8_matmul: x {tuple(x_codes.shape)} and codes {tuple(codes.shape)} do not fit")
    m, k = x_codes.shape
    n = codes.shape[0]
    if x_scales.shape != (m, -(-k // _BLOCK)) or x_scales.device != dev:
        raise ValueError(f"fp8_matmul: x's scales must be {(m, -(-k // _BLOCK))} on {dev}, got {tuple(x_scales.shape)}")
    if bias is not None:
        _check_bias("fp8_matmul", bias, n, dev)
    if k == 0:
        return _empty_sum(m, n, bias, out_dtype, dev)
    if forward_ad._current_level >= 0 or torch.is_grad_enabled() and (
            x_codes.requires_grad or x_scales.requires_grad or codes.requires_grad or scales.requires_grad
            or (bias is not None and bias.requires_grad)):
        return NoGradient.apply("fp8_matmul", _matmul, x_codes, x_scales, codes, scales, bias, out_dtype)
    return _matmul(x_codes, x_scales, codes, scales, bias, out_dtype)


def _matmul(x_codes: Tensor, x_scales: Tensor, codes: Tensor, scales: Tensor, bias: Optional[Tensor],
            out_dtype: torch.dtype) -> Tensor:
    dev = x_codes.device
    (m, k), n = x_codes.shape, codes.shape[0]
    bias_ptr, bias_dtype = (None, 0) if bias is None else (bias.data_ptr(), _IN_DTYPES[bias.dtype])
    ld = x_codes.stride(0) if m > 1 else k
    if (k > 1 and x_codes.stride(1) != 1) or not k <= ld <= _PITCH_MAX:
        x_codes, ld = x_codes.contiguous(), k
    if not x_scales.is_contiguous():
        x_scales = x_scales.contiguous()
    out = _dense((m, n), out_dtype, dev)
    need = _matmul_workspace(m, k, n)
    work = _dense((need,), torch.uint8, dev) if need else None
    with _on(dev):
        rc = _lib.lib().lrq_fp8_matmul(x_codes.data_ptr(), x_scales.data_ptr(), m, k, ld, codes.data_ptr(), scales.data_ptr(), n,
                                       bias_ptr, bias_dtype, out.data_ptr(), _IN_DTYPES[out_dtype],
                                       work.data_ptr() if need else None, need, _stream(dev))
    if rc:
        _lib.check(rc, "lrq_fp8_matmul")
    return out


@functools.lru_cache(maxsize=4096)
def _linear_workspace(rows: int, k: int, n: int) -> int:
    return _lib.lib().lrq_fp8_block_linear_workspace(rows, k, n)


def fp8_block_linear(x: Tensor, codes: Tensor, scales: Tensor, bias: Optional[Tensor] = None) -> Tensor:
    """A linear layer in FP8: ``x`` [..., K] is quantized to e4m3 in 1x128 blocks
    (as ``fp8_block_quant(x, (1, 128))``) and multiplied with ``codes`` [N, K]
    and float32 ``scales`` [ceil(N/128), ceil(K/128)] -> [..., N] in x's dtype.

    Sums are ``fp8_matmul``'s.  Up to four tokens take one launch, more take two or
    three.  No gradient: a backward pass through the result raises.
    """
    _check_input(x, "fp8_block_linear")
    dev = x.device
    codes, scales = check_tiles("fp8_block_linear", codes, scales, dev)
    shape = x.shape
    if not shape or codes.dim() != 2 or shape[-1] != codes.shape[1]:
        raise ValueError(f"fp8_block_linear: x {tuple(shape)} and codes {tuple(codes.shape)} do not fit")
    n, k = codes.shape
    if bias is not None:
        _check_bias("fp8_block_linear", bias, n, dev)
    if k == 0:
        return _empty_sum(_prod(shape[:-1]), n, bias, x.dtype, dev).view(*shape[:-1], n)
    if forward_ad._current_level >= 0 or torch.is_grad_enabled() and (
            x.requires_grad or codes.requires_grad or scales.requires_grad or (bias is not None and bias.requires_grad)):
        return NoGradient.apply("fp8_block_linear", _block_linear, x, codes, scales, bias)
    return _block_linear(x, codes, scales, bias)


def _block_linear(x: Tensor, codes: Tensor, scales: Tensor, bias: Optional[Tensor]) -> Tensor:
    dev, shape = x.device, x.shape
    n, k = codes.shape
    bias_ptr, bias_dtype = (None, 0) if bias is None else (bias.data_ptr(), _IN_DTYPES[bias.dtype])
    if x.is_contiguous():
        rows, ld = x.numel() // k, k
    else:
        rows = x.numel() // k
        x = x.reshape(rows, k)
        ld = x.stride(0) if rows > 1 else k
        if (k > 1 and x.stride(1) != 1) or not k <= ld <= _PITCH_MAX:
            x, ld = x.contiguous(), k
    out = _dense((*shape[:-1], n), x.dtype, dev)
    need = _linear_workspace(rows, k, n)
    work = _dense((need,), torch.uint8, dev) if need else None
    dtype = _IN_DTYPES[x.dtype]
    with _on(dev):
        rc = _lib.lib().lrq_fp8_block_linear(x.data_ptr(), dtype, rows, k, ld, codes.data_ptr(), scales.data_ptr(), n, bias_ptr,
                                             bias_dtype, out.data_ptr(), work.data_ptr() if need else None, need, _stream(dev))
    if rc:
        _lib.check(rc, "lrq_fp8_block_linear")
    return out
