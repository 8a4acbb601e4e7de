"""``fp8_matmul`` and ``fp8_block_linear`` against float64 products of the same codes and scales."""

from __future__ import annotations

import pytest
import torch

from lumenrl_amd.quantization import fp8_block_linear, fp8_block_quant, fp8_matmul, quantize_fp8_blockwise

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def weight(n, k, seed=0):
    """Every code but the NaNs, scales over two binades."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    codes = torch.randint(0, 256, (n, k), generator=g, device=DEV, dtype=torch.uint8)
    codes[(codes & 0x7F) == 0x7F] = 0x30
    scales = (torch.rand(-(-n // 128), -(-k // 128), generator=g, device=DEV) * 3 + 1) * 1e-4
    return codes.view(torch.float8_e4m3fn), scales


def acts(m, k, dtype, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(m, k, generator=g, device=DEV)
    x[:, k // 3] *= 40.0
    return x.to(dtype)


def spread(scales, rows, cols, block=(128, 128)):
    s = scales.double()
    return s.repeat_interleave(block[0], 0)[:rows].repeat_interleave(block[1], 1)[:, :cols]


def check(y, x_codes, x_scales, codes, scales, bias=None, many=False):
    """|y - exact| within the result's rounding and the sums' own bound.

    A block sums 128 exact products in float32, K/128 blocks and 8 waves' parts follow, each step off by at most
    2^-23 of the terms' magnitude, and the product of the two scales by 2^-24.  16-bit results of more than
    four tokens come from matrix instructions that drop what is 2^-13 below the block's largest product: 128 times
    that for each block."""
    (m, k), n = x_codes.shape, codes.shape[0]
    xd = x_codes.double() * spread(x_scales, m, k, (1, 128))
    wd = codes.double() * spread(scales, n, k)
    want, size = xd @ wd.T, xd.abs() @ wd.abs().T
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    half = torch.finfo(y.dtype).eps / 2
    least = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}[y.dtype]
    bound = half * want.abs() * 1.01 + (128 + k // 128 + 12) * 2.0 ** -23 * size + least
    if (m > 4 or many) and y.dtype != torch.float32:
        for b in range(0, k, 128):
            top = xd[:, b: b + 128].abs().amax(1)[:, None] * wd[:, b: b + 128].abs().amax(1)[None]
            bound += 128 * 2.0 ** -13 * top
    off = (y.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


# tokens of each kernel (up to four: dot products; up to 64: K in parts; tiles of four sizes), weights cut in every way
SHAPES = [(1, 1, 1), (2, 77, 2100), (4, 4100, 515), (1, 5000, 1032), (1, 4096, 4096), (3, 200, 130), (16, 130, 1104), (16, 64, 12288), (17, 129, 384), (33, 1, 1100), (64, 300, 272),
          (65, 127, 15), (65, 128, 128), (100, 130, 144), (777, 1500, 1100), (2000, 2040, 1040), (1999, 2041, 1041), (4100, 3850, 272),
          (130, 190, 1036), (300, 129, 1164), (2000, 2040, 1048), (4100, 3850, 268), (70, 65, 4), (400, 12300, 128), (1100, 6200, 144),
          (1536, 300, 1041), (1600, 513, 129), (1536, 4000, 7), (1540, 130, 2046)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul_vs_float64(m, n, k, dtype):
    x_codes, x_scales = fp8_block_quant(acts(m, k, torch.bfloat16, m), (1, 128))
    codes, scales = weight(n, k, n + k)
    bias = torch.randn(n, device=DEV).to(TYPES[n % 3]) if m % 2 else None
    y = fp8_matmul(x_codes, x_scales, codes, scales, bias, out_dtype=dtype)
    assert y.shape == (m, n) and y.dtype == dtype
    check(y, x_codes, x_scales, codes, scales, bias)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_is_the_product_of_the_quantized_activations(m, n, k, dtype):
    x = acts(m, k, dtype, m + 7)
    codes, scales = weight(n, k, n + k + 1)
    y = fp8_block_linear(x, codes, scales)
    x_codes, x_scales = fp8_block_quant(x, (1, 128))
    check(y, x_codes, x_scales, codes, scales)


def test_weights_as_the_framework_quantizes_them():
    w = torch.randn(520, 1000, device=DEV, dtype=torch.bfloat16) * 0.02
    codes, scales = quantize_fp8_blockwise(w)
    x = acts(40, 1000, torch.bfloat16)
    check(fp8_block_linear(x, codes, scales), *fp8_block_quant(x, (1, 128)), codes, scales)


@pytest.mark.parametrize("m", [2, 40, 300])
def test_strides_leading_dims_and_alignment(m):
    n, k = 270, 400
    codes, scales = weight(n, k)
    big = acts(m, 3 * k + 7, torch.bfloat16)
    for x in (big[:, 5: 5 + k], big[:, 16: 16 + k], big[:, : 2 * k: 2], big.t()[:k].t()):
        check(fp8_block_linear(x, codes, scales), *fp8_block_quant(x, (1, 128)), codes, scales)
    x = acts(2 * m, k, torch.float16).view(2, m, k)
    y = fp8_block_linear(x, codes, scales)
    assert y.shape == (2, m, n)
    check(y.view(-1, n), *fp8_block_quant(x.view(-1, k), (1, 128)), codes, scales)
    # codes whose rows are a view's, off their 16-byte boundaries, and a weight that is a transpose
    xc, xs = fp8_block_quant(acts(m, k, torch.bfloat16), (1, 128))
    wide = torch.zeros(m, 3 * k + 5, dtype=torch.uint8, device=DEV)
    for at in (0, 3, 16):
        wide[:, at: at + k] = xc.view(torch.uint8)
        view = wide.view(torch.float8_e4m3fn)[:, at: at + k]
        check(fp8_matmul(view, xs, codes, scales, out_dtype=torch.float32), xc, xs, codes, scales)
    turned = codes.view(torch.uint8).t().contiguous().t().view(torch.float8_e4m3fn)
    check(fp8_matmul(xc, xs, turned, scales, out_dtype=torch.float32), xc, xs, codes, scales)
    shifted = torch.zeros(n * k + 1, dtype=torch.uint8, device=DEV)[1:].view(n, k).copy_(codes.view(torch.uint8))
    check(fp8_matmul(xc, xs, shifted.view(torch.float8_e4m3fn), scales, out_dtype=torch.float32), xc, xs, codes, scales)


@pytest.mark.parametrize("m", [4, 30, 200])
def test_nan_inf_and_zero_rows_stay_in_their_rows(m):
    n, k = 150, 300
    codes, scales = weight(n, k)
    x = acts(m, k, torch.bfloat16)
    x[0, 7], x[1, 290], x[2] = float("nan"), float("-inf"), 0.0
    y = fp8_block_linear(x, codes, scales)
    assert bool(y[:2].isnan().all()) and bool((y[2] == 0).all())
    rest = x[3:]
    check(y[3:], *fp8_block_quant(rest, (1, 128)), codes, scales)


def test_empty_extents():
    codes, scales = weight(64, 256)
    assert fp8_block_linear(torch.zeros(0, 256, device=DEV), codes, scales).shape == (0, 64)
    assert fp8_block_linear(torch.zeros(2, 0, 256, device=DEV), codes, scales).shape == (2, 0, 64)
    assert fp8_block_linear(torch.zeros(5, 256, device=DEV), codes[:0], scales[:0]).shape == (5, 0)
    none = torch.empty(64, 0, dtype=torch.float8_e4m3fn, device=DEV)
    b = torch.randn(64, device=DEV)
    y = fp8_block_linear(torch.zeros(3, 0, device=DEV), none, torch.empty(1, 0, device=DEV), b)
    assert torch.equal(y, b.expand(3, 64))


def test_other_stream_and_graph():
    codes, scales = weight(512, 640)
    for m in (3, 50, 500):
        x = acts(m, 640, torch.bfloat16)
        want = fp8_block_linear(x, codes, scales)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = fp8_block_linear(x, codes, scales)
        side.synchronize()
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = fp8_block_linear(x, codes, scales)
        for seed in range(3):
            x.copy_(acts(m, 640, torch.bfloat16, seed))
            graph.replay()
            assert torch.equal(y, fp8_block_linear(x, codes, scales))


@pytest.mark.parametrize("m", [3, 50, 130])
def test_rows_far_apart_and_results_past_32_bits(m):
    """Codes of x whose rows lie 2^22 bytes apart, at the end of them."""
    pitch, k, n = 1 << 22, 256, 192
    wide = torch.zeros((m, pitch), dtype=torch.uint8, device=DEV)
    xc, xs = fp8_block_quant(acts(m, k, torch.bfloat16), (1, 128))
    codes, scales = weight(n, k)
    for at in (0, pitch - k):
        wide[:, at: at + k] = xc.view(torch.uint8)
        check(fp8_matmul(wide.view(torch.float8_e4m3fn)[:, at: at + k], xs, codes, scales), xc, xs, codes, scales)


def test_a_result_of_more_than_2_31_cells():
    codes, scales = weight(65536, 128)
    x = acts(40000, 128, torch.bfloat16)
    y = fp8_block_linear(x, codes, scales)
    for rows in (slice(0, 3), slice(39997, 40000)):
        check(y[rows], *fp8_block_quant(x[rows], (1, 128)), codes, scales, many=True)


@pytest.mark.parametrize("m", [3, 8, 100])
def test_rows_further_apart_than_offsets_reach(m):
    """The last token of each sequence, [m, 2048, 4096][:, -1]: a pitch of 2^23."""
    codes, scales = weight(150, 4096)
    hidden = torch.zeros(m, 2048, 4096, dtype=torch.bfloat16, device=DEV)
    hidden[:, -1] = acts(m, 4096, torch.bfloat16)
    xc, xs = fp8_block_quant(hidden[:, -1].contiguous(), (1, 128))
    check(fp8_block_linear(hidden[:, -1], codes, scales), xc, xs, codes, scales)
    wide = torch.zeros(m, (1 << 22) + 16, dtype=torch.uint8, device=DEV)
    wide[:, 16: 16 + 4096] = xc.view(torch.uint8)
    check(fp8_matmul(wide.view(torch.float8_e4m3fn)[:, 16: 16 + 4096], xs, codes, scales), xc, xs, codes, scales)


def test_more_rows_than_a_launch_takes():
    """2^28 rows of one value: as many blocks, and with 16 threads each the 2^32 of one launch.  A lone value's scale and
    quotient are off by 2^-24 each, its code is 448, and the result rounds once."""
    x = torch.randn(1 << 28, 1, dtype=torch.bfloat16, device=DEV)
    codes = torch.full((1, 1), 2.0, device=DEV).to(torch.float8_e4m3fn)
    y = fp8_block_linear(x, codes, torch.ones(1, 1, device=DEV))
    assert bool(((y.float() - 2 * x.float()).abs() <= (2.0 ** -8 + 2.0 ** -22) * 2 * x.float().abs()).all())


def test_operands_that_are_no_tensors_are_refused_by_name():
    codes, scales = weight(64, 256)
    x = acts(4, 256, torch.bfloat16)
    xc, xs = fp8_block_quant(x, (1, 128))
    for call in (lambda: fp8_matmul(xc, None, codes, scales), lambda: fp8_matmul(xc, xs, codes, scales, 1.0),
                 lambda: fp8_block_linear(x, codes, scales, [0.0] * 64), lambda: fp8_block_linear(x, codes, None)):
        with pytest.raises(TypeError, match="fp8_(matmul|block_linear): "):
            call()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_whole_numbers_are_exact(m, n, k, dtype):
    """Codes of 0, 1 and 2 either way and scales of 1 to 8: every product, block's sum and sum of blocks is a whole number below
    2^24 (k x 4 x 64), which no instruction drops bits of, in any order.  So a result is the exact one, rounded once; a code that
    is lost, misplaced or read twice shows."""
    g = torch.Generator(device=DEV).manual_seed(m + n + k)

    def codes(rows):
        return torch.randint(-2, 3, (rows, k), generator=g, device=DEV).float().to(torch.float8_e4m3fn)

    def scales(rows):
        return torch.pow(2.0, torch.randint(0, 4, (rows, -(-k // 128)), generator=g, device=DEV).float())

    xc, xs, wc, ws = codes(m), scales(m), codes(n), scales(-(-n // 128))
    want = ((xc.double() * spread(xs, m, k, (1, 128))) @ (wc.double() * spread(ws, n, k)).T).to(dtype)
    assert torch.equal(fp8_matmul(xc, xs, wc, ws, out_dtype=dtype), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [s for s in SHAPES if s[2] >= 128])
def test_the_whole_is_as_near_as_the_results_own_rounding(m, n, k, dtype):
    """Normal activations and weights, no channel above the rest: half a step at most an element, and what the instructions drop.

    That is below 2^-13 of a block's largest product, some 4 x 4 times the norm's share of both operands, each product's one way
    or the other: 2^-13 x 16 / sqrt(128), over the blocks as over their sum; none of it for float32 results or up to four tokens,
    whose sums are off by (128 + k / 128 + 12) 2^-23 at most if all terms had one sign, and by that of their norm here."""
    g = torch.Generator(device=DEV).manual_seed(m + 2 * n + k)
    x = torch.randn(m, k, generator=g, device=DEV).to(dtype)
    codes, scales = quantize_fp8_blockwise(torch.randn(n, k, generator=g, device=DEV) * 0.02)
    xc, xs = fp8_block_quant(x, (1, 128))
    want = (xc.double() * spread(xs, m, k, (1, 128))) @ (codes.double() * spread(scales, n, k)).T
    off = float((fp8_block_linear(x, codes, scales).double() - want).norm() / want.norm())
    drop = 2.0 ** -13 * 16 / 128 ** 0.5 if m > 4 and dtype != torch.float32 else 0.0
    assert off < torch.finfo(dtype).eps / 2 + drop + (128 + k // 128 + 12) * 2.0 ** -23, off
