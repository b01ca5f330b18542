"""8-bit quantisation, bit for bit, and the block-scaled product against 64 bits.

Quantisation is IEEE 32-bit arithmetic and one rounding to e4m3, so torch on the CPU gives the same
bits.  The product's values are exact in 32 bits; their sums are 32-bit, over 128 columns on the
tensor core and then over blocks: at most (128 + blocks) roundings, each 2**-23 of the sum of
magnitudes (the tensor core may cut instead of round), and one rounding to the 16-bit output.
"""

import math

import pytest
import torch

from inferkernellab_b200 import (check_device_errors, fp8_linear, quantize_fp8,
                                 quantize_fp8_weight)

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _blocks(x, block_rows):
    """fp32 [row blocks, block_rows, col blocks, 128] of a CPU matrix, zero padded."""
    rows, cols = x.shape
    rb, cb = -(-rows // block_rows), -(-cols // 128)
    wide = torch.zeros((rb * block_rows, cb * 128))
    wide[:rows, :cols] = x.float()
    return wide.view(rb, block_rows, cb, 128)


def _quantized(x, block_rows):
    x = x.cpu()
    b = _blocks(x, block_rows)
    peak = b.abs().amax(dim=(1, 3))
    peak = torch.where(peak < 2.0 ** -100, 0.0, peak)
    inverse = torch.where(peak == 0, 0.0, peak.reciprocal() * 448.0)
    q = (b * inverse[:, None, :, None]).to(torch.float8_e4m3fn)
    q = q.reshape(b.shape[0] * block_rows, -1)[:x.shape[0], :x.shape[1]]
    return q, peak / 448.0


def _same(got, want):
    q, s = got[0].cpu(), got[1].cpu()
    assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float32
    assert q.shape == want[0].shape and s.shape == want[1].shape
    nan = want[0].float().isnan()
    assert torch.equal(q.float().isnan(), nan)
    assert torch.equal(q.contiguous().view(torch.uint8)[~nan], want[0].contiguous().view(torch.uint8)[~nan])
    assert torch.equal(s.nan_to_num(nan=-1), want[1].nan_to_num(nan=-1))


def _normal(shape, seed, dtype, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(shape, generator=gen, device="cuda")).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 16), (3, 127), (5, 128), (64, 129), (33, 144),
                                       (7, 1000), (2, 4096), (257, 640), (31, 14336)])
def test_quantisation_bit_for_bit(dtype, rows, cols):
    x = _normal((rows, cols), rows * cols, DTYPES[dtype], 4.0)
    _same(quantize_fp8(x), _quantized(x, 1))
    _same(quantize_fp8_weight(x), _quantized(x, 128))
    wide = _normal((rows, cols + 5), rows + cols, DTYPES[dtype])
    view = wide[:, 3:3 + cols]  # unaligned rows
    _same(quantize_fp8(view), _quantized(view, 1))
    _same(quantize_fp8_weight(view), _quantized(view, 128))
    q, _ = quantize_fp8(x)
    assert q.stride(0) % 16 == 0


def test_blocks_of_zeros_tiny_and_infinite_values():
    x = _normal((8, 512), 3, torch.bfloat16)
    x[0] = 0
    x[1] = 2.0 ** -120
    x[2, 130] = math.inf
    x[3, 130] = math.nan
    x[4] = torch.finfo(torch.bfloat16).max
    x[5, 0] = 2.0 ** 100
    x[6, :256] = -0.0
    got = quantize_fp8(x)
    _same(got, _quantized(x, 1))
    back = got[0].float() * got[1].repeat_interleave(128, 1)
    assert bool((back[:2] == 0).all())
    assert bool(back[2:4, 128:256].isnan().any(dim=1).all())
    assert not bool(back[2:4, 256:].isnan().any()) and not bool(back[4:].isnan().any())
    assert quantize_fp8(x[:0])[0].shape == (0, 512)


def _weights(n, k, seed):
    w = _normal((n, k), seed, torch.bfloat16, 0.05)
    pitch = -(-k // 16) * 16
    q, s = quantize_fp8_weight(w)
    assert q.stride(0) == pitch
    return q, s


def _exact(xq, xs, wq, ws):
    """(value, sum of magnitudes) in 64 bits from the 8-bit values and scales."""
    m, k = xq.shape
    n = wq.shape[0]
    x, w = xq.to(torch.float32).double(), wq.to(torch.float32).double()
    value = torch.zeros((m, n), dtype=torch.float64, device=x.device)
    size = torch.zeros_like(value)
    row = torch.arange(n, device=x.device) // 128
    for b in range(-(-k // 128)):
        part = slice(128 * b, min(k, 128 * b + 128))
        scale = xs[:, b:b + 1].double() * ws[row, b].double()
        value += x[:, part] @ w[:, part].t() * scale
        size += x[:, part].abs() @ w[:, part].t().abs() * scale
    return value, size


def _close(got, value, size, blocks, dtype):
    unit = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    bound = unit * value.abs() + (128 + blocks) * 2.0 ** -23 * size + 2.0 ** -25
    worst = float(((got.double() - value).abs() / bound).max())
    assert worst <= 1.001, worst


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [
    (1, 1, 16), (1, 128, 128), (1, 6144, 4096), (2, 129, 144), (15, 200, 1024), (16, 127, 256),
    (17, 384, 112), (31, 1000, 2048), (33, 257, 4096), (64, 4096, 1024), (65, 300, 400),
    (100, 513, 14336), (128, 128, 640), (129, 130, 768), (200, 1000, 512), (256, 256, 256),
    (257, 385, 1040), (700, 2049, 384), (1000, 7, 2048), (2048, 1024, 128),
    # enough tiles for pairs of CTAs: ragged in every direction, one block and many
    (2100, 2309, 272), (300, 9500, 1040), (4097, 1281, 16), (2560, 2048, 4096)])
def test_product_against_64_bits(dtype, m, n, k):
    dtype = DTYPES[dtype]
    x = _normal((m, k), m + n + k, dtype, 2.0)
    wq, ws = _weights(n, k, n * 3 + k)
    got = fp8_linear(x, wq, ws)
    assert got.shape == (m, n) and got.dtype == dtype
    xq, xs = quantize_fp8(x)
    value, size = _exact(xq, xs, wq, ws)
    _close(got, value, size, xs.shape[1], dtype)
    assert torch.equal(fp8_linear(x, wq, ws), got)  # no dependence on timing
    assert torch.equal(fp8_linear(xq, wq, ws, x_scales=xs, dtype=dtype), got)
    assert check_device_errors() == 0


def test_bias_out_strides_and_scale_layouts():
    m, n, k = 37, 260, 528
    x = _normal((m, k + 8), 5, torch.bfloat16)[:, 1:1 + k]  # unaligned rows
    wq, ws = _weights(n, k, 6)
    bias = _normal((2 * n,), 7, torch.bfloat16)[::2]
    xq, xs = quantize_fp8(x)
    value, size = _exact(xq, xs, wq, ws)
    wide = torch.full((m, n + 9), 5.0, dtype=torch.bfloat16, device="cuda")
    got = fp8_linear(x, wq, ws, bias=bias, out=wide[:, 3:3 + n])
    assert got.data_ptr() == wide[:, 3:].data_ptr()
    _close(got, value + bias.double(), size + bias.double().abs(), xs.shape[1], torch.bfloat16)
    assert bool((wide[:, :3] == 5).all()) and bool((wide[:, 3 + n:] == 5).all())
    plain = fp8_linear(x, wq, ws)
    # x on rows that TMA cannot address, scales in the other orders
    odd = torch.empty((m, k + 1), dtype=torch.float8_e4m3fn, device="cuda")[:, :k]
    odd.copy_(xq)
    assert torch.equal(fp8_linear(odd, wq, ws, x_scales=xs.contiguous()), plain)
    assert torch.equal(fp8_linear(xq, wq, ws.t().contiguous().t(), x_scales=xs), plain)
    # one row given many times, in both types; a weight of one row
    rows = fp8_linear(xq[:1].expand(5, k), wq, ws, x_scales=xs[:1].expand(5, -1))
    assert torch.equal(rows, plain[:1].expand(5, n))
    assert torch.equal(fp8_linear(x[:1].expand(5, k), wq, ws), plain[:1].expand(5, n))
    assert torch.equal(fp8_linear(x, wq[:1], ws[:1]), plain[:, :1])
    with pytest.raises(ValueError, match="overlap"):
        fp8_linear(x, wq[:1].expand(7, k), ws[:1])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = fp8_linear(x, wq, ws)
    stream.synchronize()
    assert torch.equal(other, plain)


@pytest.mark.parametrize("m", [5, 150])
def test_rows_are_independent(m):
    """A NaN or infinity in one token leaves the others as they are; so do other tokens' values."""
    x = _normal((m, 1024), 8, torch.bfloat16)
    wq, ws = _weights(384, 1024, 9)
    clean = fp8_linear(x, wq, ws)
    dirty = x.clone()
    dirty[2, 700] = math.nan
    dirty[4, 3] = math.inf
    got = fp8_linear(dirty, wq, ws)
    assert bool(got[2].isnan().all()) and bool(got[4].isnan().all())
    rest = [i for i in range(m) if i not in (2, 4)]
    assert torch.equal(got[rest], clean[rest])
    assert torch.equal(fp8_linear(x[1:2], wq, ws)[0].float().isnan(), torch.zeros(384, dtype=torch.bool, device="cuda"))
    zero = fp8_linear(torch.zeros_like(x), wq, ws)
    assert bool((zero == 0).all())


def test_products_on_several_streams_at_once():
    """Every kind of tile (few, many tokens, split K, pairs) beside every other."""
    xs = [_normal((m, 1024), m, torch.bfloat16) for m in (2500, 1, 64, 700)]
    wq, ws = _weights(2560, 1024, 21)
    want = [fp8_linear(x, wq, ws) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for i, stream in enumerate(streams):
        with torch.cuda.stream(stream):
            got.append([fp8_linear(xs[(i + j) % 4], wq, ws) for j in range(4)])
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        assert all(torch.equal(out, want[(i + j) % 4]) for j, out in enumerate(outs))
    assert check_device_errors() == 0


def test_refusals():
    x = _normal((4, 256), 1, torch.bfloat16)
    wq, ws = _weights(130, 256, 2)
    assert fp8_linear(x[:0], wq, ws).shape == (0, 130)
    xq, xs = quantize_fp8(x)
    for match, call in (
            ("float8_e4m3fn", lambda: fp8_linear(x, wq.float(), ws)),
            ("weight's K", lambda: fp8_linear(x[:, :128], wq, ws)),
            ("weight_scales", lambda: fp8_linear(x, wq, ws[:1])),
            ("weight_scales", lambda: fp8_linear(x, wq, ws.double())),
            ("16-byte", lambda: fp8_linear(x[:, :100].contiguous(), wq[:, :100].contiguous(), ws[:, :1].contiguous())),
            ("x_scales", lambda: fp8_linear(xq, wq, ws)),
            ("x_scales", lambda: fp8_linear(xq, wq, ws, x_scales=xs[:2])),
            ("belong to", lambda: fp8_linear(x, wq, ws, x_scales=xs)),
            ("has its dtype", lambda: fp8_linear(x, wq, ws, dtype=torch.float16)),
            ("x must be", lambda: fp8_linear(x.float(), wq, ws)),
            ("result must be", lambda: fp8_linear(xq, wq, ws, x_scales=xs, dtype=torch.float32)),
            ("bias", lambda: fp8_linear(x, wq, ws, bias=x[0])),
            ("out must", lambda: fp8_linear(x, wq, ws, out=x)),
            ("2-D", lambda: quantize_fp8(x[0])),
            ("2-D", lambda: quantize_fp8(x.float())),
            ("2-D", lambda: quantize_fp8_weight(x.cpu()))):
        with pytest.raises(ValueError, match=match):
            call()
