"""Projections in 8-bit floating point (e4m3) with block scales.

``quantize_fp8`` gives activations one scale per row and 128 columns, ``quantize_fp8_weight`` a
weight one scale per 128 x 128 block, and ``fp8_linear`` multiplies the two on the tensor cores with
32-bit sums.  A decode step reads every weight once, so 8 bits halve its bytes against bfloat16.
The reference has no 8-bit path.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ops import _DTYPE_CODE, _ERROR_WORDS, _raw_stream

BLOCK = 128  # columns (and weight rows) that share a scale


def _matrix16(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.ndim != 2 or t.get_device() < 0 or t.dtype not in _DTYPE_CODE:
        raise ValueError(f"{name} must be a 2-D float16/bfloat16 CUDA tensor")
    if t.shape[1] <= 0:
        raise ValueError(f"{name} must have at least one column")
    return t if t.stride(1) == 1 else t.contiguous()


def _empty_fp8(rows: int, cols: int, device: torch.device) -> torch.Tensor:
    """Uninitialised e4m3 ``[rows, cols]`` whose rows start on 16-byte boundaries."""
    pitch = -(-cols // 16) * 16
    t = torch.empty((rows, pitch), dtype=torch.float8_e4m3fn, device=device)
    return t if pitch == cols else t[:, :cols]


def quantize_fp8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, scales)`` of 16-bit activations ``[M, K]``: ``x ~ q * scales`` with a scale per row and
    128 columns.

    ``scales[m, b] = max |x[m, 128 b : 128 b + 128]| / 448``; ``q`` is e4m3 ``[M, K]``, the nearest
    value of ``x * (448 * (1 / max))``, with rows on 16-byte boundaries, and ``scales`` float32
    ``[M, ceil(K / 128)]``, stored block by block (the order in which ``fp8_linear`` reads it).  A
    block whose largest magnitude is below 2**-100 becomes zeros; one that holds a NaN or an
    infinity stands for NaN.
    """
    x = _matrix16(x, "x")
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    q = _empty_fp8(rows, cols, x.device)
    scales = torch.empty_strided((rows, blocks), (1, rows), dtype=torch.float32, device=x.device)
    _lib.check(_lib.load().b200_quantize_fp8(
        x.data_ptr(), rows, cols, x.stride(0), _DTYPE_CODE[x.dtype], 1, q.data_ptr(), q.stride(0),
        scales.data_ptr(), 1, rows, _raw_stream(x.get_device())))
    return q, scales


def quantize_fp8_weight(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, scales)`` of a 16-bit weight ``[N, K]`` with a scale per 128 x 128 block: e4m3 ``[N, K]``
    and float32 ``[ceil(N / 128), ceil(K / 128)]``, as ``fp8_linear`` takes them."""
    weight = _matrix16(weight, "weight")
    rows, cols = weight.shape
    q = _empty_fp8(rows, cols, weight.device)
    scales = torch.empty((-(-rows // BLOCK), -(-cols // BLOCK)), dtype=torch.float32,
                         device=weight.device)
    _lib.check(_lib.load().b200_quantize_fp8(
        weight.data_ptr(), rows, cols, weight.stride(0), _DTYPE_CODE[weight.dtype], BLOCK,
        q.data_ptr(), q.stride(0), scales.data_ptr(), scales.stride(0), 1,
        _raw_stream(weight.get_device())))
    return q, scales


def fp8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor, *,
               x_scales: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ weight.T (+ bias)`` with an e4m3 ``weight`` ``[N, K]`` and its ``weight_scales``
    ``[ceil(N / 128), ceil(K / 128)]``.

    ``x`` is 16-bit ``[M, K]``, quantised as by ``quantize_fp8`` on the way, or already e4m3 with its
    ``x_scales`` ``[M, ceil(K / 128)]``.  The result ``[M, N]`` has ``x``'s dtype (``dtype``, by
    default bfloat16, if ``x`` is e4m3); products are summed in 32 bits and rounded once.  ``weight``
    rows have to start on 16-byte boundaries (``K`` a multiple of 16, or padded rows).
    """
    index = weight.get_device()
    if weight.ndim != 2 or weight.dtype != torch.float8_e4m3fn or index < 0:
        raise ValueError("weight must be a 2-D float8_e4m3fn CUDA tensor")
    outs, cols = weight.shape
    if x.ndim != 2 or x.shape[1] != cols or x.get_device() != index:
        raise ValueError("x must be [M, K] with the weight's K, on its device")
    blocks = -(-cols // BLOCK)
    if (weight_scales.shape != (-(-outs // BLOCK), blocks)
            or weight_scales.dtype != torch.float32 or weight_scales.get_device() != index):
        raise ValueError("weight_scales must be float32 [ceil(N / 128), ceil(K / 128)] on the "
                         "weight's device")
    w_stride, w_step = weight.stride()
    if w_step != 1 or w_stride % 16 or weight.data_ptr() % 16:
        raise ValueError("weight rows must be contiguous and start on 16-byte boundaries "
                         "(K a multiple of 16, or padded rows)")
    rows = x.shape[0]
    workspace, sx, xs_row, xs_block = None, None, 0, 0
    if x.dtype == torch.float8_e4m3fn:
        if x_scales is None:
            raise ValueError("an e4m3 x needs its x_scales")
        if (x_scales.shape != (rows, blocks) or x_scales.dtype != torch.float32
                or x_scales.get_device() != index):
            raise ValueError("x_scales must be float32 [M, ceil(K / 128)] on x's device")
        if x.stride(1) != 1 or x.stride(0) % 16 or x.stride(0) < cols or x.data_ptr() % 16:
            padded = _empty_fp8(rows, cols, x.device)
            padded.copy_(x)
            x = padded
        dtype = dtype or torch.bfloat16
        x_code = _lib.B200_E4M3
        sx, (xs_row, xs_block) = x_scales.data_ptr(), x_scales.stride()
    else:
        if x_scales is not None:
            raise ValueError("x_scales belong to an e4m3 x")
        if dtype is not None and dtype != x.dtype:
            raise ValueError("the result of a 16-bit x has its dtype")
        dtype = x.dtype
        x_code = _DTYPE_CODE.get(dtype)
        if x_code is None:
            raise ValueError("x must be float16, bfloat16 or float8_e4m3fn")
        if x.stride(1) != 1:
            x = x.contiguous()
        # the 8-bit rows, on 16-byte boundaries, and the scales, block by block
        nbytes = rows * (-(-cols // 16) * 16 + 4 * blocks)
        workspace = weight.new_empty(nbytes)  # one byte an element
    code = _DTYPE_CODE.get(dtype)
    if code is None:
        raise ValueError("the result must be float16 or bfloat16")
    if bias is not None:
        if bias.shape != (outs,) or bias.dtype != dtype or bias.get_device() != index:
            raise ValueError("bias must be [N] with the result's dtype and device")
        bias = bias if bias.is_contiguous() else bias.contiguous()
    if out is None:
        out = weight.new_empty((rows, outs), dtype=dtype)
    elif (out.shape != (rows, outs) or out.dtype != dtype or out.get_device() != index
          or out.stride(1) != 1):
        raise ValueError("out must be [M, N] with the result's dtype, on the weight's device")
    elif rows > 1 and out.stride(0) < outs:
        raise ValueError("rows of out must not overlap")
    ws_row, ws_block = weight_scales.stride()
    args = _lib.Fp8LinearArgs(rows, outs, cols, x.stride(0), w_stride, out.stride(0), xs_row,
                              xs_block, ws_row, ws_block, code, x_code)
    _lib.check(_lib.load().b200_fp8_linear(
        ctypes.byref(args), x.data_ptr(), sx, weight.data_ptr(), weight_scales.data_ptr(),
        bias.data_ptr() if bias is not None else None, out.data_ptr(),
        workspace.data_ptr() if workspace is not None else None,
        workspace.numel() if workspace is not None else 0,
        _ERROR_WORDS.get(weight.device).data_ptr(), _raw_stream(index)))
    return out
