"""Batched token sampling from given uniform numbers, one launch per batch.

The reference's runner samples request by request with torch ops
(``hf_benchmark.py:581-605``: divide by the temperature, sort, softmax, cumulative sum, scatter,
multinomial).  ``sample_tokens`` does a whole batch on the device with no host work, each request
with its own settings, and its result depends on nothing but its inputs.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .ops import _stream_ptr

_LOGITS_CODE = {torch.float16: _lib.B200_F16, torch.bfloat16: _lib.B200_BF16,
                torch.float32: _lib.B200_F32}


def _setting(value, name: str, rows: int, device: torch.device, dtype: torch.dtype, default,
             check):
    """(device pointer or None, scalar) of a setting given as a number or one entry per row."""
    if value is None:
        return None, None, default
    if isinstance(value, torch.Tensor) and value.ndim > 0:
        if value.shape != (rows,) or value.dtype != dtype or value.device != device:
            raise ValueError(f"{name} must hold one {str(dtype)[6:]} entry per row on the logits "
                             "device")
        value = value if value.is_contiguous() else value.contiguous()
        return value, value.data_ptr(), default
    value = type(default)(value)
    if not check(value):
        raise ValueError(f"{name} is out of range: {value}")
    return None, None, value


def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor, *, temperature=1.0, top_k=None,
                  top_p=None, min_p=None):
    """Draw one token per row of ``logits`` ``[B, V]`` (float16, bfloat16 or float32).

    With ``w = exp((logits - max) / temperature)`` and the tokens of a row in order of ``w`` (equal
    ones by index), a token is kept if ``w >= min_p``, if it is among the first ``top_k`` of those,
    and if what precedes it of those has less than ``top_p`` of their mass.  The token is the first
    one, in order of index, at which the running mass of the kept ones passes ``uniforms[b]`` times
    their sum; ``uniforms`` is float32 ``[B]`` in ``[0, 1)``.  ``temperature=0`` takes the first
    largest logit.

    Each setting is a number or a tensor with one entry per row (float32; ``top_k`` int32).
    Numbers are checked; tensors are not read on the host: a temperature that is not positive is
    greedy, ``top_k <= 0``, ``top_p >= 1`` and ``min_p <= 0`` are off, as ``None`` is.  NaN logits
    count as ``-inf``; a row that holds nothing else gives token -1 and log-probabilities ``-inf``.

    Returns ``(tokens, logprobs, sampling_logprobs)``: int64 ``[B]``, and float32 ``[B]`` log
    probabilities of the token under the temperature alone and among the kept tokens (those of
    temperature 1 where it is 0).  Nothing is read back to the host.
    """
    if logits.ndim != 2 or logits.device.type != "cuda":
        raise ValueError("logits must be a CUDA tensor with shape [B, V]")
    code = _LOGITS_CODE.get(logits.dtype)
    if code is None:
        raise ValueError("logits must be float16, bfloat16 or float32")
    rows, vocab = logits.shape
    if vocab <= 0:
        raise ValueError("logits must have at least one column")
    device = logits.device
    if uniforms.shape != (rows,) or uniforms.dtype != torch.float32 or uniforms.device != device:
        raise ValueError("uniforms must hold one float32 entry per row on the logits device")
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    if not uniforms.is_contiguous():
        uniforms = uniforms.contiguous()
    f32 = torch.float32
    # The first of each triple keeps a contiguous copy alive until the launch.
    t_keep, t_ptr, t = _setting(temperature, "temperature", rows, device, f32, 1.0,
                                lambda v: 0.0 <= v < math.inf)
    k_keep, k_ptr, k = _setting(top_k, "top_k", rows, device, torch.int32, 0,
                                lambda v: 0 <= v < 2 ** 31)
    p_keep, p_ptr, p = _setting(top_p, "top_p", rows, device, f32, 1.0, lambda v: 0.0 < v <= 1.0)
    m_keep, m_ptr, m = _setting(min_p, "min_p", rows, device, f32, 0.0, lambda v: 0.0 <= v <= 1.0)
    tokens = torch.empty(rows, dtype=torch.int64, device=device)
    logprobs = torch.empty((2, rows), dtype=f32, device=device)
    args = _lib.SampleArgs(rows, logits.stride(0), vocab, code, t, k, p, m)
    out = logprobs.data_ptr()
    _lib.check(_lib.load().b200_sample_tokens(
        ctypes.byref(args), logits.data_ptr(), uniforms.data_ptr(), t_ptr, k_ptr, p_ptr, m_ptr,
        tokens.data_ptr(), out, out + 4 * rows, _stream_ptr(device)))
    return tokens, logprobs[0], logprobs[1]
