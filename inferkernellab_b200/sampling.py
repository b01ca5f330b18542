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
from .ops import _raw_stream

_LOGITS_CODE = {torch.float16: _lib.B200_F16, torch.bfloat16: _lib.B200_BF16,
                torch.float32: _lib.B200_F32}


def _number(value, name: str, off, check):
    """A setting given as a number (``None``: off), checked."""
    if value is None:
        return off
    if isinstance(off, int) and not isinstance(value, int) and not float(value).is_integer():
        raise ValueError(f"{name} must be a whole number: {value}")
    value = type(off)(value)
    if not check(value):
        raise ValueError(f"{name} is out of range: {value}")
    return value


def _per_row(value: torch.Tensor, name: str, uniforms: torch.Tensor, dtype) -> torch.Tensor:
    """A setting given as one entry per row, contiguous."""
    if (value.dtype != dtype or value.shape != uniforms.shape
            or value.get_device() != uniforms.get_device()):
        raise ValueError(f"{name} must hold one {str(dtype)[6:]} entry per row on the logits device")
    return value if value.is_contiguous() else value.contiguous()


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
    index = logits.get_device()
    if logits.ndim != 2 or index < 0:
        raise ValueError("logits must be a CUDA tensor with shape [B, V]")
    code = _LOGITS_CODE.get(logits.dtype)
    if code is None:
        raise ValueError("logits must be float16, bfloat16 or float32")
    rows, vocab = logits.shape
    if vocab <= 0:
        raise ValueError("logits must have at least one column")
    f32 = torch.float32
    if uniforms.dtype != f32 or uniforms.shape != (rows,) or uniforms.get_device() != index:
        raise ValueError("uniforms must hold one float32 entry per row on the logits device")
    row_stride, column_stride = logits.stride()
    if column_stride != 1:
        logits = logits.contiguous()
        row_stride = vocab
    if not uniforms.is_contiguous():
        uniforms = uniforms.contiguous()
    t, k, p, m = 1.0, 0, 1.0, 0.0
    t_ptr = k_ptr = p_ptr = m_ptr = None
    if isinstance(temperature, torch.Tensor):
        temperature = _per_row(temperature, "temperature", uniforms, f32)
        t_ptr = temperature.data_ptr()
    else:
        t = _number(temperature, "temperature", 1.0, lambda v: 0.0 <= v < math.inf)
        if t > 0.0:
            t = max(t, 2.0 ** -149)  # positive in 32 bits, too
    if isinstance(top_k, torch.Tensor):
        top_k = _per_row(top_k, "top_k", uniforms, torch.int32)
        k_ptr = top_k.data_ptr()
    else:
        k = _number(top_k, "top_k", 0, lambda v: 0 <= v < 2 ** 31)
    if isinstance(top_p, torch.Tensor):
        top_p = _per_row(top_p, "top_p", uniforms, f32)
        p_ptr = top_p.data_ptr()
    else:
        p = _number(top_p, "top_p", 1.0, lambda v: 0.0 < v <= 1.0)
    if isinstance(min_p, torch.Tensor):
        min_p = _per_row(min_p, "min_p", uniforms, f32)
        m_ptr = min_p.data_ptr()
    else:
        m = _number(min_p, "min_p", 0.0, lambda v: 0.0 <= v <= 1.0)
    tokens = uniforms.new_empty(rows, dtype=torch.int64)
    logprobs, sampling = torch.empty_like(uniforms), torch.empty_like(uniforms)
    args = _lib.SampleArgs(rows, row_stride, vocab, code, t, k, p, m)
    _lib.check(_lib.load().b200_sample_tokens(
        ctypes.byref(args), logits.data_ptr(), uniforms.data_ptr(), t_ptr, k_ptr, p_ptr, m_ptr,
        tokens.data_ptr(), logprobs.data_ptr(), sampling.data_ptr(), _raw_stream(index)))
    return tokens, logprobs, sampling
