"""``qk_norm_rope_append`` against a 64-bit evaluation.

One rounding to the 16-bit type (relative 2**-8 for bfloat16, 2**-11 for float16, absolute 2**-25
below its normal range) plus 32-bit arithmetic: a handful of roundings of 2**-24 of the two terms of
the rotation, taken as 2**-20 of their magnitudes.
"""

import pytest
import torch

from inferkernellab_b200 import PagedKVCache, _lib, check_device_errors, qk_norm_rope_append

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _turned(x, weight, cos, sin, eps):
    """(value, bound on the magnitudes that enter it) in 64 bits."""
    x = x.double()
    y = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * weight.double()
    rd = cos.shape[1]
    c, s = cos.double()[:, None], sin.double()[:, None]
    r = y[..., :rd]
    half = torch.cat((-r[..., rd // 2:], r[..., :rd // 2]), -1)
    value = torch.cat((r * c + half * s, y[..., rd:]), -1)
    size = torch.cat(((r * c).abs() + (half * s).abs(), y[..., rd:].abs()), -1)
    return value, size


def _close(got, want, size, dtype):
    unit = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    bound = unit * want.abs() + 2.0 ** -20 * size + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126)
    worst = (got.double() - want).abs() / bound
    assert float(worst.max()) <= 1.001, float(worst.max())


def _inputs(tokens, hq, hkv, dim, rd, dtype, seed, pad=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    qkv = (3 * normal(tokens, (hq + 2 * hkv) * dim + pad)).to(dtype)[:, pad:]
    q = qkv[:, :hq * dim].view(tokens, hq, dim)
    k = qkv[:, hq * dim:(hq + hkv) * dim].view(tokens, hkv, dim)
    v = qkv[:, (hq + hkv) * dim:].view(tokens, hkv, dim)
    qw, kw = ((1 + 0.2 * normal(dim)).to(dtype) for _ in range(2))
    angle = 100 * normal(tokens, rd)  # cos/sin of the two halves need not agree
    return q, k, v, qw, kw, angle.cos().to(dtype), angle.sin().to(dtype)


def _run(tokens, hq, hkv, dim, rd, dtype, slot_dtype=torch.int32, pad=0, block=16, eps=1e-6):
    q, k, v, qw, kw, cos, sin = _inputs(tokens, hq, hkv, dim, rd, dtype, tokens + dim + rd, pad)
    blocks = -(-tokens // block) + 3
    cache = PagedKVCache(blocks, block, hkv, dim, num_layers=3, dtype=dtype, device="cuda")
    cache.k.fill_(7.0)
    cache.v.fill_(7.0)
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    slots = torch.randperm(blocks * block, generator=gen, device="cuda")[:tokens].to(slot_dtype)
    if tokens > 4:
        slots[3] = -1  # a padding token: rotated q, no append
    keep = [t.clone() for t in (q, k, v)]
    out = qk_norm_rope_append(q, k, v, qw, kw, cos, sin, cache, slots, layer=1, eps=eps)
    assert all(torch.equal(a, b) for a, b in zip((q, k, v), keep))
    _close(out, *_turned(q, qw, cos, sin, eps), dtype)
    live = slots >= 0
    at = slots[live].long()
    got_k, got_v = (t[1].reshape(-1, hkv, dim) for t in (cache.k, cache.v))
    value, size = _turned(k, kw, cos, sin, eps)
    _close(got_k[at], value[live], size[live], dtype)
    assert torch.equal(got_v[at], v[live])
    untouched = torch.ones(blocks * block, dtype=torch.bool, device="cuda")
    untouched[at] = False
    assert bool((got_k[untouched] == 7).all()) and bool((got_v[untouched] == 7).all())
    assert bool((cache.k[::2] == 7).all()) and bool((cache.v[::2] == 7).all())
    assert check_device_errors() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,hq,hkv,dim,rd", [
    (1, 32, 8, 128, 128), (53, 32, 8, 128, 128), (300, 8, 2, 64, 64), (17, 4, 4, 16, 16),
    (9, 6, 3, 32, 32), (33, 4, 1, 256, 256), (21, 16, 2, 128, 64), (13, 4, 2, 64, 48),
    (11, 4, 2, 64, 20), (19, 3, 1, 80, 80), (8, 2, 2, 96, 32), (6, 2, 1, 34, 2), (5, 1, 1, 2, 2),
    (7, 96, 16, 128, 128)])
def test_against_64_bits(dtype, tokens, hq, hkv, dim, rd):
    _run(tokens, hq, hkv, dim, rd, DTYPES[dtype])


def test_index_types_alignment_and_eps():
    _run(40, 8, 2, 128, 128, torch.bfloat16, slot_dtype=torch.int64)
    _run(40, 8, 2, 128, 128, torch.bfloat16, pad=3)  # rows off the 16-byte grid
    _run(40, 8, 2, 64, 64, torch.float16, block=1, eps=0.5)
    _run(2500, 4, 2, 64, 64, torch.bfloat16)


def test_zero_rows_huge_rows_and_nan_stay_in_their_place():
    q, k, v, qw, kw, cos, sin = _inputs(4, 2, 1, 128, 128, torch.bfloat16, 1)
    q, k = q.clone(), k.clone()
    q[0, 0] = 0
    q[1, 1] = torch.randn(128, device="cuda").to(torch.bfloat16) * 2.0 ** 60  # squares overflow bf16 only
    q[2, 0, 5] = float("nan")
    cache = PagedKVCache(2, 16, 1, 128, dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(4, dtype=torch.int32, device="cuda")
    out = qk_norm_rope_append(q, k, v, qw, kw, cos, sin, cache, slots)
    assert bool((out[0, 0] == 0).all())
    value, size = _turned(q, qw, cos, sin, 1e-6)
    _close(out[1], value[1], size[1], torch.bfloat16)
    assert bool(out[2, 0].isnan().all()) and not bool(out[2, 1].isnan().any())


def test_bad_slot_no_tokens_and_refusals():
    q, k, v, qw, kw, cos, sin = _inputs(3, 4, 2, 64, 64, torch.bfloat16, 2)
    cache = PagedKVCache(2, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    cache.k.zero_()
    slots = torch.tensor([0, 32, 1], dtype=torch.int32, device="cuda")
    out = torch.empty((3, 4, 64), dtype=torch.bfloat16, device="cuda")
    assert qk_norm_rope_append(q, k, v, qw, kw, cos, sin, cache, slots, out=out) is out
    assert check_device_errors() == _lib.DEVERR_BAD_SLOT
    assert bool((cache.k[0, 0, 2:] == 0).all()) and bool((cache.k[0, 1] == 0).all())
    none = qk_norm_rope_append(q[:0], k[:0], v[:0], qw, kw, cos[:0], sin[:0], cache, slots[:0])
    assert none.shape == (0, 4, 64)

    def refused(match, error=ValueError, **kw_):
        a = dict(query=q, key=k, value=v, q_weight=qw, k_weight=kw, cos=cos, sin=sin, cache=cache,
                 slots=slots) | kw_
        with pytest.raises(error, match=match):
            qk_norm_rope_append(**a)

    refused("layout", key=k[:, :1], value=v[:, :1])
    refused("layer", IndexError, layer=1)
    refused("q_weight", q_weight=qw[:32])
    refused("one row per token", cos=cos[:2], sin=sin[:2])
    refused("even", cos=cos[:, :3], sin=sin[:, :3])
    refused("cache dtype", query=q.half())
    refused("cache dtype", cos=cos.float(), sin=sin.float())
    refused("counts", slots=slots[:2])
    refused("int32 or int64", slots=slots.float())
    refused("same CUDA device", slots=slots.cpu())
    refused("eps", eps=-1.0)
    refused("out must", out=out.half())
    refused("divisible", query=q[:, :3])
