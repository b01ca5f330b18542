"""``sample_tokens`` called from several host threads, and on rows that only its exact search cuts."""

import ctypes
import math
import threading

import pytest
import torch

from inferkernellab_b200 import _lib, sample_tokens
from tests.test_gpu_sampling import _check, _delta, _logits

pytestmark = pytest.mark.gpu


def test_host_threads_with_rows_of_different_sizes():
    """Launches that need much and little shared memory, from threads that do not wait for each
    other: the C entry point in a tight loop, outside the interpreter lock."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    lib, calls = _lib.load(), 4000
    jobs = []
    for rows, vocab in [(1, 128256), (1, 500), (1, 100000), (1, 3000)]:
        x = 3 * torch.randn((rows, vocab), generator=gen, device="cuda").bfloat16()
        u = torch.rand(rows, generator=gen, device="cuda")
        want = sample_tokens(x, u, top_k=40)[0]
        token, a, b = torch.zeros_like(want), torch.zeros_like(u), torch.zeros_like(u)
        args = _lib.SampleArgs(rows, vocab, vocab, _lib.B200_BF16, 1.0, 40, 1.0, 0.0)
        stream = torch.cuda.Stream()
        jobs.append((x, u, want, token, a, b, args, stream, (
            ctypes.byref(args), x.data_ptr(), u.data_ptr(), None, None, None, None,
            token.data_ptr(), a.data_ptr(), b.data_ptr(), stream.cuda_stream)))
    torch.cuda.synchronize()
    start, refused = threading.Barrier(len(jobs)), []

    def work(call):
        start.wait()
        for _ in range(calls):
            if lib.b200_sample_tokens(*call) != _lib.B200_OK:
                refused.append(_lib.last_error())

    threads = [threading.Thread(target=work, args=job[-1:]) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not refused, (len(refused), refused[0])
    for _, _, want, token, *_ in jobs:
        assert torch.equal(token, want)


def test_a_temperature_below_32_bits_is_not_greedy():
    """1e-50 is no 32-bit number, but it is positive: equal largest logits are drawn from, and the
    log-probabilities are those of that temperature, not of 1."""
    logits = torch.tensor([[1.0, 2.0, 2.0, 0.0]] * 2, device="cuda")
    uniforms = torch.tensor([0.1, 0.6], device="cuda")
    tokens, logprobs, sampling = sample_tokens(logits, uniforms, temperature=1e-50)
    assert tokens.tolist() == [1, 2]
    half = torch.full_like(uniforms, 0.5)
    assert torch.allclose(logprobs.exp(), half) and torch.allclose(sampling.exp(), half)
    assert sample_tokens(logits, uniforms, temperature=0.0)[0].tolist() == [1, 1]


def _near(rows, vocab, dtype, seed):
    """Rows whose tokens are all likely: no filter leaves few of them."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = 0.6 * torch.rand((rows, vocab), generator=gen, device="cuda")
    return x.to(dtype), torch.rand(rows, generator=gen, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [5003, 50001])
@pytest.mark.parametrize("setting", [
    dict(min_p=0.7), dict(min_p=1.0), dict(temperature=0.5, min_p=0.4, top_p=0.8),
    dict(min_p=0.7, top_k=4000), dict(min_p=0.7, top_k=4000, top_p=0.3)])
def test_min_p_where_many_tokens_pass(dtype, vocab, setting):
    logits, uniforms = _near(4, vocab, dtype, vocab)
    args = dict(temperature=1.0, top_k=None, top_p=None, min_p=None) | setting
    got = sample_tokens(logits, uniforms, **args)
    _check(logits, uniforms, got, **args)
    assert all(torch.equal(a, b) for a, b in zip(got, sample_tokens(logits, uniforms, **args)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("setting", [dict(min_p=0.7), dict(top_k=3000), dict(top_p=0.5),
                                     dict(min_p=0.6, top_k=4000, top_p=0.9)])
@pytest.mark.parametrize("spread", ["near", "wide"])
def test_greedy_rows_with_filters(dtype, setting, spread):
    """The token is the first largest; its sampling log-probability is that among the kept tokens
    at temperature 1.  Kept sums are off by _delta as the masses are, and a cut that 32 and 64 bits
    make at neighbouring tokens moves them by one token's weight more, at most 1 of the sum."""
    logits, uniforms = (_near if spread == "near" else _logits)(5, 20011, dtype, 8)
    args = dict(temperature=0.0, top_k=None, top_p=None, min_p=None) | setting
    got = sample_tokens(logits, uniforms, **args)
    _check(logits, uniforms, got, **args)
    x = logits.double()
    w = (x - x.amax(dim=1, keepdim=True)).exp()
    w = w.sort(dim=1, descending=True, stable=True).values
    kept = w >= (args["min_p"] or 0.0)
    if args["top_k"]:
        kept[:, args["top_k"]:] = False
    sums = (w * kept).cumsum(dim=1)
    if args["top_p"]:
        kept &= sums - w < args["top_p"] * sums[:, -1:]
    total = (w * kept).sum(dim=1)
    for a, b in zip(got[2].tolist(), total.tolist()):
        assert abs(math.exp(-a) - b) <= 1 + b * (2 * _delta(20011) + 2.0 ** -20)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("setting", [dict(temperature=0.8), dict(temperature=0.0),
                                     dict(temperature=1.2, min_p=0.02)])
def test_large_batches(dtype, setting):
    """More rows than the SMs hold at once."""
    logits, uniforms = _logits(400, 9001, dtype, 77)
    args = dict(temperature=1.0, top_k=None, top_p=None, min_p=None) | setting
    _check(logits, uniforms, sample_tokens(logits, uniforms, **args), **args)
