"""``sample_tokens`` called from several host threads, and on rows that only its exact search cuts."""

import ctypes
import threading

import pytest
import torch

from inferkernellab_b200 import _lib, sample_tokens

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
