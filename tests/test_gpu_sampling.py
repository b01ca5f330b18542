"""``sample_tokens`` against a 64-bit evaluation of its definition.

Masses are whole numbers of 2**-31 of the largest weight, from 32-bit weights.  Against 64 bits a
weight is off by 3 roundings of its exponent's argument x (3 * 2**-24 * |x|, |x| <= 22 where it
counts), 2 units in the last place of exp, and half a mass unit: relative to the row's mass that is
at most DELTA = 22 * 3 * 2**-24 + 2**-22 + V * 2**-32.  So the token's interval of the running mass
has to hold the uniform number within DELTA, and rows whose top-p cut falls closer than DELTA to a
boundary (where 32 and 64 bits may cut differently) are only held to the cut that was made.
"""

import math

import pytest
import torch

from inferkernellab_b200 import sample_tokens

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _delta(vocab):
    return 22 * 3 * 2.0 ** -24 + 2.0 ** -22 + vocab * 2.0 ** -32


def _check_row(logits, u, t, k, p, m, token, logprob, sampling):
    """One row against the definition in 64 bits (CPU)."""
    x = logits.double().cpu()
    x = torch.where(x.isnan(), -math.inf, x)
    vocab = x.numel()
    delta = _delta(vocab)
    peak = x.max()
    if peak == -math.inf:
        assert token == -1 and logprob == -math.inf and sampling == -math.inf
        return
    if peak == math.inf:
        z = torch.where(x == math.inf, 0.0, -math.inf)
    else:
        z = (x - peak) / (t if t > 0 else 1.0)
    w = z.exp()
    order = w.sort(descending=True, stable=True).indices
    ranked = w[order]
    n = int((ranked >= m).sum()) if m > 0 else vocab
    if k > 0:
        n = min(n, k)
    sums = ranked[:n].cumsum(0)
    sure = True
    if p < 1:
        before = (sums - ranked[:n]) / sums[-1]
        sure = bool((before - p).abs().min() > 2 * delta)
        n = max(1, int((before < p).sum()))
    kept = torch.zeros(vocab, dtype=torch.bool)
    kept[order[:n]] = True
    assert abs(logprob - float(z[token] - w.sum().log())) <= 2 * delta + 2.0 ** -22 * (1 + abs(logprob))
    if t <= 0:
        assert token == int((x == peak).nonzero()[0])
        return
    if not sure:
        return
    assert kept[token]
    total = w[kept].sum()
    running = (w * kept).cumsum(0) / total
    high = float(running[token])
    low = high - float(w[token] / total)
    assert low - 2 * delta <= u <= high + 2 * delta, (low, u, high)
    want = float(z[token] - total.log())
    assert abs(sampling - want) <= 2 * delta + 2.0 ** -22 * (1 + abs(sampling))


def _check(logits, uniforms, got, temperature, top_k, top_p, min_p):
    tokens, logprobs, sampling = (v.cpu().tolist() for v in got)

    def at(v, i, off):
        return off if v is None else float(v[i]) if isinstance(v, torch.Tensor) else float(v)

    for i in range(logits.shape[0]):
        _check_row(logits[i], float(uniforms[i]), at(temperature, i, 1.0), int(at(top_k, i, 0)),
                   at(top_p, i, 1.0), at(min_p, i, 0.0), tokens[i], logprobs[i], sampling[i])


def _logits(rows, vocab, dtype, seed, spread=2.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = spread * torch.randn((rows, vocab), generator=gen, device="cuda")
    x[:, :: max(1, vocab // 20)] += 8 * torch.rand(x[:, :: max(1, vocab // 20)].shape, generator=gen,
                                                 device="cuda")
    return x.to(dtype), torch.rand(rows, generator=gen, device="cuda")


SETTINGS = {
    "plain": dict(temperature=0.8),
    "greedy": dict(temperature=0.0),
    "top_k": dict(temperature=1.0, top_k=40),
    "top_p": dict(temperature=1.3, top_p=0.92),
    "min_p": dict(temperature=0.7, min_p=0.03),
    "all": dict(temperature=1.1, top_k=300, top_p=0.9, min_p=0.001),
    "hot": dict(temperature=50.0, top_p=0.7),
}


@pytest.mark.parametrize("setting", SETTINGS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(3, 1), (4, 2), (5, 31), (7, 250), (2, 4097), (3, 32773),
                                        (2, 128257)])
def test_sampling_against_64_bits(rows, vocab, dtype, setting):
    logits, uniforms = _logits(rows, vocab, DTYPES[dtype], rows * vocab)
    args = dict(temperature=1.0, top_k=None, top_p=None, min_p=None) | SETTINGS[setting]
    if args["top_k"]:
        args["top_k"] = min(args["top_k"], vocab)
    _check(logits, uniforms, sample_tokens(logits, uniforms, **args), **args)


@pytest.mark.parametrize("dtype", DTYPES)
def test_settings_per_row_strided_rows_and_another_stream(dtype):
    rows, vocab = 37, 5003
    base, uniforms = _logits(rows, vocab + 5, DTYPES[dtype], 3)
    logits = base[:, 3:3 + vocab]  # odd start and row stride: unaligned rows
    i = torch.arange(rows, device="cuda")
    args = dict(temperature=torch.where(i % 4 == 0, 0.0, 0.5 + 0.05 * i), top_k=(i % 5 * 30).int(),
                top_p=0.5 + 0.5 * (i % 6) / 5, min_p=torch.where(i % 3 == 0, 0.02, 0.0))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = sample_tokens(logits, uniforms, **args)
    stream.synchronize()
    _check(logits, uniforms, got, **args)
    again = sample_tokens(logits, uniforms, **args)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    flipped = sample_tokens(logits.t().contiguous().t(), uniforms, **args)  # column-major logits
    assert all(torch.equal(a, b) for a, b in zip(got, flipped))


@pytest.mark.parametrize("vocab", [700, 60000, 128256])
def test_equal_logits_are_cut_and_drawn_by_index(vocab):
    """All weights 1: every mass is exact, so the token is known exactly."""
    uniforms = torch.tensor([0.0, 0.25, 0.5, 0.999, 1 - 2.0 ** -24, 1.0], device="cuda")
    logits = torch.full((6, vocab), 3.0, device="cuda", dtype=torch.bfloat16)
    tokens, logprobs, sampling = sample_tokens(logits, uniforms)
    want = [min(int(float(u) * vocab), vocab - 1) for u in uniforms]
    assert tokens.tolist() == want
    assert torch.allclose(logprobs, torch.full_like(logprobs, -math.log(vocab)), rtol=1e-6)
    k = vocab - 77
    assert sample_tokens(logits, uniforms, top_k=k)[0].tolist() == [min(int(float(u) * k), k - 1)
                                                                  for u in uniforms]
    half = -(-vocab // 2)
    tokens, _, sampling = sample_tokens(logits, uniforms, top_p=0.5)
    assert tokens.tolist() == [min(int(float(u) * half), half - 1) for u in uniforms]
    assert torch.allclose(sampling, torch.full_like(sampling, -math.log(half)), rtol=1e-6)
    tokens, _, _ = sample_tokens(logits, uniforms, top_k=600, top_p=0.5)
    assert tokens.tolist() == [min(int(float(u) * 300), 299) for u in uniforms]
    assert sample_tokens(logits, uniforms, temperature=0.0)[0].tolist() == [0] * 6


def test_many_tokens_in_one_bin_of_the_search():
    """Logits closer than the first histogram resolves, in 32 bits, with and without repeats."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    rows, vocab = 4, 40000
    near = 1e-3 * torch.rand((rows, vocab), generator=gen, device="cuda")
    coarse = (near * 3000).round() / 3000  # a few values, each thousands of times
    uniforms = torch.rand(rows, generator=gen, device="cuda")
    for logits in (near, coarse):
        for args in (dict(top_k=9000), dict(top_p=0.3), dict(top_k=20000, top_p=0.6)):
            full = dict(temperature=1.0, top_k=None, top_p=None, min_p=None) | args
            got = sample_tokens(logits, uniforms, **full)
            n = full["top_k"] or vocab
            order = logits.sort(dim=1, descending=True, stable=True).indices
            tokens, _, sampling = got
            rank = (order == tokens[:, None]).int().argmax(dim=1)
            # weights differ by less than 1e-3, so a cut by mass is one by count within that
            most = n * (full["top_p"] or 1.0) * (1 + 2e-3) + 1
            assert bool((rank < most).all())
            assert torch.allclose(sampling, torch.full_like(sampling, -math.log(n * (full["top_p"] or 1.0))),
                                  atol=3e-3)


def test_a_cut_below_the_drawable_weights():
    """top_k reaches past the tokens that have any mass: all that do are kept, none beyond drawn."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    logits = torch.full((8, 20000), -60.0, device="cuda")
    logits -= torch.rand(logits.shape, generator=gen, device="cuda")
    logits[:, 500:900:4] = torch.randn((8, 100), generator=gen, device="cuda")
    uniforms = torch.rand(8, generator=gen, device="cuda")
    args = dict(temperature=1.0, top_k=3000, top_p=None, min_p=None)
    got = sample_tokens(logits, uniforms, **args)
    _check(logits, uniforms, got, **args)
    assert bool(((got[0] >= 500) & (got[0] < 900)).all())
    one = sample_tokens(logits, uniforms, top_k=1)[0]
    assert torch.equal(one, logits.argmax(dim=1))


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_rows(dtype):
    dt = DTYPES[dtype]
    lowest = torch.finfo(dt).min
    inf, nan = math.inf, math.nan
    rows = [
        [-inf] * 6,                       # nothing left
        [nan] * 6,
        [-inf, nan, -inf, -inf, nan, -inf],
        [-inf, -inf, 2.0, -inf, -inf, -inf],
        [lowest, lowest, 1.0, lowest, 0.5, lowest],
        [lowest] * 6,                     # all equal, however low
        [nan, 1.0, nan, 1.0, -inf, 0.0],
        [inf, 0.0, inf, 5.0, nan, -inf],  # only the infinite ones can be drawn
    ]
    logits = torch.tensor(rows, device="cuda", dtype=dt)
    for u in (0.0, 0.49, 0.51, 0.999):
        uniforms = torch.full((len(rows),), u, device="cuda")
        for args in (dict(), dict(temperature=0.0), dict(top_k=2), dict(top_p=0.8), dict(min_p=0.5)):
            full = dict(temperature=1.0, top_k=None, top_p=None, min_p=None) | args
            got = sample_tokens(logits, uniforms, **full)
            _check(logits, uniforms, got, **full)
    tokens = sample_tokens(logits, torch.full((len(rows),), 0.7, device="cuda"))[0].tolist()
    assert tokens[:4] == [-1, -1, -1, 2] and tokens[5] == 4 and tokens[7] == 2


def test_temperatures_at_the_ends_of_the_range():
    logits = torch.tensor([[1.0, 2.0, 2.0, -math.inf]] * 4, device="cuda")
    uniforms = torch.tensor([0.1, 0.6, 0.1, 0.9], device="cuda")
    temperature = torch.tensor([1e-45, 1e-45, math.inf, math.inf], device="cuda")
    tokens, _, sampling = sample_tokens(logits, uniforms, temperature=temperature)
    assert tokens.tolist() == [1, 2, 0, 2]  # the two largest; then all three alike
    assert torch.allclose(sampling.exp(), torch.tensor([0.5, 0.5, 1 / 3, 1 / 3], device="cuda"))
    tokens = sample_tokens(logits, uniforms, temperature=torch.tensor([math.nan, -1.0, 0.0, 0.0],
                                                                      device="cuda"))[0]
    assert tokens.tolist() == [1] * 4


@pytest.mark.parametrize("setting", SETTINGS)
def test_tokens_do_not_depend_on_the_batch(setting):
    """A batch gives a row fewer CTAs than a row by itself: the masses are whole, the token the same."""
    logits, uniforms = _logits(300, 20011, torch.bfloat16, 12)
    together = sample_tokens(logits, uniforms, **SETTINGS[setting])
    for i in range(0, 300, 37):
        alone = sample_tokens(logits[i:i + 1], uniforms[i:i + 1], **SETTINGS[setting])
        assert torch.equal(alone[0], together[0][i:i + 1])
        for a, b in zip(alone[1:], together[1:]):
            assert torch.allclose(a, b[i:i + 1], rtol=0, atol=2.0 ** -20)  # sums in another order


def test_distribution_of_many_draws():
    """Evenly spaced uniform numbers reproduce the kept probabilities to one draw in n."""
    n = 4096
    row = torch.tensor([2.0, 0.0, 1.0, -math.inf, 1.5, -1.0, 0.5], device="cuda")
    uniforms = (torch.arange(n, device="cuda") + 0.5) / n
    tokens = sample_tokens(row.repeat(n, 1), uniforms, temperature=0.9, top_k=5)[0]
    p = torch.softmax(torch.where(row >= 0, row, -math.inf) / 0.9, 0)
    counts = torch.bincount(tokens, minlength=7).float() / n
    assert bool(((counts - p).abs() <= 1.5 / n).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("setting", ["plain", "greedy", "top_p", "all"])
def test_the_largest_vocabulary(dtype, setting):
    logits, uniforms = _logits(2, 376832, DTYPES[dtype], 31)
    args = dict(temperature=1.0, top_k=None, top_p=None, min_p=None) | SETTINGS[setting]
    _check(logits, uniforms, sample_tokens(logits, uniforms, **args), **args)


def test_no_rows_and_refusals():
    logits = torch.randn((0, 11), device="cuda")
    assert [v.shape for v in sample_tokens(logits, torch.empty(0, device="cuda"))] == [(0,)] * 3
    logits, u = torch.randn((3, 11), device="cuda"), torch.rand(3, device="cuda")
    with pytest.raises(ValueError, match="B, V"):
        sample_tokens(logits[0], u)
    with pytest.raises(ValueError, match="float16"):
        sample_tokens(logits.double(), u)
    with pytest.raises(ValueError, match="uniforms"):
        sample_tokens(logits, u.double())
    with pytest.raises(ValueError, match="uniforms"):
        sample_tokens(logits, u[:2])
    with pytest.raises(ValueError, match="CUDA"):
        sample_tokens(logits.cpu(), u)
    for bad in (dict(temperature=-1.0), dict(temperature=math.nan), dict(top_k=-1), dict(top_p=0.0),
                dict(top_p=1.5), dict(min_p=-0.1), dict(min_p=2.0)):
        with pytest.raises(ValueError, match="out of range"):
            sample_tokens(logits, u, **bad)
    with pytest.raises(ValueError, match="top_k must hold"):
        sample_tokens(logits, u, top_k=torch.ones(3, device="cuda"))
    with pytest.raises(ValueError, match="min_p must hold"):
        sample_tokens(logits, u, min_p=torch.ones(2, device="cuda"))
    with pytest.raises(ValueError, match="limited"):
        sample_tokens(torch.zeros((1, 400000), device="cuda", dtype=torch.float16), u[:1])
