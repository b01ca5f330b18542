"""The runner's device sampler where a request fails or ends before the others."""

import math

import pytest
import torch

from inferkernellab_b200 import check_device_errors, llama, sample_tokens
from inferkernellab_b200.llama import LlamaPagedDecodeRunner, load_random_llama

pytestmark = pytest.mark.gpu

PROMPTS = ((1, 2, 3, 4, 5, 9, 11, 3, 2), (6, 7, 8), tuple(range(20, 60)))


def _runner(**kw):
    model = load_random_llama(vocab_size=128, hidden_size=64, intermediate_size=128, num_layers=2,
                              num_attention_heads=4, num_kv_heads=2, max_position_embeddings=256,
                              rope_theta=10_000.0, seed=2026, device="cuda", dtype=torch.bfloat16)
    return LlamaPagedDecodeRunner(model, PROMPTS, **(dict(max_new_tokens=5, block_size=4,
                                                          sampler="device") | kw))


def _without_logits(runner, request_id, step, value):
    """The logits of one request at one step become ``value`` throughout."""
    plain, calls = runner._logits_for, []

    def replaced(requests):
        logits = plain(requests)
        if len(calls) == step:
            logits = logits.clone()
            logits[[r.request_id for r in requests].index(request_id)] = value
        calls.append(1)
        return logits

    runner._logits_for = replaced


@pytest.mark.parametrize("cuda_graph", [False, True])
@pytest.mark.parametrize("step,value", [(0, math.nan), (2, math.nan), (4, -math.inf)])
def test_a_request_with_nothing_to_draw_ends_alone(cuda_graph, step, value):
    whole = _runner(cuda_graph=cuda_graph).run()
    runner = _runner(cuda_graph=cuda_graph)
    _without_logits(runner, 1, step, value)
    got = runner.run()
    assert got.finish_reasons == ("length", "error", "length") and got.cache_released
    assert got.generated_tokens[1] == whole.generated_tokens[1][:step]
    for i in (0, 2):
        assert len(got.generated_tokens[i]) == 5
        # greedy: the others' tokens, up to a tie that a smaller batch's products may break
        assert got.generated_tokens[i][:step + 1] == whole.generated_tokens[i][:step + 1]
    for tokens, a, b in zip(got.generated_tokens, got.token_logprobs, got.sampling_logprobs):
        assert len(tokens) == len(a) == len(b) and all(map(math.isfinite, a + b))
    assert check_device_errors() == 0


def test_no_request_has_anything_to_draw():
    runner = _runner()
    for rid in range(3):
        _without_logits(runner, rid, 0, math.nan)
    got = runner.run()
    assert got.generated_tokens == ((), (), ()) and got.finish_reasons == ("error",) * 3
    assert got.cache_released


def _draws(runner, monkeypatch):
    """Uniform numbers by request, in the order of its steps, of a run."""
    drawn = {}
    plain_logits, ids = runner._logits_for, []

    def logits_for(requests):
        ids[:] = [r.request_id for r in requests]
        return plain_logits(requests)

    def sample(logits, uniforms, **kw):
        for rid, u in zip(ids, uniforms.tolist()):
            drawn.setdefault(rid, []).append(u)
        return sample_tokens(logits, uniforms, **kw)

    runner._logits_for = logits_for
    with monkeypatch.context() as patch:
        patch.setattr(llama, "sample_tokens", sample)
        result = runner.run()
    return drawn, result


def test_a_request_draws_the_same_numbers_when_another_ends(monkeypatch):
    kw = dict(temperature=1.0, seed=11, max_new_tokens=8, samples_per_prompt=2)
    whole, result = _draws(_runner(**kw), monkeypatch)
    assert {rid: len(v) for rid, v in whole.items()} == {rid: 8 for rid in range(6)}
    # an end token that one request alone draws first, not at its last step
    firsts = [tokens[:4] for tokens in result.generated_tokens]
    eos = next(t for tokens in firsts for t in tokens if sum(t in other for other in firsts) == 1)
    runner = _runner(**kw, eos_token_ids=[eos])
    some, ended = _draws(runner, monkeypatch)
    assert min(len(t) for t in ended.generated_tokens) < 8  # somebody has left early
    for rid, numbers in some.items():
        assert numbers == whole[rid][:len(numbers)], rid
    assert any(len(v) == 8 for v in some.values())
