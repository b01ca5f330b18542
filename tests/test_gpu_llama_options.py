"""The runner's sampled, branching, 8-bit and per-head-norm paths."""

import math

import pytest
import torch

from inferkernellab_b200 import PagedKVCache, check_device_errors
from inferkernellab_b200.llama import LlamaPagedDecodeRunner, correctness, load_random_llama

pytestmark = pytest.mark.gpu

PROMPTS = ((1, 2, 3, 4, 5, 9, 11, 3, 2), (6, 7, 8), tuple(range(20, 60)))  # 40: whole pages of 4


def _model(dtype=torch.bfloat16, hidden=64, heads=4, kv_heads=2, layers=2, qk_norm=False):
    return load_random_llama(vocab_size=128, hidden_size=hidden, intermediate_size=2 * hidden,
                             num_layers=layers, num_attention_heads=heads, num_kv_heads=kv_heads,
                             max_position_embeddings=256, rope_theta=10_000.0, seed=2026,
                             device="cuda", dtype=dtype, qk_norm=qk_norm)


def _run(model, prompts=PROMPTS, **kw):
    return LlamaPagedDecodeRunner(model, prompts, **(dict(max_new_tokens=5, block_size=4) | kw)).run()


def _assert_logits(report):
    assert report["logits_max_error"] <= report["logits_tolerance"], report


def test_fork_copies_the_partial_page_in_every_layer():
    cache = PagedKVCache(20, 16, 2, 64, num_layers=3, dtype=torch.bfloat16, device="cuda")
    cache.k.normal_()
    cache.v.normal_()
    k, v = cache.k.clone(), cache.v.clone()
    table = cache.allocate_request(0, 41)
    forks = cache.fork_request(table, 41, [1, 2])
    for fork in forks:
        assert fork[:2] == table[:2] and fork[2] not in table
        for got, want in ((cache.k, k), (cache.v, v)):
            assert torch.equal(got[:, fork[2], :9], want[:, table[2], :9])
            assert torch.equal(got[:, fork[2], 9:], want[:, fork[2], 9:])
    assert forks[0][2] != forks[1][2]
    assert check_device_errors() == 0


def test_device_sampler_is_the_torch_one_where_nothing_is_random():
    model = _model()
    torch_run, device_run = _run(model), _run(model, sampler="device")
    assert device_run.generated_tokens == torch_run.generated_tokens
    scored = _run(model, eos_token_ids=[127])  # the torch path that records log-probabilities
    if scored.generated_tokens == device_run.generated_tokens:
        for a, b in ((scored.token_logprobs, device_run.token_logprobs),
                     (scored.sampling_logprobs, device_run.sampling_logprobs)):
            assert torch.allclose(torch.tensor(a), torch.tensor(b), atol=1e-4)


@pytest.mark.parametrize("cuda_graph", [False, True])
def test_samples_of_a_prompt_share_its_prefill(cuda_graph):
    model = _model()
    kw = dict(sampler="device", temperature=1.0, top_k=40, top_p=0.95, min_p=0.001, seed=7,
              samples_per_prompt=4, cuda_graph=cuda_graph, max_new_tokens=6)
    result = _run(model, **kw)
    assert len(result.generated_tokens) == 12
    assert result.prefill_tokens == 4 * sum(map(len, PROMPTS)) and result.cache_released
    # every sample's logits are those of its own tokens
    prompts = [p for p in PROMPTS for _ in range(4)]
    _assert_logits(correctness(model, prompts, result))
    for i in range(3):
        assert len(set(result.generated_tokens[4 * i:4 * i + 4])) > 1  # they went apart
    assert all(len(lp) == 6 and all(x <= 0 for x in lp) for lp in result.token_logprobs)
    assert all(a <= b + 1e-5 for x, y in zip(result.token_logprobs, result.sampling_logprobs)
               for a, b in zip(x, y))  # the cut only raises what is left
    again = _run(model, **kw)
    assert again.generated_tokens == result.generated_tokens
    # pages: a prompt's full pages once, not four times
    alone = _run(model, [p for p in PROMPTS for _ in range(4)], **(kw | dict(samples_per_prompt=1)))
    assert result.used_blocks_peak < alone.used_blocks_peak


def test_greedy_samples_are_all_the_same():
    model = _model()
    base = _run(model)
    many = _run(model, samples_per_prompt=3, prefix_caching=True)
    assert many.generated_tokens == tuple(t for t in base.generated_tokens for _ in range(3))


def _plain_forward(model, tokens):
    """Logits of the last token: the decoder with its head norms, 32-bit arithmetic."""
    inner, cfg = model.model, model.config
    heads, kv = cfg.num_attention_heads, cfg.num_key_value_heads
    dim = cfg.hidden_size // heads
    n = len(tokens)
    x = inner.embed_tokens(torch.tensor(tokens, device="cuda")).float()

    def norm(t, m):
        return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + m.variance_epsilon) * m.weight.float()

    def linear(t, m):
        return t @ m.weight.float().t()

    cos, sin = (t[0].float() for t in inner.rotary_emb(x[None], torch.arange(n, device="cuda")[None]))

    def turn(t):
        half = torch.cat((-t[..., dim // 2:], t[..., :dim // 2]), -1)
        return t * cos[:, None] + half * sin[:, None]

    mask = torch.full((n, n), -math.inf, device="cuda").triu(1)
    for layer in inner.layers:
        a, y = layer.self_attn, norm(x, layer.input_layernorm)
        q = turn(norm(linear(y, a.q_proj).view(n, heads, dim), a.q_norm))
        k = turn(norm(linear(y, a.k_proj).view(n, kv, dim), a.k_norm)).repeat_interleave(heads // kv, 1)
        v = linear(y, a.v_proj).view(n, kv, dim).repeat_interleave(heads // kv, 1)
        p = torch.softmax(torch.einsum("qhd,khd->hqk", q, k) * dim ** -0.5 + mask, -1)
        x = x + linear(torch.einsum("hqk,khd->qhd", p, v).reshape(n, -1), a.o_proj)
        y = norm(x, layer.post_attention_layernorm)
        x = x + linear(torch.nn.functional.silu(linear(y, layer.mlp.gate_proj)) * linear(y, layer.mlp.up_proj),
                       layer.mlp.down_proj)
    return linear(norm(x[-1], inner.norm), model.lm_head)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("cuda_graph", [False, True])
def test_norms_of_queries_and_keys(dtype, cuda_graph):
    model = _model(dtype, qk_norm=True)
    result = _run(model, cuda_graph=cuda_graph)
    tol = 3e-2 if dtype == torch.bfloat16 else 5e-3  # as against the eager model
    with torch.inference_mode():
        for i, (prompt, tokens) in enumerate(zip(PROMPTS, result.generated_tokens)):
            for step in range(len(tokens)):
                want = _plain_forward(model, list(prompt) + list(tokens[:step]))
                got = result.decode_logits[step][i].cuda()
                assert float((got - want).abs().max()) <= tol
    assert check_device_errors() == 0


def test_8_bit_projections_follow_the_model():
    """Seven products a layer whose inputs and weights are rounded to 3 bits after the leading one:
    2**-4 / sqrt(3) of noise for each of the two, so about 5 % a product and, over two layers of
    residual sums, 5 % * sqrt(7 * 2) = 19 % at most of the logits."""
    model = _model(hidden=256, heads=4, kv_heads=2)
    full, small = _run(model, max_new_tokens=1), _run(model, max_new_tokens=1, projections="fp8")
    error = (small.prompt_logits - full.prompt_logits).norm() / full.prompt_logits.norm()
    assert 0 < float(error) < 0.19
    eager, graph = (_run(model, projections="fp8", cuda_graph=g) for g in (False, True))
    assert eager.generated_tokens == graph.generated_tokens
    assert check_device_errors() == 0


def test_all_of_them_together():
    model = _model(hidden=256, heads=2, kv_heads=1, qk_norm=True)
    kw = dict(projections="fp8", sampler="device", temperature=0.8, top_p=0.9, samples_per_prompt=3,
              max_new_tokens=8, block_size=16)
    a, b = _run(model, cuda_graph=True, **kw), _run(model, cuda_graph=False, **kw)
    assert a.generated_tokens == b.generated_tokens and a.cache_released
    assert check_device_errors() == 0


def test_options_are_checked():
    model = _model()
    for bad in (dict(sampler="host"), dict(projections="int4"), dict(samples_per_prompt=0),
                dict(top_k=3), dict(min_p=0.1), dict(sampler="device", top_k=-1),
                dict(sampler="device", min_p=2.0)):
        with pytest.raises(ValueError):
            LlamaPagedDecodeRunner(model, PROMPTS, max_new_tokens=1, **bad)
