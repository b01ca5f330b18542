"""Config-5 end-to-end decoder benchmark: Llama-3-8B shape on 1..8 B200s.

``python -m inferkernellab_b200.e2e_bench`` (one GPU) or
``torchrun --nproc-per-node N -m inferkernellab_b200.e2e_bench`` (N GPUs).

Workload: a random-init Llama-3-8B-shaped decoder --
32 layers, hidden 4096, 32 query / 8 KV heads, head_dim 128, intermediate
14336, vocab 128256, RMSNorm, RoPE theta 5e5, bf16 weights ~ N(0, 0.02) --
serving 256 requests whose prompt token ids and lengths (uniform in
[64, 1024]) are drawn from a seeded generator: batched prefill under a
2048-token budget, then 128 greedy decode steps.

Parallelism: the requests are partitioned contiguously over the ranks (one
process per GPU, each with its own weights replica and block pool); every
decode step all-gathers the sampled token ids over NCCL -- the only collective.
``value`` = tokens generated by all ranks in the steady-state decode steps /
the max over ranks of their time (the first decode step, which also captures
the CUDA graph, is reported separately).  ``--scaling strong`` keeps the 256
requests fixed as GPUs are added; ``--scaling weak`` gives every GPU 256.  The weights
are initialised on the GPU (same N(0, 0.02) scheme as the reference's
``_load_model``, GPU random stream), which is the practical way to build an
8B model; correctness at this scale is covered by the small-model parity tests.
"""

from __future__ import annotations

import argparse
import datetime
import json
import os
import sys
import time

import torch

from .llama import (LlamaPagedDecodeRunner, allgather_token_exchange, load_random_llama,
                    partition_requests)


def make_prompts(num_requests: int, min_len: int, max_len: int, vocab: int, seed: int):
    gen = torch.Generator().manual_seed(seed)
    lens = torch.randint(min_len, max_len + 1, (num_requests,), generator=gen).tolist()
    return [torch.randint(0, vocab, (n,), generator=gen).tolist() for n in lens]


class _StepTrace:
    """Wraps the runner's decode hook: a torch.profiler (CUPTI) device trace over
    decode steps [a, b), summarised as device microseconds per step per kernel."""

    def __init__(self, runner, spec: str):
        a, b = (int(x) for x in spec.split(":"))
        if not 0 <= a < b:
            raise ValueError("--trace-steps wants A:B with 0 <= A < B")
        self.first, self.stop, self.step, self.prof = a, b, 0, None
        self._decode = runner.runtime.decode_fn
        runner.runtime.decode_fn = self._hook

    def _hook(self, requests):
        from torch.profiler import ProfilerActivity, profile

        if self.step == self.first:
            torch.cuda.synchronize()
            self.prof = profile(activities=[ProfilerActivity.CUDA])
            self.prof.__enter__()
        self._decode(requests)
        self.step += 1
        if self.step == self.stop and self.prof is not None:
            torch.cuda.synchronize()
            self.prof.__exit__(None, None, None)

    def summary(self) -> dict:
        if self.prof is None or self.step < self.stop:
            return {"trace": "decode steps not reached"}
        steps = self.stop - self.first
        per: dict[str, list] = {}
        for ev in self.prof.events():
            if ev.device_type != torch.autograd.DeviceType.CUDA:
                continue
            entry = per.setdefault(ev.name, [0, 0.0])
            entry[0] += 1
            entry[1] += ev.device_time_total
        total = sum(v[1] for v in per.values())
        rows = sorted(per.items(), key=lambda kv: -kv[1][1])
        return {"trace": f"decode steps {self.first}..{self.stop - 1}, device time per step",
                "device_us_per_step": round(total / steps, 1),
                "kernels": [{"name": name[:160], "launches_per_step": n // steps,
                             "us_per_step": round(t / steps, 1),
                             "share": round(t / total, 4)} for name, (n, t) in rows[:24]]}


def main(argv=None) -> int:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--requests", type=int, default=256)
    p.add_argument("--min-prompt", type=int, default=64)
    p.add_argument("--max-prompt", type=int, default=1024)
    p.add_argument("--max-new-tokens", type=int, default=128)
    p.add_argument("--layers", type=int, default=32)
    p.add_argument("--hidden", type=int, default=4096)
    p.add_argument("--heads", type=int, default=32)
    p.add_argument("--kv-heads", type=int, default=8)
    p.add_argument("--intermediate", type=int, default=14336)
    p.add_argument("--vocab", type=int, default=128256)
    p.add_argument("--rope-theta", type=float, default=5e5)
    p.add_argument("--block-size", type=int, default=16)
    p.add_argument("--max-num-batched-tokens", type=int, default=2048)
    p.add_argument("--seed", type=int, default=0)
    p.add_argument("--no-cuda-graph", action="store_true",
                   help="launch the decode step eagerly instead of replaying one CUDA graph")
    p.add_argument("--scaling", choices=("strong", "weak"), default="strong",
                   help="strong: --requests in total; weak: --requests per GPU")
    p.add_argument("--shared-prefix", type=int, default=0, metavar="L",
                   help="prepend the same L seeded tokens (a common system prompt) to every prompt")
    p.add_argument("--prefix-caching", action="store_true",
                   help="share the KV blocks of common prompt prefixes (PrefixCache)")
    p.add_argument("--sync-steps", action="store_true",
                   help="synchronise after every decode step (the reference runner's per-step "
                        "wall clock); default: the host prepares step N+1 while step N runs")
    p.add_argument("--unfused-decode", action="store_true",
                   help="rotary append and attention as two launches per layer (A/B check)")
    p.add_argument("--projections", choices=("model", "fp8"), default="model",
                   help="fp8: 8-bit weights and activations with block scales (added to the "
                        "model's 16-bit weights; faster for few requests and prefill, slower "
                        "for large decode batches)")
    p.add_argument("--qk-norm", action="store_true",
                   help="a norm on every query and key head of every layer")
    p.add_argument("--sampler", choices=("torch", "device"), default="torch",
                   help="device: one sampling launch per step for the whole batch")
    p.add_argument("--temperature", type=float, default=0.0)
    p.add_argument("--top-k", type=int, default=0)
    p.add_argument("--top-p", type=float, default=1.0)
    p.add_argument("--min-p", type=float, default=0.0)
    p.add_argument("--samples-per-prompt", type=int, default=1, metavar="N",
                   help="prefill every prompt once and fork it into N requests")
    p.add_argument("--trace-steps", default=None, metavar="A:B",
                   help="record a CUPTI kernel trace of decode steps A..B-1 (rank 0) and "
                        "print the per-kernel device time per step as a second JSON line")
    args = p.parse_args(argv)

    world = int(os.environ.get("WORLD_SIZE", "1"))
    rank = int(os.environ.get("RANK", "0"))
    local = int(os.environ.get("LOCAL_RANK", "0"))
    device = torch.device("cuda", local)
    torch.cuda.set_device(device)
    if world > 1:
        torch.distributed.init_process_group("nccl", timeout=datetime.timedelta(seconds=300),
                                             device_id=device)
    try:
        total_requests = args.requests * (world if args.scaling == "weak" else 1)
        prompts = make_prompts(total_requests, args.min_prompt, args.max_prompt, args.vocab,
                               args.seed)
        if args.shared_prefix > 0:
            head = make_prompts(1, args.shared_prefix, args.shared_prefix, args.vocab,
                                args.seed + 1)[0]
            prompts = [head + p for p in prompts]
        per = -(-len(prompts) // world)
        part = partition_requests(len(prompts), world, rank)
        mine = prompts[part.start:part.stop]
        t0 = time.perf_counter()
        model = load_random_llama(vocab_size=args.vocab, hidden_size=args.hidden,
                                  intermediate_size=args.intermediate, num_layers=args.layers,
                                  num_attention_heads=args.heads, num_kv_heads=args.kv_heads,
                                  max_position_embeddings=(args.max_prompt + args.shared_prefix
                                                           + args.max_new_tokens),
                                  rope_theta=args.rope_theta, seed=args.seed, device=device,
                                  dtype=torch.bfloat16, init_on_device=True,
                                  qk_norm=args.qk_norm)
        init_s = time.perf_counter() - t0
        exchange = (allgather_token_exchange(max_local=per * args.samples_per_prompt)
                    if world > 1 else None)
        runner = LlamaPagedDecodeRunner(model, mine, max_new_tokens=args.max_new_tokens,
                                        block_size=args.block_size,
                                        max_num_batched_tokens=args.max_num_batched_tokens,
                                        token_exchange=exchange, collect_logits=False,
                                        cuda_graph=not args.no_cuda_graph,
                                        prefix_caching=args.prefix_caching,
                                        sync_steps=args.sync_steps,
                                        fused_decode=False if args.unfused_decode else "auto",
                                        projections=args.projections, sampler=args.sampler,
                                        temperature=args.temperature, top_k=args.top_k,
                                        top_p=args.top_p, min_p=args.min_p,
                                        samples_per_prompt=args.samples_per_prompt)
        trace = _StepTrace(runner, args.trace_steps) if (args.trace_steps and rank == 0) else None
        if world > 1:
            torch.distributed.barrier()
        torch.cuda.synchronize()
        result = runner.run()
        steps = result.decode_step_wall_ms
        # The first decode step also captures the CUDA graph (a one-time set-up);
        # the steady-state rate is taken over the remaining steps.
        steady = steps[1:] if len(steps) > 1 else steps
        decode_ms = sum(steady)
        requests = len(mine) * args.samples_per_prompt
        tokens_steady = float(requests * len(steady))
        stats = torch.tensor([decode_ms, result.prefill_wall_ms, result.decode_p50_ms,
                              tokens_steady, float(steps[0]), sum(steps),
                              float(result.prefix_cached_tokens)],
                             dtype=torch.float64, device=device)
        if world > 1:
            gathered = [torch.empty_like(stats) for _ in range(world)]
            torch.distributed.all_gather(gathered, stats)
        else:
            gathered = [stats]
        if rank == 0:
            g = torch.stack(gathered).cpu()
            decode_max = float(g[:, 0].max())
            tokens = float(g[:, 3].sum())
            all_tokens = float(len(prompts) * args.samples_per_prompt * args.max_new_tokens)
            record = {
                "metric": f"decode tok/s (config5 Llama-3-8B-shaped, {len(prompts)} requests)",
                "value": round(tokens / (decode_max / 1e3), 1),
                "unit": "tok/s", "n_gpus": world, "scaling": args.scaling,
                "steady_decode_ms_max_over_ranks": round(decode_max, 2),
                "tpot_p50_ms_max_over_ranks": round(float(g[:, 2].max()), 3),
                "first_step_ms_incl_graph_capture": round(float(g[:, 4].max()), 2),
                "all_steps_tok_s": round(all_tokens / (float(g[:, 5].max()) / 1e3), 1),
                "prefill_ms_max_over_ranks": round(float(g[:, 1].max()), 2),
                "prefix_cached_tokens": int(g[:, 6].sum()),
                "generated_tokens": int(all_tokens),
                "requests_per_rank": per, "prompt_tokens_total": sum(len(x) for x in prompts),
                "model_init_s": round(init_s, 2),
                "peak_memory_gb_rank0": round(result.peak_memory_allocated_bytes / 1e9, 2),
                "peak_kv_gb_rank0": round(result.peak_kv_memory_bytes / 1e9, 2),
                "config": {"layers": args.layers, "hidden": args.hidden, "heads": args.heads,
                           "kv_heads": args.kv_heads, "intermediate": args.intermediate,
                           "vocab": args.vocab, "rope_theta": args.rope_theta,
                           "block_size": args.block_size, "budget": args.max_num_batched_tokens,
                           "prompt_len": [args.min_prompt, args.max_prompt],
                           "shared_prefix": args.shared_prefix,
                           "prefix_caching": args.prefix_caching,
                           "max_new_tokens": args.max_new_tokens, "seed": args.seed,
                           "dtype": "bf16", "backend": "b200_paged",
                           "decode_step": "eager" if args.no_cuda_graph else "cuda_graph",
                           "sync_each_step": args.sync_steps,
                           "fused_decode": "off" if args.unfused_decode else "auto"},
            }
            chosen = {"projections": args.projections, "qk_norm": args.qk_norm,
                      "sampler": args.sampler, "temperature": args.temperature,
                      "top_k": args.top_k, "top_p": args.top_p, "min_p": args.min_p,
                      "samples_per_prompt": args.samples_per_prompt}
            record["config"] |= {k: v for k, v in chosen.items() if v != p.get_default(k)}
            print(json.dumps(record), flush=True)
            if trace is not None:
                print(json.dumps(trace.summary()), flush=True)
    finally:
        if world > 1:
            torch.distributed.destroy_process_group()
    return 0


if __name__ == "__main__":
    sys.exit(main())
