"""The operators of a sampled, branching decode step, as cases that can be timed and compared.

Every case names one operator of the package and one workload.  ``run`` computes it either in
plain form (elementary torch operations, 32-bit arithmetic, rounded once at the end) or, with
``own`` set, through the package's public entry points.  ``exact`` gives the same outputs from
the definition in 64 bits.

==============  =================================================================================
operator        what it is in a serving step
==============  =================================================================================
``sample``      next tokens of a batch from its logits: temperature, min-p, top-k, top-p, and one
                given uniform number per request
``pages``       physical KV pages copied to other pages in every layer (a request that forks, a
                pool that is compacted), and block tables rewritten to the new ids
``qk_norm``     RMS norm of every query and key head, rotary embedding and KV append in one pass
``quantize``    16-bit activations to 8-bit floating point with a scale per row and 128 columns
``linear``      the projection of 16-bit activations with an 8-bit weight that has a scale per
                128 x 128 block
==============  =================================================================================
"""

import math
import types

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E4M3_MAX = 448.0
FLUSH = 2.0 ** -100  # a block whose largest magnitude is below this counts as zero


# ------------------------------------------------------------------------------------- cases

def listed():
    return [
        # One interactive request: the latency of a single row of the 128256-token vocabulary.
        dict(name="sample one request", op="sample", rows=1, vocab=128256, dtype="bf16", mode="top_p"),
        # A continuous batch whose requests each bring their own sampling settings.
        dict(name="sample mixed batch", op="sample", rows=64, vocab=128256, dtype="bf16", mode="mixed"),
        # The largest decode batch with 32-bit logits; an odd vocabulary leaves its rows unaligned.
        dict(name="sample wide odd", op="sample", rows=256, vocab=128257, dtype="f32", mode="top_k"),
        # One request forks in a small model: its last, partly filled page is copied.
        dict(name="fork one page", op="pages", pages=1, layers=4, pool=64, block=16, kv_heads=8, dim=128,
             dtype="bf16", part=True, tables=1, width=64),
        # A fragmented pool is compacted: half of its pages move, every block table is rewritten.
        dict(name="compact pool", op="pages", pages=900, layers=16, pool=2048, block=16, kv_heads=8, dim=128,
             dtype="bf16", part=False, tables=256, width=512),
        # One decode step of one request.
        dict(name="qk_norm one token", op="qk_norm", tokens=1, heads=32, kv_heads=8, dim=128, rotary=128,
             block=16, dtype="bf16"),
        # A prefill batch of several requests, an odd number of tokens.
        dict(name="qk_norm prefill", op="qk_norm", tokens=8191, heads=32, kv_heads=8, dim=128, rotary=128,
             block=16, dtype="bf16"),
        # The hidden states of a decode batch ahead of a projection.
        dict(name="quantize decode", op="quantize", rows=64, cols=4096, dtype="bf16"),
        # The MLP's intermediate activations of a prefill batch.
        dict(name="quantize prefill", op="quantize", rows=8191, cols=14336, dtype="bf16"),
        # The fused q|k|v projection of one request.
        dict(name="linear one token", op="linear", rows=1, cols=4096, outs=6144, dtype="bf16"),
        # The gate|up projection of a decode batch: bound by the weight's bytes.
        dict(name="linear decode batch", op="linear", rows=64, cols=4096, outs=28672, dtype="bf16"),
        # The gate|up projection of a prefill batch: bound by the tensor cores.
        dict(name="linear prefill", op="linear", rows=4099, cols=4096, outs=28672, dtype="bf16"),
    ]


def _between(rng, low, high):
    """A whole number in [low, high], even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["sample", "sample", "pages", "qk_norm", "qk_norm", "quantize", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "sample":
        return dict(op=op, rows=_between(rng, 1, 256), vocab=_between(rng, 250, 128256),
                    dtype=rng.choice(["bf16", "f16", "f32"]),
                    mode=rng.choice(["plain", "greedy", "top_k", "top_p", "min_p", "mixed"]))
    if op == "pages":
        return dict(op=op, pages=_between(rng, 1, 500), layers=rng.randint(1, 8), pool=rng.randint(1100, 1500),
                    block=rng.choice([8, 16, 32]), kv_heads=rng.choice([1, 2, 4, 8]),
                    dim=rng.choice([64, 128]), dtype=dtype, part=rng.random() < 0.5,
                    tables=_between(rng, 1, 256), width=rng.randint(1, 300))
    if op == "qk_norm":
        kv_heads = rng.choice([1, 2, 4, 8])
        dim = rng.choice([64, 128])
        return dict(op=op, tokens=_between(rng, 1, 8000), heads=kv_heads * rng.choice([1, 2, 4]),
                    kv_heads=kv_heads, dim=dim, rotary=rng.choice([dim, dim, dim // 2]), block=16, dtype=dtype)
    cols = rng.choice([1024, 2048, 4096, 14336, 16 * (2 * _between(rng, 4, 200) + 1)])
    if op == "quantize":
        return dict(op=op, rows=_between(rng, 1, 8000), cols=cols, dtype=dtype)
    outs = rng.choice([2 * _between(rng, 50, 3000) + 1, 1024, 4096, 6144])
    return dict(op=op, rows=_between(rng, 1, 4000), cols=cols, outs=outs, dtype=dtype)


def work(case):
    op = case["op"]
    if op == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "f32" else 2) + case["rows"] * 32, "flops": 4 * n}
    if op == "pages":
        page = case["block"] * case["kv_heads"] * case["dim"] * 2
        copied = 2 * case["pages"] * case["layers"] * page * (0.5 if case["part"] else 1.0)
        return {"bytes": 2 * copied + 2 * 4 * case["tables"] * case["width"], "flops": 0}
    if op == "qk_norm":
        row = (case["heads"] + 2 * case["kv_heads"]) * case["dim"] * 2
        return {"bytes": case["tokens"] * (2 * row + 2 * case["rotary"] * 2 + 8),
                "flops": case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"] * 7}
    if op == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": 3 * n + case["rows"] * -(-case["cols"] // 128) * 4, "flops": 3 * n}
    m, k, n = case["rows"], case["cols"], case["outs"]
    return {"bytes": 2 * m * k + n * k + 2 * m * n + 4 * (-(-k // 128)) * (-(-n // 128)), "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------ inputs

def _settings(mode, rows, device):
    """Per-request temperature, top_k, top_p, min_p of a sampling mode."""
    i = torch.arange(rows, device=device)
    temperature = 0.6 + 0.1 * (i % 7).float()
    top_k = torch.zeros(rows, dtype=torch.int32, device=device)
    top_p = torch.ones(rows, device=device)
    min_p = torch.zeros(rows, device=device)
    if mode == "greedy":
        temperature = torch.zeros_like(temperature)
    elif mode == "top_k":
        top_k = (20 + 15 * (i % 5)).int()
    elif mode == "top_p":
        top_p = 0.9 + 0.02 * (i % 5).float()
    elif mode == "min_p":
        min_p = 0.02 + 0.02 * (i % 4).float()
    elif mode == "mixed":
        kind = i % 5
        temperature = torch.where(kind == 0, torch.zeros_like(temperature), temperature)
        top_k = torch.where((kind == 2) | (kind == 4), 50, 0).int()
        top_p = torch.where((kind == 1) | (kind == 2), 0.95, 1.0)
        min_p = torch.where((kind == 3) | (kind == 4), 0.05, 0.0)
    return temperature, top_k, top_p, min_p


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = dict(case=case)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device)

    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        logits = 2.2 * normal(rows, vocab)
        # Some likely continuations above the bulk, and ids that the tokenizer never emits.
        likely = torch.randint(0, vocab, (rows, 200), generator=gen, device=device)
        logits.scatter_add_(1, likely, 10 * torch.rand((rows, 200), generator=gen, device=device))
        logits[:, vocab - vocab // 200:] = float("-inf")
        s["logits"] = logits.to(dtype)
        s["uniforms"] = torch.rand(rows, generator=gen, device=device)
        s["temperature"], s["top_k"], s["top_p"], s["min_p"] = _settings(case["mode"], rows, device)
    elif case["op"] == "pages":
        s["cache"] = _Cache(case["pool"], case["block"], case["kv_heads"], case["dim"], case["layers"], dtype, device)
        s["cache"].k.normal_(generator=gen)
        s["cache"].v.normal_(generator=gen)
        order = torch.randperm(case["pool"], generator=gen, device=device).int()
        n = case["pages"]
        s["src"], s["dst"] = order[:n].clone(), order[n:2 * n].clone()
        s["tokens"] = None
        if case["part"]:
            s["tokens"] = torch.randint(1, case["block"] + 1, (n,), generator=gen, device=device, dtype=torch.int32)
        # What the allocator's plan says: the new id of every page, its own where it stays.
        s["page_map"] = torch.arange(case["pool"], dtype=torch.int32, device=device)
        s["page_map"][s["src"].long()] = s["dst"]
        live = order[torch.cat([torch.arange(n, device=device), torch.arange(2 * n, case["pool"], device=device)])]
        at = torch.randint(0, live.numel(), (case["tables"], case["width"]), generator=gen, device=device)
        s["tables"] = live[at]
    elif case["op"] == "qk_norm":
        t, hq, hkv, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        # Views of one fused projection's output, as the model has them.
        qkv = (2 * normal(t, (hq + 2 * hkv) * d)).to(dtype)
        s["q"] = qkv[:, :hq * d].view(t, hq, d)
        s["k"] = qkv[:, hq * d:(hq + hkv) * d].view(t, hkv, d)
        s["v"] = qkv[:, (hq + hkv) * d:].view(t, hkv, d)
        s["q_weight"], s["k_weight"] = ((1 + 0.1 * normal(d)).to(dtype) for _ in range(2))
        rd = case["rotary"]
        position = torch.randint(0, 8192, (t, 1), generator=gen, device=device).float()
        angle = position * 5e5 ** (-torch.arange(0, rd, 2, device=device).float() / rd)
        angle = torch.cat([angle, angle], dim=1)
        s["cos"], s["sin"] = angle.cos().to(dtype), angle.sin().to(dtype)
        pool = -(-t // case["block"]) + 4
        s["cache"] = _Cache(pool, case["block"], hkv, d, 1, dtype, device)
        s["cache"].k.zero_()
        s["cache"].v.zero_()
        s["slots"] = torch.randperm(pool * case["block"], generator=gen, device=device)[:t].int()
    else:
        x = normal(case["rows"], case["cols"])
        x = x * (1 + 20 * (torch.rand(case["cols"], generator=gen, device=device) < 0.002).float())  # outlier channels
        s["x"] = x.to(dtype)
        if case["op"] == "linear":
            n, k = case["outs"], case["cols"]
            w = 0.02 * normal(n, k)
            nb, kb = -(-n // 128), -(-k // 128)
            padded = torch.zeros(nb * 128, kb * 128, device=device)
            padded[:n, :k] = w
            scales = padded.view(nb, 128, kb, 128).abs().amax(dim=(1, 3)) / E4M3_MAX
            w = w / scales.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
            s["weight"], s["weight_scales"] = w.to(torch.float8_e4m3fn), scales
    return s


class _Cache:
    """A paged cache's storage and layout, which is all that the operators read of one."""

    def __init__(self, blocks, block, kv_heads, dim, layers, dtype, device):
        self.layout = types.SimpleNamespace(num_layers=layers, num_blocks=blocks, block_size=block,
                                            num_kv_heads=kv_heads, head_dim=dim)
        self.k = torch.empty((layers, blocks, block, kv_heads, dim), dtype=dtype, device=device)
        self.v = torch.empty_like(self.k)


# --------------------------------------------------------------------------------------- run

def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    import inferkernellab_b200 as b200

    op = s["case"]["op"]
    if op == "sample":
        return b200.sample_tokens(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"],
                                  top_p=s["top_p"], min_p=s["min_p"])
    if op == "pages":
        b200.copy_kv_pages(s["cache"], s["src"], s["dst"], tokens=s["tokens"])
        tables = b200.remap_block_tables(s["tables"], s["page_map"])
        return s["cache"].k, s["cache"].v, tables
    if op == "qk_norm":
        q = b200.qk_norm_rope_append(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["cos"], s["sin"],
                                     s["cache"], s["slots"], eps=1e-6)
        return q, s["cache"].k, s["cache"].v
    if op == "quantize":
        return b200.quantize_fp8(s["x"])
    return b200.fp8_linear(s["x"], s["weight"], s["weight_scales"])


def _run_plain(s):
    return {"sample": _plain_sample, "pages": _plain_pages, "qk_norm": _plain_qk_norm, "quantize": _plain_quantize,
            "linear": _plain_linear}[s["case"]["op"]](s)


def _plain_sample(s):
    """Weights exp((l - max) / T); tokens in order of weight (ties: lowest index) are cut by min_p, then
    top_k, then top_p of what is left; the token is where the running sum of the kept weights, in order
    of index and in units of 2**-31, passes u times their sum."""
    logits = s["logits"].float()
    logits = torch.where(logits.isnan(), -torch.inf, logits)
    peak = logits.amax(dim=1, keepdim=True)
    greedy = s["temperature"] <= 0
    inverse = (1.0 / torch.where(greedy, 1.0, s["temperature"])).clamp(max=torch.finfo(torch.float32).max)
    x = (logits - peak) * inverse[:, None]
    x = torch.where(peak.isinf(), torch.where(logits == torch.inf, 0.0, -torch.inf), x)
    w = torch.exp(x)
    q = (w * 2.0 ** 31).round().to(torch.int64)
    order = torch.sort(w, dim=1, descending=True, stable=True).indices
    ws, qs = w.gather(1, order), q.gather(1, order)
    at = torch.arange(w.shape[1], device=w.device)
    top_k = torch.where(s["top_k"] <= 0, w.shape[1], s["top_k"])
    keep = (ws >= s["min_p"][:, None]) & (at < top_k[:, None])
    mass = (qs * keep).sum(dim=1, keepdim=True)
    before = (qs * keep).cumsum(dim=1) - qs * keep
    target = s["top_p"].double()[:, None] * mass.double()
    keep &= (before.double() < target) | (s["top_p"][:, None] >= 1) | (at == 0)
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    sums = (q * kept).cumsum(dim=1)
    total = sums[:, -1:]
    t = torch.minimum((s["uniforms"].double()[:, None] * total.double()).floor().long(), total - 1)
    token = (sums <= t).sum(dim=1)
    token = torch.where(greedy, torch.where(logits == peak, at, w.shape[1]).amin(dim=1), token)
    chosen = x.gather(1, token[:, None])[:, 0]
    logprob = chosen - torch.log(w.sum(dim=1))
    sampling = chosen - torch.log((w * kept).sum(dim=1))
    return token, logprob, sampling


def _plain_pages(s):
    src, dst, cache = s["src"].long(), s["dst"].long(), s["cache"]
    if s["tokens"] is None:
        cache.k[:, dst] = cache.k[:, src]
        cache.v[:, dst] = cache.v[:, src]
    else:
        copied = torch.arange(cache.k.shape[2], device=src.device) < s["tokens"][:, None]
        copied = copied[None, :, :, None, None]
        cache.k[:, dst] = torch.where(copied, cache.k[:, src], cache.k[:, dst])
        cache.v[:, dst] = torch.where(copied, cache.v[:, src], cache.v[:, dst])
    return cache.k, cache.v, s["page_map"][s["tables"].long()]


def _plain_norm_rope(x, weight, cos, sin):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + 1e-6) * weight.float()
    rd = cos.shape[-1]
    turned, rest = x[..., :rd], x[..., rd:]
    half = torch.cat([-turned[..., rd // 2:], turned[..., :rd // 2]], dim=-1)
    return torch.cat([turned * cos.float()[:, None] + half * sin.float()[:, None], rest], dim=-1)


def _plain_qk_norm(s):
    cache, slots = s["cache"], s["slots"].long()
    q = _plain_norm_rope(s["q"], s["q_weight"], s["cos"], s["sin"]).to(s["q"].dtype)
    k = _plain_norm_rope(s["k"], s["k_weight"], s["cos"], s["sin"]).to(s["k"].dtype)
    cache.k[0].flatten(0, 1)[slots] = k
    cache.v[0].flatten(0, 1)[slots] = s["v"]
    return q, cache.k, cache.v


def _plain_quantize_values(x):
    rows, cols = x.shape
    blocks = -(-cols // 128)
    padded = torch.nn.functional.pad(x.float(), (0, blocks * 128 - cols)).view(rows, blocks, 128)
    peak = padded.abs().amax(dim=2)
    peak = torch.where(peak < FLUSH, 0.0, peak)
    scales = peak / E4M3_MAX
    inverse = torch.where(peak == 0, 0.0, E4M3_MAX / peak)
    q = (padded * inverse[:, :, None]).to(torch.float8_e4m3fn)
    return q, scales


def _plain_quantize(s):
    q, scales = _plain_quantize_values(s["x"])
    return q.view(s["x"].shape[0], -1)[:, :s["x"].shape[1]].contiguous(), scales


def _plain_linear(s):
    x, weight = s["x"], s["weight"]
    q, scales = _plain_quantize_values(x)
    values = (q.float() * scales[:, :, None]).flatten(1)[:, :x.shape[1]]
    ws = s["weight_scales"].repeat_interleave(128, 0)[:weight.shape[0]].repeat_interleave(128, 1)[:, :weight.shape[1]]
    return (values @ (weight.float() * ws).t()).to(x.dtype)


# ------------------------------------------------------------------------------------- exact

def exact(case, seed):
    s = prepare(case, seed)
    return {"sample": _exact_sample, "pages": _exact_pages, "qk_norm": _exact_qk_norm, "quantize": _exact_quantize,
            "linear": _exact_linear}[case["op"]](s)


def _exact_sample(s):
    """Request by request: probabilities in 64 bits, ranked, cut, and drawn from.  The token itself is a
    whole number and has no 64-bit value; its two log-probabilities have."""
    logprobs, samplings = [], []
    for row in range(s["logits"].shape[0]):
        values = s["logits"][row].double()
        t = float(s["temperature"][row])
        p = torch.softmax(values / (t if t > 0 else 1.0), dim=0)
        ranked, ids = p.sort(descending=True, stable=True)
        n = int((ranked >= float(s["min_p"][row]) * ranked[0]).sum())
        if int(s["top_k"][row]) > 0:
            n = min(n, int(s["top_k"][row]))
        if float(s["top_p"][row]) < 1:
            cumulative = ranked[:n].cumsum(0)
            n = 1 + int((cumulative[:-1] < float(s["top_p"][row]) * cumulative[-1]).sum())
        chosen = ids[:n].sort().values
        sums = p[chosen].cumsum(0)
        at = int(torch.searchsorted(sums, float(s["uniforms"][row]) * sums[-1], right=True))
        token = int(values.argmax()) if t <= 0 else int(chosen[min(at, n - 1)])
        logprobs.append(torch.log(p[token]))
        samplings.append(torch.log(p[token]) - torch.log(sums[-1]))
    return None, torch.stack(logprobs), torch.stack(samplings)


def _exact_pages(s):
    """A copy has the source's very values: page after page."""
    k, v = s["cache"].k.double(), s["cache"].v.double()
    block = k.shape[2]
    counts = [block] * s["src"].numel() if s["tokens"] is None else s["tokens"].tolist()
    for a, b, n in zip(s["src"].tolist(), s["dst"].tolist(), counts):
        k[:, b, :n] = k[:, a, :n]
        v[:, b, :n] = v[:, a, :n]
    return k, v, None


def _exact_qk_norm(s):
    def turned(x, weight):
        x, weight, rd = x.double(), weight.double(), s["cos"].shape[1]
        y = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * weight
        z, h = y.clone(), rd // 2
        c, n = s["cos"].double()[:, None], s["sin"].double()[:, None]
        z[..., :h] = y[..., :h] * c[..., :h] - y[..., h:rd] * n[..., :h]
        z[..., h:rd] = y[..., h:rd] * c[..., h:] + y[..., :h] * n[..., h:]
        return z

    k, v = s["cache"].k.double(), s["cache"].v.double()
    block = k.shape[2]
    pages, offsets = s["slots"].long() // block, s["slots"].long() % block
    k[0, pages, offsets] = turned(s["k"], s["k_weight"])
    v[0, pages, offsets] = s["v"].double()
    return turned(s["q"], s["q_weight"]), k, v


def _exact_blocks(x):
    """The 8-bit values (nearest, ties to even, of x / scale) and the scales, in 64 bits."""
    rows, cols = x.shape
    blocks = -(-cols // 128)
    wide = torch.zeros(rows, blocks * 128, dtype=torch.float64, device=x.device)
    wide[:, :cols] = x.double()
    scales = wide.view(rows, blocks, 128).abs().amax(2) / E4M3_MAX
    unit = wide / scales.clamp(min=1e-300).repeat_interleave(128, 1)
    # 3 bits after the leading one, and steps of 2**-9 below 2**-6
    step = torch.exp2(torch.floor(torch.log2(unit.abs().clamp(min=2.0 ** -6))) - 3)
    return ((unit / step).round() * step)[:, :cols], scales


def _exact_quantize(s):
    return _exact_blocks(s["x"])


def _exact_linear(s):
    values, scales = _exact_blocks(s["x"])
    n, k = s["weight"].shape
    weight = s["weight"].double()
    out = torch.zeros(values.shape[0], n, dtype=torch.float64, device=values.device)
    column = torch.arange(n, device=values.device) // 128
    for b in range(scales.shape[1]):
        part = slice(128 * b, min(k, 128 * (b + 1)))
        out += (values[:, part] @ weight[:, part].t()) * scales[:, b:b + 1] * s["weight_scales"].double()[column, b]
    return out
