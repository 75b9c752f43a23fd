"""A server's step beside its attention, as cases that can be timed and checked: the adapters of many requests, the norms and rotation of
queries and keys, what is said about the tokens that come out, and pages that several requests share.

Kinds:

* ``lora``      ``lora.lora_add_``: every request's low-rank adapter beside a projection that all share;
* ``norm``      ``paged_kv.paged_norm_rope_append``: RMS norm of every query and key head and its rotation in one pass, keys and values into the cache;
* ``logprobs``  ``logprobs.token_logprobs``: log probability of given tokens, entropy and the most likely alternatives; with ``grad`` the gradient too;
* ``fork``      ``paged_kv.paged_fork`` and ``paged_copy``: requests that go on from where others are, sharing their full pages;
* ``branch``    ``paged_fork`` and ``paged_release``: the same without the copies, and the branches given up again;
* ``compact``   ``paged_kv.paged_compact`` and ``paged_copy``: the pages in use moved to the front of the cache.

Sizes are those of the Llama-2-7B / Mistral-7B / Llama-2-70B / Llama-3-8B layers and vocabularies that the framework's benchmarks and tests use, or
generic ones of that range.
"""
import math
import random

import torch

own = False
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
DEVICE = "cuda"
HEADS = ((32, 32), (32, 8), (64, 8), (20, 20), (14, 2), (8, 1), (40, 8))
WIDTHS = (896, 2048, 4096, 5120, 8192, 11008, 14336)
OUTPUTS = ("896", "2048", "4096", "11008", "14336", "4096+1024+1024", "896+128+128", "4096+4096+4096", "8192+1024+1024", "11008+11008", "2040")
VOCABS = (32000, 128256, 50257, 2048, 999)


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one request with its adapter on the output projection of a 7B layer: the smallest call, a launch or two
        {"name": "lora_token", "kind": "lora", "requests": 1, "new_lo": 1, "new_hi": 1, "adapters": 4, "rank": 16, "in": 4096, "out": "4096", "dtype": "fp16"},
        # a decode batch on a merged projection with grouped heads, as many adapters as half the requests
        {"name": "lora_tokens", "kind": "lora", "requests": 64, "new_lo": 1, "new_hi": 1, "adapters": 32, "rank": 16, "in": 4096, "out": "4096+1024+1024",
         "dtype": "bf16"},
        # a step that mixes decoding requests and chunks of odd length, rank 64 into a feed-forward
        {"name": "lora_mixed", "kind": "lora", "requests": 40, "new_lo": 1, "new_hi": 300, "adapters": 12, "rank": 64, "in": 4096, "out": "11008", "dtype": "fp16"},
        # the prompts of a step
        {"name": "lora_prompts", "kind": "lora", "requests": 8, "new_lo": 300, "new_hi": 4000, "adapters": 5, "rank": 32, "in": 4096, "out": "14336", "dtype": "bf16"},
        # a decode batch of a grouped-query layer whose heads are normalised, 8-bit cache
        {"name": "norm_tokens", "kind": "norm", "tokens": 32, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "cache": "e5m2", "page": 16},
        # the prompts of a step
        {"name": "norm_prompts", "kind": "norm", "tokens": 8001, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "cache": "bf16", "page": 32},
        # one answer's next token, with the five likeliest
        {"name": "logprobs_token", "kind": "logprobs", "rows": 1, "vocab": 32000, "dtype": "fp16", "top_k": 5, "temperature": 1.0, "masked": 0.0, "grad": False},
        # a large decode batch over a large vocabulary, with twenty alternatives and part of the vocabulary ruled out
        {"name": "logprobs_batch", "kind": "logprobs", "rows": 256, "vocab": 128256, "dtype": "bf16", "top_k": 20, "temperature": 0.7, "masked": 0.2, "grad": False},
        # a training step's loss on packed samples, forward and backward: log probabilities and an entropy bonus
        {"name": "logprobs_train", "kind": "logprobs", "rows": 4001, "vocab": 32000, "dtype": "bf16", "top_k": 0, "temperature": 1.0, "masked": 0.0, "grad": True},
        # four samples of one prompt: the launches count
        {"name": "fork_few", "kind": "fork", "requests": 3, "forks": 4, "held_lo": 100, "held_hi": 3000, "page": 16, "kv_heads": 8, "dim": 128, "layers": 8,
         "cache": "bf16"},
        # a beam search over many requests, which drops its branches again
        {"name": "branch_many", "kind": "branch", "requests": 100, "forks": 300, "held_lo": 100, "held_hi": 8000, "page": 16},
        # a cache after hours of requests that came and went, moved together before a part of it is given back
        {"name": "compact", "kind": "compact", "requests": 40, "held_lo": 100, "held_hi": 2000, "page": 32, "spare": 2.0, "kv_heads": 8, "dim": 128, "layers": 6,
         "cache": "e5m2"},
    ]


def _log(rng, lo, hi):
    """a whole number spread evenly over the logarithm of [lo, hi]"""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("lora", "lora", "norm", "logprobs", "logprobs", "fork", "branch", "compact"))
    page, dtype = rng.choice((8, 16, 32, 64, 24)), rng.choice(("fp16", "bf16"))
    heads, kv_heads = rng.choice(HEADS)
    dim = rng.choice((64, 128, 128, 96, 256))
    lens = rng.randrange(1 << 20)
    if kind == "norm":
        return {"kind": kind, "tokens": _log(rng, 1, 6000 * 4096 // (heads * dim + 1) if heads * dim > 4096 else 6000), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "dtype": dtype, "cache": rng.choice(("e5m2", dtype)), "page": page}
    if kind == "logprobs":
        vocab, grad = rng.choice(VOCABS), rng.random() < 0.5
        return {"kind": kind, "rows": _log(rng, 1, min(4000, 130_000_000 // vocab // (1 if grad else 2))), "vocab": vocab, "dtype": rng.choice(("fp16", "bf16", "fp32")),
                "top_k": rng.choice((0, 1, 5, 20)), "temperature": rng.choice((1.0, 0.7, 1.5)), "masked": rng.choice((0.0, 0.0, 0.3)), "grad": grad}
    if kind == "lora":
        while True:
            lo = _log(rng, 1, 1000)
            case = {"kind": kind, "requests": _log(rng, 1, 100), "new_lo": lo, "new_hi": rng.choice((lo, _log(rng, lo, 4000))), "adapters": _log(rng, 1, 40),
                    "rank": rng.choice((8, 16, 16, 32, 64, 128)), "in": rng.choice(WIDTHS), "out": rng.choice(OUTPUTS), "dtype": dtype, "lens": lens}
            w = work(case)
            if w["bytes"] <= 4e8 and w["flops"] <= 3e10:
                return case
    held_lo = _log(rng, 1, 2000)
    case = {"kind": kind, "requests": _log(rng, 1, 100), "held_lo": held_lo, "held_hi": _log(rng, held_lo, 4000), "page": page, "lens": lens}
    if kind == "compact":
        case["spare"] = rng.choice((1.1, 1.5, 3.0))
    else:
        case["forks"] = _log(rng, 1, 200)
    if kind != "branch":
        pages = sum(-(-h // page) for h in _held(case)) * case.get("spare", 1.0) + case.get("forks", 0)
        size = 2 * page * kv_heads * dim * pages
        case |= {"kv_heads": kv_heads, "dim": dim, "layers": max(1, min(rng.choice((1, 4, 9)), int(4e8 / size))), "cache": rng.choice(("e5m2", dtype))}
    return case


def _new(case):
    """new tokens of every request, the same for every seed so that the work is the case's own; of requests that may bring a chunk three in four
    bring one token"""
    rng, lo, hi = random.Random(case.get("lens", 1)), case["new_lo"], case["new_hi"]
    return [lo if lo == 1 and i % 4 else _log(rng, max(lo, min(hi, 17)), hi) for i in range(case["requests"])]


def _held(case):
    """tokens that every request holds: of three requests one ends with a full page"""
    rng = random.Random(case.get("lens", 1))
    held = [_log(rng, case["held_lo"], case["held_hi"]) for _ in range(case["requests"])]
    return [-(-h // case["page"]) * case["page"] if i % 3 == 2 else h for i, h in enumerate(held)]


def _adapter_of(case):
    """the adapter of every request; one in eight has none"""
    rng = random.Random(case.get("lens", 1) + 1)
    return [-1 if i % 8 == 7 else rng.randrange(case["adapters"]) for i in range(case["requests"])]


def _splits(case):
    return [int(n) for n in case["out"].split("+")]


def _parents(case):
    rng = random.Random(case.get("lens", 1) + 2)
    return [rng.randrange(case["requests"]) for _ in range(case["forks"])]


# ------------------------------------------------------------------ what a program has in hand
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE)


def _cache(case, pages, g):
    x = torch.randn((pages, case["page"], case["kv_heads"], case["dim"]), generator=g, device=DEVICE, dtype=torch.float16)
    return x.to(torch.float8_e5m2).view(torch.uint8) if case["cache"] == "e5m2" else x.to(DTYPES[case["cache"]])


def _tables(dim):
    """cosines and sines of 20000 positions, rotate-half layout"""
    freq = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=DEVICE) / dim)
    a = torch.arange(20000, dtype=torch.float64, device=DEVICE)[:, None] * freq
    return torch.cat([a.cos(), a.cos()], -1).float(), torch.cat([a.sin(), a.sin()], -1).float()


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    return {"kind": kind, "case": case} | {"lora": _have_lora, "norm": _have_norm, "logprobs": _have_logits}.get(kind, _have_pages)(case, g)


def _have_lora(case, g):
    new, ids, splits, dtype = _new(case), _adapter_of(case), _splits(case), DTYPES[case["dtype"]]
    k, n, r, count = case["in"], sum(splits), case["rank"], case["adapters"]
    t = sum(new)
    return {"new": new, "ids": ids, "splits": splits, "x": _randn(g, t, k).to(dtype), "out": _randn(g, t, n).to(dtype),
            "a": (_randn(g, count, len(splits), r, k) * k ** -0.5).to(dtype), "b": (_randn(g, count, n, r) * 0.5 * r ** -0.5).to(dtype),
            "scales": 0.5 + 1.5 * torch.rand(count, generator=g, device=DEVICE), "adapter_ids": _ints(ids), "cu": _ints([0] + new).cumsum(0, dtype=torch.int32)}


def _have_norm(case, g):
    t, heads, kv, dim, dtype = case["tokens"], case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    pages = -(-t // case["page"]) + 3
    cos, sin = _tables(dim)
    at = torch.arange(t, device=DEVICE)
    order = torch.randperm(pages, generator=g, device=DEVICE)
    # heads of very different size, as a projection gives them
    size = torch.exp2(2 * _randn(g, t, heads + 2 * kv, 1))
    return {"qkv": (_randn(g, t, heads + 2 * kv, dim) * size).flatten(1).to(dtype), "q_weight": (1 + 0.3 * _randn(g, dim)).to(dtype),
            "k_weight": (1 + 0.3 * _randn(g, dim)).to(dtype), "eps": 1e-6, "cos": cos, "sin": sin, "k_cache": _cache(case, pages, g), "v_cache": _cache(case, pages, g),
            "positions": torch.randint(0, 20000 - t, (1,), generator=g, device=DEVICE) + at, "slots": order[at // case["page"]] * case["page"] + at % case["page"]}


def _have_logits(case, g):
    rows, vocab, k = case["rows"], case["vocab"], case["top_k"]
    logits = (3 * _randn(g, rows, vocab)).to(DTYPES[case["dtype"]])
    tokens = torch.randint(0, vocab, (rows,), generator=g, device=DEVICE)
    if case["masked"]:                                   # what a grammar or a filter has ruled out; the tokens are none of it
        out = torch.rand(rows, vocab, generator=g, device=DEVICE) < case["masked"]
        logits.masked_fill_(out.scatter(1, tokens[:, None], False), -math.inf)
    s = {"logits": logits, "tokens": tokens}
    if case["grad"]:
        s["tokens"] = torch.where(torch.rand(rows, generator=g, device=DEVICE) < 0.05, -100, tokens)      # a sample's prompt and padding
        logits.requires_grad_()
        s["grads"] = [_randn(g, rows) / rows, -0.01 * torch.rand(rows, generator=g, device=DEVICE) / rows] + ([_randn(g, rows, k) / rows] if k else [])
    return s


def _have_pages(case, g):
    held, page = _held(case), case["page"]
    had = [-(-h // page) for h in held]
    used = sum(had)
    forks = case.get("forks", 0)
    pages = int(used * case.get("spare", 1.0)) + forks + 5
    width = max(had) + 2
    order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((len(held) + forks, width), -1, dtype=torch.int32, device=DEVICE)
    cols = torch.arange(width, device=DEVICE)[None]
    table[:len(held)][cols < _ints(had)[:, None]] = order[:used]
    s = {"table": table, "free_pages": torch.cat([order[used:], torch.full((used,), -1, dtype=torch.int32, device=DEVICE)]), "free_count": _ints([pages - used]),
         "shared": torch.zeros(pages, dtype=torch.int32, device=DEVICE)}
    if case["kind"] == "compact":
        # every fifth request shares the first half of its neighbour's pages, and its own are free; two pages are nobody's
        for i in range(1, len(held), 5):
            both = min(had[i], had[i - 1]) // 2
            if both:
                back = table[i, :both].clone()
                table[i, :both] = table[i - 1, :both]
                s["shared"][table[i, :both].long()] += 1
                count = int(s["free_count"])
                s["free_pages"][count:count + both] = back
                s["free_count"] += both
        s["free_count"] -= 2
    else:
        s["lens"] = _ints(held + [0] * forks)
        s["parents"], s["children"] = _ints(_parents(case)), torch.arange(len(held), len(held) + forks, dtype=torch.int32, device=DEVICE)
        s["done"] = torch.arange(len(held) + forks, device=DEVICE) >= len(held)
    if case["kind"] != "branch":
        s["caches"] = [_cache(case, pages, g) for _ in range(2 * case["layers"])]
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _run_own(s)
    return {"lora": _plain_lora, "norm": _plain_norm, "logprobs": _plain_logprobs, "fork": _plain_fork_copy, "branch": _plain_branch, "compact": _plain_compact_copy}[s["kind"]](s)


def _values(cache):
    """e5m2 bytes as the numbers that they stand for"""
    return cache.view(torch.float8_e5m2) if cache.dtype == torch.uint8 else cache


def _run_own(s):
    case, kind = s["case"], s["kind"]
    if kind == "lora":
        from ipex_llm_b200.transformers.lora import lora_add_
        return lora_add_(s["out"], s["x"], s["a"], s["b"], s["scales"], s["adapter_ids"], s["cu"], splits=s["splits"])
    if kind == "logprobs":
        from ipex_llm_b200.transformers.logprobs import token_logprobs
        got = token_logprobs(s["logits"], s["tokens"], top_k=case["top_k"], temperature=case["temperature"])
        out = {"logprobs": got.logprobs, "entropy": got.entropy}
        if case["top_k"]:
            out |= {"top_ids": got.top_ids, "top_logprobs": got.top_logprobs}
        if case["grad"]:
            given = [got.logprobs, got.entropy] + ([got.top_logprobs] if case["top_k"] else [])
            out["grad"], = torch.autograd.grad(given, s["logits"], s["grads"])
        return {name: t.detach() for name, t in out.items()}
    from ipex_llm_b200.transformers import paged_kv
    if kind == "norm":
        paged_kv.paged_norm_rope_append(s["qkv"], case["heads"], case["kv_heads"], case["dim"], s["q_weight"], s["k_weight"], s["eps"], s["cos"], s["sin"], s["positions"],
                                        s["slots"], s["k_cache"], s["v_cache"])
        return {"qkv": s["qkv"], "k_cache": _values(s["k_cache"]), "v_cache": _values(s["v_cache"])}
    if kind == "compact":
        c = paged_kv.paged_compact(s["table"], s["free_pages"], s["free_count"], s["shared"])
        paged_kv.paged_copy(c.src, c.dst, s["caches"])
        return {"table": c.block_table, "free_pages": c.free_pages, "free_count": c.free_count, "shared": c.shared, "src": c.src, "dst": c.dst,
                "caches": [_values(x) for x in s["caches"]]}
    left = s["free_count"] if kind == "branch" else None
    f = paged_kv.paged_fork(s["parents"], s["children"], s["lens"], s["table"], s["free_pages"], s["free_count"], s["shared"], case["page"], free_left=left)
    out = {"src": f.src, "dst": f.dst, "missing": f.missing, "free_count": f.free_count, "lens": s["lens"], "table": s["table"], "shared": s["shared"], "free_pages": s["free_pages"]}
    if kind == "branch":
        paged_kv.paged_release(s["done"], s["table"], s["free_pages"], s["free_count"], shared=s["shared"])
        return out
    paged_kv.paged_copy(f.src, f.dst, s["caches"])
    return out | {"caches": [_values(x) for x in s["caches"]]}


def _plain_lora(s):
    x, out, new, scales = s["x"], s["out"], s["new"], s["scales"]
    a, b = s["a"].flatten(1, 2), s["b"].split(s["splits"], dim=1)
    rank = s["a"].shape[2]
    if max(new) == 1:                                    # a batch of tokens, each with its adapter's weights
        ids = s["adapter_ids"].long()
        at = ids.clamp(min=0)
        h = torch.bmm(a[at].float(), x.float()[:, :, None]) * scales[at, None, None]
        more = torch.cat([torch.bmm(w[at].float(), h[:, i * rank:(i + 1) * rank]) for i, w in enumerate(b)], 1)[..., 0]
        out.copy_(torch.where((ids >= 0)[:, None], out.float() + more, out.float()))
        return out
    first = 0
    for n, i in zip(new, s["ids"]):
        if i >= 0:
            rows = slice(first, first + n)
            h = (x[rows].float() @ a[i].float().T) * scales[i]
            out[rows] = (out[rows].float() + torch.cat([h[:, j * rank:(j + 1) * rank] @ w[i].float().T for j, w in enumerate(b)], 1)).to(out.dtype)
        first += n
    return out


def _to_cache(x, cache):
    """values in the cache's form: e5m2 saturates at its largest number"""
    return x.float().clamp(-57344, 57344).to(torch.float8_e5m2).view(torch.uint8) if cache.dtype == torch.uint8 else x


def _plain_norm(s):
    case, qkv = s["case"], s["qkv"]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    x = qkv.view(-1, heads + 2 * kv, dim)
    y = x[:, :heads + kv].float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + s["eps"])
    y = torch.cat([y[:, :heads] * s["q_weight"].float(), y[:, heads:] * s["k_weight"].float()], 1)
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    half = torch.cat([-y[..., dim // 2:], y[..., :dim // 2]], -1)
    x[:, :heads + kv] = (y * cos + half * sin).to(x.dtype)
    s["k_cache"].view(-1, kv, dim)[s["slots"]] = _to_cache(x[:, heads:heads + kv], s["k_cache"])
    s["v_cache"].view(-1, kv, dim)[s["slots"]] = _to_cache(x[:, heads + kv:], s["v_cache"])
    return {"qkv": qkv, "k_cache": _values(s["k_cache"]), "v_cache": _values(s["v_cache"])}


def _plain_logprobs(s):
    case, tokens = s["case"], s["tokens"]
    k, temperature = case["top_k"], case["temperature"]
    logits = s["logits"].detach()
    z = logits.float() / temperature
    z -= z.amax(-1, keepdim=True)
    logp = z - z.exp().sum(-1, keepdim=True).log()
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    here = tokens >= 0
    at = tokens.clamp(min=0)[:, None]
    out = {"logprobs": torch.where(here, logp.gather(1, at)[:, 0], 0.0), "entropy": entropy}
    if k:
        ids = torch.sort(logits.float(), dim=-1, descending=True, stable=True).indices[:, :k].contiguous()
        out |= {"top_ids": ids, "top_logprobs": logp.gather(1, ids)}
    if case["grad"]:
        given = torch.where(here, s["grads"][0], 0.0)
        total = given + s["grads"][2].sum(-1) if k else given
        grad = -p * total[:, None] - s["grads"][1][:, None] * torch.where(p > 0, p * (logp + entropy[:, None]), 0.0)
        grad.scatter_add_(1, at, given[:, None])
        if k:
            grad.scatter_add_(1, ids, s["grads"][2])
        out["grad"] = (grad / temperature).to(logits.dtype)
    return out


def _plain_copy(src, dst, caches):
    there = (src >= 0) & (dst >= 0)
    a, b = src[there].long(), dst[there].long()
    for c in caches:
        c[b] = c[a]


def _plain_fork(s, left):
    page, table, lens, count = s["case"]["page"], s["table"], s["lens"], s["free_count"]
    par, ch = s["parents"].long(), s["children"].long()
    held, rows = lens[par], table[par]
    full, need = held // page, held % page != 0
    rank = need.cumsum(0) - need.long()
    index = count - 1 - rank
    fresh = torch.where(index >= 0, s["free_pages"][index.clamp(min=0)], -1)
    cols = torch.arange(table.shape[1], device=table.device)[None]
    src = torch.where(need, rows.gather(1, full.long().clamp(max=table.shape[1] - 1)[:, None])[:, 0], -1)
    dst = torch.where(need, fresh, -1).int()
    whole = cols < full[:, None]
    table[ch] = torch.where(whole, rows, torch.where((cols == full[:, None]) & need[:, None], fresh[:, None], -1)).int()
    # rows of the table as they are: entries behind the full pages count for nothing
    s["shared"].index_add_(0, rows.clamp(min=0).flatten().long(), (whole & (rows >= 0)).flatten().int())
    lens[ch] = held
    short = count - need.sum()
    out = {"src": src, "dst": dst, "missing": (-short).clamp(min=0).int(), "free_count": short.clamp(min=0).int()}
    if left is not None:
        out["free_count"] = left.copy_(out["free_count"])
    return out | {"lens": lens, "table": table, "shared": s["shared"], "free_pages": s["free_pages"]}


def _plain_fork_copy(s):
    out = _plain_fork(s, None)
    _plain_copy(out["src"], out["dst"], s["caches"])
    return out | {"caches": [_values(x) for x in s["caches"]]}


def _plain_branch(s):
    out = _plain_fork(s, s["free_count"])
    table, shared, count, stack = s["table"], s["shared"], s["free_count"], s["free_pages"]
    n = shared.numel()
    entry = torch.where(s["done"][:, None], table, -1).flatten().long()
    named = entry >= 0
    at = torch.where(named, entry, n)
    times = torch.zeros(n + 1, dtype=torch.int32, device=at.device).index_add_(0, at, torch.ones_like(at, dtype=torch.int32))[:n]
    order = torch.arange(at.numel(), device=at.device)
    first = torch.full((n + 1,), at.numel(), device=at.device).scatter_reduce_(0, at, order, "amin")
    free = named & (first[at] == order) & (times > shared)[at.clamp(max=n - 1)]
    to = torch.where(free, count + free.cumsum(0) - 1, n)
    longer = torch.cat([stack, stack.new_zeros(1)])
    longer[to] = entry.int()
    stack.copy_(longer[:n])
    count += free.sum().int()
    shared.copy_((shared - times).clamp(min=0))
    table[s["done"]] = -1
    return out


def _plain_compact_copy(s):
    table, stack, shared = s["table"], s["free_pages"], s["shared"]
    n, count = shared.numel(), int(s["free_count"])
    used = torch.zeros(n + 1, dtype=torch.bool, device=table.device)
    used[torch.where(table >= 0, table, n).flatten().long()] = True
    used = used[:n]
    free = torch.zeros_like(used)
    free[stack[:count].long()] = True
    free &= ~used
    holes, high = free.nonzero()[:, 0], used.nonzero()[:, 0].flip(0)
    m = min(holes.numel(), high.numel())
    m = int((holes[:m] < high[:m]).sum())
    src, dst = torch.full((n,), -1, dtype=torch.int32, device=table.device), torch.full((n,), -1, dtype=torch.int32, device=table.device)
    src[:m], dst[:m] = high[:m].int(), holes[:m].int()
    to = torch.arange(n, dtype=torch.int32, device=table.device)
    to[high[:m]] = dst[:m]
    moved = shared.clone()
    moved[holes[:m]] = shared[high[:m]]
    moved[high[:m]] = 0
    free[holes[:m]] = False
    free[high[:m]] = True
    left = free.nonzero()[:, 0].flip(0).int()
    out_stack = torch.full_like(stack, -1)
    out_stack[:left.numel()] = left
    _plain_copy(src, dst, s["caches"])
    return {"table": torch.where(table >= 0, to[table.clamp(min=0).long()], -1), "free_pages": out_stack, "free_count": _ints([left.numel()]), "shared": moved,
            "src": src, "dst": dst, "caches": [_values(x) for x in s["caches"]]}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "lora":
        new, ids, n, k, r = _new(case), _adapter_of(case), sum(_splits(case)), case["in"], case["rank"]
        s = len(_splits(case))
        t = sum(c for c, i in zip(new, ids) if i >= 0)
        weights = len({i for i in ids if i >= 0}) * r * (s * k + n)
        return {"bytes": 2 * (t * (k + 2 * n) + weights), "flops": 2 * t * r * (s * k + n)}
    if kind == "norm":
        t, heads, kv, dim = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        kept = 1 if case["cache"] == "e5m2" else 2
        return {"bytes": t * (dim * (2 * (heads + 2 * kv) + 2 * (heads + kv) + 2 * kv * kept) + 4 * dim + 16), "flops": 7 * t * (heads + kv) * dim}
    if kind == "logprobs":
        size = case["rows"] * case["vocab"]
        each = 4 if case["dtype"] == "fp32" else 2
        # the logits in, and their gradient out
        return {"bytes": size * each * (2 if case["grad"] else 1) + case["rows"] * (16 + 12 * case["top_k"]), "flops": size * (9 if case["grad"] else 5)}
    held, page = _held(case), case["page"]
    had = [-(-h // page) for h in held]
    if kind == "compact":
        used, size = sum(had), int(sum(had) * case["spare"]) + 5
        moves = used * (size - used) // size
        return {"bytes": _page_bytes(case) * 2 * moves + 4 * (2 * used + 6 * size), "flops": used}
    parents = _parents(case)
    named, copies = sum(had[p] for p in parents), sum(held[p] % page != 0 for p in parents)
    if kind == "branch":
        return {"bytes": 4 * (6 * named + 4 * len(parents)), "flops": 2 * named}
    return {"bytes": 2 * copies * _page_bytes(case) + 4 * (4 * named + 4 * len(parents)), "flops": named}


def _page_bytes(case):
    """one page of all layers' keys and values"""
    return 2 * case["layers"] * case["page"] * case["kv_heads"] * case["dim"] * (1 if case["cache"] == "e5m2" else 2)


# ------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    kind = case["kind"]
    if kind not in ("lora", "norm", "logprobs"):
        return None                                       # whole numbers and copies: there is nothing to round
    s = prepare(case, seed)
    return {"lora": _exact_lora, "norm": _exact_norm, "logprobs": _exact_logprobs}[kind](case, s)


def _exact_lora(case, s):
    out = s["out"].double()
    ids = torch.repeat_interleave(s["adapter_ids"], s["cu"][1:] - s["cu"][:-1])
    for i in range(case["adapters"]):
        rows = (ids == i).nonzero()[:, 0]
        if rows.numel() == 0:
            continue
        x, first = s["x"][rows].double(), 0
        for j, n in enumerate(_splits(case)):
            # the adapter as one matrix
            whole = s["b"][i, first:first + n].double() @ s["a"][i, j].double()
            for part in rows.split(4096):
                out[part, first:first + n] += float(s["scales"][i]) * (s["x"][part].double() @ whole.T)
            first += n
    return out


def _exact_norm(case, s):
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    x = s["qkv"].double().view(case["tokens"], -1, dim)
    angle = s["positions"].double()[:, None, None] * torch.exp2(-math.log2(10000.0) * 2 / dim * torch.arange(dim // 2, device=DEVICE, dtype=torch.float64))
    n = heads + kv
    weight = torch.stack([s["q_weight"]] * heads + [s["k_weight"]] * kv).double()
    y = x[:, :n] * weight / torch.sqrt(torch.linalg.vector_norm(x[:, :n], dim=-1, keepdim=True) ** 2 / dim + s["eps"])
    z = torch.polar(torch.ones_like(angle), angle) * torch.complex(y[..., :dim // 2].contiguous(), y[..., dim // 2:].contiguous())
    x = torch.cat([torch.cat([z.real, z.imag], -1), x[:, n:]], 1)
    out = {"qkv": x.reshape(case["tokens"], -1)}
    for name, first in (("k_cache", heads), ("v_cache", n)):
        rows = x[:, first:first + kv]
        if case["cache"] == "e5m2":                       # the bytes hold the rounded activations' nearest e5m2 values
            rows = rows.to(DTYPES[case["dtype"]]).to(torch.float8_e5m2).double()
        whole = _values(s[name]).double()
        whole.view(-1, kv, dim)[s["slots"]] = rows
        out[name] = whole
    return out


def _exact_logprobs(case, s):
    k, rows = case["top_k"], case["rows"]
    parts = []
    for first in range(0, rows, 512):
        at = slice(first, first + 512)
        tokens = s["tokens"][at]
        z = s["logits"].detach()[at].double() / case["temperature"]
        q = torch.log_softmax(z, -1)
        w = torch.softmax(z, -1)
        h = torch.special.entr(w).sum(-1)
        token = torch.where(tokens < 0, 0.0, q.gather(1, tokens.clamp(min=0)[:, None])[:, 0])
        part = {"logprobs": token, "entropy": h}
        if k:
            ids = torch.argsort(-s["logits"].detach()[at].double(), dim=-1, stable=True)[:, :k]
            part |= {"top_ids": ids, "top_logprobs": q.gather(1, ids)}
        if case["grad"]:
            coefficient = torch.zeros_like(z)
            coefficient.scatter_add_(1, tokens.clamp(min=0)[:, None], torch.where(tokens < 0, 0.0, s["grads"][0][at].double())[:, None])
            if k:
                coefficient.scatter_add_(1, ids, s["grads"][2][at].double())
            # entropy = -sum w q, and dw = w (dz - sum w dz)
            surprise = torch.where(w > 0, q, 0.0) + h[:, None]
            part["grad"] = (coefficient - w * coefficient.sum(-1, keepdim=True) - s["grads"][1][at].double()[:, None] * w * surprise) / case["temperature"]
        parts.append(part)
    return {name: torch.cat([p[name] for p in parts]) for name in parts[0]}
