"""Serving many requests from one paged key/value cache, as cases that can be timed and checked.

Kinds (each one call of ``ipex_llm_b200.transformers.paged_kv``):

* ``step``    ``paged_step``: from what every request holds and brings, the pages that it still needs, its block table, and for every new
              token its position and its slot in the cache;
* ``append``  ``paged_rope_append``: rotary embedding of the new tokens' queries and keys in the merged projection's output, keys and values
              into their slots;
* ``paged``   ``sdp_paged``: attention of every request's new tokens (one, or a chunk of a prompt) over its pages;
* ``packed``  ``sdp_packed``: causal attention of whole prompts that lie behind one another, straight from the projection's output.

The cache is [pages, page_size, kv heads, head_dim], of the activations' type or e5m2 bytes.  Head counts and sizes are those of the
Llama-2-7B / Mistral-7B / Llama-2-70B layers that the framework's benchmarks and tests use, or generic ones of that range.
"""
import math
import random

import torch

own = False
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
DEVICE = "cuda"
HEADS = ((32, 32), (32, 8), (64, 8), (20, 20), (14, 2), (8, 1), (40, 8))


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # a small server's decode step: 32 requests with one new token each, where the launch is most of the time
        {"name": "step_decode", "kind": "step", "requests": 32, "held_lo": 100, "held_hi": 4000, "new_lo": 1, "new_hi": 1, "page": 16},
        # a large server's step, in which some requests bring a chunk of their prompt and most one token
        {"name": "step_mixed", "kind": "step", "requests": 500, "held_lo": 1, "held_hi": 16000, "new_lo": 1, "new_hi": 700, "page": 64},
        # one token of a 7B layer into an 8-bit cache
        {"name": "append_token", "kind": "append", "tokens": 1, "heads": 32, "kv_heads": 32, "dim": 128, "dtype": "fp16", "cache": "e5m2", "page": 16},
        # the prompts of a step, 8000 tokens of a grouped-query layer
        {"name": "append_prompts", "kind": "append", "tokens": 8000, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "cache": "bf16", "page": 32},
        # one request alone at 4000 tokens, 7B heads, 8-bit cache: the shortest attention
        {"name": "token_alone", "kind": "paged", "requests": 1, "held_lo": 4000, "held_hi": 4000, "new_lo": 1, "new_hi": 1, "heads": 32, "kv_heads": 32, "dim": 128,
         "dtype": "fp16", "cache": "e5m2", "page": 16},
        # a decode batch of requests of very different lengths, grouped heads, 8-bit cache
        {"name": "tokens_fp8", "kind": "paged", "requests": 64, "held_lo": 100, "held_hi": 16000, "new_lo": 1, "new_hi": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "dtype": "bf16", "cache": "e5m2", "page": 16},
        # the same with 70B heads and the cache in the activations' type
        {"name": "tokens_bf16", "kind": "paged", "requests": 100, "held_lo": 200, "held_hi": 8000, "new_lo": 1, "new_hi": 1, "heads": 64, "kv_heads": 8, "dim": 128,
         "dtype": "bf16", "cache": "bf16", "page": 64},
        # a chunk of a long prompt over what the request already holds
        {"name": "chunk", "kind": "paged", "requests": 1, "held_lo": 16000, "held_hi": 16000, "new_lo": 512, "new_hi": 512, "heads": 32, "kv_heads": 8, "dim": 128,
         "dtype": "bf16", "cache": "bf16", "page": 32},
        # a step of a server that mixes both: most requests decode, some bring a chunk of odd length; small heads
        {"name": "mixed", "kind": "paged", "requests": 40, "held_lo": 10, "held_hi": 5000, "new_lo": 1, "new_hi": 300, "heads": 20, "kv_heads": 20, "dim": 64,
         "dtype": "fp16", "cache": "e5m2", "page": 16},
        # a few short prompts, small heads
        {"name": "prompts_short", "kind": "packed", "requests": 7, "new_lo": 17, "new_hi": 300, "heads": 20, "kv_heads": 20, "dim": 64, "dtype": "fp16"},
        # prompts of very different lengths, grouped heads
        {"name": "prompts_ragged", "kind": "packed", "requests": 8, "new_lo": 200, "new_hi": 4000, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16"},
        # one long prompt with 7B heads
        {"name": "prompt_long", "kind": "packed", "requests": 1, "new_lo": 8000, "new_hi": 8000, "heads": 32, "kv_heads": 32, "dim": 128, "dtype": "fp16"},
    ]


def _log(rng, lo, hi):
    """a whole number spread evenly over the logarithm of [lo, hi]"""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("step", "append", "paged", "paged", "packed"))
    page = rng.choice((8, 16, 32, 64, 128, 24))
    if kind == "step":
        lo = _log(rng, 1, 4000)
        return {"kind": kind, "requests": _log(rng, 1, 500), "held_lo": lo, "held_hi": _log(rng, lo, 16000), "new_lo": 1, "new_hi": _log(rng, 1, 700),
                "page": page, "lens": rng.randrange(1 << 20)}
    heads, kv_heads = rng.choice(HEADS)
    dim, dtype = rng.choice((64, 128, 128, 96, 256)), rng.choice(("fp16", "bf16"))
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype}
    if kind == "append":
        return case | {"tokens": _log(rng, 1, 4000), "cache": rng.choice(("e5m2", dtype)), "page": page}
    case["lens"] = rng.randrange(1 << 20)
    for _ in range(200):
        requests = _log(rng, 1, 100)
        if kind == "packed":
            lo = _log(rng, 1, 2000)
            more = {"requests": requests, "new_lo": lo, "new_hi": _log(rng, lo, 8000)}
        else:
            lo = _log(rng, 1, 16000)
            more = {"requests": requests, "held_lo": lo, "held_hi": _log(rng, lo, 16000), "new_lo": 1,
                    "new_hi": 1 if rng.random() < 0.5 else _log(rng, 1, 600), "cache": rng.choice(("e5m2", dtype)), "page": page}
        new, held = _lengths(case | more)
        w, longest = work(case | more), max(h + n for h, n in zip(held, new))
        # no more work, and no more scores and padded keys in the plain form, than the largest listed cases
        if w["bytes"] <= 8e8 and w["flops"] <= 5e11 and requests * longest * max(heads * max(new), 2 * kv_heads * dim) <= 2.1e9:
            break
    return case | more


def _lengths(case):
    """(new tokens, tokens held before) of every request: the same for every seed, so that the work is the case's own.  Lengths spread over
    the logarithm of their range; of requests that may bring a chunk three in four bring one token"""
    rng, n = random.Random(case.get("lens", 1)), case["requests"]
    lo, hi = case["new_lo"], case["new_hi"]
    if case["kind"] == "packed":
        return [_log(rng, lo, hi) for _ in range(n)], [0] * n
    new = [1 if hi > 1 and n > 1 and i % 4 else _log(rng, max(lo, min(hi, 17)), hi) for i in range(n)]
    return new, [_log(rng, case["held_lo"], case["held_hi"]) for _ in range(n)]


# ------------------------------------------------------------------ what a program has in hand
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _tables(dim):
    """cosines and sines of 20000 positions, rotate-half layout"""
    freq = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=DEVICE) / dim)
    a = torch.arange(20000, dtype=torch.float64, device=DEVICE)[:, None] * freq
    return torch.cat([a.cos(), a.cos()], -1).float(), torch.cat([a.sin(), a.sin()], -1).float()


def _cache(case, pages, g):
    """random contents: what earlier requests left in pages and rows that nobody holds is no zero either"""
    shape = (pages, case["page"], case["kv_heads"], case["dim"])
    x = torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float16)
    return x.to(torch.float8_e5m2).view(torch.uint8) if case["cache"] == "e5m2" else x.to(DTYPES[case["cache"]])


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    s = {"kind": kind, "case": case}
    if kind == "append":
        t, heads, kv, dim = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        pages = -(-t // case["page"]) + 3
        s["qkv"] = torch.randn(t, (heads + 2 * kv) * dim, generator=g, device=DEVICE).to(DTYPES[case["dtype"]])
        s["k_cache"], s["v_cache"] = _cache(case, pages, g), _cache(case, pages, g)
        s["cos"], s["sin"] = _tables(dim)
        s["positions"] = torch.randint(0, 20000 - t, (1,), generator=g, device=DEVICE) + torch.arange(t, device=DEVICE)
        order = torch.randperm(pages, generator=g, device=DEVICE)
        at = torch.arange(t, device=DEVICE)
        s["slots"] = order[at // case["page"]] * case["page"] + at % case["page"]
        return s
    new, held = _lengths(case)
    s["max_new"], s["max_len"], s["tokens"] = max(new), max(h + n for h, n in zip(held, new)), sum(new)
    if kind == "packed":
        width = (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        qkv = torch.randn(s["tokens"], width, generator=g, device=DEVICE).to(DTYPES[case["dtype"]])
        s["q"], s["k"], s["v"] = qkv.view(s["tokens"], -1, case["dim"]).split([case["heads"], case["kv_heads"], case["kv_heads"]], dim=1)
        s["cu"] = _ints([0] + new).cumsum(0, dtype=torch.int32)
        return s
    width = -(-max(s["max_len"], 1) // case["page"]) + 2
    had = [-(-h // case["page"]) for h in held]
    total = [-(-(h + n) // case["page"]) for h, n in zip(held, new)]
    if kind == "step":
        pages = sum(total) + 9
        order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
        table = torch.full((len(new), width), -1, dtype=torch.int32, device=DEVICE)
        cols = torch.arange(width, device=DEVICE)[None]
        table[cols < _ints(had)[:, None]] = order[:sum(had)]
        free = pages - sum(had)
        s["free_pages"] = torch.cat([order[sum(had):], torch.full((sum(had),), -1, dtype=torch.int32, device=DEVICE)])
        s["free_count"], s["table"], s["new"], s["held"] = _ints([free]), table, _ints(new), _ints(held)
        return s
    pages = sum(total) + 3
    order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((len(new), width), -1, dtype=torch.int32, device=DEVICE)
    table[torch.arange(width, device=DEVICE)[None] < _ints(total)[:, None]] = order[:sum(total)]
    s["table"], s["seq_lens"], s["cu"] = table, _ints([h + n for h, n in zip(held, new)]), _ints([0] + new).cumsum(0, dtype=torch.int32)
    s["k_cache"], s["v_cache"] = _cache(case, pages, g), _cache(case, pages, g)
    s["q"] = (1.5 * torch.randn(s["tokens"], case["heads"], case["dim"], generator=g, device=DEVICE)).to(DTYPES[case["dtype"]])
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _run_own(s)
    return {"step": _plain_step, "append": _plain_append, "paged": _plain_paged, "packed": _plain_packed}[s["kind"]](s)


def _values(cache):
    """e5m2 bytes as the numbers that they stand for"""
    return cache.view(torch.float8_e5m2) if cache.dtype == torch.uint8 else cache


def _run_own(s):
    from ipex_llm_b200.transformers import paged_kv
    case = s["case"]
    if s["kind"] == "step":
        st = paged_kv.paged_step(s["new"], s["held"], s["table"], s["free_pages"], s["free_count"], case["page"], s["tokens"])
        return {"table": s["table"], "cu": st.cu_seqlens, "seq_lens": st.seq_lens, "positions": st.positions, "slots": st.slots, "free": st.free_count, "missing": st.missing}
    if s["kind"] == "append":
        paged_kv.paged_rope_append(s["qkv"], case["heads"], case["kv_heads"], case["dim"], s["cos"], s["sin"], s["positions"], s["slots"], s["k_cache"], s["v_cache"])
        return {"qkv": s["qkv"], "k_cache": _values(s["k_cache"]), "v_cache": _values(s["v_cache"])}
    if s["kind"] == "paged":
        return paged_kv.sdp_paged(s["q"], s["k_cache"], s["v_cache"], s["table"], s["seq_lens"], s["cu"], case["dim"] ** -0.5, max_query_len=s["max_new"])
    return paged_kv.sdp_packed(s["q"], s["k"], s["v"], s["cu"], case["dim"] ** -0.5, max_seqlen=s["max_new"])


def _plain_step(s):
    page, new, held, table = s["case"]["page"], s["new"].long(), s["held"].long(), s["table"]
    had, want = (held + page - 1) // page, (held + new + page - 1) // page
    need = want - had
    before = need.cumsum(0) - need
    cols = torch.arange(table.shape[1], device=table.device)[None]
    index = before[:, None] + cols - had[:, None]                        # which of this step's new pages
    fresh = torch.where(index < s["free_count"], s["free_pages"][(s["free_count"] - 1 - index).clamp(0, s["free_pages"].numel() - 1)], -1)
    table.copy_(torch.where((cols >= had[:, None]) & (cols < want[:, None]), fresh, table))
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    at = torch.arange(s["tokens"], device=table.device)
    row = torch.searchsorted(cu[1:], at, right=True).clamp(max=new.numel() - 1)
    positions = held[row] + at - cu[row]
    held_by = table[row, positions // page].long()
    slots = torch.where(held_by >= 0, held_by * page + positions % page, -1)
    left = s["free_count"] - need.sum()
    return {"table": table, "cu": cu.int(), "seq_lens": (held + new).int(), "positions": positions, "slots": slots, "free": left.clamp(min=0).int(), "missing": (-left).clamp(min=0).int()}


def _to_cache(x, cache):
    """values in the cache's form: e5m2 saturates at its largest number"""
    return x.float().clamp(-57344, 57344).to(torch.float8_e5m2).view(torch.uint8) if cache.dtype == torch.uint8 else x


def _plain_append(s):
    case, qkv = s["case"], s["qkv"]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    x = qkv.view(-1, heads + 2 * kv, dim)
    turned = x[:, :heads + kv].float()
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    half = torch.cat([-turned[..., dim // 2:], turned[..., :dim // 2]], -1)
    x[:, :heads + kv] = (turned * cos + half * sin).to(x.dtype)
    s["k_cache"].view(-1, kv, dim)[s["slots"]] = _to_cache(x[:, heads:heads + kv], s["k_cache"])
    s["v_cache"].view(-1, kv, dim)[s["slots"]] = _to_cache(x[:, heads + kv:], s["v_cache"])
    return {"qkv": qkv, "k_cache": _values(s["k_cache"]), "v_cache": _values(s["v_cache"])}


def _attend(q, k, v, cu, lens, max_new, scale):
    """q [T, H, D] by request -> [R, n, H, D]; k, v [R, L, G, D] in 32 bits; request r's i-th of n_r tokens sees the keys up to len_r - n_r + i"""
    cu = cu.long()
    new = cu[1:] - cu[:-1]
    i = torch.arange(max_new, device=q.device)
    at = cu[:-1, None] + i[None]
    group = q.shape[1] // k.shape[2]
    rows = q[at.clamp(max=q.shape[0] - 1)].float().unflatten(2, (k.shape[2], group)).permute(0, 2, 3, 1, 4)        # [R, G, H / G, n, D]
    scores = (rows.flatten(2, 3) @ k.permute(0, 2, 3, 1)).unflatten(2, (group, max_new))
    scores *= scale
    sees = torch.arange(k.shape[1], device=q.device) <= (lens.long() - new)[:, None, None] + i[:, None]
    scores.masked_fill_(~sees[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores.flatten(2, 3) @ v.permute(0, 2, 1, 3)).unflatten(2, (group, max_new)) / total
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3)[i[None] < new[:, None]].to(q.dtype)


def _plain_paged(s):
    page = s["case"]["page"]
    table = s["table"][:, :-(-s["max_len"] // page)].long().clamp(min=0)
    k, v = (_values(s[n])[table].flatten(1, 2).float() for n in ("k_cache", "v_cache"))
    # rows that a request does not hold are whatever was there: they must not reach a product
    held = (torch.arange(k.shape[1], device=k.device) < s["seq_lens"][:, None])[..., None, None]
    return _attend(s["q"], torch.where(held, k, 0.0), torch.where(held, v, 0.0), s["cu"], s["seq_lens"], s["max_new"], s["case"]["dim"] ** -0.5)


def _plain_packed(s):
    cu = s["cu"].long()
    new = cu[1:] - cu[:-1]
    i = torch.arange(s["max_new"], device=cu.device)
    at = (cu[:-1, None] + i).clamp(max=s["tokens"] - 1)
    held = (i < new[:, None])[..., None, None]
    k, v = (torch.where(held, s[n][at].float(), 0.0) for n in ("k", "v"))
    return _attend(s["q"], k, v, s["cu"], new, s["max_new"], s["case"]["dim"] ** -0.5)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind, dim = case["kind"], case.get("dim", 0)
    if kind == "append":
        t, heads, kv = case["tokens"], case["heads"], case["kv_heads"]
        kept = 1 if case["cache"] == "e5m2" else 2
        moved = 2 * (heads + 2 * kv) + 2 * (heads + kv) + 2 * kv * kept            # the projection in, its queries and keys out, both caches
        return {"bytes": t * (dim * moved + 4 * dim + 16), "flops": 3 * t * (heads + kv) * dim}
    new, held = _lengths(case)
    if kind == "step":
        pages = sum(-(-(h + n) // case["page"]) - -(-h // case["page"]) for h, n in zip(held, new))
        return {"bytes": 20 * len(new) + 8 * pages + 16 * sum(new), "flops": 4 * sum(new)}
    heads, kv = case["heads"], case["kv_heads"]
    seen = sum(n * h + n * (n + 1) // 2 for h, n in zip(held, new))
    size = 1 if case.get("cache") == "e5m2" else 2
    keys = sum(h + n for h, n in zip(held, new))
    return {"bytes": 4 * sum(new) * heads * dim + 2 * keys * kv * dim * size, "flops": 4 * seen * heads * dim}


# ------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    if case["kind"] == "step":
        return None                                       # whole numbers: there is nothing to round
    s = prepare(case, seed)
    if case["kind"] == "append":
        x = s["qkv"].double().view(case["tokens"], -1, case["dim"])
        angle = s["positions"].double()[:, None, None] * torch.exp2(-math.log2(10000.0) * 2 / case["dim"] * torch.arange(case["dim"] // 2, device=DEVICE, dtype=torch.float64))
        n = case["heads"] + case["kv_heads"]
        z = torch.polar(torch.ones_like(angle), angle) * torch.complex(x[:, :n, :case["dim"] // 2].contiguous(), x[:, :n, case["dim"] // 2:].contiguous())
        x = torch.cat([torch.cat([z.real, z.imag], -1), x[:, n:]], 1)
        out = {"qkv": x.reshape(case["tokens"], -1)}
        for name, first in (("k_cache", case["heads"]), ("v_cache", n)):
            rows = x[:, first:first + case["kv_heads"]]
            if case["cache"] == "e5m2":                   # the bytes hold the rounded activations' nearest e5m2 values
                rows = rows.to(DTYPES[case["dtype"]]).to(torch.float8_e5m2).double()
            whole = _values(s[name]).double()
            whole.view(-1, case["kv_heads"], case["dim"])[s["slots"]] = rows
            out[name] = whole
        return out
    new, held = _lengths(case)
    out, first = torch.empty(s["tokens"], case["heads"], case["dim"], dtype=torch.float64, device=DEVICE), 0
    group = case["heads"] // case["kv_heads"]
    for r, (n, h) in enumerate(zip(new, held)):
        if case["kind"] == "packed":
            keys, values = s["k"][first:first + n], s["v"][first:first + n]
        else:
            pages = s["table"][r, :-(-(h + n) // case["page"])].long()
            keys, values = (_values(s[name])[pages].flatten(0, 1)[:h + n] for name in ("k_cache", "v_cache"))
        for head in range(case["heads"]):
            score = s["q"][first:first + n, head].double() @ keys[:, head // group].double().T / math.sqrt(case["dim"])
            score = score.masked_fill(torch.ones_like(score, dtype=torch.bool).triu(h + 1), -math.inf)
            out[first:first + n, head] = torch.softmax(score, -1) @ values[:, head // group].double()
        first += n
    return out
