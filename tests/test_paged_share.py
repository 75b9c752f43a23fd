"""Pages that several rows share (transformers/paged_kv.py): forks, releases, copies and moves against whole numbers computed here one after the other, the
norms in front of the rotation against 64 bits, and a server that uses them with everything else that a step has."""
import ctypes
import math
import random

import pytest
import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def paged(native_lib):
    from ipex_llm_b200.transformers import paged_kv
    return paged_kv


def dev_ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------ forks
def fork_statement(parents, children, lens, table, stack, shared, page):
    table, stack, shared, lens, src, dst, missing = [list(r) for r in table], list(stack), list(shared), list(lens), [], [], 0
    R, width = len(table), len(table[0])
    for p, c in zip(parents, children):
        if not (0 <= p < R and 0 <= c < R) or p == c:
            src.append(-1)
            dst.append(-1)
            continue
        held = max(lens[p], 0)
        full = min(held // page, width)
        row = table[p][:full]
        for pg in row:
            if 0 <= pg < len(shared):
                shared[pg] += 1
        if held % page and held // page < width:
            src.append(table[p][full])
            dst.append(stack.pop() if stack else -1)
            missing += dst[-1] < 0
            row = row + [dst[-1]]
        else:
            src.append(-1)
            dst.append(-1)
        table[c] = row + [-1] * (width - len(row))
        lens[c] = lens[p]
    return table, lens, shared, src, dst, len(stack), missing


def fill(held, page, width, pages, rng, rows):
    order = list(range(pages))
    rng.shuffle(order)
    table = []
    for h in held:
        row = [order.pop() for _ in range(min(-(-h // page), width))]
        table.append(row + [-1] * (width - len(row)))
    return table + [[rng.choice((-1, 7)) for _ in range(width)] for _ in range(rows - len(held))], order


def check_fork(paged, dev, held, parents, children, page, width, rows, spare=None, in_place=False, pad=0):
    rng = random.Random(len(parents) * 100 + page)
    pages = sum(-(-h // page) for h in held) + len(parents) + 3
    table, stack = fill(held, page, width, pages, rng, rows)
    if spare is not None:
        stack = stack[:spare]
    lens = held + [rng.randrange(5) for _ in range(rows - len(held))]
    shared = [rng.randrange(3) for _ in range(pages)]
    want = fork_statement(parents, children, lens, table, stack, shared, page)
    wide = torch.full((rows, width + pad), 99, dtype=torch.int32, device=dev)
    t = wide[:, :width]
    t.copy_(dev_ints(table, dev))
    free, count, sh, ln = dev_ints(stack + [-1] * (pages - len(stack)), dev), dev_ints([len(stack)], dev), dev_ints(shared, dev), dev_ints(lens, dev)
    before = free.clone()
    got = paged.paged_fork(dev_ints(parents, dev), dev_ints(children, dev), ln, t, free, count, sh, page, free_left=count if in_place else None)
    assert t.tolist() == want[0] and ln.tolist() == want[1] and sh.tolist() == want[2] and got.src.tolist() == want[3] and got.dst.tolist() == want[4]
    assert got.free_count.tolist() == [want[5]] and got.missing.tolist() == [want[6]] and torch.equal(free, before)
    assert count.tolist() == [want[5] if in_place else len(stack)] and bool((wide[:, width:] == 99).all())


FORKS = [([5], [0], [1], 4, 3, 2), ([8], [0], [1], 4, 3, 2), ([0, 7], [0, 1, 1, 1], [2, 3, 4, 5], 4, 3, 6), ([16, 3, 33], [2, 0, 2, 1, 2], [9, 3, 4, 8, 5], 16, 5, 10),
         ([9, 4], [0, -1, 1, 2, 5, 1], [2, 3, 1, 7, 4, 3], 4, 3, 5), ([50], [0, 0], [2, 1], 8, 4, 3), ([7], [0], [1], 1, 7, 2), ([40], [0], [1], 8, 5, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("held,parents,children,page,width,rows", FORKS)
@pytest.mark.parametrize("in_place,pad", [(False, 0), (True, 5)])
def test_fork(paged, cuda_device, held, parents, children, page, width, rows, in_place, pad):
    check_fork(paged, cuda_device, held, parents, children, page, width, rows, in_place=in_place, pad=pad)


@pytest.mark.gpu
@pytest.mark.parametrize("spare", [0, 1, 2])
def test_forks_without_enough_pages(paged, cuda_device, spare):
    check_fork(paged, cuda_device, [5, 9, 8], [0, 1, 2, 0, 1], [3, 4, 5, 6, 7], 4, 4, 8, spare=spare)


@pytest.mark.gpu
@pytest.mark.parametrize("requests,forks,width,page", [(3, 40, 300, 16), (100, 300, 60, 8), (200, 1024, 9, 4), (50, 1500, 33, 32), (1, 2100, 5, 4), (2, 3, 20000, 1)])
def test_many_forks(paged, cuda_device, requests, forks, width, page):
    rng = random.Random(forks)
    held = [rng.randrange(width * page + 1) for _ in range(requests)]
    children = list(range(requests, requests + forks))
    rng.shuffle(children)
    check_fork(paged, cuda_device, held, [rng.randrange(requests) for _ in range(forks)], children, page, width, requests + forks)


@pytest.mark.gpu
def test_no_forks(paged, cuda_device):
    i = lambda x: dev_ints(x, cuda_device)                                                        # noqa: E731
    got = paged.paged_fork(i([]), i([]), i([3]), i([[1, -1]]), i([0, 2]), i([2]), i([0, 0]), 4)
    assert got.src.numel() == 0 and got.free_count.tolist() == [2] and got.missing.tolist() == [0]


# ------------------------------------------------------------------ releases
def release_statement(done, table, stack, shared, pages, first_col):
    """(table, stack, shared): a page goes back in the place of the entry that names it first"""
    table, stack, shared, times, order = [list(r) for r in table], list(stack), list(shared), {}, []
    for r, row in enumerate(table):
        if not done[r]:
            continue
        for c in range(first_col[r], len(row)):
            if 0 <= row[c] < pages:
                times[row[c]] = times.get(row[c], 0) + 1
                if times[row[c]] == 1:
                    order.append(row[c])
            row[c] = -1
    for p in order:
        if times[p] > shared[p]:
            stack.append(p)
        shared[p] = max(shared[p] - times[p], 0)
    return table, stack[:pages], shared


def check_release(paged, dev, done, table, stack, shared, pages, held=None, page=None):
    width = len(table[0])
    want = release_statement(done, table, stack, shared, pages, [0 if held is None else min(-(-max(h, 0) // page), width) for h in held or done])
    t, free, count, sh = dev_ints(table, dev), dev_ints(stack + [-1] * (pages - len(stack)), dev), dev_ints([len(stack)], dev), dev_ints(shared, dev)
    more = {} if held is None else {"held": dev_ints(held, dev), "page_size": page}
    paged.paged_release(torch.tensor(done, dtype=torch.bool, device=dev), t, free, count, shared=sh, **more)
    n = int(count)
    assert n == len(want[1]) and free[:n].tolist() == want[1] and t.tolist() == want[0] and sh.tolist() == want[2]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,pages", [(1, 1, 1), (2, 3, 9), (7, 40, 60), (64, 33, 400), (40, 300, 2000), (1100, 9, 3000), (5, 5000, 9000), (9, 1000, 20000)])
@pytest.mark.parametrize("what", ["all", "some", "none", "behind"])
def test_release_of_shared_pages(paged, cuda_device, rows, width, pages, what):
    """rows that share beginnings, entries that are no page, rows that name a page twice"""
    rng = random.Random(rows * width)
    order = list(range(pages))
    rng.shuffle(order)
    table, owners = [], [0] * pages
    for r in range(rows):
        if table and rng.random() < 0.6:                               # a fork: the beginning of an earlier row
            old = rng.choice(table)
            n = rng.randrange(width + 1)
            row = old[:n] + [-1] * (width - n)
        else:
            n = min(rng.randrange(width + 1), len(order))
            row = [order.pop() for _ in range(n)] + [-1] * (width - n)
        if rng.random() < 0.1:
            row[rng.randrange(width)] = rng.choice((-5, pages, pages + 3))
        for p in set(row):
            if 0 <= p < pages:
                owners[p] += 1
        table.append(row)
    shared = [max(n - 1, 0) for n in owners]
    done = [{"all": True, "none": False}.get(what, rng.random() < 0.6) for _ in range(rows)]
    held = [rng.randrange(-1, 4 * width + 9) for _ in range(rows)] if what == "behind" else None
    check_release(paged, cuda_device, done, table, order, shared, pages, held, 4)


@pytest.mark.gpu
def test_release_of_counts_that_are_too_small(paged, cuda_device):
    """more rows name a page than the counts say: it goes back once, and the stack never takes more than it holds"""
    check_release(paged, cuda_device, [True] * 4, [[1, 2], [1, 2], [1, 0], [1, 1]], [], [0, 1, 5], 3)
    check_release(paged, cuda_device, [True] * 2, [[0, 1, 2], [2, 1, 0]], [0, 1], [0, 0, 0], 3)


# ------------------------------------------------------------------ moves
def compact_statement(table, stack, shared, pages):
    used = {p for row in table for p in row if 0 <= p < pages}
    free = sorted({p for p in stack if 0 <= p < pages} - used)
    high = sorted(used, reverse=True)
    moves = [(u, f) for u, f in zip(high, free) if f < u]
    to, shared = dict(moves), list(shared)
    for u, f in moves:
        shared[f], shared[u] = shared[u], 0
    left = sorted((set(free) - {f for _, f in moves}) | {u for u, _ in moves}, reverse=True)
    return [[to.get(p, p) for p in row] for row in table], left, shared, moves


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,pages,density", [(1, 1, 1, 1.0), (1, 3, 8, 0.5), (6, 10, 100, 0.5), (40, 30, 1500, 0.7), (300, 40, 9000, 0.9), (3, 7000, 30000, 0.6), (9, 9, 500, 0.0)])
@pytest.mark.parametrize("reserved", [0, 3])
@pytest.mark.parametrize("with_shared", [True, False])
def test_compact(paged, cuda_device, rows, width, pages, density, reserved, with_shared):
    rng = random.Random(pages + reserved)
    order = list(range(pages))
    rng.shuffle(order)
    kept = [order.pop() for _ in range(min(reserved, pages - 1))]
    table = []
    for r in range(rows):
        if table and rng.random() < 0.3:
            row = list(rng.choice(table))
        else:
            n = min(int(width * density * rng.random() + 0.5), len(order))
            row = [order.pop() for _ in range(n)] + [-1] * (width - n)
        table.append(row)
    if rows > 3:
        table[2][width - 1] = pages + 4                                # no page: it stays what it is
    owners = [0] * pages
    for row in table:
        for p in row:
            if 0 <= p < pages:
                owners[p] += 1
    shared = [max(n - 1, 0) for n in owners]
    for p in kept:
        shared[p] = 5
    want = compact_statement(table, order, shared, pages)
    wide = torch.full((rows, width + 3), 99, dtype=torch.int32, device=cuda_device)
    wide[:, :width] = dev_ints(table, cuda_device)
    t, free, count, sh = wide[:, :width], dev_ints(order + [-1] * (pages - len(order)), cuda_device), dev_ints([len(order)], cuda_device), dev_ints(shared, cuda_device)
    keep = [x.clone() for x in (t, free, count, sh)]
    got = paged.paged_compact(t, free, count, sh if with_shared else None)
    assert all(torch.equal(a, b) for a, b in zip(keep, (t, free, count, sh)))
    m = len(want[3])
    assert got.block_table.tolist() == want[0] and got.free_count.tolist() == [len(want[1])]
    assert got.free_pages.tolist() == want[1] + [-1] * (pages - len(want[1]))
    assert got.src.tolist() == [u for u, _ in want[3]] + [-1] * (pages - m) and got.dst.tolist() == [f for _, f in want[3]] + [-1] * (pages - m)
    assert (got.shared.tolist() == want[2]) if with_shared else got.shared is None
    again = paged.paged_compact(got.block_table, got.free_pages, got.free_count, got.shared)
    assert not bool((again.src >= 0).any()) and torch.equal(again.block_table, got.block_table) and torch.equal(again.free_pages, got.free_pages)


# ------------------------------------------------------------------ copies
def layouts(dev):
    g = torch.Generator(device=dev).manual_seed(3)
    r = lambda *s: torch.randint(0, 255, s, generator=g, device=dev, dtype=torch.uint8)           # noqa: E731
    half = lambda *s: r(*s[:-1], 2 * s[-1]).view(torch.float16)                                   # noqa: E731
    return {"plain": [half(20, 16, 4, 64) for _ in range(6)], "bytes": [r(20, 16, 2, 96) for _ in range(3)], "heads first": [half(20, 4, 16, 64).transpose(1, 2) for _ in range(2)],
            "keys and values in one": list(half(20, 2, 8, 2, 32).unbind(1)), "odd pages": [half(20, 3, 1, 7) for _ in range(2)] + [r(20, 5, 3)], "off 16 bytes": [half(20 * 64 + 8)[1:1 + 20 * 64].view(20, 4, 2, 8)],
            "mixed": [half(20, 8, 2, 64), r(20, 8, 2, 64), half(30, 8, 2, 64), r(20, 2000)], "many": [half(20, 4, 1, 16) for _ in range(300)], "large": [half(20, 128, 8, 128)],
            "one page": [half(1, 4, 4)]}


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["plain", "bytes", "heads first", "keys and values in one", "odd pages", "off 16 bytes", "mixed", "many", "large", "one page"])
def test_copies(paged, cuda_device, name):
    caches = layouts(cuda_device)[name]
    src, dst = [3, -1, 7, 3, 0, 25, 2, 19, 18], [1, 4, -1, 5, 6, 8, 60, 17, 9]
    want = [c.clone() for c in caches]
    for w in want:
        for a, b in zip(src, dst):
            if 0 <= a < len(w) and 0 <= b < len(w):
                w[b] = w[a]
    paged.paged_copy(dev_ints(src, cuda_device), dev_ints(dst, cuda_device), caches)
    assert all(torch.equal(c.contiguous().view(torch.uint8), w.contiguous().view(torch.uint8)) for c, w in zip(caches, want))


@pytest.mark.gpu
def test_copies_of_nothing(paged, cuda_device):
    c = torch.zeros(3, 4, device=cuda_device)
    paged.paged_copy(dev_ints([], cuda_device), dev_ints([], cuda_device), [c])
    paged.paged_copy(dev_ints([1], cuda_device), dev_ints([2], cuda_device), [])


@pytest.mark.gpu
def test_copies_beyond_32_bits(paged, cuda_device):
    c = torch.empty(70000, 16, 8, 128, dtype=torch.float16, device=cuda_device).view(torch.int16)
    c[69999], c[3] = 7, 9
    paged.paged_copy(dev_ints([69999, 3], cuda_device), dev_ints([2, 69998], cuda_device), [c])
    assert bool((c[2] == 7).all()) and bool((c[69998] == 9).all()) and bool((c[3] == 9).all())


# ------------------------------------------------------------------ norms and rotation
def rotated(x, cos, sin):
    half = cos.shape[-1] // 2
    y = x.clone()
    y[..., :half] = x[..., :half] * cos[:, None, :half].double() - x[..., half:2 * half] * sin[:, None, :half].double()
    y[..., half:2 * half] = x[..., half:2 * half] * cos[:, None, :half].double() + x[..., :half] * sin[:, None, :half].double()
    return y


def tables(dim, n, dev, dtype):
    a = torch.arange(n, dtype=torch.float64, device=dev)[:, None] * 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=dev) / dim)
    return torch.cat([a.cos(), a.cos()], -1).to(dtype), torch.cat([a.sin(), a.sin()], -1).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cached", ["e5m2", "same", None])
@pytest.mark.parametrize("T,heads,kv_heads,dim,rotary,table_type,w_type", [
    (1, 32, 8, 128, 128, "f32", "same"), (7, 4, 2, 64, 64, "same", "f32"), (300, 14, 2, 96, 32, "f32", "same"), (33, 8, 1, 256, 256, "same", "same"), (65, 3, 3, 80, 80, "f32", "f32"),
    (20, 2, 1, 48, 6, "same", "same"), (40, 0, 2, 64, 64, "f32", "same"), (130, 8, 4, 128, 0, "f32", "same"), (5, 3, 1, 17, 10, "f32", "f32"), (9, 2, 2, 272, 272, "same", "same"),
    (2000, 4, 4, 16, 16, "f32", "same"), (11, 5, 1, 224, 96, "f32", "f32")])
def test_norm_and_append(paged, cuda_device, dtype, cached, T, heads, kv_heads, dim, rotary, table_type, w_type):
    g = torch.Generator(device=cuda_device).manual_seed(T)
    page, width, eps = 8, (heads + 2 * kv_heads) * dim, 1e-5
    pages, n = T // page + 3, heads + kv_heads
    whole = torch.randn(T, width + 16, generator=g, device=cuda_device)
    whole[:, :width] *= torch.exp2(6 * torch.randn(T, heads + 2 * kv_heads, 1, generator=g, device=cuda_device)).clamp(2.0 ** -12, 2.0 ** 10).expand(-1, -1, dim).reshape(T, width)
    whole = whole.to(dtype)
    qkv = whole[:, :width]
    qkv[0, :dim] = 0.0                                                 # a head of zeros
    before = whole.clone()
    w_dtype = torch.float32 if w_type == "f32" else dtype
    qw, kw = ((1 + torch.randn(dim, generator=g, device=cuda_device)).to(w_dtype) for _ in range(2))
    caches = [None, None]
    if cached:
        caches = [torch.randn(pages, kv_heads, page, dim, generator=g, device=cuda_device).to(dtype).transpose(1, 2) for _ in range(2)]
        if cached == "e5m2":
            caches = [c.to(torch.float8_e5m2).view(torch.uint8) for c in caches]
    held = [c.clone() if cached else None for c in caches]
    slots = torch.randperm(pages * page, generator=g, device=cuda_device)[:T]
    if T > 30:
        slots[5], slots[6] = pages * page, -1
    positions = torch.randint(0, 500, (T,), generator=g, device=cuda_device)
    positions[-1] = 10 ** 10                                           # beyond the tables: the last row
    cos, sin = tables(max(rotary, 2), 500, cuda_device, torch.float32 if table_type == "f32" else dtype)
    paged.paged_norm_rope_append(qkv, heads, kv_heads, dim, qw, kw, eps, *((cos, sin) if rotary else (None, None)), positions if rotary else None, slots if cached else None, *caches)
    x = before[:, :width].double().view(T, heads + 2 * kv_heads, dim)[:, :n]
    weight = torch.cat([qw.double().expand(heads, dim), kw.double().expand(kv_heads, dim)])
    y = x * weight / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    at = positions.clamp(max=499)
    want = rotated(y, cos[at], sin[at]) if rotary else y
    # squares: dim additions at most, halved by the root; the root 2^-22; three products and the sum of two
    size = rotated(y.abs(), cos[at].abs(), -sin[at].abs()).abs() + y.abs() if rotary else y.abs()
    got = qkv.double().view(T, -1, dim)[:, :n]
    low = 2.0 ** -25 if dtype == torch.float16 else 0.0                # half a step of fp16's smallest numbers
    assert bool(((got - want).abs() <= HALF[dtype] * want.abs() + (2.0 ** -21 + 2.0 ** -25 * (dim / 8 + 8)) * 2 * size + low).all())
    assert not bool(got[0, 0].any())
    assert torch.equal(whole[:, width:], before[:, width:]) and torch.equal(qkv[:, n * dim:], before[:, n * dim:width])
    if not cached:
        return
    now = qkv.reshape(T, -1, dim)
    for cache, old, rows in zip(caches, held, (now[:, heads:n], now[:, n:])):
        flat, was = cache.reshape(pages * page, kv_heads, dim), old.reshape(pages * page, kv_heads, dim).clone()
        ok = (slots >= 0) & (slots < pages * page)
        was[slots[ok]] = rows[ok].float().clamp(-57344, 57344).to(torch.float8_e5m2).view(torch.uint8) if cached == "e5m2" else rows[ok]
        assert torch.equal(flat.view(torch.uint8), was.view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 68])
def test_norms_of_heads_that_are_not_finite_stay_there(paged, cuda_device, dim):
    x = torch.ones(3, 4 * dim, dtype=torch.bfloat16, device=cuda_device)
    x[1, dim + 3], x[1, 2 * dim + 1] = math.nan, math.inf
    w = torch.ones(dim, device=cuda_device)
    paged.paged_norm_rope_append(x, 2, 1, dim, w, w, 0.0, None, None, None, None, None, None)
    x = x.view(3, 4, dim).float()
    assert bool(torch.isnan(x[1, 1]).all()) and bool((x[1, 2, 2:] == 0).all()) and bool((x[[0, 2]] == 1).all()) and bool((x[1, [0, 3]] == 1).all())


# ------------------------------------------------------------------ together
def serve(paged, dev, dtype, eight, forked):
    """a server's steps with everything that they have beside the attention: prompts, then samples of them that go on by themselves -- as forks, or (``forked``
    false) as requests that bring the prompt once more -- then some that end, and the cache moved together.  Returns what every sample said"""
    from ipex_llm_b200.transformers.logprobs import token_logprobs
    from ipex_llm_b200.transformers.lora import lora_add_
    H, G, D, K, page, pages, V, R, layers = 4, 2, 64, 128, 8, 120, 300, 8, 2
    g = torch.Generator(device=dev).manual_seed(11)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)                                       # noqa: E731
    W = [(r((H + 2 * G) * D, K) * K ** -0.5).to(dtype) for _ in range(layers)]
    O = [(r(K, H * D) * (H * D) ** -0.5).to(dtype) for _ in range(layers)]                        # noqa: E741
    A, B = (r(3, 3, 16, K) * K ** -0.5).to(dtype), (r(3, (H + 2 * G) * D, 16) * 0.2).to(dtype)
    scales, qw, kw = torch.tensor([0.5, 1.0, 2.0], device=dev), 1 + 0.2 * r(D), 1 + 0.2 * r(D)
    emb, head = r(V, K).to(dtype), (r(V, K) * K ** -0.5).to(dtype)
    cos, sin = tables(D, 200, dev, torch.float32)
    caches = [[torch.zeros(pages, page, G, D, dtype=torch.uint8 if eight else dtype, device=dev) for _ in range(2)] for _ in range(layers)]
    table, stack = torch.full((R, 12), -1, dtype=torch.int32, device=dev), torch.randperm(pages, generator=g, device=dev).int()
    count, shared, held = dev_ints([pages], dev), torch.zeros(pages, dtype=torch.int32, device=dev), torch.zeros(R, dtype=torch.int32, device=dev)
    ids = dev_ints([0, -1, 0, 0, -1, 2, 1, 1], dev)                    # row 2, 3 sample row 0's prompt, row 4 row 1's

    def step(tokens, new):
        nonlocal held
        st = paged.paged_step(dev_ints(new, dev), held, table, stack, count, page, len(tokens), free_left=count)
        assert st.missing.item() == 0
        x = emb[torch.tensor(tokens, device=dev)]
        for (kc, vc), w, o in zip(caches, W, O):
            qkv = torch.cat([x[i:i + 1] @ w.T for i in range(len(tokens))])                       # a row at a time: the same whatever lies beside it
            lora_add_(qkv, x, A, B, scales, ids, st.cu_seqlens, splits=[H * D, G * D, G * D])
            paged.paged_norm_rope_append(qkv, H, G, D, qw, kw, 1e-6, cos, sin, st.positions, st.slots, kc, vc)
            y = paged.sdp_paged(qkv[:, :H * D].view(-1, H, D), kc, vc, table, st.seq_lens, st.cu_seqlens)
            x = x + torch.cat([y[i].reshape(1, -1) @ o.T for i in range(len(tokens))])
        held = st.seq_lens
        return torch.cat([x[i:i + 1] @ head.T for i in range(len(tokens))]), st.cu_seqlens.tolist()
    prompts = {0: [5, 9, 2, 7, 1, 8, 3, 3, 6, 4, 11], 1: list(range(20, 36))}                     # 11 tokens: a page and a part; 16: two pages
    said = {}
    if forked:
        step(prompts[0] + prompts[1], [11, 16, 0, 0, 0, 0, 0, 0])
        f = paged.paged_fork(dev_ints([0, 0, 1], dev), dev_ints([2, 3, 4], dev), held, table, stack, count, shared, page, free_left=count)
        assert f.missing.item() == 0 and (f.dst >= 0).tolist() == [True, True, False]
        paged.paged_copy(f.src, f.dst, [c for pair in caches for c in pair])
    else:
        step(prompts[0] + prompts[1] + prompts[0] * 2 + prompts[1], [11, 16, 11, 11, 16, 0, 0, 0])
    last = {0: [4], 1: [17], 2: [41], 3: [250], 4: [90]}
    for turn in range(12):
        rows = sorted(last)
        logits, cu = step([t for r_ in rows for t in last[r_]], [len(last.get(r_, [])) for r_ in range(R)])
        got = token_logprobs(logits, torch.tensor([7 + r_ for r_ in rows], device=dev), 3)
        for n, r_ in enumerate(rows):
            said.setdefault(r_, []).append((got.logprobs[n].item(), got.entropy[n].item(), got.top_ids[n].tolist()))
            last[r_] = [got.top_ids[n, turn % 2].item()]
        if turn == 4:
            done = torch.zeros(R, dtype=torch.bool, device=dev)
            done[[0, 3]] = True                                        # the parent goes, one sample of it stays
            paged.paged_release(done, table, stack, count, shared=shared)
            held = held.masked_fill(done, 0)
            del last[0], last[3]
        if turn == 7:
            c = paged.paged_compact(table, stack, count, shared)
            paged.paged_copy(c.src, c.dst, [x for pair in caches for x in pair])
            table.copy_(c.block_table), stack.copy_(c.free_pages), count.copy_(c.free_count), shared.copy_(c.shared)
            used = table[table >= 0]
            assert int(used.max()) < used.unique().numel() == pages - count.item()
    paged.paged_release(torch.ones(R, dtype=torch.bool, device=dev), table, stack, count, shared=shared)
    assert count.tolist() == [pages] and sorted(stack.tolist()) == list(range(pages)) and not bool(shared.any()) and bool((table == -1).all())
    return said


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,eight", [(torch.bfloat16, False), (torch.float16, True)])
def test_a_server_with_shared_pages(paged, cuda_device, dtype, eight):
    """samples that share their prompt's pages say what samples with a prompt of their own say.  The prompts of the two runs lie in other tiles and are summed in
    another order, so single results may differ by roundings: a log probability by the 0.15 that a dozen roundings of 2^-8 of logits of up to 3 can add up to"""
    a, b = (serve(paged, cuda_device, dtype, eight, f) for f in (True, False))
    assert a.keys() == b.keys()
    for r in a:
        for (lp, h, ids), (lp2, h2, ids2) in zip(a[r], b[r]):
            assert abs(lp - lp2) < 0.15 and abs(h - h2) < 0.15
            if ids != ids2:                                            # two alternatives that are that near change places: the texts part
                break


@pytest.mark.gpu
def test_recorded_forks_and_releases(paged, cuda_device):
    dev, page, width, R, pages = cuda_device, 4, 6, 8, 60
    i = lambda x: dev_ints(x, dev)                                                                # noqa: E731
    table, stack, count, shared, lens = torch.full((R, width), -1, dtype=torch.int32, device=dev), torch.arange(pages, dtype=torch.int32, device=dev), i([pages]), \
        torch.zeros(pages, dtype=torch.int32, device=dev), torch.zeros(R, dtype=torch.int32, device=dev)
    cache = torch.arange(pages * 64, device=dev, dtype=torch.float16).view(pages, page, 1, 16)
    parents, children, done = i([0, 0, 1]), i([4, 5, 6]), torch.zeros(R, dtype=torch.bool, device=dev)

    def cycle():
        f = paged.paged_fork(parents, children, lens, table, stack, count, shared, page, free_left=count)
        paged.paged_copy(f.src, f.dst, [cache])
        paged.paged_release(done, table, stack, count, shared=shared)
        c = paged.paged_compact(table, stack, count, shared)
        return (*f, *c)
    cycle()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    state = (table, stack, count, shared, lens, cache)
    with torch.cuda.graph(graph):
        out = cycle()
    for held, gone in (([9, 4, 0, 0], [4]), ([3, 20, 7, 0], [0, 6, 5])):
        table.fill_(-1), shared.zero_(), stack.copy_(torch.arange(pages, dtype=torch.int32)), count.fill_(pages), done.zero_()
        paged.paged_step(i(held + [0] * 4), torch.zeros_like(lens), table, stack, count, page, sum(held), free_left=count)
        lens.copy_(i(held + [0] * 4))
        done[gone] = True
        start = [x.clone() for x in state]
        graph.replay()
        first = [x.clone() for x in (*state, *out)]
        for x, y in zip(state, start):
            x.copy_(y)
        again = cycle()
        assert all(torch.equal(a, b) for a, b in zip(first, (*state, *again)))


@pytest.mark.gpu
def test_on_other_streams_at_once(paged, cuda_device):
    """releases and moves keep their scratch to themselves"""
    rng = random.Random(1)
    pages, rows, width = 5000, 100, 40
    jobs = []
    for _ in range(6):
        table, stack = fill([rng.randrange(width * 4) for _ in range(rows)], 4, width, pages, rng, rows)
        done = [rng.random() < 0.5 for _ in range(rows)]
        want = release_statement(done, table, stack, [0] * pages, pages, [0] * rows)
        jobs.append((done, want, compact_statement(want[0], want[1], [0] * pages, pages), dev_ints(table, cuda_device), dev_ints(stack + [-1] * (pages - len(stack)), cuda_device),
                     dev_ints([len(stack)], cuda_device), torch.zeros(pages, dtype=torch.int32, device=cuda_device), torch.tensor(done, device=cuda_device)))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for n, (_, _, _, table, stack, count, shared, done) in enumerate(jobs):
        with torch.cuda.stream(streams[n % 3]):
            paged.paged_release(done, table, stack, count, shared=shared)
            got.append(paged.paged_compact(table, stack, count, shared))
    torch.cuda.synchronize()
    for (_, want, moved, table, stack, count, _, _), c in zip(jobs, got):
        assert table.tolist() == want[0] and stack[:len(want[1])].tolist() == want[1] and c.block_table.tolist() == moved[0] and c.src[:len(moved[3])].tolist() == [u for u, _ in moved[3]]


@pytest.mark.gpu
def test_the_python_statements_say_the_same(paged, cuda_device, monkeypatch):
    """what serves where the native host side is not to be had"""
    dev, page, width, R, pages = cuda_device, 4, 6, 8, 60
    i = lambda x: dev_ints(x, dev)                                                                # noqa: E731
    results = []
    for native in (True, False):
        if not native:
            monkeypatch.setattr(paged, "_native", lambda *args: None)
        for in_place in (False, True):
            table, stack, count = torch.full((R, width + 3), -1, dtype=torch.int32, device=dev)[:, :width], torch.arange(pages, dtype=torch.int32, device=dev), i([pages])
            shared, held = torch.zeros(pages, dtype=torch.int32, device=dev), i([9, 4, 23, 0, 0, 0, 0, 0])
            st = paged.paged_step(held, torch.zeros_like(held), table, stack, count, page, 36, free_left=count)
            g = torch.Generator(device=dev).manual_seed(5)
            caches = [torch.zeros(pages, page, 2, 64, dtype=torch.float16, device=dev) for _ in range(2)]
            qkv, w, cos = torch.randn(36, 8 * 64, generator=g, device=dev).half(), torch.rand(64, generator=g, device=dev), torch.rand(50, 32, generator=g, device=dev)
            paged.paged_norm_rope_append(qkv, 4, 2, 64, w, w, 1e-6, cos, cos, st.positions, st.slots, *caches)
            bare = qkv.clone()
            paged.paged_norm_rope_append(bare, 4, 2, 64, w, w, 1e-6, None, None, None, None, None, None)
            f = paged.paged_fork(i([0, 0, 2]), i([4, 5, 6]), held, table, stack, count, shared, page, free_left=count if in_place else None)
            count = f.free_count
            paged.paged_copy(f.src, f.dst, caches)
            paged.paged_release(torch.tensor([0, 0, 1, 0, 1, 0, 0, 0], dtype=torch.uint8, device=dev), table, stack, count, held=i([0, 0, 5, 0, 0, 0, 0, 0]), page_size=page, shared=shared)
            paged.paged_release(torch.tensor([1, 0, 0, 0, 0, 0, 0, 0], dtype=torch.bool, device=dev), table, stack, count, shared=shared)
            c = paged.paged_compact(table, stack, count, shared)
            results.append((*f, *c, *paged.paged_compact(table, stack, count)[:3], table.clone(), shared, held, qkv, bare, *caches))
    for r in results[1:]:
        assert len(r) == len(results[0]) and all(torch.equal(a, b) for a, b in zip(r, results[0]))


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_autograd_hears_of_the_norms(paged, cuda_device, monkeypatch, native):
    if not native:
        monkeypatch.setattr(paged, "_native", lambda *args: None)
    qkv = torch.randn(3, 256, device=cuda_device).half()
    w, scale = torch.ones(64, device=cuda_device), torch.ones(256, device=cuda_device, dtype=torch.float16, requires_grad=True)
    y = qkv * scale
    paged.paged_norm_rope_append(qkv, 2, 1, 64, w, w, 1e-6, None, None, None, None, None, None)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


# ------------------------------------------------------------------ refusals
@pytest.mark.gpu
def test_refusals(paged, cuda_device):
    dev = cuda_device
    i = lambda *n: torch.zeros(n, dtype=torch.int32, device=dev)                                  # noqa: E731
    h = lambda *n: torch.zeros(n, dtype=torch.float16, device=dev)                                # noqa: E731
    table, free, one, done = i(3, 4), i(9), i(1), torch.zeros(3, dtype=torch.bool, device=dev)
    slots = torch.zeros(6, dtype=torch.int64, device=dev)
    c, w = h(3, 16, 2, 64), h(64)
    f = lambda **k: paged.paged_fork(**({"parents": i(2), "children": i(2), "context_lens": i(3), "block_table": table, "free_pages": free, "free_count": one, "shared": i(9),   # noqa: E731
                                         "page_size": 16} | k))
    n = lambda **k: paged.paged_norm_rope_append(**({"qkv": h(6, 512), "n_heads": 4, "n_kv_heads": 2, "head_dim": 64, "q_weight": w, "k_weight": w, "eps": 1e-6, "cos": h(9, 64),   # noqa: E731
                                                     "sin": h(9, 64), "positions": slots, "slots": slots, "k_cache": c, "v_cache": c} | k))
    bad = [lambda: f(parents=i(3)), lambda: f(children=i(2).long()), lambda: f(context_lens=i(2)), lambda: f(shared=i(8)), lambda: f(page_size=0), lambda: f(free_count=i(2)),
           lambda: f(free_left=i(2)), lambda: f(block_table=table.t()), lambda: f(parents=i(2).cpu()), lambda: f(shared=i(9).cpu()), lambda: f(free_pages=i(0), shared=i(0)),
           lambda: paged.paged_release(done, table, free, one, shared=i(8)), lambda: paged.paged_release(done, table, free, one, shared=i(9).cpu()),
           lambda: paged.paged_release(done, table, free, one, shared=i(9).long()), lambda: paged.paged_release(done, table, free, one, held=i(3), shared=i(9)),
           lambda: paged.paged_copy(i(2), i(3), [c]), lambda: paged.paged_copy(i(2).long(), i(2).long(), [c]), lambda: paged.paged_copy(i(2), i(2), [c.cpu()]),
           lambda: paged.paged_copy(i(2), i(2), [c[:, :, :1]]), lambda: paged.paged_copy(i(2), i(2), [c[:1].expand(3, -1, -1, -1)]), lambda: paged.paged_copy(i(2), i(2), [h(5)]),
           lambda: paged.paged_copy(i(2), i(2), [c.clone().requires_grad_()]), lambda: paged.paged_copy(i(2), i(2), [h(0, 3)]),
           lambda: paged.paged_compact(table.long(), free, one), lambda: paged.paged_compact(table, free, i(2)), lambda: paged.paged_compact(table, free, one, i(8)),
           lambda: paged.paged_compact(table, i(0), one), lambda: paged.paged_compact(table, free.cpu(), one),
           lambda: n(qkv=h(6, 500)), lambda: n(qkv=h(6, 512).float()), lambda: n(q_weight=h(63)), lambda: n(k_weight=w.float()), lambda: n(eps=-1.0), lambda: n(eps=math.nan), lambda: n(k_cache=None),
           lambda: n(cos=None), lambda: n(cos=h(9, 66), sin=h(9, 66)), lambda: n(slots=slots[:5]), lambda: n(positions=slots[:5]), lambda: n(q_weight=w.cpu()), lambda: n(k_cache=c[..., :32], v_cache=c[..., :32]),
           lambda: n(qkv=h(1, 512).expand(6, 512)), lambda: n(qkv=h(6, 512).requires_grad_()), lambda: n(q_weight=w.clone().requires_grad_()), lambda: n(k_cache=c[:, :, :1], v_cache=c[:, :, :1])]
    for k, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {k} was taken")
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="tangent"):
            n(k_weight=torch.autograd.forward_ad.make_dual(w, w))
    f(), n(), n(k_cache=None, v_cache=None, slots=None)


def test_refusals_on_the_cpu(paged, native_lib):
    i = lambda *n: torch.zeros(n, dtype=torch.int32)                                              # noqa: E731
    x, w = torch.zeros(2, 256, dtype=torch.float16), torch.zeros(64, dtype=torch.float16)
    for call in (lambda: paged.paged_fork(i(1), i(1), i(2), i(2, 3), i(5), i(1), i(5), 16), lambda: paged.paged_release(torch.zeros(2, dtype=torch.bool), i(2, 3), i(5), i(1), shared=i(5)),
                 lambda: paged.paged_copy(i(1), i(1), [x]), lambda: paged.paged_compact(i(2, 3), i(5), i(1)),
                 lambda: paged.paged_norm_rope_append(x, 2, 1, 64, w, w, 1e-6, None, None, None, None, None, None)):
        with pytest.raises(RuntimeError, match="CUDA device"):
            call()
    lib, some = native_lib._lib, 4096                                  # never read: every call is refused before anything is launched

    def refused(name, good, changes, code=1):
        for at, value in changes:
            args = list(good)
            args[at] = value
            assert getattr(lib, name)(*args) == code, (name, at, value)
    refused("lowbit_paged_fork_cuda", [some, some, 2, some, some, 4, 3, 4, some, 9, some, some, some, 16, some, some, some, None],
            [(a, None) for a in (0, 1, 3, 4, 8, 10, 11, 12, 14, 15, 16)] + [(2, 0), (2, (1 << 30) + 1), (5, 3), (6, 0), (6, (1 << 28) + 1), (7, 0), (9, 0), (9, (1 << 30) + 1), (13, 0)])
    refused("lowbit_paged_share_release_cuda", [some, some, 4, 3, some, 4, 4, some, 9, some, some, some, 1 << 20, None],
            [(a, None) for a in (0, 4, 7, 9, 10)] + [(2, 0), (3, 0), (5, 3), (6, 0), (8, 0), (8, (1 << 30) + 1)])
    refused("lowbit_paged_share_release_cuda", [some, some, 4, 3, some, 4, 4, some, 9, some, some, some, 1 << 20, None], [(11, None), (11, 4098), (12, 87)], 4)
    refused("lowbit_paged_compact_cuda", [some, 4, 3, 4, some, 9, some, some, some, some, some, some, some, some, some, 1 << 20, None],
            [(a, None) for a in (0, 4, 6, 7, 8, 9, 10, 11, 12, 13)] + [(1, 3), (2, 0), (3, 0), (5, 0), (5, (1 << 30) + 1)])
    refused("lowbit_paged_compact_cuda", [some, 4, 3, 4, some, 9, some, some, some, some, some, some, some, some, some, 1 << 20, None], [(14, None), (15, 143)], 4)
    at = (ctypes.c_void_p * 1)(some)
    refused("lowbit_paged_copy_cuda", [some, some, 2, at, 1, 9, 64, 64, None], [(0, None), (1, None), (2, -1), (3, None), (4, -1), (5, 0), (6, 63), (7, 0), (3, (ctypes.c_void_p * 1)(None))])
    strides = (ctypes.c_int64 * 3)(2048, 128, 64)
    refused("lowbit_paged_norm_rope_append_cuda", [some, 1, 512, 6, 4, 2, 64, 64, some, some, 1, 1e-6, some, some, 1, 64, 9, some, some, some, strides, some, strides, 1, 3, 16, None],
            [(a, None) for a in (0, 8, 9, 12, 13, 17, 18, 19, 20, 21, 22)] + [(1, 0), (2, 511), (3, -1), (4, -1), (5, 0), (6, 0), (7, 66), (7, 63), (10, 3), (11, -1.0), (11, math.nan), (14, 3), (15, 31),
                                                                        (16, 0), (23, 2), (24, 0), (25, 0)])


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_autograd_hears_of_caches_and_lists(paged, cuda_device, monkeypatch, native):
    """whatever the operators write over: caches, and whole numbers that a graph has kept as indices"""
    if not native:
        monkeypatch.setattr(paged, "_native", lambda *args: None)
    dev = cuda_device
    i = lambda x: dev_ints(x, dev)                                                                # noqa: E731
    w, scale, rows = torch.ones(64, device=dev), torch.ones(64, device=dev, dtype=torch.float16, requires_grad=True), torch.ones(12, 2, device=dev, requires_grad=True)
    slots = torch.arange(3, device=dev)
    with torch.inference_mode():
        keeps_no_count = torch.zeros(4, 8, 1, 64, dtype=torch.float16, device=dev)

    def state():
        return {"qkv": torch.randn(3, 256, device=dev).half(), "k_cache": torch.zeros(4, 8, 1, 64, dtype=torch.float16, device=dev), "v_cache": torch.zeros(4, 8, 1, 64, dtype=torch.float16, device=dev),
                "lens": i([9, 0, 0]), "table": i([[3, 2], [0, 0], [0, 0]]), "stack": i([0, 1, 0, 0]), "count": i([2]), "shared": i([0, 0, 0, 0])}

    def norms(s):
        paged.paged_norm_rope_append(s["qkv"], 2, 1, 64, w, w, 1e-6, None, None, None, slots, s["k_cache"], s["v_cache"])

    def fork(s):
        paged.paged_fork(i([0]), i([1]), s["lens"], s["table"], s["stack"], s["count"], s["shared"], 8, free_left=s["count"])

    def release(s):
        paged.paged_release(torch.tensor([True, False, False], device=dev), s["table"], s["stack"], s["count"], shared=s["shared"])
    for call, names in ((norms, ("qkv", "k_cache", "v_cache")), (lambda s: paged.paged_copy(i([0]), i([2]), [s["k_cache"], s["v_cache"]]), ("k_cache", "v_cache")),
                        (lambda s: paged.paged_copy(i([-1, 3]), i([1, 0]), [s["k_cache"], keeps_no_count, s["v_cache"].view(torch.uint8)]), ("k_cache", "v_cache")),
                        (fork, ("lens", "table", "count", "shared")), (release, ("table", "stack", "count", "shared"))):
        for name in names:
            s = state()
            kept = s[name]
            y = torch.nn.functional.embedding(kept, rows) if kept.dtype == torch.int32 else kept.view(-1, 64) * scale
            call(s)
            with pytest.raises(RuntimeError, match="modified by an inplace"):
                y.sum().backward()
        s = state()
        y = sum(t.float().sum() for t in s.values()) * scale.sum()     # what is read alone stays
        call(s)
        y.backward()
    s = state() | {"k_cache": keeps_no_count, "v_cache": keeps_no_count.clone()}
    norms(s)
    table = i([[1, 2]])
    y = torch.nn.functional.embedding(table, rows)
    paged.paged_compact(table, i([0, 3, 0, 0]), i([2]))                # writes over nothing
    y.sum().backward()
