"""The paged key/value cache (transformers/paged_kv.py): bookkeeping against whole numbers computed here, the cache write and the two
attentions against 64-bit statements.

Bounds.  A rounding is off by half a step, h(t) = finfo(t).eps / 2 of the value.  An attention's output is rounded once, h(out) |o|; its
probabilities may be rounded to the type t of the values in the product (the activations', fp16 over e5m2), each h(t) of itself, which moves
the output by up to h(t) (a + |o|) with a = sum p |v| / sum p.  The sums: a score's D products drop up to 2^-23 of their absolute sum in
each of D / 8 steps, and that much of its probability; exp2 2^-22; the products with the values up to 2^-23 of a in each of L / 8 steps."""
import ctypes
import math

import pytest
import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def paged(native_lib):
    from ipex_llm_b200.transformers import paged_kv
    yield paged_kv
    if torch.cuda.is_available():
        assert not native_lib.lowbit_gemm_wait_expired()


# ------------------------------------------------------------------ pages, slots, positions
def step_statement(new, held, table, stack, page, n_tokens):
    """the same in whole numbers: (table, cu, seq_lens, positions, slots, left, missing); the table's rows as lists"""
    table, stack, missing = [list(row) for row in table], list(stack), 0
    cu, lens, positions, slots = [0], [], [], []
    for r, (n, h) in enumerate(zip(new, held)):
        for c in range(-(-h // page), -(-(h + n) // page)):
            if c >= len(table[r]):
                missing += 1
            elif stack:
                table[r][c] = stack.pop()
            else:
                table[r][c] = -1
                missing += 1
        for p in range(h, h + n):
            c = p // page
            pg = table[r][c] if c < len(table[r]) else -1
            positions.append(p)
            slots.append(pg * page + p % page if pg >= 0 else -1)
        cu.append(cu[-1] + n)
        lens.append(h + n)
    pad = n_tokens - len(slots)
    return table, cu, lens, (positions + [0] * pad)[:n_tokens], (slots + [-1] * pad)[:n_tokens], len(stack), missing


def start(held, page, width, pages, g, spare=None):
    """a table that holds what the requests hold, and the stack of free pages (``spare`` of them)"""
    order = torch.randperm(pages, generator=g).tolist()
    table = []
    for h in held:
        row = [order.pop() for _ in range(min(-(-h // page), width))]
        table.append(row + [-1] * (width - len(row)))
    return table, order if spare is None else order[:spare]


STEPS = [([1], [0], 16, 4), ([1], [15], 16, 4), ([1], [16], 16, 4), ([1, 1, 1], [0, 31, 32], 16, 8), ([0, 5, 0, 40, 1], [3, 0, 0, 7, 64], 8, 16),
         ([100, 1, 300], [0, 0, 1], 1, 400), ([33, 17], [20, 6], 7, 20), ([0, 0], [9, 0], 4, 4), ([700], [3], 128, 9)]


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [0, 3, 200])
@pytest.mark.parametrize("new,held,page,width", STEPS)
def test_step(paged, cuda_device, new, held, page, width, pad):
    check_step(paged, cuda_device, new, held, page, width, sum(new) + pad)


@pytest.mark.gpu
@pytest.mark.parametrize("R,page", [(31, 16), (33, 64), (1000, 16), (1024, 8), (1025, 32), (2500, 16)])
def test_step_of_many_requests(paged, cuda_device, R, page):
    g = torch.Generator().manual_seed(R)
    held = torch.randint(0, 500, (R,), generator=g).tolist()
    new = [n if i % 5 == 0 else 1 for i, n in enumerate(torch.randint(0, 90, (R,), generator=g).tolist())]
    check_step(paged, cuda_device, new, held, page, -(-600 // page), sum(new) + 5)


@pytest.mark.gpu
@pytest.mark.parametrize("spare", [0, 1, 3])
@pytest.mark.parametrize("new,held,page,width", [([40, 5, 20], [0, 3, 1], 8, 8), ([1, 1, 1, 1], [8, 16, 7, 24], 8, 8), ([30, 90], [2, 1], 8, 4)])
def test_step_without_enough_pages(paged, cuda_device, new, held, page, width, spare):
    """earlier requests are served first; what is left gets -1, and the count of it; the same where the table is too narrow"""
    check_step(paged, cuda_device, new, held, page, width, sum(new), spare)


def check_step(paged, dev, new, held, page, width, n_tokens, spare=None):
    g = torch.Generator().manual_seed(sum(new) + page)
    pages = sum(-(-h // page) for h in held) + sum(-(-n // page) + 1 for n in new) + 2
    table, stack = start(held, page, width, pages, g, spare)
    want = step_statement(new, held, table, stack, page, n_tokens)
    on = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)                                 # noqa: E731
    wide = torch.full((len(new), width + 3), 77, dtype=torch.int32, device=dev)                   # rows of a wider table
    wide[:, :width] = on(table)
    free = torch.full((pages,), -5, dtype=torch.int32, device=dev)
    free[:len(stack)] = on(stack)
    count = on([len(stack)])
    for in_place in (False, True):
        t = wide.clone()
        st = paged.paged_step(on(new), on(held), t[:, :width], free, count, page, n_tokens, free_left=count if in_place else None)
        assert t[:, :width].tolist() == want[0] and bool((t[:, width:] == 77).all())
        assert (st.cu_seqlens.tolist(), st.seq_lens.tolist(), st.positions.tolist(), st.slots.tolist()) == want[1:5]
        assert (st.free_count.item(), st.missing.item()) == want[5:]
        assert count.item() == (want[5] if in_place else len(stack))


@pytest.mark.gpu
def test_fewer_rows_than_tokens(paged, cuda_device):
    """rows of the step beyond those asked for are not written anywhere"""
    on = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)                         # noqa: E731
    st = paged.paged_step(on([3, 9]), on([0, 0]), torch.full((2, 4), -1, dtype=torch.int32, device=cuda_device), on([4, 5, 6, 7]), on([4]), 4, 5)
    assert st.positions.tolist() == [0, 1, 2, 0, 1] and st.slots.tolist() == [28, 29, 30, 24, 25] and st.cu_seqlens.tolist() == [0, 3, 12]


@pytest.mark.gpu
@pytest.mark.parametrize("width", [1, 5, 40, 1500])
def test_release_returns_every_page_once(paged, cuda_device, width):
    g = torch.Generator().manual_seed(width)
    R, pages = 9, 9 * width + 4
    held = torch.randint(0, width * 4 + 1, (R,), generator=g).tolist()
    table, stack = start(held, 4, width, pages, g)
    done = [True, False, True, True, False, False, True, False, True]
    free = torch.full((pages,), -5, dtype=torch.int32, device=cuda_device)
    free[:len(stack)] = torch.tensor(stack, dtype=torch.int32, device=cuda_device)
    count = torch.tensor([len(stack)], dtype=torch.int32, device=cuda_device)
    t = torch.tensor(table, dtype=torch.int32, device=cuda_device)
    for _ in range(2):                                                                            # the second time there is nothing to return
        paged.paged_release(torch.tensor(done, device=cuda_device), t, free, count)
        want = stack + [p for row, d in zip(table, done) if d for p in row if p >= 0]
        assert count.item() == len(want) and free[:len(want)].tolist() == want and bool((free[len(want):] == -5).all())
        assert t.tolist() == [[-1] * width if d else row for row, d in zip(table, done)]


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 2])
def test_lengths_that_32_bits_cannot_add(paged, cuda_device, page):
    """a request that would bring its end beyond 2^31: what its row can name is handed out once, and the counts are the largest that there are"""
    most = (1 << 31) - 1
    on = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)                         # noqa: E731
    for new, held in (([most], [1]), ([2, most, most], [1, 3, 2]), ([most, most], [most, 0])):
        R, width = len(new), 4
        had = [min(-(-h // page), width) for h in held]
        table = [[10 * r + c if c < had[r] else -1 for c in range(width)] for r in range(R)]
        stack = list(range(100, 130))
        want, left = [list(row) for row in table], list(stack)
        for r in range(R):
            for c in range(had[r], min(-(-(held[r] + new[r]) // page), width)):
                want[r][c] = left.pop()
        t, count = on(table), on([len(stack)])
        st = paged.paged_step(on(new), on(held), t, on(stack), count, page, 6)
        assert t.tolist() == want and st.free_count.item() == len(left)
        ends = [0]
        for n in new:
            ends.append(ends[-1] + n)
        assert st.cu_seqlens.tolist() == [min(e, most) for e in ends] and st.seq_lens.tolist() == [min(h + n, most) for h, n in zip(held, new)]
        for i, (p, s) in enumerate(zip(st.positions.tolist(), st.slots.tolist())):
            r = next(r for r in range(R) if ends[r + 1] > i)
            at = held[r] + i - ends[r]
            assert p == at and s == (want[r][at // page] * page + at % page if at // page < width else -1)
        assert st.missing.item() > most // 8


def test_a_table_of_more_entries_than_32_bits_is_refused(native_lib):
    lib, p = native_lib._lib, ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p)
    assert lib.lowbit_paged_step_cuda(p, p, 1 << 16, p, 1 << 15, 1 << 15, p, 8, p, p, 16, 3, p, p, p, p, p, None) != 0
    assert "lowbit_paged_step_cuda" in lib.b200_lowbit_last_error_string().decode()
    lib.b200_lowbit_clear_error()


def owned_once(table, stack, count, pages):
    """every page is named by one row or lies on the stack, once"""
    return sorted([x for row in table.tolist() for x in row if x >= 0] + stack[:int(count)].tolist()) == list(range(pages))


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("new,held,page,width,spare,victim", [([40, 5, 20], [3, 9, 17], 8, 9, 3, 1), ([1, 1, 1, 1], [8, 16, 7, 24], 8, 8, 1, 3), ([30, 2, 90], [2, 60, 1], 8, 4, 5, 1),
                                                              ([700, 1, 2000], [5, 900, 16], 1, 2100, 800, 1)])
def test_a_step_that_ran_short_is_taken_back_and_repeated(paged, cuda_device, new, held, page, width, spare, victim, in_place):
    """pages that it handed out go back, a request goes, and the step is repeated: every page stays somebody's, once"""
    g = torch.Generator().manual_seed(page + sum(new))
    pages = sum(min(-(-h // page), width) for h in held) + spare
    table, stack = start(held, page, width, pages, g)
    on = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)                         # noqa: E731
    t, free, count = on(table), torch.full((pages,), -5, dtype=torch.int32, device=cuda_device), on([len(stack)])
    free[:len(stack)] = on(stack)
    st = paged.paged_step(on(new), on(held), t, free, count, page, sum(new), free_left=count if in_place else None)
    assert st.missing.item() > 0 and owned_once(t, free, st.free_count, pages)
    everyone = torch.ones(len(new), dtype=torch.bool, device=cuda_device)
    paged.paged_release(everyone, t, free, st.free_count, on(held), page)
    assert t.tolist() == table and st.free_count.item() == len(stack) and owned_once(t, free, st.free_count, pages)
    paged.paged_release(torch.arange(len(new), device=cuda_device) == victim, t, free, st.free_count)
    new[victim:victim + 1], held[victim:victim + 1] = [0], [0]
    again = paged.paged_step(on(new), on(held), t, free, st.free_count, page, sum(new))
    assert owned_once(t, free, again.free_count, pages)
    want = [min(-(-(h + n) // page), width) for h, n in zip(held, new)]
    wanted = sum(want) - sum(min(-(-h // page), width) for h in held)
    assert again.free_count.item() == max(st.free_count.item() - wanted, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [3, 40, 1500])
def test_tokens_that_a_request_drops_give_their_pages_back(paged, cuda_device, width):
    g = torch.Generator().manual_seed(width)
    R, page, pages = 7, 4, 7 * width + 4
    held = torch.randint(0, width * page + 1, (R,), generator=g).tolist()
    keep = [min(int(x * (h + 9)), h + 3) for x, h in zip(torch.rand(R, generator=g).tolist(), held)]   # a few more than they hold: nothing goes
    keep[0], keep[1] = -2, 0
    done = [True, True, False, True, True, False, True]
    table, stack = start(held, page, width, pages, g)
    on = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)                         # noqa: E731
    wide, free, count = torch.full((R, width + 3), 77, dtype=torch.int32, device=cuda_device), torch.full((pages,), -5, dtype=torch.int32, device=cuda_device), on([len(stack)])
    wide[:, :width], free[:len(stack)] = on(table), on(stack)
    first = [min(-(-max(k, 0) // page), width) for k in keep]
    for _ in range(2):                                                                            # the second time there is nothing to return
        paged.paged_release(torch.tensor(done, device=cuda_device), wide[:, :width], free, count, on(keep), page)
        want = stack + [p for row, d, f in zip(table, done, first) if d for p in row[f:] if p >= 0]
        assert count.item() == len(want) and free[:len(want)].tolist() == want and bool((free[len(want):] == -5).all())
        assert wide[:, :width].tolist() == [row[:f] + [-1] * (width - f) if d else row for row, d, f in zip(table, done, first)] and bool((wide[:, width:] == 77).all())


# ------------------------------------------------------------------ the write into the cache
def rotated(x, cos, sin):
    """64 bits: x [T, H, D], tables [T, rotary width]"""
    R = cos.shape[-1]
    c, s = cos.double()[:, None], sin.double()[:, None]
    a = x[..., :R]
    return torch.cat([a * c + torch.cat([-a[..., R // 2:], a[..., :R // 2]], -1) * s, x[..., R:]], -1)


def tables(dim, n, dev, dtype=torch.float32):
    a = torch.arange(n, device=dev, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, dim, 2, device=dev, dtype=torch.float64) / dim)
    return torch.cat([a.cos()] * 2, -1).to(dtype), torch.cat([a.sin()] * 2, -1).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("T,heads,kv_heads,dim,rotary,table_type", [(1, 32, 32, 128, 128, "f32"), (7, 4, 2, 64, 64, "same"), (300, 14, 2, 96, 32, "f32"), (33, 8, 1, 256, 256, "same"),
                                                                    (65, 3, 3, 80, 80, "f32"), (20, 2, 1, 48, 6, "same"), (40, 0, 2, 64, 64, "f32"), (130, 8, 4, 128, 0, "f32")])
def test_append(paged, cuda_device, dtype, eight, T, heads, kv_heads, dim, rotary, table_type):
    g = torch.Generator(device=cuda_device).manual_seed(T)
    page, width = 8, (heads + 2 * kv_heads) * dim
    pages = T // page + 3
    whole = torch.randn(T, width + 16, generator=g, device=cuda_device).to(dtype)                 # rows with something between them
    qkv = whole[:, :width]
    qkv[0, -1] = 60000.0                                                                          # saturates in e5m2 (57344)
    before = whole.clone()
    # the layout of a cache whose heads come before its rows
    caches = [torch.randn(pages, kv_heads, page, dim, generator=g, device=cuda_device).to(dtype).transpose(1, 2) for _ in range(2)]
    if eight:
        caches = [c.to(torch.float8_e5m2).view(torch.uint8) for c in caches]
    held = [c.clone() for c in caches]
    slots = torch.randperm(pages * page, generator=g, device=cuda_device)[:T]
    slots[T // 2] = -1 if T > 1 else slots[0]
    if T > 30:
        slots[5] = pages * page                                                                   # no slot of the cache
    positions = torch.randint(0, 500, (T,), generator=g, device=cuda_device)
    positions[-1] = 10 ** 10                                                                      # beyond the tables: the last row
    cos, sin = tables(max(rotary, 2), 500, cuda_device, torch.float32 if table_type == "f32" else dtype)
    paged.paged_rope_append(qkv, heads, kv_heads, dim, *((cos, sin) if rotary else (None, None)), positions if rotary else None, slots, *caches)
    x = before[:, :width].double().view(T, heads + 2 * kv_heads, dim)
    n = heads + kv_heads
    if rotary:
        at = positions.clamp(max=499)
        want = rotated(x[:, :n], cos[at], sin[at])
        # two products, one sum, one rounding
        scale = rotated(x[:, :n].abs(), cos[at].abs(), -sin[at].abs())
        got = qkv.double().view(T, -1, dim)[:, :n]
        assert bool(((got - want).abs() <= HALF[dtype] * want.abs() + 2.0 ** -22 * (scale.abs() + want.abs() + x[:, :n].abs().amax()) + 1e-7).all())
    else:
        assert torch.equal(qkv, before[:, :width])
    assert torch.equal(whole[:, width:], before[:, width:])
    assert torch.equal(qkv[:, n * dim:], before[:, n * dim:width])                                # the values stay
    now = qkv.reshape(T, -1, dim)
    for cache, old, rows in zip(caches, held, (now[:, heads:n], now[:, n:])):
        flat, was = cache.reshape(pages * page, kv_heads, dim), old.reshape(pages * page, kv_heads, dim).clone()
        ok = (slots >= 0) & (slots < pages * page)
        # the bytes are those of the rounded activations, and everything else stays
        was[slots[ok]] = rows[ok].float().clamp(-57344, 57344).to(torch.float8_e5m2).view(torch.uint8) if eight else rows[ok]
        assert torch.equal(flat.view(torch.uint8), was.view(torch.uint8))


# ------------------------------------------------------------------ attention
def statement(q, k, v, cu, lens, scale, causal=True):
    """64 bits.  q [T, H, D]; k, v: lists of [len_r, G, D]; returns the outputs, the same with |v|, and the largest absolute sum of a score"""
    out, absolute, largest = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device), 0.0
    group = q.shape[1] // k[0].shape[1]
    for r in range(len(lens)):
        a, b, n = cu[r], cu[r + 1], lens[r]
        if a == b or n == 0:
            continue
        kr, vr = (t.double().repeat_interleave(group, 1) for t in (k[r], v[r]))
        s = torch.einsum("ihd,jhd->hij", q[a:b].double(), kr) * scale
        largest = max(largest, float(torch.einsum("ihd,jhd->hij", q[a:b].double().abs(), kr.abs()).max()) * scale)
        if causal:
            unseen = torch.arange(n, device=q.device)[None] > n - (b - a) + torch.arange(b - a, device=q.device)[:, None]
            s = s.masked_fill(unseen, -math.inf)
        p = torch.softmax(s, -1)
        p = torch.where(torch.isnan(p), torch.zeros_like(p), p)
        out[a:b] = torch.einsum("hij,jhd->ihd", p, vr)
        absolute[a:b] = torch.einsum("hij,jhd->ihd", p, vr.abs())
    return out, absolute, largest


def bound(want, absolute, largest, dtype, p_dtype, dim, keys):
    score = dim / 8 * largest * 2.0 ** -23 + 2.0 ** -22
    return HALF[dtype] * want.abs() + HALF[p_dtype] * (absolute + want.abs()) + (2 * score + (keys / 8 + 8) * 2.0 ** -23) * absolute + 1e-7


def requests(dev, new, held, heads, kv_heads, dim, dtype, eight, page, seed=0, q_scale=1.5, stale=math.nan):
    """(q, caches, table, lens, cu, the keys and values of every request): rows and pages that nobody holds are ``stale``"""
    g = torch.Generator(device=dev).manual_seed(seed + sum(new) + 7 * len(new))
    lens = [h + n for h, n in zip(held, new)]
    counts = [-(-n // page) for n in lens]
    pages, width = sum(counts) + 2, max(counts + [1]) + 1
    caches = [torch.full((pages, page, kv_heads, dim), stale, device=dev).to(torch.float8_e5m2 if eight else dtype) for _ in range(2)]
    order = torch.randperm(pages, generator=g, device=dev)
    table = torch.full((len(new), width), -1, dtype=torch.int32, device=dev)
    rows, first = [[], []], 0
    for r, (c, n) in enumerate(zip(counts, lens)):
        mine = order[first:first + c]
        first += c
        table[r, :c] = mine.int()
        for cache, keep in zip(caches, rows):
            x = torch.randn(n, kv_heads, dim, generator=g, device=dev).to(cache.dtype)
            keep.append(x)
            at = mine[torch.arange(n, device=dev) // page] * page + torch.arange(n, device=dev) % page
            cache.view(torch.uint8 if eight else torch.int16).view(-1, kv_heads, dim)[at] = x.view(torch.uint8 if eight else torch.int16)
    q = (q_scale * torch.randn(sum(new), heads, dim, generator=g, device=dev)).to(dtype)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    on = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)                                 # noqa: E731
    if eight:
        caches = [c.view(torch.uint8) for c in caches]
    return q, caches, table, on(lens), on(cu), rows, cu, lens


def check_paged(paged, dev, new, held, heads, kv_heads, dim, dtype, eight, page, scale=None, hint=None, **kw):
    q, caches, table, lens, cu, rows, cu_list, len_list = requests(dev, new, held, heads, kv_heads, dim, dtype, eight, page, **kw)
    scale = dim ** -0.5 if scale is None else scale
    got = paged.sdp_paged(q, *caches, table, lens, cu, scale, max_query_len=hint)
    if eight:
        rows = [[x.half() for x in part] for part in rows]
    want, absolute, largest = statement(q, *rows, cu_list, len_list, scale)
    limit = bound(want, absolute, largest, dtype, torch.float16 if eight else dtype, dim, max(len_list))
    far = (got.double() - want).abs()
    assert bool((far <= limit).all()), f"{float((far / limit).max()):.2f} of the bound"
    return got


KINDS = [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True), (torch.bfloat16, True)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 128), (8, 2, 128), (8, 1, 64), (2, 2, 96), (7, 1, 80), (16, 1, 128), (6, 2, 256), (5, 5, 16), (3, 1, 192)])
@pytest.mark.parametrize("held,page", [([0], 16), ([1, 15, 16, 17, 0], 16), ([127, 128, 129, 5, 1000], 8), ([255, 300, 31, 32, 33], 1), ([3000, 2, 700], 24)])
def test_single_tokens(paged, cuda_device, dtype, eight, heads, kv_heads, dim, held, page):
    check_paged(paged, cuda_device, [1] * len(held), held, heads, kv_heads, dim, dtype, eight, page, hint=1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 128), (8, 2, 128), (8, 1, 64), (2, 2, 96), (7, 1, 80), (6, 2, 256), (3, 1, 192), (5, 1, 32)])
@pytest.mark.parametrize("new,held,page", [([2], [0], 16), ([5, 1, 3], [100, 0, 16], 16), ([128], [0], 32), ([129, 1, 17], [3, 500, 0], 24), ([300, 2, 0, 64], [1000, 30, 40, 64], 64),
                                           ([33, 257], [127, 1], 8)])
def test_chunks(paged, cuda_device, dtype, eight, heads, kv_heads, dim, new, held, page):
    check_paged(paged, cuda_device, new, held, heads, kv_heads, dim, dtype, eight, page)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
@pytest.mark.parametrize("R,heads,kv_heads", [(3, 32, 8), (70, 8, 2), (300, 4, 4), (1100, 2, 1)])
def test_many_requests_of_different_lengths(paged, cuda_device, dtype, eight, R, heads, kv_heads):
    g = torch.Generator().manual_seed(R)
    held = [int(2 ** float(x)) for x in torch.rand(R, generator=g) * (11 if R < 100 else 8)]
    for most in (1, 40):
        new = [1 if i % 4 else 1 + int(x) for i, x in enumerate(torch.randint(0, most, (R,), generator=g))]
        check_paged(paged, cuda_device, new, held, heads, kv_heads, 128, dtype, eight, 16, hint=most)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
@pytest.mark.parametrize("new,held", [([1], [9000]), ([700], [2500]), ([1, 300, 1], [6000, 1500, 3])])
@pytest.mark.parametrize("q_scale", [0.05, 4.0, 40.0])
def test_flat_and_steep_softmax(paged, cuda_device, dtype, eight, new, held, q_scale):
    """nearly equal probabilities over many keys, and scores of hundreds that pick single ones"""
    check_paged(paged, cuda_device, new, held, 8, 2, 128, dtype, eight, 16, q_scale=q_scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,eight,big", [(torch.float16, False, 2.0 ** 12), (torch.float16, False, 1.0), (torch.bfloat16, False, 2.0 ** 90), (torch.bfloat16, False, 2.0 ** 12),
                                             (torch.float16, True, 2.0 ** 12), (torch.bfloat16, True, 2.0 ** 90), (torch.bfloat16, True, 2.0 ** 12)])
@pytest.mark.parametrize("new,held", [([1], [700]), ([3, 1], [20, 300]), ([40], [200]), ([300, 70], [0, 900])])
def test_scores_beyond_what_32_bits_tell_apart(paged, cuda_device, dtype, eight, big, new, held):
    """scores of 10^4 to 10^31, whose neighbours in 32 bits lie up to 10^24 apart: a row takes the value of its largest, far ahead of the others"""
    heads, kv_heads, dim = 4, 2, 64
    q, caches, table, lens, cu, rows, cu_list, len_list = requests(cuda_device, new, held, heads, kv_heads, dim, dtype, eight, 16)
    q, kind = (whole(q).double() * big).to(dtype), torch.float8_e5m2 if eight else dtype
    k = [(whole(x).float() * 4096).to(kind) for x in rows[0]]
    for r, x in enumerate(k):
        j = torch.arange(len(x), device=cuda_device)
        caches[0][table[r, j // 16].long(), j % 16] = x.view(torch.uint8) if eight else x
    got = paged.sdp_paged(q, *caches, table, lens, cu)
    assert bool(torch.isfinite(got).all())
    for r, (a, b, n) in enumerate(zip(cu_list, cu_list[1:], len_list)):
        s = torch.einsum("ihd,jhd->hij", q[a:b].double(), k[r].double().repeat_interleave(2, 1)) * dim ** -0.5          # exact: whole numbers of few bits
        s = s.masked_fill(torch.arange(n, device=cuda_device)[None] > n - (b - a) + torch.arange(b - a, device=cuda_device)[:, None], -math.inf)
        top = s.topk(min(2, n), -1).values
        # the second is behind by more than the scores' rounding and than any weight that counts
        clear = (top[..., 0] - top[..., -1] > 64 + top[..., 0].abs() * 2.0 ** -20) | (torch.arange(b - a, device=cuda_device)[None] + n - (b - a) == 0)
        want = rows[1][r].to(dtype).repeat_interleave(2, 1).permute(1, 0, 2).gather(1, s.argmax(-1)[..., None].expand(-1, -1, dim)).transpose(0, 1)
        assert bool((clear.float().mean() > 0.5)) and torch.equal(got[a:b][clear.t()], want[clear.t()])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
def test_requests_without_keys_and_rows_behind_the_last(paged, cuda_device, dtype, eight):
    q, caches, table, lens, cu, rows, cu_list, len_list = requests(cuda_device, [3, 0, 1, 150], [20, 9, 4, 7], 8, 2, 64, dtype, eight, 16)
    lens[0], lens[3] = 0, 140                                   # a request without keys; one whose first ten tokens see none
    out = torch.full((q.shape[0] + 9, 8, 64), 5.0, dtype=dtype, device=cuda_device)
    wide = torch.cat([q, torch.full((9, 8, 64), math.nan, dtype=dtype, device=cuda_device)])
    got = paged.sdp_paged(wide, *caches, table, lens, cu, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert bool((out[:3] == 0).all()) and bool((out[4:14] == 0).all()) and bool((out[q.shape[0]:] == 5).all())
    if eight:
        rows = [[x.half() for x in part] for part in rows]
    rows = [[x[:n] for x, n in zip(part, lens.tolist())] for part in rows]
    want, absolute, largest = statement(q, *rows, cu_list, lens.tolist(), 64 ** -0.5)
    want[4:14], absolute[4:14] = 0, 0
    limit = bound(want, absolute, largest, dtype, torch.float16 if eight else dtype, 64, 157)
    assert bool(((out[:q.shape[0]].double() - want).abs() <= limit).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
@pytest.mark.parametrize("new", [[1, 1, 1], [200, 150, 90]])
def test_values_that_are_not_numbers_stay_with_their_request(paged, cuda_device, dtype, eight, new):
    """another request's infinities and NaN, and a page that does not exist, reach no row of the others"""
    q, caches, table, lens, cu, rows, cu_list, len_list = requests(cuda_device, new, [300, 31, 77], 4, 2, 128, dtype, eight, 16)
    want = paged.sdp_paged(q, *caches, table, lens, cu)
    bad = {torch.float16: 0x7e00, torch.bfloat16: 0x7fc0}[dtype]
    for cache in caches:
        cache.view(torch.uint8 if eight else torch.int16)[table[1, 1].long(), 3] = 0x7f if eight else bad
    got = paged.sdp_paged(q, *caches, table, lens, cu)
    a, b = cu_list[1], cu_list[2]
    assert torch.equal(got[:a], want[:a]) and torch.equal(got[b:], want[b:]) and bool(torch.isnan(got[b - 1]).all())
    table[1, 0] = -1
    table[2, 2] = 10 ** 6
    got = paged.sdp_paged(q, *caches, table, lens, cu)
    assert torch.equal(got[:a], want[:a]) and bool(torch.isnan(got[b - 1]).all()) and bool(torch.isnan(got[-1]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
@pytest.mark.parametrize("new,held", [([1, 1, 1, 1], [31, 300, 2000, 48]), ([3, 1, 2, 16], [29, 300, 64, 32]), ([32, 10, 200, 300], [0, 60, 900, 20]), ([1, 20, 1, 40], [31, 45, 65, 30])])
@pytest.mark.parametrize("page", [16, 4])
def test_a_request_that_holds_more_than_its_row_can_name(paged, cuda_device, dtype, eight, new, held, page):
    """its rows are NaN, as for a page that is not there, and not the attention of other positions; one that fills its row is not touched by it"""
    q, caches, table, lens, cu, rows, cu_list, len_list = requests(cuda_device, new, held, 4, 2, 64, dtype, eight, page)
    width = 32 // page
    got = paged.sdp_paged(q, *caches, table[:, :width], lens, cu)
    if eight:
        rows = [[x.half() for x in part] for part in rows]
    want, absolute, largest = statement(q, *rows, cu_list, len_list, 64 ** -0.5)
    limit = bound(want, absolute, largest, dtype, torch.float16 if eight else dtype, 64, 32)
    assert len_list[0] == 32
    for r, n in enumerate(len_list):
        a, b = cu_list[r], cu_list[r + 1]
        if n > 32:
            assert bool(torch.isnan(got[a:b]).all()), r
        else:
            assert bool(((got[a:b].double() - want[a:b]).abs() <= limit[a:b]).all()), r


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,eight", [KINDS[1], KINDS[3]])
def test_a_cache_beyond_32_bits(paged, cuda_device, dtype, eight):
    """offsets of more than 2^32 elements, and a layout with the heads in front of the rows"""
    page, kv_heads, dim, pages = 16, 2, 128, (1 << 32) // (16 * 2 * 128) + 40
    kind = torch.uint8 if eight else dtype
    caches = [torch.zeros(pages, kv_heads, page, dim, dtype=kind, device=cuda_device).transpose(1, 2) for _ in range(2)]
    g = torch.Generator(device=cuda_device).manual_seed(5)
    table = torch.tensor([[pages - 1, 3, pages - 7], [2, pages - 2, -1]], dtype=torch.int32, device=cuda_device)
    lens, cu = torch.tensor([40, 19], dtype=torch.int32, device=cuda_device), torch.tensor([0, 20, 21], dtype=torch.int32, device=cuda_device)
    rows = [[], []]
    for r, n in enumerate((40, 19)):
        for cache, keep in zip(caches, rows):
            x = torch.randn(n, kv_heads, dim, generator=g, device=cuda_device).to(torch.float8_e5m2 if eight else dtype)
            keep.append(x.half() if eight else x)
            for j in range(n):
                cache[int(table[r, j // page]), j % page] = x[j].view(torch.uint8) if eight else x[j]
    q = torch.randn(21, 4, dim, generator=g, device=cuda_device).to(dtype)
    got = paged.sdp_paged(q, *caches, table, lens, cu)
    want, absolute, largest = statement(q, *rows, [0, 20, 21], [40, 19], dim ** -0.5)
    assert bool(((got.double() - want).abs() <= bound(want, absolute, largest, dtype, torch.float16 if eight else dtype, dim, 40)).all())


@pytest.mark.gpu
def test_views_and_layouts(paged, cuda_device):
    """queries inside the merged projection's output, outputs with room between the heads, heads before rows, a misaligned query"""
    dev, dtype = cuda_device, torch.bfloat16
    q, caches, table, lens, cu, rows, cu_list, len_list = requests(dev, [1, 70, 4], [90, 33, 8], 8, 2, 64, dtype, False, 16)
    want = paged.sdp_paged(q, *caches, table, lens, cu)
    flat = torch.randn(q.shape[0], 12 * 64, device=dev).to(dtype)
    flat[:, :8 * 64] = q.flatten(1)
    view = flat.view(q.shape[0], 12, 64)[:, :8]
    turned = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in caches]
    out = torch.full((q.shape[0], 8, 96), 3.0, device=dev).to(dtype)
    paged.sdp_paged(view, *turned, table, lens, cu, out=out[..., :64])
    assert torch.equal(out[..., :64], want) and bool((out[..., 64:] == 3).all())
    odd = torch.empty(q.numel() + 1, dtype=dtype, device=dev)[1:].view(q.shape)
    odd.copy_(q)
    assert odd.data_ptr() % 16 and torch.equal(paged.sdp_paged(odd, *caches, table, lens, cu), want)


# ------------------------------------------------------------------ packed prompts
def check_packed(paged, dev, lens, heads, kv_heads, dim, dtype, causal=True, q_scale=1.5, hint=True, pad=0):
    g = torch.Generator(device=dev).manual_seed(sum(lens) + heads)
    T = sum(lens)
    x = torch.randn(T + pad, heads + 2 * kv_heads, dim, generator=g, device=dev)
    x[:, :heads] *= q_scale
    x = x.to(dtype)
    x[T:] = math.nan                                            # padding behind the last prompt
    q, k, v = x.split([heads, kv_heads, kv_heads], 1)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    out = torch.full((T + pad, heads, dim), 7.0, dtype=dtype, device=dev)
    got = paged.sdp_packed(q, k, v, torch.tensor(cu, dtype=torch.int32, device=dev), is_causal=causal, max_seqlen=max(lens) if hint else None, out=out)
    assert bool((got[T:] == 7).all())
    parts = [[t[a:b] for a, b in zip(cu, cu[1:])] for t in (k, v)]
    want, absolute, largest = statement(q[:T], *parts, cu, lens, dim ** -0.5, causal)
    limit = bound(want, absolute, largest, dtype, dtype, dim, max(lens))
    far = (got[:T].double() - want).abs()
    assert bool((far <= limit).all()), f"{float((far / limit).max()):.2f} of the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 128), (8, 2, 128), (8, 1, 64), (2, 2, 96), (7, 1, 80), (6, 2, 256), (3, 1, 192), (12, 4, 64), (5, 1, 16)])
@pytest.mark.parametrize("lens", [[1], [1, 1, 2], [64, 63, 65], [128, 1, 127, 129], [0, 300, 0, 5], [517, 256]])
def test_packed(paged, cuda_device, dtype, heads, kv_heads, dim, lens):
    check_packed(paged, cuda_device, lens, heads, kv_heads, dim, dtype, hint=sum(lens) % 2 == 0, pad=sum(lens) % 3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads,dim,lens", [(4, 2, 128, [1, 130, 700]), (2, 2, 64, [90, 257]), (2, 1, 256, [300])])
def test_packed_without_a_causal_mask(paged, cuda_device, dtype, heads, kv_heads, dim, lens):
    check_packed(paged, cuda_device, lens, heads, kv_heads, dim, dtype, causal=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,heads,kv_heads", [([2100, 900, 33], 32, 8), ([3000], 8, 8), ([40] * 90, 8, 2), ([1 + i % 7 for i in range(700)], 4, 2)])
@pytest.mark.parametrize("q_scale", [0.05, 1.5, 20.0])
def test_packed_long_and_many(paged, cuda_device, dtype, lens, heads, kv_heads, q_scale):
    check_packed(paged, cuda_device, lens, heads, kv_heads, 128, dtype, q_scale=q_scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_packed_neighbours_do_not_meet(paged, cuda_device, dtype):
    """infinities and NaN of one prompt reach no row of another"""
    g = torch.Generator(device=cuda_device).manual_seed(3)
    lens, cu = [70, 30, 200, 5], [0, 70, 100, 300, 305]
    q, k, v = (torch.randn(305, h, 128, generator=g, device=cuda_device).to(dtype) for h in (4, 2, 2))
    on = torch.tensor(cu, dtype=torch.int32, device=cuda_device)
    want = paged.sdp_packed(q, k, v, on)
    k[80], v[81], v[299] = math.nan, math.inf, -math.inf
    got = paged.sdp_packed(q, k, v, on)
    for r, bad in enumerate((False, True, True, False)):
        if not bad:
            assert torch.equal(got[cu[r]:cu[r + 1]], want[cu[r]:cu[r + 1]])
    assert bool(torch.isnan(got[99]).any()) and not bool(torch.isfinite(got[299]).any())


# ------------------------------------------------------------------ together, recorded, on other streams
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,eight", [(torch.float16, True), (torch.bfloat16, False)])
def test_a_server(paged, cuda_device, dtype, eight):
    """requests come, run and go: pages are handed out and come back, and every step's attention is that over all of a request's own tokens"""
    dev, heads, kv_heads, dim, page, pages, rows = cuda_device, 8, 2, 64, 8, 60, 5
    g = torch.Generator(device=dev).manual_seed(1)
    on = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)                                 # noqa: E731
    kind = torch.uint8 if eight else dtype
    caches = [torch.full((pages, page, kv_heads, dim), 0x7f, dtype=torch.uint8, device=dev) if eight else torch.full((pages, page, kv_heads, dim), math.nan, dtype=kind, device=dev)
              for _ in range(2)]
    cos, sin = tables(dim, 300, dev)
    table, stack, count = torch.full((rows, 20), -1, dtype=torch.int32, device=dev), torch.arange(pages, dtype=torch.int32, device=dev), on([pages])
    held, past = [0] * rows, [[[], []] for _ in range(rows)]
    plan = [[9, 0, 30, 1, 0], [1, 17, 1, 1, 0], [1, 1, 1, 0, 5], "0", [40, 1, 1, 0, 1], [1, 1, 1, 8, 1], "24", [1, 1, 12, 1, 3], [1, 1, 1, 1, 1]]
    for step in plan:
        if isinstance(step, str):
            done = torch.zeros(rows, dtype=torch.bool, device=dev)
            for r in map(int, step):
                done[r], held[r], past[r] = True, 0, [[], []]
            paged.paged_release(done, table, stack, count)
            continue
        T = sum(step)
        st = paged.paged_step(on(step), on(held), table, stack, count, page, T, free_left=count)
        qkv = torch.randn(T, (heads + 2 * kv_heads) * dim, generator=g, device=dev).to(dtype)
        paged.paged_rope_append(qkv, heads, kv_heads, dim, cos, sin, st.positions, st.slots, *caches)
        x = qkv.view(T, -1, dim)
        got = paged.sdp_paged(x[:, :heads], *caches, table, st.seq_lens, st.cu_seqlens)
        cu = st.cu_seqlens.tolist()
        for r in range(rows):
            for part, first in zip(past[r], (heads, heads + kv_heads)):
                new = x[cu[r]:cu[r + 1], first:first + kv_heads]
                part.append(new.to(torch.float8_e5m2).half() if eight else new)
            held[r] += step[r]
        k, v = ([torch.cat(past[r][i]) for r in range(rows)] for i in (0, 1))
        want, absolute, largest = statement(x[:, :heads], k, v, cu, held, dim ** -0.5)
        assert bool(((got.double() - want).abs() <= bound(want, absolute, largest, dtype, torch.float16 if eight else dtype, dim, 300)).all())
        if held == step and not eight:                          # nobody held anything before: the prompts' own attention says the same
            packed = paged.sdp_packed(x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:], st.cu_seqlens)
            assert bool(((packed.double() - want).abs() <= bound(want, absolute, largest, dtype, dtype, dim, 300)).all())
        assert st.missing.item() == 0 and count.item() == pages - sum(-(-h // page) for h in held)
    paged.paged_release(torch.ones(rows, dtype=torch.bool, device=dev), table, stack, count)
    assert sorted(stack.tolist()) == list(range(pages)) and count.item() == pages


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
def test_a_recorded_step_serves_other_lengths(paged, cuda_device, dtype, eight):
    """one graph of step, write and attention, replayed while the lengths on the device move; two graphs of it do not meet in a workspace"""
    dev, heads, kv_heads, dim, page, R, width = cuda_device, 8, 2, 128, 16, 6, 80
    g = torch.Generator(device=dev).manual_seed(2)
    pages = R * width
    kind = torch.uint8 if eight else dtype
    caches = [torch.randn(pages, page, kv_heads, dim, generator=g, device=dev).to(torch.float8_e5m2).view(torch.uint8) if eight
              else torch.randn(pages, page, kv_heads, dim, generator=g, device=dev).to(kind) for _ in range(2)]
    table = torch.randperm(pages, generator=g, device=dev).to(torch.int32).view(R, width)          # every page handed out: nothing to take
    keep = table.clone()
    stack, count = torch.zeros(1, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    new, held = torch.ones(R, dtype=torch.int32, device=dev), torch.zeros(R, dtype=torch.int32, device=dev)
    qkv = torch.randn(16, (heads + 2 * kv_heads) * dim, generator=g, device=dev).to(dtype)
    cos, sin = tables(dim, 2000, dev)

    def call(x):
        st = paged.paged_step(new, held, table, stack, count, page, 16)
        paged.paged_rope_append(x, heads, kv_heads, dim, cos, sin, st.positions, st.slots, *caches)
        out = torch.zeros(16, heads, dim, dtype=dtype, device=dev)
        return paged.sdp_paged(x.view(16, -1, dim)[:, :heads], *caches, table, st.seq_lens, st.cu_seqlens, out=out, max_query_len=4)

    side, recorded = torch.cuda.Stream(), []
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(qkv.clone())
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        graph, x = torch.cuda.CUDAGraph(), qkv.clone()
        with torch.cuda.graph(graph):
            y = call(x)
        recorded.append((graph, x, y))
    for counts, lens in (([1] * 6, [5, 100, 31, 0, 700, 64]), ([4, 1, 0, 3, 2, 4], [1201, 2, 9, 1, 641, 4]), ([1, 0, 0, 0, 0, 0], [1000, 0, 0, 0, 0, 0])):
        new.copy_(torch.tensor(counts, dtype=torch.int32))
        held.copy_(torch.tensor(lens, dtype=torch.int32))
        # a new token that opens a page gets none here (the stack is empty): its entry becomes -1
        before = [c.clone() for c in caches]
        opens = bool((((held + new + page - 1) // page) > ((held + page - 1) // page)).any())
        for graph, x, y in recorded:
            for c, b in zip(caches, before):
                c.copy_(b)
            table.copy_(keep)
            x.copy_(qkv)
            graph.replay()
        results = [y.clone() for _, _, y in recorded]
        assert torch.equal(*[torch.nan_to_num(r) for r in results])
        for c, b in zip(caches, before):
            c.copy_(b)
        table.copy_(keep)
        want = call(qkv.clone())
        assert torch.equal(torch.nan_to_num(want), torch.nan_to_num(results[0])) and (opens or not bool(torch.isnan(want[:sum(counts)]).any()))


@pytest.mark.gpu
def test_the_python_statements_say_the_same(paged, cuda_device, monkeypatch):
    """what serves where the native host side is not to be had, a lone token with any stride among it"""
    dev = cuda_device
    on = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)                                 # noqa: E731
    results = []
    for native in (True, False):
        if not native:
            monkeypatch.setattr(paged, "_native", lambda *args: None)
        g = torch.Generator(device=dev).manual_seed(8)
        for T in (1, 5):
            table, free, count = torch.full((1, 4), -1, dtype=torch.int32, device=dev), on([3, 1, 0, 2]), on([4])
            st = paged.paged_step(on([T]), on([0]), table, free, count, 2, T)
            cos, sin = tables(64, 50, dev)
            caches = [torch.zeros(4, 2, 2, 64, dtype=torch.float16, device=dev) for _ in range(2)]
            qkv = torch.randn(T, 8 * 64, generator=g, device=dev).half()
            if T == 1:
                qkv = qkv.as_strided((1, 512), (1, 1))
            paged.paged_rope_append(qkv, 4, 2, 64, cos, sin, st.positions, st.slots, *caches)
            x = qkv.view(T, 8, 64)
            results.append((*st, table, qkv.clone(), *caches, paged.sdp_paged(x[:, :4], *caches, table, st.seq_lens, st.cu_seqlens, max_query_len=T),
                            paged.sdp_packed(x[:, :4], x[:, 4:6], x[:, 6:], st.cu_seqlens)))
    for a, b in ((results[0], results[2]), (results[1], results[3])):
        assert all(torch.equal(x, y) for x, y in zip(a, b)) and len(a) == len(b)


@pytest.mark.gpu
def test_on_other_streams_at_once(paged, cuda_device):
    """two streams, other lengths on each, many calls in flight: every result is that of the call alone"""
    sets = [requests(cuda_device, new, held, 8, 2, 128, torch.bfloat16, eight, 16, seed=i)
            for i, (new, held, eight) in enumerate([([1] * 5, [3000, 20, 700, 1, 90], False), ([300, 1], [20, 900], False), ([1, 1], [5000, 6], True)])]
    call = lambda s: paged.sdp_paged(s[0], *s[1], s[2], s[3], s[4])                               # noqa: E731
    want = [call(s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [[] for _ in sets]
    for _ in range(20):
        for stream, s, keep in zip(streams, sets, got):
            with torch.cuda.stream(stream):
                keep.append(call(s))
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for keep, w in zip(got, want) for x in keep)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
@pytest.mark.parametrize("new,held", [([1, 1], [20, 7000]), ([2, 300], [700, 5000])])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 1, 64), (64, 1, 128), (256, 1, 128), (128, 1, 256)])
def test_many_heads_on_one(paged, cuda_device, dtype, eight, new, held, heads, kv_heads, dim):
    """a kv head's keys in the parts of many blocks, for 16 rows and more, up to the most heads that there may be; a hint beyond all rows is no hint"""
    check_paged(paged, cuda_device, new, held, heads, kv_heads, dim, dtype, eight, 16, hint=1 << 62)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
@pytest.mark.parametrize("new,rows", [([3, 9], 5), ([40, 300, 7], 200), ([1, 1, 1], 2)])
def test_tokens_behind_the_last_row(paged, cuda_device, dtype, eight, new, rows):
    """a list that names more rows than there are: those that are there see the keys that they would see with the others"""
    q, caches, table, lens, cu = requests(cuda_device, new, [100 + 30 * i for i in range(len(new))], 4, 2, 64, dtype, eight, 16)[:5]
    there = cu.clamp(max=rows)
    fewer = lens - (cu - there).diff()
    want = paged.sdp_paged(q[:rows], *caches, table, fewer, there)
    assert torch.equal(paged.sdp_paged(q[:rows], *caches, table, lens, cu), want) and not bool(torch.isnan(want).any())


# ------------------------------------------------------------------ what is rounded, and what is not
# P enters its product as two values of type t, the second with what the rounding of the first left: h(t)^2 of itself is lost, and nothing else but
# the result is rounded.  In fp16 neither part has bits below 2^-24, half of which a stored value may be off by; a row's largest key is stored as
# at least 2^LIFT, so that moves the output by up to 2^(-25 - LIFT) sum |v|.
# Queries and keys are small whole numbers here: the scores' sums are exact in 32 bits, and what is left is the exponent e = score log2(e), whose
# factor is off by 2^-23 of itself and which is rounded (with up to 16 beside it) once in the exponential and once whenever the row's reference moves:
# by more than 2^4 each time, and where the parts of warps and blocks meet (2).
LIFT = 11


def bound_once(want, absolute, steepest, v_sum, dtype, p_dtype, keys):
    e = 1.4427 * steepest
    score = 2.0 ** -22 + 0.7 * (e * 2.0 ** -23 + (2 * e + 16) * 2.0 ** -24 * (3 + 2 * e / 4))
    lost = HALF[p_dtype] ** 2 * absolute + (2.0 ** (-25 - LIFT) * v_sum if p_dtype == torch.float16 else 0)
    # an output of fp16 has no bits below 2^-24 either
    return HALF[dtype] * want.abs() + 2.0 ** -25 + (1 + HALF[dtype]) * (lost + (2 * score + (keys / 8 + 8) * 2.0 ** -23) * absolute)


def check_once(got, q, k, v, cu, lens, scale, dtype, p_dtype, causal=True):
    heads = q.shape[1]
    want, absolute, _ = statement(q, k, v, cu, lens, scale, causal)
    steepest = max(float(torch.einsum("ihd,jhd->hij", q[a:b].double(), x.double().repeat_interleave(heads // x.shape[1], 1)).abs().max()) * scale
                   for x, a, b in zip(k, cu, cu[1:]))
    v_sum = torch.cat([x.double().abs().sum(0).repeat_interleave(heads // x.shape[1], 0)[None].expand(b - a, -1, -1) for x, a, b in zip(v, cu, cu[1:])])
    limit = bound_once(want, absolute, steepest, v_sum, dtype, p_dtype, max(lens))
    return float(((got.double() - want).abs() / limit).max())


def whole(x):
    return x.float().round().clamp(-4, 4).to(x.dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 128), (8, 1, 64), (16, 1, 128), (6, 2, 256), (5, 5, 16), (12, 1, 96)])
@pytest.mark.parametrize("new,held,page", [([1, 1, 1], [30, 150, 7], 16), ([1], [150], 1), ([1], [900], 32), ([1, 3, 1], [100, 90, 33], 24)])
def test_tokens_round_the_result_alone(paged, cuda_device, dtype, eight, heads, kv_heads, dim, new, held, page):
    """values that nearly cancel, so that the weights' own error is not behind the result's rounding; up to 8 rows a request, and up to 16"""
    new = [min(n, 16 * kv_heads // heads) for n in new]
    q, caches, table, lens, cu, rows, cu_list, len_list = requests(cuda_device, new, held, heads, kv_heads, dim, dtype, eight, page)
    q, kind = whole(q), torch.float8_e5m2 if eight else dtype
    turned = [[whole(x) for x in rows[0]], [(x.float() + 8 - 16 * (torch.arange(len(x), device=cuda_device) % 2)[:, None, None]).to(kind) for x in rows[1]]]
    for cache, part in zip(caches, turned):
        for r, x in enumerate(part):
            j = torch.arange(len(x), device=cuda_device)
            cache[table[r, j // page].long(), j % page] = x.view(torch.uint8) if eight else x
    k, v = ([x.half() if eight else x for x in part] for part in turned)
    scale = 0.25 * dim ** -0.5
    got = paged.sdp_paged(q, *caches, table, lens, cu, scale, max_query_len=max(new))
    assert check_once(got, q, k, v, cu_list, len_list, scale, dtype, torch.float16 if eight else dtype) <= 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (8, 1, 64), (6, 2, 256)])
@pytest.mark.parametrize("new,held,page", [([130], [0], 16), ([70, 200], [30, 20], 24), ([40], [100], 4), ([150], [800], 32)])
def test_chunks_round_the_result_alone(paged, cuda_device, dtype, eight, heads, kv_heads, dim, new, held, page):
    q, caches, table, lens, cu, rows, cu_list, len_list = requests(cuda_device, new, held, heads, kv_heads, dim, dtype, eight, page)
    q, keys = whole(q), caches[0].view(torch.float8_e5m2) if eight else caches[0]
    caches[0] = whole(keys).view(torch.uint8) if eight else whole(keys)
    k, v = ([x.half() if eight else x for x in part] for part in (map(whole, rows[0]), rows[1]))
    scale = 0.25 * dim ** -0.5
    got = paged.sdp_paged(q, *caches, table, lens, cu, scale)
    assert check_once(got, q, k, v, cu_list, len_list, scale, dtype, torch.float16 if eight else dtype) <= 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads,dim,lens", [(8, 2, 128, [500, 33, 157]), (4, 4, 64, [200]), (3, 1, 256, [90, 140])])
@pytest.mark.parametrize("causal", [True, False])
def test_prompts_round_the_result_alone(paged, cuda_device, dtype, heads, kv_heads, dim, lens, causal):
    g = torch.Generator(device=cuda_device).manual_seed(dim)
    q, k, v = (1.5 * torch.randn(sum(lens), heads + 2 * kv_heads, dim, generator=g, device=cuda_device)).to(dtype).split([heads, kv_heads, kv_heads], 1)
    q, k, cu, scale = whole(q), whole(k), [0], 0.25 * dim ** -0.5
    for n in lens:
        cu.append(cu[-1] + n)
    got = paged.sdp_packed(q, k, v, torch.tensor(cu, dtype=torch.int32, device=cuda_device), scale, is_causal=causal)
    k, v = ([t[a:b] for a, b in zip(cu, cu[1:])] for t in (k, v))
    assert check_once(got, q, k, v, cu, lens, scale, dtype, dtype, causal) <= 1


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("keys", [30, 150])
@pytest.mark.parametrize("cancel", [0, 8])
def test_the_bound_tells_probabilities_of_one_value(dtype, keys, cancel):
    """an oracle that rounds its probabilities once is outside it, one that keeps what that left is inside"""
    g = torch.Generator().manual_seed(keys)
    q, k, v = ((1.5 * torch.randn(n, 2, 128, generator=g)).to(dtype) for n in (40, keys, keys))
    q, k, scale = whole(q), whole(k), 0.25 * 128 ** -0.5
    v = (v.float() + cancel - 2 * cancel * (torch.arange(keys) % 2)[:, None, None]).to(dtype)
    s = torch.einsum("ihd,jhd->hij", q.float(), k.float()) * scale
    p = torch.exp(s - s.amax(-1, keepdim=True))
    high = p.to(dtype).float()
    for parts, inside in ((high, False), (high + (p - high).to(dtype).float(), True)):
        o = (torch.einsum("hij,jhd->ihd", parts, v.float()) / p.sum(-1).t()[..., None]).to(dtype)
        assert (check_once(o, q, [k], [v], [0, 40], [keys], scale, dtype, dtype, False) <= 1) == inside


def one_key_above(dev, lens, kv_heads, dim, dtype, depths, sink):
    """keys and values of every request: key ``sink`` with a value of zero, the others ``depths`` nats below it (in turn) with values of 16000 to 49000"""
    g = torch.Generator(device=dev).manual_seed(sum(lens))
    k, v = [], []
    for n in lens:
        x = torch.zeros(n, kv_heads, dim, device=dev)
        x[..., 0] = -torch.tensor(depths, device=dev, dtype=torch.float32)[torch.arange(n, device=dev) % len(depths)][:, None]
        y = 16384 * (1 + 2 * torch.rand(n, kv_heads, dim, generator=g, device=dev))
        x[min(sink, n - 1)], y[min(sink, n - 1)] = 0, 0
        k.append(x.to(dtype))
        v.append(y.to(dtype))
    return k, v


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
@pytest.mark.parametrize("depths", [[14.0], [20.0], [24.0], [12.0, 14.0, 16.0, 20.0, 24.0]])
@pytest.mark.parametrize("new,held,heads,kv_heads,page", [([1], [500], 4, 4, 16), ([1, 1], [3000, 700], 8, 1, 24), ([1, 1], [900, 40], 16, 1, 16), ([40], [1000], 4, 2, 16), ([200, 90], [0, 300], 8, 2, 4)])
def test_keys_far_below_the_largest_count(paged, cuda_device, dtype, eight, depths, new, held, heads, kv_heads, page):
    """a key that takes nearly all of the weight and gives nothing: the output is that of the others, 2^-17 to 2^-35 of it each"""
    dim, lens, cu = 64, [h + n for h, n in zip(held, new)], [0]
    for n in new:
        cu.append(cu[-1] + n)
    q, caches, table, lens_on, cu_on = requests(cuda_device, new, held, heads, kv_heads, dim, dtype, eight, page)[:5]
    q = torch.zeros_like(q)
    q[..., 0] = 1
    k, v = one_key_above(cuda_device, lens, kv_heads, dim, torch.float8_e5m2 if eight else dtype, depths, 3)
    for r, n in enumerate(lens):
        j = torch.arange(n, device=cuda_device)
        for cache, x in zip(caches, (k[r], v[r])):
            cache[table[r, j // page].long(), j % page] = x.view(torch.uint8) if eight else x
    if eight:
        k, v = ([x.half() for x in part] for part in (k, v))
    got = paged.sdp_paged(q, *caches, table, lens_on, cu_on, 1.0, max_query_len=max(new))
    assert check_once(got, q, k, v, cu, lens, 1.0, dtype, torch.float16 if eight else dtype) <= 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("depths", [[20.0], [24.0], [12.0, 14.0, 16.0, 20.0, 24.0]])
@pytest.mark.parametrize("causal", [True, False])
def test_keys_far_below_the_largest_count_in_prompts(paged, cuda_device, dtype, depths, causal):
    lens, cu = [700, 60], [0, 700, 760]
    k, v = one_key_above(cuda_device, lens, 2, 64, dtype, depths, 0)
    q = torch.zeros(760, 4, 64, dtype=dtype, device=cuda_device)
    q[..., 0] = 1
    got = paged.sdp_packed(q, torch.cat(k), torch.cat(v), torch.tensor(cu, dtype=torch.int32, device=cuda_device), 1.0, is_causal=causal)
    assert check_once(got, q, k, v, cu, lens, 1.0, dtype, dtype, causal) <= 1


# ------------------------------------------------------------------ waits
def waiting_calls(paged, dev):
    t, b = torch.float16, torch.bfloat16
    sets = {"tokens": requests(dev, [1] * 40, [2500] * 40, 8, 2, 128, b, False, 16), "tokens, e5m2": requests(dev, [1] * 40, [2500] * 40, 8, 2, 128, t, True, 16),
            "chunk": requests(dev, [600], [3000], 8, 2, 128, b, False, 16), "chunk, e5m2": requests(dev, [600], [3000], 8, 2, 128, b, True, 16),
            "chunk without boxes": requests(dev, [600], [3000], 8, 2, 64, t, False, 4)}
    calls = {name: lambda s=s: paged.sdp_paged(s[0], *s[1], s[2], s[3], s[4]) for name, s in sets.items()}
    q = torch.randn(3000, 12, 64, generator=torch.Generator(device=dev).manual_seed(4), device=dev).to(t)
    cu = torch.tensor([0, 900, 3000], dtype=torch.int32, device=dev)
    return {**calls, "prompts": lambda: paged.sdp_packed(q[:, :4], q[:, 4:8], q[:, 8:], cu)}


WAITING = ["tokens", "tokens, e5m2", "chunk", "chunk, e5m2", "chunk without boxes", "prompts"]


@pytest.mark.gpu
@pytest.mark.parametrize("clocks", [20, 100000])
@pytest.mark.parametrize("name", WAITING)
def test_a_wait_that_runs_out_is_reported_once(paged, native_lib, cuda_device, name, clocks):
    """below zero half of a launch's copies never come, and the waits for them run out after that many clocks; the next call says so, and
    the one after is right"""
    call = waiting_calls(paged, cuda_device)[name]
    want = call()
    assert not native_lib.lowbit_gemm_wait_expired()
    native_lib._lib.lowbit_debug_set_wait_limit(-clocks)
    try:
        call()
    finally:
        native_lib._lib.lowbit_debug_set_wait_limit(0)
    assert native_lib.lowbit_gemm_wait_expired()
    with pytest.raises(native_lib.LowBitNativeError, match="ran out"):
        call()
    assert not native_lib.lowbit_gemm_wait_expired()
    assert torch.equal(call(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("clocks", [1, 300, 1500, 6000, 30000])
@pytest.mark.parametrize("name", WAITING)
def test_wherever_a_wait_runs_out_the_next_call_is_right(paged, native_lib, cuda_device, name, clocks):
    """limits of the order of the kernels' own waits: they run out in the middle of the work, or not at all"""
    call = waiting_calls(paged, cuda_device)[name]
    want = call()
    for _ in range(2):
        native_lib._lib.lowbit_debug_set_wait_limit(clocks)
        try:
            call()
        except native_lib.LowBitNativeError as e:
            assert "ran out" in str(e)
        finally:
            native_lib._lib.lowbit_debug_set_wait_limit(0)
        if native_lib.lowbit_gemm_wait_expired():
            with pytest.raises(native_lib.LowBitNativeError, match="ran out"):
                call()
            torch.cuda.synchronize()
        assert torch.equal(call(), want)


# ------------------------------------------------------------------ what is refused
def test_refusals_without_a_device(native_lib):
    """bad arguments are refused before anything touches a device"""
    lib, p = native_lib._lib, ctypes.cast(ctypes.create_string_buffer(4096 + 16), ctypes.c_void_p)
    p = ctypes.c_void_p(p.value + 15 & ~15)
    s2, s3, odd = (ctypes.c_int64 * 2)(256, 64), (ctypes.c_int64 * 3)(1024, 64, 64), (ctypes.c_int64 * 2)(256, 65)

    def refused(rc, needle):
        msg = lib.b200_lowbit_last_error_string().decode()
        lib.b200_lowbit_clear_error()
        return rc != 0 and needle in msg

    step = lambda R=2, width=4, stride=4, pages=8, page=16, n=3, table=p: lib.lowbit_paged_step_cuda(               # noqa: E731
        p, p, R, table, stride, width, p, pages, p, p, page, n, p, p, p, p, p, None)
    for bad in (dict(R=0), dict(width=0), dict(stride=3), dict(pages=0), dict(page=0), dict(n=-1), dict(table=None)):
        assert refused(step(**bad), "lowbit_paged_step_cuda"), bad
    assert refused(lib.lowbit_paged_release_cuda(p, 0, p, 4, 4, p, 8, p, None), "lowbit_paged_release_cuda")
    append = lambda dtype=1, cache=1, T=3, heads=2, kv=1, dim=64, rotary=64, cos=p, stride=256, pages=4: lib.lowbit_paged_rope_append_cuda(   # noqa: E731
        p, dtype, stride, T, heads, kv, dim, rotary, cos, p, 0, 64, 10, p, p, p, s3, p, s3, cache, pages, 16, None)
    for bad in (dict(dtype=0, cache=0), dict(cache=2), dict(kv=0), dict(rotary=66), dict(rotary=31), dict(cos=None), dict(stride=255), dict(pages=0), dict(T=-1)):
        assert refused(append(**bad), "lowbit_paged_rope_append_cuda"), bad

    def attend(q=p, dtype=1, q_strides=s2, T=4, cache=1, pages=4, page=16, table=p, width=2, R=2, heads=4, kv=2, dim=64, scale=0.1):
        return lib.lowbit_sdp_paged_cuda(q, dtype, q_strides, T, p, s3, p, s3, cache, pages, page, table, width, width, p, p, R, heads, kv, dim, scale, T, p, s2, p, 0, None)
    for bad in (dict(q=None), dict(dtype=0, cache=0), dict(cache=2), dict(cache=0), dict(q_strides=odd), dict(T=-1), dict(pages=0), dict(page=0), dict(table=None), dict(width=0),
                dict(R=0), dict(kv=3), dict(dim=72), dict(dim=272), dict(scale=0.0), dict(scale=math.nan), dict(page=1 << 30), dict(q=ctypes.c_void_p(p.value + 2))):
        assert refused(attend(**bad), "lowbit_sdp_paged_cuda"), bad

    def packed(q=p, dtype=1, strides=s2, T=4, R=2, heads=4, kv=2, dim=64, scale=0.1):
        return lib.lowbit_sdp_packed_cuda(q, dtype, strides, T, p, strides, p, strides, p, R, heads, kv, dim, scale, 1, T, p, s2, p, 0, None)
    for bad in (dict(q=None), dict(dtype=0), dict(dtype=19), dict(strides=odd), dict(T=-1), dict(T=1 << 31), dict(R=0), dict(heads=5), dict(dim=24), dict(scale=-1.0)):
        assert refused(packed(**bad), "lowbit_sdp_packed_cuda"), bad


def test_refusals_on_the_cpu(paged):
    i = lambda *n: torch.zeros(n, dtype=torch.int32)                                              # noqa: E731
    x = torch.zeros(2, 4, 64, dtype=torch.float16)
    c = torch.zeros(3, 16, 4, 64, dtype=torch.float16)
    for call in (lambda: paged.paged_step(i(2), i(2), i(2, 4), i(5), i(1), 16, 2), lambda: paged.paged_release(torch.zeros(2, dtype=torch.bool), i(2, 4), i(5), i(1)),
                 lambda: paged.paged_rope_append(x.view(2, 256), 2, 1, 64, None, None, None, torch.zeros(2, dtype=torch.int64), c[:, :, :1], c[:, :, :1]),
                 lambda: paged.sdp_paged(x, c, c, i(2, 4), i(2), i(3)), lambda: paged.sdp_packed(x, x, x, i(3))):
        with pytest.raises(RuntimeError, match="CUDA device"):
            call()
    for t in (x.float().requires_grad_(), x.clone().requires_grad_()):
        with pytest.raises(RuntimeError, match="backward"):
            paged.sdp_packed(t, x, x, i(3))


def derivatives(paged, dev):
    """(name, call): every operator with each of its tensors in turn wanting a gradient (``wants``) or carrying a tangent"""
    fw = torch.autograd.forward_ad
    i = lambda *n: torch.zeros(n, dtype=torch.int32, device=dev)                                  # noqa: E731
    h = lambda *n: torch.zeros(n, dtype=torch.float16, device=dev)                                # noqa: E731
    at = torch.zeros(6, dtype=torch.int64, device=dev)
    append = lambda qkv, k, v, cos, sin: paged.paged_rope_append(qkv, 4, 2, 64, cos, sin, at, at, k, v)              # noqa: E731
    attend = lambda q, k, v, out: paged.sdp_paged(q, k, v, i(2, 4), i(2), i(3), out=out)                               # noqa: E731
    packed = lambda q, k, v, out: paged.sdp_packed(q, k, v, i(3), out=out)                                            # noqa: E731
    q, c, p = h(6, 4, 64), h(3, 16, 2, 64), h(6, 2, 64)
    for name, call, tensors in (("append", append, (h(6, 512), c, c, h(9, 64), h(9, 64))), ("paged", attend, (q, c, c, h(6, 4, 64))), ("packed", packed, (q, p, p, h(6, 4, 64))),
                                ("paged, plain", lambda *t: attend(*t, None), (q, c, c)), ("packed, plain", lambda *t: packed(*t, None), (q, p, p))):
        for n in range(len(tensors)):
            def run(change, call=call, tensors=tensors, n=n):
                return call(*(change(t) if j == n else t.clone() for j, t in enumerate(tensors)))
            yield f"{name} {n}", lambda run=run: run(lambda t: t.clone().requires_grad_()), lambda run=run: run(lambda t: fw.make_dual(t.clone(), torch.ones_like(t)))


def check_derivatives(paged, dev):
    for name, wants, carries in derivatives(paged, dev):
        with pytest.raises(RuntimeError, match="backward"):
            wants()
            pytest.fail(name)
        for mode in (torch.enable_grad, torch.no_grad):                                           # no_grad does not end forward mode
            with mode(), torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="tangent"):
                carries()
                pytest.fail(name)


def test_what_would_need_a_derivative_is_refused_on_the_cpu(paged):
    check_derivatives(paged, "cpu")


@pytest.mark.gpu
def test_what_would_need_a_derivative_is_refused(paged, cuda_device):
    check_derivatives(paged, cuda_device)
    for _, wants, _ in derivatives(paged, cuda_device):
        with torch.no_grad():
            wants()


def test_what_a_row_keeps_is_refused_without_a_device(native_lib, paged):
    lib, p = native_lib._lib, ctypes.cast(ctypes.create_string_buffer(4096), ctypes.c_void_p)
    behind = lambda done=p, held=p, R=2, stride=4, width=4, page=16, pages=8, table=p: lib.lowbit_paged_release_behind_cuda(   # noqa: E731
        done, held, R, table, stride, width, page, p, pages, p, None)
    for bad in (dict(done=None), dict(held=None), dict(R=0), dict(stride=3), dict(width=0), dict(page=0), dict(pages=0), dict(table=None)):
        assert behind(**bad) != 0 and "lowbit_paged_release_behind_cuda" in lib.b200_lowbit_last_error_string().decode(), bad
        lib.b200_lowbit_clear_error()


@pytest.mark.gpu
def test_what_a_row_keeps_is_refused(paged, cuda_device):
    i = lambda *n: torch.zeros(n, dtype=torch.int32, device=cuda_device)                          # noqa: E731
    done = torch.zeros(2, dtype=torch.bool, device=cuda_device)
    for held, page in ((i(2), None), (None, 16), (i(3), 16), (i(2).long(), 16), (i(2), 0), (i(2).cpu(), 16)):
        with pytest.raises(RuntimeError):
            paged.paged_release(done, i(2, 4), i(5), i(1), held, page)


@pytest.mark.gpu
def test_refusals(paged, cuda_device):
    dev = cuda_device
    i = lambda *n: torch.zeros(n, dtype=torch.int32, device=dev)                                  # noqa: E731
    h = lambda *n: torch.zeros(n, dtype=torch.float16, device=dev)                                # noqa: E731
    q, c, table, lens, cu = h(6, 4, 64), h(3, 16, 2, 64), i(2, 4), i(2), i(3)
    bad = [lambda: paged.paged_step(i(2), i(3), table, i(5), i(1), 16, 2), lambda: paged.paged_step(i(2), i(2).long(), table, i(5), i(1), 16, 2),
           lambda: paged.paged_step(i(2), i(2), table.t(), i(5), i(1), 16, 2), lambda: paged.paged_step(i(2), i(2), i(3, 4), i(5), i(1), 16, 2),
           lambda: paged.paged_step(i(2), i(2), table, i(5), i(1), 0, 2), lambda: paged.paged_step(i(2), i(2), table, i(5), i(1).cpu(), 16, 2),
           lambda: paged.paged_step(i(0), i(0), i(0, 4), i(5), i(1), 16, 2), lambda: paged.paged_step(i(2), i(2), table, i(5), i(1), 16, -1),
           lambda: paged.paged_release(i(2), table, i(5), i(1)), lambda: paged.paged_release(torch.zeros(3, dtype=torch.bool, device=dev), table, i(5), i(1)),
           lambda: paged.sdp_paged(q.float(), c.float(), c.float(), table, lens, cu), lambda: paged.sdp_paged(q, c.bfloat16(), c.bfloat16(), table, lens, cu),
           lambda: paged.sdp_paged(q, c, c[:, :, :1], table, lens, cu), lambda: paged.sdp_paged(q, c[..., :32], c[..., :32], table, lens, cu),
           lambda: paged.sdp_paged(h(6, 3, 64), c, c, table, lens, cu), lambda: paged.sdp_paged(h(6, 4, 72), h(3, 16, 2, 72), h(3, 16, 2, 72), table, lens, cu),
           lambda: paged.sdp_paged(h(6, 4, 272), h(3, 16, 2, 272), h(3, 16, 2, 272), table, lens, cu), lambda: paged.sdp_paged(q, c, c, table, i(3), cu),
           lambda: paged.sdp_paged(q, c, c, table, lens, i(4)), lambda: paged.sdp_paged(q, c, c, table, lens, cu.long()), lambda: paged.sdp_paged(q, c, c, table, lens, cu, scale=0.0),
           lambda: paged.sdp_paged(q, c, c, table, lens, cu, out=h(6, 4, 32)), lambda: paged.sdp_paged(q, c, c, table, lens, cu, max_query_len=-1),
           lambda: paged.sdp_paged(q, c, c, table.long(), lens, cu), lambda: paged.sdp_paged(q, c, c, table, lens.cpu(), cu),
           lambda: paged.sdp_paged(q, h(3, 16, 2, 68)[..., :64], c, table, lens, cu),
           lambda: paged.sdp_packed(q, h(5, 2, 64), h(5, 2, 64), cu), lambda: paged.sdp_packed(q, h(6, 3, 64), h(6, 3, 64), cu), lambda: paged.sdp_packed(q, h(6, 2, 64), h(6, 2, 64).bfloat16(), cu),
           lambda: paged.paged_rope_append(h(6, 512), 4, 2, 64, None, None, None, torch.zeros(5, dtype=torch.int64, device=dev), c, c),
           lambda: paged.paged_rope_append(h(6, 500), 4, 2, 64, None, None, None, torch.zeros(6, dtype=torch.int64, device=dev), c, c),
           lambda: paged.paged_rope_append(h(1, 512).expand(6, 512), 4, 2, 64, None, None, None, torch.zeros(6, dtype=torch.int64, device=dev), c, c),
           lambda: paged.paged_rope_append(h(6, 512), 4, 2, 64, h(9, 66), h(9, 66), torch.zeros(6, dtype=torch.int64, device=dev), torch.zeros(6, dtype=torch.int64, device=dev), c, c)]
    for n, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {n} was taken")
    wants = c.clone().requires_grad_()
    for call in (lambda: paged.sdp_paged(q, wants, c, table, lens, cu), lambda: paged.sdp_paged(q, c, wants, table, lens, cu)):
        with pytest.raises(RuntimeError, match="backward"):
            call()
    wide = h(6, 514, 64)                                                                          # more heads on one than a unit has rows
    for call in (lambda: paged.sdp_paged(wide, h(3, 16, 2, 64), h(3, 16, 2, 64), table, lens, cu), lambda: paged.sdp_packed(wide, q[:, :2], q[:, :2], cu)):
        with pytest.raises(RuntimeError, match="bad argument"):
            call()
    assert paged.sdp_paged(q[:0], c, c, table, lens, cu).shape == (0, 4, 64) and paged.sdp_packed(q[:0], q[:0], q[:0], cu).shape == (0, 4, 64)
