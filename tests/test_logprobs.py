"""Log probabilities of tokens (transformers/logprobs.py) against 64-bit statements.

Bounds.  The exponent of an element is one multiply-add of the logit and the factor log2 e / temperature, which is itself rounded: off by 2^-22 of the
largest |z| / temperature of its row in all; the power adds 2^-22 and the sum of a row's V powers one rounding, 2^-24, for each of the V / 256 / 4 pieces
that a thread adds up and some 40 where threads and blocks meet.  A log probability is off by that sum; an entropy by the same, weighted with the mean distance
of an exponent from the reference, below H + 40 (the reference follows the maximum within 2^4, and the sum is below 2^32); a gradient by that of its
probabilities, and is rounded once, finfo(t).eps / 2."""
import math

import pytest
import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TYPES = list(HALF)


@pytest.fixture(scope="module")
def lp(native_lib):
    from ipex_llm_b200.transformers import logprobs
    return logprobs


def statement(logits, tokens, k, temperature):
    z = logits.detach().double() / temperature
    q = torch.log_softmax(z, -1)
    w = q.exp()
    h = torch.special.entr(w).sum(-1)
    here = (tokens >= 0) & (tokens < z.shape[-1])
    token = torch.where(here, q.gather(-1, tokens.clamp(0, z.shape[-1] - 1)[..., None])[..., 0], 0.0)
    ids = torch.sort(logits.detach().double(), dim=-1, descending=True, stable=True).indices[..., :k]
    return q, w, h, token, ids, q.gather(-1, ids)


def slack(logits, temperature):
    """of a log probability, by row"""
    z = logits.detach().double() / temperature
    z = torch.where(torch.isinf(z) | (z.abs() > 1e30), 0.0, z).abs().amax(-1)
    return 2.0 ** -22 * (z + 4) + 2.0 ** -24 * (logits.shape[-1] / 1024 + 40)


def check(got, logits, tokens, k, temperature):
    q, w, h, token, ids, top = statement(logits, tokens, k, temperature)
    tol = slack(logits, temperature)
    near = lambda a, b, t: (a.double() == b) | ((a.double() - b).abs() <= t + 2.0 ** -23 * b.abs())       # noqa: E731  equal: infinities too
    assert bool(near(got.logprobs, token, tol).all())
    assert bool(((got.entropy.double() - h).abs() <= tol * (h + 40)).all())
    if k:
        assert torch.equal(got.top_ids, ids)
        assert bool(near(got.top_logprobs, top, tol[..., None]).all())
    else:
        assert got.top_ids is None and got.top_logprobs is None


def make(rows, V, dtype, dev, masked=0.0, spread=3.0, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + rows * 7 + V)
    logits = (spread * torch.randn(rows, V, generator=g, device=dev)).to(dtype)
    tokens = torch.randint(0, V, (rows,), generator=g, device=dev)
    if masked:
        out = torch.rand(rows, V, generator=g, device=dev) < masked
        logits.masked_fill_(out, -math.inf)
        logits[:, 0] = 0.5                                             # something is left in every row
    if rows > 2:
        tokens[1], tokens[2] = -100, V
    return logits, tokens


SIZES = [(1, 1), (1, 7), (3, 40), (2, 999), (5, 2048), (1, 32000), (33, 4099), (700, 2056), (2, 128256), (9, 50257)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", SIZES)
@pytest.mark.parametrize("k,temperature,masked", [(0, 1.0, 0.0), (1, 0.7, 0.3), (5, 1.0, 0.0), (20, 1.5, 0.9), (32, 0.3, 0.0)])
def test_values(lp, cuda_device, dtype, rows, V, k, temperature, masked):
    logits, tokens = make(rows, V, dtype, cuda_device, masked)
    k = min(k, V)
    check(lp.token_logprobs(logits, tokens, k, temperature), logits, tokens, k, temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [50, 999, 20000, 70000])
@pytest.mark.parametrize("shape", ["even", "rising", "falling", "few values", "in one thread", "even but one", "all but two masked", "signs of zero", "pairs"])
def test_orders_and_ties(lp, cuda_device, dtype, V, shape):
    """the alternatives of rows where the largest lie together, are many or are equal"""
    i = torch.arange(V, device=cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(V)
    rows = {"even": torch.zeros(V, device=cuda_device), "rising": i / V * 8, "falling": -i / V * 8, "few values": torch.randint(0, 3, (V,), generator=g, device=cuda_device).float(),
            "in one thread": (i // 8 % 256 == 3).float() * 5 + i / V, "even but one": (i == V - 1).float(), "signs of zero": torch.where(i % 2 == 0, 0.0, -0.0),
            "all but two masked": torch.where((i == 11) | (i == V - 3), 1.0, -math.inf), "pairs": torch.randint(0, V // 2, (V,), generator=g, device=cuda_device).float() / V}
    logits = torch.stack([rows[shape], rows[shape].flip(0)]).to(dtype)
    tokens = torch.tensor([11, V - 12], device=cuda_device)
    for k in (1, 20, 32):
        check(lp.token_logprobs(logits, tokens, k, 1.0), logits, tokens, k, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [300, 40001])
@pytest.mark.parametrize("low", [-1e4, -1e9, -1e12, -1e25, -1e29, -3e30, -1e37])
def test_masks_of_large_numbers(lp, cuda_device, dtype, V, low):
    """what masks are written with: numbers whose exponents have lost their differences, in front of the others, behind them, and alone"""
    logits, tokens = make(6, V, dtype, cuda_device)
    logits[0, :V // 2] = low
    logits[1, V // 2:] = low
    logits[2, torch.arange(V, device=cuda_device) % 3 > 0] = low
    logits[3] = low
    logits[4] = low
    logits[4, V // 3] = low / 2
    logits[5, 1:] = low
    tokens[:] = V // 3
    check(lp.token_logprobs(logits, tokens, 9, 1.0), logits, tokens, 9, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [1e-7, 1e-3, 30.0, 1e7])
@pytest.mark.parametrize("dtype", TYPES)
def test_temperatures(lp, cuda_device, dtype, temperature):
    logits, tokens = make(5, 3001, dtype, cuda_device, masked=0.3)
    logits[3] = torch.finfo(dtype).min
    logits[4, 7:] = torch.finfo(dtype).min
    logits[4, :7] = torch.arange(7) / 8
    tokens[3:] = 5
    check(lp.token_logprobs(logits, tokens, 6, temperature), logits, tokens, 6, temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [300, 40001])
def test_masks_infinities_and_nan(lp, cuda_device, dtype, V):
    low = torch.finfo(dtype).min
    logits, tokens = make(9, V, dtype, cuda_device)
    logits[0, 5:] = -math.inf
    logits[1, 5:] = low                                                # masks of the type's lowest value
    logits[2] = low                                                    # ... that leave nothing: the row is even
    logits[3] = -math.inf
    logits[4, V // 2] = math.nan
    logits[5, V - 1] = math.inf
    logits[6] = math.nan
    logits[7] = torch.finfo(dtype).max / 2
    tokens[:] = 3
    k = 7
    got = lp.token_logprobs(logits, tokens, k, 1.0)
    fine = torch.tensor([0, 1, 2, 7, 8], device=cuda_device)
    check(lp.TokenLogprobs(*(t[fine] for t in got)), logits[fine], tokens[fine], k, 1.0)
    for row in (3, 4, 5, 6):
        assert all(bool(torch.isnan(t[row]).all()) for t in (got.logprobs, got.entropy, got.top_logprobs)), row
        ids = got.top_ids[row].tolist()
        assert all(-1 <= i < V for i in ids) and len({i for i in ids if i >= 0}) == len([i for i in ids if i >= 0])
    assert got.top_ids[3].tolist() == list(range(k)) and got.top_ids[6].tolist() == [-1] * k
    token = lp.token_logprobs(logits[:1], tokens[:1] + 100, 0, 1.0)     # a token that cannot come
    assert token.logprobs.item() == -math.inf


def gradient(logits, tokens, ids, k, temperature, gs):
    """64 bits: the gradient, and the absolute sums that its rounding errors are of"""
    q, w, h, *_ = statement(logits, tokens, k, temperature)
    V = q.shape[-1]
    coefficient = torch.zeros_like(q)
    here = (tokens >= 0) & (tokens < V)
    if gs[0] is not None:
        coefficient.scatter_add_(1, tokens.clamp(0, V - 1)[:, None], torch.where(here, gs[0].double(), 0.0)[:, None])
    if k and gs[2] is not None:
        coefficient.scatter_add_(1, ids, gs[2].double())
    gh = gs[1].double()[:, None] if gs[1] is not None else 0.0
    surprise = torch.where(w > 0, q, 0.0) + h[:, None]
    want = (coefficient - w * coefficient.sum(-1, keepdim=True) - gh * w * surprise) / temperature
    size = (w * coefficient.abs().sum(-1, keepdim=True) + abs(gh) * w * (torch.where(w > 0, q, 0.0).abs() + h[:, None] + 1)) / temperature
    return want, size, coefficient.abs() / temperature


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(1, 1), (2, 7), (3, 999), (5, 2048), (700, 520), (3, 32000), (2, 50257), (1, 128256)])
@pytest.mark.parametrize("k,temperature,masked,which", [(0, 1.0, 0.0, (1, 1, 0)), (20, 0.7, 0.3, (1, 1, 1)), (3, 1.5, 0.0, (0, 0, 1)), (5, 1.0, 0.0, (0, 1, 0)), (0, 2.0, 0.9, (1, 0, 0))])
def test_gradients(lp, cuda_device, dtype, rows, V, k, temperature, masked, which):
    logits, tokens = make(rows, V, dtype, cuda_device, masked)
    k = min(k, V)
    if k:
        tokens[0] = logits[0].float().argmax()                         # the token is an alternative too
    leaf = logits.clone().requires_grad_()
    got = lp.token_logprobs(leaf, tokens, k, temperature)
    check(lp.TokenLogprobs(*(t.detach() if t is not None else None for t in got)), logits, tokens, k, temperature)
    outs = [got.logprobs, got.entropy] + ([got.top_logprobs] if k else [])
    g = torch.Generator(device=cuda_device).manual_seed(V)
    gs = [torch.randn(o.shape, generator=g, device=cuda_device) for o in outs] + [None] * (3 - len(outs))
    used = [i for i in range(len(outs)) if which[i]]
    grad, = torch.autograd.grad([outs[i] for i in used], leaf, [gs[i] for i in used])
    gs = [x if which[i] else None for i, x in enumerate(gs)]
    if k and gs[2] is not None:                                        # alternatives that cannot come: none is asked for
        gs[2] = gs[2]
    want, size, single = gradient(logits, tokens, got.top_ids, k, temperature, gs)
    tol = slack(logits, temperature)[:, None]
    assert grad.dtype == dtype and grad.shape == logits.shape
    bound = HALF[dtype] * want.abs() + 2 * tol * size + 2.0 ** -22 * (single + size) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126)
    assert bool(((grad.double() - want).abs() <= bound).all())


@pytest.mark.gpu
def test_gradients_by_differences(lp, cuda_device):
    """the directional derivative against a central difference of the operator's own outputs"""
    logits, tokens = make(6, 300, torch.float32, cuda_device, spread=1.5)
    g = torch.Generator(device=cuda_device).manual_seed(5)
    direction = torch.randint(0, 2, logits.shape, generator=g, device=cuda_device).float() * 2 - 1
    gs = [torch.randn(6, generator=g, device=cuda_device) for _ in range(2)] + [torch.randn(6, 4, generator=g, device=cuda_device)]
    step = 2.0 ** -5

    # the alternatives are those of the middle: where two lie within 2 steps of one another the sorted values have a kink there, at which they change
    # places, and a difference across it mixes their weights
    ids = lp.token_logprobs(logits, tokens, 4, 1.0).top_ids

    def value(x):
        got = lp.token_logprobs(x, tokens, 0, 1.0)
        top = torch.stack([lp.token_logprobs(x, ids[:, k].contiguous(), 0, 1.0).logprobs for k in range(4)], 1)
        return [(o.double() * w.double()).flatten(1).sum(1) if o.dim() > 1 else o.double() * w.double() for o, w in zip((got.logprobs, got.entropy, top), gs)]
    leaf = logits.clone().requires_grad_()
    got = lp.token_logprobs(leaf, tokens, 4, 1.0)
    grad, = torch.autograd.grad([got.logprobs, got.entropy, got.top_logprobs], leaf, gs)
    plus, minus = value(logits + step * direction), value(logits - step * direction)
    slope = sum((p - m) / (2 * step) for p, m in zip(plus, minus))
    # third derivatives of log sum exp along +-1 are at most 2, of the entropy at most 6 (its log factor at most log 300 more); outputs are off by 2^-17
    weight = gs[0].abs() + gs[2].abs().sum(1) + 6 * gs[1].abs()
    bound = step ** 2 / 6 * 8 * weight.double() + 2.0 ** -17 / step * weight.double() * 2
    assert bool(((grad.double() * direction.double()).sum(1) - slope).abs().le(bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_of_masked_rows(lp, cuda_device, dtype):
    """rows of the type's lowest value, of one token alone, and rows without probabilities, whose NaN stays in its row"""
    logits, tokens = make(6, 4000, dtype, cuda_device)
    logits[0, 1:] = -math.inf
    logits[1] = torch.finfo(dtype).min
    logits[2, 7:] = torch.finfo(dtype).min
    logits[3] = -math.inf
    logits[4, 9] = math.nan
    tokens[:] = 0
    leaf = logits.clone().requires_grad_()
    got = lp.token_logprobs(leaf, tokens, 0, 1.0)
    gs = [torch.ones(6, device=cuda_device), torch.full((6,), 0.5, device=cuda_device), None]
    grad, = torch.autograd.grad([got.logprobs, got.entropy], leaf, gs[:2])
    fine = torch.tensor([0, 1, 2, 5], device=cuda_device)
    want, size, single = gradient(logits[fine], tokens[fine], None, 0, 1.0, [x[fine] for x in gs[:2]] + [None])
    bound = HALF[dtype] * want.abs() + (2 * slack(logits[fine], 1.0)[:, None] + 2.0 ** -22) * size + 2.0 ** -22 * single + 2.0 ** -25
    assert bool(((grad[fine].double() - want).abs() <= bound).all())
    assert bool(torch.isnan(grad[3]).all()) and bool(torch.isnan(grad[4]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(lp, cuda_device, dtype):
    """rows of a wider tensor, off 16 bytes, of every other position, of three dimensions, transposed, none"""
    wide, tokens = make(12, 5003, dtype, cuda_device)
    for view in (wide[:, 1:4000], wide[:, 3:], wide[::3, 2:2050]):
        t = tokens[:view.shape[0]] % view.shape[1]
        check(lp.token_logprobs(view, t, 5, 0.9), view, t, 5, 0.9)
        leaf = wide.clone().requires_grad_()
        at = {wide.shape[0]: slice(None), 4: slice(None, None, 3)}[view.shape[0]]
        part = leaf[at, view.storage_offset():view.storage_offset() + view.shape[1]]
        got = lp.token_logprobs(part, t, 0, 0.9)
        got.logprobs.sum().backward()
        want, size, single = gradient(view, t, None, 0, 0.9, [torch.ones_like(got.logprobs), None, None])
        grad = leaf.grad[at, view.storage_offset():view.storage_offset() + view.shape[1]].double()
        bound = HALF[dtype] * want.abs() + (2 * slack(view, 0.9)[:, None] + 2.0 ** -22) * size + 2.0 ** -22 * single + 2.0 ** -25
        assert bool(((grad - want).abs() <= bound).all())
    cube = wide[:, :999].reshape(3, 4, 999)
    got = lp.token_logprobs(cube, tokens.view(3, 4) % 999, 3, 1.0)
    assert got.logprobs.shape == (3, 4) and got.top_ids.shape == (3, 4, 3) and got.top_logprobs.shape == (3, 4, 3)
    check(got, cube, tokens.view(3, 4) % 999, 3, 1.0)
    turned = wide[:, :64].t()
    check(lp.token_logprobs(turned, torch.zeros(64, dtype=torch.int64, device=cuda_device), 2, 1.0), turned, torch.zeros(64, dtype=torch.int64, device=cuda_device), 2, 1.0)
    none = lp.token_logprobs(wide[:0], tokens[:0], 4)
    assert none.logprobs.shape == (0,) and none.top_ids.shape == (0, 4)
    one = lp.token_logprobs(wide[0], tokens[0], 2)
    assert one.logprobs.shape == () and one.top_ids.shape == (2,)
    leaf = wide[:0].clone().requires_grad_()
    lp.token_logprobs(leaf, tokens[:0]).logprobs.sum().backward()
    assert leaf.grad.shape == leaf.shape


@pytest.mark.gpu
def test_rows_beyond_32_bits(lp, cuda_device):
    rows, V = 70000, 32000
    logits = torch.empty(rows, V, dtype=torch.float16, device=cuda_device).uniform_(-4, 4)
    tokens = torch.randint(0, V, (rows,), device=cuda_device)
    got = lp.token_logprobs(logits, tokens, 3)
    at = torch.tensor([0, 1, 67107, 67109, rows - 1], device=cuda_device)
    check(lp.TokenLogprobs(*(t[at] for t in got)), logits[at], tokens[at], 3, 1.0)


@pytest.mark.gpu
def test_the_same_every_time_and_on_other_streams(lp, cuda_device):
    logits, tokens = make(40, 30000, torch.bfloat16, cuda_device)
    want = lp.token_logprobs(logits, tokens, 20)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams * 2:
        with torch.cuda.stream(s):
            got.append(lp.token_logprobs(logits, tokens, 20))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


@pytest.mark.gpu
def test_recorded_with_its_gradient(lp, cuda_device):
    logits, tokens = make(20, 3001, torch.bfloat16, cuda_device)
    leaf = logits.clone().requires_grad_()
    w = torch.randn(20, device=cuda_device)

    def step():
        got = lp.token_logprobs(leaf, tokens, 5)
        grad, = torch.autograd.grad([got.logprobs, got.entropy], leaf, [w, w])
        return got.logprobs, got.top_ids, grad
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2):
        fresh, other = make(20, 3001, torch.bfloat16, cuda_device, seed=seed)
        with torch.no_grad():
            leaf.copy_(fresh)
        tokens.copy_(other)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


@pytest.mark.gpu
def test_no_recording_beside_a_living_graph(lp, cuda_device):
    """the refusal of what the engine could not record, by the node alone: nothing of it is launched"""
    for shape in ((20, 301), (4, 5, 301)):
        leaf = torch.randn(shape, device=cuda_device).requires_grad_()
        tokens = torch.zeros(shape[:-1], dtype=torch.int64, device=cuda_device)
        alive = lp.token_logprobs(leaf, tokens)
        with pytest.raises(RuntimeError, match="outside the recording"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                lp.token_logprobs(leaf, tokens)
        alive.logprobs.sum().backward()
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            grad, = torch.autograd.grad(lp.token_logprobs(leaf, tokens).logprobs.sum(), leaf)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, leaf.grad)
        # what lives of another stream joins the recording
        want, leaf.grad = leaf.grad, None
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            kept = lp.token_logprobs(leaf, tokens)
            kept.logprobs.sum().backward()
        torch.cuda.synchronize()
        leaf.grad = None
        recorded = torch.cuda.CUDAGraph()
        with torch.cuda.graph(recorded):
            lp.token_logprobs(leaf, tokens).logprobs.sum().backward()
        recorded.replay()
        torch.cuda.synchronize()
        assert torch.equal(leaf.grad, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_the_python_statements_say_the_same(lp, cuda_device, monkeypatch, dtype):
    """what serves where the native host side is not to be had; three dimensions go through it"""
    logits, tokens = make(24, 3001, dtype, cuda_device, 0.2)
    w = torch.randn(24, 7, device=cuda_device)
    results = []
    for native, shape in ((True, (24,)), (True, (4, 6)), (False, (24,)), (False, (2, 3, 4))):
        monkeypatch.setattr(lp.paged_kv, "_native", lp.paged_kv._native if native else lambda *args: None)
        for k in (0, 5):
            leaf = logits.clone().view(*shape, 3001).requires_grad_()
            got = lp.token_logprobs(leaf, tokens.view(shape), k, 0.8)
            loss = (got.logprobs.flatten() * w[:, 0]).sum() + (got.entropy.flatten() * w[:, 1]).sum()
            if k:
                loss = loss + (got.top_logprobs.view(24, 5) * w[:, 2:]).sum()
            loss.backward()
            with torch.no_grad():
                again = lp.token_logprobs(leaf, tokens.view(shape), k, 0.8)
            results.append([t.detach().reshape(24, -1) for t in (*got, *again, leaf.grad) if t is not None])
    for i, r in enumerate(results):
        assert len(r) == len(results[i % 2]) and all(torch.equal(a, b) for a, b in zip(r, results[i % 2]))


@pytest.mark.gpu
def test_outputs_by_themselves_and_saved_elsewhere(lp, cuda_device):
    """a gradient of one output, none of the others; what was saved comes back from the host, or in another layout; a parameter; twice through one graph"""
    logits, tokens = make(9, 2000, torch.float32, cuda_device)
    def grad_of(what, hooks=None, parameter=False):                                               # noqa: E306
        leaf = torch.nn.Parameter(logits.clone()) if parameter else logits.clone().requires_grad_()
        with hooks or torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t):
            got = lp.token_logprobs(leaf, tokens, 4)
        sum(getattr(got, n).sum() for n in what).backward(retain_graph=True)
        first = leaf.grad.clone()
        leaf.grad = None
        sum(getattr(got, n).sum() for n in what).backward()
        assert torch.equal(first, leaf.grad)
        with pytest.raises(RuntimeError, match="second time"):
            sum(getattr(got, n).sum() for n in what).backward()
        return first
    turned = torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2 else t)
    for what in (["logprobs"], ["entropy"], ["top_logprobs"], ["entropy", "logprobs"]):
        want = grad_of(what)
        assert torch.equal(grad_of(what, torch.autograd.graph.save_on_cpu()), want)
        assert torch.equal(grad_of(what, turned), want) and torch.equal(grad_of(what, parameter=True), want)


@pytest.mark.gpu
def test_calls_at_once_from_threads(lp, cuda_device):
    import threading
    jobs = [make(5 + i, 9000 + i, torch.bfloat16, cuda_device) for i in range(6)]
    want = [lp.token_logprobs(x, t, 7) for x, t in jobs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                leaf = jobs[i][0].clone().requires_grad_()
                got = lp.token_logprobs(leaf, jobs[i][1], 7)
                got.logprobs.sum().backward()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])) or not bool(torch.isfinite(leaf.grad).all()):
                    wrong.append(i)
    torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.gpu
def test_refusals(lp, cuda_device):
    x, t = torch.zeros(4, 50, device=cuda_device), torch.zeros(4, dtype=torch.int64, device=cuda_device)
    for call in (lambda: lp.token_logprobs(x.double(), t), lambda: lp.token_logprobs(x, t.int()), lambda: lp.token_logprobs(x, t[:3]), lambda: lp.token_logprobs(x, t.cpu()),
                 lambda: lp.token_logprobs(x, t, 33), lambda: lp.token_logprobs(x[:, :5], t, 6), lambda: lp.token_logprobs(x, t, -1), lambda: lp.token_logprobs(x, t, 0, 0.0),
                 lambda: lp.token_logprobs(x, t, 0, -1.0), lambda: lp.token_logprobs(x, t, 0, math.inf), lambda: lp.token_logprobs(x, t, 0, 1e-9), lambda: lp.token_logprobs(x, t, 0, 1e9), lambda: lp.token_logprobs(x, t, 0, math.nan), lambda: lp.token_logprobs(x[:, :0], t)):
        with pytest.raises(RuntimeError):
            call()
    leaf = x.clone().requires_grad_()
    grad, = torch.autograd.grad(lp.token_logprobs(leaf, t).logprobs.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError):
            lp.token_logprobs(torch.autograd.forward_ad.make_dual(x, x), t)
    got = lp.token_logprobs(leaf, t, 2)
    assert not got.top_ids.requires_grad and got.top_logprobs.requires_grad
    with torch.no_grad():
        leaf.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        got.logprobs.sum().backward()


def test_refusals_on_the_cpu(lp, native_lib):
    with pytest.raises(RuntimeError, match="CUDA device"):
        lp.token_logprobs(torch.zeros(2, 9), torch.zeros(2, dtype=torch.int64))
    lib = native_lib._lib
    some = 4096                                                        # never read: every call is refused before anything is launched
    good = [some, 1, 100, 2, 100, some, 1.0, 4, some, some, some, some, some, None]
    for i, bad in ((0, None), (1, 3), (1, -1), (2, 99), (3, -1), (4, 0), (4, 1 << 31), (5, None), (6, 0.0), (6, math.nan), (7, 33), (7, -1), (8, None), (9, None), (10, None),
                   (11, None), (12, 4100), (0, 4097)):
        args = list(good)
        args[i] = bad
        assert lib.lowbit_token_logprobs_cuda(*args) == 1, (i, bad)
    good = [some, 1, 100, 2, 100, some, 1.0, 4, some, None, None, None, some, some, 100, None]
    for i, bad in ((0, None), (1, 3), (2, 99), (5, None), (6, -1.0), (7, 101), (8, None), (12, None), (12, 4100), (13, None), (13, 4097), (14, 99)):
        args = list(good)
        args[i] = bad
        assert lib.lowbit_token_logprobs_grad_cuda(*args) == 1, (i, bad)


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("shape", [(12,), (3, 4)])
def test_what_was_saved_in_another_layout(lp, cuda_device, monkeypatch, native, shape):
    """the gradient's node in Python, which serves three dimensions too, looks at what a hook brings back as the native one does"""
    if not native:
        monkeypatch.setattr(lp.paged_kv, "_native", lambda *args: None)
    logits, tokens = make(12, 700, torch.float32, cuda_device)
    logits, tokens = logits.view(*shape, 700), tokens.view(shape)
    g = torch.Generator(device=cuda_device).manual_seed(2)
    gs = [torch.randn(*shape, *more, generator=g, device=cuda_device) for more in ((), (), (4,))]

    def grad_of(unpack):
        leaf = logits.clone().requires_grad_()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            got = lp.token_logprobs(leaf, tokens, 4, 0.8)
            return torch.autograd.grad([got.logprobs, got.entropy, got.top_logprobs], leaf, gs)[0]
    want = grad_of(lambda t: t)
    turned = lambda t: t.t().contiguous().t() if t.dim() == 2 else t                              # noqa: E731
    apart = lambda t: torch.stack([t, t], -1).flatten(-2)[..., ::2]                               # noqa: E731  every other element of a wider one
    alone = lambda width: lambda t: turned(t) if t.dim() == 2 and t.shape[1] == width else t      # noqa: E731
    for unpack in (turned, apart, alone(4), alone(700)):
        assert torch.equal(grad_of(unpack), want)
    for unpack in (lambda t: t.int() if t.dtype == torch.int64 else t, lambda t: t.half() if t.shape[-1] == 4 and t.dtype == torch.float32 else t, lambda t: t.cpu()):
        with pytest.raises(RuntimeError, match="came back as something else"):
            grad_of(unpack)


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_no_recording_of_a_leaf_s_view_nor_without_the_native_side(lp, cuda_device, monkeypatch, native):
    """the refusals alone: no backward pass is recorded here beside a graph that lives.  Without the native host side nobody can look at a leaf's node, so that
    a recording takes no leaf that wants a gradient"""
    leaf = torch.randn(4, 6, 301, device=cuda_device).requires_grad_()
    tokens = torch.zeros(4, 6, dtype=torch.int64, device=cuda_device)
    forms = [(leaf, tokens), (leaf[:, :-1], tokens[:, 1:]), (leaf[0], tokens[0]), (leaf[1, :, :9], tokens[1])]
    wants = [lp.token_logprobs(x.detach(), t) for x, t in forms]
    if not native:
        monkeypatch.setattr(lp.paged_kv.linears, "_host", False)
    alive = lp.token_logprobs(leaf, tokens)
    for x, t in forms:
        with pytest.raises(RuntimeError, match="recording"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                lp.token_logprobs(x, t)
    alive.logprobs.sum().backward()
    del alive, x, forms
    for take, want in zip((lambda x: (x, tokens), lambda x: (x[:, :-1], tokens[:, 1:]), lambda x: (x[0], tokens[0]), lambda x: (x[1, :, :9], tokens[1])), wants):
        if native:                                                     # nothing lives any more
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got = lp.token_logprobs(*take(leaf))
                grad, = torch.autograd.grad(got.logprobs.sum(), leaf)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got.logprobs, want.logprobs) and bool(torch.isfinite(grad).all())
            del got, grad
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph), torch.no_grad():                 # no gradient is asked for
            got = lp.token_logprobs(*take(leaf))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got.logprobs, want.logprobs) and torch.equal(got.entropy, want.entropy)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = lp.token_logprobs(*take(leaf.detach()))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got.logprobs, want.logprobs)


# ------------------------------------------------------------------ bounds that masked entries do not widen
def tight(logits, tokens, k, temperature):
    """what the results may be off by: (log probability of the token, entropy, of the alternatives; of every entry's probability, relative; of the entropy and an entry's log
    probability together).

    An exponent is taken relative to a reference within 2^4 above its row's largest: one multiply-add or a difference and a product, and a factor with
    three roundings, so it is off by 2^-21 of its own distance from the largest (and of those 4); entries of probability 0 add nothing to any sum.  A power adds 2^-22; sums add
    2^-24 for each of the V / 512 additions of a thread and some 40 where threads and blocks meet; a base-2 logarithm below 32 adds 2^-23 of that.  The entropy
    is the logarithm of the sum less the mean exponent, whose absolute mean is below that of the distances and 4."""
    q, w, h, token, ids, top = statement(logits, tokens, k, temperature)
    z = logits.detach().double() / temperature
    dist = z.amax(-1, keepdim=True) - z
    U = torch.where(w > 0, dist, 0.0) + 4
    R = 2.0 ** -22 + 2.0 ** -24 * (z.shape[-1] / 512 + 40)
    off = 2.0 ** -21 * U
    mean = (w * U).sum(-1)
    of_sum = (w * off).sum(-1) + R + 2.0 ** -18
    of_h = (w * (U * R + off * (1 + U))).sum(-1) + of_sum + 2.0 ** -23 * (mean + 32)
    here = (tokens >= 0) & (tokens < z.shape[-1])
    at = tokens.clamp(0, z.shape[-1] - 1)[:, None]
    own = lambda i: 2.0 ** -21 * (dist.gather(1, i) + 4) + of_sum[:, None] + 2.0 ** -23 * q.gather(1, i).abs()       # noqa: E731  the entry's own distance, masked or not
    return torch.where(here, own(at)[:, 0], 0.0), of_h, own(ids), off + of_sum[:, None], 2 * (off + of_sum[:, None] + of_h[:, None])


def held(got, logits, tokens, k, temperature):
    """whether results lie within the tight bounds; numbers that 32 bits cannot hold are their infinity"""
    _, _, h, token, ids, top = statement(logits, tokens, k, temperature)
    a, b, c, *_ = tight(logits, tokens, k, temperature)
    near = lambda x, y, t: bool(((x.double() == y.float().double()) | ((x.double() - y).abs() <= t)).all())          # noqa: E731
    return near(got.logprobs, token, a) and near(got.entropy, h, b) and (not k or torch.equal(got.top_ids, ids) and near(got.top_logprobs, top, c))


MASKS = ["front", "behind", "between", "everything", "all but one", "all but the first", "half as low", "in every thread", "a few left"]


def masked_rows(V, dtype, dev, low):
    logits, tokens = make(len(MASKS), V, dtype, dev, seed=3)
    i = torch.arange(V, device=dev)
    for row, out in enumerate((i < V // 2, i >= V // 2, i % 3 > 0, i >= 0, i != V // 3, i > 0, i >= 0, i // 8 % 2 == 0, i * 7919 % V >= 9)):
        logits[row, out] = low
    logits[6, V // 3] = low / 2
    tokens[:] = V // 3
    return logits, tokens


def lows(dtype):
    return [-1e4, torch.finfo(dtype).min] + ([-1e9, -1e12, -1e25, -1e29, -3e30, -1e37] if dtype != torch.float16 else []) + [-math.inf]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [300, 40001, 128256])
def test_masks_do_not_blur_what_is_left(lp, cuda_device, dtype, V):
    """as test_masks_of_large_numbers, with the bounds of what the masks leave"""
    for low in lows(dtype):
        logits, tokens = masked_rows(V, dtype, cuda_device, low)
        if low == -math.inf:
            logits[3], logits[6] = 0.0, 1.0                            # rows of nothing else have no probabilities
        for k, temperature in ((9, 1.0), (0, 0.7), (20, 3.0), (1, 1e-3), (5, 1e4)):
            got = lp.token_logprobs(logits, tokens, k, temperature)
            assert held(got, logits, tokens, k, temperature), (low, k, temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V,k,temperature,masked", [(3, 999, 5, 1.0, 0.0), (33, 4099, 20, 0.7, 0.9), (2, 128256, 20, 1.5, 0.3), (800, 2056, 0, 0.3, 0.0), (5, 3001, 6, 1e-7, 0.3), (5, 3001, 6, 1e7, 0.3)])
def test_values_within_the_bounds_of_what_counts(lp, cuda_device, dtype, rows, V, k, temperature, masked):
    logits, tokens = make(rows, V, dtype, cuda_device, masked)
    assert held(lp.token_logprobs(logits, tokens, k, temperature), logits, tokens, k, temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [300, 40001])
def test_gradients_of_what_masks_leave(lp, cuda_device, dtype, V):
    for low in lows(dtype):
        logits, tokens = masked_rows(V, dtype, cuda_device, low)
        if low == -math.inf:
            logits[3], logits[6] = 0.0, 1.0
        g = torch.Generator(device=cuda_device).manual_seed(V)
        gs = [torch.randn(len(MASKS), *more, generator=g, device=cuda_device) for more in ((), (), (5,))]
        for temperature in (1.0, 0.7):
            leaf = logits.clone().requires_grad_()
            got = lp.token_logprobs(leaf, tokens, 5, temperature)
            grad, = torch.autograd.grad(list(got[:2]) + [got.top_logprobs], leaf, gs)
            q, w, h, *_ = statement(logits, tokens, 5, temperature)
            want, size, single = gradient(logits, tokens, got.top_ids, 5, temperature, gs)
            *_, of_p, of_both = tight(logits, tokens, 5, temperature)
            weight = gs[1].double().abs()[:, None] * w / temperature
            bound = HALF[dtype] * want.abs() + 2 * of_p * size + weight * (of_both + 2.0 ** -22 * 8) + 2.0 ** -22 * (single + size) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126)
            assert bool(((grad.double() - want).abs() <= bound).all()), (low, temperature)


def test_the_bounds_refuse_planted_mistakes(lp):
    """on the CPU: results of 64 bits are taken, and those with a mistake in what the masks leave are not"""
    for dtype in TYPES:
        for low in lows(dtype):
            logits, tokens = masked_rows(300, dtype, torch.device("cpu"), low)
            if low == -math.inf:
                logits[3], logits[6] = 0.0, 1.0
            _, w, h, token, ids, top = statement(logits, tokens, 5, 1.0)
            right = lp.TokenLogprobs(token.float(), h.float(), ids, top.float())
            assert held(right, logits, tokens, 5, 1.0)
            for row in (0, 1, 2, 7, 8):                                # sums that are lost, counted twice, or off in the fourth digit
                for name, value in (("logprobs", 0.0), ("logprobs", token[row] - math.log(2)), ("logprobs", token[row] + 1e-3), ("entropy", 0.0), ("entropy", h[row] + 1e-3),
                                    ("top_logprobs", top[row] - 1e-3), ("top_ids", ids[row].flip(0))):
                    if name == "logprobs" and token[row] < -1e3:       # this token is ruled out: its own distance
                        continue
                    wrong = right._replace(**{name: getattr(right, name).clone()})
                    getattr(wrong, name)[row] = value
                    assert not held(wrong, logits, tokens, 5, 1.0), (dtype, low, row, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [0.7, 1.0, 2.0, 1e3, 1e7])
def test_logits_of_the_type_s_whole_range(lp, cuda_device, dtype, temperature):
    """the difference from the row's largest may pass 32 bits where its quotient by the temperature does not, and the other way round"""
    big = torch.finfo(dtype).max
    logits = torch.zeros(6, 3000, dtype=dtype, device=cuda_device)
    for row, (a, b) in enumerate(((big / 2, -big), (big, -big), (big, big / 4), (0.0, -big), (-big / 4, -big), (1e30, -big))):
        logits[row, ::2], logits[row, 1::2] = a, b
        logits[row, 5] = 0.0 if row < 3 else -big / 2
    for token in (0, 1, 5):
        tokens = torch.full((6,), token, device=cuda_device)
        for k in (0, 32):
            assert held(lp.token_logprobs(logits, tokens, k, temperature), logits, tokens, k, temperature)
    tokens[::2] = 1
    leaf = logits.clone().requires_grad_()
    got = lp.token_logprobs(leaf, tokens, 4, temperature)
    gs = [torch.ones(6, device=cuda_device), torch.full((6,), 0.5, device=cuda_device), torch.ones(6, 4, device=cuda_device)]
    grad, = torch.autograd.grad([got.logprobs, got.entropy, got.top_logprobs], leaf, gs)
    want, size, single = gradient(logits, tokens, got.top_ids, 4, temperature, gs)
    *_, of_p, of_both = tight(logits, tokens, 4, temperature)
    w = statement(logits, tokens, 4, temperature)[1]
    bound = HALF[dtype] * want.abs() + 2 * of_p * size + 0.5 * w / temperature * (of_both + 2.0 ** -19) + 2.0 ** -22 * (single + size) + 2.0 ** -126
    assert bool(((grad.double() - want).abs() <= bound).all())
