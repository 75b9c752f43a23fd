"""Adapters of many requests (transformers/lora.py) against 64-bit statements.

Bounds.  x A^T: the K products of an element drop up to 2^-23 of their absolute sum in each of K / 16 steps of two MMAs, and some 20 times where warps and
parts meet.  Its two 16-bit values leave 2^-16 of it (bf16) or 2^-21 (fp16, with 2^-38 of its row's largest).  The product with B drops up to 2^-23 of
its absolute sum in each of its rank / 4 steps.  `out` is rounded once, finfo(t).eps / 2, behind an addition in 32 bits."""
import math

import pytest
import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEFT = {torch.float16: 2.0 ** -21, torch.bfloat16: 2.0 ** -16}


@pytest.fixture(scope="module")
def lora(native_lib):
    from ipex_llm_b200.transformers import lora
    return lora


def rows_of(lens, ids, T):
    """the adapter of every row"""
    flat = [i for n, i in zip(lens, ids) for _ in range(n)]
    return torch.tensor(flat + [-1] * (T - len(flat)))


def make(lens, ids, K, splits, rank, adapters, dtype, dev, pad=0, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + sum(lens) + K + rank)
    T, N = sum(lens) + pad, sum(splits)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)                                       # noqa: E731
    return {"out": r(T, N).to(dtype), "x": r(T, K).to(dtype), "a": (r(adapters, len(splits), rank, K) * K ** -0.5).to(dtype), "b": (r(adapters, N, rank) * 0.3).to(dtype),
            "scales": 0.25 + 2 * torch.rand(adapters, generator=g, device=dev), "ids": torch.tensor(ids, dtype=torch.int32, device=dev),
            "cu": torch.tensor([0] + lens, dtype=torch.int32, device=dev).cumsum(0, dtype=torch.int32), "splits": splits}


def statement(s, lens, ids):
    """the result, and what it may be off by"""
    dtype, dev = s["x"].dtype, s["x"].device
    T, K = s["x"].shape
    rank = s["b"].shape[2]
    rows = rows_of(lens, ids, T).to(dev)
    want, bound = s["out"].double(), torch.zeros(s["out"].shape, dtype=torch.float64, device=dev)
    for i in range(s["b"].shape[0]):
        at = (rows == i).nonzero()[:, 0]
        first = 0
        for j, n in enumerate(s["splits"]):
            x, a, b, c = s["x"][at].double(), s["a"][i, j].double(), s["b"][i, first:first + n].double(), float(s["scales"][i])
            h, size = x @ a.T, x.abs() @ a.abs().T
            want[at, first:first + n] += c * (h @ b.T)
            off = 2.0 ** -23 * (K / 16 + 20) * size + LEFT[dtype] * h.abs() + (2.0 ** -38 * h.abs().amax(-1, keepdim=True) if h.numel() else 0)
            bound[at, first:first + n] += c * (off @ b.abs().T + 2.0 ** -23 * (rank / 4 + 4) * (h.abs() @ b.abs().T))
            first += n
    return want, HALF[dtype] * want.abs() + bound + 2.0 ** -23 * s["out"].double().abs() * (bound > 0) + (2.0 ** -25 if dtype == torch.float16 else 0)


def run(lora, s, **more):
    args = {"splits": s["splits"]} | more
    out = s["out"].clone()
    got = lora.lora_add_(out, s["x"], s["a"], s["b"], s["scales"], s["ids"], s["cu"], **args)
    assert got is out
    return out


def check(lora, s, lens, ids):
    want, bound = statement(s, lens, ids)
    got = run(lora, s)
    assert bool(((got.double() - want).abs() <= bound).all())
    nobody = rows_of(lens, [i if 0 <= i < s["b"].shape[0] else -1 for i in ids], s["x"].shape[0]).to(got.device) < 0
    assert torch.equal(got[nobody], s["out"][nobody])
    return got


CASES = [([1], [0], 1), ([1], [-1], 1), ([1, 1, 1, 1, 1], [2, 0, 2, -1, 1], 3), ([0, 3, 0, 17], [1, 0, 5, 1], 2), ([16, 1, 15, 33], [0, 1, 2, 0], 4), ([64, 1, 63, 200], [3, -1, 0, 3], 4),
         ([300], [0], 1), ([1] * 40 + [250] + [1] * 30, [i % 7 for i in range(71)], 7), ([1] * 300, [i * 5 % 67 for i in range(300)], 67), ([2, 1, 3] * 230, [i % 3 - 1 for i in range(690)], 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,ids,adapters", CASES)
@pytest.mark.parametrize("K,splits,rank", [(8, [8], 8), (256, [256], 16), (1000, [136, 40, 40], 24), (4096, [520], 64), (96, [128, 128], 128)])
def test_rows_take_their_adapters(lora, cuda_device, dtype, lens, ids, adapters, K, splits, rank):
    check(lora, make(lens, ids, K, splits, rank, adapters, dtype, cuda_device, pad=5), lens, ids)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("K,splits,rank", [(14336, [4096], 16), (4096, [4096, 1024, 1024], 32), (4096, [11008, 11008], 8), (2048, [2040], 256), (512, [64] * 8, 256), (8, [8, 8], 256)])
@pytest.mark.parametrize("lens", [[1, 1, 1], [100, 1, 300]])
def test_layer_sizes(lora, cuda_device, dtype, K, splits, rank, lens):
    ids = [1, -1, 0]
    check(lora, make(lens, ids, K, splits, rank, 2, dtype, cuda_device), lens, ids)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens", [[3, 1], [200, 130]])
def test_only_the_result_is_rounded(lora, cuda_device, dtype, lens):
    """`out` takes the product away again: what is left is far below what one 16-bit value of x A^T leaves"""
    s = make(lens, [0, 1], 512, [256], 32, 2, dtype, cuda_device)
    s["out"].zero_()
    s["out"] = (-statement(s, lens, [0, 1])[0]).to(dtype)
    want, bound = statement(s, lens, [0, 1])
    check(lora, s, lens, [0, 1])
    # with one value
    first = s["x"].double() @ s["a"][0, 0].double().T
    once = s["out"][:lens[0]].double() + float(s["scales"][0]) * (first[:lens[0]].to(dtype).double() @ s["b"][0].double().T)
    assert bool(((once - want[:lens[0]]).abs() > bound[:lens[0]]).any())


@pytest.mark.gpu
def test_products_beyond_fp16(lora, cuda_device):
    """x A^T of 10^6 and of 10^-6, which fp16 cannot hold, and a B that brings them back"""
    for up in (2.0 ** 7, 2.0 ** -9):
        s = make([5, 90], [0, 1], 256, [64], 16, 2, torch.float16, cuda_device)
        s["x"] *= up
        s["a"] *= up * 64 if up > 1 else up
        s["b"] *= 2.0 ** -12 if up > 1 else 2.0 ** 8
        want, bound = statement(s, [5, 90], [0, 1])
        assert bool(torch.isfinite(want).all())
        check(lora, s, [5, 90], [0, 1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens", [[1, 1, 1, 1], [40, 300, 7, 90]])
def test_what_is_not_finite_stays_in_its_row(lora, cuda_device, dtype, lens):
    ids = [0, 1, 0, -1]
    s = make(lens, ids, 256, [64, 64], 16, 3, dtype, cuda_device, pad=3)
    clean = run(lora, s)
    s["x"][lens[0]:sum(lens[:2])] = math.nan                           # a request's activations
    s["x"][sum(lens):] = math.inf                                      # padding
    s["a"][2], s["b"][2] = math.nan, math.inf                          # an adapter that nobody has
    got = run(lora, s)
    rows = torch.ones(len(got), dtype=torch.bool, device=cuda_device)
    rows[lens[0]:sum(lens[:2])] = False
    assert torch.equal(got[rows], clean[rows]) and bool(torch.isnan(got[~rows]).all())


@pytest.mark.gpu
def test_layouts(lora, cuda_device):
    lens, ids = [30, 1, 60], [1, 0, 1]
    s = make(lens, ids, 128, [96], 16, 2, torch.bfloat16, cuda_device)
    want = run(lora, s)
    T = sum(lens)
    wide_x, wide_out = torch.zeros(T, 160, dtype=torch.bfloat16, device=cuda_device), torch.full((T, 128), 7.0, dtype=torch.bfloat16, device=cuda_device)
    wide_x[:, 16:144], wide_out[:, 24:120] = s["x"], s["out"]
    wide_a, wide_b = torch.zeros(4, 1, 16, 128, dtype=torch.bfloat16, device=cuda_device), torch.zeros(2, 16, 96, dtype=torch.bfloat16, device=cuda_device)
    wide_a[::2] = s["a"]
    wide_b.copy_(s["b"].transpose(1, 2))
    lora.lora_add_(wide_out[:, 24:120], wide_x[:, 16:144], wide_a[::2], wide_b.transpose(1, 2), s["scales"], s["ids"], s["cu"])
    assert torch.equal(wide_out[:, 24:120], want) and bool((wide_out[:, :24] == 7).all()) and bool((wide_out[:, 120:] == 7).all())
    odd = torch.zeros(T, 131, dtype=torch.bfloat16, device=cuda_device)
    odd[:, 3:] = s["x"]                                                # rows off 16 bytes
    out = s["out"].clone()
    lora.lora_add_(out, odd[:, 3:], s["a"][:, 0], s["b"], s["scales"], s["ids"], s["cu"])        # one projection: a without the splits
    assert torch.equal(out, want)
    none = lora.lora_add_(out[:0], s["x"][:0], s["a"], s["b"], s["scales"], s["ids"], s["cu"])
    assert none.shape == (0, 96)


@pytest.mark.gpu
def test_lists_that_do_not_fit_the_rows(lora, cuda_device):
    """more tokens than rows, requests in a padded batch, an adapter that is not there"""
    s = make([20, 30, 4], [0, 9, 1], 64, [64], 8, 2, torch.float16, cuda_device)
    want = run(lora, s)
    assert torch.equal(want[20:50], s["out"][20:50])
    cut = {**s, "x": s["x"][:52], "out": s["out"][:52]}
    assert torch.equal(run(lora, cut), want[:52])


@pytest.mark.gpu
def test_offsets_beyond_32_bits(lora, cuda_device):
    """a tensor of more than 2^32 bytes, in which the last rows have an adapter"""
    T, K, N = 150000, 16384, 16
    x = torch.empty(T, K, dtype=torch.float16, device=cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(1)
    x[-40:] = torch.randn(40, K, generator=g, device=cuda_device).half()
    s = make([40], [0], K, [N], 8, 1, torch.float16, cuda_device)
    s["x"] = x[-40:].clone()
    want = run(lora, s)
    out = torch.zeros(T, N, dtype=torch.float16, device=cuda_device)
    out[-40:] = s["out"]
    ids, cu = torch.tensor([-1, 0], dtype=torch.int32, device=cuda_device), torch.tensor([0, T - 40, T], dtype=torch.int32, device=cuda_device)
    lora.lora_add_(out, x, s["a"], s["b"], s["scales"], ids, cu)
    # other tiles than above: other sums of the same products
    assert bool(((out[-40:] - want).double().abs() <= 2 * statement(s, [40], [0])[1]).all()) and not bool(out[:-40].any())


@pytest.mark.gpu
def test_the_same_every_time_and_on_other_streams(lora, cuda_device):
    lens = [1] * 30 + [200, 100]
    s = make(lens, [i % 5 for i in range(32)], 1024, [512], 32, 5, torch.bfloat16, cuda_device)
    want = run(lora, s)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for st in streams * 2:
        with torch.cuda.stream(st):
            got.append(run(lora, s))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.gpu
def test_a_recorded_call_serves_other_requests(lora, cuda_device):
    lens = [1] * 8 + [50]
    s = make(lens, [0] * 9, 256, [128, 64], 16, 3, torch.float16, cuda_device)
    base, out = s["out"].clone(), s["out"].clone()
    lora.lora_add_(out, s["x"], s["a"], s["b"], s["scales"], s["ids"], s["cu"], splits=s["splits"])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lora.lora_add_(out, s["x"], s["a"], s["b"], s["scales"], s["ids"], s["cu"], splits=s["splits"])
    for lens, ids in (([3, 0, 20, 1, 1, 1, 1, 1, 10], [2, 0, -1, 1, 1, 0, 0, 2, 2]), ([58] + [0] * 8, [1] * 9)):
        s["cu"].copy_(torch.tensor([0] + lens, dtype=torch.int32, device=cuda_device).cumsum(0))
        s["ids"].copy_(torch.tensor(ids, dtype=torch.int32))
        out.copy_(base)
        graph.replay()
        assert torch.equal(out, run(lora, s))
        check(lora, s, lens, ids)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [255, 256, 257, 321])
@pytest.mark.parametrize("rank", [8, 48, 64, 136])
def test_where_the_launches_change(lora, cuda_device, rows, rank):
    lens, ids = [rows - 70, 1, 69], [2, 0, 1]
    check(lora, make(lens, ids, 520, [264, 8], rank, 3, torch.float16, cuda_device), lens, ids)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,ids,adapters", [
    ([1] * 2000, [0] * 2000, 1), ([1] * 600, [i % 600 for i in range(600)], 600), ([3, 0, 5, 1] * 300, [i * 7 % 9 - 1 for i in range(1200)], 8), ([1500, 1, 1023, 1024, 1025, 6], [1, 0, 1, 2, 1, -1], 3),
    ([2] * 700 + [1100], [i * 31 % 5003 for i in range(701)], 5000), ([64] * 6, [4999, 0, 4096, 4095, 4999, 5000], 5000)])
def test_orders_of_many_rows(lora, cuda_device, lens, ids, adapters):
    """more requests and more adapters than a block looks at at a time, stretches of every kind, an adapter for each, one for all"""
    check(lora, make(lens, ids, 16, [8, 16], 8, adapters, torch.float16, cuda_device, pad=9), lens, ids)


@pytest.mark.gpu
def test_a_list_that_goes_back(lora, cuda_device):
    """of many rows none is taken twice: a request has what lies behind all in front of it"""
    s = make([400, 200], [0, 1], 64, [64], 8, 3, torch.bfloat16, cuda_device)
    want = run(lora, s)
    for cu, ids in (([0, 400, 100, 400, 350, 600], [0, 2, 2, 2, 1]), ([-50, 400, 600, 0, 600], [0, 1, 2, 2])):
        odd = {**s, "cu": torch.tensor(cu, dtype=torch.int32, device=cuda_device), "ids": torch.tensor(ids, dtype=torch.int32, device=cuda_device)}
        assert torch.equal(run(lora, odd), want)


@pytest.mark.gpu
def test_rows_far_apart(lora, cuda_device):
    """rows of 2^27 elements: as many at a time as a 32-bit offset in 16 bytes reaches"""
    T, step = 270, 1 << 27
    if torch.cuda.mem_get_info()[0] < T * step * 2 + (4 << 30):
        pytest.skip("needs 73 GB")
    lens, ids = [200, 30, 40], [0, -1, 1]
    s = make(lens, ids, 64, [64], 16, 2, torch.float16, cuda_device)
    want = run(lora, s)
    far = torch.empty(T * step, dtype=torch.float16, device=cuda_device).as_strided((T, 64), (step, 1))
    far.copy_(s["out"])
    lora.lora_add_(far, s["x"], s["a"], s["b"], s["scales"], s["ids"], s["cu"])
    assert torch.equal(far, want)
    far.copy_(s["x"])
    assert torch.equal(run(lora, {**s, "x": far}), want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 5, 300])
def test_the_python_statements_say_the_same(lora, cuda_device, monkeypatch, rows):
    s = make([rows], [1], 256, [128, 64], 16, 2, torch.bfloat16, cuda_device)
    native = run(lora, s)
    monkeypatch.setattr(lora.paged_kv, "_native", lambda *args: None)
    assert torch.equal(run(lora, s), native)
    whole = {**s, "splits": [192], "a": s["a"][:, :1].contiguous()}
    assert torch.equal(run(lora, {**whole, "a": whole["a"][:, 0], "splits": None}), check(lora, whole, [rows], [1]))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 7, 300])
@pytest.mark.parametrize("native", [True, False])
def test_rows_that_share_memory(lora, cuda_device, monkeypatch, rows, native):
    """the output is the input, lies some way into it, or beside it in one buffer"""
    if not native:
        monkeypatch.setattr(lora.paged_kv, "_native", lambda *args: None)
    s = make([rows], [0], 256, [256], 16, 1, torch.float16, cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(rows)
    buffer = torch.randn(rows + 3, 768, generator=g, device=cuda_device).half()
    for x_at, out_at in (((0, 0), (0, 0)), ((0, 0), (0, 128)), ((0, 128), (0, 0)), ((0, 0), (1, 0)), ((0, 0), (0, 256)), ((0, 512), (0, 0)), ((0, 0), (2, 640))):
        flat = buffer.clone().view(-1)
        x, out = (flat.as_strided((rows, 256), (768, 1), 768 * r + c) for r, c in (x_at, out_at))
        case = {**s, "x": x.clone(), "out": out.clone()}
        want = run(lora, case)
        lora.lora_add_(out, x, s["a"], s["b"], s["scales"], s["ids"], s["cu"])
        assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_autograd_hears_of_it(lora, cuda_device, monkeypatch, native):
    if not native:
        monkeypatch.setattr(lora.paged_kv, "_native", lambda *args: None)
    s = make([3], [0], 64, [64], 8, 1, torch.float16, cuda_device)
    w = torch.ones(64, device=cuda_device, dtype=torch.float16, requires_grad=True)
    out = s["out"].clone()
    y = out * w
    lora.lora_add_(out, s["x"], s["a"], s["b"], s["scales"], s["ids"], s["cu"], splits=[64])
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    with torch.inference_mode():
        fresh = s["out"].clone()
    lora.lora_add_(fresh, s["x"], s["a"], s["b"], s["scales"], s["ids"], s["cu"], splits=[64])
    assert torch.equal(fresh, out)


@pytest.mark.gpu
def test_calls_at_once_from_threads(lora, cuda_device):
    import threading
    jobs = [make([50 * i + 1, 20], [0, 1], 512, [256], 16, 2, torch.bfloat16, cuda_device) for i in range(6)]
    want = [run(lora, s) for s in jobs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            wrong.extend(i for _ in range(20) if not torch.equal(run(lora, jobs[i]), want[i]))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.gpu
def test_refusals(lora, cuda_device):
    s = make([3, 2], [0, 1], 64, [32, 32], 16, 2, torch.float16, cuda_device)
    names = ("out", "x", "a", "b", "scales", "ids", "cu")

    def call(splits=(32, 32), **changed):
        lora.lora_add_(*({**s, **changed}[n] for n in names), splits=splits)
    call()
    bad = [{"x": s["x"].float()}, {"out": s["out"].bfloat16()}, {"a": s["a"].bfloat16()}, {"x": s["x"][:4]}, {"x": s["x"][:, :56]}, {"b": s["b"][:, :56]}, {"b": s["b"][:, :, :8]}, {"a": s["a"][:1]},
           {"scales": s["scales"].half()}, {"scales": s["scales"][:1]}, {"ids": s["ids"].long()}, {"ids": s["ids"][:1]}, {"cu": s["cu"].long()}, {"cu": s["cu"][:2]},
           {"splits": (32, 24)}, {"splits": (36, 28)}, {"splits": (64,)}, {"splits": None}, {"splits": (64, 0)}, {"ids": s["ids"].cpu()}, {"scales": s["scales"].cpu()}, {"a": s["a"][0]},
           {"a": s["a"][:, :, :12], "b": s["b"][:, :, :12]}, {"x": s["x"][:, :60], "a": s["a"][..., :60]}, {"out": torch.zeros(5, 67, dtype=torch.float16, device=cuda_device)[:, 3:]},
           {"out": s["out"].t().contiguous().t()}, {"out": s["out"][0].expand(5, 64)}]
    for i, more in enumerate(bad):
        with pytest.raises(RuntimeError):
            call(**more)
            pytest.fail(f"call {i} was taken")
    for n in ("out", "x", "a", "b", "scales"):
        with pytest.raises(RuntimeError, match="backward"):
            call(**{n: s[n].clone().requires_grad_()})
        with torch.autograd.forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="tangent"):
                call(**{n: torch.autograd.forward_ad.make_dual(s[n], torch.ones_like(s[n]))})
        with torch.no_grad():
            call(**{n: s[n].clone().requires_grad_()})


def test_refusals_on_the_cpu(lora, native_lib):
    s = make([3, 2], [0, 1], 64, [32], 16, 2, torch.float16, torch.device("cpu"))
    with pytest.raises(RuntimeError, match="CUDA device"):
        lora.lora_add_(s["out"], s["x"], s["a"], s["b"], s["scales"], s["ids"], s["cu"])
    import ctypes
    lib, some = native_lib._lib, 4096                                  # never read: every call is refused before anything is launched
    splits = (ctypes.c_int * 2)(32, 32)
    good = [some, 64, 1, 5, 64, some, 2 * 16 * 64, some, 64 * 16, 16, some, 2, some, some, 2, splits, 2, some, 64, None, 0, None]
    for i, bad in ((0, None), (0, 4100), (1, 56), (1, 68), (2, 0), (3, -1), (3, 1 << 40), (4, 60), (4, 0), (4, (1 << 20) + 8), (5, None), (6, 100), (7, None), (8, 100), (9, 12), (9, 264), (9, 0), (10, None), (11, 0),
                   (12, None), (13, None), (14, 0), (15, None), (15, (ctypes.c_int * 2)(32, 12)), (15, (ctypes.c_int * 2)(64, 0)), (16, 0), (16, 9), (17, None), (17, 4104), (18, 56)):
        args = list(good)
        args[i] = bad
        assert lib.lowbit_lora_add_cuda(*args) == 1, (i, bad)
    good[3], good[19], good[20] = 3000, some, 1 << 30
    for i, bad in ((19, None), (19, 4100), (20, 3000 * 2 * 16 * 4)):
        args = list(good)
        args[i] = bad
        assert lib.lowbit_lora_add_cuda(*args) == 4, (i, bad)
    assert lib.lowbit_lora_workspace_size(64, 64, 64, 16, 2, 3, 4) == 0 and lib.lowbit_lora_workspace_size(3000, 64, 64, 16, 2, 3, 4) >= 3000 * (32 * 4 + 4)


# ------------------------------------------------------------------ three launches: which calls take them is a rule of cost, so every test here asks for it
def launches(lora, s):
    """1, or 3 where the call needs a workspace"""
    L, S, R, K = s["a"].shape
    return 3 if lora.ggml.lowbit_lora_workspace_size(s["x"].shape[0], K, s["out"].shape[1], R, S, L, s["ids"].shape[0]) else 1


def many(dtype, dev, K=256, splits=(128, 64), rank=16, pad=3, adapters=12, requests=40, seed=0):
    """requests of one token and chunks, of more adapters than one launch takes"""
    lens = [1 if i % 3 else 2 + i % 37 for i in range(requests)]
    ids = [i * 5 % (adapters + 1) - 1 for i in range(requests)]
    return make(lens, ids, K, list(splits), rank, adapters, dtype, dev, pad=pad, seed=seed), lens, ids


def by_rows(cu, ids, adapters, T):
    """the adapter of every row: a request has what lies behind all in front of it and before its own end, none behind the list's end"""
    rows = [-1] * T
    for r, i in enumerate(ids):
        for t in range(max(max(cu[:r + 1]), 0), min(cu[r + 1], cu[-1], T)):
            rows[t] = i if 0 <= i < adapters else -1
    return rows


SPREADS = [(256, (128, 64), 16), (1000, (136, 40, 40), 24), (512, (520,), 64), (96, (128, 128), 128), (64, (72,), 256), (2048, (2040,), 48)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("K,splits,rank", SPREADS)
def test_three_launches_on_streams_recorded_and_from_threads(lora, cuda_device, dtype, K, splits, rank):
    import threading
    s, lens, ids = many(dtype, cuda_device, K, splits, rank)
    assert launches(lora, s) == 3
    want = check(lora, s, lens, ids)
    torch.cuda.synchronize()
    got = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            got.extend(run(lora, s) for _ in range(4))
    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert len(got) == 12 and all(torch.equal(g, want) for g in got)
    # recorded, and repeated for other requests
    out = s["out"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lora.lora_add_(out, s["x"], s["a"], s["b"], s["scales"], s["ids"], s["cu"], splits=s["splits"])
    T = s["x"].shape[0]
    for lens, ids in ((lens, ids), ([0] * 39 + [T], [3] * 40), ([T // 40] * 40, [i % 14 - 1 for i in range(40)]), ([T - 60] + [1] * 39, [0] + list(range(39)))):
        s["cu"].copy_(torch.tensor([0] + lens, dtype=torch.int32, device=cuda_device).cumsum(0))
        s["ids"].copy_(torch.tensor(ids, dtype=torch.int32))
        out.copy_(s["out"])
        graph.replay()
        assert torch.equal(out, check(lora, s, lens, ids))


@pytest.mark.gpu
def test_three_launches_of_rows_far_apart(lora, cuda_device):
    """rows of 2^27 elements: 256 of them at a time, a request on both sides of the border and others behind it"""
    T, step = 270, 1 << 27
    if torch.cuda.mem_get_info()[0] < T * step * 2 + (4 << 30):
        pytest.skip("needs 73 GB")
    lens, ids = [20] * 12 + [10, 9, 8], [0, 1, 2, 3, -1, 5, 6, 7, 8, 9, 1, 2, 3, 4, 5]
    s = make(lens, ids, 64, [64], 16, 10, torch.float16, cuda_device, pad=3)
    assert launches(lora, s) == 3
    want = run(lora, s)
    far = torch.empty(T * step, dtype=torch.float16, device=cuda_device).as_strided((T, 64), (step, 1))
    far.copy_(s["out"])
    lora.lora_add_(far, s["x"], s["a"], s["b"], s["scales"], s["ids"], s["cu"])
    value, bound = statement(s, lens, ids)
    assert bool(((far.double() - value).abs() <= bound).all()) and torch.equal(far[-3:], s["out"][-3:]) and torch.equal(far[80:100], s["out"][80:100])
    far.copy_(s["x"])
    got = run(lora, {**s, "x": far})
    assert bool(((got.double() - value).abs() <= bound).all()) and torch.equal(got[-3:], want[-3:])


@pytest.mark.gpu
@pytest.mark.parametrize("R", [40, 1100])
def test_three_launches_of_a_list_that_goes_back(lora, cuda_device, R):
    """the running maximum within a block's look at the requests, and from one look to the next"""
    T, adapters = 400, 9
    g = torch.Generator().manual_seed(R)
    cu = [-30] + (torch.arange(R) * T // R + torch.randint(-60, 30, (R,), generator=g)).tolist()
    ids = torch.randint(-1, adapters + 1, (R,), generator=g).tolist()
    for end in (T + 5, T - 11):
        s = make([T], [0], 64, [64], 8, adapters, torch.bfloat16, cuda_device)
        cu[-1] = end
        s["cu"], s["ids"] = (torch.tensor(v, dtype=torch.int32, device=cuda_device) for v in (cu, ids))
        assert launches(lora, s) == 3
        check(lora, s, [1] * T, by_rows(cu, ids, adapters, T))


@pytest.mark.gpu
@pytest.mark.parametrize("up", [2.0 ** 7, 2.0 ** -9])
def test_three_launches_of_products_beyond_fp16(lora, cuda_device, up):
    """as above: rows of very different size, and what brings them back through memory"""
    s, lens, ids = many(torch.float16, cuda_device, splits=(64, 24))
    s["x"] *= up
    s["x"][::3] *= 2.0 ** -6
    s["a"] *= up * 64 if up > 1 else up
    s["b"] *= 2.0 ** -12 if up > 1 else 2.0 ** 8
    assert launches(lora, s) == 3 and bool(torch.isfinite(statement(s, lens, ids)[0]).all())
    check(lora, s, lens, ids)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_three_launches_round_the_result_alone(lora, cuda_device, dtype):
    s, lens, ids = many(dtype, cuda_device, 512, (256,), 32)
    assert launches(lora, s) == 3
    s["out"].zero_()
    s["out"] = (-statement(s, lens, ids)[0]).to(dtype)
    check(lora, s, lens, ids)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_three_launches_keep_what_is_not_finite_in_its_row(lora, cuda_device, dtype):
    s, lens, ids = many(dtype, cuda_device)
    ids = [2 if i == 11 else i for i in ids]                           # nobody has the last adapter
    s["ids"].copy_(torch.tensor(ids, dtype=torch.int32))
    assert launches(lora, s) == 3
    clean = run(lora, s)
    nan = torch.zeros(len(clean), dtype=torch.bool, device=cuda_device)
    for r in (3, 9, 21):                                               # chunks, and one of their rows alone
        assert ids[r] >= 0 and lens[r] > 1
        nan[sum(lens[:r]):sum(lens[:r + 1]) if r != 9 else sum(lens[:r]) + 1] = True
    s["x"][nan] = math.nan
    s["x"][sum(lens):] = math.inf
    s["a"][11], s["b"][11] = math.nan, math.inf
    got = run(lora, s)
    assert torch.equal(got[~nan], clean[~nan]) and bool(torch.isnan(got[nan]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_three_launches_of_views_and_shared_memory(lora, cuda_device, monkeypatch, native):
    """rows of wider tensors, rows off 16 bytes, the output in the input's place; with the native host side and without"""
    s, lens, ids = many(torch.bfloat16, cuda_device, 256, (256,), 16, pad=0)
    assert launches(lora, s) == 3
    want = check(lora, s, lens, ids)
    if not native:
        monkeypatch.setattr(lora.paged_kv, "_native", lambda *args: None)
    assert torch.equal(run(lora, s), want)
    T = sum(lens)
    wide_x, wide_out, odd = (torch.full((T, n), 7.0, dtype=torch.bfloat16, device=cuda_device) for n in (304, 288, 259))
    wide_x[:, 16:272], wide_out[:, 24:280], odd[:, 3:] = s["x"], s["out"], s["x"]
    lora.lora_add_(wide_out[:, 24:280], wide_x[:, 16:272], s["a"], s["b"], s["scales"], s["ids"], s["cu"])
    assert torch.equal(wide_out[:, 24:280], want) and bool((wide_out[:, :24] == 7).all()) and bool((wide_out[:, 280:] == 7).all())
    assert torch.equal(run(lora, {**s, "x": odd[:, 3:]}), want)
    both = s["x"].clone()                                              # x += adapters of x
    case = {**s, "out": s["x"]}
    assert torch.equal(lora.lora_add_(both, both, s["a"], s["b"], s["scales"], s["ids"], s["cu"]), run(lora, case))


@pytest.mark.gpu
@pytest.mark.parametrize("adapters,K,splits,rank", [(1, 520, (264, 8), 64), (3, 520, (264, 8), 136), (8, 520, (264, 8), 8), (8, 4096, (4096,), 16), (8, 96, (64,), 48)])
def test_both_sides_of_where_the_launches_change(lora, cuda_device, adapters, K, splits, rank):
    """the last number of rows that takes one launch, and the first that takes three"""
    for T in range(max(adapters, 2), 5000):
        args = (K, sum(splits), rank, len(splits), adapters, adapters)
        if lora.ggml.lowbit_lora_workspace_size(T, *args):
            break
    assert lora.ggml.lowbit_lora_workspace_size(T, *args) > 0 == lora.ggml.lowbit_lora_workspace_size(T - 1, *args)
    for rows, expect in ((T - 1, 1), (T, 3)):
        lens = [rows // adapters] * (adapters - 1)
        lens.append(rows - sum(lens))
        s = make(lens, list(range(adapters)), K, list(splits), rank, adapters, torch.float16, cuda_device)
        assert launches(lora, s) == expect
        check(lora, s, lens, list(range(adapters)))
