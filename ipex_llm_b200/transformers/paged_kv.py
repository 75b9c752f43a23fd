"""A paged key/value cache for many requests that come and go, and the operators around it -- what the reference's serving engine
(its vLLM integration) keeps beside the one-batch caches of transformers/kv.py.

The cache of a layer is two tensors [pages, page_size, kv_heads, head_dim], of the activations' type or uint8 (e5m2 bytes, the format of
``DynamicFp8Cache``).  Request r's tokens lie in the pages that row r of the block table names, in order; a token's slot is
``page * page_size + row``.  The new tokens of a step are packed: those of request r are rows ``cu_seqlens[r]`` to ``cu_seqlens[r + 1]``
of every activation.

A step of a server is ``paged_step`` once (pages, slots, positions: one launch, nothing comes back to the host, so a step can be recorded),
then per layer ``paged_rope_append`` on the projection's output and ``sdp_paged`` -- or ``sdp_packed`` where every request starts with its
whole prompt -- and ``paged_release`` for requests that are done.  None of them has a backward pass: tensors that want a
gradient, or carry a tangent of forward mode, are refused.
"""
import math
from typing import NamedTuple

import torch

from ipex_llm_b200.utils.common import invalidInputError, LazyModule

ggml = LazyModule("ipex_llm_b200.ggml.model.llama.llama_cpp")      # loaded by the first call of one of its kernels
linears = LazyModule("ipex_llm_b200.transformers.low_bit_linear")   # their native host side has these operators' too

_HALF = (torch.float16, torch.bfloat16)


class PagedStep(NamedTuple):
    """what ``paged_step`` finds out about a step, all on the device"""
    cu_seqlens: torch.Tensor          # int32 [R + 1]: first packed row of every request
    seq_lens: torch.Tensor            # int32 [R]: tokens that a request holds once its new ones are written
    positions: torch.Tensor           # int64 [n_tokens]: position of every packed row, 0 behind the last
    slots: torch.Tensor               # int64 [n_tokens]: its slot, -1 behind the last and where no page was to be had
    free_count: torch.Tensor          # int32 [1]: free pages left
    missing: torch.Tensor             # int32 [1]: pages that were not to be had


def _native(name, *args):
    """the plain call in one native call (csrc/host/paged_host.cpp); None where the statements here serve or refuse it"""
    host = linears._host if linears._host is not None else linears._load_host()
    out = getattr(host, name)(*args) if host else None
    if type(out) is int:
        ggml._check(out, "lowbit_" + name)
    return out


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)


def _device(*tensors):
    """the one CUDA device that all of them are on"""
    dev = tensors[0].device
    invalidInputError(dev.type == "cuda", "the paged cache's operators run on a CUDA device (there is no CPU path)")
    for t in tensors[1:]:
        invalidInputError(t.device == dev, f"tensors on {dev} and {t.device}")
    return dev


def _ints(t, n, name, dtype=torch.int32):
    invalidInputError(t.dtype == dtype and t.dim() == 1 and t.shape[0] == n and t.is_contiguous(), f"{name} must be a contiguous {dtype} [{n}]")


def _table(block_table):
    invalidInputError(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.stride(1) == 1 and block_table.numel() > 0
                      and block_table.stride(0) >= block_table.shape[1], "block_table must be an int32 [requests, pages] with contiguous rows")


def _no_grad(*tensors):
    """none of them (None: not given) wants a gradient or carries a tangent"""
    tensors = [t for t in tensors if t is not None]
    invalidInputError(not (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)), "the paged cache's operators have no backward pass")
    invalidInputError(all(torch.autograd.forward_ad.unpack_dual(t).tangent is None for t in tensors), "the paged cache's operators have no forward-mode derivative (a tensor carries a tangent)")


def _caches(k_cache, v_cache, dtype, head_dim):
    invalidInputError(k_cache.dim() == 4 and v_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.dtype == v_cache.dtype
                      and k_cache.stride(3) == 1 and v_cache.stride(3) == 1 and k_cache.numel() > 0,
                      "caches must be two [pages, page_size, kv_heads, head_dim] with contiguous heads")
    invalidInputError(k_cache.dtype in (dtype, torch.uint8), f"a {k_cache.dtype} cache beside {dtype} activations")
    invalidInputError(k_cache.shape[3] == head_dim, f"the cache's heads have {k_cache.shape[3]} elements, the activations' {head_dim}")


def paged_step(query_lens, context_lens, block_table, free_pages, free_count, page_size, n_tokens, free_left=None):
    """Pages, slots and positions of a step in one launch.

    ``query_lens`` / ``context_lens`` int32 [R]: tokens that every request brings, and holds already; ``block_table`` int32 [R, width],
    -1 where a request has no page: the pages that the new tokens need are entered (in place); ``free_pages`` int32 [N] with ``free_count``
    int32 [1]: the stack that they come off, the last first; ``n_tokens``: rows of the step's activations (at least the sum of
    ``query_lens``: what is behind it is padding).  ``free_left``: where the number of pages left goes, a new tensor by default;
    ``free_count`` itself for a server's loop.  Returns a ``PagedStep``.

    Where ``missing`` is not 0 the pages that there were have been handed out, to earlier requests first.  The step is repeated after it has been
    taken back, ``paged_release(every row, block_table, free_pages, the count that it left, context_lens, page_size)``, and somebody has gone: what the
    table names behind ``context_lens`` is written over, and pages that only it named would be nobody's.  The same holds for tokens that a request
    drops.  The count that the next call gets is the one that this call left: an older one hands pages out twice."""
    out = _native("paged_step", query_lens, context_lens, block_table, free_pages, free_count, page_size, n_tokens, free_left)
    if out is not None:
        return PagedStep._make(out)
    R = query_lens.shape[0]
    dev = _device(query_lens, context_lens, block_table, free_pages, free_count)
    _ints(query_lens, R, "query_lens")
    _ints(context_lens, R, "context_lens")
    _table(block_table)
    invalidInputError(R > 0 and block_table.shape[0] == R, f"{R} requests, {block_table.shape[0]} rows of the block table")
    _ints(free_pages, free_pages.shape[0], "free_pages")
    _ints(free_count, 1, "free_count")
    page_size, n_tokens = int(page_size), int(n_tokens)
    invalidInputError(page_size > 0 and n_tokens >= 0 and free_pages.shape[0] > 0, "page_size and the number of pages must be positive")
    if free_left is None:
        free_left = torch.empty(1, dtype=torch.int32, device=dev)
    else:
        _device(free_count, free_left)
        _ints(free_left, 1, "free_left")
    out = PagedStep(torch.empty(R + 1, dtype=torch.int32, device=dev), torch.empty(R, dtype=torch.int32, device=dev),
                    torch.empty(n_tokens, dtype=torch.int64, device=dev), torch.empty(n_tokens, dtype=torch.int64, device=dev), free_left,
                    torch.empty(1, dtype=torch.int32, device=dev))
    with torch.cuda.device(dev):
        ggml.lowbit_paged_step(query_lens, context_lens, block_table, free_pages, free_count, free_left, page_size, out.cu_seqlens, out.seq_lens,
                               out.positions, out.slots, out.missing, _stream(dev))
    return out


def paged_release(done, block_table, free_pages, free_count, held=None, page_size=None):
    """Requests that are done give their pages back: rows of ``block_table`` with ``done`` (bool or uint8 [R]) set go onto the stack
    ``free_pages`` / ``free_count`` and become -1, in place.  With ``held`` (int32 [R]: tokens that they keep) and the ``page_size`` they give back
    only what lies behind those: a step that found too few pages is taken back so, and tokens that a request drops.  A page that several rows name
    would go back once for each."""
    dev = _device(done, block_table, free_pages, free_count)
    invalidInputError(done.dtype in (torch.bool, torch.uint8) and done.dim() == 1 and done.is_contiguous() and done.shape[0] > 0, "done must be a contiguous bool [R]")
    _table(block_table)
    invalidInputError(block_table.shape[0] == done.shape[0], f"{done.shape[0]} requests, {block_table.shape[0]} rows of the block table")
    _ints(free_pages, free_pages.shape[0], "free_pages")
    _ints(free_count, 1, "free_count")
    invalidInputError((held is None) == (page_size is None), "held and page_size come together")
    if held is not None:
        _device(done, held)
        _ints(held, done.shape[0], "held")
        invalidInputError(int(page_size) > 0, "page_size must be positive")
    with torch.cuda.device(dev):
        if held is None:
            ggml.lowbit_paged_release(done, block_table, free_pages, free_count, _stream(dev))
        else:
            ggml.lowbit_paged_release_behind(done, held, block_table, page_size, free_pages, free_count, _stream(dev))


def paged_rope_append(qkv, n_heads, n_kv_heads, head_dim, cos, sin, positions, slots, k_cache, v_cache):
    """Rotary embedding of the query and key heads of the merged projection's output ``qkv`` [T, (n_heads + 2 n_kv_heads) * head_dim], in
    place, and the write of keys and values into their ``slots`` (int64 [T], none twice; -1: not written).  ``cos`` / ``sin`` [positions, rotary width]
    in the rotate_half layout, indexed by ``positions`` (int64 [T]; beyond the tables: their last row); a rotary width below head_dim
    leaves the other elements; None: no rotation.  e5m2 caches keep the rounded activations' nearest value, saturating."""
    if _native("paged_append", qkv, n_heads, n_kv_heads, head_dim, cos, sin, positions, slots, k_cache, v_cache) is not None:
        return
    _no_grad(qkv, cos, sin, k_cache, v_cache)
    invalidInputError(qkv.dim() == 2 and qkv.dtype in _HALF and qkv.shape[1] == (n_heads + 2 * n_kv_heads) * head_dim and (qkv.stride(1) == 1 or qkv.numel() == 0),
                      f"qkv must be a half-precision [T, {(n_heads + 2 * n_kv_heads) * head_dim}] with contiguous rows")
    invalidInputError(qkv.shape[0] <= 1 or qkv.stride(0) >= qkv.shape[1], "the rows of qkv overlap")
    T, rotary = qkv.shape[0], 0
    dev = _device(qkv, slots, k_cache, v_cache)
    _ints(slots, T, "slots", torch.int64)
    _caches(k_cache, v_cache, qkv.dtype, head_dim)
    invalidInputError(k_cache.shape[2] == n_kv_heads, f"the cache has {k_cache.shape[2]} kv heads, the activations {n_kv_heads}")
    invalidInputError((cos is None) == (sin is None), "cos and sin come together")
    if cos is not None:
        _device(qkv, cos, sin, positions)
        _ints(positions, T, "positions", torch.int64)
        invalidInputError(cos.dim() == 2 and cos.shape == sin.shape and cos.dtype == sin.dtype and cos.dtype in _HALF + (torch.float32,)
                          and cos.stride(1) == 1 and cos.stride() == sin.stride() and cos.shape[0] > 0, "cos / sin must be two [positions, rotary width] of one type")
        rotary = cos.shape[1]
        invalidInputError(0 < rotary <= head_dim and rotary % 2 == 0, f"rotary width {rotary} with heads of {head_dim} elements")
    if T == 0:
        return
    with torch.cuda.device(dev):
        ggml.lowbit_paged_rope_append(qkv, n_heads, n_kv_heads, head_dim, rotary, cos, sin, positions, slots, k_cache, v_cache, _stream(dev))


def _attention_args(query, n_kv_heads, cu_seqlens, scale, out):
    invalidInputError(query.dim() == 3 and query.dtype in _HALF, "queries must be a half-precision [T, heads, head_dim]")
    T, H, D = query.shape
    invalidInputError(H % n_kv_heads == 0 and D % 16 == 0 and 0 < D <= 256, f"unsupported attention shape ({H} heads over {n_kv_heads}, head_dim {D})")
    invalidInputError(cu_seqlens.dtype == torch.int32 and cu_seqlens.dim() == 1 and cu_seqlens.shape[0] >= 2 and cu_seqlens.is_contiguous(),
                      "cu_seqlens must be a contiguous int32 [requests + 1]")
    scale = 1 / math.sqrt(D) if scale is None else float(scale)
    invalidInputError(scale > 0, "the scale must be positive")
    if not _rows_aligned(query):
        query = query.clone(memory_format=torch.contiguous_format)
    if out is None:
        out = torch.empty((T, H, D), dtype=query.dtype, device=query.device)
    else:
        invalidInputError(out.shape == query.shape and out.dtype == query.dtype and out.device == query.device and _rows_aligned(out),
                          "out must have the queries' shape, type and device and 16-byte aligned rows")
    return query, scale, out


def _rows_aligned(t):
    """rows of the last dimension contiguous and on 16 bytes"""
    unit = 16 // t.element_size()
    return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % unit == 0 for s in t.stride()[:-1])


def sdp_paged(query, k_cache, v_cache, block_table, seq_lens, cu_seqlens, scale=None, max_query_len=None, out=None):
    """Attention of every request's new tokens over its pages (``paged_rope_append`` has written the new tokens' own keys).

    ``query`` [T, heads, head_dim], packed; request r's i-th of n new tokens sees keys 0 .. seq_lens[r] - n + i, grouped heads as in
    ``scaled_dot_product_attention``, at most 256 on one kv head (128 where head_dim is above 128).  ``max_query_len``: no request brings more
    new tokens (1 for a decode step; the rows of one that does are undefined); never knowing is right, knowing saves launches.  A token that
    sees no key gives zeros; rows behind the last request are left as they are in ``out``, a new tensor by default.  Pages outside the
    cache (-1) make their request's rows NaN, and so do more tokens than its row of the table can name; keys or values that are not finite may do so to all rows of their request."""
    if out is None:
        result = _native("sdp_paged", query, k_cache, v_cache, block_table, seq_lens, cu_seqlens, scale, max_query_len)
        if result is not None:
            return result
    _no_grad(query, k_cache, v_cache, out)
    dev = _device(query, k_cache, v_cache, block_table, seq_lens, cu_seqlens)
    _table(block_table)
    _caches(k_cache, v_cache, query.dtype, query.shape[-1])
    invalidInputError(_rows_aligned(k_cache) and _rows_aligned(v_cache), "the caches' rows must be 16-byte aligned")
    query, scale, out = _attention_args(query, k_cache.shape[2], cu_seqlens, scale, out)
    T, H, D = query.shape
    R = block_table.shape[0]
    _ints(seq_lens, R, "seq_lens")
    invalidInputError(cu_seqlens.shape[0] == R + 1, f"{R} rows of the block table, {cu_seqlens.shape[0] - 1} requests in cu_seqlens")
    invalidInputError(block_table.shape[1] * k_cache.shape[1] < 1 << 31, "a request's pages hold fewer than 2^31 tokens")
    most = T if max_query_len is None else int(max_query_len)
    invalidInputError(most >= 0, "max_query_len must not be negative")
    if T == 0:
        return out
    with torch.cuda.device(dev):
        ws = torch.empty(ggml.lowbit_sdp_paged_workspace_size(T, R, H, k_cache.shape[2], D, most), dtype=torch.uint8, device=dev)
        ggml.lowbit_sdp_paged(query, k_cache, v_cache, block_table, seq_lens, cu_seqlens, scale, most, out, ws, _stream(dev))
    return out


def sdp_packed(query, key, value, cu_seqlens, scale=None, is_causal=True, max_seqlen=None, out=None):
    """Attention of whole prompts that lie behind one another, each over itself: ``query`` [T, heads, head_dim], ``key`` / ``value``
    [T, kv_heads, head_dim] (views of the merged projection's output serve), prompt r = rows cu_seqlens[r] .. cu_seqlens[r + 1].
    ``max_seqlen``: no prompt is longer.  Rows behind the last prompt are left as they are in ``out``."""
    if out is None:
        result = _native("sdp_packed", query, key, value, cu_seqlens, scale, is_causal, max_seqlen)
        if result is not None:
            return result
    _no_grad(query, key, value, out)
    dev = _device(query, key, value, cu_seqlens)
    invalidInputError(key.dim() == 3 and key.shape == value.shape and key.shape[0] == query.shape[0] and key.shape[2] == query.shape[-1] and key.shape[1] > 0
                      and key.dtype == query.dtype and value.dtype == query.dtype, "keys and values must be [T, kv_heads, head_dim] of the queries' type")
    query, scale, out = _attention_args(query, key.shape[1], cu_seqlens, scale, out)
    key, value = (t if _rows_aligned(t) else t.clone(memory_format=torch.contiguous_format) for t in (key, value))
    T, H, D = query.shape
    most = T if max_seqlen is None else int(max_seqlen)
    invalidInputError(most >= 0, "max_seqlen must not be negative")
    if T == 0:
        return out
    with torch.cuda.device(dev):
        ws = torch.empty(ggml.lowbit_sdp_packed_workspace_size(T, cu_seqlens.shape[0] - 1, H, key.shape[1], D, most), dtype=torch.uint8, device=dev)
        ggml.lowbit_sdp_packed(query, key, value, cu_seqlens, scale, is_causal, most, out, ws, _stream(dev))
    return out
