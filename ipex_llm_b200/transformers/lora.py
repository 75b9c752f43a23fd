"""Low-rank adapters of many requests at once, beside a projection that all of them share (a ``LowBitLinear`` whose weight stays packed): the reference's
serving engine loads such adapters next to its low-bit model and gives every request its own.

The rows of a step are packed as for the paged cache (transformers/paged_kv.py): those of request r are rows ``cu_seqlens[r]`` to ``cu_seqlens[r + 1]``.
After ``y = linear(x)``, ``lora_add_(y, x, ...)`` adds every request's own ``scale * (x A^T) B^T`` in place."""
import torch

from ipex_llm_b200.utils.common import invalidInputError, LazyModule

ggml = LazyModule("ipex_llm_b200.ggml.model.llama.llama_cpp")      # loaded by the first call of one of its kernels
paged_kv = LazyModule("ipex_llm_b200.transformers.paged_kv")        # its native host side has this operator's too

_HALF = (torch.float16, torch.bfloat16)
RANK_MOST, SPLITS_MOST = 256, 8


def _rows_aligned(t):
    return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and (t.shape[0] <= 1 or t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1])


def _overlap(a, b):
    """whether matrices of as many rows share memory: columns of one buffer side by side do not"""
    size, rows = a.element_size(), a.shape[0]
    at = [(t.data_ptr(), t.data_ptr() + ((rows - 1) * t.stride(0) * (rows > 1) + t.shape[1]) * size) for t in (a, b)]
    if at[0][1] <= at[1][0] or at[1][1] <= at[0][0]:
        return False
    if rows <= 1 or a.stride(0) != b.stride(0):
        return True
    behind = (at[1][0] - at[0][0]) % (a.stride(0) * size)
    return behind < a.shape[1] * size or behind + b.shape[1] * size > a.stride(0) * size


def lora_add_(out, x, a, b, scales, adapter_ids, cu_seqlens, splits=None):
    """``out`` [T, N] += scale (x A^T) B^T for every row whose request has an adapter, in place; returns ``out``.

    ``x`` [T, K]; ``a`` [adapters, rank, K] and ``b`` [adapters, N, rank], all fp16 or all bf16; ``scales`` fp32 [adapters]; ``adapter_ids`` int32 [requests],
    outside [0, adapters): none, and such rows stay as they are; ``cu_seqlens`` int32 [requests + 1] (``PagedStep.cu_seqlens``): rows behind the last request
    stay too.  The rank is a multiple of 8 up to 256 (adapters of a smaller one: rows of zeros), K (at most 2^20) and N multiples of 8.

    ``splits``: the widths of the projections that ``out`` merges (queries, keys and values: 4096, 1024, 1024), each with an A of its own: ``a`` is then
    [adapters, len(splits), rank, K], and columns of a projection take the product with its A.

    x A^T is summed in 32 bits and enters the second product as two 16-bit values, which leave out 2^-16 of it (bf16) or 2^-22 (fp16); ``out`` is rounded once, by
    2^-8 or 2^-11.  So the former shows only where ``out`` all but cancels what is added.  One launch, or three for more rows or larger products; nothing
    comes back to the host, and the lists are read on the device: a recorded step serves other requests.  An ``x`` that shares memory with ``out`` is copied first.  There is no backward pass: tensors that want a
    gradient or carry a tangent are refused."""
    if splits is not None:
        splits = [int(n) for n in splits]
    if paged_kv._native("lora_add", out, x, a, b, scales, adapter_ids, cu_seqlens, splits) is not None:
        return out
    tensors = (out, x, a, b, scales)
    dev = x.device
    invalidInputError(dev.type == "cuda", "adapters run on a CUDA device (there is no CPU path)")
    for t in tensors + (adapter_ids, cu_seqlens):
        invalidInputError(t.device == dev, f"tensors on {dev} and {t.device}")
    invalidInputError(not (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)), "lora_add_ has no backward pass")
    invalidInputError(all(torch.autograd.forward_ad.unpack_dual(t).tangent is None for t in tensors), "lora_add_ has no forward-mode derivative (a tensor carries a tangent)")
    invalidInputError(x.dim() == 2 and out.dim() == 2 and x.dtype in _HALF and out.dtype == x.dtype and a.dtype == x.dtype and b.dtype == x.dtype,
                      "x [T, K], out [T, N] and the adapters must be fp16 or bf16, all of one type")
    T, K = x.shape
    N = out.shape[1]
    splits = [N] if splits is None else splits
    if a.dim() == 3:
        a = a.unsqueeze(1)
    invalidInputError(a.dim() == 4 and b.dim() == 3, "a must be [adapters, (splits,) rank, K] and b [adapters, N, rank]")
    L, S, R = a.shape[:3]
    invalidInputError(out.shape[0] == T and a.shape[3] == K and b.shape[0] == L and b.shape[1] == N and b.shape[2] == R and L > 0,
                      f"x {list(x.shape)}, out {list(out.shape)}, a {list(a.shape)} and b {list(b.shape)} do not belong together")
    invalidInputError(0 < len(splits) <= SPLITS_MOST and len(splits) == S and sum(splits) == N and all(n > 0 and n % 8 == 0 for n in splits),
                      f"splits must be up to {SPLITS_MOST} multiples of 8, one for each A, that add up to {N}")
    invalidInputError(0 < R <= RANK_MOST and R % 8 == 0 and K % 8 == 0 and 0 < K <= 1 << 20,
                      f"rank {R} and K {K} must be multiples of 8, the rank at most {RANK_MOST}, K at most 2^20")
    invalidInputError(scales.dtype == torch.float32 and scales.shape == (L,) and scales.is_contiguous(), f"scales must be a contiguous fp32 [{L}]")
    invalidInputError(adapter_ids.dtype == torch.int32 and adapter_ids.dim() == 1 and adapter_ids.is_contiguous() and adapter_ids.shape[0] > 0,
                      "adapter_ids must be a contiguous int32 [requests]")
    invalidInputError(cu_seqlens.dtype == torch.int32 and cu_seqlens.shape == (adapter_ids.shape[0] + 1,) and cu_seqlens.is_contiguous(),
                      f"cu_seqlens must be a contiguous int32 [{adapter_ids.shape[0] + 1}]")
    if T == 0:
        return out
    invalidInputError(_rows_aligned(out), "the rows of out must be contiguous and 16-byte aligned")
    if not _rows_aligned(x) or _overlap(out, x):
        x = x.clone(memory_format=torch.contiguous_format)
    a, b = (t if t[0].is_contiguous() and t.data_ptr() % 16 == 0 and t.stride(0) % 8 == 0 and (t.shape[0] == 1 or t.stride(0) >= t[0].numel())
            else t.clone(memory_format=torch.contiguous_format) for t in (a, b))
    with torch.cuda.device(dev):
        ws = torch.empty(ggml.lowbit_lora_workspace_size(T, K, N, R, S, L, adapter_ids.shape[0]), dtype=torch.uint8, device=dev)
        ggml.lowbit_lora_add(x, a, b, scales, adapter_ids, cu_seqlens, splits, out, ws, torch._C._cuda_getCurrentRawStream(dev.index))
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)
    return out
