"""What a row of logits says about its tokens: the log probability of a given token, the entropy, the most likely alternatives -- what a server
answers beside its tokens (the reference's serving engine returns them with each; the greedy pick of the recorded decode step reads the same logits)
and what a loss on token probabilities is made of, with its gradient."""
from typing import NamedTuple, Optional

import torch

from ipex_llm_b200.utils.common import invalidInputError, LazyModule

ggml = LazyModule("ipex_llm_b200.ggml.model.llama.llama_cpp")      # loaded by the first call of one of its kernels
paged_kv = LazyModule("ipex_llm_b200.transformers.paged_kv")        # its native host side has this operator's too

_TYPES = (torch.float16, torch.bfloat16, torch.float32)
TOP_MOST = 32                                                       # alternatives of a row


class TokenLogprobs(NamedTuple):
    """what ``token_logprobs`` says, in 32 bits whatever the logits' type"""
    logprobs: torch.Tensor                      # fp32, the tokens' shape: log probability of the given token, 0 where that is outside the vocabulary
    entropy: torch.Tensor                       # fp32, the tokens' shape
    top_ids: Optional[torch.Tensor]             # int64 [..., top_k]: the largest logits in order, of equal ones the lower id first; None without top_k
    top_logprobs: Optional[torch.Tensor]        # fp32 [..., top_k]


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)


def _forward(logits, tokens, temperature, top_k, keep):
    rows, dev = logits.shape[0], logits.device
    f32 = {"dtype": torch.float32, "device": dev}
    logprobs, entropy = torch.empty(rows, **f32), torch.empty(rows, **f32)
    ids = torch.empty(rows, top_k, dtype=torch.int64, device=dev) if top_k else None
    top = torch.empty(rows, top_k, **f32) if top_k else None
    stats = torch.empty(rows, 4, **f32) if keep else None
    with torch.cuda.device(dev):
        ggml.lowbit_token_logprobs(logits, tokens, temperature, top_k, logprobs, entropy, ids, top, stats, _stream(dev))
    return logprobs, entropy, ids, top, stats


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature, top_k):
        logprobs, entropy, ids, top, stats = _forward(logits, tokens, temperature, top_k, True)
        ctx.save_for_backward(logits, tokens, ids, stats)
        ctx.more = temperature, top_k
        if not top_k:
            return logprobs, entropy
        ctx.mark_non_differentiable(ids)
        return logprobs, entropy, ids, top

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logprobs, g_entropy, _=None, g_top=None):
        logits, tokens, ids, stats = ctx.saved_tensors
        temperature, top_k = ctx.more
        # a hook for saved tensors may have brought them back in another layout, or as something else, which the kernel could not see
        if logits.stride(1) != 1 or logits.shape[0] > 1 and logits.stride(0) < logits.shape[1]:
            logits = logits.contiguous()
        tokens, stats, ids = (t if t is None else t.contiguous() for t in (tokens, stats, ids))
        invalidInputError(logits.is_cuda and logits.dtype in _TYPES and stats.dtype == torch.float32 and tokens.dtype == torch.int64 and (ids is None or ids.dtype == torch.int64)
                          and all(t is None or t.device == logits.device for t in (tokens, stats, ids)), "what token_logprobs saved came back as something else")
        given = [None if g is None else g.contiguous() for g in (g_logprobs, g_entropy, g_top)]
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        with torch.cuda.device(logits.device):
            ggml.lowbit_token_logprobs_grad(logits, tokens, temperature, top_k, ids, *given, stats, grad, _stream(logits.device))
        return grad, None, None, None


def token_logprobs(logits, tokens, top_k=0, temperature=1.0):
    """Log probabilities of ``tokens`` (int64 [...]) under softmax(``logits`` / ``temperature``) with ``logits`` [..., vocabulary] (fp16, bf16 or fp32), the
    entropy of every row in nats, and its ``top_k`` (at most 32) most likely tokens: one launch, one pass over logits [rows, vocabulary].  More dimensions are brought to that
    first, by a copy where rows do not follow one another (``logits[:, :-1]``), and their gradient's node is one in Python.  ``temperature`` and ``top_k`` are the
    call's, for all rows: a recorded call keeps them.

    A token outside the vocabulary (-100) has log probability 0 and no gradient of it.  Logits of -inf are tokens that cannot come: probability 0, nothing to
    the entropy, and among the alternatives last.  A row that has no probabilities -- a NaN, +inf, or nothing but -inf in it -- gives NaN, and -1 among the
    alternatives where it has fewer numbers than ``top_k``.

    Where the logits want a gradient, ``logprobs``, ``entropy`` and ``top_logprobs`` have one: another launch, which reads the logits again and writes their
    gradient, rounded once to their type.  The logits must not be overwritten before it.  It has no derivative of its own.
    The temperature lies between 1e-7 and 1e7.  A recording refuses logits that are a leaf, or a view of one, of which something lives that was computed on
    the default stream: their gradient cannot be recorded.  Without the native host side, which alone can see that, it refuses every leaf that wants a gradient."""
    out = paged_kv._native("token_logprobs", logits, tokens, top_k, temperature)
    if out is not None:
        return TokenLogprobs._make(out)
    invalidInputError(logits.dim() >= 1 and logits.dtype in _TYPES and logits.shape[-1] > 0, "logits must be fp16, bf16 or fp32 [..., vocabulary]")
    invalidInputError(logits.device.type == "cuda", "token_logprobs runs on a CUDA device (there is no CPU path)")
    invalidInputError(tokens.dtype == torch.int64 and tokens.device == logits.device and tokens.shape == logits.shape[:-1],
                      f"tokens must be int64 {list(logits.shape[:-1])} on the logits' device")
    top_k, temperature, V = int(top_k), float(temperature), logits.shape[-1]
    invalidInputError(0 <= top_k <= min(TOP_MOST, V), f"top_k must be between 0 and {min(TOP_MOST, V)}")
    invalidInputError(1e-7 <= temperature <= 1e7, "the temperature must be between 1e-7 and 1e7")
    if not paged_kv.linears._host and torch.is_grad_enabled() and logits.requires_grad and torch.cuda.is_current_stream_capturing():
        invalidInputError(not (logits._base if logits._is_view() else logits).is_leaf,
                          "logits that are a leaf with a gradient take no part in a recording without the native host side: what lives of them may end the process")
    shape = tokens.shape
    rows = logits.reshape(-1, V)
    if rows.shape[0] > 1 and (rows.stride(1) != 1 or rows.stride(0) < V) or V > 1 and rows.stride(1) != 1:
        rows = rows.contiguous()
    flat = tokens.reshape(-1).contiguous()
    if torch.is_grad_enabled() and logits.requires_grad or torch.autograd.forward_ad.unpack_dual(logits).tangent is not None:
        logprobs, entropy, *more = _TokenLogprobs.apply(rows, flat, temperature, top_k)
    else:
        logprobs, entropy, *more = _forward(rows, flat, temperature, top_k, False)
    ids, top = more[:2] if top_k else (None, None)
    if logits.dim() != 2:
        logprobs, entropy = logprobs.view(shape), entropy.view(shape)
        if top_k:
            ids, top = ids.view(*shape, top_k), top.view(*shape, top_k)
    return TokenLogprobs(logprobs, entropy, ids, top)
