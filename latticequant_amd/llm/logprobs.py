"""Log probabilities of given tokens, with entropies and top alternatives.

What a decode step answers with beside its token (``accept_drafts`` takes the same
logits), and what an evaluation of a compressed cache sums: the reference's
llm/perplexity_eval.py takes a cross entropy of logits for that.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .. import _lib as L
from .paged import _no_grad

MAX_TOP = L.LQ_LOGPROBS_MAX_TOP


class TokenLogprobs(NamedTuple):
    """What token_logprobs returns, in the shape of its tokens."""
    logprob: torch.Tensor                  # fp32: log softmax at the given token
    entropy: torch.Tensor                  # fp32: -sum p log p
    top_ids: Optional[torch.Tensor]        # (..., top) int64, most likely first; None without top
    top_logprobs: Optional[torch.Tensor]   # (..., top) fp32


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top: int = 0) -> TokenLogprobs:
    """logits: (..., V) fp16, bf16 or fp32, rows of any strides with a contiguous last
    dimension (others are copied); tokens: (...) int64 or None (log probabilities 0 then);
    top: 0..64 alternatives, at most V.  Natural logarithms.
    A negative token names none: its log probability is 0; one of V or more gives NaN.
    Logits of -inf weigh nothing; a row of nothing else, or with a NaN or +inf, is NaN.
    Alternatives are in order of their logits, the lower id first of equal ones, NaN above
    all.  Nothing waits for the device."""
    if logits.dim() < 1 or logits.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise ValueError("logits must be (..., V) fp16, bf16 or fp32")
    dev = logits.device
    shape, V = logits.shape[:-1], logits.shape[-1]
    if tokens is not None and (tokens.shape != shape or tokens.dtype is not torch.int64 or tokens.device != dev):
        raise ValueError("tokens must be int64 of the logits' leading shape, on their device")
    if V < 1 or not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"top must be 0..{MAX_TOP}, at most the vocabulary")
    if dev.type != "cuda":
        raise ValueError("logits must be on the GPU")
    _no_grad("token_logprobs", logits)
    lib = L.lib()
    with L.on_device(dev):
        x = logits
        if x.stride(-1) != 1 and V > 1:
            x = x.contiguous()
        if x.dim() != 2:
            x = x.reshape(-1, V)
        n = x.shape[0]
        both = torch.empty((2,) + shape, dtype=torch.float32, device=dev)
        logprob, entropy = both.unbind()
        ids = tops = None
        if top:
            ids = torch.empty(shape + (top,), dtype=torch.int64, device=dev)
            tops = both.new_empty(shape + (top,))
        if n:
            tok = None if tokens is None else tokens.contiguous()
            at = both.data_ptr()
            L.check(lib.lq_token_logprobs(x.data_ptr(), L.dtype_code(x.dtype), x.stride(0), n, V,
                                          None if tok is None else tok.data_ptr(), top, at, at + 4 * n, L.ptr(ids),
                                          L.ptr(tops), L.raw_stream(dev)), "lq_token_logprobs")
    return TokenLogprobs(logprob, entropy, ids, tops)
