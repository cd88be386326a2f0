"""How probable the tokens of a model are: log probabilities of given tokens, the entropy of their distributions, the best alternatives.

candle's examples draw a token from the logits and drop the rest (candle-transformers/src/generation/mod.rs:60-130); a program that scores, ranks or filters
what a model has said needs these numbers, from one read of the logits.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import capi
from .capi import CandleQError

_ELEM = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}


class TokenLogProbs(NamedTuple):
    logprob: torch.Tensor | None        # f32 [rows], of the given tokens
    entropy: torch.Tensor               # f32 [rows], in nats
    top_logprobs: torch.Tensor          # f32 [rows, top], descending
    top_ids: torch.Tensor               # int64 [rows, top]; the lower index first among equals


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None = None, top: int = 0) -> TokenLogProbs:
    """logits: CUDA [..., vocab], f32, f16 or bf16; tokens: whole numbers of the leading shape.  top: 0 .. 32 alternatives.  Sums are f32 and so are the results.

    A negative token counts as no token: its log probability is 0.  One beyond the vocabulary gives NaN.  Logits of -inf are tokens that cannot be: their
    log probability is -inf.  A row with a NaN or +inf, or with nothing but -inf, is no distribution: its numbers are NaN and its ids -1."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda or logits.dim() < 1:
        raise CandleQError("token_logprobs needs CUDA logits [..., vocab]: there is no CPU path")
    if logits.dtype not in _ELEM:
        raise CandleQError(f"Expected f32/f16/bf16, got {logits.dtype}")
    shape, dev = logits.shape, logits.device
    vocab, flat = shape[-1], len(shape) == 2
    if vocab == 0 or not 0 <= top <= min(32, vocab):
        raise CandleQError(f"token_logprobs: 0 <= top <= min(32, vocab), got {top} of {vocab}")
    x = logits if flat else logits.reshape(-1, vocab)
    rows, step = x.shape[0], x.stride(0)
    if (x.stride(1) != 1 and vocab > 1) or (rows > 1 and step < 0):
        x, step = x.contiguous(), vocab
    lead = shape[:-1]
    tokens_at = logprob = logprob_at = None
    entropy = torch.empty(rows, dtype=torch.float32, device=dev)
    if tokens is not None:
        if tokens.shape != lead or tokens.is_floating_point() or tokens.dtype == torch.bool or tokens.get_device() != logits.get_device():
            raise CandleQError(f"token_logprobs: tokens must be whole numbers of shape {list(lead)} on {dev}")
        if not flat:
            tokens = tokens.reshape(-1)
        if tokens.dtype != torch.int64 or not tokens.is_contiguous():
            tokens = tokens.to(torch.int64).contiguous()
        logprob = torch.empty_like(entropy)
        tokens_at, logprob_at = tokens.data_ptr(), logprob.data_ptr()
    best = torch.empty((rows, top), dtype=torch.float32, device=dev)
    ids = torch.empty_like(best, dtype=torch.int64)
    if rows:
        lib = capi.lib()
        with capi.on_device(dev):
            nbytes = lib.cq_token_logprobs_scratch_bytes(rows, vocab, top)
            if nbytes == 0:
                raise CandleQError(f"token_logprobs: {rows} rows of {vocab} are too many for one call")
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            lib.cq_token_logprobs(x.data_ptr(), _ELEM[x.dtype], step if rows > 1 else vocab, rows, vocab, tokens_at, top, logprob_at, entropy.data_ptr(), best.data_ptr(),
                                  ids.data_ptr(), scratch.data_ptr(), capi.stream_of(dev))
        capi.check("token_logprobs")
    if flat:
        return TokenLogProbs(logprob, entropy, best, ids)
    return TokenLogProbs(None if logprob is None else logprob.view(lead), entropy.view(lead), best.view(*lead, top), ids.view(*lead, top))
