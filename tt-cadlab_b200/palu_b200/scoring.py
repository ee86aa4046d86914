"""Log probabilities of given tokens, the entropy and the top alternatives of rows of logits.

What a server answers next to its tokens, and what scores a prompt (perplexity, the quality measure of a compressed
cache): one kernel over the logits as the LM head wrote them (bf16 or fp32), without an fp32 copy, a softmax or a sort.
The reference decodes greedily and has none of this (palu_tt/generate.py:53-62).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from palu_b200 import _lib

MAX_TOP = 32


class TokenLogprobs(NamedTuple):
    """``logprob`` [N] of the given tokens and ``entropy`` [N] of the rows (nats, fp32); ``top_logprob`` [N, k] fp32 and
    ``top_id`` [N, k] int64, highest first."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprob: torch.Tensor
    top_id: torch.Tensor


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """Per row of ``logits`` [N, vocab] (bf16 or fp32, rows of any stride): the log probability of ``tokens`` [N] (int64 or
    int32), the entropy, and the ``top`` (at most 32) highest log probabilities with their ids (palu_token_logprobs).

    Equal logits are ordered by the lower id. A negative token stands for none and gives 0; one at or past the vocabulary
    gives NaN. A logit of -inf has probability 0; a row of -inf only, or with a NaN or +inf in it, has no distribution:
    its log probabilities and entropy are NaN. Everything is computed in fp32."""
    dtype, dev = logits.dtype, logits.device
    if not logits.is_cuda or not tokens.is_cuda:
        _lib.require_cuda(logits, tokens)
    if logits.dim() != 2 or (dtype != torch.bfloat16 and dtype != torch.float32) or not 1 <= logits.shape[1] < 2**31:
        raise RuntimeError(f"logits must be bf16 or fp32 [N, vocab], got {dtype} {tuple(logits.shape)}")
    n, vocab = logits.shape
    wide = tokens.dtype == torch.int64
    if tokens.dim() != 1 or tokens.shape[0] != n or not (wide or tokens.dtype == torch.int32):
        raise RuntimeError(f"tokens must be [{n}] int64 or int32, got {tokens.dtype} {tuple(tokens.shape)}")
    if tokens.device != dev:
        raise RuntimeError(f"tokens are on {tokens.device}, logits on {dev}")
    top = int(top)
    if not 0 <= top <= MAX_TOP or top > vocab:
        raise RuntimeError(f"top must be in [0, {min(MAX_TOP, vocab)}] (at most 32, at most the vocabulary), got {top}")
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return token_logprobs(logits, tokens, top)
    ld, step = logits.stride()
    if step != 1 or (n > 1 and ld < vocab):
        logits = logits.contiguous()
        ld = vocab
    tokens = tokens.contiguous()
    empty, f32 = torch.empty, torch.float32
    lp, tv = empty(n, dtype=f32, device=dev), empty(n, top, dtype=f32, device=dev)
    ent = torch.empty_like(lp)
    ti = empty(n, top, dtype=torch.int64, device=dev)
    _lib.check(_lib.load().palu_token_logprobs(
        logits.data_ptr(), ld, _lib.PALU_BF16 if dtype == torch.bfloat16 else _lib.PALU_F32, n, vocab, tokens.data_ptr(), wide, top,
        lp.data_ptr(), ent.data_ptr(), tv.data_ptr(), ti.data_ptr(), _lib.stream_handle(dev)))
    return TokenLogprobs(lp, ent, tv, ti)
