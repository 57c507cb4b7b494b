"""Scores of given tokens from a model's logits.

What the evaluation harness makes of the logits that ``CompressionBackend.run_decode`` returns
(perplexity of a continuation, how sure the model was), and what a server returns as the log
probabilities of a prompt or of sampled tokens, in one pass over the logits
(``knlp_b200_token_score``): the reference computes them with ``log_softmax`` over the whole
vocabulary in fp32 (compute_ppl of its harnesses).  CUDA tensors only.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib, ops


class TokenScores(NamedTuple):
    logprob: torch.Tensor  # fp32 [...]
    entropy: torch.Tensor  # fp32 [...], nats
    rank: torch.Tensor  # int32 [...], 1 = no logit is larger
    top_ids: torch.Tensor  # int64 [..., k], descending, lower index first among equals
    top_logprobs: torch.Tensor  # fp32 [..., k]


def token_logprobs(logits: torch.Tensor, token_ids: torch.Tensor, top_k: int = 0) -> TokenScores:
    """Log probability, rank and alternatives of ``token_ids`` [...] under ``logits``
    [..., vocab] (float32 / float16 / bfloat16, -inf masks a token), with the entropy of each
    distribution.

    A negative id marks a row without a token: logprob 0, rank 0.  An id >= vocab gives NaN and
    rank 0.  A row without a logit above -inf has entropy 0 and log probabilities -inf; NaN or
    +inf logits make the row's logprob and entropy NaN, and NaN counts as the largest.
    ``top_k`` <= 64."""
    dev = ops._need_cuda(logits, token_ids)
    dt = ops._dt(logits)
    if token_ids.dtype != torch.int64:
        raise TypeError("token_ids must be int64")
    if logits.dim() < 1 or logits.shape[:-1] != token_ids.shape:
        raise ValueError("expected logits [..., vocab] and token_ids [...]")
    vocab = logits.shape[-1]
    if vocab == 0:
        raise ValueError("the vocabulary is empty")
    if not 0 <= top_k <= min(_lib.MAX_TOP, vocab):
        raise ValueError(f"top_k must lie in [0, min({_lib.MAX_TOP}, vocab)]")
    x = logits
    if x.dim() != 2:
        x = x.reshape(-1, vocab)
    if vocab > 1 and x.stride(1) != 1:
        x = x.contiguous()
    ids = token_ids.reshape(-1)
    if not ids.is_contiguous():
        ids = ids.contiguous()
    n = ids.numel()
    if max(n, vocab) >= 2 ** 31:
        raise ValueError("too many rows or too large a vocabulary")
    shape = tuple(token_ids.shape)
    logprob = torch.empty(shape, dtype=torch.float32, device=dev)
    entropy = torch.empty_like(logprob)
    rank = torch.empty(shape, dtype=torch.int32, device=dev)
    top_ids = torch.empty(shape + (top_k,), dtype=torch.int64, device=dev)
    top_lp = torch.empty(shape + (top_k,), dtype=torch.float32, device=dev)
    if n:
        with ops._on(dev):
            rc = _lib.load().knlp_b200_token_score(
                x.data_ptr(), dt, x.stride(0), ids.data_ptr(), n, vocab, top_k,
                logprob.data_ptr(), entropy.data_ptr(), rank.data_ptr(),
                top_ids.data_ptr() if top_k else None, top_lp.data_ptr() if top_k else None,
                ops._stream(dev))
        _lib.check(rc, "knlp_b200_token_score")
    return TokenScores(logprob, entropy, rank, top_ids, top_lp)
