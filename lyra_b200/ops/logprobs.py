"""Scores of given tokens from logits (``csrc/elementwise/token_logprobs.cu``): log probability, entropy and the most likely
alternatives in one pass over the logits; the gradient of the first two is one more kernel."""

from __future__ import annotations

from typing import NamedTuple

import torch

from lyra_b200.ops import native

MAX_TOP_K = 32
MAX_VOCAB = 1 << 22      # on a GPU: a single warp may have to sweep a row of nothing but ties, in less time than a wait is given


class TokenLogprobs(NamedTuple):
    """``logprob, entropy [...]`` fp32 (differentiable), ``top_logprobs [..., k]`` fp32 and ``top_ids [..., k]`` int64 (not)."""

    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_ids: torch.Tensor


def check_arguments(logits: torch.Tensor, targets: torch.Tensor, top_k: int, vocab_size: int | None) -> int:
    """Refuses what neither path computes; returns the number of columns that take part."""
    if logits.ndim < 1 or tuple(targets.shape) != tuple(logits.shape[:-1]):
        raise ValueError(f"targets {tuple(targets.shape)} must have the shape of the logits' rows {tuple(logits.shape[:-1])}")
    if targets.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"targets must be int32 or int64, got {targets.dtype}")
    if targets.device != logits.device:
        raise ValueError(f"targets on {targets.device}, logits on {logits.device}")
    vocab = logits.shape[-1] if vocab_size is None else int(vocab_size)
    if not 1 <= vocab <= logits.shape[-1]:
        raise ValueError(f"vocab_size {vocab} must lie in 1..{logits.shape[-1]}")
    if not 0 <= top_k <= min(MAX_TOP_K, vocab):
        raise ValueError(f"top_k {top_k} must lie in 0..{min(MAX_TOP_K, vocab)}")
    return vocab


def _forward(logits, targets, k: int, vocab: int, norm: torch.Tensor | None):
    N, dev = logits.shape[0], logits.device
    logprob, entropy = torch.empty(N, dtype=torch.float32, device=dev), torch.empty(N, dtype=torch.float32, device=dev)
    top_lp, top_id = torch.empty(N, k, dtype=torch.float32, device=dev), torch.empty(N, k, dtype=torch.int64, device=dev)
    if N:
        fn = native.function("lyra_token_logprobs", "pippppppiiilpp")
        native.check(fn(logits.data_ptr(), logits.dtype == torch.bfloat16, targets.data_ptr(), logprob.data_ptr(), entropy.data_ptr(),
                        norm.data_ptr() if norm is not None else None, top_lp.data_ptr(), top_id.data_ptr(), N, vocab, k, logits.stride(0),
                        native.status_word().data_ptr(), native.stream_address()), "lyra_token_logprobs")
        native.count_launch()
    return logprob, entropy, top_lp, top_id


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, k, vocab):
        norm = torch.empty(2, logits.shape[0], dtype=torch.float32, device=logits.device)      # row maxima and log sums, for the gradient
        logprob, entropy, top_lp, top_id = _forward(logits, targets, k, vocab, norm)
        ctx.save_for_backward(logits, targets, norm, entropy)
        ctx.vocab = vocab
        ctx.mark_non_differentiable(top_lp, top_id)
        ctx.set_materialize_grads(False)
        return logprob, entropy, top_lp, top_id

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logprob, g_entropy, *_):
        logits, targets, norm, entropy = ctx.saved_tensors
        if g_logprob is None and g_entropy is None:
            return None, None, None, None
        N, W = logits.shape
        grad = torch.empty(N, W, dtype=logits.dtype, device=logits.device)
        if N:
            gl = g_logprob.float().contiguous() if g_logprob is not None else None
            gh = g_entropy.float().contiguous() if g_entropy is not None else None
            address = lambda t: t.data_ptr() if t is not None else None
            with native.on_device(logits):
                fn = native.function("lyra_token_logprobs_bwd", "pippppppiiilp")
                native.check(fn(logits.data_ptr(), logits.dtype == torch.bfloat16, grad.data_ptr(), targets.data_ptr(), norm.data_ptr(), entropy.data_ptr(),
                                address(gl), address(gh), N, ctx.vocab, W, logits.stride(0), native.stream_address()), "lyra_token_logprobs_bwd")
            native.count_launch()
        return grad, None, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top_k: int, vocab: int) -> TokenLogprobs:
    """CUDA path; the arguments have passed :func:`check_arguments`. Rows may be strided, elements of a row may not."""
    if logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"logits must be fp32 or bf16 on a GPU, got {logits.dtype}")
    if vocab > MAX_VOCAB:
        raise ValueError(f"token_logprobs takes at most {MAX_VOCAB} columns on a GPU, got {vocab}")
    lead = logits.shape[:-1]
    rows, flat = logits, targets
    if logits.ndim != 2:
        rows, flat = logits.reshape(-1, logits.shape[-1]), targets.reshape(-1)
    if rows.shape[0] and (rows.stride(1) != 1 or rows.stride(0) < rows.shape[1]):
        rows = rows.contiguous()                              # transposed logits, or one row expanded to many
    if flat.dtype != torch.int64 or not flat.is_contiguous():
        flat = flat.long().contiguous()
    with native.on_device(logits):
        if torch.is_grad_enabled() and rows.requires_grad:
            out = _TokenLogprobs.apply(rows, flat, top_k, vocab)
        else:
            out = _forward(rows, flat, top_k, vocab, None)
    return TokenLogprobs(*out) if logits.ndim == 2 else TokenLogprobs(*(t.reshape((*lead, *t.shape[1:])) for t in out))
