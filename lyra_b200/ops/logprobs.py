"""Scores of given tokens from logits (``csrc/elementwise/token_logprobs.cu``): log probability, entropy and the most likely
alternatives in one pass over the logits; the gradient of the first two is one more kernel."""

from __future__ import annotations

from typing import NamedTuple

import torch

from lyra_b200.ops import native
from lyra_b200.ops.native import c_int, c_ll, ptr

MAX_TOP_K = 32


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


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, k, vocab):
        N, W = logits.shape
        dev = logits.device
        logprob, entropy = torch.empty(2, N, dtype=torch.float32, device=dev).unbind(0)
        norm = torch.empty(2, N, dtype=torch.float32, device=dev)          # row maxima and log sums, for the gradient
        top_lp = torch.empty(N, k, dtype=torch.float32, device=dev)
        top_id = torch.empty(N, k, dtype=torch.int64, device=dev)
        if N:
            native.check(native.kernels().lyra_token_logprobs(ptr(logits), c_int(int(logits.dtype == torch.bfloat16)), ptr(targets), ptr(logprob),
                                                              ptr(entropy), ptr(norm), ptr(top_lp), ptr(top_id), c_int(N), c_int(vocab), c_int(k),
                                                              c_ll(logits.stride(0)), native.stream_ptr()), "lyra_token_logprobs")
            native.count_launch()
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
            with native.on_device(logits):
                native.check(native.kernels().lyra_token_logprobs_bwd(ptr(logits), c_int(int(logits.dtype == torch.bfloat16)), ptr(grad), ptr(targets),
                                                                      ptr(norm), ptr(entropy), ptr(gl), ptr(gh), c_int(N), c_int(ctx.vocab), c_int(W),
                                                                      c_ll(logits.stride(0)), native.stream_ptr()), "lyra_token_logprobs_bwd")
            native.count_launch()
        return grad, None, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top_k: int, vocab: int) -> TokenLogprobs:
    """CUDA path; the arguments have passed :func:`check_arguments`. Rows may be strided, elements of a row may not."""
    if logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"logits must be fp32 or bf16 on a GPU, got {logits.dtype}")
    lead = logits.shape[:-1]
    rows = logits.reshape(-1, logits.shape[-1])
    if rows.shape[0] and (rows.stride(1) != 1 or rows.stride(0) < rows.shape[1]):
        rows = rows.contiguous()                              # transposed logits, or one row expanded to many
    with native.on_device(logits):
        out = _TokenLogprobs.apply(rows, targets.reshape(-1).long().contiguous(), top_k, vocab)
    return TokenLogprobs(*(t.reshape(*lead, *t.shape[1:]) for t in out))
