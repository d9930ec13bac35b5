"""Scoring tokens: the log probabilities of given tokens under a row of logits,
the distribution's entropy and its top alternatives, with the gradient that a
policy update or a distillation needs (csrc/scoring.cu, through the C ABI).

The training loss (trunk.cross_entropy_sum) gives one sum; an answer's tokens are
scored one by one, and a policy-gradient step weighs each token's gradient.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib

MAX_TOP = 32


class TokenLogprobs(NamedTuple):
    """logprob, entropy (R) fp32; top_idx (R, k) int64 and top_logprob (R, k) fp32,
    or None without alternatives."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_idx: Optional[torch.Tensor]
    top_logprob: Optional[torch.Tensor]


def _forward(logits, targets, top_k, temperature, ignore_index, want_stats):
    R, V = logits.shape
    dev = logits.device
    logprob = torch.empty(R, dtype=torch.float32, device=dev)
    entropy = torch.empty(R, dtype=torch.float32, device=dev)
    top_lp = torch.empty(R, top_k, dtype=torch.float32, device=dev) if top_k else None
    top_idx = torch.empty(R, top_k, dtype=torch.int64, device=dev) if top_k else None
    stats = torch.empty(R, 4, dtype=torch.float32, device=dev) if want_stats else None
    _lib.call_on(dev.index, "mom_logprobs_fwd", logits.data_ptr(), _code(logits), logits.stride(0) if R > 1 else V,
                 targets.data_ptr(), R, V, ignore_index, temperature, top_k, logprob.data_ptr(), entropy.data_ptr(),
                 top_lp.data_ptr() if top_k else None, top_idx.data_ptr() if top_k else None,
                 stats.data_ptr() if want_stats else None)
    return logprob, entropy, top_lp, top_idx, stats


def _code(t):
    return _lib.BF16 if t.dtype == torch.bfloat16 else _lib.F32


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top_k, temperature, ignore_index):
        logprob, entropy, top_lp, top_idx, stats = _forward(logits, targets, top_k, temperature, ignore_index, True)
        ctx.save_for_backward(logits, targets, stats, top_idx)
        ctx.meta = (top_k, temperature, ignore_index)
        ctx.set_materialize_grads(False)
        if top_k:
            ctx.mark_non_differentiable(top_idx)
            return logprob, entropy, top_lp, top_idx
        return logprob, entropy

    @staticmethod
    def backward(ctx, g_logprob, g_entropy, g_top=None, _g_idx=None):
        if torch.is_grad_enabled():
            raise RuntimeError("token_logprobs: its gradient has no gradient (create_graph=True)")
        logits, targets, stats, top_idx = ctx.saved_tensors
        top_k, temperature, ignore_index = ctx.meta
        R, V = logits.shape
        if g_logprob is None and g_entropy is None and g_top is None:
            return None, None, None, None, None
        g = [None if t is None else t.to(torch.float32).contiguous() for t in (g_logprob, g_entropy, g_top)]
        dlogits = torch.empty(R, V, dtype=logits.dtype, device=logits.device)
        _lib.call_on(logits.device.index, "mom_logprobs_bwd", logits.data_ptr(), _code(logits),
                     logits.stride(0) if R > 1 else V, targets.data_ptr(), stats.data_ptr(),
                     top_idx.data_ptr() if top_k else None, top_k, *(None if t is None else t.data_ptr() for t in g), R,
                     V, ignore_index, temperature, dlogits.data_ptr())
        return dlogits, None, None, None, None


def token_logprobs(logits, targets, *, top_k: int = 0, temperature: float = 1.0, ignore_index: int = -100):
    """Log probabilities of targets (R) under softmax(logits / temperature), logits
    (R, V) bf16 or fp32 (rows may be strided), with each row's entropy and, for
    top_k > 0 (at most 32), its top_k greatest logits in order: ties to the lowest
    index, NaN above all. A row whose target is ignore_index has logprob 0 (and no
    gradient from it); a target outside [0, V) gives a logprob of NaN. A logit of -inf
    has probability 0, a finite mask what its softmax gives; a row with a NaN or +inf,
    or of nothing but -inf, gives NaN.
    Sums are fp32 whatever the logits' dtype; the gradient has the logits' dtype.
    Differentiable in logprob, entropy and top_logprob. Returns TokenLogprobs."""
    if not logits.is_cuda or logits.dtype not in (torch.bfloat16, torch.float32):
        raise RuntimeError(f"token_logprobs takes bf16 or fp32 CUDA logits, got {logits.dtype} on {logits.device}")
    if forward_ad._current_level >= 0:
        _lib.no_tangent("token_logprobs", logits)
    shape = logits.shape
    if len(shape) != 2 or shape[1] == 0 or targets.shape != shape[:1] or targets.device != logits.device or \
            targets.dtype.is_floating_point:
        raise RuntimeError(f"token_logprobs: logits (R, V) and integer targets (R,) on one device, got "
                           f"{tuple(shape)} and {tuple(targets.shape)} {targets.dtype}")
    R, V = shape
    top_k, temperature = int(top_k), float(temperature)
    if not 0 <= top_k <= min(MAX_TOP, V):
        raise RuntimeError(f"token_logprobs: top_k {top_k} must be in [0, {min(MAX_TOP, V)}]")
    if not 1e-6 <= temperature <= 1e6:
        raise RuntimeError(f"token_logprobs: temperature {temperature} must be in [1e-6, 1e6]")
    if not logits.is_contiguous() and (V > 1 and logits.stride(1) != 1 or R > 1 and logits.stride(0) < V):
        logits = logits.contiguous()
    if targets.dtype != torch.int64 or not targets.is_contiguous():
        targets = targets.to(torch.int64).contiguous()
    if logits.requires_grad and torch.is_grad_enabled():
        out = _TokenLogprobs.apply(logits, targets, top_k, temperature, int(ignore_index))
        return TokenLogprobs(out[0], out[1], *((out[3], out[2]) if top_k else (None, None)))
    logprob, entropy, top_lp, top_idx, _ = _forward(logits, targets, top_k, temperature, int(ignore_index), False)
    return TokenLogprobs(logprob, entropy, top_idx, top_lp)


__all__ = ["MAX_TOP", "TokenLogprobs", "token_logprobs"]
