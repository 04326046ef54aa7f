"""Log probabilities of given tokens, entropy and the most likely tokens (native csrc/logprobs.cu).

``token_logprobs`` reads materialised logits once and returns what scoring, serving and fine-tuning
on scores need; unlike ``chunked_cross_entropy``, which keeps only a mean loss, it keeps each token's
value and is differentiable in all of them. Sums are fp32 whatever the logits' type; the gradient is
computed in fp32 and rounded once to it.

The reference project has only the mean cross entropy.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from .. import _native as nat
from .reference import token_logprobs_ref

MAX_TOP_K = 32
_BAD_TARGET = 3 << 24 | 1  # the kernel's status: code 3 (bad argument), site 1

_status: dict[int, torch.Tensor] = {}


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor | None       # [...] fp32 log p of the targets (0 where ignored)
    entropy: torch.Tensor               # [...] fp32, in nats
    top_logprobs: torch.Tensor | None   # [..., top_k] fp32, descending
    top_tokens: torch.Tensor | None     # [..., top_k] int64


def _status_word(device: torch.device) -> torch.Tensor:
    return nat.status_word(_status, device)


def check_status(device: torch.device | None = None) -> None:
    """Raise (and clear it) if a kernel met a target outside the vocabulary on ``device``, or on any without
    one (waits for every stream of it)."""
    for idx, t in nat.status_of(_status, device):
        if t.is_cuda:
            torch.cuda.synchronize(t.device)
        v = int(t.item())
        if v:
            t.zero_()
            raise RuntimeError(f"token_logprobs on cuda:{idx}: a target is outside the vocabulary (status {v:#x})")


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, targets, top_k, ignore_index):
        M, V = x.shape
        dev = x.device
        f32 = torch.float32
        logprobs = torch.empty(M, dtype=f32, device=dev) if targets is not None else None
        entropy = torch.empty(M, dtype=f32, device=dev)
        stats = torch.empty((M, 2), dtype=f32, device=dev) if ctx is not None else None  # for the backward pass
        top = torch.empty((M, top_k), dtype=f32, device=dev) if top_k else None
        ids = torch.empty((M, top_k), dtype=torch.int64, device=dev) if top_k else None
        with nat.on_device(dev):
            nat.call("nfb_logprobs_fwd", nat.DT[x.dtype], x.data_ptr(), x.stride(0), M, V, nat.ptr(targets),
                     ignore_index, top_k, nat.ptr(logprobs), entropy.data_ptr(), nat.ptr(stats), nat.ptr(top),
                     nat.ptr(ids), _status_word(dev).data_ptr(), nat.stream(dev))
        if ctx is not None:
            ctx.set_materialize_grads(False)
            ctx.save_for_backward(x, targets, stats, entropy, ids)
            ctx.top_k, ctx.ignore_index = top_k, ignore_index
            if ids is not None:
                ctx.mark_non_differentiable(ids)
        return logprobs, entropy, top, ids

    @staticmethod
    def backward(ctx, g_logprobs, g_entropy, g_top, _):
        # (the wrapper for double differentiation only where a graph of the gradient is wanted: it costs
        # as much host time as the launch)
        if torch.is_grad_enabled():
            return _first_order(ctx, g_logprobs, g_entropy, g_top)
        return _TokenLogprobs._gradient(ctx, g_logprobs, g_entropy, g_top)

    @staticmethod
    def _gradient(ctx, g_logprobs, g_entropy, g_top):
        x, targets, stats, entropy, ids = ctx.saved_tensors
        if g_logprobs is None and g_entropy is None and g_top is None:
            return None, None, None, None
        M, V = x.shape
        g_logprobs, g_entropy, g_top = (None if g is None else g.contiguous() for g in (g_logprobs, g_entropy, g_top))
        dev = x.device
        dx = torch.empty((M, V), dtype=x.dtype, device=dev)
        with nat.on_device(dev):
            nat.call("nfb_logprobs_bwd", nat.DT[x.dtype], x.data_ptr(), x.stride(0), M, V, nat.ptr(targets),
                     ctx.ignore_index, ctx.top_k, nat.ptr(ids), nat.ptr(g_logprobs), nat.ptr(g_entropy),
                     nat.ptr(g_top), stats.data_ptr(), entropy.data_ptr(), dx.data_ptr(), nat.stream(dev))
        return dx, None, None, None


def _reference_on_device(x, targets, top_k, ignore_index, word):
    """The reference without its index check: a target outside the vocabulary (torch's gather would abort the
    process's GPU context) gives NaN, no gradient, and the status that the kernel sets in ``word``."""
    if targets is None:
        return token_logprobs_ref(x, None, top_k, ignore_index)
    bad = (targets != ignore_index) & ((targets < 0) | (targets >= x.shape[1]))
    given, *rest = token_logprobs_ref(x, targets.masked_fill(bad, ignore_index), top_k, ignore_index)
    word.copy_(torch.where(bad.any(), torch.full_like(word, _BAD_TARGET), word))
    return given.masked_fill(bad, float("nan")), *rest


# gradients of the gradient raise instead of being silently zero
_first_order = once_differentiable(_TokenLogprobs._gradient)


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor | None = None, top_k: int = 0,
                   ignore_index: int = -100, force_reference: bool = False) -> TokenLogprobs:
    """log p of ``targets`` [...] int64 under ``logits`` [..., V], the entropy of each row and its ``top_k``
    (at most 32) most likely tokens, equal logits in the order of their index.

    Gradients flow from ``logprobs``, ``entropy`` and ``top_logprobs`` to ``logits``. A target equal to
    ``ignore_index`` has log p 0 and no gradient; its row's entropy and alternatives are computed all the
    same. A masked logit is -inf; a row of nothing else has log p -inf, entropy 0 and no gradient. A row
    with a NaN or +inf logit gives NaN (and unspecified alternatives). A target outside the vocabulary
    gives NaN and is reported by ``check_status`` (on the CPU it raises). Nothing waits for the host; a call
    can be captured in a CUDA graph after a first one outside of it (refused before), its backward pass only while no
    eager autograd graph of the same leaves is alive (torch ties their gradients to that graph's stream).
    Rows may begin anywhere; the backward pass is about four times faster where their distance is V plus a multiple
    of 16 bytes (a vocabulary of V padded to V + 8 16-bit logits rather than to V + 3). Only the reference has
    forward-mode derivatives.
    """
    if logits.dim() < 1 or not logits.is_floating_point():
        raise TypeError(f"logits must be a floating-point tensor [..., V], got {tuple(logits.shape)} {logits.dtype}")
    V = logits.shape[-1]
    lead = logits.shape[:-1]
    if not 0 <= top_k <= min(MAX_TOP_K, V):
        raise ValueError(f"top_k {top_k} is not in 0..{min(MAX_TOP_K, V)}")
    if V < 1:
        raise ValueError("the vocabulary is empty")
    if targets is not None:
        if targets.dtype != torch.int64:
            raise TypeError(f"targets must be int64, got {targets.dtype}")
        if targets.shape != lead or targets.device != logits.device:
            raise ValueError(f"targets must be {tuple(lead)} on {logits.device}, got {tuple(targets.shape)} on "
                             f"{targets.device}")
    top_k, ignore_index = int(top_k), int(ignore_index)
    flat = len(lead) == 1
    x = logits if flat else logits.reshape(-1, V)
    t = targets if flat or targets is None else targets.reshape(-1)
    if force_reference or not (nat.HAS_NATIVE and x.is_cuda and x.dtype in nat.DT):
        r = _reference_on_device(x, t, top_k, ignore_index, _status_word(x.device)) if x.is_cuda else \
            token_logprobs_ref(x, t, top_k, ignore_index)
    else:
        if nat.has_tangent(x):
            raise RuntimeError("token_logprobs has no forward-mode derivative on a GPU: use force_reference")
        if x.stride(1) != 1 and V > 1:
            x = x.contiguous()
        t = None if t is None else t.contiguous()
        if x.requires_grad and torch.is_grad_enabled():
            r = _TokenLogprobs.apply(x, t, top_k, ignore_index)
        else:
            r = _TokenLogprobs.forward(None, x, t, top_k, ignore_index)
    if flat:
        return TokenLogprobs(*r)
    lp, h, top, ids = r
    return TokenLogprobs(None if lp is None else lp.view(lead), h.view(lead),
                         None if top is None else top.view(*lead, top_k),
                         None if ids is None else ids.view(*lead, top_k))


__all__ = ["MAX_TOP_K", "TokenLogprobs", "check_status", "token_logprobs"]
