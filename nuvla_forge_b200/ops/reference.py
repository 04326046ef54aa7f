"""Pure-PyTorch reference implementations (test oracle and CPU fallback).

Every native kernel in :mod:`nuvla_forge_b200.ops` has an fp32-computing
reference here. Parity: nuvla_forge/kernels/reference.py:22-96 (same functions
and signatures for the three fused ops), plus references for the ops the
reference left to PyTorch (attention, RMSNorm, image normalisation, patchify).
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

IMAGENET_MEAN = (0.485, 0.456, 0.406)
IMAGENET_STD = (0.229, 0.224, 0.225)


def _per_row(c: torch.Tensor, tokens_per_sample: int) -> torch.Tensor:
    """[B, N] per-sample vector -> [B*T, N], row m taking sample m // T."""
    return torch.repeat_interleave(c, tokens_per_sample, dim=0)


def adaln_residual_rmsnorm_ref(x, y, gate, weight, scale, shift, tokens_per_sample: int, eps: float = 1e-6):
    """h = x + gate*y; out = rmsnorm(h) * weight * (1 + scale) + shift.

    x, y: [M, N]; gate, scale, shift: [B, N] with M = B * tokens_per_sample;
    weight: [N]. Returns (h, out) in x's dtype.
    """
    g = _per_row(gate, tokens_per_sample).to(torch.float32)
    s = _per_row(scale, tokens_per_sample).to(torch.float32)
    sh = _per_row(shift, tokens_per_sample).to(torch.float32)
    h = (x.to(torch.float32) + g * y.to(torch.float32)).to(x.dtype)
    hf = h.to(torch.float32)
    inv = torch.rsqrt(hf.square().mean(dim=-1, keepdim=True) + eps)
    out = hf * inv * weight.to(torch.float32) * (1.0 + s) + sh
    return h, out.to(x.dtype)


def rmsnorm_ref(x, weight, eps: float = 1e-6):
    xf = x.to(torch.float32)
    inv = torch.rsqrt(xf.square().mean(dim=-1, keepdim=True) + eps)
    return (xf * inv * weight.to(torch.float32)).to(x.dtype)


def add_rmsnorm_ref(x, y, weight, eps: float = 1e-6):
    """h = x + y; out = rmsnorm(h) * weight. Returns (h, out)."""
    h = (x.to(torch.float32) + y.to(torch.float32)).to(x.dtype)
    return h, rmsnorm_ref(h, weight, eps)


def swiglu_ref(a, b):
    """silu(a) * b computed in fp32, returned in a's dtype."""
    return (F.silu(a.to(torch.float32)) * b.to(torch.float32)).to(a.dtype)


def chunked_cross_entropy_ref(hidden, lm_weight, targets, ignore_index: int = -100):
    """Unchunked mean cross entropy over hidden @ lm_weight.T, in fp32."""
    logits = hidden.to(torch.float32) @ lm_weight.to(torch.float32).t()
    return F.cross_entropy(logits, targets, ignore_index=ignore_index, reduction="mean")


def attention_ref(q, k, v, causal: bool = False, scale: float | None = None):
    """Softmax attention in fp32. q [B, Hq, S, D], k/v [B, Hkv, L, D] (GQA when Hkv < Hq)."""
    hq, hkv = q.shape[1], k.shape[1]
    if hkv != hq:
        rep = hq // hkv
        k = k.repeat_interleave(rep, dim=1)
        v = v.repeat_interleave(rep, dim=1)
    qf, kf, vf = (t.to(torch.float32) for t in (q, k, v))
    sc = scale if scale is not None else 1.0 / math.sqrt(q.shape[-1])
    s = torch.einsum("bhsd,bhld->bhsl", qf, kf) * sc
    if causal:
        S, L = s.shape[-2], s.shape[-1]
        mask = torch.ones(S, L, dtype=torch.bool, device=s.device).tril(L - S)
        s = s.masked_fill(~mask, float("-inf"))
    p = torch.softmax(s, dim=-1)
    return torch.einsum("bhsl,bhld->bhsd", p, vf).to(q.dtype)


def _cache_slots(page_table, positions, n_pages: int, page_size: int):
    """(page, slot) of each position [B, T]; raises on a position or page id out of range."""
    if positions.numel() and (int(positions.min()) < 0 or int(positions.max()) >= page_table.shape[1] * page_size):
        raise IndexError("a position lies outside the pages of its sequence")
    page = page_table.long().gather(1, positions // page_size)
    if page.numel() and (int(page.min()) < 0 or int(page.max()) >= n_pages):
        raise IndexError("a page id lies outside the cache")
    return page, positions % page_size


def rotate_ref(x, cos, sin, interleaved: bool = False):
    """Rotates the first 2 * half values of each head of x [B, T, H, D] by cos / sin [B, T, half], in fp32."""
    half = cos.shape[-1]
    xf = x.to(torch.float32)
    c, s = cos[:, :, None], sin[:, :, None]
    if interleaved:
        a, b = xf[..., 0:2 * half:2], xf[..., 1:2 * half:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    else:
        a, b = xf[..., :half], xf[..., half:2 * half]
        turned = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    return torch.cat([turned.to(x.dtype), x[..., 2 * half:]], dim=-1)


def append_kv_ref(k, v, k_cache, v_cache, page_table, lengths, counts=None, q=None, cos=None, sin=None,
                  interleaved: bool = False):
    """Stores the rotated keys and the values of tokens t < counts[b] at positions lengths[b] + t; returns rotated q."""
    B, T = k.shape[:2]
    t = torch.arange(T, device=k.device)
    pos = lengths.long()[:, None] + t
    live = t < counts[:, None] if counts is not None else torch.ones_like(pos, dtype=torch.bool)
    if cos is not None:
        if bool(((pos < 0) | (pos >= cos.shape[0]))[live].any()):
            raise IndexError("a position lies outside the cos / sin tables")
        at = pos.clamp(0, max(cos.shape[0] - 1, 0))
        k = rotate_ref(k, cos[at], sin[at], interleaved)
        q = rotate_ref(q, cos[at], sin[at], interleaved) if q is not None else None
    rows = torch.arange(B, device=k.device)[:, None].expand(B, T)[live]
    page, slot = _cache_slots(page_table[rows], pos[live][:, None], k_cache.shape[0], k_cache.shape[1])
    k_cache[page[:, 0], slot[:, 0]] = k[live]
    v_cache[page[:, 0], slot[:, 0]] = v[live]
    return q


def paged_attention_ref(q, k_cache, v_cache, page_table, lengths, scale: float | None = None):
    """Softmax attention in fp32 of q [B, 1, Hq, D] over each sequence's first lengths[b] cached tokens."""
    B, _, hq, d = q.shape
    n_pages, ps, hkv, _ = k_cache.shape
    out = torch.zeros((B, 1, hq, d), dtype=q.dtype, device=q.device)
    for b, n in enumerate(lengths.tolist()):
        if n < 0:
            raise IndexError("a length is negative")
        if n == 0:
            continue
        page, slot = _cache_slots(page_table[b:b + 1], torch.arange(n, device=q.device)[None], n_pages, ps)
        # attention_ref leaves a row of -inf scores as NaN; a query no key is left for answers 0
        k, v = (c[page, slot].transpose(1, 2) for c in (k_cache, v_cache))
        o = attention_ref(q[b:b + 1].transpose(1, 2), k, v, scale=scale)
        kf = k.to(torch.float32).repeat_interleave(hq // hkv, dim=1)
        sc = scale if scale is not None else 1.0 / math.sqrt(d)
        s = torch.einsum("bhsd,bhld->bhsl", q[b:b + 1].transpose(1, 2).to(torch.float32), kf) * sc
        o = torch.where((s == float("-inf")).all(dim=-1, keepdim=True), torch.zeros_like(o), o)
        out[b:b + 1] = o.transpose(1, 2)
    return out


def token_logprobs_ref(logits, targets=None, top_k: int = 0, ignore_index: int = -100):
    """(log p of the targets or None, entropy, top log p or None, top ids or None) of logits [M, V], in fp32
    (fp64 logits: in fp64). A row without a finite logit: log p -inf, entropy 0, no gradient."""
    x = logits if logits.dtype == torch.float64 else logits.to(torch.float32)
    dead = (x == float("-inf")).all(dim=-1, keepdim=True)
    logp = torch.log_softmax(torch.where(dead, torch.zeros_like(x), x), dim=-1)
    p = logp.exp()
    entropy = -(p * torch.where(p > 0, logp, torch.zeros_like(logp))).sum(dim=-1)
    entropy = torch.where(dead[:, 0], torch.zeros_like(entropy), entropy)
    none = torch.full((), float("-inf"), dtype=x.dtype, device=x.device)
    given = top = ids = None
    if targets is not None:
        keep = targets != ignore_index
        lp = logp.gather(1, torch.where(keep, targets, torch.zeros_like(targets))[:, None])
        given = torch.where(keep, torch.where(dead, none, lp)[:, 0], torch.zeros_like(entropy))
    if top_k:
        ids = torch.sort(x.detach(), dim=-1, descending=True, stable=True)[1][:, :top_k].contiguous()
        top = torch.where(dead, none, logp.gather(1, ids))
    return given, entropy, top, ids


def normalise_images_ref(images, dtype=torch.bfloat16, mean=IMAGENET_MEAN, std=IMAGENET_STD):
    """uint8 [..., 3, H, W] -> (v/255 - mean[c]) / std[c] in ``dtype``."""
    x = images.to(torch.float32) / 255.0
    m = torch.tensor(mean, dtype=torch.float32, device=x.device).view(3, 1, 1)
    s = torch.tensor(std, dtype=torch.float32, device=x.device).view(3, 1, 1)
    return ((x - m) / s).to(dtype)


def patchify_ref(images_hwc, patch: int, kpad: int | None = None, dtype=torch.bfloat16,
                 mean=IMAGENET_MEAN, std=IMAGENET_STD):
    """uint8 [n, H, W, 3] -> normalised patch rows [n, (H/p)*(W/p), kpad] in (c, ky, kx) order."""
    n, H, W, _ = images_hwc.shape
    p = patch
    x = images_hwc.to(torch.float32) / 255.0
    m = torch.tensor(mean, dtype=torch.float32, device=x.device)
    s = torch.tensor(std, dtype=torch.float32, device=x.device)
    x = (x - m) / s                                        # [n, H, W, 3]
    x = x.view(n, H // p, p, W // p, p, 3).permute(0, 1, 3, 5, 2, 4)  # [n, hp, wp, 3, p, p]
    x = x.reshape(n, (H // p) * (W // p), 3 * p * p)
    k = 3 * p * p
    if kpad is not None and kpad > k:
        x = F.pad(x, (0, kpad - k))
    return x.to(dtype)
