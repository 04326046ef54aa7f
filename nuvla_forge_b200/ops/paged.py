"""Paged key-value cache: append with position rotation, and attention of one new token (native csrc/paged.cu).

``append_kv`` stores new keys and values where a page table says, rotating the keys (and the
queries, when given) by their position on the way; ``paged_attention`` attends one query per
sequence over its cached tokens. Together they are one decoding step of the backbone; the prompt
enters the cache with the same ``append_kv`` while ``ops.attention`` computes its outputs.

Layout: pools ``[n_pages, page_size, Hkv, D]`` for keys and values (the projection-native order of
``ops.attention``), ``page_table`` [B, W] int32 page ids, ``lengths`` [B] int32. Token p of sequence
b is in page ``page_table[b, p // page_size]``, slot ``p % page_size``; any page size works. Lengths
and page ids stay on the device: neither op waits for the host, both can be captured in a CUDA
graph (after a first call outside of one, which creates the device's status word; refused before),
and several streams can run them at once on caches of their own.

A position or page id out of range cannot be refused without reading it back: the kernels skip the
token and set a status word that ``check_status`` (and the trainer's health monitor) raises on. On
the CPU the reference raises IndexError. Neither op has a derivative.

The reference project has no decoding path.
"""

from __future__ import annotations

import torch

from .. import _native as nat
from .reference import append_kv_ref, paged_attention_ref

MAX_HEAD_DIM = 256

_status: dict[int, torch.Tensor] = {}


def _status_word(device: torch.device) -> torch.Tensor:
    return nat.status_word(_status, device)


def check_status(device: torch.device | None = None) -> None:
    """Raise (and clear it) if a kernel met a position, length or page id out of range on ``device``, or on any without
    one (waits for every stream of it)."""
    for idx, t in nat.status_of(_status, device):
        if t.is_cuda:
            torch.cuda.synchronize(t.device)
        v = int(t.item())
        if v:
            t.zero_()
            raise RuntimeError(f"paged cache on cuda:{idx}: a position, length or page id is out of range "
                               f"(status {v:#x}, site {v & 0xFFFFFF})")


def _check_cache(k_cache, v_cache, page_table, lengths, like, heads: int, dim: int, batch: int) -> None:
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError(f"k_cache and v_cache must both be [n_pages, page_size, Hkv, D], got "
                         f"{tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    if heads < 1 or dim < 1 or k_cache.shape[1] < 1 or k_cache.shape[2] != heads or k_cache.shape[3] != dim:
        raise ValueError(f"cache {tuple(k_cache.shape)} does not hold {heads} heads of {dim}")
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        raise ValueError("the cache's last dimension must be contiguous")
    if k_cache.dtype != like.dtype or v_cache.dtype != like.dtype:
        raise TypeError(f"cache dtypes {k_cache.dtype} and {v_cache.dtype} differ from the tokens' {like.dtype}")
    if page_table.dtype != torch.int32 or lengths.dtype != torch.int32:
        raise TypeError("page_table and lengths must be int32")
    if page_table.dim() != 2 or page_table.shape[0] != batch or lengths.shape != (batch,):
        raise ValueError(f"page_table must be [{batch}, W] and lengths [{batch}], got {tuple(page_table.shape)} "
                         f"and {tuple(lengths.shape)}")
    dev = like.device
    if not (k_cache.device == v_cache.device == page_table.device == lengths.device == dev):
        raise ValueError("all tensors must be on one device")


def _inner(t: torch.Tensor) -> torch.Tensor:
    return t if _rows_ok(t) else t.contiguous()


# What a call's shapes, strides, types and devices (never its addresses) decide: the checks, the array of
# sizes and strides, the workspace size. A decoding loop repeats them, and checking them anew took longer
# than the small kernels run.
_plans: dict[tuple, tuple] = {}
_MAX_PLANS = 4096


def _keep(key: tuple, plan: tuple) -> tuple:
    if len(_plans) >= _MAX_PLANS:
        _plans.clear()
    _plans[key] = plan
    return plan


def _sig(t: torch.Tensor) -> tuple:
    return t.shape, t.stride(), t.dtype, t.device


def _native(t: torch.Tensor) -> bool:
    return nat.HAS_NATIVE and t.is_cuda and t.dtype in nat.DT


def _rows_ok(*tensors) -> bool:
    """Whether the kernels read the tensors as they are: unit inner stride, or (``contiguous`` returns an empty
    tensor as it is) nothing to read."""
    return all(t is None or t.dim() == 0 or t.stride(-1) == 1 or t.shape[-1] <= 1 or t.numel() == 0 for t in tensors)


def _append_plan(key, k, v, k_cache, v_cache, page_table, lengths, counts, q, cos, sin, interleaved) -> tuple:
    if k.dim() != 4 or v.shape != k.shape:
        raise ValueError(f"k and v must both be [B, T, Hkv, D], got {tuple(k.shape)} and {tuple(v.shape)}")
    B, T, Hkv, D = k.shape
    _check_cache(k_cache, v_cache, page_table, lengths, k, Hkv, D, B)
    if v.dtype != k.dtype or v.device != k.device:
        raise TypeError("k and v must share dtype and device")
    if q is not None and (q.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != D or q.dtype != k.dtype
                          or q.device != k.device):
        raise ValueError(f"q must be [{B}, {T}, Hq, {D}] of {k.dtype} on {k.device}, got {tuple(q.shape)} {q.dtype}")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin must be given together")
    half = 0
    if cos is not None:
        half = cos.shape[-1]
        if cos.dim() != 2 or cos.shape != sin.shape or not 0 < 2 * half <= D or cos.shape[0] < 1:
            raise ValueError(f"cos and sin must be [positions, half] with 2 * half <= {D}, got {tuple(cos.shape)} "
                             f"and {tuple(sin.shape)}")
        if cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.device != k.device or sin.device != k.device:
            raise TypeError("cos and sin must be fp32 on the tokens' device")
    if counts is not None and (counts.dtype != torch.int32 or counts.shape != (B,) or counts.device != k.device):
        raise TypeError(f"counts must be [{B}] int32 on {k.device}")
    if any(n > 1 and s == 0 for c in (k_cache, v_cache) for n, s in zip(c.shape, c.stride())):
        raise ValueError("the cache must not be an expanded tensor: its slots would share memory")
    ready = _rows_ok(k, v, page_table, lengths, counts, q) and (
        cos is None or (cos.is_contiguous() and sin.is_contiguous()))
    dims = None
    if ready:
        Hq, qs = (q.shape[2], q.stride()[:3]) if q is not None else (0, (0, 0, 0))
        dims = nat.int64s(B, T, Hq, Hkv, D, half, int(interleaved), k_cache.shape[1], k_cache.shape[0],
                          page_table.shape[1], cos.shape[0] if half else 0, *qs, *k.stride()[:3], *v.stride()[:3],
                          *k_cache.stride()[:3], *v_cache.stride()[:3], page_table.stride(0))
    return _keep(key, (_native(k), dims))


def append_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              page_table: torch.Tensor, lengths: torch.Tensor, counts: torch.Tensor | None = None,
              q: torch.Tensor | None = None, cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
              interleaved: bool = False, force_reference: bool = False) -> torch.Tensor | None:
    """Store tokens k, v [B, T, Hkv, D] behind each sequence's ``lengths[b]`` cached tokens, in place.

    Token t of sequence b goes to position ``lengths[b] + t``; with ``counts`` [B] int32 only the
    first ``counts[b]`` of its T tokens are stored (a padded batch; 0 leaves the sequence as it is).
    With ``cos`` and ``sin`` ([positions, half] fp32, row p for position p) the first ``2 * half``
    values of each key head, and of each head of ``q`` [B, T, Hq, D], are rotated: value i with
    value half + i, or with ``interleaved`` neighbours (2i, 2i + 1); in fp32, rounded once.

    Returns q rotated (a new tensor; padding rows too, at most by the tables' last row), a copy of q
    without tables, or None without q. ``lengths`` is not changed. The slots that one call writes
    must be distinct.
    """
    key = (_sig(k), _sig(v), _sig(k_cache), _sig(v_cache), _sig(page_table), _sig(lengths),
           counts is not None and _sig(counts), q is not None and _sig(q), cos is not None and _sig(cos),
           sin is not None and _sig(sin), bool(interleaved))
    plan = _plans.get(key)
    if plan is None:
        plan = _append_plan(key, k, v, k_cache, v_cache, page_table, lengths, counts, q, cos, sin, interleaved)
    native, dims = plan
    if (k.requires_grad or v.requires_grad or k_cache.requires_grad or v_cache.requires_grad
            or (q is not None and q.requires_grad)
            or (cos is not None and (cos.requires_grad or sin.requires_grad))) and torch.is_grad_enabled():
        raise RuntimeError("append_kv has no backward pass: call it under torch.no_grad()")
    if nat.has_tangent(k, v, k_cache, v_cache, q, cos, sin):
        raise RuntimeError("append_kv has no forward-mode derivative")
    if force_reference or not native:
        out = append_kv_ref(k, v, k_cache, v_cache, page_table, lengths, counts, q, cos, sin, interleaved)
        return out.clone() if out is q and q is not None else out
    if dims is None:
        if cos is not None:
            cos, sin = cos.contiguous(), sin.contiguous()
        return append_kv(_inner(k), _inner(v), k_cache, v_cache, _inner(page_table), _inner(lengths),
                         None if counts is None else _inner(counts), None if q is None else _inner(q), cos, sin,
                         interleaved)
    out = None if q is None else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dev = k.device
    with nat.on_device(dev):
        nat.call("nfb_append_kv", nat.DT[k.dtype], nat.ptr(q), k.data_ptr(), v.data_ptr(), nat.ptr(out),
                 k_cache.data_ptr(), v_cache.data_ptr(), page_table.data_ptr(), lengths.data_ptr(),
                 nat.ptr(counts), nat.ptr(cos), nat.ptr(sin), dims, _status_word(dev).data_ptr(), nat.stream(dev))
    return out


def _attention_plan(key, q, k_cache, v_cache, page_table, lengths) -> tuple:
    if q.dim() != 4 or q.shape[1] != 1:
        raise ValueError(f"q must be [B, 1, Hq, D], got {tuple(q.shape)}")
    B, _, Hq, D = q.shape
    Hkv = k_cache.shape[2] if k_cache.dim() == 4 else 0
    _check_cache(k_cache, v_cache, page_table, lengths, q, Hkv, D, B)
    if Hkv < 1 or Hq % Hkv:
        raise ValueError(f"{Hkv} key heads do not divide {Hq} query heads")
    if not 0 < D <= MAX_HEAD_DIM:
        raise ValueError(f"head size {D} is not in 1..{MAX_HEAD_DIM}")
    native, dims, ws, aligned = _native(q), None, 0, False
    if native and _rows_ok(q, page_table, lengths):
        n_pages, ps = k_cache.shape[:2]
        W = page_table.shape[1]
        dims = nat.int64s(B, Hq, Hkv, D, ps, n_pages, W, q.stride(0), q.stride(2), Hq * D, D, *k_cache.stride()[:3],
                          *v_cache.stride()[:3], page_table.stride(0))
        # which kernel runs is left to the addresses where the rest allows the tensor-core one: room for either
        strides = (q.stride(0), q.stride(2), *k_cache.stride()[:3], *v_cache.stride()[:3])
        tiled = q.element_size() == 2 and D in (32, 64, 96, 128) and all(n % 8 == 0 for n in strides)
        plain, mma = (int(nat.lib().nfb_paged_attn_ws(kind, B, Hq, Hkv, D, ps * W)) if kind == 0 or tiled else -1
                      for kind in (0, 1))
        ws, aligned = max(plain, mma), plain < 0
        if ws < 0:
            raise ValueError(f"{B} sequences of up to {ps * W} tokens and {Hkv} key heads are more than the kernel's "
                             f"2^31 (sequence, head, 16-token tile) units: narrow the page table")
    return _keep(key, (native, dims, ws, aligned, D ** -0.5))


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    lengths: torch.Tensor, scale: float | None = None,
                    force_reference: bool = False) -> torch.Tensor:
    """softmax(scale q k^T) v of one query per sequence over its first ``lengths[b]`` cached tokens.

    q [B, 1, Hq, D] (grouped queries: Hkv divides Hq, D <= 256); returns [B, 1, Hq, D]. ``scale``
    defaults to D ** -0.5. A sequence of length 0 answers zeros; what the pages hold behind a
    sequence's length is never used. Statistics and sums are fp32, whatever the cache's type; of a weight
    p <= 1, 16 bits or more meet the values (fp16: all but 2^-20 p or 2^-39).
    """
    key = (_sig(q), _sig(k_cache), _sig(v_cache), _sig(page_table), _sig(lengths))
    plan = _plans.get(key)
    if plan is None:
        plan = _attention_plan(key, q, k_cache, v_cache, page_table, lengths)
    native, dims, n_ws, aligned, default = plan
    if (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad) and torch.is_grad_enabled():
        raise RuntimeError("paged_attention has no backward pass: call it under torch.no_grad()")
    if nat.has_tangent(q, k_cache, v_cache):
        raise RuntimeError("paged_attention has no forward-mode derivative")
    sc = default if scale is None else float(scale)
    if force_reference or not native:
        return paged_attention_ref(q, k_cache, v_cache, page_table, lengths, sc)
    if dims is None:
        return paged_attention(_inner(q), k_cache, v_cache, _inner(page_table), _inner(lengths), sc)
    if aligned and (q.data_ptr() | k_cache.data_ptr() | v_cache.data_ptr()) % 16:
        raise ValueError("a page table as wide as this one needs queries and caches that begin on 16 bytes")
    dev = q.device
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    # the caching allocator's memory, new for each call and held until its kernels are launched: calls on other
    # streams, in other threads and in other graphs have theirs
    ws = torch.empty(n_ws, dtype=torch.float32, device=dev) if n_ws else None
    with nat.on_device(dev):
        nat.call("nfb_paged_attn", nat.DT[q.dtype], q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                 page_table.data_ptr(), lengths.data_ptr(), out.data_ptr(), nat.ptr(ws), dims, sc,
                 _status_word(dev).data_ptr(), nat.stream(dev))
    return out


__all__ = ["MAX_HEAD_DIM", "append_kv", "check_status", "paged_attention"]
