"""Paged cache append and attention on the GPU against plain 64-bit implementations.

Tolerances. A stored or returned value is rounded once to its type: eps / 2 relative. A rotation in
fp32 is two products and a sum: at most 4 * 2^-24 of |a| + |b|. Attention: a score z = scale q.k in
fp32 is off by at most dz = (D + 4) 2^-24 scale sum |q k| plus one rounding of the scaled result, so a
weight by 2 dz relative; sums over L weights, their exponentials and weights kept as two 16-bit parts
(2^-16 for bf16) add (L + 64) 2^-24 + 2^-16 at most. All of it multiplies max |v|.
"""

import math

import pytest
import torch

from nuvla_forge_b200 import _native as nat
from nuvla_forge_b200.ops import append_kv, paged, paged_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def _pool(n_pages, ps, hk, d, dtype, g):
    return (torch.randn(n_pages, ps, hk, d, generator=g, device=DEV).to(dtype),
            torch.randn(n_pages, ps, hk, d, generator=g, device=DEV).to(dtype))


def _table(B, W, n_pages, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(n_pages, generator=g)[: B * W].reshape(B, W).to(DEV, torch.int32)


def _attend64(q, kc, vc, table, lengths, scale):
    """(out, max |v|, bound on the error of a score) per sequence and head, one sequence at a time."""
    B, _, H, D = q.shape
    ps, hk = kc.shape[1:3]
    out = torch.zeros(B, 1, H, D, dtype=torch.float64, device=q.device)
    vmax = torch.zeros(B, 1, H, 1, dtype=torch.float64, device=q.device)
    dz = torch.zeros_like(vmax)
    for b, n in enumerate(lengths.tolist()):
        if n == 0:
            continue
        pages = table[b, : -(-n // ps)].long()
        k = kc[pages].flatten(0, 1)[:n].double().repeat_interleave(H // hk, 1)
        v = vc[pages].flatten(0, 1)[:n].double().repeat_interleave(H // hk, 1)
        z = torch.einsum("hd,lhd->hl", q[b, 0].double(), k) * scale
        mag = torch.einsum("hd,lhd->hl", q[b, 0].double().abs(), k.abs()) * abs(scale)
        out[b, 0] = torch.einsum("hl,lhd->hd", torch.softmax(z, -1), v)
        vmax[b, 0, :, 0] = v.abs().amax((0, 2))
        dz[b, 0, :, 0] = mag.amax(-1) * (D + 4) * 2.0 ** -24 + z.abs().amax(-1) * 2.0 ** -23
    return out, vmax, dz


def _check_attention(out, q, kc, vc, table, lengths, scale=None):
    scale = scale if scale is not None else q.shape[-1] ** -0.5
    ref, vmax, dz = _attend64(q, kc, vc, table, lengths, scale)
    L = int(lengths.max()) if lengths.numel() else 0
    tol = torch.finfo(q.dtype).eps / 2 * ref.abs() + (2 * dz + (L + 64) * 2.0 ** -24 + 2.0 ** -16) * vmax
    if q.dtype == torch.float16:
        tol = tol + 2.0 ** -25                        # half a step of the subnormals
    bad = (out.double() - ref).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((out.double() - ref).abs() / (tol + 1e-30)).max()))
    assert torch.equal(out[lengths == 0], torch.zeros_like(out[lengths == 0]))
    paged.check_status()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hk,d", [(4, 4, 64), (16, 8, 128), (24, 8, 128), (6, 1, 96), (12, 4, 32), (16, 1, 128),
                                     (17, 1, 64), (40, 1, 128), (3, 3, 80), (2, 1, 256), (5, 5, 24), (2, 2, 1)])
def test_attention_head_layouts(dtype, hq, hk, d):
    g = _gen(hq * 1000 + d)
    kc, vc = _pool(40, 16, hk, d, dtype, g)
    table = _table(5, 7, 40, 1)
    lengths = torch.tensor([0, 1, 33, 112, 17], dtype=torch.int32, device=DEV)
    q = (torch.randn(5, 1, hq, d, generator=g, device=DEV) * 2).to(dtype)
    _check_attention(paged_attention(q, kc, vc, table, lengths), q, kc, vc, table, lengths)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ps", [1, 3, 16, 24, 48, 64, 1024])
def test_attention_page_sizes_and_lengths_around_their_ends(dtype, ps):
    g = _gen(ps)
    W = -(-200 // ps) + 1
    lengths = torch.tensor([1, 15, 16, 17, ps, ps + 1, max(ps - 1, 1), 31, 32, 47, 200, 0], device=DEV).clamp(max=W * ps)
    lengths = lengths.to(torch.int32)
    B = lengths.numel()
    n_pages = B * W + 2
    kc, vc = _pool(n_pages, ps, 2, 64, dtype, g)
    table = _table(B, W, n_pages, 2)
    # what no sequence may read: slots behind the lengths hold NaN and infinities
    for b, n in enumerate(lengths.tolist()):
        for w in range(W):
            lo = max(0, min(ps, n - w * ps))
            kc[int(table[b, w]), lo:] = float("nan")
            vc[int(table[b, w]), lo:] = float("inf")
    q = torch.randn(B, 1, 4, 64, generator=g, device=DEV).to(dtype)
    _check_attention(paged_attention(q, kc, vc, table, lengths), q, kc, vc, table, lengths)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,hq,hk,d,L", [(1, 16, 8, 128, 20011), (3, 8, 1, 64, 5000), (70, 4, 2, 64, 600),
                                         (300, 2, 1, 64, 40), (2, 6, 6, 96, 3392)])
def test_attention_long_and_many_sequences(dtype, B, hq, hk, d, L):
    g = _gen(B + L)
    ps = 64
    W = -(-L // ps)
    kc, vc = _pool(B * W + 1, ps, hk, d, dtype, g)
    table = _table(B, W, B * W + 1, 3)
    lengths = torch.randint(0, L + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
    lengths[0] = L
    q = torch.randn(B, 1, hq, d, generator=g, device=DEV).to(dtype)
    out = paged_attention(q, kc, vc, table, lengths)
    _check_attention(out, q, kc, vc, table, lengths)
    for _ in range(3):                                # the join adds in a fixed order
        assert torch.equal(out, paged_attention(q, kc, vc, table, lengths))


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64)])
@pytest.mark.parametrize("longest", [500, 8192, 70000])
def test_attention_many_sequences_and_a_few_long_ones(dtype, d, longest):
    """More (sequence, head) pairs than the GPU holds: each has a block for its first 8192 tokens, and what lies
    behind them is divided. Sequences share pages here (a table may name a page more than once)."""
    g = _gen(longest + d)
    B, ps, pages = 300, 64, 300
    kc, vc = _pool(pages, ps, 8, d, dtype, g)
    W = -(-longest // ps)
    table = torch.randint(0, pages, (B, W), generator=g, device=DEV, dtype=torch.int32)
    lengths = torch.randint(0, min(longest, 90), (B,), generator=g, device=DEV, dtype=torch.int32)
    for i, n in enumerate((longest, 8191, 8192, 8193, 8208, 8209, 12345, 0, 1, longest)):
        lengths[29 * i] = min(n, longest)
    q = torch.randn(B, 1, 16, d, generator=g, device=DEV).to(dtype)
    out = paged_attention(q, kc, vc, table, lengths)
    _check_attention(out, q, kc, vc, table, lengths)
    assert torch.equal(out, paged_attention(q, kc, vc, table, lengths))
    lengths.clamp_(max=5)                             # the same table, only short sequences
    _check_attention(paged_attention(q, kc, vc, table, lengths), q, kc, vc, table, lengths)


def test_attention_large_scores_and_custom_scale():
    """Scores of several hundred: the weights collapse to one token; a growing maximum rescales the sums."""
    g = _gen(5)
    kc, vc = _pool(20, 16, 2, 64, torch.bfloat16, g)
    kc *= torch.linspace(0.1, 12, 20, device=DEV).to(torch.bfloat16)[:, None, None, None]
    table = torch.arange(20, dtype=torch.int32, device=DEV)[None]
    lengths = torch.tensor([320], dtype=torch.int32, device=DEV)
    q = (torch.randn(1, 1, 4, 64, generator=g, device=DEV) * 4).to(torch.bfloat16)
    for scale in (None, 1.0, 0.0, -0.5):
        _check_attention(paged_attention(q, kc, vc, table, lengths, scale=scale), q, kc, vc, table, lengths, scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_infinite_and_nan_values_in_live_places(dtype):
    g = _gen(6)
    kc, vc = _pool(4, 16, 1, 64, dtype, g)
    table = torch.tensor([[2, 0], [1, 3]], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([20, 20], dtype=torch.int32, device=DEV)
    q = torch.rand(2, 1, 2, 64, generator=g, device=DEV).to(dtype) + 1
    kc[1] = kc[3] = -float("inf")                     # sequence 1: every score is -inf
    kc[2, 3] = -float("inf")                          # sequence 0: one token is masked by its key
    out = paged_attention(q, kc, vc, table, lengths)
    assert not out[1].any()
    live = [i for i in range(20) if i != 3]
    k = torch.cat([kc[2], kc[0]])[live, 0].double()
    v = torch.cat([vc[2], vc[0]])[live, 0].double()
    ref = torch.softmax(q[0, 0].double() @ k.T / 8, -1) @ v
    tol = torch.finfo(dtype).eps / 2 * ref.abs() + (64 * 80 * 2.0 ** -24 + 2.0 ** -16) * v.abs().max()
    assert ((out[0, 0].double() - ref).abs() <= tol).all()
    kc[2, 5, 0, 7] = float("nan")
    assert paged_attention(q, kc, vc, table, lengths)[0].isnan().all()


def test_attention_strided_inputs():
    """Queries cut from a fused projection, heads-first caches, a table cut from a wider one."""
    g = _gen(7)
    for dtype in (torch.bfloat16, torch.float32):
        k0, v0 = (torch.randn(30, 4, 32, 64, generator=g, device=DEV).to(dtype) for _ in range(2))  # heads first
        kc, vc = k0.transpose(1, 2), v0.transpose(1, 2)
        table = _table(3, 9, 30, 4)[:, 1:6]
        lengths = torch.tensor([160, 77, 5], dtype=torch.int32, device=DEV)
        q = torch.randn(3, 1, 16, 64, generator=g, device=DEV).to(dtype)[:, :, 4:12]
        _check_attention(paged_attention(q, kc, vc, table, lengths), q, kc, vc, table, lengths)
        odd = torch.randn(30 * 32 * 4 * 65 + 1, generator=g, device=DEV).to(dtype)[1:].view(30, 32, 4, 65)
        kc, vc = odd[..., :64], odd[..., 1:]          # rows that start anywhere
        _check_attention(paged_attention(q, kc, vc, table, lengths), q, kc, vc, table, lengths)
        qt = torch.randn(3, 1, 64, 8, generator=g, device=DEV).to(dtype).transpose(2, 3)
        _check_attention(paged_attention(qt, kc, vc, table, lengths), qt, kc, vc, table, lengths)


def test_attention_empty_calls():
    kc, vc = _pool(2, 16, 2, 64, torch.bfloat16, _gen(8))
    e = torch.zeros(0, dtype=torch.int32, device=DEV)
    out = paged_attention(torch.zeros(0, 1, 4, 64, device=DEV, dtype=torch.bfloat16), kc, vc, e.view(0, 1), e)
    assert out.shape == (0, 1, 4, 64)
    # no pages at all: only empty sequences
    q = torch.ones(2, 1, 4, 64, device=DEV, dtype=torch.bfloat16)
    z = torch.zeros(2, dtype=torch.int32, device=DEV)
    assert not paged_attention(q, kc, vc, z.view(2, 1)[:, :0], z).any()
    assert not paged_attention(q, kc[:0], vc[:0], z.view(2, 1), z).any()


def test_bad_lengths_and_pages_are_reported_and_skipped():
    """Every index is checked before it is used; the good sequence of the batch is answered all the same."""
    g = _gen(9)
    for dtype in (torch.bfloat16, torch.float32):
        kc, vc = _pool(6, 16, 2, 64, dtype, g)
        q = torch.randn(2, 1, 4, 64, generator=g, device=DEV).to(dtype)
        good = paged_attention(q[1:], kc, vc, torch.tensor([[1, 2]], dtype=torch.int32, device=DEV),
                               torch.tensor([30], dtype=torch.int32, device=DEV))
        for row, n in (([0, 6], 30), ([-1, 0], 30), ([2 ** 31 - 1, 0], 3), ([0, 3], 33), ([0, 3], -5), ([0, 3], 2 ** 31 - 1)):
            table = torch.tensor([row, [1, 2]], dtype=torch.int32, device=DEV)
            out = paged_attention(q, kc, vc, table, torch.tensor([n, 30], dtype=torch.int32, device=DEV))
            assert torch.allclose(out[1].float(), good[0].float(), rtol=2 ** -7, atol=2 ** -9)
            with pytest.raises(RuntimeError, match="out of range"):
                paged.check_status()
            paged.check_status()                      # raising clears it
        kb, vb = kc.clone(), vc.clone()
        k, v = (torch.randn(2, 2, 2, 64, generator=g, device=DEV).to(dtype) for _ in range(2))
        for row, n in (([6, 0], 3), ([-7, 0], 3), ([0, 3], 31), ([0, 3], -1), ([0, 3], 2 ** 31 - 1)):
            kc.copy_(kb), vc.copy_(vb)
            table = torch.tensor([row, [1, 2]], dtype=torch.int32, device=DEV)
            append_kv(k, v, kc, vc, table, torch.tensor([n, 8], dtype=torch.int32, device=DEV))
            assert torch.equal(kc[1, 8:10], k[1]) and torch.equal(vc[1, 8:10], v[1])
            with pytest.raises(RuntimeError, match="out of range"):
                paged.check_status()
        kc.copy_(kb)
        cos = torch.ones(9, 32, device=DEV)           # the table ends inside the sequence
        append_kv(k, v, kc, vc, table, torch.tensor([2, 8], dtype=torch.int32, device=DEV), cos=cos, sin=cos * 0)
        assert torch.equal(kc[1, 8], k[1, 0]) and torch.equal(kc[1, 9], kb[1, 9])
        with pytest.raises(RuntimeError, match="out of range"):
            paged.check_status()


# ------------------------------------------------------------------------------------------ append
def _append64(k, v, kc, vc, table, starts, counts, q, cos, sin, pairs):
    """(cache k, cache v, q) in 64 bits, one token at a time, and which slots were written."""
    ps = kc.shape[1]
    half = cos.shape[-1] if cos is not None else 0
    a = list(range(0, 2 * half, 2)) if pairs else list(range(half))
    b = [i + 1 for i in a] if pairs else list(range(half, 2 * half))

    def turn(x, p):
        x = x.double().clone()
        if half:
            c, s = cos[p].double(), sin[p].double()
            xa, xb = x[..., a], x[..., b]
            x[..., a], x[..., b] = xa * c - xb * s, xb * c + xa * s
        return x

    kd, vd, qd = kc.double(), vc.double(), None if q is None else q.double().clone()
    for i in range(k.shape[0]):
        for t in range(k.shape[1]):
            p = int(starts[i]) + t
            if q is not None:
                qd[i, t] = turn(q[i, t], min(p, cos.shape[0] - 1) if half else p)
            if counts is None or t < int(counts[i]):
                kd[table[i, p // ps], p % ps] = turn(k[i, t], p)
                vd[table[i, p // ps], p % ps] = v[i, t].double()
    return kd, vd, qd


def _check_append(dtype, B, T, hq, hk, d, ps, half, pairs, ragged, seed=0, view=True, with_q=True, odd=False):
    g = _gen(seed)
    pad = 1 if odd else 0
    qkv = torch.randn(B, T, hq + 2 * hk, d + pad, generator=g, device=DEV).to(dtype)[..., pad:]
    q, k, v = qkv.split([hq, hk, hk], dim=2)
    if not view:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    longest = 37 + T
    W = -(-longest // ps)
    kc, vc = _pool(B * W + 2, ps, hk, d, dtype, g)
    table = _table(B, W, B * W + 2, seed)
    starts = torch.randint(0, 38, (B,), generator=g, device=DEV, dtype=torch.int32)
    counts = torch.randint(0, T + 1, (B,), generator=g, device=DEV, dtype=torch.int32) if ragged else None
    cos = sin = None
    if half:
        ang = torch.rand(longest, half, generator=g, device=DEV) * 2 * math.pi
        cos, sin = ang.cos(), ang.sin()
    rk, rv, rq = _append64(k, v, kc, vc, table, starts, counts, q, cos, sin, pairs)
    before = kc.clone()
    out = append_kv(k, v, kc, vc, table, starts, counts, q=q if with_q else None, cos=cos, sin=sin, interleaved=pairs)
    paged.check_status()
    assert torch.equal(vc.double(), rv)
    still = rk == before.double()
    assert torch.equal(kc[still], before[still])      # slots that no token went to, and what is not rotated
    eps = torch.finfo(dtype).eps / 2
    # |a| + |b| of a pair is at most 12 here; a subnormal fp16 result is rounded by 2^-25
    tol = 12 * 4 * 2.0 ** -24 + 2.0 ** -25
    assert ((kc.double() - rk).abs() <= eps * rk.abs() + tol).all()
    if with_q:
        assert out.is_contiguous() and out.shape == q.shape
        assert ((out.double() - rq).abs() <= eps * rq.abs() + tol).all()
    else:
        assert out is None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,hq,hk,d,ps,half,pairs,ragged", [
    (1, 1, 4, 4, 64, 16, 32, False, False), (5, 1, 16, 8, 128, 64, 64, False, True),
    (3, 7, 16, 8, 128, 16, 32, True, True), (2, 33, 6, 1, 96, 24, 48, False, True),
    (2, 5, 3, 3, 80, 3, 20, True, False), (4, 3, 2, 2, 64, 1, 0, False, True),
    (2, 3, 2, 1, 24, 5, 8, False, False), (2, 3, 2, 1, 26, 5, 13, True, False), (1, 2, 1, 1, 2, 4, 1, False, False),
    (2, 4, 2, 1, 256, 16, 128, True, False), (1, 2, 2, 2, 7, 2, 3, False, False), (70, 2, 4, 2, 64, 16, 32, False, True),
    (2, 3, 5, 1, 320, 8, 16, False, False)])
def test_append(dtype, B, T, hq, hk, d, ps, half, pairs, ragged):
    _check_append(dtype, B, T, hq, hk, d, ps, half, pairs, ragged)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_layouts(dtype):
    _check_append(dtype, 3, 9, 4, 2, 64, 16, 32, False, True, seed=1, view=False)
    _check_append(dtype, 3, 9, 4, 2, 64, 16, 32, False, True, seed=2, with_q=False)
    _check_append(dtype, 3, 9, 4, 2, 64, 16, 32, True, True, seed=3, odd=True)       # rows that start anywhere
    _check_append(dtype, 3, 9, 4, 2, 64, 16, 0, False, True, seed=4)                 # no tables: q is copied


def test_append_padding_rows_and_empty_calls():
    g = _gen(11)
    kc, vc = _pool(4, 16, 2, 64, torch.bfloat16, g)
    k, v, q = (torch.randn(1, 6, 2, 64, generator=g, device=DEV).to(torch.bfloat16) for _ in range(3))
    table = torch.tensor([[3, 1]], dtype=torch.int32, device=DEV)
    # the padded rows lie behind the pages and behind the tables: nothing of them is an error
    cos = torch.ones(32, 32, device=DEV)
    starts, counts = (torch.tensor([n], dtype=torch.int32, device=DEV) for n in (30, 2))
    kb = kc.clone()
    out = append_kv(k, v, kc, vc, table, starts, counts, q=q, cos=cos, sin=cos * 0)
    paged.check_status()
    assert torch.equal(kc[1, 14:], k[0, :2]) and torch.equal(out, q)
    kb[1, 14:] = k[0, :2]
    assert torch.equal(kc, kb)
    assert append_kv(k[:, :0], v[:, :0], kc, vc, table, starts, q=q[:, :0]).shape == (1, 0, 2, 64)
    append_kv(k[:0], v[:0], kc, vc, table[:0], starts[:0])
    assert torch.equal(kc, kb)


def test_refusals_on_the_gpu():
    kc, vc = _pool(4, 16, 2, 64, torch.bfloat16, _gen(12))
    table = torch.tensor([[0, 1]], dtype=torch.int32, device=DEV)
    n = torch.tensor([3], dtype=torch.int32, device=DEV)
    k = torch.zeros(1, 1, 2, 64, device=DEV, dtype=torch.bfloat16)
    for bad in (dict(page_table=table.cpu()), dict(lengths=n.cpu()), dict(k_cache=kc.cpu(), v_cache=vc.cpu())):
        with pytest.raises(ValueError, match="one device"):
            append_kv(**{**dict(k=k, v=k, k_cache=kc, v_cache=vc, page_table=table, lengths=n), **bad})
        with pytest.raises(ValueError, match="one device"):
            paged_attention(**{**dict(q=k, k_cache=kc, v_cache=vc, page_table=table, lengths=n), **bad})
    with pytest.raises(RuntimeError, match="no_grad"):
        paged_attention(k.requires_grad_(True), kc, vc, table, n)
    wide = table[:, :1].expand(1, 2 ** 27)                   # a table (of one entry) for 2^31 tokens
    with pytest.raises(ValueError, match="narrow the page table"):
        paged_attention(torch.zeros(1, 1, 64, 64, device=DEV), torch.zeros(4, 16, 64, 64, device=DEV),
                        torch.zeros(4, 16, 64, 64, device=DEV), wide, n)


def test_mixed_calls_and_other_current_stream():
    """The same shapes with other strides, types and options use plans of their own."""
    g = _gen(16)
    for dtype in (torch.bfloat16, torch.float32, torch.bfloat16):
        for heads_first in (False, True):
            for pairs in (False, True):
                kc, vc = _pool(6, 16, 2, 64, dtype, g)
                if heads_first:
                    kc, vc = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (kc, vc))
                table = torch.tensor([[3, 1]], dtype=torch.int32, device=DEV)
                start = torch.tensor([13], dtype=torch.int32, device=DEV)
                k, v, q = (torch.randn(1, 1, h, 64, generator=g, device=DEV).to(dtype) for h in (2, 2, 4))
                ang = torch.rand(20, 32, generator=g, device=DEV) * 6
                rk, rv, rq = _append64(k, v, kc, vc, table, start, None, q, ang.cos(), ang.sin(), pairs)
                out = append_kv(k, v, kc, vc, table, start, q=q, cos=ang.cos(), sin=ang.sin(), interleaved=pairs)
                eps = torch.finfo(dtype).eps / 2
                for x, r in ((kc, rk), (vc, rv), (out, rq)):
                    assert ((x.double() - r).abs() <= eps * r.abs() + 48 * 2.0 ** -24).all()
                n = start + 1
                _check_attention(paged_attention(out, kc, vc, table, n), out, kc, vc, table, n)


def test_offsets_past_32_bits():
    """A pool of more than 2^31 values: the last page is written and read through 64-bit offsets."""
    pages = 2 ** 31 // (64 * 8 * 128) + 3
    kc = torch.zeros(pages, 64, 8, 128, device=DEV, dtype=torch.bfloat16)
    vc = torch.zeros_like(kc)
    g = _gen(13)
    k, v = (torch.randn(1, 40, 8, 128, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    table = torch.tensor([[pages - 1, 0]], dtype=torch.int32, device=DEV)
    zero, n = torch.zeros(1, dtype=torch.int32, device=DEV), torch.tensor([40], dtype=torch.int32, device=DEV)
    append_kv(k, v, kc, vc, table, zero)
    assert torch.equal(kc[-1, :40], k[0]) and torch.equal(vc[-1, :40], v[0])
    q = torch.randn(1, 1, 16, 128, generator=g, device=DEV).to(torch.bfloat16)
    _check_attention(paged_attention(q, kc, vc, table, n), q, kc, vc, table, n)


def test_two_streams_and_two_captured_graphs_at_once():
    """Calls on two streams, then two captured graphs replayed together, share no workspace."""
    g = _gen(14)
    sets = []
    for i in range(2):
        kc, vc = _pool(200, 16, 4, 128, torch.bfloat16, g)
        table = _table(2, 90, 200, i)
        lengths = torch.tensor([1440, 700 + i], dtype=torch.int32, device=DEV)
        q = torch.randn(2, 1, 8, 128, generator=g, device=DEV).to(torch.bfloat16)
        sets.append((q, kc, vc, table, lengths))
    want = [paged_attention(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged_attention(*sets[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])
    graphs, outs = [], []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(paged_attention(*sets[i]))
        graphs.append(gr)
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(outs[i], want[i]) for i in range(2))
    sets[0][4].copy_(torch.tensor([3, 0], dtype=torch.int32))     # a replay follows the lengths on the device
    graphs[0].replay()
    torch.cuda.synchronize()
    _check_attention(outs[0], *sets[0])


def test_native_kernels_run():
    kc, vc = _pool(4, 16, 2, 64, torch.bfloat16, _gen(15))
    t = torch.tensor([[0, 1]], dtype=torch.int32, device=DEV)
    n = torch.tensor([3], dtype=torch.int32, device=DEV)
    x = torch.zeros(1, 1, 2, 64, device=DEV, dtype=torch.bfloat16)
    nat.reset_launch_count()
    append_kv(x, x, kc, vc, t, n)
    paged_attention(x, kc, vc, t, n)
    assert nat.launch_count() == 2
