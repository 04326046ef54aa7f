"""Paged cache and token scores on the CPU: the references against their definitions, and every refusal."""

import math

import pytest
import torch

from nuvla_forge_b200.ops import append_kv, paged_attention, token_logprobs


def _cache(n_pages=6, ps=4, hk=2, d=8, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n_pages, ps, hk, d, generator=g).to(dtype), torch.randn(n_pages, ps, hk, d, generator=g).to(dtype))


def _append_args(B=2, T=3, hk=2, d=8, dtype=torch.float32):
    k, v = torch.randn(B, T, hk, d).to(dtype), torch.randn(B, T, hk, d).to(dtype)
    kc, vc = _cache(hk=hk, d=d, dtype=dtype)
    table = torch.tensor([[4, 1], [0, 3]], dtype=torch.int32)[:B]
    lengths = torch.tensor([2, 5], dtype=torch.int32)[:B]
    return dict(k=k, v=v, k_cache=kc, v_cache=vc, page_table=table, lengths=lengths)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("half", [0, 2, 4])
def test_append_writes_each_token_where_its_table_says(interleaved, half):
    torch.manual_seed(1)
    a = _append_args()
    counts = torch.tensor([3, 2], dtype=torch.int32)
    q = torch.randn(2, 3, 4, 8)
    ang = torch.arange(8, dtype=torch.float64)[:, None] * (0.3 + torch.arange(half, dtype=torch.float64))
    cos, sin = (ang.cos().float(), ang.sin().float()) if half else (None, None)
    want_k, want_v, want_q = a["k_cache"].double(), a["v_cache"].double(), q.double().clone()

    def turn(x, p):  # complex rotation, pair by pair
        x = x.double().clone()
        for i in range(half):
            ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, half + i)
            z = torch.complex(x[..., ia], x[..., ib]) * torch.polar(torch.ones(()).double(), ang[p, i])
            x[..., ia], x[..., ib] = z.real, z.imag
        return x

    for b in range(2):
        for t in range(3):
            p = int(a["lengths"][b]) + t
            want_q[b, t] = turn(q[b, t], p)
            if t < counts[b]:
                page, slot = int(a["page_table"][b, p // 4]), p % 4
                want_k[page, slot] = turn(a["k"][b, t], p)
                want_v[page, slot] = a["v"][b, t].double()
    out = append_kv(**a, counts=counts, q=q, cos=cos, sin=sin, interleaved=interleaved)
    # a pair's fp32 turn: two products and a sum, each rounded, of values below 8, and the table's rounding
    tol = 8 * 4 * 2.0 ** -24
    assert (out.double() - want_q).abs().max() <= tol
    assert (a["k_cache"].double() - want_k).abs().max() <= tol
    assert torch.equal(a["v_cache"].double(), want_v)
    assert out.data_ptr() != q.data_ptr()


def test_append_without_queries_returns_none_and_zero_counts_change_nothing():
    a = _append_args()
    before = a["k_cache"].clone(), a["v_cache"].clone()
    assert append_kv(**a, counts=torch.zeros(2, dtype=torch.int32)) is None
    assert torch.equal(a["k_cache"], before[0]) and torch.equal(a["v_cache"], before[1])


def test_append_refusals():
    a = _append_args()
    ok = torch.ones(8, 4)
    bad = [
        (ValueError, dict(k=a["k"][0])),
        (ValueError, dict(v=a["v"][:, :2])),
        (ValueError, dict(k=a["k"][:, :, :0], v=a["v"][:, :, :0], k_cache=a["k_cache"][:, :, :0], v_cache=a["v_cache"][:, :, :0])),
        (ValueError, dict(k_cache=a["k_cache"][..., :4], v_cache=a["v_cache"][..., :4])),
        (ValueError, dict(k_cache=a["k_cache"][0])),
        (ValueError, dict(k_cache=a["k_cache"].transpose(2, 3).contiguous().transpose(2, 3))),
        (ValueError, dict(k_cache=a["k_cache"][:1].expand(6, -1, -1, -1))),
        (TypeError, dict(k_cache=a["k_cache"].bfloat16(), v_cache=a["v_cache"].bfloat16())),
        (TypeError, dict(page_table=a["page_table"].long())),
        (TypeError, dict(lengths=a["lengths"].long())),
        (ValueError, dict(lengths=a["lengths"][:1])),
        (ValueError, dict(page_table=a["page_table"][:1])),
        (TypeError, dict(counts=torch.tensor([1, 1]))),
        (TypeError, dict(counts=torch.tensor([1], dtype=torch.int32))),
        (ValueError, dict(q=torch.randn(2, 3, 4, 4))),
        (ValueError, dict(q=torch.randn(2, 2, 4, 8))),
        (ValueError, dict(cos=ok)),
        (ValueError, dict(cos=ok, sin=ok[:4])),
        (ValueError, dict(cos=torch.ones(8, 5), sin=torch.ones(8, 5))),
        (ValueError, dict(cos=torch.ones(0, 4), sin=torch.ones(0, 4))),
        (TypeError, dict(cos=ok.double(), sin=ok.double())),
        (RuntimeError, dict(k=a["k"].clone().requires_grad_(True))),
        (IndexError, dict(lengths=torch.tensor([2, 6], dtype=torch.int32))),
        (IndexError, dict(lengths=torch.tensor([-1, 5], dtype=torch.int32))),
        (IndexError, dict(page_table=torch.tensor([[4, 6], [0, 3]], dtype=torch.int32))),
        (IndexError, dict(page_table=torch.tensor([[-4, 1], [0, 3]], dtype=torch.int32))),
        (IndexError, dict(cos=torch.ones(7, 4), sin=torch.ones(7, 4))),
    ]
    for err, change in bad:
        with pytest.raises(err):
            append_kv(**{**a, **change})


@pytest.mark.parametrize("hq,hk", [(4, 4), (6, 2), (5, 1)])
def test_paged_attention_reference_against_64_bits(hq, hk):
    torch.manual_seed(2)
    kc, vc = _cache(n_pages=9, ps=3, hk=hk)
    kc[7], vc[7] = float("nan"), float("inf")            # a page no sequence has
    table = torch.tensor([[4, 1, 8], [0, 3, 7], [2, 5, 6]], dtype=torch.int32)
    lengths = torch.tensor([9, 6, 0], dtype=torch.int32)
    q = torch.randn(3, 1, hq, 8)
    out = paged_attention(q, kc, vc, table, lengths)
    for b in range(3):
        for h in range(hq):
            if lengths[b] == 0:
                assert torch.equal(out[b, 0, h], torch.zeros(8))
                continue
            pos = range(int(lengths[b]))
            K = torch.stack([kc[table[b, p // 3], p % 3, h // (hq // hk)].double() for p in pos])
            V = torch.stack([vc[table[b, p // 3], p % 3, h // (hq // hk)].double() for p in pos])
            w = torch.softmax(K @ q[b, 0, h].double() / math.sqrt(8), dim=0)
            # 9 fp32 terms of values below 4: 64 roundings in all cover scores, exponentials and sums
            assert (out[b, 0, h].double() - w @ V).abs().max() <= 64 * 4 * 2.0 ** -24


def test_paged_attention_refusals():
    kc, vc = _cache()
    table, lengths = torch.tensor([[4, 1]], dtype=torch.int32), torch.tensor([5], dtype=torch.int32)
    base = dict(q=torch.randn(1, 1, 4, 8), k_cache=kc, v_cache=vc, page_table=table, lengths=lengths)
    bad = [
        (ValueError, dict(q=torch.randn(1, 2, 4, 8))),
        (ValueError, dict(q=torch.randn(1, 4, 8))),
        (ValueError, dict(q=torch.randn(1, 1, 3, 8))),
        (ValueError, dict(q=torch.randn(1, 1, 4, 4))),
        (ValueError, dict(q=torch.randn(2, 1, 4, 8))),
        (ValueError, dict(q=torch.randn(1, 1, 4, 0), k_cache=kc[..., :0], v_cache=vc[..., :0])),
        (ValueError, dict(k_cache=kc[:, :, :0], v_cache=vc[:, :, :0])),
        (ValueError, dict(v_cache=vc[:5])),
        (ValueError, dict(k_cache=kc[0])),
        (TypeError, dict(k_cache=kc.half(), v_cache=vc.half())),
        (TypeError, dict(lengths=lengths.long())),
        (TypeError, dict(page_table=table.long())),
        (RuntimeError, dict(q=torch.randn(1, 1, 4, 8, requires_grad=True))),
        (IndexError, dict(lengths=torch.tensor([9], dtype=torch.int32))),
        (IndexError, dict(lengths=torch.tensor([-1], dtype=torch.int32))),
        (IndexError, dict(page_table=torch.tensor([[6, 1]], dtype=torch.int32))),
    ]
    for err, change in bad:
        with pytest.raises(err):
            paged_attention(**{**base, **change})
    wide = torch.zeros(2, 4, 1, 264)
    with pytest.raises(ValueError, match="256"):
        paged_attention(torch.zeros(1, 1, 1, 264), wide, wide, table, lengths)


def test_token_logprobs_reference_values_ties_and_masks():
    x = torch.tensor([[1.0, 3.0, 3.0, -float("inf"), 0.0],
                      [-float("inf")] * 5,
                      [0.0, -0.0, 0.0, -1.0, 0.0]])
    t = torch.tensor([2, 1, -100])
    r = token_logprobs(x, t, top_k=3)
    p = torch.softmax(x[0].double(), 0)
    assert abs(float(r.logprobs[0]) - float(p[2].log())) < 1e-6
    assert abs(float(r.entropy[0]) + float((p[p > 0] * p[p > 0].log()).sum())) < 1e-6
    assert r.top_tokens.tolist() == [[1, 2, 0], [0, 1, 2], [0, 1, 2]]
    assert float(r.logprobs[1]) == -float("inf") and float(r.entropy[1]) == 0.0
    assert float(r.logprobs[2]) == 0.0
    one = token_logprobs(torch.zeros(2, 1), torch.zeros(2, dtype=torch.int64), top_k=1)
    assert one.logprobs.tolist() == [0.0, 0.0] and one.entropy.tolist() == [0.0, 0.0]
    lead = token_logprobs(torch.randn(2, 3, 7), torch.zeros(2, 3, dtype=torch.int64), top_k=2)
    assert lead.logprobs.shape == (2, 3) and lead.top_tokens.shape == (2, 3, 2)
    bare = token_logprobs(torch.randn(7))
    assert bare.logprobs is None and bare.top_tokens is None and bare.entropy.shape == ()


def test_token_logprobs_reference_gradient_against_differences():
    torch.manual_seed(3)
    x = torch.randn(4, 9, dtype=torch.float64)
    x[0, 3] = -float("inf")
    x[2] = -float("inf")
    t = torch.tensor([1, -100, 4, 8])
    g1, g2, g3 = torch.randn(4).double(), torch.randn(4).double(), torch.randn(4, 3).double()

    def f(z):
        r = token_logprobs(z, t, top_k=3)
        live = torch.tensor([0, 1, 3])
        return sum(((a * g)[live]).sum() for a, g in ((r.logprobs, g1), (r.entropy, g2), (r.top_logprobs, g3)))

    z = x.clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(f(z), z)
    assert torch.isfinite(grad).all() and float(grad[0, 3]) == 0.0 and not grad[2].any()
    for _ in range(4):
        d = torch.randn_like(x)
        h = 1e-5
        num = float(f(x + h * d) - f(x - h * d)) / (2 * h)
        assert abs(num - float((grad * d).sum())) < 1e-8    # the error of central differences, h^2 f''' / 6


def test_token_logprobs_refusals():
    x, t = torch.randn(3, 9), torch.zeros(3, dtype=torch.int64)
    for err, args, kw in [
        (ValueError, (x, t), dict(top_k=10)),
        (ValueError, (x, t), dict(top_k=-1)),
        (ValueError, (torch.randn(3, 64), t), dict(top_k=33)),
        (ValueError, (x, t[:2]), {}),
        (TypeError, (x, t.int()), {}),
        (TypeError, (x.long(), t), {}),
        (ValueError, (torch.randn(3, 0), t), {}),
        (RuntimeError, (x, t + 9), {}),                     # torch's index check
        (RuntimeError, (x, t - 1), {}),
    ]:
        with pytest.raises(err):
            token_logprobs(*args, **kw)


def test_status_words_of_the_new_ops_reach_the_health_monitor():
    from nuvla_forge_b200.health import DeviceFault, HealthMonitor
    from nuvla_forge_b200.ops import logprobs, paged

    for mod, name in ((paged, "paged_cache"), (logprobs, "logprobs")):
        mod._status[97] = torch.tensor([(3 << 24) | 1], dtype=torch.int32)
        try:
            with pytest.raises(DeviceFault, match=f"{name}@cuda:97: bad argument at site 1"):
                HealthMonitor(torch.device("cpu")).check_now()
            with pytest.raises(RuntimeError, match="cuda:97"):
                mod.check_status()
        finally:
            del mod._status[97]
