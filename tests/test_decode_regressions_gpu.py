"""Cached decoding and scores on the GPU: calls that once went wrong."""

import pytest
import torch
from torch.autograd import forward_ad

from nuvla_forge_b200 import _native as nat
from nuvla_forge_b200.models import NuVLA, NuVLAConfig
from nuvla_forge_b200.ops import logprobs as lp
from nuvla_forge_b200.ops import paged
from nuvla_forge_b200.serve import ReasoningDecoder

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _model(dtype, **over):
    torch.manual_seed(0)
    cfg = NuVLAConfig.preset("tiny", vocab_size=1000, n_instruction=8, n_reasoning=40, **over)
    model = NuVLA(cfg)
    with torch.no_grad():
        model.lm_head.mul_(10.0)
    model = model.to(DEV, dtype)
    images = torch.randint(0, 256, (4, cfg.n_images, 128, 128, 3), dtype=torch.uint8, device=DEV)
    return model, images, torch.randint(0, 1000, (4, 8), device=DEV)


def test_bad_targets_of_64_bit_logits_are_reported():
    x = torch.randn(4, 50, device=DEV, dtype=torch.float64, requires_grad=True)
    t = torch.tensor([3, -100, 50, 8], device=DEV)
    for logits, forced in ((x, False), (x.float(), True)):
        r = lp.token_logprobs(logits, t, top_k=2, force_reference=forced)
        assert r.logprobs[2].isnan() and r.logprobs[[0, 1, 3]].isfinite().all()
        assert torch.autograd.grad(r.logprobs[[0, 2, 3]].sum(), x)[0].isfinite().all()
        with pytest.raises(RuntimeError, match="outside the vocabulary"):
            lp.check_status()
    lp.check_status()


@pytest.mark.parametrize("graph", [False, True])
def test_two_streams_share_a_decoder_one_call_at_a_time(graph):
    model, images, text = _model(torch.bfloat16)
    texts = [text] + [torch.randint(0, 1000, (4, 8), device=DEV) for _ in range(3)]
    dec = ReasoningDecoder(model, 4, 8, max_new=12, graph=graph)
    want = [dec(images, t) for t in texts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, t in enumerate(texts):
        with torch.cuda.stream(streams[i % 2]):
            if i == 0:
                torch.cuda._sleep(20_000_000)         # the others are enqueued before the first one runs
            got.append(dec(images, t))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    paged.check_status()


def test_empty_calls_of_any_stride():
    kc, vc = (torch.zeros(2, 16, 2, 64, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    e = torch.zeros(0, dtype=torch.int32, device=DEV)
    q = torch.zeros(0, 1, 64, 4, device=DEV, dtype=torch.bfloat16).transpose(2, 3)
    assert paged.paged_attention(q, kc, vc, e.view(0, 1), e).shape == (0, 1, 4, 64)
    k = torch.zeros(0, 3, 64, 2, device=DEV, dtype=torch.bfloat16).transpose(2, 3)
    assert paged.append_kv(k, k, kc, vc, e.view(0, 1), e, q=k).shape == (0, 3, 2, 64)
    k = torch.zeros(2, 0, 64, 2, device=DEV, dtype=torch.bfloat16).transpose(2, 3)
    n = torch.zeros(2, dtype=torch.int32, device=DEV)
    assert paged.append_kv(k, k, kc, vc, n.view(2, 1), n, q=k).shape == (2, 0, 2, 64)
    paged.check_status()


def test_workspace_is_held_until_the_kernels_are_launched(monkeypatch):
    """Another thread that allocates on the same stream in the meantime must not be handed the call's workspace."""
    kc, vc = (torch.randn(100, 16, 4, 64, device=DEV).to(torch.bfloat16) for _ in range(2))
    table = torch.arange(100, dtype=torch.int32, device=DEV)[None]
    lengths = torch.tensor([1600], dtype=torch.int32, device=DEV)
    q = torch.randn(1, 1, 8, 64, device=DEV).to(torch.bfloat16)
    want = paged.paged_attention(q, kc, vc, table, lengths)
    call, seen = nat.call, []

    def between(name, *args):
        ws = args[7]
        assert name == "nfb_paged_attn" and ws is not None
        n = int(nat.lib().nfb_paged_attn_ws(1, 1, 8, 4, 64, 1600))
        other = [torch.empty(n, device=DEV) for _ in range(4)]       # of the workspace's size
        seen.append(all(not t.data_ptr() <= ws < t.data_ptr() + 4 * n for t in other))
        return call(name, *args)

    monkeypatch.setattr(nat, "call", between)
    got = paged.paged_attention(q, kc, vc, table, lengths)
    assert seen == [True] and torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nats", [10, 14, 18])
@pytest.mark.parametrize("B,hk,d,L", [(1, 1, 64, 768), (2, 4, 96, 700), (300, 8, 128, 8192)])
def test_a_tail_of_small_weights_keeps_its_share(dtype, nats, B, hk, d, L):
    """Four tokens with values of 0 (one for each warp) hold nearly all the mass; the output is what the tail
    gives. p = exp(-nats), at least 2^-26: relative to the output, a weight as two 16-bit parts is off by 2^-16
    (bf16) or 2^-20 + 2^-39 / p <= 2^-13 + 2^-20 (fp16), its exponential by 2^-22 and the score's three roundings
    by 3 * 18 * 2^-24 < 2^-18, the sums by 2^-23 for each of the L / 16 + 64 steps. The output is rounded once."""
    ps = 16
    pages = -(-L // ps)
    g = torch.Generator(DEV).manual_seed(nats + L)
    kc = torch.zeros(pages, ps, hk, d, device=DEV, dtype=dtype)
    kc[..., 0] = -nats                                # scores: exact, 0 for the four and -nats for the tail
    vc = (1 + torch.rand(pages, ps, hk, d, generator=g, device=DEV)).to(dtype)
    kc[:4, 5], vc[:4, 5] = 0, 0
    q = torch.zeros(B, 1, hk, d, device=DEV, dtype=dtype)
    q[..., 0] = 1
    table = torch.arange(pages, dtype=torch.int32, device=DEV).expand(B, pages)
    lengths = torch.full((B,), L, dtype=torch.int32, device=DEV)
    out = paged.paged_attention(q, kc, vc, table, lengths, scale=1.0)
    z = kc.flatten(0, 1)[:L, :, 0].double()
    want = torch.einsum("lh,lhd->hd", torch.softmax(z, 0), vc.flatten(0, 1)[:L].double())
    rel = 2.0 ** -13 + 2.0 ** -16 + 2.0 ** -18 + 2.0 ** -20 + (L / 16 + 64) * 2.0 ** -23 + torch.finfo(dtype).eps / 2
    # (fp16: outputs below 2^-14 are rounded to a multiple of 2^-24)
    assert ((out[:, 0].double() - want).abs() <= rel * want + (2.0 ** -25 if dtype == torch.float16 else 0)).all()
    paged.check_status()


def test_forward_mode_derivatives_are_refused():
    x, d = (torch.randn(3, 90, device=DEV) for _ in range(2))
    kc = torch.randn(4, 16, 2, 64, device=DEV)
    k, n = torch.randn(2, 1, 2, 64, device=DEV), torch.tensor([3, 4], dtype=torch.int32, device=DEV)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, d)
        with pytest.raises(RuntimeError, match="forward-mode"):
            lp.token_logprobs(dual)
        with pytest.raises(RuntimeError, match="forward-mode"), torch.no_grad():
            lp.token_logprobs(dual)
        assert forward_ad.unpack_dual(lp.token_logprobs(dual, force_reference=True).entropy).tangent is not None
        dk = forward_ad.make_dual(k, k)
        with pytest.raises(RuntimeError, match="forward-mode"):
            paged.paged_attention(dk, kc, kc, n.view(2, 1), n)
        with pytest.raises(RuntimeError, match="forward-mode"):
            paged.append_kv(dk, k, kc, kc.clone(), n.view(2, 1), n)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda z: lp.token_logprobs(z).entropy, (x,), (d,))


def test_unfused_decoding_is_a_reference_of_its_own(monkeypatch):
    """Plain operators decode, the kernels score what was decoded; fp32, tolerance as for the fused decoder."""
    model, images, text = _model(torch.float32, text_heads=4, text_kv_heads=2)
    plain = NuVLA(NuVLAConfig.preset("tiny", vocab_size=1000, n_instruction=8, n_reasoning=40, text_heads=4,
                                     text_kv_heads=2, fused=False)).to(DEV)
    plain.load_state_dict(model.state_dict())
    call, names = nat.call, set()
    monkeypatch.setattr(nat, "call", lambda name, *a: (names.add(name), call(name, *a))[1])
    dec = ReasoningDecoder(plain, 4, 8, max_new=8, top_k=3, page_size=16)
    a = dec(images, text)
    assert dec.graph is None and not names & {"nfb_append_kv", "nfb_paged_attn", "nfb_logprobs_fwd"}
    seq = torch.cat([text, a.tokens], 1)
    with torch.no_grad():
        s = model.score_text(images, seq[:, :-1], seq[:, 1:], top_k=3)
    assert "nfb_logprobs_fwd" in names
    assert (s.logprobs[:, 7:] - a.logprobs).abs().max() < 1e-2 and (s.entropy[:, 7:] - a.entropy).abs().max() < 1e-2


def test_check_status_waits_for_kernels_on_other_streams():
    kc = torch.zeros(2, 16, 2, 64, device=DEV, dtype=torch.bfloat16)
    table, n = torch.tensor([[5]], dtype=torch.int32, device=DEV), torch.tensor([3], dtype=torch.int32, device=DEV)
    q = torch.zeros(1, 1, 2, 64, device=DEV, dtype=torch.bfloat16)
    x, t = torch.zeros(2, 40, device=DEV), torch.tensor([3, 40], device=DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
        paged.paged_attention(q, kc, kc, table, n)    # a page id out of range: skipped and reported
        lp.token_logprobs(x, t)
    with pytest.raises(RuntimeError, match="out of range"):
        paged.check_status()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
        lp.token_logprobs(x, t)
    with pytest.raises(RuntimeError, match="outside the vocabulary"):
        lp.check_status()
    paged.check_status()


@pytest.fixture
def no_status_words():
    kept = {m: dict(m._status) for m in (paged, lp)}
    for m in kept:
        m._status.clear()
    yield
    for m, words in kept.items():
        m._status.clear()
        m._status.update(words)


def _small_calls():
    kc = torch.zeros(2, 16, 2, 64, device=DEV, dtype=torch.bfloat16)
    n = torch.tensor([3], dtype=torch.int32, device=DEV)
    q = torch.zeros(1, 1, 2, 64, device=DEV, dtype=torch.bfloat16)
    tables = [torch.tensor([[i]], dtype=torch.int32, device=DEV) for i in (0, 5)]
    x, targets = torch.zeros(2, 40, device=DEV), [torch.tensor([3, i], device=DEV) for i in (4, 40)]
    return [(lambda bad, t=t: paged.paged_attention(q, kc, kc, t[bad], n)) for t in (tables,)] + \
        [lambda bad: lp.token_logprobs(x, targets[bad])]


def test_a_first_call_in_a_capture_is_refused(no_status_words):
    for call, mod in zip(_small_calls(), (paged, lp)):
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="outside of the capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call(0)
        assert not mod._status
        call(0)                                       # outside of it, then in one
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(0)
        g.replay()
        mod.check_status()


def test_an_error_on_another_stream_outlives_the_first_calls_status_word(no_status_words):
    calls = _small_calls()
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for call, mod in zip(calls, (paged, lp)):
        with torch.cuda.stream(a):
            torch.cuda._sleep(50_000_000)
            call(0)
        with torch.cuda.stream(b):
            call(1)
        with pytest.raises(RuntimeError, match="out"):
            mod.check_status()


def test_a_wide_table_is_refused_only_by_the_kernel_that_would_run():
    """2^30 units of the tensor-core kernel, of 16 query heads each; the plain one counts 4 heads to a unit."""
    g = torch.Generator(DEV).manual_seed(3)
    kc, vc = (torch.randn(4, 16, 64, 64, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(1, 1, 1024, 64, generator=g, device=DEV).to(torch.bfloat16)
    table, n = torch.tensor([[2, 0, 3]], dtype=torch.int32, device=DEV), torch.tensor([40], dtype=torch.int32, device=DEV)
    wide = torch.zeros(1, 2 ** 24, dtype=torch.int32, device=DEV)
    wide[:, :3] = table
    want = paged.paged_attention(q, kc, vc, table, n)
    out = paged.paged_attention(q, kc, vc, wide, n)   # the same function; another division adds in another order
    assert torch.allclose(out.float(), want.float(), rtol=2 ** -7, atol=2 ** -9)
    odd = torch.zeros(q.numel() + 1, device=DEV, dtype=torch.bfloat16)[1:].view(q.shape)
    with pytest.raises(ValueError, match="16 bytes"):
        paged.paged_attention(odd, kc, vc, wide, n)
    with pytest.raises(ValueError, match="narrow the page table"):
        paged.paged_attention(q.float(), kc.float(), vc.float(), wide, n)
    paged.check_status()


def test_calls_without_query_heads():
    kc, n = torch.zeros(4, 16, 2, 64, device=DEV, dtype=torch.bfloat16), torch.tensor([3, 4], dtype=torch.int32, device=DEV)
    for dtype in (torch.bfloat16, torch.float32):
        c, q = kc.to(dtype), torch.zeros(2, 1, 0, 64, device=DEV, dtype=dtype)
        assert paged.paged_attention(q, c, c, n.view(2, 1) - 3, n).shape == (2, 1, 0, 64)
        k = torch.ones(2, 1, 2, 64, device=DEV, dtype=dtype)
        assert paged.append_kv(k, k, c, c.clone(), n.view(2, 1) - 3, n, q=q).shape == (2, 1, 0, 64)
        assert torch.equal(c[0, 3], k[0, 0]) and torch.equal(c[1, 4], k[1, 0])
    paged.check_status()
