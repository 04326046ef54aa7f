"""Cached decoding and scores on the CPU: calls that once went wrong."""

import contextlib
import subprocess
import sys
import threading
import time

import pytest
import torch
from torch.autograd import forward_ad

from nuvla_forge_b200 import _native as nat
from nuvla_forge_b200._build import lib_path
from nuvla_forge_b200.models import NuVLA, NuVLAConfig, layers
from nuvla_forge_b200.models.layers import PagedKVCache, run_blocks
from nuvla_forge_b200.ops import logprobs as lp
from nuvla_forge_b200.ops import paged
from nuvla_forge_b200.serve import ReasoningDecoder


# two fp32 evaluations of one small network (width 64, depth 2): a few hundred roundings of 2^-24 of
# values below 30
TOL = 300 * 30 * 2.0 ** -24


def _model(**over):
    torch.manual_seed(0)
    cfg = NuVLAConfig.preset("tiny", image_size=32, n_views=2, n_frames=1, vision_dim=64, vision_depth=1, vision_heads=2,
                             text_dim=64, text_depth=2, text_heads=4, text_kv_heads=2, text_ffn=128, dit_dim=64,
                             dit_depth=1, dit_heads=2, vocab_size=120, n_instruction=5, n_reasoning=9, **over)
    model = NuVLA(cfg)
    with torch.no_grad():
        model.lm_head.mul_(20.0)                      # clear winners among the tokens
    images = torch.randint(0, 256, (3, 2, 32, 32, 3), dtype=torch.uint8)
    text = torch.randint(0, 120, (3, 5))
    return model, images, text


def test_reference_scores_of_device_tensors_never_index_with_a_bad_target():
    """On a GPU torch's gather would abort the context; the same code runs here with its own status word."""
    torch.manual_seed(0)
    x = torch.randn(4, 9, dtype=torch.float64, requires_grad=True)
    good = lp.token_logprobs(x, torch.tensor([3, -100, 0, 8]), top_k=2)
    for bad in (9, -1, 2 ** 62, -2 ** 63):
        word = torch.zeros(1, dtype=torch.int32)
        given, entropy, top, ids = lp._reference_on_device(x, torch.tensor([3, -100, bad, 8]), 2, -100, word)
        assert int(word) == 3 << 24 | 1
        assert given[2].isnan() and torch.equal(given[[0, 1, 3]], good.logprobs[[0, 1, 3]])
        assert torch.equal(entropy, good.entropy) and torch.equal(top, good.top_logprobs) and torch.equal(ids, good.top_tokens)
        (dx,) = torch.autograd.grad(given.sum(), x)
        (want,) = torch.autograd.grad(good.logprobs[[0, 3]].sum(), x, retain_graph=True)
        assert torch.equal(dx, want)
    word = torch.zeros(1, dtype=torch.int32)
    given, *_ = lp._reference_on_device(x, torch.tensor([3, -100, 0, 8]), 2, -100, word)
    assert torch.equal(given, good.logprobs) and int(word) == 0
    assert lp._reference_on_device(x, None, 0, -100, word)[0] is None
    with pytest.raises(RuntimeError):
        lp.token_logprobs(x, torch.tensor([3, -100, 9, 8]))       # a CPU tensor: torch's own check


def test_two_threads_share_a_decoder_one_call_at_a_time(monkeypatch):
    """Calls in each other's buffers count positions past their end (on a GPU a device assert)."""
    model, images, text = _model()
    texts = [text, torch.randint(0, 120, (3, 5))]
    want = [ReasoningDecoder(model, 3, 5, max_new=4)(images, t) for t in texts]
    dec = ReasoningDecoder(model, 3, 5, max_new=4)
    busy, most, got, read = [0], [0], [None, None], model.read_prompt

    def slow(*args):
        busy[0] += 1
        most[0] = max(most[0], busy[0])
        time.sleep(0.2)
        h = read(*args)
        busy[0] -= 1
        return h

    monkeypatch.setattr(model, "read_prompt", slow)

    def call(i):
        got[i] = dec(images, texts[i])

    threads = [threading.Thread(target=call, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert most[0] == 1
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_empty_tensors_of_any_stride_are_read_as_they_are():
    """``contiguous`` leaves an empty tensor's strides, so asking it for unit ones never ended."""
    for t in (torch.zeros(0, 1, 64, 8).transpose(2, 3), torch.zeros(2, 8, 0, 4).permute(0, 2, 3, 1),
              torch.zeros(3, 0, dtype=torch.int32).T, torch.zeros(4, 6)[:, ::2], torch.zeros(4, 6).T[:, 1:3]):
        assert paged._rows_ok(paged._inner(t))


def test_forward_mode_derivatives_are_right_or_refused():
    torch.manual_seed(0)
    x, d = torch.randn(3, 9, dtype=torch.float64), torch.randn(3, 9, dtype=torch.float64)
    t = torch.tensor([1, 8, 0])
    k, kc = torch.randn(2, 1, 2, 8), torch.randn(4, 4, 2, 8)
    table, n = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32), torch.tensor([3, 4], dtype=torch.int32)
    with forward_ad.dual_level():
        r = lp.token_logprobs(forward_ad.make_dual(x, d), t)
        logp = torch.log_softmax(x, -1)
        want = d.gather(1, t[:, None])[:, 0] - (logp.exp() * d).sum(-1)
        assert (forward_ad.unpack_dual(r.logprobs).tangent - want).abs().max() < 1e-12
        dual = forward_ad.make_dual(k, torch.ones_like(k))
        for bad in (dict(k=dual, v=k), dict(k=k, v=dual), dict(k=k, v=k, q=dual)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                paged.append_kv(**bad, k_cache=kc.clone(), v_cache=kc.clone(), page_table=table, lengths=n)
        for q, c in ((dual, kc), (k, forward_ad.make_dual(kc, kc))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                paged.paged_attention(q, c, kc, table, n)
        paged.paged_attention(k, kc, kc, table, n)    # nothing dual among the arguments


def test_append_refuses_angles_that_require_a_gradient():
    k, kc = torch.randn(2, 1, 2, 8), torch.randn(4, 4, 2, 8)
    table, n = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32), torch.tensor([3, 4], dtype=torch.int32)
    one, learned = torch.ones(8, 4), torch.ones(8, 4, requires_grad=True)
    for cos, sin in ((learned, one), (one, learned)):
        with pytest.raises(RuntimeError, match="no_grad"):
            paged.append_kv(k, k, kc, kc.clone(), table, n, cos=cos, sin=sin)
        with torch.no_grad():
            paged.append_kv(k, k, kc, kc.clone(), table, n, cos=cos, sin=sin)


def test_states_behind_a_stop_token_are_those_of_the_returned_tokens():
    model, images, text = _model()
    free = ReasoningDecoder(model, 3, 5, max_new=7)(images, text)
    stop = int(free.tokens[1, 2])
    z0 = torch.randn(1, model.cfg.horizon, model.cfg.traj_dim)
    plans = []
    for max_new in (7, 9):
        a = ReasoningDecoder(model, 3, 5, max_new=max_new, stop_token=stop)(images, text)
        assert int(a.lengths[1]) <= 3
        with torch.no_grad():
            whole = model.context(images, torch.cat([text, a.tokens], 1))
            assert (a.states - whole).abs().max() < TOL
            one = model.context(images[1:2], torch.cat([text[1:2], a.tokens[1:2, : int(a.lengths[1])]], 1))
            assert a.context(1).shape == one.shape and (a.context(1) - one).abs().max() < TOL
            plans.append(model.dit.sample(a.context(1), steps=2, z0=z0))
    assert (plans[0] - plans[1]).abs().max() < TOL


def test_every_score_behind_a_stop_token_is_zero():
    model, images, text = _model()
    free = ReasoningDecoder(model, 3, 5, max_new=7, top_k=3)(images, text)
    stop = int(free.tokens[1, 2])
    a = ReasoningDecoder(model, 3, 5, max_new=7, top_k=3, stop_token=stop)(images, text)
    n = int(a.lengths[1])
    assert n < 7 and (a.top_tokens[1, n:] == stop).all()
    for x in (a.logprobs, a.entropy, a.top_logprobs):
        assert not x[1, n:].any() and x[1, :n].all()
    assert torch.equal(a.top_tokens[1, :n], free.top_tokens[1, :n])
    with torch.no_grad():
        model.text_norm.weight.fill_(float("nan"))    # scores that are NaN are not 0 times NaN behind the stop
    dec = ReasoningDecoder(model, 3, 5, max_new=3, stop_token=0)
    b = dec(images, text)
    for i in range(3):
        n = int(b.lengths[i])
        assert b.logprobs[i, :n].isnan().all() and not b.logprobs[i, n:].any()


@torch.no_grad()
def test_several_tokens_do_not_enter_a_cache_that_holds_some():
    """They would attend to one another alone; one at a time they see what is stored."""
    model, _, _ = _model()
    x = torch.randn(2, 6, 64)
    whole = run_blocks(model.text_blocks, x, model.text_norm)
    cache = PagedKVCache(2, 2, 8, 2, 16, page_size=4, dtype=torch.float32)

    def feed(t0, t1):
        cache.begin(t1 - t0)
        h = run_blocks(model.text_blocks, x[:, t0:t1], model.text_norm, cache=cache)
        cache.advance()
        return h

    for _ in range(2):
        first = feed(0, 4)
        with pytest.raises(ValueError, match="one at a time"):
            feed(4, 6)
        h = torch.cat([first, feed(4, 5), feed(5, 6)], 1)
        assert (h - whole).abs().max() < TOL
        cache.reset()


@pytest.mark.parametrize("fused", [False, True])
def test_decoding_honours_the_models_choice_of_kernels(fused, monkeypatch):
    model, images, text = _model(fused=fused)
    asked = []
    for name in ("append_kv", "paged_attention"):
        op = getattr(layers, name)
        monkeypatch.setattr(layers, name, lambda *a, op=op, **kw: (asked.append(kw["force_reference"]), op(*a, **kw))[1])
    ReasoningDecoder(model, 3, 5, max_new=2)(images, text)
    assert len(asked) >= 6 and all(f is not fused for f in asked)


@pytest.mark.parametrize("mod", [paged, lp])
def test_check_status_is_about_the_device_it_is_given(mod):
    bad = (3 << 24) | 1
    mod._status.update({97: torch.tensor([bad], dtype=torch.int32), 98: torch.tensor([bad], dtype=torch.int32)})
    try:
        mod.check_status(torch.device("cpu"))
        mod.check_status(torch.device("cuda", 96))
        with pytest.raises(RuntimeError, match="cuda:98"):
            mod.check_status(torch.device("cuda", 98))
        mod.check_status(torch.device("cuda", 98))    # raising cleared it
        with pytest.raises(RuntimeError, match="cuda:97"):
            mod.check_status()                        # the other device's is still there
        mod.check_status()
    finally:
        del mod._status[97], mod._status[98]


@pytest.mark.parametrize("mod", [paged, lp])
def test_a_status_word_made_under_inference_mode_can_be_cleared(mod):
    with torch.inference_mode():
        word = mod._status_word(torch.device("cpu", 99))
        word.fill_((3 << 24) | 1)
    try:
        assert not word.is_inference()
        with pytest.raises(RuntimeError, match="cuda:99"):
            mod.check_status()
        mod.check_status()
    finally:
        del mod._status[99]


def test_a_cache_counts_the_tokens_that_are_stored():
    """append_kv stores none for a negative count and all for one past the tokens."""
    c = PagedKVCache(1, 3, 10, 1, 4, page_size=3, dtype=torch.float32)
    c.begin(2, torch.tensor([5, -1, 1], dtype=torch.int32))
    c.layer(0).append(torch.ones(3, 2, 1, 4), torch.ones(3, 2, 1, 4))
    assert c.seen.tolist() == [2, 0, 1] and float(c.k[0].sum()) == 3 * 4
    c.advance()
    assert c.lengths.tolist() == [2, 0, 1]


def test_cache_refuses_sizes_that_it_cannot_hold():
    for bad in (dict(page_size=0), dict(page_size=-3), dict(max_len=0), dict(batch_size=0), dict(kv_heads=0)):
        with pytest.raises(ValueError, match="at least 1"):
            PagedKVCache(**{**dict(n_layers=1, batch_size=2, max_len=10, kv_heads=1, head_dim=4, page_size=3), **bad})
    model, images, text = _model()
    with pytest.raises(ValueError, match="at least 1"):
        ReasoningDecoder(model, 3, 5, max_new=2, page_size=0)
    cache = model.new_cache(3, 4, page_size=3)        # room in the last page behind max_len is not the cache's
    with pytest.raises(ValueError, match="do not fit"):
        model.read_prompt(images, text, cache)
    with pytest.raises(ValueError, match="do not fit"):
        cache.begin(5)


def test_a_call_runs_with_the_models_device_current(monkeypatch):
    """The GEMMs launch on the current device; the constructor's warm-up and capture had it set."""
    model, images, text = _model()
    dec = ReasoningDecoder(model, 3, 5, max_new=2)
    inside, seen, read = [], [], model.read_prompt

    @contextlib.contextmanager
    def on_device(device):
        inside.append(device)
        yield
        inside.pop()

    monkeypatch.setattr(nat, "on_device", on_device)
    monkeypatch.setattr(model, "read_prompt", lambda *a: (seen.append(list(inside)), read(*a))[1])
    dec(images, text)
    assert seen == [[model.lm_head.device]]


def test_a_decoder_built_under_inference_mode_answers_outside_of_it():
    model, images, text = _model()
    want = ReasoningDecoder(model, 3, 5, max_new=3)(images, text)
    with torch.inference_mode():
        dec = ReasoningDecoder(model, 3, 5, max_new=3)
        inside = dec(images, text)
    for a in (inside, dec(images, text)):
        assert all(torch.equal(x, y) for x, y in zip(a, want))


def test_a_workspace_of_no_heads_is_asked_for_without_a_division_by_zero():
    """In a process of its own: the division ended it."""
    if not lib_path().exists():
        pytest.skip("the native library is not built")
    code = f"import ctypes; f = ctypes.CDLL({str(lib_path())!r}).nfb_paged_attn_ws"
    code += """
from ctypes import c_int, c_int64 as L
f.restype, f.argtypes = L, [c_int] + [L] * 5
print([f(kind, *args) for kind in (0, 1) for args in ((2, 0, 1, 64, 100), (0, 4, 2, 64, 100))])
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and r.stdout.strip() == "[0, 0, 0, 0]", (r.returncode, r.stderr[-500:])
    kc, n = torch.randn(4, 4, 2, 8), torch.tensor([3, 4], dtype=torch.int32)
    assert paged.paged_attention(torch.zeros(2, 1, 0, 8), kc, kc, n.view(2, 1) % 4, n).shape == (2, 1, 0, 8)


def test_context_of_an_answer_counted_from_the_end():
    model, images, text = _model()
    a = ReasoningDecoder(model, 3, 5, max_new=3)(images, text)
    assert torch.equal(a.context(-1), a.context(2)) and a.context(-1).shape == (1, a.states.shape[1], 64)
    with pytest.raises(IndexError):
        a.context(3)
