"""Answering on the GPU: prompt, cached steps in a graph, scores and gradient together."""

import pytest
import torch

from nuvla_forge_b200 import _native as nat
from nuvla_forge_b200.models import NuVLA, NuVLAConfig
from nuvla_forge_b200.ops import paged
from nuvla_forge_b200.serve import GraphedPlanner, ReasoningDecoder

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


def test_fp32_decoding_matches_scoring_of_its_own_tokens():
    """Cached decoding and one pass over the whole sequence are the same function; in fp32 (depth 4, width 256,
    a few thousand roundings of 2^-24 of values below 30) they agree to 1e-2 of a nat, where a wrong page or
    mask moves a log probability by whole nats."""
    model, images, text = _model(torch.float32, text_heads=4, text_kv_heads=2)
    for graph in (False, True):
        dec = ReasoningDecoder(model, 4, 8, max_new=24, top_k=3, page_size=16, graph=graph)
        a = dec(images, text)
        dec.check_status()
        seq = torch.cat([text, a.tokens], 1)
        with torch.no_grad():
            s = model.score_text(images, seq[:, :-1], seq[:, 1:], top_k=3)
        assert (s.logprobs[:, 7:] - a.logprobs).abs().max() < 1e-2
        assert (s.entropy[:, 7:] - a.entropy).abs().max() < 1e-2
        with torch.no_grad():
            assert (model.context(images, seq) - a.states).abs().max() < 1e-2


def test_bf16_graph_replays_what_runs_eagerly():
    model, images, text = _model(torch.bfloat16)
    eager = ReasoningDecoder(model, 4, 8, max_new=40, graph=False)(images, text)
    dec = ReasoningDecoder(model, 4, 8, max_new=40)
    planner = GraphedPlanner(model, 4, dec.n_prompt + 40, steps=2)
    for _ in range(2):
        nat.reset_launch_count()
        a = dec(images, text)
        assert nat.launch_count() > 0
        for x, y in zip(a, eager):
            assert torch.equal(x, y)
        assert planner(a.states).shape == (4, 8, 3)
    dec.check_status()
    paged.check_status()
    text2 = torch.randint(0, 1000, (4, 8), device=DEV)
    eager2 = ReasoningDecoder(model, 4, 8, max_new=40, graph=False)(images, text2)
    assert torch.equal(dec(images, text2).tokens, eager2.tokens)
    stop = int(eager.tokens[0, 5])
    for graph in (False, True):
        b = ReasoningDecoder(model, 4, 8, max_new=40, stop_token=stop, graph=graph)(images, text)
        n = int((eager.tokens[0] == stop).nonzero()[0]) + 1
        assert int(b.lengths[0]) == n and torch.equal(b.tokens[0, :n], eager.tokens[0, :n])
        assert (b.tokens[0, n:] == stop).all()


def test_training_on_scores_runs_native_kernels():
    """A step on log probabilities and entropy through the native op: every parameter of the text path gets a
    finite gradient."""
    model, images, _ = _model(torch.bfloat16)
    text, targets = (torch.randint(0, 1000, (4, 48), device=DEV) for _ in range(2))
    w = torch.randn(4, 48, device=DEV)
    r = model.score_text(images, text, targets)
    ((r.logprobs * w).sum() - 0.01 * r.entropy.sum()).backward()
    for name, p in model.named_parameters():
        if name.startswith(("text_", "lm_head", "encoder", "vision_proj")):
            assert p.grad is not None and p.grad.isfinite().all(), name
    assert model.lm_head.grad.abs().max() > 0
