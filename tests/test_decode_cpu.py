"""Answering with the reasoning head on the CPU: cache, decoder and scores against recomputation (fp32)."""

import pytest
import torch

from nuvla_forge_b200.models import NuVLA, NuVLAConfig
from nuvla_forge_b200.models.layers import PagedKVCache
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


@torch.no_grad()
def _by_recomputation(model, images, text, n):
    """Greedy tokens, log probabilities, entropies and states with the whole sequence run for every token."""
    out = []
    for _ in range(n):
        logp = torch.log_softmax(model.text_logits(model.context(images, text)[:, -1]).double(), -1)
        lp, tok = logp.max(-1)
        out.append((tok, lp, -(logp.exp() * logp).sum(-1)))
        text = torch.cat([text, tok[:, None]], 1)
    tok, lp, h = (torch.stack(x, 1) for x in zip(*out))
    return tok, lp, h, model.context(images, text)


@pytest.mark.parametrize("page_size", [1, 7, 64])
def test_decoder_matches_recomputation(page_size):
    model, images, text = _model()
    dec = ReasoningDecoder(model, 3, 5, max_new=6, top_k=4, page_size=page_size)
    tok, lp, h, states = _by_recomputation(model, images, text, 6)
    for _ in range(2):                                # the second call starts from an empty cache again
        a = dec(images, text)
        assert torch.equal(a.tokens, tok) and torch.equal(a.top_tokens[..., 0], tok)
        assert (a.logprobs.double() - lp).abs().max() < TOL and (a.entropy.double() - h).abs().max() < TOL
        assert a.states.shape == states.shape and (a.states - states).abs().max() < TOL
        assert a.top_logprobs.shape == (3, 6, 4) and (a.top_logprobs.diff(dim=-1) <= 0).all()
        assert a.lengths.tolist() == [6, 6, 6]
    images2 = torch.randint(0, 256, images.shape, dtype=torch.uint8)
    assert torch.equal(dec(images2, text).tokens, _by_recomputation(model, images2, text, 6)[0])
    # the answer's states condition the planner
    assert model.dit.sample(a.states, steps=2).shape == (3, model.cfg.horizon, 3)


def test_stop_token_ends_a_sequence_and_leaves_the_others():
    model, images, text = _model()
    free = ReasoningDecoder(model, 3, 5, max_new=7)(images, text)
    stop = int(free.tokens[1, 2])
    a = ReasoningDecoder(model, 3, 5, max_new=7, stop_token=stop)(images, text)
    for b in range(3):
        hits = (free.tokens[b] == stop).nonzero().flatten().tolist()
        n = hits[0] + 1 if hits else 7
        assert int(a.lengths[b]) == n
        assert torch.equal(a.tokens[b, :n], free.tokens[b, :n]) and (a.tokens[b, n:] == stop).all()
        assert (a.logprobs[b, :n] - free.logprobs[b, :n]).abs().max() < TOL and not a.logprobs[b, n:].any()


def test_scores_of_given_text_and_their_gradient():
    model, images, _ = _model()
    text, targets = torch.randint(0, 120, (3, 14)), torch.randint(0, 120, (3, 14))
    targets[0, :5] = -100
    r = model.score_text(images, text, targets, top_k=3)
    assert r.logprobs.shape == (3, 14) and r.top_tokens.shape == (3, 14, 3)
    loss = -r.logprobs.sum() / (targets != -100).sum()
    g1 = torch.autograd.grad(loss, (model.lm_head, model.text_embed.weight))
    ce = model(images, text_tokens=text, text_targets=targets)
    g2 = torch.autograd.grad(ce["loss"], (model.lm_head, model.text_embed.weight))
    assert abs(float(loss.detach()) - float(ce["reason_loss"])) < TOL
    for a, b in zip(g1, g2):
        assert (a - b).abs().max() < TOL
    # decoding scores its own tokens as this does
    a = ReasoningDecoder(model, 3, 5, max_new=9)(images, text[:, :5])
    seq = torch.cat([text[:, :5], a.tokens], 1)
    s = model.score_text(images, seq[:, :-1], seq[:, 1:])
    assert (s.logprobs[:, 4:] - a.logprobs).abs().max() < TOL and (s.entropy[:, 4:] - a.entropy).abs().max() < TOL


def test_refusals():
    model, images, text = _model()
    for kw in (dict(max_new=10), dict(max_new=0), dict(top_k=0), dict(top_k=33)):
        with pytest.raises(ValueError):
            ReasoningDecoder(model, 3, 5, **kw)
    dec = ReasoningDecoder(model, 3, 5, max_new=2)
    with pytest.raises(ValueError, match="instructions"):
        dec(images, text[:, :4])
    with pytest.raises(ValueError, match="instructions"):
        dec(images[:2], text[:2])
    ref = NuVLA(NuVLAConfig(image_size=32, vision_dim=64, vision_depth=1, vision_heads=2, fusion_depth=1, text_depth=1,
                            dit_depth=1, dit_heads=2, vocab_size=50))
    with pytest.raises(ValueError, match="causal backbone"):
        ReasoningDecoder(ref, 1, 4, max_new=2)
    with pytest.raises(ValueError, match="causal backbone"):
        ref.score_text(images, text, text)


def test_cache_grows_by_counts():
    c = PagedKVCache(1, 2, 10, 1, 4, page_size=3, dtype=torch.float32)
    assert c.k[0].shape == (8, 3, 1, 4)
    c.begin(3)
    c.layer(0).append(torch.ones(2, 3, 1, 4), torch.ones(2, 3, 1, 4))
    c.advance()
    c.begin(1, torch.tensor([1, 0], dtype=torch.int32))
    c.layer(0).append(torch.full((2, 1, 1, 4), 2.0), torch.full((2, 1, 1, 4), 2.0))
    c.advance()
    assert c.lengths.tolist() == [4, 3]
    assert float(c.k[0][1, 0, 0, 0]) == 2.0 and not c.k[0][5].any()
