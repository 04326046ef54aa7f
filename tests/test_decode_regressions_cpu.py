"""Cached decoding and scores on the CPU: calls that once went wrong."""

import pytest
import torch

from nuvla_forge_b200.ops import logprobs as lp


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
