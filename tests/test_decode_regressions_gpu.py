"""Cached decoding and scores on the GPU: calls that once went wrong."""

import pytest
import torch

from nuvla_forge_b200.ops import logprobs as lp

pytestmark = pytest.mark.gpu
DEV = "cuda"


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
