"""The cache attention serves: a gradient through it is refused, not left out."""
import pytest
import torch

import tda_b200
from tests.test_gpu_cache4 import filled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["softmax", "threshold"])
@pytest.mark.parametrize("wants", [0, 1, 2])
def test_backward_raises(form, wants):
    cache, table, lengths, _, q1, q2 = filled([5, 40], 4, 2, 64, 16, torch.bfloat16, 1, form == "threshold", poison=False)
    lam = torch.full((1, 4, 1, 1), 0.4, device="cuda")

    def call(a, b, l):
        if form == "softmax":
            return tda_b200.cache4_softmax_attention(a, b, cache, table, lengths, l)
        return tda_b200.cache4_threshold_attention(a, b, cache, table, lengths, 0.9, l)

    plain = call(q1, q2, lam)
    assert not plain.requires_grad
    xs = [q1, q2, lam]
    xs[wants] = xs[wants].clone().requires_grad_(True)
    out = call(*xs)
    assert out.requires_grad and torch.equal(out.detach(), plain)
    with pytest.raises(RuntimeError, match="no backward"):
        out.float().sum().backward()
    with torch.no_grad():
        assert not call(*xs).requires_grad
