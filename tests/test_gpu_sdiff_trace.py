"""Traced calls give the plain call's bits."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import tda_b200
from tests.test_gpu_softmax_differential import make

pytestmark = pytest.mark.gpu


def test_same_bits():
    xs, dout, lam = make(1, 2, 2, 200, 200, 64, torch.bfloat16, seed=14)
    fn = lambda *a: tda_b200.differential_softmax_attention(*a)
    want = fn(*xs, lam)
    torch._dynamo.reset()
    compiled = torch.compile(fn, fullgraph=True, backend="aot_eager")
    assert torch.equal(compiled(*xs, lam), want)
    assert torch.equal(make_fx(fn, tracing_mode="fake")(*xs, lam)(*xs, lam), want)
    leaves = [x.detach().requires_grad_(True) for x in xs]
    with torch.no_grad():
        assert torch.equal(compiled(*leaves, lam), want)
    out, o12, lse = torch.ops.tda.sdiff_fwd(*xs, lam, 0.125, True, None, False)
    assert torch.equal(out, want) and o12.numel() == lse.numel() == 0
    a = torch.autograd.grad(compiled(*leaves, lam), leaves, dout)
    b = torch.autograd.grad(fn(*leaves, lam), leaves, dout)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
