"""Gradients where a key that queries see holds a NaN or an infinity: the same
entries are finite as in the 64-bit form, wherever in a tile the key lies."""
import math

import pytest
import torch

import tda_b200
from tests.sdiff_reference import attention64, rel
from tests.test_gpu_sdiff_nonfinite import poisoned
from tests.test_gpu_softmax_differential import GRAD_TOL, NAMES, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_backward(dtype, D, causal, bad):
    for index in range(32):
        which = index % 2
        xs, dout, lam = poisoned(dtype, D, index, bad, which, causal)
        leaves = [x.detach().requires_grad_(True) for x in xs]
        out = tda_b200.differential_softmax_attention(*leaves, lam, causal=causal)
        grads = torch.autograd.grad(out, leaves, dout)
        for name, g, r in zip(NAMES, grads, attention64(*xs, lam, causal=causal, dout=dout)[1:6]):
            fine = torch.isfinite(r)
            assert torch.equal(torch.isfinite(g), fine), (name, index)
            if fine.any():
                assert rel(g[fine], r[fine]) <= GRAD_TOL[dtype], (name, index)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_a_lone_key_that_is_nan(dtype, D, causal):
    """Its weight is not 1: the gradients of queries and keys are NaN there, and zeros for a lone key that is a number."""
    xs, dout, lam = make(3, 2, 1, 40, 40, D, dtype, seed=2)
    xs[2][1, 0, 0, 5] = math.nan
    lengths = torch.tensor([1, 1, 30], dtype=torch.int32, device="cuda")
    leaves = [x.detach().requires_grad_(True) for x in xs]
    out = tda_b200.differential_softmax_attention(*leaves, lam, causal=causal, key_lengths=lengths)
    grads = torch.autograd.grad(out, leaves, dout)
    for name, g, r in zip(NAMES, grads, attention64(*xs, lam, causal=causal, lengths=lengths, dout=dout)[1:6]):
        assert torch.equal(torch.isfinite(g), torch.isfinite(r)), name
        if name != "dv":
            assert float(g[0].abs().max()) == 0.0
