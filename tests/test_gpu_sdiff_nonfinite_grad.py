"""Gradients where a key that queries see holds a NaN or an infinity: the same
entries are finite as in the 64-bit form, wherever in a tile the key lies."""
import math

import pytest
import torch

import tda_b200
from tests.sdiff_reference import attention64, rel
from tests.test_gpu_sdiff_nonfinite import poisoned
from tests.test_gpu_softmax_differential import GRAD_TOL, NAMES

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
