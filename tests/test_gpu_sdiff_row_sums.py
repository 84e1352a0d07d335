"""dk where the rows' sums D, subtracted inside the products in 16-bit pieces, are
small or large in themselves (fp16).

Rows are peaked (queries four times a normal variate), so that dS is no smaller
than fp16's normal numbers and D's own precision shows.  Tolerance: that of
gradients at N(0,1), which a power of two on dout does not change, and the
rounding of the result."""
import pytest
import torch

import tda_b200
from tests.sdiff_reference import attention64, rel
from tests.test_gpu_softmax_differential import GRAD_TOL, NAMES, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [1e-4, 1e-3, 1.0, 100.0])
@pytest.mark.parametrize("D,causal", [(64, False), (128, False), (64, True)])
def test_dk(D, causal, size):
    xs, dout, lam = make(2, 2, 1, 256, 256, D, torch.float16, seed=D)
    xs[0], xs[1] = xs[0] * 4, xs[1] * 4
    dout = (dout.float() * size).half()
    leaves = [x.detach().requires_grad_(True) for x in xs]
    out = tda_b200.differential_softmax_attention(*leaves, lam, causal=causal)
    grads = torch.autograd.grad(out, leaves, dout)
    for name, g, r in list(zip(NAMES, grads, attention64(*xs, lam, causal=causal, dout=dout)[1:6]))[2:4]:
        assert rel(g, r) <= GRAD_TOL[torch.float16] + rel(r.half(), r), (name, rel(g, r), rel(r.half(), r))
