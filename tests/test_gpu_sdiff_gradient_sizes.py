"""fp16 gradients whose upstream gradient is far from 1, as a mean loss or a
scaled one gives it.

Tolerance: scaling dout by a power of two scales every gradient by it, so the
relative error that holds at N(0,1), GRAD_TOL, holds at any size, but for what
fp16 itself cannot hold of the result: the 64-bit gradient rounded once."""
import pytest
import torch

import tda_b200
from tests.sdiff_reference import attention64, rel
from tests.test_gpu_softmax_differential import GRAD_TOL, NAMES, make

pytestmark = pytest.mark.gpu

SHAPES = [
    # B, H, Hkv, Sq, Sk, D, causal, peak (factor on the queries: rows with a few large weights)
    (1, 4, 2, 256, 256, 64, True, 1.0),
    (2, 2, 1, 256, 256, 64, False, 4.0),
    (1, 2, 2, 300, 700, 128, True, 1.0),
    (1, 2, 1, 2048, 2048, 64, False, 1.0),
]


def check(xs, dout, lam, causal, scale=None):
    leaves = [x.detach().requires_grad_(True) for x in xs]
    l = lam.clone().requires_grad_(True)
    out = tda_b200.differential_softmax_attention(*leaves, l, scale, causal)
    grads = torch.autograd.grad(out, leaves + [l], dout)
    ref = attention64(*xs, lam, scale, causal, dout=dout)
    for name, g, r in zip(NAMES, grads, ref[1:6]):
        once = r.to(torch.float16)
        assert torch.isfinite(once).all()  # the case is one that fp16 holds
        assert torch.isfinite(g).all(), name
        assert rel(g, r) <= GRAD_TOL[torch.float16] + rel(once, r), (name, rel(g, r), rel(once, r))
    return grads


@pytest.mark.parametrize("size", [1e-2, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("shape", SHAPES)
def test_small(shape, size):
    B, H, Hkv, Sq, Sk, D, causal, peak = shape
    xs, dout, lam = make(B, H, Hkv, Sq, Sk, D, torch.float16, seed=Sk)
    xs[0], xs[1] = xs[0] * peak, xs[1] * peak
    check(xs, (dout.float() * size).half(), lam, causal)


@pytest.mark.parametrize("D", [64, 128])
def test_small_values(D):
    """dP is as small as the values are."""
    xs, dout, lam = make(1, 4, 2, 256, 256, D, torch.float16, seed=D)
    xs[4] = (xs[4].float() * 1e-3).half()
    check(xs, (dout.float() * 1e-2).half(), lam, True)


@pytest.mark.parametrize("size,value", [(1000.0, 16.0), (16.0, 1000.0)])
def test_large(size, value):
    """dS, near 1e5, is past what fp16 holds; no gradient is."""
    xs, dout, lam = make(1, 4, 2, 256, 256, 64, torch.float16, seed=5)
    for i in range(4):
        xs[i] = xs[i] * 8
    xs[4] = xs[4] * value
    check(xs, dout * size, 0.25 * lam, False, 0.125 / 64)


def test_heads_of_different_sizes():
    """Each kv head by its own size: one head's gradient does not cost another's."""
    xs, dout, lam = make(2, 4, 4, 256, 256, 64, torch.float16, seed=6)
    f = torch.tensor([100.0, 1e-4, 1.0, 1e-3], device="cuda")[None, :, None, None]
    g = torch.tensor([1.0, 1e-1], device="cuda")[:, None, None, None]
    dout = (dout.float() * f * g).half()
    leaves = [x.detach().requires_grad_(True) for x in xs]
    out = tda_b200.differential_softmax_attention(*leaves, lam)
    grads = torch.autograd.grad(out, leaves, dout)
    for name, gr, r in zip(NAMES, grads, attention64(*xs, lam, dout=dout)[1:6]):
        for b in range(2):
            for h in range(4):
                once = r[b, h].to(torch.float16)
                assert rel(gr[b, h], r[b, h]) <= GRAD_TOL[torch.float16] + rel(once, r[b, h]), (name, b, h)


@pytest.mark.parametrize("lam", [300.0, -300.0, 1e-3])
def test_lambda_of_any_size(lam):
    xs, dout, l = make(1, 2, 1, 200, 200, 64, torch.float16, seed=7)
    check(xs, (dout.float() * 1e-2).half(), torch.full_like(l, lam), True)


def test_many_small_weights():
    """dv where every weight is below 2^-14, fp16's least normal number: rows of 65536 keys."""
    xs, dout, lam = make(1, 1, 1, 256, 65536, 64, torch.float16, seed=8)
    leaves = [x.detach().requires_grad_(True) for x in xs]
    out = tda_b200.differential_softmax_attention(*leaves, lam, causal=False)
    (dv,) = torch.autograd.grad(out, leaves[4:], 64 * dout)
    r = attention64(*xs, lam, causal=False, dout=64 * dout)[5]
    assert rel(dv, r) <= GRAD_TOL[torch.float16] + rel(r.half(), r), rel(dv, r)


def test_large_scores_and_large_sums():
    """L of some 10^5 in units of the raw score, D of some 10^5: the other columns of the tables."""
    xs, dout, lam = make(1, 2, 1, 256, 256, 64, torch.float16, seed=3)
    for i in range(4):
        xs[i] = xs[i] * 32
    xs[4], dout = xs[4] * 30, dout * 300
    leaves = [x.detach().requires_grad_(True) for x in xs]
    scale = 2 * 0.125 / 1024
    out = tda_b200.differential_softmax_attention(*leaves, lam, scale)
    grads = torch.autograd.grad(out, leaves, dout)
    for name, g, r in list(zip(NAMES, grads, attention64(*xs, lam, scale, dout=dout)[1:6])):
        assert rel(g, r) <= GRAD_TOL[torch.float16] + rel(r.half(), r), (name, rel(g, r))
