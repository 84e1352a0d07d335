"""A NaN or an infinity in a key that a query sees: the same entries of the
output and of the gradients are finite as in the 64-bit form, wherever in a tile
the key lies."""
import math

import pytest
import torch

import tda_b200
from tests.sdiff_reference import attention64, rel
from tests.test_gpu_softmax_differential import OUT_TOL, make

pytestmark = pytest.mark.gpu

S, AT = 300, 32  # keys 32-63: for the rows from 128 on they lie in a tile that no mask cuts


def poisoned(dtype, D, index, bad, which, causal):
    xs, dout, lam = make(1, 2, 1, S, S, D, dtype, seed=index)
    xs[2 + which][0, 0, AT + index, 3] = bad
    return xs, dout, lam


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_forward(dtype, D, causal, bad):
    for index in range(32):
        for which in range(2):
            xs, _, lam = poisoned(dtype, D, index, bad, which, causal)
            out = tda_b200.differential_softmax_attention(*xs, lam, causal=causal)
            ref = attention64(*xs, lam, causal=causal)
            fine = torch.isfinite(ref)
            assert torch.equal(torch.isfinite(out), fine), (index, which)
            if fine.any():
                assert rel(out[fine], ref[fine]) <= OUT_TOL[dtype], (index, which)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scores_of_minus_infinity(dtype):
    """They have no weight, also where a whole tile of keys holds no other."""
    xs, _, lam = make(1, 1, 1, 140, 256, 64, dtype, seed=3)
    xs[0][..., 0] = 1.0
    xs[2][:, :, :200, 0] = -math.inf
    out = tda_b200.differential_softmax_attention(*xs, lam, causal=False)
    ref = attention64(*xs, lam, causal=False)
    assert torch.isfinite(out).all() and rel(out, ref) <= OUT_TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_queries_and_the_first_key(dtype, causal, bad):
    """Rows of nothing but NaN, a row whose only score is one, rows without a number at their maximum."""
    for tensor, row in ((0, 0), (0, 130), (1, 299), (2, 0), (3, 0), (3, 299)):
        xs, _, lam = make(1, 2, 1, S, S, 64, dtype, seed=row)
        xs[tensor][0, 0, row, 7] = bad
        out = tda_b200.differential_softmax_attention(*xs, lam, causal=causal)
        ref = attention64(*xs, lam, causal=causal)
        fine = torch.isfinite(ref)
        assert torch.equal(torch.isfinite(out), fine), (tensor, row)
        assert not fine.all()
        if fine.any():
            assert rel(out[fine], ref[fine]) <= OUT_TOL[dtype], (tensor, row)
